"""models.llama.TeacherLogits: distillation through the chunked LM head, the trainers, tensor
parallelism and context parallelism, against torch.autograd and one process.

Gradient tolerances are those of the label path's own tests (the same bf16 model around the head):
2.5 % of the greatest element on the CPU, 5 % on the GPU, 3 % between one and two ranks."""
import pytest
import torch

import logits_oracle as oracle
from dist_util import run_ranks
from service_account_auth_improvements_amd.models.llama import Llama, LlamaConfig, TeacherLogits
from service_account_auth_improvements_amd.models.llama_ref import _logits, _weights
from service_account_auth_improvements_amd.parallel.context import shard_tokens
from service_account_auth_improvements_amd.parallel.state import ParallelState


def _targets(B, S, V, K, lse=False, temp=1.0, seed=0, device="cpu", empty=True):
    g = torch.Generator().manual_seed(seed)
    ids = torch.stack([torch.randperm(V, generator=g)[:K] for _ in range(B * S)]).view(B, S, K)
    z = torch.randn(B, S, K, generator=g) * 2
    if empty:
        ids[:, S // 2] = -1               # tokens that are not trained on
        ids[0, 1, K // 2:] = -1
    L = torch.logsumexp(z / temp, -1) + 0.2 if lse else None
    return TeacherLogits(ids.to(device), z.to(device), temp, None if L is None else L.to(device))


def _reference(m, tok, t, scale):
    """Loss and gradients by autograd over the 64-bit formula's gradient of fp32 logits."""
    W = _weights(m, torch.float32)
    logits = _logits(m, tok, W, torch.float32).reshape(-1, m.cfg.vocab_size)
    f = t.reshape(-1)
    loss, dx, _, _ = oracle.distill(logits.detach().cpu(), f.ids.cpu(), f.logits.cpu(), f.temperature,
                                    None if f.lse is None else f.lse.cpu())
    logits.backward((dx * scale).float().to(logits.device))
    return float(loss.sum() * scale), W


def _check(m, W, tol):
    for n, w in W.items():
        g, r = m.G(n).float(), w.grad
        rel = ((g - r).abs().max() / r.abs().max().clamp_min(1e-8)).item()
        assert rel < tol, (n, rel)


@pytest.mark.parametrize("lse,temp", [(False, 1.0), (True, 2.0)])
def test_gradients_match_autograd(lse, temp):
    cfg = LlamaConfig.preset("tiny")
    m = Llama(cfg, ParallelState(), device="cpu", seed=3).allocate()
    m.head_chunk = 24                     # several chunks, the last one shorter
    B, S = 2, 32
    tok = torch.randint(0, cfg.vocab_size, (B, S), generator=torch.Generator().manual_seed(1))
    t = _targets(B, S, cfg.vocab_size, 12, lse, temp)
    loss = float(m.forward_backward(tok, t))
    ref, W = _reference(m, tok, t, 1.0 / (B * S))
    assert abs(loss - ref) < 1e-2 * ref
    _check(m, W, 2.5e-2)
    assert abs(float(m.forward_loss(tok, t)) - loss) < 1e-5 * abs(loss)


def test_one_sure_entry_is_the_label_loss():
    cfg = LlamaConfig.preset("tiny")
    tok, lab = torch.randint(0, cfg.vocab_size, (2, 2, 32), generator=torch.Generator().manual_seed(2))
    out = []
    for target in (lab, TeacherLogits(lab.unsqueeze(-1), torch.randn(2, 32, 1))):
        m = Llama(cfg, ParallelState(), device="cpu", seed=4).allocate()
        out.append((float(m.forward_backward(tok, target)), m.mats.grads.float().clone()))
    assert abs(out[0][0] - out[1][0]) < 1e-5 * out[0][0]
    # bf16 logit gradients that differ by a rounding now and then: 2^-8 of the greatest, through the backward pass
    assert (out[0][1] - out[1][1]).abs().max() < 2 ** -7 * out[0][1].abs().max()


def test_trainer_step_takes_teacher_micro_batches():
    from service_account_auth_improvements_amd.runtime.trainer import TrainConfig, Trainer
    V = LlamaConfig.preset("tiny").vocab_size
    toks = torch.randint(0, V, (2, 2, 32), generator=torch.Generator().manual_seed(5))
    ts = [_targets(2, 32, V, 6, True, 1.5, seed=s) for s in (1, 2)]
    tr = Trainer(TrainConfig(model="tiny", seq_len=32, lr=0.0, micro_batch=2, grad_accum=2), ParallelState())
    loss = float(tr.train_step([(toks[0], ts[0]), (toks[1], ts[1])]))
    got = tr.reduced_grads(tr.model.mats)
    big = Trainer(TrainConfig(model="tiny", seq_len=32, lr=0.0, micro_batch=4), ParallelState())
    both = TeacherLogits(torch.cat([t.ids for t in ts]), torch.cat([t.logits for t in ts]), 1.5, torch.cat([t.lse for t in ts]))
    ref = float(big.train_step([(toks.reshape(4, 32), both)]))
    want = big.reduced_grads(big.model.mats)
    assert abs(loss - ref) < 1e-3 * ref
    assert (got - want).abs().max() < 2e-2 * want.abs().max()


def test_targets_are_cut_like_labels():
    t = _targets(2, 8, 50, 3, True)
    assert t.shape == (2, 8) and t.numel() == 16
    half = shard_tokens(t, 2, 1)
    assert torch.equal(half.ids, t.ids[:, 4:]) and torch.equal(half.lse, t.lse[:, 4:]) and half.logits.is_contiguous()
    flat = t.reshape(-1)
    assert torch.equal(flat[3:5].logits, t.logits.reshape(16, 3)[3:5])
    for bad in ((t.ids, t.logits[..., :2], None), (t.ids[0, 0], t.logits[0, 0], None), (t.ids, t.logits, t.lse[:1])):
        if bad[0].dim() == 1:
            with pytest.raises(ValueError):
                TeacherLogits(bad[0], bad[1])
        else:
            with pytest.raises(ValueError):
                TeacherLogits(bad[0], bad[1], 1.0, bad[2])


def _tp_body(rank, world, lse):
    from service_account_auth_improvements_amd.parallel.state import init_distributed
    st = init_distributed(tp=world, pp=1, device="cpu")
    cfg = LlamaConfig.preset("tiny")
    m = Llama(cfg, st, device="cpu", seed=9, full_init=True).allocate()
    m.head_chunk = 40
    tok = torch.randint(0, cfg.vocab_size, (2, 32), generator=torch.Generator().manual_seed(3))
    loss = m.forward_backward(tok, _targets(2, 32, cfg.vocab_size, 10, lse, 1.3))
    return float(loss), {s.name: m.G(s.name).float().clone() for g in m.groups for s in g.specs}


@pytest.mark.parametrize("lse", [False, True])
def test_tensor_parallel_matches_one_rank(lse):
    cfg = LlamaConfig.preset("tiny")
    ref = Llama(cfg, ParallelState(), device="cpu", seed=9, full_init=True).allocate()
    tok = torch.randint(0, cfg.vocab_size, (2, 32), generator=torch.Generator().manual_seed(3))
    want = float(ref.forward_backward(tok, _targets(2, 32, cfg.vocab_size, 10, lse, 1.3)))
    for rank, (loss, grads) in enumerate(run_ranks(_tp_body, world=2, args=(lse,))):
        assert abs(loss - want) < 1e-2 * want
        sl = Llama(cfg, ParallelState(tp=2, tp_rank=rank), device="cpu", seed=9, full_init=True)._tp_slicers()
        for name, g in grads.items():
            r = ref.G(name).float()
            r = sl[name][1](r) if name in sl else r
            assert (g - r).abs().max() < 3e-2 * r.abs().max(), (rank, name)


def _cp_body(rank, world):
    from service_account_auth_improvements_amd.parallel.state import init_distributed
    from service_account_auth_improvements_amd.runtime.trainer import TrainConfig, Trainer
    st = init_distributed(tp=1, device="cpu")
    cfg = LlamaConfig.preset("tiny").with_(n_heads=4, n_kv_heads=2)
    tr = Trainer(TrainConfig(model="tiny", seq_len=64, micro_batch=2, lr=0.0, bucket_mb=1, context_parallel=True), st, mcfg=cfg,
                 full_init=True)
    tok = torch.randint(0, cfg.vocab_size, (2, 64), generator=torch.Generator().manual_seed(6))
    loss = tr.train_step([(tok, _targets(2, 64, cfg.vocab_size, 5, True))])
    return float(loss)


def test_context_parallel_losses_average_to_one_process():
    from service_account_auth_improvements_amd.runtime.trainer import TrainConfig, Trainer
    cfg = LlamaConfig.preset("tiny").with_(n_heads=4, n_kv_heads=2)
    tr = Trainer(TrainConfig(model="tiny", seq_len=64, micro_batch=2, lr=0.0), ParallelState(), mcfg=cfg, full_init=True)
    tok = torch.randint(0, cfg.vocab_size, (2, 64), generator=torch.Generator().manual_seed(6))
    want = float(tr.train_step([(tok, _targets(2, 64, cfg.vocab_size, 5, True))]))
    losses = run_ranks(_cp_body, world=2)
    assert abs(sum(losses) / 2 - want) < 5e-3 * want


@pytest.mark.gpu
@pytest.mark.parametrize("preset,S,K,lse", [("tiny", 128, 12, False), ("small", 256, 64, True)])
def test_gradients_match_autograd_gpu(preset, S, K, lse):
    cfg = LlamaConfig.preset(preset)
    m = Llama(cfg, ParallelState(device=torch.device("cuda:0")), device="cuda:0", seed=3).allocate()
    m.head_chunk = 100
    tok = torch.randint(0, cfg.vocab_size, (2, S), generator=torch.Generator().manual_seed(1)).cuda()
    t = _targets(2, S, cfg.vocab_size, K, lse, 1.5, device="cuda:0")
    loss = float(m.forward_backward(tok, t))
    ref, W = _reference(m, tok, t, 1.0 / (2 * S))
    assert abs(loss - ref) < 1e-2 * ref
    _check(m, W, 5e-2)
