"""Calls of the operators over logits at the limits of what they take: no rows, the longest rows, a
launch that fails, and outputs over inputs."""
import ctypes

import pytest
import torch

import logits_oracle as oracle
from service_account_auth_improvements_amd import ops
from service_account_auth_improvements_amd.ops import _ext


def _no_rows(device, V, lse):
    x = torch.zeros(0, V, dtype=torch.bfloat16, device=device)
    ids, z = torch.zeros(0, 3, dtype=torch.long, device=device), torch.zeros(0, 3, device=device)
    L = torch.zeros(0, device=device) if lse else None
    loss, d = ops.distill_topk_fused(x, ids, z, 1.0, 1.0, L)
    assert loss.shape == (0,) and d.shape == (0, V)
    st = ops.distill_topk_stats(x, ids, z, 1.0, L)
    assert st.shape[0] == 0
    loss, d = ops.distill_topk_grad(x, ids, z, ops.distill_topk_join(st[None]), 1.0, 1.0, L)
    assert loss.shape == (0,) and d.shape == (0, V)
    xv = x.clone().requires_grad_()
    (d,) = torch.autograd.grad(ops.distill_topk(xv, ids, z, 1.0, L), xv, torch.zeros(0, device=device))
    assert d.shape == (0, V)
    xv, tok = x.clone().requires_grad_(), torch.zeros(0, dtype=torch.long, device=device)
    logp, ent, top, tlp = ops.token_logprobs(xv, tok, 1.0, min(2, V))
    (d,) = torch.autograd.grad([logp, ent], xv, [torch.zeros(0, device=device)] * 2)
    assert d.shape == (0, V) and top.shape == tlp.shape == (0, min(2, V))


@pytest.mark.parametrize("lse", [False, True])
@pytest.mark.parametrize("V", [1, 100])
def test_no_rows(V, lse):
    _no_rows("cpu", V, lse)


@pytest.mark.gpu
@pytest.mark.parametrize("lse", [False, True])
@pytest.mark.parametrize("V", [1, 100, 300001])
def test_no_rows_gpu(V, lse):
    _no_rows("cuda:0", V, lse)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("V", [491519, 491520])
def test_longest_rows_with_a_teacher_lse(V, dtype):
    g = torch.Generator().manual_seed(V)
    x = (torch.randn(2, V, generator=g) * 2).to(dtype)
    ids = torch.cat([torch.randint(0, V - 1, (2, 63), generator=g).sort(1).values, torch.full((2, 1), V - 1)], 1)
    z = torch.randn(2, 64, generator=g) + 4
    lse = torch.logsumexp(z, 1) + 0.3
    rl, rd, size, lsize = oracle.distill(x, ids, z, 1.0, lse)
    loss, d = ops.distill_topk_fused(x.cuda(), ids.cuda(), z.cuda(), 1.0, 1.0, lse.cuda())
    oracle.close(loss, rl, (1 + lsize) * 4 * oracle.sum_bound(V), "loss")
    oracle.close(d, rd, oracle.grad_bound(rd, size, 60.0, V, dtype), "dlogits")


@pytest.mark.skipif(torch.cuda.is_available(), reason="launches with null pointers, which only fail where there is no device")
def test_a_launch_that_fails_is_returned():
    lib = ctypes.CDLL(str(_ext.lib_path()))
    n, L, I, F, D = ctypes.c_void_p(0), ctypes.c_long, ctypes.c_int, ctypes.c_float, ctypes.c_double
    assert lib.kf_token_logprobs(n, I(0), L(64), L(1), I(64), n, L(-100), F(1), n, n, n, I(0), n, n, n, n) >= 1000
    assert lib.kf_token_logprobs_bwd(n, I(0), L(64), n, L(64), L(1), I(64), n, L(-100), n, n, n, n, F(1), n) >= 1000
    for mode, V in ((0, 64), (0, 4), (1, 64), (2, 64)):
        stats = (ctypes.c_float * 16)()
        assert lib.kf_distill_topk(n, I(0), L(V), n, L(V), L(1), I(V), L(0), L(V), n, I(0), L(1), n, I(0), L(1), n, I(1), D(1), n, F(1), n, n,
                                   stats, I(mode), n) >= 1000
    # nothing to launch
    assert lib.kf_token_logprobs(n, I(0), L(64), L(0), I(64), n, L(-100), F(1), n, n, n, I(0), n, n, n, n) == 0


@pytest.mark.gpu
def test_out_over_another_input_is_refused():
    T, V, K = 4, 128, 5
    buf = torch.zeros(T, V + 8, device="cuda")
    x, beside = buf[:, :V], buf[:, V:V + K]
    other = torch.zeros(T, V, device="cuda")
    ids, z = torch.arange(K, device="cuda").repeat(T, 1), torch.randn(T, K, device="cuda")
    f, st, tok = torch.zeros(T, device="cuda"), torch.zeros(T, 2, device="cuda"), torch.zeros(T, dtype=torch.long, device="cuda")
    stats = ops.distill_topk_stats(x, ids, z)
    n = stats.shape[1]
    flat = other.view(-1)
    whole = flat.view(torch.int64)
    refused = {
        "teacher logits": lambda: ops.distill_topk_fused(x, ids, x[:, :K], 1.0, out=x),
        "teacher logits,": lambda: ops.distill_topk_fused(x, ids, other[:, 3:3 + K], 1.0, out=other),
        "ids": lambda: ops.distill_topk_fused(x, whole[:T * K].view(T, K), z, 1.0, out=other),
        "lse": lambda: ops.distill_topk_fused(x, ids, z, 1.0, 1.0, flat[-T:], out=other),
        "scale": lambda: ops.distill_topk_fused(x, ids, z, flat[7:8], out=other),
        "stats": lambda: ops.distill_topk_grad(x, ids, z, flat[:T * n].view(T, n), 1.0, out=other),
        "tokens": lambda: ops.token_logprobs_bwd(x, whole[:T], st, f, f, out=other),
        "stats,": lambda: ops.token_logprobs_bwd(x, tok, flat[:2 * T].view(T, 2), f, f, out=other),
        "entropy": lambda: ops.token_logprobs_bwd(x, tok, st, flat[:T], f, out=other),
        "dlogp": lambda: ops.token_logprobs_bwd(x, tok, st, f, flat[:T], out=other),
        "dentropy": lambda: ops.token_logprobs_bwd(x, tok, st, f, f, flat[:T], out=other),
    }
    for name, call in refused.items():
        with pytest.raises(RuntimeError, match="out overlaps the " + name.rstrip(",")):
            call()
    # beside the logits in one buffer, and the logits themselves: taken
    beside.copy_(z)
    x.normal_(generator=torch.Generator("cuda").manual_seed(0))
    want = ops.distill_topk_fused(x, ids, z, 1.0)
    got = ops.distill_topk_fused(x, ids, beside, 1.0, out=x)
    assert torch.equal(got[0], want[0]) and torch.equal(x, want[1]) and torch.equal(beside, z)
