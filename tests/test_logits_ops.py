"""ops.token_logprobs* and ops.distill_topk* on the CPU: their fp32 reference against the 64-bit
oracle and against differences, refusals, and a vocabulary in parts."""
import pytest
import torch

import logits_oracle as oracle
from service_account_auth_improvements_amd import ops

F32 = torch.float32


def _x(T, V, dtype=F32, seed=0, spread=3.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(T, V, generator=g) * spread).to(dtype)


def _tok(T, V, seed=1):
    return torch.randint(0, V, (T,), generator=torch.Generator().manual_seed(seed))


@pytest.mark.parametrize("T,V,dtype,temp,top", [(1, 1, F32, 1.0, 1), (5, 37, torch.bfloat16, 0.7, 8), (4, 300, torch.float16, 2.0, 20),
                                                (3, 5000, F32, 1.0, 128), (0, 11, F32, 1.0, 3)])
def test_logprobs_reference(T, V, dtype, temp, top):
    x, tok = _x(T, V, dtype), _tok(T, V)
    if T > 2:
        tok[1] = -100
        x[2, ::3] = float("-inf")
        x[2, int(tok[2])] = 1.0
    logp, ent, stats, ids, tlp = ops.token_logprobs_fwd(x, tok, temp, top)
    rl, rh, ri, rt = oracle.logprobs(x, tok, temp, top)
    oracle.close(logp, rl, oracle.logp_bound(rl, V), "logp")
    oracle.close(ent, rh, oracle.entropy_bound(rh, V), "entropy")
    assert torch.equal(ids, ri)
    oracle.close(tlp, rt, oracle.logp_bound(rt, V), "top")
    g, h = torch.randn(T), torch.randn(T)
    d = ops.token_logprobs_bwd(x, tok, stats, ent, g, h, temp)
    ref, size = oracle.logprobs_grad(x, tok, g, h, temp)
    oracle.close(d, ref, oracle.grad_bound(ref, size, 60.0, V, dtype), "dlogits")


def test_logprobs_gradient_by_differences():
    x, tok = _x(3, 9).double(), _tok(3, 9)

    def f(v):
        logp, H, _, _ = oracle.logprobs(v, tok, 1.5)
        return (logp * torch.tensor([1.0, -2.0, 0.5]) + H * torch.tensor([0.3, 0.1, -0.7])).sum()
    step, num = 1e-5, torch.zeros(3, 9).double()
    for i in range(3):
        for j in range(9):
            e = torch.zeros_like(x)
            e[i, j] = step
            num[i, j] = (f(x + e) - f(x - e)) / (2 * step)
    xv = x.float().requires_grad_()
    logp, ent, _, _ = ops.token_logprobs(xv, tok, 1.5)
    (d,) = torch.autograd.grad([logp, ent], xv, [torch.tensor([1.0, -2.0, 0.5]), torch.tensor([0.3, 0.1, -0.7])])
    # x is rounded to fp32 (relative 2^-24, second derivatives of order 10) and the difference is of order step^2
    oracle.close(d, num, 1e-5, "difference")


def _teacher(T, V, K, seed=2, lse=False, temp=1.0):
    g = torch.Generator().manual_seed(seed)
    ids = torch.stack([torch.randperm(V, generator=g)[:K] for _ in range(T)]) if T else torch.zeros(0, K, dtype=torch.long)
    z = torch.randn(T, K, generator=g) * 2
    return ids, z, (torch.logsumexp(z / temp, 1) + 0.1 if lse else None)


@pytest.mark.parametrize("lse", [False, True])
@pytest.mark.parametrize("T,V,K,temp", [(6, 50, 7, 1.0), (4, 2000, 64, 2.5), (3, 5, 5, 1.0), (0, 9, 2, 1.0), (2, 300, 256, 0.5)])
def test_distill_reference(T, V, K, temp, lse):
    x = _x(T, V)
    ids, z, L = _teacher(T, V, K, lse=lse, temp=temp)
    if T > 3:
        ids[1] = -1                       # a row without entries
        ids[2, 3:] = -1
        ids[3, 1] = ids[3, 0]             # the same id twice
    loss, d = ops.distill_topk_fused(x, ids, z, 0.5, temp, L)
    rl, rd, size, lsize = oracle.distill(x, ids, z, temp, L)
    oracle.close(loss, rl, (1 + lsize) * 4 * oracle.sum_bound(V), "loss")
    oracle.close(d, rd * 0.5, oracle.grad_bound(rd * 0.5, size * 0.5, 60.0, V, F32), "dlogits")
    xv = x.clone().requires_grad_()
    rows = torch.rand(T)
    lo = ops.distill_topk(xv, ids, z, temp, L)
    (da,) = torch.autograd.grad(lo, xv, rows)
    oracle.close(lo, rl, (1 + lsize) * 4 * oracle.sum_bound(V), "autograd loss")
    oracle.close(da, rd * rows[:, None], oracle.grad_bound(rd, size, 60.0, V, F32), "autograd dlogits")


def test_distill_gradient_by_differences():
    x = _x(2, 11).double()
    ids, z, L = _teacher(2, 11, 4, lse=True)
    step, num = 1e-5, torch.zeros(2, 11).double()
    f = lambda v: oracle.distill(v, ids, z, 1.0, L)[0].sum()          # noqa: E731
    for i in range(2):
        for j in range(11):
            e = torch.zeros_like(x)
            e[i, j] = step
            num[i, j] = (f(x + e) - f(x - e)) / (2 * step)
    _, d = ops.distill_topk_fused(x.float(), ids, z, 1.0, 1.0, L)
    oracle.close(d, num, 1e-5, "difference")


@pytest.mark.parametrize("lse", [False, True])
@pytest.mark.parametrize("cuts", [(0, 40, 97), (0, 1, 97), (0, 30, 31, 97)])
def test_distill_in_vocabulary_parts(cuts, lse):
    V, temp = 97, 1.7
    x = _x(5, V)
    x[4, :cuts[1]] = float("-inf")        # a part without any mass
    ids, z, L = _teacher(5, V, 9, lse=lse, temp=temp)
    ids[0, 2:] = -1
    ids[1] = -1
    ids[4] = torch.arange(V - 9, V)
    whole, dw = ops.distill_topk_fused(x, ids, z, 2.0, temp, L)
    parts = list(zip(cuts[:-1], cuts[1:]))
    st = [ops.distill_topk_stats(x[:, a:b].contiguous(), ids, z, temp, L, a, V) for a, b in parts]
    joined = ops.distill_topk_join(torch.stack(st), temp)
    for a, b in parts:
        loss, d = ops.distill_topk_grad(x[:, a:b].contiguous(), ids, z, joined, 2.0, temp, L, a, V)
        oracle.close(loss, whole, 64 * oracle.EPS * (1 + whole.abs()), "loss")
        oracle.close(d, dw[:, a:b], 64 * oracle.EPS * (1 + dw[:, a:b].abs()), "dlogits")


def test_entry_in_a_part_of_nothing_but_minus_infinity():
    x = _x(2, 20)
    x[0, :8] = float("-inf")
    ids, z = torch.tensor([[3, 12], [3, 12]]), torch.zeros(2, 2)
    whole, dw = ops.distill_topk_fused(x, ids, z, 1.0)
    st = torch.stack([ops.distill_topk_stats(x[:, a:b].contiguous(), ids, z, 1.0, None, a, 20) for a, b in ((0, 8), (8, 20))])
    for a, b in ((0, 8), (8, 20)):
        loss, d = ops.distill_topk_grad(x[:, a:b].contiguous(), ids, z, ops.distill_topk_join(st), 1.0, 1.0, None, a, 20)
        oracle.close(loss, whole, 64 * oracle.EPS * (1 + whole[1].abs()), "loss")
        oracle.close(d, dw[:, a:b], 64 * oracle.EPS, "dlogits")
    assert whole[0] == float("inf")


def test_overwritten_logits_are_noticed_by_autograd():
    x, tok = _x(2, 9), _tok(2, 9)
    xv = (x.clone().requires_grad_() * 1.0)
    logp, ent, _, _ = ops.token_logprobs(xv, tok)
    with torch.no_grad():
        _, _, st, _, _ = ops.token_logprobs_fwd(xv, tok)
        ops.token_logprobs_bwd(xv, tok, st, ent.detach(), torch.ones(2), out=xv)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        logp.sum().backward()


def test_distill_border_rows():
    # everything covered; student without mass outside; student without mass at an entry; id behind the end
    x = torch.zeros(4, 6)
    x[1, 3:] = float("-inf")
    x[2, 0] = float("-inf")
    ids = torch.tensor([[0, 1, 2, 3, 4, 5], [0, 1, 2, -1, -1, -1], [0, 1, -1, -1, -1, -1], [6, 0, 1, -1, -1, -1]])
    z = torch.randn(4, 6, generator=torch.Generator().manual_seed(0))
    zz = z.masked_fill(ids < 0, float("-inf"))
    loss, d = ops.distill_topk_fused(x, ids, z, 1.0, 1.0, torch.logsumexp(zz, 1) + 1e-3)
    assert torch.isfinite(loss[:2]).all() and torch.isfinite(d[:3]).all()
    assert loss[2] == float("inf") and torch.isnan(loss[3]) and torch.isnan(d[3]).all()


REFUSALS = {
    "integer logits": lambda k: k["lp"](k["x"].long(), k["tok"]),
    "fp64 logits": lambda k: k["lp"](k["x"].double(), k["tok"]),
    "1-D logits": lambda k: k["lp"](k["x"][0], k["tok"]),
    "no vocabulary": lambda k: k["lp"](k["x"][:, :0], k["tok"]),
    "inner stride": lambda k: k["lp"](k["x"][:, ::2], k["tok"]),
    "int32 tokens": lambda k: k["lp"](k["x"], k["tok"].int()),
    "token count": lambda k: k["lp"](k["x"], k["tok"][:2]),
    "top negative": lambda k: k["lp"](k["x"], k["tok"], 1.0, -1),
    "top above V": lambda k: k["lp"](k["x"], k["tok"], 1.0, 41),
    "top above 128": lambda k: k["lp"](torch.cat([k["x"]] * 5, 1), k["tok"], 1.0, 129),
    "temperature 0": lambda k: k["lp"](k["x"], k["tok"], 0.0),
    "temperature NaN": lambda k: k["lp"](k["x"], k["tok"], float("nan")),
    "temperature negative": lambda k: k["lp"](k["x"], k["tok"], -1.0),
    "stats shape": lambda k: k["bwd"](k["x"], k["tok"], k["f"], k["f"], k["f"]),
    "upstream type": lambda k: k["bwd"](k["x"], k["tok"], k["st"], k["f"], k["f"].half()),
    "upstream stride": lambda k: k["bwd"](k["x"], k["tok"], k["st"], k["f"], k["f"][:1].expand(3)),
    "out type": lambda k: k["bwd"](k["x"], k["tok"], k["st"], k["f"], k["f"], out=k["x"].half()),
    "out shape": lambda k: k["bwd"](k["x"], k["tok"], k["st"], k["f"], k["f"], out=k["x"][:2]),
    "out rows shared": lambda k: k["bwd"](k["x"], k["tok"], k["st"], k["f"], k["f"], out=k["x"][:1].expand(3, 40)),
    "ids type": lambda k: k["kd"](k["x"], k["ids"].short(), k["z"], 1.0),
    "ids rows": lambda k: k["kd"](k["x"], k["ids"][:2], k["z"], 1.0),
    "ids stride": lambda k: k["kd"](k["x"], k["ids"][:, ::2], k["z"][:, :2], 1.0),
    "teacher shape": lambda k: k["kd"](k["x"], k["ids"], k["z"][:, :2], 1.0),
    "teacher type": lambda k: k["kd"](k["x"], k["ids"], k["z"].double(), 1.0),
    "too many entries": lambda k: k["kd"](k["x"], k["ids"][:, :1].repeat(1, 257), k["z"][:, :1].repeat(1, 257), 1.0),
    "lse type": lambda k: k["kd"](k["x"], k["ids"], k["z"], 1.0, 1.0, k["f"].half()),
    "lse length": lambda k: k["kd"](k["x"], k["ids"], k["z"], 1.0, 1.0, k["f"][:2]),
    "scale of two": lambda k: k["kd"](k["x"], k["ids"], k["z"], k["f"][:2]),
    "scale type": lambda k: k["kd"](k["x"], k["ids"], k["z"], k["f"][:1].half()),
    "part behind the vocabulary": lambda k: k["st_"](k["x"], k["ids"], k["z"], 1.0, None, 10, 49),
    "part before the vocabulary": lambda k: k["st_"](k["x"], k["ids"], k["z"], 1.0, None, -1, 49),
    "joined statistics": lambda k: k["gr"](k["x"], k["ids"], k["z"], k["st"], 1.0),
    "rest over a long row": lambda k: k["kd"](k["f"][:1].expand(3, 1)[:, :1].to(torch.bfloat16).repeat(1, 491521), k["ids"], k["z"], 1.0, 1.0,
                                              k["f"]),
}


def refusal_args(device):
    g = torch.Generator().manual_seed(0)
    x = torch.randn(3, 40, generator=g).to(device)
    return {"x": x, "tok": torch.tensor([0, 1, 2], device=device), "f": torch.zeros(3, device=device), "st": torch.zeros(3, 2, device=device),
            "ids": torch.randint(0, 40, (3, 4), generator=g).to(device), "z": torch.randn(3, 4, generator=g).to(device),
            "lp": ops.token_logprobs_fwd, "bwd": ops.token_logprobs_bwd, "kd": ops.distill_topk_fused,
            "st_": ops.distill_topk_stats, "gr": ops.distill_topk_grad}


@pytest.mark.parametrize("what", sorted(REFUSALS))
def test_refusals(what):
    with pytest.raises(RuntimeError, match="token_logprobs|distill_topk"):
        REFUSALS[what](refusal_args("cpu"))
