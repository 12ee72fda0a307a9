"""The rest bucket of ops.distill_topk* where the student's mass outside the teacher's ids is next to
nothing: whole rows, vocabulary parts and autograd against the formula in 64 bits, through logarithms."""
import pytest
import torch

import logits_oracle as oracle
from service_account_auth_improvements_amd import ops

BF16, FP16, F32 = torch.bfloat16, torch.float16, torch.float32
NEG = float("-inf")


def _exact(x, ids, z, temperature, lse):
    """(loss, gradient, size of the loss's terms, size of the gradient's) with o the softmax among the
    logits outside the ids and R their mass:  dx = o (W R - r) / temperature outside, (p W - q) / temperature
    inside.  Ids are distinct and all present."""
    T, V = x.shape
    x, z, lse = x.double() / temperature, z.double() / temperature, lse.double()[:, None]
    lp = torch.log_softmax(x, 1)
    inside = torch.zeros(T, V, dtype=torch.bool).scatter_(1, ids, True)
    out = x.masked_fill(inside, NEG)
    mo = out.amax(1, keepdim=True)
    none = torch.isneginf(mo)                                       # no mass outside
    d = torch.where(none, out, out - mo)
    lo = torch.log(torch.exp(d).sum(1, keepdim=True))               # logits at the type's lowest value cancel exactly
    top = x.amax(1, keepdim=True)
    lR = torch.where(none, NEG, mo - top + lo - torch.log(torch.exp(x - top).sum(1, keepdim=True)))
    lq = z - lse
    q = torch.exp(lq)
    r = (1 - q.sum(1, keepdim=True)).clamp(min=0)
    W = q.sum(1, keepdim=True) + r
    use = (r > 0) & ~none
    lpk = lp.gather(1, ids)
    part = torch.where(use, r * (torch.log(r) - lR), 0.0)
    loss = (torch.where(q != 0, q * (lq - lpk), 0.0)).sum(1) + part[:, 0]
    lsize = (torch.where(q != 0, q * (lq.abs() + lpk.abs()), 0.0)).sum(1) + torch.where(use, r * (torch.log(r).abs() + lR.abs()), 0.0)[:, 0]
    o = torch.where(none, 0.0, torch.exp(d - lo))
    ru = torch.where(use, r, 0.0)
    qs = torch.zeros(T, V).double().scatter_(1, ids, q)
    dx = torch.where(inside, lp.exp() * W - qs, o * (W * lR.exp() - ru)) / temperature
    size = torch.where(inside, lp.exp() * W + qs, o * (W * lR.exp() + ru)) / temperature
    return loss, dx, lsize, size


def _case(T, V, K, dtype, temperature, gaps, seed=0):
    """Row t: the ids' logits around 0, all others gaps[t] nats (after the temperature) below."""
    g = torch.Generator().manual_seed(seed)
    gap = torch.tensor([gaps[t % len(gaps)] for t in range(T)])[:, None]
    x = (torch.randn(T, V, generator=g) - gap) * temperature
    ids = torch.stack([torch.randperm(V, generator=g)[:K] for _ in range(T)])
    x.scatter_(1, ids, torch.randn(T, K, generator=g) * temperature)
    z = torch.randn(T, K, generator=g) * 2 * temperature
    lse = torch.logsumexp(z / temperature, 1) + 0.2                 # a rest of 0.18
    return x.to(dtype), ids, z, lse


def _hold(device, x, ids, z, temperature, lse, scale=1.0, far=300.0, cuts=None):
    V, dtype = x.shape[1], x.dtype
    rl, rd, lsize, size = _exact(x, ids, z, temperature, lse)
    lb = (1 + lsize) * 4 * oracle.sum_bound(V)
    gb = oracle.grad_bound(rd * scale, size * scale, far, V, dtype)
    x, ids, z, lse = (t.to(device) for t in (x, ids, z, lse))
    loss, d = ops.distill_topk_fused(x, ids, z, scale, temperature, lse)
    oracle.close(loss, rl, lb, "loss")
    oracle.close(d, rd * scale, gb, "dlogits")
    xv = x.clone().requires_grad_()
    lo = ops.distill_topk(xv, ids, z, temperature, lse)
    (da,) = torch.autograd.grad(lo, xv, torch.full((x.shape[0],), scale, device=device))
    oracle.close(lo, rl, lb, "autograd loss")
    oracle.close(da, rd * scale, gb, "autograd dlogits")
    cols = list(zip((0, *(cuts or (V // 3, V // 3 + 1))), (*(cuts or (V // 3, V // 3 + 1)), V)))
    st = torch.stack([ops.distill_topk_stats(x[:, a:b], ids, z, temperature, lse, a, V) for a, b in cols])
    joined = ops.distill_topk_join(st, temperature)
    for a, b in cols:
        lp, dp = ops.distill_topk_grad(x[:, a:b], ids, z, joined, scale, temperature, lse, a, V)
        oracle.close(lp, rl, 2 * lb, "parts' loss")                 # the parts' sums are scaled once more
        oracle.close(dp, rd[:, a:b] * scale, 2 * gb[:, a:b], "parts' dlogits")


GAPS = [20.0, 60.0, 80.0, 86.0, 88.0, 95.0, 104.0, 200.0]


def _outside_far_below(device, V, dtype, temperature, scale):
    x, ids, z, lse = _case(8, V, min(4, V - 1), dtype, temperature, GAPS)
    _hold(device, x, ids, z, temperature, lse, scale)


@pytest.mark.parametrize("V,dtype,temperature,scale", [(1000, F32, 1.0, 1.0), (1000, F32, 0.1, 256.0), (1000, BF16, 1.0, 65536.0),
                                                       (5, F32, 1.0, 1.0), (300, FP16, 0.05, 256.0), (3000, F32, 1e-4, 1.0)])
def test_outside_far_below(V, dtype, temperature, scale):
    _outside_far_below("cpu", V, dtype, temperature, scale)


@pytest.mark.gpu
@pytest.mark.parametrize("V,dtype,temperature,scale", [(1000, F32, 1.0, 1.0), (1000, F32, 0.1, 256.0), (1000, BF16, 1.0, 65536.0),
                                                       (5, F32, 1.0, 1.0), (300, FP16, 0.05, 256.0), (3000, F32, 1e-4, 1.0),
                                                       (40003, BF16, 1.0, 1.0), (128256, BF16, 0.1, 256.0), (150001, F32, 1.0, 65536.0)])
def test_outside_far_below_gpu(V, dtype, temperature, scale):
    _outside_far_below("cuda:0", V, dtype, temperature, scale)


def _borders(device, V):
    T, K = 6, 3
    x, ids, z, lse = _case(T, V, K, F32, 1.0, [40.0])
    inside = torch.zeros(T, V, dtype=torch.bool).scatter_(1, ids, True)
    low = torch.finfo(F32).min
    x[0] = torch.where(inside[0], x[0], NEG)                        # no mass outside: the rest is left out
    x[1] = torch.where(inside[1], x[1], low)                        # masked by the lowest value: next to none is some
    x[2] = torch.where(inside[2], x[2], NEG)                        # a single logit outside, 150 below
    x[2, int((~inside[2]).nonzero()[-1])] = -150.0
    x[3] = torch.where(inside[3], x[3] - 120.0, x[3] + 40.0)        # the student's mass is all outside
    x[4] = torch.where(inside[4], NEG, 0.0)
    x[4, ids[4]] = torch.tensor([0.0, -1.0, -2.0])
    x[5] = torch.where(inside[5], low, x[5])                        # every id at the lowest value
    x[5, ids[5, 0]] = 200.0
    z[5] = torch.tensor([0.0, NEG, NEG])                            # entries without mass there
    lse[5] = 1.0
    _hold(device, x, ids, z, 1.0, lse)


@pytest.mark.parametrize("V", [50, 700])
def test_borders_of_the_rest(V):
    _borders("cpu", V)


@pytest.mark.gpu
@pytest.mark.parametrize("V", [50, 700, 30001, 131081])
def test_borders_of_the_rest_gpu(V):
    _borders("cuda:0", V)


def test_gradient_by_differences():
    x, ids, z, lse = _case(2, 9, 3, F32, 1.0, [90.0, 110.0])
    x, step = x.double(), 1e-4
    num = torch.zeros(2, 9).double()
    for i in range(2):
        for j in range(9):
            e = torch.zeros_like(x)
            e[i, j] = step
            num[i, j] = (_exact(x + e, ids, z, 1.0, lse)[0] - _exact(x - e, ids, z, 1.0, lse)[0])[i] / (2 * step)
    _, d = ops.distill_topk_fused(x.float(), ids, z, 1.0, 1.0, lse)
    # the difference's own error is step^2, its rounding 1e-14 / step; x is rounded to fp32: 110 * 2^-24 on the logits
    oracle.close(d, num, 3e-5, "difference")


def _small_rest(device, V, dtype, zt, temperature):
    """Teachers that leave next to nothing, to students that have still less there: the outside's gradient
    is the rest's, and as exact as any other."""
    T, K = 6, 7
    x, ids, z, _ = _case(T, V, K, dtype, temperature, [25.0, 40.0])
    z = z.to(zt)
    full = torch.logsumexp(z.double() / temperature, 1)
    lse = (full + torch.tensor([1e-6, 1e-5, 1e-4, 3e-6, 1e-6, 0.0]).double()).float()
    lse[5] = float(full[5].float()) * (1 - 1e-6) if full[5] > 0 else float(full[5].float()) * (1 + 1e-6)    # entries above one: no rest
    _hold(device, x, ids, z, temperature, lse, far=80.0)


@pytest.mark.parametrize("V,dtype,zt,temperature", [(1000, F32, F32, 1.0), (300, BF16, BF16, 0.7), (5000, F32, FP16, 0.1)])
def test_small_rest(V, dtype, zt, temperature):
    _small_rest("cpu", V, dtype, zt, temperature)


@pytest.mark.gpu
@pytest.mark.parametrize("V,dtype,zt,temperature", [(1000, F32, F32, 1.0), (300, BF16, BF16, 0.7), (5000, F32, FP16, 0.1), (40000, BF16, F32, 1.3),
                                                    (150001, F32, BF16, 1.0)])
def test_small_rest_gpu(V, dtype, zt, temperature):
    _small_rest("cuda:0", V, dtype, zt, temperature)
