"""64-bit oracles of the operators over logits, and the bounds their results are held to."""
import math

import torch

NEG, NAN = float("-inf"), float("nan")
EPS = 2.0 ** -24            # half a step of fp32


def softmax_parts(x, temperature):
    """x [T, V] any float -> (p, ln p) in 64 bits; a row of nothing but -inf, with +inf or NaN is NaN."""
    x = x.double() / temperature
    m = x.amax(1, keepdim=True) if x.shape[0] else x[:, :1]
    d = torch.where(torch.isfinite(m), x - m, x)          # logits at the type's lowest value cancel exactly
    lp = d - torch.log(torch.exp(d).sum(1, keepdim=True))
    gone = torch.isneginf(x).all(1) | torch.isposinf(x).any(1) | torch.isnan(x).any(1)
    lp = lp.masked_fill(gone[:, None], NAN)
    return lp.exp(), lp


def sum_bound(V):
    """Relative error, in fp32, of a row's sum of exponentials: one rounding per add of a thread's
    V / 256 terms at most and of the joins, and the exponential's own two steps."""
    return EPS * (V / 256 + 64)


def logprobs(x, tokens, temperature=1.0, top=0, ignore=-100):
    T, V = x.shape
    p, lp = softmax_parts(x, temperature)
    dead = tokens == ignore
    bad = ~dead & ((tokens < 0) | (tokens >= V))
    logp = lp.gather(1, tokens.clamp(0, V - 1)[:, None])[:, 0].masked_fill(bad, NAN).masked_fill(dead, 0.0)
    H = -torch.where(p == 0, p, p * lp).sum(1).masked_fill(dead, 0.0)
    order = torch.sort(x.double() + 0.0, dim=1, descending=True, stable=True).indices[:, :top]
    tlp = lp.gather(1, order).masked_fill(dead[:, None], 0.0)
    return logp, H, order.masked_fill(dead[:, None], -1), tlp


def logp_bound(ref, V):
    """|error| of a log-probability: the sum's, and four roundings of the distance to the maximum."""
    return sum_bound(V) + 4 * EPS * ref.abs().nan_to_num(0.0, 0.0, 0.0)


def entropy_bound(ref, V):
    """The sum's error enters ln s once and the weighted sum (of size H, twice) once more."""
    return 4 * sum_bound(V) * (1 + ref.abs().nan_to_num(0.0, 0.0, 0.0))


def logprobs_grad(x, tokens, g, h, temperature=1.0, ignore=-100):
    """(gradient, the size its roundings are measured against) in 64 bits."""
    T, V = x.shape
    p, lp = softmax_parts(x, temperature)
    H = -torch.where(p == 0, p, p * lp).sum(1, keepdim=True)
    g, h = g.double()[:, None], h.double()[:, None]
    l0 = torch.where(p == 0, torch.zeros_like(lp), lp)
    d = -g * p - h * p * (l0 + H)
    size = g.abs() * p + h.abs() * p * (l0.abs() + H)
    dead = (tokens == ignore)[:, None]
    bad = ~dead & ((tokens < 0) | (tokens >= V))[:, None]
    hit = torch.zeros_like(p).scatter_(1, tokens.clamp(0, V - 1)[:, None], 1.0)
    d = (d + g * hit) / temperature
    size = (size + g.abs() * hit) / temperature
    return d.masked_fill(bad, NAN).masked_fill(dead, 0.0), size.nan_to_num(0.0)


def grad_bound(ref, size, lp_max, V, dtype):
    """Half a step of the output's type on the value, the arithmetic's relative error (the sum's, and
    that of 2^y for |y| up to lp_max) on the terms' size, and what the type flushes to zero."""
    half = torch.finfo(dtype).eps / 2
    return ref.abs().nan_to_num(0.0) * half * 1.001 + 4 * (sum_bound(V) + EPS * (16 + 4 * lp_max)) * size + \
        torch.finfo(dtype).tiny * (half if dtype == torch.float16 else 1.0)


def distill(x, ids, z, temperature=1.0, lse=None):
    """(loss rows, gradient rows, size of the gradient's terms, size of the loss's terms) in 64 bits."""
    T, V = x.shape
    p, lp = softmax_parts(x, temperature)
    ids = ids.long()
    loss, dx, size = torch.zeros(T).double(), torch.zeros(T, V).double(), torch.zeros(T, V).double()
    lsize = torch.zeros(T).double()
    for t in range(T):
        ent = [(int(i), float(v)) for i, v in zip(ids[t], z[t].double()) if i >= 0]
        if any(i >= V for i, _ in ent):
            loss[t], dx[t] = NAN, NAN
            continue
        v = torch.tensor([e[1] for e in ent]).double() / temperature
        if lse is None:
            if not ent or torch.isneginf(v).all():
                continue
            lq = v - v.max() - torch.log(torch.exp(v - v.max()).sum())
            r = 0.0
        else:
            lq = v - float(lse[t])
            r = max(0.0, 1.0 - float(lq.exp().sum()))
            if not ent or bool((lq.exp() == 0).all()):
                continue
        q = lq.exp()
        at = torch.tensor([e[0] for e in ent])
        inside = torch.zeros(V, dtype=torch.bool)
        inside[at] = True
        use = q != 0
        loss[t] = (q * (lq - lp[t, at]))[use].sum()
        lsize[t] = (q * (lq.abs() + lp[t, at].abs()))[use].sum()
        R = float(p[t][~inside].sum())
        W = float(q.sum()) + r
        k = torch.full((V,), W).double()
        if r > 0 and R != 0:
            loss[t] += r * (math.log(r) - (math.log(R) if R == R else NAN))
            lsize[t] += r * (abs(math.log(r)) + abs(math.log(R) if R == R else 0))
            k[~inside] -= r / R
        qs = torch.zeros(V).double().index_add_(0, at, q)
        dx[t] = (p[t] * k - qs) / temperature
        size[t] = (p[t] * (W + (k - W).abs()) + qs) / temperature
    return loss, dx, size.nan_to_num(0.0), lsize.nan_to_num(0.0, 0.0, 0.0)


def close(got, ref, bound, what):
    """Equal infinities and NaN in the same places, the rest within ``bound``."""
    got, ref = got.detach().double().cpu(), ref.double().cpu()
    bound = bound.double().cpu() if torch.is_tensor(bound) else torch.full_like(ref, bound)
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    fin = torch.isfinite(ref)
    assert torch.equal(torch.isfinite(got), fin), (what, "finite in other places")
    assert torch.equal(torch.isnan(got), torch.isnan(ref)), (what, "NaN in other places")
    inf = torch.isinf(ref)
    assert torch.equal(got[inf], ref[inf]), what
    err = (got - ref).abs()[fin]
    over = err - bound.expand_as(ref)[fin]
    if err.numel():
        i = int(over.argmax())
        assert over[i] <= 0, (what, f"off by {err[i]:.3e}, bound {(err - over)[i]:.3e}, value {ref[fin][i]:.6g}")
