"""Plain-PyTorch fp32 reference implementations of every kernel in ``ops/csrc``.

They define the semantics the HIP kernels are tested against (numerics tests compare the
gfx950 kernel to these on the same inputs) and they serve CPU tensors in CPU-only tests
(the gloo multi-process tests of the parallel engines run the model through them).
"""
from __future__ import annotations

import math

import torch
import torch.nn.functional as F


def rmsnorm_fwd(a, b, w, eps):
    """Returns (y, h, rstd) with h = a + b (rounded to a's dtype) or h = a."""
    h = a if b is None else (a.float() + b.float()).to(a.dtype)
    hf = h.float()
    rstd = torch.rsqrt(hf.pow(2).mean(-1) + eps)
    y = (hf * rstd.unsqueeze(-1) * w.float()).to(a.dtype)
    return y, (h if b is not None else h.new_empty(0)), rstd.reshape(-1)


def rmsnorm_bwd(dy, h, rstd, w, dres=None):
    """Returns (dh, dw) in fp32 math, dh cast to h.dtype, dw fp32."""
    H = h.shape[-1]
    hf = h.float().reshape(-1, H)
    dyf = dy.float().reshape(-1, H)
    r = rstd.reshape(-1, 1).float()
    g = dyf * w.float()
    dot = (g * hf).sum(-1, keepdim=True)
    dh = r * g - hf * (r ** 3) * dot / H
    if dres is not None:
        dh = dh + dres.float().reshape(-1, H)
    dw = (dyf * hf * r).sum(0)
    return dh.to(h.dtype).reshape(h.shape), dw


def rope_tables(max_pos: int, head_dim: int, theta: float = 500000.0, device=None):
    """fp32 cos/sin tables [max_pos, head_dim/2] computed in fp64 (Llama-3 RoPE)."""
    inv = 1.0 / (theta ** (torch.arange(0, head_dim, 2, dtype=torch.float64) / head_dim))
    t = torch.arange(max_pos, dtype=torch.float64)
    f = torch.outer(t, inv)
    return f.cos().float().to(device), f.sin().float().to(device)


def rope_(x, nheads, head_dim, cos_t, sin_t, pos=None, seq_len=None, inverse=False):
    """In-place half-split rotary on the first nheads*head_dim columns of x [T, C]."""
    T = x.shape[0]
    p = pos.long() if pos is not None else torch.arange(T, device=x.device) % seq_len
    c = cos_t[p].unsqueeze(1)  # [T,1,D/2]
    s = sin_t[p].unsqueeze(1)
    if inverse:
        s = -s
    v = x[:, : nheads * head_dim].float().reshape(T, nheads, head_dim)
    a, b = v[..., : head_dim // 2], v[..., head_dim // 2:]
    out = torch.cat([a * c - b * s, b * c + a * s], dim=-1)
    x[:, : nheads * head_dim] = out.reshape(T, nheads * head_dim).to(x.dtype)
    return x


def swiglu_fwd(gu):
    F_ = gu.shape[-1] // 2
    g, u = gu[..., :F_].float(), gu[..., F_:].float()
    return (F.silu(g) * u).to(gu.dtype)


def swiglu_bwd(gu, dout):
    F_ = gu.shape[-1] // 2
    g, u = gu[..., :F_].float(), gu[..., F_:].float()
    d = dout.float()
    s = torch.sigmoid(g)
    du = d * g * s
    dg = d * u * s * (1 + g * (1 - s))
    return torch.cat([dg, du], dim=-1).to(gu.dtype)


def cross_entropy(logits, labels, ignore_index=-100, scale=None):
    """Returns (loss_rows fp32, lse fp32, dlogits fp32) for mean-style scaling `scale`."""
    lf = logits.float()
    lse = torch.logsumexp(lf, dim=-1)
    valid = labels != ignore_index
    safe = labels.clamp(min=0)
    xy = lf.gather(1, safe.unsqueeze(1)).squeeze(1)
    loss = torch.where(valid, lse - xy, torch.zeros_like(lse))
    if scale is None:
        scale = 1.0 / max(int(valid.sum()), 1)
    p = torch.softmax(lf, dim=-1)
    p[torch.arange(p.shape[0], device=p.device)[valid], safe[valid]] -= 1.0
    p = p * scale
    p[~valid] = 0
    return loss, lse, p


FLOATS = (torch.bfloat16, torch.float16, torch.float32)
TOP_MAX, DISTILL_K_MAX, DISTILL_REST_V_MAX = 128, 256, 491520    # the GPU kernels' limits


def _need(ok, msg):
    if not ok:
        raise RuntimeError(msg)


def _check_logits(x, temperature, op):
    _need(x.dtype in FLOATS, f"{op}: logits must be bfloat16, float16 or float32")
    _need(x.dim() == 2 and x.shape[1] >= 1 and (x.shape[1] == 1 or x.stride(1) == 1),
          f"{op}: logits must be [T, V] with V >= 1 and unit inner stride")
    _need(1e-4 <= temperature <= 1e4, f"{op}: temperature must be between 1e-4 and 1e4")


def _check_tokens(tokens, x, op):
    _need(tokens.device == x.device and tokens.dtype == torch.int64 and tuple(tokens.shape) == (x.shape[0],),
          f"{op}: tokens must be int64 [T] on the logits' device")


def _check_rows(t, x, tail, op, name):
    _need(t.device == x.device and t.dtype == torch.float32 and t.is_contiguous()
          and tuple(t.shape) == (x.shape[0], *tail), f"{op}: {name} must be contiguous float32 on the logits' device")


def _check_out(out, x, op):
    _need(out.device == x.device and out.dtype == x.dtype and out.shape == x.shape
          and (x.shape[1] == 1 or out.stride(1) == 1) and (x.shape[0] <= 1 or out.stride(0) >= x.shape[1]),
          f"{op}: out must have the logits' type, shape and device, unit inner stride and rows of their own")


def token_logprobs(logits, tokens, temperature=1.0, top=0, ignore_index=-100):
    """(logp, entropy, stats [T, 2] = (max, log2 of the sum), top ids, top logp): ops.token_logprobs_fwd."""
    op = "token_logprobs"
    _check_logits(logits, temperature, op)
    _need(0 <= top <= min(TOP_MAX, logits.shape[1]), f"{op}: top must be 0 to {TOP_MAX} and at most V")
    _check_tokens(tokens, logits, op)
    V = logits.shape[1]
    x = logits.float()
    m = x.amax(1, keepdim=True)
    d = x - m
    e = torch.exp(d / temperature)
    s = e.sum(1, keepdim=True)
    logs = torch.log(s)
    lp = d / temperature - logs
    dead = tokens == ignore_index
    bad = ~dead & ((tokens < 0) | (tokens >= V))
    logp = lp.gather(1, tokens.clamp(0, V - 1).unsqueeze(1)).squeeze(1)
    logp = logp.masked_fill(bad, float("nan")).masked_fill(dead, 0.0)
    p = e / s
    ent = -torch.where(p == 0, p, p * lp).sum(1).masked_fill(dead, 0.0)
    stats = torch.cat([m, logs / math.log(2.0)], 1).masked_fill(dead.unsqueeze(1), 0.0)
    # NaN first, then descending, equal values (-0 and +0 too) by ascending id
    ids = torch.sort(x + 0.0, dim=1, descending=True, stable=True).indices[:, :top]
    tlp = lp.gather(1, ids).masked_fill(dead.unsqueeze(1), 0.0)
    return logp, ent, stats, ids.masked_fill(dead.unsqueeze(1), -1), tlp


def token_logprobs_bwd(logits, tokens, stats, entropy, dlogp, dentropy, temperature, ignore_index, out):
    op = "token_logprobs_bwd"
    _check_logits(logits, temperature, op)
    _check_tokens(tokens, logits, op)
    _check_rows(stats, logits, (2,), op, "stats")
    _check_rows(entropy, logits, (), op, "entropy")
    for t, name in ((dlogp, "dlogp"), (dentropy, "dentropy")):
        if t is not None:
            _check_rows(t, logits, (), op, name)
    if out is None:
        out = torch.empty(logits.shape, dtype=logits.dtype)
    _check_out(out, logits, op)
    V = logits.shape[1]
    z = torch.zeros(logits.shape[0], 1)
    g = z if dlogp is None else dlogp.unsqueeze(1)
    h = z if dentropy is None else dentropy.unsqueeze(1)
    lp = (logits.float() - stats[:, :1]) / temperature - stats[:, 1:] * math.log(2.0)
    p = torch.exp(lp)
    d = -g * p - h * torch.where(p == 0, p, p * (lp + entropy.unsqueeze(1)))
    d.scatter_add_(1, tokens.clamp(0, V - 1).unsqueeze(1), g)
    dead = tokens == ignore_index
    bad = ~dead & ((tokens < 0) | (tokens >= V))
    d = (d / temperature).masked_fill(bad.unsqueeze(1), float("nan")).masked_fill(dead.unsqueeze(1), 0.0)
    return out.copy_(d)


def distill_topk(logits, ids, z, lse, temperature, scale, scale_h, rows, vocab_start, vocab_size, mode, stats, out):
    """ops.distill_topk_*: mode 0 loss rows and gradient; 1 loss rows and statistics [T, 9]; 2 loss rows
    and gradient from joined statistics.  Returns (loss, statistics, gradient)."""
    op = "distill_topk"
    _check_logits(logits, temperature, op)
    T, V = logits.shape
    _need(ids.device == logits.device and ids.dtype in (torch.int64, torch.int32) and ids.dim() == 2
          and ids.shape[0] == T and (ids.shape[1] <= 1 or ids.stride(1) == 1),
          f"{op}: ids must be int64 or int32 [T, K] with unit inner stride on the logits' device")
    _need(ids.shape[1] <= DISTILL_K_MAX, f"{op}: at most {DISTILL_K_MAX} entries a row")
    _need(z.dtype in FLOATS, f"{op}: teacher logits must be bfloat16, float16 or float32")
    _need(z.device == logits.device and z.shape == ids.shape and (z.shape[1] <= 1 or z.stride(1) == 1),
          f"{op}: teacher logits must be [T, K] with unit inner stride on the logits' device")
    if lse is not None:
        _check_rows(lse, logits, (), op, "lse")
        _need(V <= DISTILL_REST_V_MAX, f"{op}: with a teacher lse at most {DISTILL_REST_V_MAX} logits a row")
    _need(vocab_start >= 0 and vocab_size >= vocab_start + V, f"{op}: the part's logits lie outside the vocabulary")
    _need(mode != 0 or vocab_size == V, f"{op}: a part of a vocabulary goes through statistics and gradient")
    if scale is not None:
        _need(scale.device == logits.device and scale.dtype == torch.float32 and scale.numel() == 1,
              f"{op}: scale must be a number or one float32 on the logits' device")
        scale_h = float(scale.reshape(-1)[0])
    if rows is not None:
        _check_rows(rows, logits, (), op, "row weights")
    if mode == 2:
        _check_rows(stats, logits, (9,), op, "stats")
    _need(mode != 1 or out is None, f"{op}: out goes with a gradient")
    if out is None:
        out = torch.empty(logits.shape, dtype=logits.dtype)
    _check_out(out, logits, op)
    nan, zero = float("nan"), torch.zeros(())
    ids = ids.long()
    has = ids >= 0
    bad = (ids >= vocab_size).any(1)
    here = (ids >= vocab_start) & (ids < vocab_start + V)
    col = torch.where(here, ids - vocab_start, V)                      # V: a column that is cut off again
    zt = torch.where(has, z.float() / temperature, float("-inf"))
    if lse is None:
        mz = zt.amax(1, keepdim=True) if zt.shape[1] else torch.full((T, 1), float("-inf"))
        mz = torch.where(torch.isneginf(mz), 0.0, mz)
        q = torch.exp(zt - mz)
        n = q.sum(1, keepdim=True)
        lq = zt - mz - torch.log(n)
        q = torch.where(n == 0, n, q / n)
        rest = torch.zeros(T)
    else:
        # in 64 bits, as the rest is often small
        lq = torch.where(has, z.double() / temperature, float("-inf")) - lse.double().unsqueeze(1)
        q = torch.where(has, torch.exp(lq), 0.0)
        rest = (1 - q.sum(1)).clamp(min=0)
    some = (q != 0).any(1)
    W = (q.sum(1) + rest).float().unsqueeze(1)
    lq, q, rest = lq.float(), q.float(), rest.float()
    x = logits.float()
    inside = torch.zeros(T, V + 1, dtype=torch.bool).scatter_(1, col, True)[:, :V]
    xk = torch.cat([x, torch.zeros(T, 1)], 1).gather(1, col)
    xo = x.masked_fill(inside, float("-inf"))                          # what lies outside, against its own greatest

    def sums(v):
        m = v.amax(1, keepdim=True)
        return m, torch.exp(torch.where(torch.isneginf(m), v, v - m) / temperature).sum(1, keepdim=True)
    if mode != 2:
        m, s = sums(x)
        mo, u = sums(xo) if lse is not None else (torch.full_like(m, float("-inf")), torch.zeros_like(m))
        ok = here & (q != 0)
        xq = torch.where(ok, q * (xk - torch.where(torch.isneginf(m), 0.0, m)), zero).sum(1, keepdim=True)
        # the student's (max, sum, outside max, outside sum, sum q (x - max), sum q here), the teacher's
        # (max and sum of the softmax, or rest and sum q) and whether the row has entries
        tm, tn = (mz * temperature, n) if lse is None else (rest.unsqueeze(1), q.sum(1, keepdim=True))
        part = torch.cat([m, s, mo, u, xq, torch.where(here, q, zero).sum(1, keepdim=True), tm, tn, torch.ones(T, 1)], 1)
    else:
        m, s, mo, u, xq = stats[:, :5].split(1, 1)
        part = None
    logs = torch.log(s)
    # ln of the mass outside
    do = torch.where(torch.isneginf(mo), zero, mo - m)
    lnR = do / temperature + torch.log(u) - logs
    live = (rest.unsqueeze(1) > 0) & (u != 0)
    loss = torch.where(q != 0, q * (lq + logs), zero).sum(1) - (xq / temperature).squeeze(1)
    r1 = rest.unsqueeze(1)
    loss = loss + torch.where(live, r1 * (torch.log(r1) - lnR), zero).squeeze(1)
    loss = loss.masked_fill(~some, 0.0).masked_fill(bad, nan)
    if mode == 1:
        return loss, part.masked_fill(~some.unsqueeze(1), 0.0).masked_fill(bad.unsqueeze(1), nan), None
    p = torch.exp((x - m) / temperature - logs)
    # outside: p W - o r with o the softmax there; R itself may vanish
    o = torch.exp(torch.where(torch.isneginf(mo), xo, xo - mo) / temperature) / torch.where(u == 0, torch.ones_like(u), u)
    dx = torch.where(inside, p, p if lse is None else o * (u * torch.exp(do / temperature) / s)) * W
    dx = dx - torch.where(live, o * r1, zero)
    dx = torch.cat([dx, torch.zeros(T, 1)], 1).scatter_add_(1, col, torch.where(here, -q, zero))[:, :V]
    dx = dx * (scale_h / temperature) * (1.0 if rows is None else rows.unsqueeze(1))
    out.copy_(dx.masked_fill(~some.unsqueeze(1), 0.0).masked_fill(bad.unsqueeze(1), nan))
    return loss, None, out


def adamw_(p, w, m, v, g, n_decay, lr, b1, b2, eps, wd, step, gscale=1.0, sumsq=None,
           max_norm=0.0):
    gf = g.float() * gscale
    if sumsq is not None and max_norm > 0:
        nrm = math.sqrt(float(sumsq)) * gscale
        gf = gf * min(1.0, max_norm / (nrm + 1e-6))
    bc1 = 1 - b1 ** step
    bc2 = 1 - b2 ** step
    decay = torch.ones_like(w)
    decay[:n_decay] = 1 - lr * wd
    m.mul_(b1).add_(gf, alpha=1 - b1)
    v.mul_(b2).addcmul_(gf, gf, value=1 - b2)
    denom = v.sqrt() / math.sqrt(bc2) + eps
    w.mul_(decay).sub_(lr * (m / bc1) / denom)
    p.copy_(w.to(p.dtype))


def attention(q, k, v, causal=True, scale=None):
    """q [B,Hq,S,D], k/v [B,Hkv,S,D] -> (o [B,Hq,S,D], lse [B,Hq,S]) in fp32 math (GQA)."""
    B, Hq, S, D = q.shape
    Hkv = k.shape[1]
    rep = Hq // Hkv
    kf = k.float().repeat_interleave(rep, dim=1)
    vf = v.float().repeat_interleave(rep, dim=1)
    scale = scale if scale is not None else 1.0 / math.sqrt(D)
    s = torch.matmul(q.float(), kf.transpose(-1, -2)) * scale
    if causal:
        Sk = k.shape[2]
        mask = torch.ones(S, Sk, dtype=torch.bool, device=q.device).tril(Sk - S)
        s = s.masked_fill(~mask, float("-inf"))
    lse = torch.logsumexp(s, dim=-1)
    p = torch.softmax(s, dim=-1)
    o = torch.matmul(p, vf)
    return o, lse
