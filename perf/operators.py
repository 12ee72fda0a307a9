"""Cases for the operators over a language model's logits: log-probabilities of given tokens (with entropy and the top
alternatives), their gradient, and distillation from a teacher's top logits with its gradient.

``own`` false: plain torch in 32 bits (64 where it matters); ``own`` true: the package's entry points."""
import math

import torch

own = False
DEV = "cuda"
IGNORE = -100
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
ESIZE = {"bf16": 2, "fp16": 2, "fp32": 4}


# ---------------------------------------------------------------- cases
def _logprobs(name, T, V, dtype="bf16", pad=0, temperature=1.0, top=0, masked=0.0, banned=0, grad=False):
    c = {"op": "logprobs_grad" if grad else "logprobs", "T": T, "V": V, "dtype": dtype, "pad": pad,
         "temperature": temperature, "top": top, "masked": masked, "banned": banned}
    return {"name": name, **c} if name else c


def _distill(name, T, V, K, dtype="bf16", pad=0, temperature=1.0, rest=False, ragged=False, ids32=False, grad=False):
    c = {"op": "distill_grad" if grad else "distill", "T": T, "V": V, "K": K, "dtype": dtype, "pad": pad,
         "temperature": temperature, "rest": rest, "ragged": ragged, "ids32": ids32}
    return {"name": name, **c} if name else c


def listed():
    return [
        # serving one sequence: the drawn token's log-probability and five alternatives, latency only
        _logprobs("lp_one_row", 1, 128256, top=5),
        # a full decode batch with the most alternatives the completions protocol asks for
        _logprobs("lp_decode_batch", 64, 128256, top=20),
        # constrained decoding: banned tokens hold -inf; a vocabulary of no round size, fp16, sampling temperature
        _logprobs("lp_banned_odd", 24, 50021, dtype="fp16", temperature=0.7, top=20, banned=3),
        # scoring a long prompt, one LM-head chunk of rows, a tenth of them padding
        _logprobs("lp_score_chunk", 4096, 128256, masked=0.1),
        # a teacher writing its targets: the 64 top tokens of every row
        _logprobs("lp_teacher_top", 2048, 128256, top=64),
        # policy gradient with an entropy bonus over one LM-head chunk
        _logprobs("lp_policy_chunk", 4096, 128256, masked=0.25, grad=True),
        # the same in 32 bits on a small odd vocabulary with padded rows
        _logprobs("lp_policy_fp32", 700, 32003, dtype="fp32", pad=13, temperature=1.3, grad=True),
        # distillation over one LM-head chunk: loss and gradient in one pass
        _distill("kd_chunk", 4096, 128256, 64),
        # teacher's tail kept as one rest bucket, softened, targets with fewer entries in some rows
        _distill("kd_rest_chunk", 2048, 128256, 32, temperature=2.0, rest=True, ragged=True, ids32=True),
        # a short sequence on a small vocabulary
        _distill("kd_small", 37, 32000, 8, dtype="fp16", temperature=4.0, ragged=True),
        # through autograd, 32 bits, odd vocabulary, many entries
        _distill("kd_autograd_fp32", 513, 50021, 200, dtype="fp32", pad=3, temperature=1.5, rest=True, grad=True),
    ]


def draw(rng):
    """One more case: rows and vocabulary spread over their logarithm, no dearer than the largest listed one."""
    def spread(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    V = spread(300, 262144)
    if rng.random() < 0.4:
        V = -(-V // 64) * 64                        # vocabularies are often padded to a multiple of 64
    T = spread(1, max(2, min(4096, 4096 * 128256 * 2 // (2 * ESIZE[dtype] * V))))
    pad = rng.choice([0, 0, 0, rng.randint(1, 130)])
    temperature = rng.choice([1.0, 1.0, round(rng.uniform(0.5, 4.0), 3)])
    kind = rng.choice(["logprobs", "logprobs", "logprobs_grad", "distill", "distill_grad"])
    if kind.startswith("logprobs"):
        top = 0 if kind == "logprobs_grad" or rng.random() < 0.25 else spread(1, 64)
        return _logprobs(None, T, V, dtype, pad, temperature, top, rng.choice([0.0, 0.3]) if T > 3 else 0.0,
                         rng.choice([0, 0, 5]), kind == "logprobs_grad")
    return _distill(None, T, V, spread(1, min(256, V // 3)), dtype, pad, temperature, rng.random() < 0.5,
                    T > 3 and rng.random() < 0.5, rng.random() < 0.5, kind == "distill_grad")


# ---------------------------------------------------------------- inputs
def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed * 1000003 + 17)
    T, V, dt = case["T"], case["V"], DTYPES[case["dtype"]]
    # logits as a trained head gives them: a broad bulk, and one continuation that stands out on most rows
    buf = torch.empty(T, V + case["pad"], device=DEV, dtype=dt).normal_(0.0, 2.0, generator=g)
    x = buf[:, :V]
    tokens = torch.randint(0, V, (T,), generator=g, device=DEV)
    lift = (_randn(g, T) * 3 + 9).to(dt)
    x.scatter_add_(1, tokens[:, None], lift[:, None])
    s = {"case": case, "logits": x}
    if case["op"].startswith("logprobs"):
        if case["banned"]:
            # every n-th token of a row's own phase is banned, never the given one
            at = torch.arange(V, device=DEV)[None, :] + torch.randint(0, V, (T, 1), generator=g, device=DEV)
            x.masked_fill_((at % case["banned"] == 0) & (torch.arange(V, device=DEV)[None, :] != tokens[:, None]),
                           float("-inf"))
        if case["masked"]:
            tokens = tokens.masked_fill(torch.rand(T, generator=g, device=DEV) < case["masked"], IGNORE)
        s["tokens"] = tokens
        if case["op"] == "logprobs_grad":
            s["dlogp"] = _randn(g, T) / T          # advantages
            s["dentropy"] = torch.full((T,), -0.01 / T, device=DEV)
            if case["dtype"] == "fp16":            # loss scaling, as fp16 training uses it
                s["dlogp"] *= 256.0 * T
                s["dentropy"] *= 256.0 * T
        return s
    K = case["K"]
    step = torch.randint(1, V // K + 1, (T, 1), generator=g, device=DEV)
    ids = (tokens[:, None] + step * torch.arange(K, device=DEV)[None, :]) % V      # distinct: K * step <= V
    z = torch.sort(_randn(g, T, K) * 2.5 + 6, dim=1, descending=True).values
    x.scatter_add_(1, ids, (0.6 * z * torch.rand(T, 1, generator=g, device=DEV)).to(dt))   # a student part-way there
    if case["ragged"]:
        n = torch.randint(0, K + 1, (T, 1), generator=g, device=DEV)               # 0: a row without a target
        ids = ids.masked_fill(torch.arange(K, device=DEV)[None, :] >= n, -1)
    s["ids"] = ids.to(torch.int32) if case["ids32"] else ids
    s["teacher"] = z.to(dt)
    s["lse"] = None
    if case["rest"]:
        zt = s["teacher"].float() / case["temperature"]
        s["lse"] = torch.logsumexp(zt, 1) + 0.02 + 0.3 * torch.rand(T, generator=g, device=DEV)
    s["scale"] = 256.0 if case["dtype"] == "fp16" else 1.0 / T
    if case["op"] == "distill_grad":
        s["drows"] = (torch.rand(T, generator=g, device=DEV) + 0.5) * s["scale"]
    return s


# ---------------------------------------------------------------- plain forms
def _plain_logprobs(x, tokens, temperature, top):
    """(logp, entropy, ids, top logp) and what the gradient needs, in 32 bits."""
    live = tokens != IGNORE
    z = x.float() / temperature
    m = z.amax(1, keepdim=True)
    e = torch.exp(z - m)
    s = e.sum(1, keepdim=True)
    logs = torch.log(s)
    logp_all = z - m - logs
    p = e / s
    zero = torch.zeros((), device=x.device)
    logp = torch.where(live, logp_all.gather(1, tokens.clamp(min=0)[:, None])[:, 0], zero)
    entropy = torch.where(live, -torch.where(p > 0, p * logp_all, zero).sum(1), zero)
    if top:
        # one whole number orders by value, then by the lower index: all different, so no tie is left open
        u = (x.float() + 0.0).view(torch.int32)
        u = torch.where(u < 0, u ^ 0x7FFFFFFF, u).long()
        at = torch.arange(x.shape[1], device=x.device)
        key = torch.topk((u << 32) + (0xFFFFFFFF - at)[None, :], top, dim=1).values
        ids = 0xFFFFFFFF - (key & 0xFFFFFFFF)
        tlp = torch.where(live[:, None], logp_all.gather(1, ids), zero)
        ids = torch.where(live[:, None], ids, torch.full_like(ids, -1))
    else:
        ids = torch.empty(x.shape[0], 0, dtype=torch.int64, device=x.device)
        tlp = torch.empty(x.shape[0], 0, device=x.device)
    return logp, entropy, ids, tlp, p, logp_all, live


def _plain_logprobs_grad(s):
    c, x, tokens = s["case"], s["logits"], s["tokens"]
    logp, entropy, _, _, p, logp_all, live = _plain_logprobs(x, tokens, c["temperature"], 0)
    zero = torch.zeros((), device=x.device)
    d = -s["dlogp"][:, None] * p
    d -= s["dentropy"][:, None] * torch.where(p > 0, p * (logp_all + entropy[:, None]), zero)
    d.scatter_add_(1, tokens.clamp(min=0)[:, None], s["dlogp"][:, None])
    d = torch.where(live[:, None], d / c["temperature"], zero)
    return logp, entropy, d.to(x.dtype)


def _plain_distill(s, rows):
    """(loss rows, gradient rows times ``rows``)."""
    c, x = s["case"], s["logits"]
    t = c["temperature"]
    ids = s["ids"].long()
    has = ids >= 0
    at = ids.clamp(min=0)
    zero = torch.zeros((), device=x.device)
    zt = (s["teacher"].float() / t).double()
    zt = torch.where(has, zt, torch.full_like(zt, float("-inf")))
    if s["lse"] is None:
        mz = zt.amax(1, keepdim=True)
        mz = torch.where(torch.isfinite(mz), mz, torch.zeros_like(mz))
        q = torch.exp(zt - mz)
        n = q.sum(1, keepdim=True)
        logq = zt - mz - torch.log(n)
        q = torch.where(n > 0, q / n, torch.zeros_like(q))
        r = torch.zeros_like(n)
        some = (n > 0)[:, 0]
    else:
        logq = zt - s["lse"].double()[:, None]
        q = torch.exp(logq)
        r = (1 - q.sum(1, keepdim=True)).clamp(min=0)          # next to a border: 64 bits
        some = (q > 0).any(1)
    w = (q.sum(1, keepdim=True) + r).float()
    q, logq, r = q.float(), logq.float(), r.float()
    z = x.float() / t
    m = z.amax(1, keepdim=True)
    e = torch.exp(z - m)
    total = e.sum(1, keepdim=True)
    lp = (z - m).gather(1, at) - torch.log(total)
    loss = torch.where(q > 0, q * (logq - lp), zero).sum(1)
    p = e / total
    if s["lse"] is None:
        d = p * w
    else:
        # entries of id -1 mark column V, which is cut off
        inside = torch.zeros(x.shape[0], x.shape[1] + 1, dtype=torch.bool, device=x.device)
        inside.scatter_(1, torch.where(has, ids, torch.full_like(ids, x.shape[1])), True)
        inside = inside[:, :-1]
        out = torch.where(inside, zero, p).sum(1, keepdim=True)
        live = (r > 0) & (out > 0)
        loss = loss + torch.where(live, r * (torch.log(r) - torch.log(out)), zero)[:, 0]
        d = torch.where(inside, p * w, p * torch.where(live, w - r / out, w))
    d.scatter_add_(1, at, torch.where(has, -q, zero))
    d = torch.where(some[:, None], d * rows / t, zero)
    return torch.where(some, loss, zero), d.to(x.dtype)


# ---------------------------------------------------------------- one pass
def run(s):
    c = s["case"]
    op = c["op"]
    if own:
        from service_account_auth_improvements_amd import ops
        if op == "logprobs":
            logp, entropy, _, ids, tlp = ops.token_logprobs_fwd(s["logits"], s["tokens"], c["temperature"], c["top"])
            return {"logp": logp, "entropy": entropy, "ids": ids, "top": tlp} if c["top"] else {"logp": logp, "entropy": entropy}
        if op == "logprobs_grad":
            logp, entropy, stats, _, _ = ops.token_logprobs_fwd(s["logits"], s["tokens"], c["temperature"])
            d = ops.token_logprobs_bwd(s["logits"], s["tokens"], stats, entropy, s["dlogp"], s["dentropy"], c["temperature"])
            return {"logp": logp, "entropy": entropy, "dlogits": d}
        if op == "distill":
            loss, d = ops.distill_topk_fused(s["logits"], s["ids"], s["teacher"], s["scale"], c["temperature"], s["lse"])
            return {"loss": loss, "dlogits": d}
        x = s["logits"].detach().requires_grad_()
        loss = ops.distill_topk(x, s["ids"], s["teacher"], c["temperature"], s["lse"])
        (d,) = torch.autograd.grad(loss, x, s["drows"])
        return {"loss": loss.detach(), "dlogits": d}
    if op == "logprobs":
        logp, entropy, ids, tlp, _, _, _ = _plain_logprobs(s["logits"], s["tokens"], c["temperature"], c["top"])
        return {"logp": logp, "entropy": entropy, "ids": ids, "top": tlp} if c["top"] else {"logp": logp, "entropy": entropy}
    if op == "logprobs_grad":
        return dict(zip(("logp", "entropy", "dlogits"), _plain_logprobs_grad(s)))
    rows = s["drows"][:, None] if op == "distill_grad" else s["scale"]
    return dict(zip(("loss", "dlogits"), _plain_distill(s, rows)))


def work(case):
    T, V, e = case["T"], case["V"], ESIZE[case["dtype"]]
    rows = T * (1.0 - case.get("masked", 0.0))      # a padding row's logits need not be read
    if case["op"] == "logprobs":
        return {"bytes": rows * V * e + T * (8 + 8 + 12 * case["top"]), "flops": 4.0 * rows * V}
    if case["op"] == "logprobs_grad":
        return {"bytes": (rows + T) * V * e + T * 24, "flops": 8.0 * rows * V}
    K = case["K"]
    side = T * (K * (e + (4 if case["ids32"] else 8)) + 4 + (4 if case["rest"] else 0))
    return {"bytes": 2.0 * T * V * e + side, "flops": 7.0 * T * V}


# ---------------------------------------------------------------- the definition, in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    x = s["logits"].double() / case["temperature"]
    lsm = x - torch.logsumexp(x, 1, keepdim=True)
    T = case["T"]
    n = torch.arange(T, device=DEV)
    if case["op"].startswith("logprobs"):
        tok = s["tokens"]
        dead = tok == IGNORE
        p = lsm.exp()
        H = torch.special.entr(p).sum(1)
        res = {"logp": lsm[n, tok.clamp(min=0)].masked_fill(dead, 0.0), "entropy": H.masked_fill(dead, 0.0)}
        if case["op"] == "logprobs_grad":
            a, b = s["dlogp"].double()[:, None], s["dentropy"].double()[:, None]
            d = (torch.special.entr(p) - p * H[:, None]) * b - a * p     # -p ln p - p H
            d[n, tok.clamp(min=0)] += a[:, 0]
            res["dlogits"] = (d / case["temperature"]).masked_fill(dead[:, None], 0.0)
        elif case["top"]:
            order = torch.sort(s["logits"].double(), dim=1, descending=True, stable=True).indices[:, :case["top"]]
            res["ids"] = order.masked_fill(dead[:, None], -1)
            res["top"] = lsm.gather(1, order).masked_fill(dead[:, None], 0.0)
        return res
    # teacher as a dense distribution over the vocabulary (ids are distinct in these inputs)
    ids = s["ids"].long()
    row, col = (ids >= 0).nonzero(as_tuple=True)
    z = torch.full_like(x, float("-inf"))
    z[row, ids[row, col]] = s["teacher"].double()[row, col] / case["temperature"]
    some = (ids >= 0).any(1)
    inside = torch.isfinite(z)
    p = lsm.exp()
    if s["lse"] is None:
        q = torch.softmax(z, 1).masked_fill(~some[:, None], 0.0)
        loss = (torch.special.xlogy(q, q) - q * lsm).sum(1)
        d = p - q
    else:
        q = (z - s["lse"].double()[:, None]).exp()
        r = (1.0 - q.sum(1)).clamp(min=0)
        R = p.masked_fill(inside, 0.0).sum(1)
        loss = (torch.special.xlogy(q, q) - q * lsm).sum(1) + torch.special.xlogy(r, r / R)
        # sum q ln p + r ln R by the chain rule: the softmax's Jacobian on q / p inside and r / R outside
        up = torch.where(inside, q / p, (r / R)[:, None])
        d = p * (up * p).sum(1, keepdim=True) - p * up
    rows = s["drows"].double()[:, None] if case["op"] == "distill_grad" else s["scale"]
    return {"loss": loss.masked_fill(~some, 0.0), "dlogits": (d * rows / case["temperature"]).masked_fill(~some[:, None], 0.0)}
