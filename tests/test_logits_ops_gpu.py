"""The gfx950 kernels of ops.token_logprobs* and ops.distill_topk* against the 64-bit oracle: types,
lengths, strides, alignments, masks, ties, streams and graphs.  All on cuda:0."""
import pytest
import torch

import logits_oracle as oracle
from service_account_auth_improvements_amd import ops
from service_account_auth_improvements_amd.ops import _ext
from test_logits_ops import REFUSALS, refusal_args

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16, FP16, F32 = torch.bfloat16, torch.float16, torch.float32
NEG = float("-inf")


@pytest.fixture(scope="module", autouse=True)
def _lib():
    assert _ext.load(), "the HIP library must load"


def _x(T, V, dtype, seed=0, pad=0, skip=0):
    """[T, V] logits in a wider buffer that starts ``skip`` elements in: any alignment."""
    g = torch.Generator().manual_seed(seed)
    buf = torch.zeros(skip + T * (V + pad) + 8, dtype=dtype, device=DEV)
    x = buf[skip:skip + T * (V + pad)].view(T, V + pad)[:, :V]
    x.copy_((torch.randn(T, V, generator=g) * 3).to(dtype))
    return x


def _tok(T, V, seed=1):
    return torch.randint(0, V, (T,), generator=torch.Generator().manual_seed(seed)).to(DEV)


def _check_fwd(x, tok, temp=1.0, top=0):
    logp, ent, stats, ids, tlp = ops.token_logprobs_fwd(x, tok, temp, top)
    V = x.shape[1]
    rl, rh, ri, rt = oracle.logprobs(x.cpu(), tok.cpu(), temp, top)
    oracle.close(logp, rl, oracle.logp_bound(rl, V), "logp")
    oracle.close(ent, rh, oracle.entropy_bound(rh, V), "entropy")
    assert torch.equal(ids.cpu(), ri)
    oracle.close(tlp, rt, oracle.logp_bound(rt, V), "top")
    return ent, stats


SHAPES = [(1, 1, 0, 0), (2, 7, 0, 0), (3, 8, 0, 1), (5, 9, 3, 0), (4, 63, 0, 5), (3, 1000, 1, 0), (2, 2047, 0, 3), (3, 16384, 0, 0),
          (3, 16385, 0, 0), (5, 32003, 13, 7), (2, 128256, 0, 0), (1, 262143, 0, 1), (300, 517, 2, 0)]


@pytest.mark.parametrize("dtype", [BF16, FP16, F32])
@pytest.mark.parametrize("T,V,pad,skip", SHAPES)
def test_logprobs_forward_backward(T, V, pad, skip, dtype):
    for temp, top in ((1.0, 0), (0.6, min(20, V)), (2.5, min(128, V))):
        x, tok = _x(T, V, dtype, 0, pad, skip), _tok(T, V)
        if T > 2:
            tok[1] = -100
        ent, stats = _check_fwd(x, tok, temp, top)
    g, h = torch.randn(T), torch.randn(T)
    ref, size = oracle.logprobs_grad(x.cpu(), tok.cpu(), g, h, temp)
    bound = oracle.grad_bound(ref, size, 60.0, V, dtype)
    d = ops.token_logprobs_bwd(x, tok, stats, ent, g.to(DEV), h.to(DEV), temp)
    oracle.close(d, ref, bound, "dlogits")
    ref1, size1 = oracle.logprobs_grad(x.cpu(), tok.cpu(), g, torch.zeros(T), temp)
    d1 = ops.token_logprobs_bwd(x, tok, stats, ent, g.to(DEV), None, temp)
    oracle.close(d1, ref1, oracle.grad_bound(ref1, size1, 60.0, V, dtype), "dlogits of logp")
    # in place, through the strided rows; what lies between the rows stays
    base = x.clone() if x._base is None else x._base.clone()
    here = ops.token_logprobs_bwd(x, tok, stats, ent, g.to(DEV), h.to(DEV), temp, out=x)
    assert here.data_ptr() == x.data_ptr() and torch.equal(x, d)
    if x._base is not None:
        gap = torch.ones_like(base, dtype=torch.bool)
        gap.as_strided(x.shape, x.stride(), x.storage_offset()).fill_(False)
        assert torch.equal(x._base[gap], base[gap])


@pytest.mark.parametrize("V", [5000, 40000])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_logprobs_masks_and_special_rows(V, dtype):
    low = torch.finfo(dtype).min
    x, tok = _x(12, V, dtype), _tok(12, V)
    ar = torch.arange(V, device=DEV)
    x[0] = NEG; x[0, int(tok[0])] = 2.0                     # one token allowed
    x[1].masked_fill_(ar % 3 != 0, NEG); tok[1] = 1         # the given one is masked
    x[2].masked_fill_(ar % 5 != 0, low)                     # masks of the type's lowest value
    x[3] = low                                              # ... and nothing else: uniform
    x[4] = low; x[4, ::2] = NEG
    x[5] = 1.5                                              # all equal: the lowest ids
    x[6, :V // 2] = NEG
    x[7, 1024:] = NEG
    x[8].masked_fill_(ar % 2 == 0, 0.0); x[8].masked_fill_(ar % 2 == 1, -0.0)   # zeros of both signs are one value
    x[9] = torch.sort(x[9], descending=True).values
    x[10] = torch.sort(x[10]).values
    x[11] = NEG; tok[11] = -100                             # padding
    tok[4] = 1
    for top in (0, 1, 17, 128):
        ent, stats = _check_fwd(x, tok, 1.3, top)
    g, h = torch.randn(12), torch.randn(12)
    ref, size = oracle.logprobs_grad(x.cpu(), tok.cpu(), g, h, 1.3)
    d = ops.token_logprobs_bwd(x, tok, stats, ent, g.to(DEV), h.to(DEV), 1.3)
    oracle.close(d, ref, oracle.grad_bound(ref, size, 60.0, V, dtype), "dlogits")


@pytest.mark.parametrize("V", [900, 5003, 40001])
def test_logprobs_nan_and_infinities(V):
    x, tok = _x(6, V, F32), _tok(6, V)
    x[0, V - 1] = float("nan")
    x[1, 3] = float("inf")
    x[2] = NEG
    x[3, 1::2] = float("nan")
    x[4] = float("nan")
    x[5, 7] = float("nan"); x[5, 2] = -float("nan"); tok[5] = -100
    ent, stats = _check_fwd(x, tok, 1.0, 100)
    d = ops.token_logprobs_bwd(x, tok, stats, ent, torch.ones(6, device=DEV), None)
    assert torch.isnan(d[:5]).all() and (d[5] == 0).all()


def test_logprobs_token_outside_the_vocabulary_is_nan():
    x = _x(3, 700, BF16)
    tok = torch.tensor([700, -1, 699], device=DEV)
    ent, stats = _check_fwd(x, tok, 1.0, 4)
    d = ops.token_logprobs_bwd(x, tok, stats, ent, torch.ones(3, device=DEV), torch.ones(3, device=DEV))
    assert torch.isnan(d[:2]).all() and torch.isfinite(d[2]).all()


# rows whose great values meet the threads' stride: more elements than are held at a time reach the
# first bound (thread groups of 4 x 8 elements, 1024 threads above 16384 logits; of 8 elements, 256 below)
@pytest.mark.parametrize("V,group,top,great", [(128256, 4, 4, 3), (128256, 4, 40, 39), (16384, 1, 40, 39), (16383, 1, 128, 127)])
@pytest.mark.parametrize("order", ["random", "rising", "equal"])
def test_top_alternatives_in_an_order_that_meets_the_stride(V, group, top, great, order):
    g = torch.Generator().manual_seed(3)
    x = torch.randn(2, V, generator=g)
    c = torch.arange(V) // 8
    hit = (c // group) % 256 < great
    up = {"random": torch.rand(V, generator=g), "rising": torch.arange(V) / V, "equal": torch.zeros(V)}[order]
    x = torch.where(hit, 20 + 4 * up, x).to(DEV)
    _check_fwd(x, _tok(2, V), 1.0, top)


@pytest.mark.parametrize("T", [1, 2, 31, 100, 255, 256, 257])
def test_few_and_many_rows(T):
    """Rows that several blocks share and rows of one block."""
    for V, top in ((20001, 0), (20001, 11), (4104, 128), (65537, 3)):
        x, tok = _x(T, V, BF16, 0, 1), _tok(T, V)
        tok[T // 2] = -100 if T > 2 else tok[T // 2]
        _check_fwd(x, tok, 0.9, top)


@pytest.mark.parametrize("V,dtype", [(70001, BF16), (66003, FP16), (36001, F32)])
def test_few_long_rows_with_masks_ties_and_orders(V, dtype):
    """Rows that several blocks share: their lists of alternatives meet in one order, whatever is equal."""
    low = torch.finfo(dtype).min
    x, tok = _x(13, V, dtype, 4, 1), _tok(13, V)
    ar = torch.arange(V, device=DEV)
    x[0] = NEG; x[0, int(tok[0])] = 2.0
    x[1] = 1.5                                              # all equal
    x[2] = low
    x[3].masked_fill_(ar % 5 != 0, low)
    x[4, 700:] = NEG                                        # one part holds all there is
    x[5, :V - 9] = NEG                                      # ... the last one
    x[6] = torch.sort(x[6].float(), descending=True).values.to(dtype)
    x[7] = torch.sort(x[7].float()).values.to(dtype)
    x[8] = (x[8].float() / 4).round().to(dtype)             # some ten values in all
    x[9, V // 2] = float("nan")
    x[10] = NEG; x[10, 1::V // 40] = 3.0
    x[11] = float("nan")
    x[12] = NEG; tok[12] = -100
    for top in (0, 1, 5, 12, 13, 20, 64, 128):              # up to and above what is ranked directly
        _check_fwd(x, tok, 1.3, top)


@pytest.mark.parametrize("T", [2, 33, 70, 127, 128, 512, 513])
@pytest.mark.parametrize("V,top", [(32769, 0), (36800, 20), (65537, 64), (65537, 128), (140001, 33)])
def test_rows_around_the_choices_of_the_launch(T, V, top):
    if T * V > 20_000_000:
        V = V // 2 + 1
    x, tok = _x(T, V, BF16, 5, 3), _tok(T, V)
    tok[T // 2] = -100
    _check_fwd(x, tok, 0.8, top)


def test_logprobs_expanded_and_broadcast_inputs():
    x = _x(1, 3001, BF16).expand(7, 3001)                    # row stride 0
    tok = _tok(7, 3001)
    _check_fwd(x, tok, 1.0, 5)
    leaf = _x(1, 3001, F32).clone().requires_grad_()
    logp, ent, _, _ = ops.token_logprobs(leaf.expand(7, 3001), tok)
    (logp.sum() + ent.mean()).backward()                     # upstream gradients are broadcast too
    ref, size = oracle.logprobs_grad(leaf.detach().cpu().expand(7, 3001), tok.cpu(), torch.ones(7), torch.full((7,), 1 / 7))
    oracle.close(leaf.grad, ref.sum(0, keepdim=True), 8 * oracle.grad_bound(ref, size, 60.0, 3001, F32).sum(0, keepdim=True), "leaf")


def test_out_that_overlaps_otherwise_is_refused():
    buf = torch.zeros(4 * 128 + 8, device=DEV)
    x = buf[:512].view(4, 128)
    st, f, tok = torch.zeros(4, 2, device=DEV), torch.zeros(4, device=DEV), _tok(4, 128)
    with pytest.raises(RuntimeError, match="overlaps"):
        ops.token_logprobs_bwd(x, tok, st, f, f, out=buf[8:520].view(4, 128))
    two = torch.zeros(4, 256, device=DEV)                    # side by side in one buffer: taken
    ops.token_logprobs_bwd(two[:, :128], tok, st, f, f, out=two[:, 128:])
    with pytest.raises(RuntimeError, match="overlaps"):
        ops.token_logprobs_bwd(two[:, :128], tok, st, f, f, out=two[:, 127:255])


@pytest.mark.parametrize("what", sorted(REFUSALS))
def test_refusals(what):
    with pytest.raises(RuntimeError, match="token_logprobs|distill_topk"):
        REFUSALS[what](refusal_args(DEV))


def test_tensors_of_another_device_are_refused():
    x, tok = _x(3, 40, F32), _tok(3, 40)
    ids, z = torch.zeros(3, 2, dtype=torch.long, device=DEV), torch.zeros(3, 2, device=DEV)
    for call in (lambda: ops.token_logprobs_fwd(x, tok.cpu()), lambda: ops.distill_topk_fused(x, ids.cpu(), z, 1.0),
                 lambda: ops.distill_topk_fused(x, ids, z.cpu(), 1.0), lambda: ops.distill_topk_fused(x, ids, z, torch.ones(1)),
                 lambda: ops.distill_topk_fused(x, ids, z, 1.0, 1.0, torch.zeros(3))):
        with pytest.raises(RuntimeError, match="device"):
            call()


# ---------------------------------------------------------------- distillation
def _teacher(T, V, K, dtype, lse, temp, seed=2):
    g = torch.Generator().manual_seed(seed)
    ids = torch.stack([torch.randperm(V, generator=g)[:K] for _ in range(T)]) if T else torch.zeros(0, K, dtype=torch.long)
    z = (torch.randn(T, K, generator=g) * 2).to(dtype)
    L = torch.logsumexp(z.float() / temp, 1) + 0.1 if lse else None
    return ids, z, L


def _check_kd(x, ids, z, temp, L, scale=0.5):
    V, dtype = x.shape[1], x.dtype
    dev = lambda t: None if t is None else t.to(DEV)          # noqa: E731
    loss, d = ops.distill_topk_fused(x, dev(ids), dev(z), scale, temp, dev(L))
    rl, rd, size, lsize = oracle.distill(x.cpu(), ids, z, temp, L)
    lb = (1 + lsize) * 4 * oracle.sum_bound(V)
    oracle.close(loss, rl, lb, "loss")
    oracle.close(d, rd * scale, oracle.grad_bound(rd * scale, size * scale, 60.0, V, dtype), "dlogits")
    xv = x.detach().clone().requires_grad_()
    rows = torch.rand(x.shape[0])
    lo = ops.distill_topk(xv, dev(ids), dev(z), temp, dev(L))
    (da,) = torch.autograd.grad(lo, xv, rows.to(DEV))
    oracle.close(lo, rl, lb, "autograd loss")
    r = rows[:, None].double()
    oracle.close(da, rd * r, oracle.grad_bound(rd * r, size * r, 60.0, V, dtype), "autograd dlogits")
    return loss, d


@pytest.mark.parametrize("lse", [False, True])
@pytest.mark.parametrize("dtype,zt", [(BF16, BF16), (FP16, F32), (F32, FP16)])
@pytest.mark.parametrize("T,V,pad,skip,K", [(1, 1, 0, 0, 1), (3, 9, 0, 1, 4), (5, 1000, 3, 0, 64), (4, 16385, 0, 5, 200), (2, 128256, 0, 0, 64),
                                            (3, 5, 0, 0, 5), (6, 300, 0, 0, 256), (4, 50, 0, 0, 0), (1, 262143, 1, 0, 8)])
def test_distill(T, V, pad, skip, K, dtype, zt, lse):
    x = _x(T, V, dtype, 0, pad, skip)
    ids, z, L = _teacher(T, V, K, zt, lse, 1.5)
    if T > 3 and K > 4:
        ids[1] = -1                                          # a row without entries
        ids[2, 3:] = -7
        ids[3, 1] = ids[3, 0]                                # the same id twice, and again
        ids[3, 4] = ids[3, 0]
    loss, d = _check_kd(x, ids, z, 1.5, L)
    # int32 ids, strided ids and teacher logits, scale on the device, in place
    wide = torch.full((T, K + 3), -1, dtype=torch.int32)
    wide[:, :K] = ids.int()
    zw = torch.zeros(T, K + 5, dtype=zt)
    zw[:, 2:K + 2] = z
    lo2, d2 = ops.distill_topk_fused(x, wide.to(DEV)[:, :K], zw.to(DEV)[:, 2:K + 2], torch.full((1,), 0.5, device=DEV), 1.5,
                                     None if L is None else L.to(DEV), out=x)
    assert d2.data_ptr() == x.data_ptr() and torch.equal(lo2, loss) and torch.equal(x, d)


# every row (skip odd, stride even) or every second one
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("V,pad,skip", [(1, 0, 1), (2, 1, 0), (8, 1, 0), (9, 0, 0), (16, 1, 1), (17, 1, 1), (520, 3, 0), (4096, 1, 0), (32769, 0, 0),
                                        (66000, 1, 0), (131072, 1, 1), (131080, 1, 0)])
def test_rows_off_a_4_byte_boundary(V, pad, skip, dtype):
    T, k = 6, min(V, 7)
    x, tok = _x(T, V, dtype, 6, pad, skip), _tok(T, V)
    x[0, 0] = x[1, 0] = 30.0                                 # the first element is the greatest
    x[2] = 0.25                                              # equal everywhere: the first ones
    x[3, 0] = NEG
    x[4, 1:] = NEG; x[4, 0] = -5.0                           # there is no other
    tok[0] = tok[1] = tok[4] = 0
    ent, stats = _check_fwd(x, tok, 1.2, k)
    _check_fwd(x[:, V // 2:], tok % (V - V // 2), 1.2, 0)
    # the same bits wherever a row lies
    there = torch.zeros(T, V + 16 - V % 8, dtype=dtype, device=DEV)[:, :V]
    there.copy_(x)
    for a, b in zip(ops.token_logprobs_fwd(x, tok, 1.2, k), ops.token_logprobs_fwd(there, tok, 1.2, k)):
        assert torch.equal(a.isnan(), b.isnan()) and torch.equal(a[~a.isnan()], b[~b.isnan()])    # V = 1 has a row of -inf
    ids = torch.stack([(torch.arange(k) * max(1, V // k) + r % 2) % V for r in range(T)])
    ids[5] = 0                                               # the first element again and again
    z = torch.linspace(2, -2, k).expand(T, k).clone()
    for L in (None, torch.logsumexp(z, 1) + 0.2):
        _check_kd(x, ids, z, 1.0, L)
    want = ops.distill_topk_fused(x, ids.to(DEV), z.to(DEV), 1.0, 1.0)[1]
    here = ops.distill_topk_fused(x, ids.to(DEV), z.to(DEV), 1.0, 1.0, out=x)[1]
    assert torch.equal(here.contiguous().view(torch.int16), want.view(torch.int16))      # bits: V = 1 has a row of -inf, all NaN


@pytest.mark.parametrize("V", [400, 20000])
@pytest.mark.parametrize("lse", [False, True])
def test_distill_masks_and_special_rows(V, lse):
    T, K = 10, 6
    x = _x(T, V, F32)
    ids, z, L = _teacher(T, V, K, F32, lse, 1.0)
    low = torch.finfo(F32).min
    x[0].masked_fill_(torch.arange(V, device=DEV) % 2 == 0, NEG)      # some of the teacher's ids are banned: +inf
    ids[0, 0] = 2
    x[1] = NEG                                                        # the student has nothing: NaN
    x[2] = low
    x[3, 5] = float("nan")
    x[4] = NEG; x[4, ids[4].to(DEV)] = 1.0                            # nothing outside
    z[5, 2] = NEG                                                     # an entry without mass
    z[6] = NEG                                                        # nothing but such
    z[7] = low
    x[8, int(ids[8, 0])] = 60.0                                       # a student that is sure: 1 - p is below fp32's step
    ids[9, 3] = V                                                     # an id behind the end
    _check_kd(x, ids, z, 1.0, L)


@pytest.mark.parametrize("lse", [False, True])
def test_distill_nan_teacher(lse):
    x = _x(2, 500, BF16)
    ids, z, L = _teacher(2, 500, 5, F32, lse, 1.0)
    z[0, 1] = float("nan")
    loss, d = ops.distill_topk_fused(x, ids.to(DEV), z.to(DEV), 1.0, 1.0, None if L is None else L.to(DEV))
    assert torch.isnan(loss[0]) and torch.isnan(d[0]).all() and torch.isfinite(loss[1]) and torch.isfinite(d[1]).all()


@pytest.mark.parametrize("lse", [False, True])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_distill_in_vocabulary_parts(dtype, lse):
    V, cuts, temp = 41001, (0, 20500, 20501, 41001), 1.7
    x = _x(5, V, dtype)
    ids, z, L = _teacher(5, V, 40, F32, lse, temp)
    ids[1] = -1
    ids[2, 0] = 20500
    ids, z, L = ids.to(DEV), z.to(DEV), None if L is None else L.to(DEV)
    whole, dw = ops.distill_topk_fused(x, ids, z, 2.0, temp, L)
    cols = list(zip(cuts[:-1], cuts[1:]))
    st = torch.stack([ops.distill_topk_stats(x[:, a:b], ids, z, temp, L, a, V) for a, b in cols])
    joined = ops.distill_topk_join(st, temp)
    rl, rd, size, lsize = oracle.distill(x.cpu(), ids.cpu(), z.cpu(), temp, None if L is None else L.cpu())
    for a, b in cols:
        loss, d = ops.distill_topk_grad(x[:, a:b], ids, z, joined, 2.0, temp, L, a, V)
        oracle.close(loss, rl, (1 + lsize) * 8 * oracle.sum_bound(V), "loss")
        oracle.close(d, 2 * rd[:, a:b], oracle.grad_bound(2 * rd[:, a:b], 2 * size[:, a:b], 60.0, V, dtype), "dlogits")


@pytest.mark.parametrize("lse", [False, True])
@pytest.mark.parametrize("T,V,dtype", [(700, 65601, BF16), (1200, 40000, FP16), (2100, 3001, BF16), (600, 40000, F32), (40, 262145, BF16)])
def test_distill_more_rows_than_blocks(T, V, dtype, lse):
    """Blocks that walk several rows: each row's result is the one it has alone, and the sampled ones the oracle's."""
    x = _x(T, V, dtype, 0, 3, 1)
    K = 20
    g = torch.Generator().manual_seed(4)
    ids = (torch.randint(0, V, (T, 1), generator=g) + torch.randint(1, V // K, (T, 1), generator=g) * torch.arange(K)) % V
    ids[::7] = -1
    ids[3::11, 5:] = -1
    z = torch.randn(T, K, generator=g) * 2
    L = torch.logsumexp(z, 1) + 0.1 if lse else None
    dev = lambda t: None if t is None else t.to(DEV)          # noqa: E731
    loss, d = ops.distill_topk_fused(x, dev(ids), dev(z), 0.5, 1.0, dev(L))
    for rows in ([0, 1, T // 2, T - 1], [255 % T, 256 % T, 257 % T, 511 % T, 512 % T]):
        sel = lambda t: None if t is None else t[rows]        # noqa: E731
        lo, da = ops.distill_topk_fused(x[rows], dev(ids[rows]), dev(z[rows]), 0.5, 1.0, dev(sel(L)))
        assert torch.equal(lo, loss[rows]) and torch.equal(da, d[rows])
    rows = [0, 1, 3, T // 2, T - 1]
    rl, rd, size, lsize = oracle.distill(x[rows].cpu(), ids[rows], z[rows], 1.0, None if L is None else L[rows])
    oracle.close(loss[rows], rl, (1 + lsize) * 4 * oracle.sum_bound(V), "loss")
    oracle.close(d[rows], rd * 0.5, oracle.grad_bound(rd * 0.5, size * 0.5, 60.0, V, dtype), "dlogits")


def test_distill_empty_rows_of_nan_logits():
    """A row without targets is 0 whatever its logits hold."""
    for V in (500, 40000, 300001):
        x = _x(3, V, F32)
        x[1], x[2] = float("nan"), float("inf")
        ids = torch.zeros(3, 4, dtype=torch.long, device=DEV)
        ids[1] = -1
        z = torch.randn(3, 4, device=DEV)
        z[2] = NEG
        for L in (None, torch.full((3,), 3.0, device=DEV)):
            loss, d = ops.distill_topk_fused(x, ids, z, 1.0, 1.0, L)
            assert torch.isfinite(loss).all() and (loss[1:] == 0).all() and (d[1:] == 0).all() and torch.isfinite(d).all()


def test_entry_in_a_part_of_nothing_but_minus_infinity():
    x = _x(2, 20, F32)
    x[0, :8] = NEG
    ids, z = torch.tensor([[3, 12], [3, 12]], device=DEV), torch.zeros(2, 2, device=DEV)
    whole, dw = ops.distill_topk_fused(x, ids, z, 1.0)
    st = torch.stack([ops.distill_topk_stats(x[:, a:b], ids, z, 1.0, None, a, 20) for a, b in ((0, 8), (8, 20))])
    for a, b in ((0, 8), (8, 20)):
        loss, d = ops.distill_topk_grad(x[:, a:b], ids, z, ops.distill_topk_join(st), 1.0, 1.0, None, a, 20)
        oracle.close(loss, whole.cpu(), 64 * oracle.EPS * (1 + whole[1].abs().cpu()), "loss")
        oracle.close(d, dw[:, a:b].cpu(), 64 * oracle.EPS, "dlogits")
    assert whole[0] == float("inf")


def test_teacher_to_student_run():
    """The operators together: a teacher's top alternatives are the student's targets, whose
    log-probabilities rise along the gradient."""
    V, T, K = 32000, 16, 64
    teacher, student = _x(T, V, BF16, 5), _x(T, V, F32, 6)
    tok = teacher.argmax(1)
    _, _, _, ids, tlp = ops.token_logprobs_fwd(teacher, tok, top=K)
    lse = torch.zeros(T, device=DEV)                          # log-probabilities: normalised already
    loss, d = ops.distill_topk_fused(student, ids, tlp, 1.0, 1.0, lse)
    rl, rd, size, lsize = oracle.distill(student.cpu(), ids.cpu(), tlp.cpu(), 1.0, lse.cpu())
    oracle.close(loss, rl, (1 + lsize) * 4 * oracle.sum_bound(V), "loss")
    oracle.close(d, rd, oracle.grad_bound(rd, size, 60.0, V, F32), "dlogits")
    before = ops.token_logprobs_fwd(student, tok)[0]
    after = ops.token_logprobs_fwd(student - 4 * d, tok)[0]
    assert (after > before).all()


# ---------------------------------------------------------------- streams, graphs, determinism
def _all_calls(x, tok, ids, z, L, g):
    logp, ent, st, top, tlp = ops.token_logprobs_fwd(x, tok, 1.1, 20)
    d = ops.token_logprobs_bwd(x, tok, st, ent, g, g, 1.1)
    loss, dk = ops.distill_topk_fused(x, ids, z, 1.0, 1.1, L)
    part = ops.distill_topk_stats(x, ids, z, 1.1, L)
    lg, dg = ops.distill_topk_grad(x, ids, z, ops.distill_topk_join(part[None], 1.1), 1.0, 1.1, L)
    return [logp, ent, st, top, tlp, d, loss, dk, part, lg, dg]


def _inputs(T, V, seed=0):
    x, tok = _x(T, V, BF16, seed), _tok(T, V, seed + 1)
    ids, z, L = _teacher(T, V, 30, F32, True, 1.1, seed + 2)
    return [x, tok, ids.to(DEV), z.to(DEV), L.to(DEV), torch.randn(T, generator=torch.Generator().manual_seed(seed)).to(DEV)]


def test_results_do_not_depend_on_the_run_or_the_stream():
    a = _inputs(33, 32003)
    one = _all_calls(*a)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        two = _all_calls(*a)
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    for p, q in zip(one, two):
        assert torch.equal(p, q)


def test_captured_and_replayed():
    a = _inputs(9, 20001)
    static = [t.clone() for t in a]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        _all_calls(*static)
    torch.cuda.current_stream().wait_stream(s)
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g1):
        o1 = _all_calls(*static)
    with torch.cuda.graph(g2):                                # a second graph of the same calls
        o2 = _all_calls(*static)
    for seed in (0, 10, 20):
        for t, n in zip(static, _inputs(9, 20001, seed)):
            t.copy_(n)
        want = _all_calls(*static)
        torch.cuda.synchronize()
        g1.replay(); g2.replay(); g1.replay()
        torch.cuda.synchronize()
        for p, q, w in zip(o1, o2, want):
            assert torch.equal(p, w) and torch.equal(q, w)


def test_captured_autograd():
    T, V = 6, 5001
    w = torch.randn(V, 32, device=DEV)
    h, tok = torch.randn(T, 32, device=DEV), _tok(T, V)
    ids, z, _ = _teacher(T, V, 7, F32, False, 1.0)
    ids, z = ids.to(DEV), z.to(DEV)

    def step(hh):
        x = torch.mm(hh.detach(), w.t()).requires_grad_()
        logp, ent, _, _ = ops.token_logprobs(x, tok)
        (d,) = torch.autograd.grad((logp - 0.1 * ent).mean() - ops.distill_topk(x, ids, z).mean(), x)
        return d
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step(h)
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step(h)
    for seed in range(3):
        h.copy_(torch.randn(T, 32, generator=torch.Generator().manual_seed(seed)))
        want = step(h)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


def test_rows_beyond_32_bit_offsets():
    """A row stride that puts the last rows more than 2^31 elements from the first."""
    V, ld, T = 1000, 715_827_883, 4
    buf = torch.empty((T - 1) * ld + V, dtype=BF16, device=DEV)
    x = buf.as_strided((T, V), (ld, 1))
    x.copy_(_x(T, V, BF16))
    tok = _tok(T, V)
    ent, st = _check_fwd(x, tok, 1.0, 9)
    g = torch.randn(T)
    ref, size = oracle.logprobs_grad(x.cpu(), tok.cpu(), g, torch.zeros(T))
    d = ops.token_logprobs_bwd(x, tok, st, ent, g.to(DEV))
    oracle.close(d, ref, oracle.grad_bound(ref, size, 60.0, V, BF16), "dlogits")
    ids, z, _ = _teacher(T, V, 8, F32, False, 1.0)
    _check_kd(x, ids, z, 1.0, None)


def test_no_rows():
    x, tok = _x(0, 100, BF16), torch.zeros(0, dtype=torch.long, device=DEV)
    logp, ent, st, ids, tlp = ops.token_logprobs_fwd(x, tok, 1.0, 5)
    assert logp.shape == (0,) and ids.shape == (0, 5)
    assert ops.token_logprobs_bwd(x, tok, st, ent, ent).shape == (0, 100)
    loss, d = ops.distill_topk_fused(x, torch.zeros(0, 3, dtype=torch.long, device=DEV), torch.zeros(0, 3, device=DEV), 1.0)
    assert loss.shape == (0,) and d.shape == (0, 100)


@pytest.mark.parametrize("other", [False, True])
def test_capture_over_a_live_graph_of_a_leaf_is_refused(other):
    x, tok = _x(3, 500, F32).clone().requires_grad_(), _tok(3, 500)
    ids, z = torch.zeros(3, 2, dtype=torch.long, device=DEV), torch.zeros(3, 2, device=DEV)
    held = (x * 2) if other else ops.token_logprobs(x, tok)[0]      # an eager graph that is still alive
    for call in (lambda: ops.token_logprobs(x, tok), lambda: ops.distill_topk(x, ids, z)):
        with pytest.raises(RuntimeError, match="earlier autograd graph"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                call()
    held.sum().backward()
    assert torch.isfinite(x.grad).all()


def test_autograd_corners():
    x, tok = _x(4, 300, F32).clone().requires_grad_(), _tok(4, 300)
    ids, z, L = (t.to(DEV) for t in _teacher(4, 300, 5, F32, True, 1.0))
    # one output used, or none
    logp, ent, top, tlp = ops.token_logprobs(x, tok, 1.0, 3)
    assert not top.requires_grad and not tlp.requires_grad
    (d,) = torch.autograd.grad(ent.sum(), x)
    ref, size = oracle.logprobs_grad(x.detach().cpu(), tok.cpu(), torch.zeros(4), torch.ones(4))
    oracle.close(d, ref, oracle.grad_bound(ref, size, 60.0, 300, F32), "entropy's")
    # 16-bit upstream gradients, no gradient wanted, leaf of another type
    xh = x.detach().half().requires_grad_()
    loss = ops.distill_topk(xh, ids, z, 1.0, L)
    loss.to(torch.bfloat16).sum().backward()
    assert xh.grad.dtype == FP16
    with torch.no_grad():
        assert not ops.distill_topk(x, ids, z).requires_grad
    assert not ops.token_logprobs(x.detach(), tok)[0].requires_grad
    # differentiable once
    for f in (lambda: ops.token_logprobs(x, tok)[0].sum(), lambda: ops.distill_topk(x, ids, z).pow(2).sum()):
        (g,) = torch.autograd.grad(f(), x, create_graph=True)
        with pytest.raises(RuntimeError, match="twice"):
            g.sum().backward()
    # logits overwritten before the backward pass
    y = x * 1.0
    lo = ops.distill_topk(y, ids, z)
    with torch.no_grad():
        y.zero_()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        lo.sum().backward()
    # refusals come through
    with pytest.raises(RuntimeError, match="distill_topk"):
        ops.distill_topk(x, ids.short(), z)
    with pytest.raises(RuntimeError, match="token_logprobs"):
        ops.token_logprobs(x, tok.int())
