"""Normed and rotated keys into the paged caches, page bounds, page choice and
attention over chosen pages (HIP) against 64-bit forms (GPU).

Tolerances.  Cache values and queries: as the norm's own test, half a step of
the type they are stored in plus 2^-24 * 32 (|z_lo| + |z_hi|); bounds and page
choices are exact.  The attention: the weights are rounded to the caches' 16-bit
type in the numerator (half a step, eps / 2), or taken with 16 significant bits
(2^-16 for each of a few factors) where q or the caches are wider; a =
scale q.k - 1/2 is off by da (2^-24 D sum|q k| scale, or 2^-15 of it with split
operands), which changes a weight by 2 da of itself; a + sqrt(a^2 + 1) loses up
to 2 (a^2 + 1) steps of 2^-24 twice over, 2^-12 for |a| <= 16; the output is
rounded to bf16, 2^-8.
"""
import math

import pytest
import torch

import smooth_attn
from oracle import paging, serving

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24
FP8 = torch.float8_e4m3fn
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


def _g(seed):
    return torch.Generator().manual_seed(seed)


def _randn(shape, dtype, seed, scale=1.0):
    return (torch.randn(shape, generator=_g(seed)) * scale).to(dtype)


def _bytes(t):
    return t.contiguous().view(torch.uint8)


def _half_step(dtype):
    return torch.finfo(dtype).eps / 2


# ---------------------------------------------------------------------------
# Norm, rotation and append.
# ---------------------------------------------------------------------------
APPEND = [
    # N, Hq, Hkv, D, P, dtype, cache, weights
    (1, 1, 1, 16, 16, BF, BF, "same"),
    (8, 32, 8, 128, 16, BF, BF, "same"),
    (77, 8, 2, 64, 16, HF, HF, "fp32"),
    (50, 4, 4, 128, 32, BF, FP8, "same"),
    (33, 6, 3, 80, 8, BF, F32, "none"),
    (20, 5, 1, 256, 16, F32, BF, "same"),
    (19, 2, 2, 512, 4, F32, F32, "same"),
    (40, 4, 1, 96, 12, HF, FP8, "fp32"),
    (1000, 32, 8, 128, 16, BF, BF, "fp32"),
    (70, 3, 2, 48, 16, F32, FP8, "none"),
]


@pytest.mark.parametrize("N,Hq,Hkv,D,P,dtype,cache,weights", APPEND)
def test_append(N, Hq, Hkv, D, P, dtype, cache, weights):
    fused = _randn((N, (Hq + 2 * Hkv) * D), dtype, 1, 1.7)
    q, k, v = (t.unflatten(1, (-1, D)) for t in fused.split([Hq * D, Hkv * D, Hkv * D], 1))
    wdt = F32 if weights == "fp32" else dtype
    qw, kw = (None, None) if weights == "none" else [(1 + 0.3 * _randn((D,), F32, s)).to(wdt) for s in (2, 3)]
    n_pages = N // P + 3
    angle = torch.rand(64, D // 2, generator=_g(4)) * 60
    cos, sin = angle.cos(), angle.sin()
    pos = torch.randint(0, 64, (N,), generator=_g(5)).to(torch.int32)
    slots = torch.randperm(n_pages * P, generator=_g(6))[:N].to(torch.int32)
    if N > 4:
        slots[1], slots[3], pos[2] = -1, n_pages * P + 3, 1000  # not stored; past the caches; past the tables
    kc, vc = (_randn((n_pages, Hkv, P, D), BF, s).to(cache) for s in (7, 8))
    kd, vd = kc.to(DEV), vc.to(DEV)
    dev = [None if t is None else t.to(DEV) for t in (qw, kw, cos, sin, pos, slots)]
    parts = [t.unflatten(1, (-1, D)) for t in fused.to(DEV).split([Hq * D, Hkv * D, Hkv * D], 1)]
    out = smooth_attn.sp2norm_paged_qk_norm_rope_append(*parts, *dev, kd, vd, block_size=P)
    assert out.dtype == dtype and out.shape == (N, Hq, D)

    p = pos.long().clamp(0, 63)
    c, s = cos[p].double()[:, None], sin[p].double()[:, None]
    yq, yk = (serving.qk_norm_rope(x.double(), None if w is None else w.double(), c, s) for x, w in ((q, qw), (k, kw)))

    def terms(x, w):
        z = (serving.qk_norm_rope(x.double(), None if w is None else w.double(), 1.0, 0.0)).abs()
        return 32 * U * (z + z.roll(D // 2, -1))

    err = (out.cpu().double() - yq).abs()
    assert (err <= _half_step(dtype) * yq.abs() + 2 * terms(q, qw) + 2.0 ** -25).all(), err.max()
    live = (slots >= 0) & (slots < n_pages * P)
    page, row = slots[live].long() // P, slots[live].long() % P
    got_k = kd.cpu().view(torch.uint8 if cache == FP8 else cache)[page, :, row].view(cache).double()
    err = (got_k - yk[live]).abs()
    low = 2.0 ** -10 if cache == FP8 else 2.0 ** -25 if cache == HF else 0.0  # half the smallest step
    assert (err <= _half_step(cache) * yk[live].abs() * (1 + 1e-6) + 2 * terms(k, kw)[live] + low).all(), err.max()
    # values are only converted, and every other row stays as it was
    ref_v, ref_k = _bytes(vc).view(n_pages, Hkv, P, -1).clone(), _bytes(kc).view(n_pages, Hkv, P, -1).clone()
    ref_v[page, :, row] = _bytes(v[live].to(cache)).view(int(live.sum()), Hkv, -1)
    assert torch.equal(_bytes(vd.cpu()).view_as(ref_v), ref_v)
    after = _bytes(kd.cpu()).view_as(ref_k).clone()
    after[page, :, row] = ref_k[page, :, row]
    assert torch.equal(after, ref_k)


def test_append_rounds_to_e4m3_as_torch_does():
    # every rounding case of the 8-bit type: v is stored as it is
    x = torch.cat([torch.linspace(-520, 520, 4001), torch.tensor([464.0, 463.9, 464.1, 448.0, 1e30, -1e30, 2.0 ** -10,
                   2.0 ** -11, 3 * 2.0 ** -10, 0.0, -0.0, float("inf"), float("-inf"), float("nan"), 0.0146, 0.0155]),
                   torch.randn(4000, generator=_g(1)) * 0.02])
    x = torch.cat([x, torch.zeros(-x.numel() % 64)]).view(-1, 1, 64)
    N = x.shape[0]
    kc = torch.zeros(N, 1, 1, 64, dtype=torch.uint8, device=DEV).view(FP8)
    vc = torch.zeros_like(kc.view(torch.uint8)).view(FP8)
    cos, sin = torch.ones(1, 32, device=DEV), torch.zeros(1, 32, device=DEV)
    zero = torch.zeros(N, dtype=torch.int32, device=DEV)
    slots = torch.arange(N, dtype=torch.int32, device=DEV)
    smooth_attn.sp2norm_paged_qk_norm_rope_append(x.to(DEV), x.to(DEV), x.to(DEV), None, None, cos, sin, zero, slots,
                                                  kc, vc, block_size=1)
    want, got = x.to(FP8), vc.cpu().view(N, 1, 64)
    nan = torch.isnan(want.float())
    assert torch.equal(torch.isnan(got.float()), nan)
    assert torch.equal(got.view(torch.uint8)[~nan], want.view(torch.uint8)[~nan])


def test_append_of_nothing_and_into_strided_caches():
    D, P = 64, 16
    kc = torch.zeros(4, 2, P, 2 * D, dtype=BF, device=DEV)[..., :D]
    vc = torch.zeros(4, P, 2, D, dtype=BF, device=DEV).transpose(1, 2)
    cos, sin = torch.ones(8, 32, device=DEV), torch.zeros(8, 32, device=DEV)
    q, k = _randn((5, 4, D), BF, 1).to(DEV), _randn((5, 2, D), BF, 2).to(DEV)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
    args = (None, None, cos, sin, i32(0, 1, 2, 3, 4), i32(5, 63, 17, 0, 40))
    out = smooth_attn.sp2norm_paged_qk_norm_rope_append(q, k, k, *args, kc, vc)
    k2, v2 = torch.zeros(4, 2, P, D, dtype=BF, device=DEV), torch.zeros(4, 2, P, D, dtype=BF, device=DEV)
    out2 = smooth_attn.sp2norm_paged_qk_norm_rope_append(q, k, k, *args, k2, v2)
    assert torch.equal(kc, k2) and torch.equal(vc, v2) and torch.equal(out, out2)
    none = smooth_attn.sp2norm_paged_qk_norm_rope_append(q[:0], k[:0], k[:0], None, None, cos, sin, i32(), i32(), k2, v2)
    assert none.shape == (0, 4, D) and torch.equal(k2, kc)


def test_64_bit_slots_and_positions_past_32_bits():
    D = 32
    cos, sin = smooth_attn.precompute_rope_cos_sin(D, 8, device=DEV)
    k = _randn((4, 2, D), BF, 1).to(DEV)
    kc, vc = (torch.zeros(2, 2, 16, D, dtype=BF, device=DEV) for _ in range(2))
    slots = torch.tensor([1 << 32, 3, -(1 << 32), (1 << 32) + 5], device=DEV)  # 0, 3, 0 and 5 in their low halves
    pos = torch.tensor([0, (1 << 32) + 1, 2, 3], device=DEV)                   # 1 in its low half; clamped to 7
    out = smooth_attn.sp2norm_paged_qk_norm_rope_append(k, k, k, None, None, cos, sin, pos, slots, kc, vc)
    assert torch.equal(vc[0, :, 3], k[1]) and int((vc != 0).any(-1).sum()) == 2
    want = smooth_attn.sp2norm_qk_norm_rope(k.transpose(0, 1)[None], k.transpose(0, 1)[None], None, None, cos, sin,
                                            positions=torch.tensor([0, 7, 2, 3], device=DEV))[0]
    assert torch.equal(out, want[0].transpose(0, 1))


def test_append_without_pages_or_query_heads():
    D = 32
    cos, sin = torch.ones(8, 16, device=DEV), torch.zeros(8, 16, device=DEV)
    k = _randn((3, 2, D), BF, 1).to(DEV)
    i32 = torch.arange(3, dtype=torch.int32, device=DEV)
    none = torch.zeros(0, 2, 16, D, dtype=BF, device=DEV)
    out = smooth_attn.sp2norm_paged_qk_norm_rope_append(k, k, k, None, None, cos, sin, i32, i32, none, none)
    kc, vc = torch.zeros(1, 2, 16, D, dtype=BF, device=DEV), torch.zeros(1, 2, 16, D, dtype=BF, device=DEV)
    empty = smooth_attn.sp2norm_paged_qk_norm_rope_append(k[:, :0], k, k, None, None, cos, sin, i32, i32, kc, vc)
    assert empty.shape == (3, 0, D) and torch.equal(kc[0, :, :3].transpose(0, 1), out) and torch.equal(vc[0, :, :3].transpose(0, 1), k)


# ---------------------------------------------------------------------------
# Bounds.
# ---------------------------------------------------------------------------
def _paged(B, Hkv, D, P, lens, dtype, seed, spare=3):
    """Random caches (rows past the lengths hold NaN), a shuffled table with
    entries that name no page past them."""
    W = max(-(-max(lens) // P), 1) + 1
    n_pages = sum(-(-n // P) for n in lens) + spare
    perm = torch.randperm(n_pages, generator=_g(seed))
    src = BF if dtype == FP8 else dtype
    kc, vc = (_randn((n_pages, Hkv, P, D), src, seed + i) for i in (1, 2))
    kc += _randn((n_pages, Hkv, 1, D), src, seed + 3)
    table = torch.full((B, W), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(lens):
        k = -(-n // P)
        table[b, :k] = perm[at:at + k].to(torch.int32)
        at += k
        if n % P:
            kc[perm[at - 1], :, n % P:] = float("nan")
            vc[perm[at - 1], :, n % P:] = float("nan")
    kc[perm[at:]] = float("nan")
    vc[perm[at:]] = float("nan")
    return kc.to(dtype), vc.to(dtype), table, torch.tensor(lens, dtype=torch.int32)


@pytest.mark.parametrize("Hkv,D,P,dtype", [
    (2, 64, 16, BF), (1, 128, 16, BF), (8, 128, 16, HF), (3, 80, 8, BF), (2, 128, 32, FP8), (1, 16, 1, FP8),
    (2, 96, 64, F32), (1, 8, 16, BF), (2, 256, 128, F32), (1, 1024, 4, F32), (1, 1024, 16, BF), (2, 48, 256, FP8)])
def test_bounds(Hkv, D, P, dtype):
    lens = [0, 1, P, P + 1, 3 * P - 1, 7 * P + P // 2]
    kc, _, table, ctx = _paged(len(lens), Hkv, D, P, lens, dtype, D + P)
    before = torch.tensor([0, 0, 0, P, P // 2, 5 * P + 1], dtype=torch.int32)
    start = torch.full((kc.shape[0], Hkv, 2, D), 9.0).to(dtype)
    want = serving.key_bounds(kc, table, before, ctx, start, P)
    bounds = start.to(DEV)
    got = smooth_attn.sp2norm_paged_key_bounds(kc.to(DEV), table.to(DEV), before.to(DEV), ctx.to(DEV), bounds,
                                               block_size=P)
    assert got is bounds
    assert torch.equal(bounds.cpu().double(), want)


def test_bounds_nan_new_tensor_and_bad_pages():
    P, D = 16, 64
    kc, _, table, ctx = _paged(3, 2, D, P, [40, 5, 17], BF, 1)
    kc[table[0, 1], 1, 3, 7] = float("nan")
    kc[table[0, 0], 0, 2, 5] = float("inf")
    table[2, 0] = 1000  # names no page
    zero = torch.zeros(3, dtype=torch.int32)
    want = serving.key_bounds(kc, table, zero, ctx, torch.zeros(kc.shape[0], 2, 2, D), P)
    got = smooth_attn.sp2norm_paged_key_bounds(kc.to(DEV), table.to(DEV), zero.to(DEV), ctx.to(DEV))
    torch.testing.assert_close(got.cpu().double(), want, rtol=0, atol=0, equal_nan=True)
    assert torch.isnan(got[table[0, 1], 1, :, 7]).all()


# ---------------------------------------------------------------------------
# Choice of pages.
# ---------------------------------------------------------------------------
def _bounds_of(kc, table, ctx, P):
    return serving.key_bounds(kc, table, torch.zeros_like(ctx), ctx, torch.zeros(kc.shape[0], kc.shape[1], 2, kc.shape[3]),
                              P).to(kc.dtype)


SELECT = [
    # Hq, Hkv, D, P, q type, cache, lens, top_k, n_first, n_last
    (32, 8, 128, 16, BF, BF, [1, 17, 500, 1024, 333], 8, 1, 1),
    (4, 4, 64, 16, HF, HF, [160, 161], 10, 0, 1),
    (8, 1, 80, 8, BF, BF, [700, 80, 8], 5, 2, 3),
    (6, 2, 96, 32, F32, F32, [900, 64, 1000], 7, 0, 0),
    (16, 2, 128, 16, BF, FP8, [2000, 31], 20, 0, 2),
    (2, 1, 256, 4, F32, BF, [300, 9], 33, 1, 1),
    (1, 1, 16, 1, BF, FP8, [3000, 50], 17, 3, 4),
    (3, 3, 512, 16, HF, HF, [200], 3, 1, 2),
    (2, 2, 1024, 16, BF, F32, [100, 40], 2, 0, 1),
    (2, 1, 8, 1, BF, BF, [5000, 600, 0], 512, 0, 1),
    (5, 1, 40, 16, F32, HF, [999], 1, 0, 1),
    (4, 2, 64, 16, FP8, BF, [400], 4, 1, 1),
]


@pytest.mark.parametrize("Hq,Hkv,D,P,qt,ct,lens,top_k,n_first,n_last", SELECT)
def test_select(Hq, Hkv, D, P, qt, ct, lens, top_k, n_first, n_last):
    kc, _, table, ctx = _paged(len(lens), Hkv, D, P, lens, ct, D + P + top_k)
    bounds = _bounds_of(kc, table, ctx, P)
    q = _randn((len(lens), Hq, 1, D), F32 if qt == FP8 else qt, 5).to(qt)
    want = serving.select_pages(q, bounds, table, ctx, top_k, n_first, n_last, P)
    got = smooth_attn.sp2norm_paged_select_pages(q.to(DEV), bounds.to(DEV), table.to(DEV), ctx.to(DEV), top_k,
                                                 n_first=n_first, n_last=n_last, block_size=P)
    assert torch.equal(got.cpu(), want)


@pytest.mark.parametrize("np_", [3, 64, 513, 1500, 5000, 17000])
def test_select_ties_infinities_and_nan(np_):
    # a few distinct scores: the border falls inside a run of equal ones
    D, P = 8, 2
    bounds = torch.zeros(np_, 1, 2, D, dtype=BF)
    bounds[:, 0, 1, 0] = torch.randint(0, 3, (np_,), generator=_g(1)).to(BF)
    q = torch.zeros(1, 1, 1, D, dtype=BF)
    q[..., 0] = 1
    table = torch.randperm(np_, generator=_g(2)).to(torch.int32)[None]
    ctx = torch.tensor([np_ * P], dtype=torch.int32)

    def check(k, first, last):
        want = serving.select_pages(q, bounds, table, ctx, k, first, last, P)
        got = smooth_attn.sp2norm_paged_select_pages(q.to(DEV), bounds.to(DEV), table.to(DEV), ctx.to(DEV), k,
                                                     n_first=first, n_last=last, block_size=P)
        assert torch.equal(got.cpu(), want), (k, first, last)

    ks = sorted({1, 2, max(1, np_ // 5), max(1, np_ // 2), max(1, np_ - 1), np_, np_ + 3})
    for k in ks:
        for first, last in ((0, 0), (0, 1), (1, 0), (1, 1)):
            if first + last <= k:
                check(k, first, last)
    bounds[np_ // 2, 0, 1, 0] = float("inf")
    bounds[np_ // 3, 0, 1, 0] = float("-inf")
    for k in ks:
        check(k, 0, 0)
    bounds[np_ - 1, 0, 0, 3] = float("inf")  # times a query of 0: NaN, above all
    bounds[0, 0, 0, 2] = float("nan")
    for k in ks:
        check(k, 0, 0)
    q.fill_(float("nan"))  # every score
    for k in ks:
        check(k, 0, 0)


def test_select_where_32_bits_would_not_do():
    # two pages whose scores differ by 2^-30 of themselves, among terms that cancel
    D, P = 64, 16
    bounds = torch.zeros(40, 1, 2, D, dtype=F32)
    bounds[:, 0, 1, 0] = 1.0
    bounds[:, 0, 1, 1] = 2.0 ** 20
    bounds[:, 0, 0, 2] = 2.0 ** 20
    bounds[27, 0, 1, 3] = 2.0 ** -10
    q = torch.zeros(1, 1, 1, D, dtype=F32)
    q[0, 0, 0, :4] = torch.tensor([1.0, 1.0, -1.0, 1.0])
    table = torch.arange(40, dtype=torch.int32)[None]
    got = smooth_attn.sp2norm_paged_select_pages(q.to(DEV), bounds.to(DEV), table.to(DEV),
                                                 torch.tensor([640], device=DEV), 2)
    assert got.tolist() == [[[27, 39]]]


# ---------------------------------------------------------------------------
# Attention over listed pages.
# ---------------------------------------------------------------------------
def _attention_tolerance(q, kc, table, ctx, pages, scale, P, o, bound, qt, ct):
    D = q.shape[-1]
    same16 = qt == ct and ct in (BF, HF)
    rounding = _half_step(ct) if same16 else 2.0 ** -14
    big = q.double().abs().amax() * kc.double().nan_to_num().abs().amax() * D * scale
    da = (U * D if same16 else 2.0 ** -15) * min(big, 16.0 * 4)
    rel = rounding + 4 * da + 2.0 ** -12
    return _half_step(BF) * o.abs() * (1 + rel) + rel * (bound + o.abs()) * 1.1 + 1e-30


SPARSE = [
    # Hq, Hkv, D, P, q, cache, lens, listed
    (32, 8, 128, 16, BF, BF, [1, 17, 500, 1024], 8),
    (4, 4, 64, 16, HF, HF, [160, 161, 5], 10),
    (8, 1, 80, 8, BF, BF, [700, 80, 8], 5),
    (6, 2, 96, 32, F32, F32, [900, 64], 7),
    (16, 2, 128, 16, BF, FP8, [2000, 31], 20),
    (2, 1, 256, 4, F32, BF, [300, 9], 33),
    (32, 1, 64, 1, BF, BF, [300, 40], 130),
    (3, 3, 512, 16, HF, HF, [200], 3),
    (2, 2, 1024, 16, BF, BF, [100, 40], 2),
    (2, 1, 128, 128, F32, HF, [999, 128], 3),
    (4, 2, 64, 2, F32, FP8, [77, 1], 40),
    (2, 2, 32, 64, BF, F32, [640], 5),
    (4, 1, 64, 16, FP8, FP8, [333], 9),
    (2, 1, 8, 16, BF, BF, [333], 9),
]


@pytest.mark.parametrize("Hq,Hkv,D,P,qt,ct,lens,n", SPARSE)
@pytest.mark.parametrize("order", ["ascending", "any"])
def test_sparse_attention(Hq, Hkv, D, P, qt, ct, lens, n, order):
    B = len(lens)
    kc, vc, table, ctx = _paged(B, Hkv, D, P, lens, ct, D + P + n)
    q = _randn((B, Hq, 1, D), F32 if qt == FP8 else qt, 5).to(qt)
    if order == "ascending":
        pages = serving.select_pages(q, _bounds_of(kc, table, ctx, P), table, ctx, n, 0, 1, P)
    else:  # any order, pages twice, outside the table, past the context
        pages = torch.randint(-2, table.shape[1] + 3, (B, Hkv, n), generator=_g(7)).to(torch.int32)
        pages[0, 0, 0] = 2 ** 31 - 1
    scale = 1 / math.sqrt(D)
    o, bound = serving.sparse_attention(q, kc, vc, table, ctx, pages, scale, P)
    got = smooth_attn.sp2norm_paged_sparse_attention(q.to(DEV), kc.to(DEV), vc.to(DEV), table.to(DEV), ctx.to(DEV),
                                                     pages.to(DEV), block_size=P)
    assert got.dtype == BF and got.shape == (B, Hq, D)
    tol = _attention_tolerance(q, kc, table, ctx, pages, scale, P, o, bound, qt, ct)
    err = (got.cpu().double() - o).abs()
    assert (err <= tol).all(), ((err - tol).max(), err.max())


def test_sparse_attention_without_tokens_is_zero():
    P, D = 16, 64
    kc, vc, table, ctx = _paged(2, 2, D, P, [40, 0], BF, 1)
    q = _randn((2, 4, 1, D), BF, 2).to(DEV)
    args = (kc.to(DEV), vc.to(DEV), table.to(DEV), ctx.to(DEV))
    none = torch.full((2, 2, 3), -1, dtype=torch.int32, device=DEV)
    assert (smooth_attn.sp2norm_paged_sparse_attention(q, *args, none) == 0).all()
    assert (smooth_attn.sp2norm_paged_sparse_attention(q, *args, none[..., :0]) == 0).all()
    all_ = torch.arange(3, dtype=torch.int32, device=DEV).expand(2, 2, 3)
    o = smooth_attn.sp2norm_paged_sparse_attention(q, *args, all_)
    assert (o[1] == 0).all() and torch.isfinite(o).all() and (o[0] != 0).any()


@pytest.mark.parametrize("dtype,D", [(BF, 128), (HF, 64), (F32, 128), (BF, 512)])
def test_sparse_attention_over_all_pages_is_the_paged_attention(dtype, D):
    P, lens = 16, [500, 33, 256, 1]
    kc, vc, table, ctx = _paged(4, 2, D, P, lens, dtype, 3)
    q = _randn((4, 8, 1, D), dtype, 4).to(DEV)
    args = (kc.to(DEV), vc.to(DEV), table.to(DEV), ctx.to(DEV))
    pages = smooth_attn.sp2norm_paged_select_pages(q, torch.zeros(kc.shape[0], 2, 2, D, dtype=dtype, device=DEV), *args[2:], 40)
    a = smooth_attn.sp2norm_paged_sparse_attention(q, *args, pages)
    b = smooth_attn.sp2norm_paged_attention(q, *args)
    # the same products in the same tiles, summed over other splits: a rounding of the output apart
    assert ((a.double() - b.double()).abs() <= 2.0 ** -7 * b.double().abs() + 2.0 ** -16).all()


def test_calls_on_another_stream_repeat_bit_for_bit():
    P, D = 16, 128
    kc, vc, table, ctx = (t.to(DEV) for t in _paged(6, 4, D, P, [700, 20, 333, 64, 1000, 5], BF, 3))
    q = _randn((6, 16, 1, D), BF, 4).to(DEV)

    def step():
        bounds = smooth_attn.sp2norm_paged_key_bounds(kc, table, torch.zeros_like(ctx), ctx)
        pages = smooth_attn.sp2norm_paged_select_pages(q, bounds, table, ctx, 10, n_first=1)
        return bounds, pages, smooth_attn.sp2norm_paged_sparse_attention(q, kc, vc, table, ctx, pages)

    want = step()
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for st in streams:  # two at once
        with torch.cuda.stream(st):
            got.append(step())
    torch.cuda.synchronize()
    for g in got:
        torch.testing.assert_close(g[0], want[0], rtol=0, atol=0, equal_nan=True)
        assert torch.equal(g[1], want[1]) and torch.equal(g[2], want[2])


# ---------------------------------------------------------------------------
# The operators together.
# ---------------------------------------------------------------------------
def _serve(B, W, P, n_pages, dtype, Hq, Hkv, D, top_k, steps, seed):
    """A few steps of a serving loop on the device (prompts, then single tokens,
    a sequence replaced on the way) and the same with the plain forms."""
    gen = _g(seed)
    cos, sin = smooth_attn.precompute_rope_cos_sin(D, W * P, device=DEV)
    qw, kw = ((1 + 0.1 * _randn((D,), F32, s)).to(dtype).to(DEV) for s in (1, 2))
    table = torch.full((B, W), -1, dtype=torch.int32, device=DEV)
    lens = torch.zeros(B, dtype=torch.int32, device=DEV)
    free = torch.randperm(n_pages, generator=gen).to(torch.int32).to(DEV)
    n_free = torch.tensor([n_pages], dtype=torch.int32, device=DEV)
    kc, vc = (torch.full((n_pages, Hkv, P, D), float("nan"), dtype=dtype, device=DEV) for _ in range(2))
    bounds = torch.zeros(n_pages, Hkv, 2, D, dtype=dtype, device=DEV)
    r_table, r_lens, r_free, r_n = table.cpu(), lens.cpu(), free.cpu(), n_pages
    keys = {}
    for step in range(steps):
        prompt = step == 0
        new = torch.randint(5, 3 * P, (B,), generator=gen) if prompt else torch.ones(B, dtype=torch.int64)
        if step == 2:
            done = torch.zeros(B, dtype=torch.bool)
            done[1] = True
            lens, n_free = smooth_attn.sp2norm_paged_release(table, lens, done.to(DEV), free, n_free, block_size=P)
            r_table, r_free, r_lens, r_n = serving.release(r_table, r_lens, done, r_free, r_n, P)
            keys = {k: v for k, v in keys.items() if k[0] != 1}
            new[1] = 2 * P + 3
        N = int(new.sum())
        x = _randn((N, Hq + 2 * Hkv, D), dtype, seed + 10 + step)
        q, k, v = x.to(DEV).split([Hq, Hkv, Hkv], 1)
        r = smooth_attn.sp2norm_paged_reserve(table, lens, new.to(DEV), free, n_free, N, block_size=P)
        qr = smooth_attn.sp2norm_paged_qk_norm_rope_append(q, k, v, qw, kw, cos, sin, r.positions, r.slots, kc, vc,
                                                           block_size=P)
        smooth_attn.sp2norm_paged_key_bounds(kc, table, lens, r.context_lens, bounds, block_size=P)
        last = (r.starts[1:] - 1).long()
        q1 = qr[last][:, :, None]
        pages = smooth_attn.sp2norm_paged_select_pages(q1, bounds, table, r.context_lens, top_k, block_size=P)
        o = smooth_attn.sp2norm_paged_sparse_attention(q1, kc, vc, table, r.context_lens, pages, block_size=P)
        w = serving.reserve(r_table, r_lens, new, r_free, r_n, N, P)
        assert torch.equal(table.cpu(), w[0]) and torch.equal(r.slots.cpu(), w[1])
        r_table, r_lens, r_n = w[0], w[5], w[6]
        lens, n_free = r.context_lens, r.n_free
        want_pages = serving.select_pages(q1.cpu(), serving.key_bounds(
            kc.cpu(), r_table, torch.zeros(B), r_lens, torch.zeros(bounds.shape), P).to(dtype), r_table, r_lens, top_k, 0, 1, P)
        assert torch.equal(pages.cpu(), want_pages), step
        ref, bound = serving.sparse_attention(q1.cpu(), kc.cpu(), vc.cpu(), r_table, r_lens, want_pages, D ** -0.5, P)
        assert ((o.cpu().double() - ref).abs() <= 2.0 ** -7 * (ref.abs() + bound)).all(), step
        # the caches hold every token's key where its sequence looks for it
        c64, s64 = cos.cpu().double(), sin.cpu().double()
        for i in range(N):
            keys[(int(w[3][i]), int(w[2][i]))] = x[i, Hq:Hq + Hkv]
        for (b, pos), raw in list(keys.items())[::7]:
            y = serving.qk_norm_rope(raw.double(), kw.cpu().double(), c64[pos], s64[pos])
            got = kc[r_table[b, pos // P], :, pos % P].cpu().double()
            assert ((got - y).abs() <= _half_step(dtype) * y.abs() + 1e-4).all()


@pytest.mark.parametrize("dtype,Hq,Hkv,D,P,top_k", [(BF, 8, 2, 64, 16, 2), (HF, 4, 4, 128, 8, 3), (F32, 4, 1, 32, 16, 4)])
def test_a_serving_loop(dtype, Hq, Hkv, D, P, top_k):
    _serve(5, 12, P, 70, dtype, Hq, Hkv, D, top_k, 6, 17)


def test_a_decode_step_replays_in_a_graph():
    B, W, P, n_pages, Hq, Hkv, D, top_k = 6, 20, 16, 130, 8, 2, 64, 5
    cos, sin = smooth_attn.precompute_rope_cos_sin(D, W * P, device=DEV)
    lens0 = [250, 31, 16, 100, 1, 77]
    kc0, vc0, table0, ctx0 = _paged(B, Hkv, D, P, lens0, BF, 5, spare=40)
    W = table0.shape[1]
    used = table0[table0 >= 0].tolist()
    free0 = torch.tensor([p for p in range(kc0.shape[0]) if p not in used] + used, dtype=torch.int32)
    n0 = torch.tensor([kc0.shape[0] - len(used)], dtype=torch.int32)
    b0 = _bounds_of(kc0, table0, ctx0, P)
    static = [t.to(DEV) for t in (kc0, vc0, table0, ctx0, free0, n0, b0)]
    x = torch.empty(B, Hq + 2 * Hkv, D, dtype=BF, device=DEV)
    ones = torch.ones(B, dtype=torch.int32, device=DEV)

    def step(state, x):
        kc, vc, table, ctx, free, n_free, bounds = state
        q, k, v = x.split([Hq, Hkv, Hkv], 1)
        r = smooth_attn.sp2norm_paged_reserve(table, ctx, ones, free, n_free, B)
        qr = smooth_attn.sp2norm_paged_qk_norm_rope_append(q, k, v, None, None, cos, sin, r.positions, r.slots, kc, vc)
        smooth_attn.sp2norm_paged_key_bounds(kc, table, ctx, r.context_lens, bounds)
        pages = smooth_attn.sp2norm_paged_select_pages(qr[:, :, None], bounds, table, r.context_lens, top_k)
        o = smooth_attn.sp2norm_paged_sparse_attention(qr[:, :, None], kc, vc, table, r.context_lens, pages)
        ctx.copy_(r.context_lens)
        n_free.copy_(r.n_free)
        return o, pages

    x.copy_(_randn(x.shape, BF, 1))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(static, x)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step(static, x)
    for d, s in zip(static, (kc0, vc0, table0, ctx0, free0, n0, b0)):
        d.copy_(s)
    eager = [t.to(DEV) for t in (kc0, vc0, table0, ctx0, free0, n0, b0)]
    for i in range(20):  # past a page's end
        x.copy_(_randn(x.shape, BF, 30 + i))
        graph.replay()
        torch.cuda.synchronize()
        want = step(eager, x.clone())
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1]), i
    for a, b in zip(static, eager):
        torch.testing.assert_close(a, b, rtol=0, atol=0, equal_nan=True)


def test_offsets_past_32_bits():
    # a cache of over 2^31 bytes a head and pages at its far end
    P, D, Hkv = 64, 128, 2
    n_pages = 150_000  # 150000 * 2 * 64 * 128 * 2 bytes = 4.9 GB
    kc = torch.zeros(n_pages, Hkv, P, D, dtype=BF, device=DEV)
    vc = torch.zeros(n_pages, Hkv, P, D, dtype=BF, device=DEV)
    ids = [n_pages - 1, 3, n_pages - 2, 70_000]
    table = torch.tensor([ids], dtype=torch.int32, device=DEV)
    lens = torch.tensor([4 * P - 5], dtype=torch.int32, device=DEV)
    N = 4 * P - 5
    x = _randn((N, 4 + 2 * Hkv, D), BF, 1).to(DEV)
    q, k, v = x.split([4, Hkv, Hkv], 1)
    pos = torch.arange(N, dtype=torch.int32, device=DEV)
    slots = table[0, (pos // P).long()] * P + pos % P
    cos, sin = smooth_attn.precompute_rope_cos_sin(D, N, device=DEV)
    smooth_attn.sp2norm_paged_qk_norm_rope_append(q, k, v, None, None, cos, sin, pos, slots, kc, vc, block_size=P)
    bounds = smooth_attn.sp2norm_paged_key_bounds(kc, table, torch.zeros_like(lens), lens, block_size=P)
    q1 = q[-1:][:, :, None]
    pages = smooth_attn.sp2norm_paged_select_pages(q1, bounds, table, lens, 3, block_size=P)
    o = smooth_attn.sp2norm_paged_sparse_attention(q1, kc, vc, table, lens, pages, block_size=P)
    # the same in a small cache
    small = [c[torch.tensor(ids, device=DEV)].contiguous() for c in (kc, vc)]
    t2 = torch.arange(4, dtype=torch.int32, device=DEV)[None]
    yk = serving.qk_norm_rope(k.cpu().double(), None, cos.cpu().double()[:, None], sin.cpu().double()[:, None])
    stored = small[0].transpose(1, 2).reshape(-1, Hkv, D)[:N].cpu().double()
    assert ((stored - yk).abs() <= _half_step(BF) * yk.abs() + 1e-4).all()
    assert torch.equal(small[1].transpose(1, 2).reshape(-1, Hkv, D)[:N], v)
    b2 = smooth_attn.sp2norm_paged_key_bounds(small[0], t2, torch.zeros_like(lens), lens, block_size=P)
    assert torch.equal(b2, bounds[torch.tensor(ids, device=DEV)])
    p2 = smooth_attn.sp2norm_paged_select_pages(q1, b2, t2, lens, 3, block_size=P)
    assert torch.equal(p2, pages)
    assert torch.equal(smooth_attn.sp2norm_paged_sparse_attention(q1, *small, t2, lens, p2, block_size=P), o)
