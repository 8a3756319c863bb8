"""Refusals of the norm and serving operators, on the CPU: argument errors are
raised before anything is launched, by the Python entry points and by the C ABI."""
import ctypes
import inspect

import pytest
import torch

import smooth_attn
from smooth_attn import _lib, qk_norm, serving

BF, F32, I32 = torch.bfloat16, torch.float32, torch.int32


def z(*shape, dtype=BF):
    return torch.zeros(shape, dtype=torch.uint8 if dtype == torch.float8_e4m3fn else dtype).view(dtype) \
        if dtype == torch.float8_e4m3fn else torch.zeros(shape, dtype=dtype)


def test_names_are_reached_from_the_package():
    for mod in (qk_norm, serving):
        for name in mod.__all__:
            assert getattr(smooth_attn, name) is getattr(mod, name)
    sig = inspect.signature(smooth_attn.sp2norm_qk_norm_rope)
    assert list(sig.parameters) == ["q", "k", "q_weight", "k_weight", "cos", "sin", "positions", "eps"]


def norm(q=None, k=None, qw=None, kw=None, cos=None, sin=None, **kw_):
    return smooth_attn.sp2norm_qk_norm_rope(z(2, 4, 8, 32) if q is None else q, z(2, 2, 8, 32) if k is None else k, qw, kw,
                                            z(8, 16, dtype=F32) if cos is None else cos,
                                            z(8, 16, dtype=F32) if sin is None else sin, **kw_)


@pytest.mark.parametrize("kwargs,match", [
    (dict(), "CUDA tensor"),
    (dict(q=z(4, 8, 32)), "B, H, T, D"),
    (dict(k=z(2, 2, 9, 32)), "k must be"),
    (dict(k=z(2, 2, 8, 32, dtype=F32)), "dtype"),
    (dict(q=z(2, 4, 8, 32, dtype=torch.float64), k=z(2, 2, 8, 32, dtype=torch.float64)), "dtype"),
    (dict(q=z(2, 4, 8, 40), k=z(2, 2, 8, 40), cos=z(8, 20, dtype=F32), sin=z(8, 20, dtype=F32)), "multiples of 16"),
    (dict(q=z(2, 4, 8, 528), k=z(2, 2, 8, 528)), "multiples of 16"),
    (dict(qw=z(16)), "q_weight"),
    (dict(kw=z(32, dtype=torch.float16)), "k_weight"),
    (dict(cos=z(8, 32, dtype=F32)), "cos and sin"),
    (dict(sin=z(7, 16, dtype=F32)), "cos and sin"),
    (dict(cos=z(7, 16, dtype=F32), sin=z(7, 16, dtype=F32)), "row for each"),
    (dict(cos=z(8, 16, dtype=I32), sin=z(8, 16, dtype=I32)), "floating point"),
    (dict(cos=torch.zeros(8, 16, requires_grad=True)), "no gradient"),
    (dict(positions=z(2, 7, dtype=I32)), "positions must be"),
    (dict(positions=z(2, 8, dtype=F32)), "integer"),
    (dict(positions=z(8, dtype=torch.bool)), "integer"),
    (dict(q=z(1, 1, 1, 16).expand(1 << 13, 1, 1 << 12, 16), k=z(1, 1, 1, 16).expand(1 << 13, 1, 1 << 12, 16),
          cos=z(1, 8, dtype=F32), sin=z(1, 8, dtype=F32)), "tokens"),
])
def test_norm_refusals(kwargs, match):
    with pytest.raises(ValueError, match=match):
        norm(**kwargs)


def test_non_tensors():
    with pytest.raises(TypeError, match="k must be a torch.Tensor"):
        norm(k=[1.0])
    with pytest.raises(TypeError):
        smooth_attn.sp2norm_paged_reserve([[0]], z(1, dtype=I32), z(1, dtype=I32), z(4, dtype=I32), z(1, dtype=I32), 4)


def reserve(table=None, lens=None, new=None, free=None, n_free=None, n=8, **kw):
    pick = lambda t, *s: z(*s, dtype=I32) if t is None else t  # noqa: E731
    return smooth_attn.sp2norm_paged_reserve(pick(table, 3, 4), pick(lens, 3), pick(new, 3), pick(free, 9), pick(n_free, 1),
                                             n, **kw)


@pytest.mark.parametrize("kwargs,match", [
    (dict(), "CUDA tensor"),
    (dict(table=z(3, 4, dtype=torch.int64)), "block_table must be"),
    (dict(table=z(12, dtype=I32)), "block_table must be"),
    (dict(table=z(4, 3, dtype=I32).t()), "consecutive"),
    (dict(table=z(1, 4, dtype=I32).expand(3, 4)), "overlap"),
    (dict(table=z(4097, 1, dtype=I32)), "at most 4096"),
    (dict(lens=z(4, dtype=I32)), "context_lens"),
    (dict(new=z(2, dtype=I32)), "new_lens"),
    (dict(free=z(9, dtype=torch.int64)), "free_pages"),
    (dict(free=z(18, dtype=I32)[::2]), "free_pages"),
    (dict(n_free=z(2, dtype=I32)), "n_free"),
    (dict(n=-1), "n_tokens"),
    (dict(block_size=0), "block_size"),
    (dict(block_size=1 << 28), "32-bit"),
])
def test_reserve_refusals(kwargs, match):
    with pytest.raises(ValueError, match=match):
        reserve(**kwargs)


def test_release_refusals():
    args = (z(3, 4, dtype=I32), z(3, dtype=I32), z(3, dtype=torch.bool), z(9, dtype=I32), z(1, dtype=I32))
    with pytest.raises(ValueError, match="CUDA tensor"):
        smooth_attn.sp2norm_paged_release(*args)
    with pytest.raises(ValueError, match="bool"):
        smooth_attn.sp2norm_paged_release(args[0], args[1], z(3, dtype=I32), *args[3:])
    with pytest.raises(ValueError, match="finished"):
        smooth_attn.sp2norm_paged_release(args[0], args[1], z(2, dtype=torch.bool), *args[3:])


def append(q=None, k=None, v=None, kc=None, vc=None, pos=None, slots=None, cos=None, **kw):
    d = lambda t, *s, dt=BF: z(*s, dtype=dt) if t is None else t  # noqa: E731
    cos = d(cos, 8, 16, dt=F32)
    return smooth_attn.sp2norm_paged_qk_norm_rope_append(
        d(q, 5, 4, 32), d(k, 5, 2, 32), d(v, 5, 2, 32), None, None, cos, cos, d(pos, 5, dt=I32), d(slots, 5, dt=I32),
        d(kc, 3, 2, 16, 32), d(vc, 3, 2, 16, 32), **kw)


@pytest.mark.parametrize("kwargs,match", [
    (dict(), "CUDA tensor"),
    (dict(q=z(5, 4, 1, 32)), "q must be"),
    (dict(v=z(5, 3, 32)), "q must be"),
    (dict(k=z(4, 2, 32), v=z(4, 2, 32)), "q must be"),
    (dict(v=z(5, 2, 32, dtype=F32)), "dtype"),
    (dict(kc=z(3, 2, 8, 32)), "k_cache"),
    (dict(vc=z(3, 2, 16, 32, dtype=F32)), "one dtype"),
    (dict(kc=z(3, 1, 16, 32), vc=z(3, 1, 16, 32)), "k_cache and v_cache"),
    (dict(kc=z(3, 2, 16, 32, dtype=torch.int8)), "paged caches"),
    (dict(kc=z(3, 2, 16, 33)[..., 1:]), "16-byte"),
    (dict(pos=z(4, dtype=I32)), "positions"),
    (dict(slots=z(5, dtype=F32)), None),
    (dict(cos=z(0, 16, dtype=F32)), "no rows"),
])
def test_append_refusals(kwargs, match):
    with pytest.raises(ValueError, match=match):
        append(**kwargs)


def test_bounds_refusals():
    kc, t, n = z(3, 2, 16, 32), z(2, 4, dtype=I32), z(2, dtype=I32)
    call = smooth_attn.sp2norm_paged_key_bounds
    for args, kw, match in [
        ((kc, t, n, n), {}, "CUDA tensor"),
        ((kc[0], t, n, n), {}, "k_cache"),
        ((kc, t, n, n), dict(block_size=8), "k_cache"),
        ((z(3, 2, 12, 32), t, n, n), dict(block_size=12), "power of two"),
        ((z(3, 2, 16, 36), t, n, n), {}, "head dims"),
        ((z(3, 2, 16, 24, dtype=torch.float8_e4m3fn), t, n, n), {}, "head dims"),
        ((kc, t[0], n, n), {}, "block_table"),
        ((kc, t, n[:1], n), {}, "from_lens"),
        ((kc, t, n, n.float()), {}, "integer"),
        ((kc, t, n, n, z(3, 2, 2, 16)), {}, "bounds"),
        ((kc, t, n, n, z(3, 2, 2, 32, dtype=F32)), {}, "bounds"),
        ((kc, t, n, n, z(3, 2, 2, 64)[..., :32]), {}, "bounds"),
    ]:
        with pytest.raises(ValueError, match=match):
            call(*args, **kw)


def test_select_and_attention_refusals():
    q, b, t, n = z(2, 4, 1, 32), z(3, 2, 2, 32), z(2, 4, dtype=I32), z(2, dtype=I32)
    call = smooth_attn.sp2norm_paged_select_pages
    for args, kw, match in [
        ((q, b, t, n, 2), {}, "CUDA tensor"),
        ((z(2, 4, 2, 32), b, t, n, 2), {}, "q must be"),
        ((q, b[:, :, 0], t, n, 2), {}, "bounds"),
        ((z(2, 3, 1, 32), b, t, n, 2), {}, "multiple of H_kv"),
        ((q.to(torch.int8), b, t, n, 2), {}, "q must be"),
        ((q, b, t, n, 0), dict(n_last=0), "top_k"),
        ((q, b, t, n, 2), dict(n_first=2), "top_k"),
        ((q, b, t, n, 2), dict(n_last=-1), "top_k"),
        ((q, b, t, n, 2), dict(block_size=24), "power of two"),
        ((q, b, t[:1], n, 2), {}, "block_table"),
        ((q, b, t, n[:1], 2), {}, "context_lens"),
    ]:
        with pytest.raises(ValueError, match=match):
            call(*args, **kw)
    kc, pages = z(3, 2, 16, 32), z(2, 2, 5, dtype=I32)
    call = smooth_attn.sp2norm_paged_sparse_attention
    for args, kw, match in [
        ((q, kc, kc, t, n, pages), {}, "CUDA tensor"),
        ((q[:, :, 0], kc, kc, t, n, pages), {}, "q must be"),
        ((q, kc, kc, t, n, pages[:, :1]), {}, "pages"),
        ((q, kc, kc, t, n, pages.float()), {}, None),
        ((q, kc, kc.float(), t, n, pages), {}, "one dtype"),
        ((z(2, 3, 1, 32), kc, kc, t, n, pages), {}, "H_q"),
        ((z(2, 66, 1, 32), kc, kc, t, n, pages), {}, "1 to 32"),
        ((z(2, 4, 1, 36), z(3, 2, 16, 36), z(3, 2, 16, 36), t, n, pages), {}, "head dim"),
        ((q, kc, kc, t, n, pages), dict(block_size=32), "k_cache"),
    ]:
        with pytest.raises(ValueError, match=match):
            call(*args, **kw)


# ---------------------------------------------------------------------------
# The C ABI: status codes before any HIP call (pointers are 16-byte aligned
# dummies that nothing dereferences).
# ---------------------------------------------------------------------------
D16, BAD = ctypes.c_void_p(16), ctypes.c_void_p(18)


def _s(*v):
    return (ctypes.c_int64 * len(v))(*v)


def test_norm_abi_errors():
    lib = _lib.load()
    good = _s(4 * 8 * 64, 8 * 64, 64, 1)

    def fwd(q=D16, B=0, Hq=4, T=8, D=64, n_pos=8, s=good, dt=_lib.SA_BF16, w=_lib.SA_BF16, cos=D16):
        return lib.sa_qk_norm_rope_fwd(q, D16, D16, D16, None, None, cos, D16, None, 0, B, Hq, 2, T, D, n_pos, s, good,
                                       good, good, 1e-6, dt, w, None)

    assert fwd() == 0
    assert fwd(B=-1) == -2 and fwd(D=72) == -6 and fwd(D=528) == -6 and fwd(dt=7) == -3
    assert fwd(w=_lib.SA_F16) == -3 and fwd(B=1, q=None) == -1 and fwd(B=1, cos=None) == -1
    assert fwd(B=1, n_pos=0) == -2 and fwd(B=1, q=BAD) == -5 and fwd(B=1, s=_s(2048, 512, 63, 1)) == -5
    assert fwd(B=1, s=_s(2048, 512, 64, 2)) == -5 and fwd(B=1 << 20, T=32) == -2 and fwd(B=1, Hq=20000) == -2
    size = lib.sa_qk_norm_rope_bwd_workspace_size(2, 32, 8, 1024, 128)
    assert size > 0 and size % (128 * 4) == 0 and lib.sa_qk_norm_rope_bwd_workspace_size(0, 32, 8, 1024, 128) == 0

    def bwd(B=1, dw=D16, ws=D16, nbytes=1 << 40):
        return lib.sa_qk_norm_rope_bwd(D16, D16, D16, D16, D16, None, dw, None, None, None, D16, D16, None, 0, B, 4, 2, 8,
                                       64, 8, good, good, good, good, good, good, 1e-6, _lib.SA_BF16, _lib.SA_BF16, ws,
                                       nbytes, None)

    assert bwd() == -1  # no dk
    assert bwd(B=0) == -6 and bwd(B=0, dw=None) == 0


def test_maps_abi_errors():
    lib = _lib.load()

    def res(B=2, W=4, P=16, n_pages=8, n=4, stride=4, table=D16, out=D16):
        return lib.sa_paged_reserve(table, D16, D16, D16, D16, out, D16, D16, D16, D16, D16, B, W, P, n_pages, n, stride,
                                    None)

    assert res(B=-1) == -2 and res(B=4097) == -6 and res(P=0) == -2 and res(n=-1) == -2 and res(stride=3) == -5
    assert res(n_pages=1 << 28) == -2 and res(W=1 << 28, stride=1 << 28) == -2 and res(table=None) == -1
    assert res(out=None) == -1
    rel = lambda B: lib.sa_paged_release(D16, D16, None, D16, D16, D16, D16, D16, B, 4, 16, 8, 4, None)  # noqa: E731
    assert rel(2) == -1 and rel(0) == -2 and rel(4097) == -6


def test_append_bounds_select_sparse_abi_errors():
    lib = _lib.load()
    t3, t4 = _s(256, 64, 1), _s(2048, 1024, 64, 1)

    def app(N=4, D=64, P=16, pages=8, kc=t4, cache=_lib.SA_BF16, slots=D16):
        return lib.sa_paged_qk_norm_rope_append(D16, D16, D16, D16, D16, D16, None, None, D16, D16, D16, slots, N, 4, 2, D,
                                                8, P, pages, t3, t3, t3, t3, kc, t4, 1e-6, _lib.SA_BF16, _lib.SA_BF16,
                                                cache, None)

    assert app(N=0) == 0 and app(N=-1) == -2 and app(D=24) == -6 and app(P=0) == -2 and app(pages=1 << 28) == -2
    assert app(cache=9) == -3 and app(slots=None) == -1 and app(kc=_s(2048, 1024, 60, 1)) == -5
    assert app(cache=_lib.SA_FP8_E4M3FN, kc=_s(2048, 1024, 72, 1)) == -5

    def bnd(B=2, D=64, P=16, W=4, stride=4, cache=_lib.SA_BF16, k=D16, s=t4):
        return lib.sa_paged_key_bounds(k, D16, D16, D16, D16, B, 2, D, P, W, 8, s, stride, cache, None)

    assert bnd(B=0) == 0 and bnd(B=-1) == -2 and bnd(P=24) == -6 and bnd(D=12) == -6 and bnd(D=1032) == -6
    assert bnd(cache=5) == -3 and bnd(stride=3) == -5 and bnd(k=None) == -1 and bnd(k=BAD) == -5
    assert bnd(W=1 << 27, stride=1 << 27) == -6 and bnd(cache=_lib.SA_FP8_E4M3FN, D=24) == -6

    def sel(B=2, Hq=4, K=2, first=0, last=1, W=4, ws=D16, nbytes=1 << 40, dt=_lib.SA_BF16, pages=D16, q=D16, s=t4):
        return lib.sa_paged_select_pages(q, D16, D16, D16, pages, B, Hq, 2, 64, 16, W, 8, K, first, last, s, W, dt,
                                         _lib.SA_BF16, ws, nbytes, None)

    assert sel(q=BAD) == -5 and sel(s=_s(2048, 60, 64, 1)) == -5 and sel(s=_s(2048, 64, 64, 2)) == -5
    assert sel(B=1 << 21) == -6

    assert sel(B=0) == 0 and sel(K=0, last=0) == 0 and sel(Hq=3) == -2 and sel(K=-1) == -2 and sel(first=2) == -2
    assert sel(last=-1) == -2 and sel(dt=3) == -3 and sel(pages=None) == -1 and sel(nbytes=8) == -7 and sel(ws=None) == -7
    assert lib.sa_paged_select_workspace_size(2, 8, 1000) == 2 * 8 * 1000 * 8

    def sparse(B=2, n=3, P=16, W=4, ws=D16, nbytes=1 << 40, pages=D16, dt=_lib.SA_BF16, Hq=4):
        return lib.sa_paged_sparse_decode(D16, D16, D16, D16, D16, D16, pages, B, Hq, 2, 64, P, W, 8, n, t4, t4, t4, t3, W,
                                          0.1, dt, ws, nbytes, None)

    assert sparse(B=0) == 0 and sparse(n=-1) == -2 and sparse(P=24) == -6 and sparse(nbytes=16) == -7
    assert sparse(ws=None) == -1 and sparse(pages=None) == -1 and sparse(dt=9) == -3 and sparse(Hq=66) == -6
    assert sparse(n=1 << 28) == -6
