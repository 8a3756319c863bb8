"""The native call path of the norm and serving operators against the Python
path: the same bits and gradients, the same refusals, and which calls it takes."""
import threading

import pytest
import torch
from torch.utils.checkpoint import checkpoint

import smooth_attn
from smooth_attn import _lib, qk_norm, serving

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, HF, F32, FP8 = torch.bfloat16, torch.float16, torch.float32, torch.float8_e4m3fn


class _Counting:
    """The native path, counting the calls that it took."""

    def __init__(self):
        self.took = 0

    def __getattr__(self, name):
        fn = getattr(_lib.host(), name)

        def call(*a):
            r = fn(*a)
            self.took += r is not None and r is not False
            return r
        return call


def both(monkeypatch, call):
    """call() on the Python path and on the native one: (Python, native, times the native path took it)."""
    got = []
    for nat in (_lib.NothingOrdinary, _Counting()):
        for mod in (qk_norm, serving):
            monkeypatch.setattr(mod, "_native", lambda nat=nat: nat)
        try:
            got.append(call())
        except Exception as e:  # noqa: BLE001
            got.append(e)
    monkeypatch.undo()
    return got[0], got[1], nat.took


def same(a, b):
    if isinstance(a, Exception) or isinstance(b, Exception):
        assert type(a) is type(b) and str(a) == str(b), (a, b)
        return
    if isinstance(a, torch.Tensor):
        assert a.dtype == b.dtype and a.shape == b.shape and a.stride() == b.stride()
        assert a.requires_grad == b.requires_grad
        a, b = (t.detach().contiguous().view(-1).view(torch.uint8) for t in (a, b))
        assert torch.equal(a, b)
        return
    assert type(a) is type(b) and len(a) == len(b)
    for x, y in zip(a, b):
        same(x, y)


def _randn(shape, dtype, seed, scale=1.0):
    x = torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * scale
    return x.to(dtype).to(DEV)


def _norm_args(dtype, B=2, Hq=8, Hkv=2, T=33, D=64, layout="bthd", weights="same", grad=True):
    def heads(H, seed):
        x = _randn((B, T, H, D) if layout == "bthd" else (B, H, T, D), dtype, seed)
        return x.transpose(1, 2) if layout == "bthd" else x

    wdt = F32 if weights == "fp32" else dtype
    w = [None, None] if weights == "none" else [1 + 0.2 * _randn((D,), wdt, s) for s in (3, 4)]
    if weights == "one":
        w[0] = None
    cos, sin = smooth_attn.precompute_rope_cos_sin(D, T, device=DEV)
    args = [heads(Hq, 1), heads(Hkv, 2), *w]
    return [None if t is None else t.detach().requires_grad_(grad) for t in args], cos, sin


@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("layout", ["bthd", "bhtd"])
@pytest.mark.parametrize("weights", ["same", "fp32", "none", "one"])
@pytest.mark.parametrize("positions", [None, "T", "BT"])
def test_norm_and_gradients(monkeypatch, dtype, layout, weights, positions):
    args, cos, sin = _norm_args(dtype, layout=layout, weights=weights)
    gen = torch.Generator().manual_seed(9)
    pos = None if positions is None else \
        torch.randint(0, 33, (33,) if positions == "T" else (2, 33), generator=gen).to(torch.int32).to(DEV)

    def call():
        y = smooth_attn.sp2norm_qk_norm_rope(*args, cos, sin, positions=pos)
        return list(y) + list(torch.autograd.grad(y, [t for t in args if t is not None],
                                                  [_randn(t.shape, dtype, 20) for t in y]))

    a, b, took = both(monkeypatch, call)
    same(a, b)
    assert took == 1


def test_norm_calls_that_python_takes(monkeypatch):
    args, cos, sin = _norm_args(BF)
    q, k, qw, kw = args
    odd = torch.zeros(q.numel() + 1, dtype=BF, device=DEV)[1:].view(q.shape)
    forms = [
        (q, k, qw.detach().float(), kw, cos, sin),       # weights of two types
        (odd, k, qw, kw, cos, sin),                      # not aligned
        (q, k, qw, kw, cos.double(), sin),               # tables of another type
        (q.transpose(2, 3).contiguous().transpose(2, 3), k, qw, kw, cos, sin),
        (q[:, :0], k, qw, kw, cos, sin),                 # nothing
    ]
    for form in forms:
        a, b, took = both(monkeypatch, lambda: smooth_attn.sp2norm_qk_norm_rope(*form))
        assert not isinstance(a, Exception), a
        same(a, b)
        assert took == 0
    pos = torch.arange(33, device=DEV)  # 64 bits
    a, b, took = both(monkeypatch, lambda: smooth_attn.sp2norm_qk_norm_rope(*args, cos, sin, positions=pos))
    same(a, b)
    assert took == 0
    for bad in [(q, k.float(), qw, kw, cos, sin), (q, k, qw[:32], kw, cos, sin), (q, k, qw, kw, cos[:5], sin[:5]),
                (q.cpu(), k, qw, kw, cos, sin), (q, k, qw, kw, cos.clone().requires_grad_(True), sin), (q, [1], qw, kw, cos, sin)]:
        a, b, took = both(monkeypatch, lambda: smooth_attn.sp2norm_qk_norm_rope(*bad))
        assert isinstance(a, (ValueError, TypeError))
        same(a, b)
        assert took == 0


def test_norm_modes(monkeypatch):
    args, cos, sin = _norm_args(BF)
    call = lambda: smooth_attn.sp2norm_qk_norm_rope(*args, cos, sin)  # noqa: E731
    with torch.no_grad():
        a, b, took = both(monkeypatch, call)
        same(a, b)
        assert took == 1 and not b[0].requires_grad
    # checkpointing runs forward again in backward
    f = lambda q, k, qw, kw: sum(t.float().square().sum() for t in smooth_attn.sp2norm_qk_norm_rope(q, k, qw, kw, cos, sin))  # noqa: E731
    plain = torch.autograd.grad(f(*args), args)
    again = torch.autograd.grad(checkpoint(f, *args, use_reentrant=False), args)
    same(list(plain), list(again))
    # only some gradients are asked for
    y = call()
    (dkw,) = torch.autograd.grad(y[1].float().sum(), args[3])
    y = call()
    full = torch.autograd.grad(y[1].float().sum(), args, allow_unused=True)
    same(dkw, full[3])
    # a second derivative is refused on both paths
    for nat in (_lib.NothingOrdinary, _lib.host()):
        for mod in (qk_norm, serving):
            monkeypatch.setattr(mod, "_native", lambda nat=nat: nat)
        x = args[0].detach().float().requires_grad_(True)
        yq, yk = smooth_attn.sp2norm_qk_norm_rope(x, x, None, None, cos, sin)
        (g,) = torch.autograd.grad(yq.square().sum() + yk.sum(), x, create_graph=True)
        with pytest.raises(RuntimeError, match="differentiate twice"):
            g.sum().backward()
        (g,) = torch.autograd.grad(smooth_attn.sp2norm_qk_norm_rope(x, x, None, None, cos, sin)[0].sum(), x,
                                   create_graph=True)  # (of a constant gradient: nothing to refuse)
        assert not g.requires_grad
    monkeypatch.undo()


def test_norm_hooks_on_the_native_path():
    args, cos, sin = _norm_args(BF)

    def run(unpack):
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, unpack):
            y = smooth_attn.sp2norm_qk_norm_rope(*args, cos, sin)
        return list(torch.autograd.grad(y, args, [torch.ones_like(t) for t in y]))

    want = run(lambda t: t)
    got = run(lambda t: t.transpose(-1, -2).contiguous().transpose(-1, -2) if t.ndim == 4 else t)
    for a, b in zip(want, got):
        assert torch.equal(a, b)
    for bad in (lambda t: t.double() if t.ndim == 4 else t, lambda t: t.cpu(), lambda t: t[..., :-16],
                lambda t: t[:, :1] if t.ndim == 4 else t):
        with pytest.raises(ValueError):
            run(bad)


def _caches(dtype, n_pages=40, Hkv=2, P=16, D=64):
    src = BF if dtype == FP8 else dtype
    return [_randn((n_pages, Hkv, P, D), src, s).to(dtype) for s in (1, 2)]


@pytest.mark.parametrize("dtype,cache", [(BF, BF), (HF, HF), (F32, F32), (BF, FP8), (HF, F32)])
def test_append(monkeypatch, dtype, cache):
    N, Hq, Hkv, D, P = 21, 8, 2, 64, 16
    x = _randn((N, Hq + 2 * Hkv, D), dtype, 3)
    q, k, v = x.split([Hq, Hkv, Hkv], 1)
    w = 1 + 0.1 * _randn((D,), dtype, 4)
    cos, sin = smooth_attn.precompute_rope_cos_sin(D, 64, device=DEV)
    pos = torch.arange(N, dtype=torch.int32, device=DEV)
    slots = torch.randperm(640, generator=torch.Generator().manual_seed(1))[:N].to(torch.int32).to(DEV)

    def call(slots=slots):
        kc, vc = _caches(cache)
        out = smooth_attn.sp2norm_paged_qk_norm_rope_append(q, k, v, w, None, cos, sin, pos, slots, kc, vc)
        return [out, kc, vc]

    a, b, took = both(monkeypatch, call)
    same(a, b)
    assert took == 1
    a, b, took = both(monkeypatch, lambda: call(slots.long()))
    same(a, b)
    assert took == 0


def test_maps(monkeypatch):
    B, W = 9, 6
    lens = torch.tensor([0, 5, 16, 17, 40, 96, 1, 2, 3], dtype=torch.int32, device=DEV)
    new = torch.tensor([3, 30, 0, 1, 7, 9, 20, 1, 1], dtype=torch.int32, device=DEV)
    free = torch.randperm(80, generator=torch.Generator().manual_seed(2)).to(torch.int32).to(DEV)
    n_free = torch.tensor([50], dtype=torch.int32, device=DEV)
    base = free[50:].repeat(2)[:B * W].view(B, W).contiguous()

    def step(lens=lens, finished=lens > 30, room=80):
        table, f = base.clone(), free.clone()
        ln, n = smooth_attn.sp2norm_paged_release(table, lens, finished, f, n_free)
        r = smooth_attn.sp2norm_paged_reserve(table, ln, new, f, n, room)
        return [table, f, ln, n, r]

    a, b, took = both(monkeypatch, step)
    same(a, b)
    assert took == 2 and isinstance(b[4], smooth_attn.PagedReservation)
    a, b, took = both(monkeypatch, lambda: step(lens=lens.long()))
    same(a, b)
    assert took == 1  # (release's lengths are 32-bit)
    a, b, took = both(monkeypatch, lambda: step(room=True))
    same(a, b)
    for bad in (dict(finished=lens), dict(room=-1), dict(lens=lens[:4])):
        a, b, took = both(monkeypatch, lambda: step(**bad))
        assert isinstance(a, ValueError)
        same(a, b)


@pytest.mark.parametrize("qt,ct", [(BF, BF), (HF, HF), (F32, F32), (BF, FP8), (F32, BF), (FP8, FP8)])
def test_sparse(monkeypatch, qt, ct):
    kc, vc = _caches(ct)
    table = torch.randperm(40, generator=torch.Generator().manual_seed(3)).to(torch.int32).to(DEV).view(2, 20)
    lens = torch.tensor([300, 77], dtype=torch.int32, device=DEV)
    q = _randn((2, 8, 1, 64), F32 if qt == FP8 else qt, 5).to(qt)

    def call(table=table, lens=lens, top_k=6, scale=None, bounds=None, **kw):
        if bounds is None:
            bounds = torch.zeros(40, 2, 2, 64, dtype=torch.uint8, device=DEV).view(FP8) if ct == FP8 else \
                torch.zeros(40, 2, 2, 64, dtype=ct, device=DEV)
        b = smooth_attn.sp2norm_paged_key_bounds(kc, table, torch.zeros_like(lens), lens, bounds)
        pages = smooth_attn.sp2norm_paged_select_pages(q, b, table, lens, top_k, **kw)
        return [b, pages, smooth_attn.sp2norm_paged_sparse_attention(q, kc, vc, table, lens, pages, scale=scale)]

    a, b, took = both(monkeypatch, call)
    same(a, b)
    assert took == 1 + (qt != FP8) + ((qt, ct) in ((BF, BF), (HF, HF), (F32, F32), (BF, FP8)))
    for kw in (dict(table=table.long()), dict(lens=lens.long()), dict(table=table.t().contiguous().t()),
               dict(top_k=30, n_first=2, n_last=3), dict(scale=0.5), dict(scale=0)):
        a, b, _ = both(monkeypatch, lambda: call(**kw))
        assert not isinstance(a, Exception), a
        same(a, b)
    for kw in (dict(top_k=0), dict(n_last=9), dict(lens=lens[:1]), dict(table=table[:1]), dict(lens=lens.float()),
               dict(bounds=torch.zeros(40, 2, 2, 32, device=DEV))):
        a, b, _ = both(monkeypatch, lambda: call(**kw))
        assert isinstance(a, ValueError), kw
        same(a, b)


def test_threads_and_streams():
    args, cos, sin = _norm_args(BF)
    want = [t.detach() for t in smooth_attn.sp2norm_qk_norm_rope(*args, cos, sin)]
    torch.cuda.synchronize()
    got = {}

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                got[i] = [t.detach() for t in smooth_attn.sp2norm_qk_norm_rope(*args, cos, sin)]
            torch.cuda.current_stream().synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for i in range(4):
        same(want, got[i])
