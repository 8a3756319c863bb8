"""RMS norm + RoPE of queries and keys (HIP) against 64-bit forms (GPU).

Tolerances.  Everything is computed in fp32 and rounded once.  An output is off
by at most half a step of its type, eps_t / 2 relative, and by the fp32 errors
in front of it: z has a relative error of a few 2^-24 (a sum of squares of
positive terms over 16 values a lane and at most 5 steps across lanes, a
reciprocal root of one step, two products), and y = z_lo cos -+ z_hi sin adds
two products and a sum, so 2^-24 * 32 * (|z_lo| + |z_hi|) covers it.  The
gradient of x is r (h - n mean(h n)): the same with r (|h| + |n| mean|h n|).  A
weight's gradient sums R rows in 32 bits, at most R in sequence: 2^-24 (32 + R)
times the sum of the terms' absolute values.  fp16 outputs below its normal
range are off by half of 2^-24 at most.
"""
import pytest
import torch

import smooth_attn
from oracle import serving

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24


def _randn(shape, dtype, seed, scale=1.0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype)


def _check(got, want, terms, dtype, what):
    """got against want (64 bits); terms: the magnitudes that fp32 errors scale with."""
    tol = torch.finfo(dtype).eps / 2 * want.abs() + terms * (1 + torch.finfo(dtype).eps)
    if dtype == torch.float16:
        tol = tol + 2.0 ** -25
    err = (got.detach().cpu().double() - want).abs()
    worst = (err - tol).max().item() if err.numel() else 0.0
    assert worst <= 0, (what, worst, err.max().item())


def _tables(n, D, seed=5):
    angle = torch.rand(n, D // 2, generator=torch.Generator().manual_seed(seed)) * 100
    return angle.cos(), angle.sin()


def _reference(x, w, cos, sin, g, eps):
    """y, dx, dw in 64 bits by autograd, and the magnitudes of their errors."""
    x64 = x.double().requires_grad_(True)
    w64 = (torch.ones(x.shape[-1]) if w is None else w).double().requires_grad_(True)
    y = serving.qk_norm_rope(x64, w64, cos.double(), sin.double(), eps)
    dx, dw = torch.autograd.grad(y, (x64, w64), g.double()) if y.numel() else (torch.zeros_like(x64), torch.zeros_like(w64))
    with torch.no_grad():
        r = torch.rsqrt((x64 * x64).mean(-1, keepdim=True) + eps)
        n = x64 * r
        z = (n * w64).abs()
        half = x.shape[-1] // 2
        y_terms = U * 32 * (z + torch.cat([z[..., half:], z[..., :half]], -1))
        ga, gb = g.double().abs()[..., :half], g.double().abs()[..., half:]
        dz = torch.cat([ga * cos.abs() + gb * sin.abs(), gb * cos.abs() + ga * sin.abs()], -1)
        h = dz * w64.abs()
        dx_terms = U * 64 * r * (h + n.abs() * (h * n.abs()).mean(-1, keepdim=True))
        R = x[..., 0].numel()
        dw_terms = U * (32 + R) * (dz * n.abs()).flatten(0, -2).sum(0)
    return y.detach(), dx, dw, y_terms, dx_terms, dw_terms


CASES = [
    # B, Hq, Hkv, T, D, dtype, weights, layout
    (1, 1, 1, 1, 16, torch.bfloat16, "same", "bhtd"),
    (2, 4, 2, 33, 32, torch.float16, "same", "bthd"),
    (2, 12, 12, 65, 64, torch.bfloat16, "fp32", "bhtd"),
    (1, 32, 8, 1, 128, torch.bfloat16, "same", "bthd"),
    (3, 32, 8, 129, 128, torch.bfloat16, "fp32", "bthd"),
    (2, 5, 3, 77, 80, torch.bfloat16, "same", "bthd"),
    (2, 7, 1, 50, 48, torch.float16, "none", "bhtd"),
    (1, 6, 2, 40, 96, torch.float32, "same", "bthd"),
    (1, 3, 3, 20, 256, torch.bfloat16, "fp32", "bthd"),
    (1, 4, 1, 19, 512, torch.float16, "same", "bhtd"),
    (1, 2, 2, 18, 272, torch.float32, "none", "bthd"),
    (1, 2, 1, 2000, 64, torch.float32, "same", "bhtd"),
    (5, 16, 2, 300, 128, torch.float16, "fp32", "bhtd"),
]


@pytest.mark.parametrize("B,Hq,Hkv,T,D,dtype,weights,layout", CASES)
def test_forward_and_gradients(B, Hq, Hkv, T, D, dtype, weights, layout):
    def heads(H, seed, scale):
        x = _randn((B, T, H, D) if layout == "bthd" else (B, H, T, D), dtype, seed, scale)
        return x.transpose(1, 2) if layout == "bthd" else x

    q, k, gq, gk = heads(Hq, 1, 2.0), heads(Hkv, 2, 0.3), heads(Hq, 3, 1.0), heads(Hkv, 4, 1.0)
    wdt = dtype if weights == "same" else torch.float32
    qw, kw = (None, None) if weights == "none" else [(1 + 0.3 * _randn((D,), torch.float32, s)).to(wdt) for s in (6, 7)]
    cos, sin = _tables(T, D)
    to = lambda t: None if t is None else t.to(DEV).requires_grad_(True)  # noqa: E731
    dev = [to(t) for t in (q, k, qw, kw)]
    yq, yk = smooth_attn.sp2norm_qk_norm_rope(*dev, cos.to(DEV), sin.to(DEV))
    assert yq.dtype == dtype and yq.shape == q.shape and yk.shape == k.shape
    leaves = [t for t in dev if t is not None]
    grads = list(torch.autograd.grad((yq, yk), leaves, (gq.to(DEV), gk.to(DEV))))
    for x, w, g, y, i in ((q, qw, gq, yq, 0), (k, kw, gk, yk, 1)):
        ry, rdx, rdw, ty, tdx, tdw = _reference(x, w, cos, sin, g, 1e-6)
        _check(y, ry, ty, dtype, "y")
        _check(grads[i], rdx, tdx, dtype, "dx")
        if w is not None:
            assert grads[2 + i].dtype == wdt
            _check(grads[2 + i], rdw, tdw, wdt, "dw")


@pytest.mark.parametrize("per_sequence", [False, True])
@pytest.mark.parametrize("kind", [torch.int32, torch.int64])
def test_positions(per_sequence, kind):
    B, Hq, Hkv, T, D, n_pos = 3, 4, 2, 21, 64, 100
    q, k = _randn((B, Hq, T, D), torch.bfloat16, 1), _randn((B, Hkv, T, D), torch.bfloat16, 2)
    cos, sin = _tables(n_pos, D)
    pos = torch.randint(0, n_pos, (B, T) if per_sequence else (T,), generator=torch.Generator().manual_seed(3)).to(kind)
    pos.view(-1)[0], pos.view(-1)[1] = -5, n_pos + 7  # clamped to the tables
    p = pos.clamp(0, n_pos - 1)
    want = lambda x: serving.qk_norm_rope(x.double(), None, *(t.double()[p][:, None] if per_sequence else t.double()[p]  # noqa: E731
                                                              for t in (cos, sin)))
    yq, yk = smooth_attn.sp2norm_qk_norm_rope(q.to(DEV), k.to(DEV), None, None, cos.to(DEV), sin.to(DEV),
                                              positions=pos.to(DEV))
    for y, x in ((yq, q), (yk, k)):
        w = want(x)
        _check(y, w, U * 64 * x.double().abs().amax(-1, keepdim=True).expand_as(w) * 4, torch.bfloat16, "y")


def test_rows_of_zeros_and_of_large_values():
    D = 64
    q = torch.zeros(1, 2, 3, D)
    q[0, 1, 0] = 1e18  # its mean square is within fp32
    q[0, 1, 1] = 1e-30
    cos, sin = _tables(3, D)
    yq, yk = smooth_attn.sp2norm_qk_norm_rope(q.to(DEV), q.to(DEV), None, None, cos.to(DEV), sin.to(DEV))
    assert torch.equal(yq[0, 0].cpu(), torch.zeros(3, D)) and torch.isfinite(yq).all()
    assert abs(yq[0, 1, 0].square().mean().item() - 1) < 1e-5
    assert torch.equal(yq.cpu(), yk.cpu())
    x = torch.full((1, 1, 1, D), float("nan"))
    y, _ = smooth_attn.sp2norm_qk_norm_rope(x.to(DEV), x.to(DEV), None, None, cos.to(DEV), sin.to(DEV))
    assert torch.isnan(y).all()


def test_gradient_against_differences():
    # fp32 everywhere: (f(x + e d) - f(x - e d)) / 2e against <grad, d>
    B, Hq, Hkv, T, D = 1, 3, 1, 6, 32
    args = [_randn((B, Hq, T, D), torch.float32, 1), _randn((B, Hkv, T, D), torch.float32, 2),
            1 + 0.2 * _randn((D,), torch.float32, 3), 1 + 0.2 * _randn((D,), torch.float32, 4)]
    cos, sin = (t.to(DEV) for t in _tables(T, D))
    gq, gk = _randn((B, Hq, T, D), torch.float32, 5).to(DEV), _randn((B, Hkv, T, D), torch.float32, 6).to(DEV)

    def f(a):
        yq, yk = smooth_attn.sp2norm_qk_norm_rope(*a, cos, sin)
        return (yq * gq).double().sum() + (yk * gk).double().sum()

    dev = [a.to(DEV).requires_grad_(True) for a in args]
    grads = torch.autograd.grad(f(dev), dev)
    e = 2.0 ** -8
    for i, g in enumerate(grads):
        d = _randn(args[i].shape, torch.float32, 10 + i).to(DEV)
        up, down = ([t.detach() + s * e * d if j == i else t.detach() for j, t in enumerate(dev)] for s in (1, -1))
        diff = ((f(up) - f(down)) / (2 * e)).item()
        want = (g.double() * d.double()).sum().item()
        # differences: e^2 / 6 of a third derivative of a few times the terms, and 2^-24 of about 400 terms over e
        assert abs(diff - want) <= 2e-3 * (g.double() * d.double()).abs().sum().item() + 2e-2, (i, diff, want)


def test_gradients_of_a_broadcast_input_and_of_one_output():
    D, T = 64, 10
    base = _randn((1, 1, T, D), torch.float32, 1).to(DEV).requires_grad_(True)
    k = _randn((2, 2, T, D), torch.float32, 2).to(DEV).requires_grad_(True)
    w = torch.ones(D, device=DEV, requires_grad=True)
    cos, sin = (t.to(DEV) for t in _tables(T, D))
    q = base.expand(2, 4, T, D)  # one row for every head and sequence
    yq, yk = smooth_attn.sp2norm_qk_norm_rope(q, k, w, w, cos, sin)  # and one weight for both
    yq.sum().backward()  # (a gradient of stride 0; none of k's output)
    ref = base.detach().double().cpu().requires_grad_(True)
    w64 = torch.ones(D, dtype=torch.float64, requires_grad=True)
    y = serving.qk_norm_rope(ref.expand(2, 4, T, D), w64, cos.double().cpu(), sin.double().cpu())
    y.sum().backward()
    torch.testing.assert_close(base.grad.cpu().double(), ref.grad, rtol=1e-5, atol=1e-5)
    torch.testing.assert_close(w.grad.cpu().double(), w64.grad, rtol=1e-5, atol=1e-4)
    assert torch.equal(k.grad, torch.zeros_like(k))


def test_strided_and_unaligned_inputs_equal_contiguous_ones():
    B, H, T, D = 2, 4, 9, 64
    wide = _randn((B, T, 3 * H * D + 8), torch.bfloat16, 1).to(DEV)
    odd = _randn((B * T * H * D + 1,), torch.bfloat16, 2).to(DEV)[1:].view(B, H, T, D)  # 2 bytes past alignment
    q = wide[..., 8:8 + H * D].unflatten(-1, (H, D)).transpose(1, 2)
    cos, sin = (t.to(DEV) for t in _tables(T, D))
    w = _randn((2 * D + 1,), torch.bfloat16, 3).to(DEV)
    a = smooth_attn.sp2norm_qk_norm_rope(q, odd, w[1:D + 1], w[::2][:D], cos, sin)
    b = smooth_attn.sp2norm_qk_norm_rope(q.contiguous(), odd.clone(), w[1:D + 1].clone(), w[::2][:D].clone(), cos, sin)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_empty_inputs():
    cos, sin = (t.to(DEV) for t in _tables(4, 32))
    w = torch.ones(32, device=DEV, requires_grad=True)
    q = torch.zeros(0, 4, 4, 32, device=DEV, requires_grad=True)
    yq, yk = smooth_attn.sp2norm_qk_norm_rope(q, q[:, :2], w, w, cos, sin)
    assert yq.shape == (0, 4, 4, 32) and yk.shape == (0, 2, 4, 32)
    (yq.sum() + yk.sum()).backward()
    assert torch.equal(w.grad, torch.zeros(32, device=DEV))


def test_no_heads_on_one_side():
    cos, sin = (t.to(DEV) for t in _tables(4, 32))
    q, w = _randn((2, 3, 4, 32), torch.float32, 1).to(DEV).requires_grad_(True), torch.ones(32, device=DEV, requires_grad=True)
    a, none = smooth_attn.sp2norm_qk_norm_rope(q, q[:, :0], w, w, cos, sin)
    none2, b = smooth_attn.sp2norm_qk_norm_rope(q[:, :0], q, w, w, cos, sin)
    assert none.shape == none2.shape == (2, 0, 4, 32) and torch.equal(a, b)
    ga = torch.autograd.grad(a.square().sum() + none.sum(), (q, w))
    gb = torch.autograd.grad(b.square().sum() + none2.sum(), (q, w))
    assert all(torch.equal(x, y) for x, y in zip(ga, gb)) and ga[0].abs().sum() > 0


def test_other_stream_and_repeatable():
    B, H, T, D = 2, 8, 500, 128
    q, k = (_randn((B, H, T, D), torch.bfloat16, s).to(DEV).requires_grad_(True) for s in (1, 2))
    w = torch.ones(D, device=DEV, requires_grad=True)
    g = _randn((B, H, T, D), torch.bfloat16, 3).to(DEV)
    cos, sin = (t.to(DEV) for t in _tables(T, D))

    def step():
        y = smooth_attn.sp2norm_qk_norm_rope(q, k, w, w, cos, sin)
        return [t.detach() for t in y] + list(torch.autograd.grad(y, (q, k, w), (g, g)))

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want, got))


def test_second_derivative_is_refused():
    q = _randn((1, 2, 4, 32), torch.float32, 1).to(DEV).requires_grad_(True)
    cos, sin = (t.to(DEV) for t in _tables(4, 32))
    yq, yk = smooth_attn.sp2norm_qk_norm_rope(q, q, None, None, cos, sin)
    (g,) = torch.autograd.grad(yq.square().sum() + yk.sum(), q, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


def test_saved_tensor_hooks():
    B, H, T, D = 1, 4, 8, 64
    q, k = (_randn((B, H, T, D), torch.bfloat16, s).to(DEV).requires_grad_(True) for s in (1, 2))
    w = torch.ones(D, device=DEV, requires_grad=True)
    cos, sin = (t.to(DEV) for t in _tables(T, D))
    g = _randn((B, H, T, D), torch.bfloat16, 3).to(DEV)

    def run(unpack):
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, unpack):
            y = smooth_attn.sp2norm_qk_norm_rope(q, k, w, w, cos, sin)
        return torch.autograd.grad(y, (q, k, w), (g, g))

    want = run(lambda t: t)
    # another layout of the same values
    got = run(lambda t: t.transpose(-1, -2).contiguous().transpose(-1, -2) if t.ndim == 4 else t)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    with pytest.raises(ValueError, match="saved"):
        run(lambda t: t[:, :2] if t.ndim == 4 and t.shape[1] == H else t)
    with pytest.raises(ValueError, match="dtype"):
        run(lambda t: t.double() if t.ndim == 4 else t)


def test_feeds_the_fused_attention():
    # norm + rotation, then attention, with one backward through both
    B, Hq, Hkv, T, D = 2, 8, 2, 96, 64
    q, k, v = (_randn((B, T, H, D), torch.float32, s).to(DEV).transpose(1, 2).requires_grad_(True)
               for s, H in ((1, Hq), (2, Hkv), (3, Hkv)))
    w = (1 + 0.1 * _randn((D,), torch.float32, 4)).to(DEV).requires_grad_(True)
    cos, sin = smooth_attn.precompute_rope_cos_sin(D, T, device=DEV)
    go = _randn((B, Hq, T, D), torch.float32, 5).to(DEV)
    yq, yk = smooth_attn.sp2norm_qk_norm_rope(q, k, w, w, cos, sin)
    o = smooth_attn.sp2norm_flash_attention(yq, yk, v)
    grads = torch.autograd.grad(o, (q, k, v, w), go)
    leaves = [t.detach().cpu().double().requires_grad_(True) for t in (q, k, v, w)]
    c, s = cos.cpu().double(), sin.cpu().double()
    a, b = (serving.qk_norm_rope(x, leaves[3], c, s) for x in leaves[:2])
    a = torch.matmul(a, b.repeat_interleave(Hq // Hkv, 1).transpose(-1, -2)) / D ** 0.5 - 0.5
    y = torch.tril((a + torch.sqrt(a * a + 1)) ** 2)
    ref = torch.matmul(y / (y.sum(-1, keepdim=True) + 1e-12), leaves[2].repeat_interleave(Hq // Hkv, 1))
    want = torch.autograd.grad(ref, leaves, go.cpu().double())
    torch.testing.assert_close(o.cpu().double(), ref, rtol=2e-5, atol=2e-5)
    for x, r in zip(grads, want):  # fp32 sums of up to a few thousand terms
        assert (x.cpu().double() - r).norm() <= 2e-5 * r.norm()


def test_training_step_replays_in_a_graph():
    B, Hq, Hkv, T, D = 2, 8, 2, 130, 128

    def make(seed):
        return [_randn((B, H, T, D), torch.bfloat16, seed + H).to(DEV) for H in (Hq, Hkv)] + \
            [(1 + 0.1 * _randn((D,), torch.float32, seed + i)).to(DEV) for i in (1, 3)]

    cos, sin = (t.to(DEV) for t in _tables(T, D))
    gq, gk = _randn((B, Hq, T, D), torch.bfloat16, 50).to(DEV), _randn((B, Hkv, T, D), torch.bfloat16, 51).to(DEV)

    def step(args):
        y = smooth_attn.sp2norm_qk_norm_rope(*args, cos, sin)
        return [t.detach() for t in y] + list(torch.autograd.grad(y, args, (gq, gk)))

    static = [t.requires_grad_(True) for t in make(1)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step(static)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step(static)
    for i in range(3):
        fresh = make(100 + i)
        with torch.no_grad():
            for d, s in zip(static, fresh):
                d.copy_(s)
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in outs]
        want = step([t.clone().requires_grad_(True) for t in fresh])
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), i


@pytest.mark.parametrize("dtype,B,T", [(torch.bfloat16, 2, 8192), (torch.float32, 2, 4096)])
def test_tensors_past_the_caches(dtype, B, T):
    # larger than the last-level cache: the same values as sequence by sequence, which is not
    Hq, Hkv, D = 32, 8, 128
    g = torch.Generator(device=DEV).manual_seed(1)
    q, gq = (torch.randn(B, T, Hq, D, generator=g, device=DEV, dtype=dtype).transpose(1, 2) for _ in range(2))
    k, gk = (torch.randn(B, T, Hkv, D, generator=g, device=DEV, dtype=dtype).transpose(1, 2) for _ in range(2))
    w = 1 + 0.1 * torch.randn(D, generator=g, device=DEV)
    cos, sin = (t.to(DEV) for t in _tables(T, D))

    def step(rows):
        args = [t[rows].detach().requires_grad_(True) for t in (q, k)] + [w.clone().requires_grad_(True) for _ in range(2)]
        y = smooth_attn.sp2norm_qk_norm_rope(*args, cos, sin)
        return [t.detach() for t in y] + list(torch.autograd.grad(y, args, (gq[rows], gk[rows])))

    whole, parts = step(slice(0, B)), [step(slice(b, b + 1)) for b in range(B)]
    for i in range(4):
        assert all(torch.equal(whole[i][b:b + 1], parts[b][i]) for b in range(B)), i
    for i in (4, 5):  # sums of 32-bit terms in another order
        torch.testing.assert_close(whole[i], sum(p[i] for p in parts), rtol=1e-4, atol=1e-2)


@pytest.mark.parametrize("leaf", ["itself", "behind views"])
@pytest.mark.parametrize("native", [True, False])
def test_capture_beside_a_living_graph_of_the_same_leaves_is_refused(native, leaf):
    # (the streams of the two graphs would wait for each other inside the capture, which ends the process)
    D, T = 64, 20
    q = _randn((1, 4, T, D), torch.bfloat16, 1).to(DEV)
    if not native:
        q = q.transpose(2, 3).contiguous().transpose(2, 3)  # a layout that the Python path takes
    q.requires_grad_(True)
    k = _randn((1, 2, T, D), torch.bfloat16, 2).to(DEV)
    cos, sin = (t.to(DEV) for t in _tables(T, D))
    ones = torch.ones(q.shape, dtype=q.dtype, device=DEV)

    def forward():
        x = q if leaf == "itself" else (q * 1).view_as(q)
        return smooth_attn.sp2norm_qk_norm_rope(x, k, None, None, cos, sin)

    def step():
        return torch.autograd.grad(forward()[0], q, ones)[0]

    want = step()
    alive = forward()
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="captured into a graph"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            step()
    assert torch.equal(torch.autograd.grad(alive[0], q, ones)[0], want)  # the living graph is as it was
    del alive
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want)
