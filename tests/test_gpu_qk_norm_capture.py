"""Captured backwards of the norm whose leaves other graphs hold (GPU)."""
import pytest
import torch

import smooth_attn
from smooth_attn import _lib

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _args(native):
    g = torch.Generator().manual_seed(1)
    D, T = 64, 20
    q = torch.randn(1, 4, T, D, generator=g).to(torch.bfloat16).to(DEV)
    if not native:
        q = q.transpose(2, 3).contiguous().transpose(2, 3)  # a layout that the Python path takes
    k = torch.randn(1, 2, T, D, generator=g).to(torch.bfloat16).to(DEV)
    angle = (torch.rand(T, D // 2, generator=g) * 9).to(DEV)
    return q.requires_grad_(True), k, angle.cos(), angle.sin(), torch.ones_like(q).detach()


@pytest.mark.parametrize("native", [True, False])
@pytest.mark.parametrize("held_by", ["graph", "accumulator"])
def test_leaves_of_a_side_stream_are_captured(native, held_by):
    # A side stream joins the capture where the engine waits for it (what the default stream cannot): so a
    # program that built its accumulators on one, as hooks on parameters do, is captured.
    q, k, cos, sin, ones = _args(native)

    def forward():
        return smooth_attn.sp2norm_qk_norm_rope(q, k, None, None, cos, sin)[0]

    def step():
        if held_by == "graph":
            return torch.autograd.grad(forward(), q, ones)[0]
        q.grad = None
        forward().backward(ones)
        return q.grad

    side, capture = torch.cuda.Stream(), torch.cuda.Stream()
    assert side != capture
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        alive = forward() if held_by == "graph" else q.view_as(q).grad_fn.next_functions[0][0]
        want = step().clone()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=capture):
        got = step()
    for i in range(3):
        with torch.no_grad():
            got.fill_(i)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want)
        other = q.detach().clone().requires_grad_(True)  # eager work between the replays
        y = smooth_attn.sp2norm_qk_norm_rope(other, k, None, None, cos, sin)[0]
        assert torch.equal(torch.autograd.grad(y, other, ones)[0], want)
    if held_by == "graph":
        assert torch.equal(torch.autograd.grad(alive, q, ones)[0], want)


def test_without_the_native_path_a_captured_backward_is_refused(monkeypatch):
    q, k, cos, sin, ones = _args(True)

    def step():
        return torch.autograd.grad(smooth_attn.sp2norm_qk_norm_rope(q, k, None, None, cos, sin)[0], q, ones)[0]

    want = step()
    monkeypatch.setattr(_lib, "_host", _lib.NothingOrdinary)
    assert torch.equal(step(), want)
    with pytest.raises(RuntimeError, match="native call path"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            step()
    assert torch.equal(step(), want)


def test_a_whole_step_is_captured_while_the_warm_up_s_loss_lives():
    # projection, norm, attention, projection; the loss of the last warm-up step on a side stream is kept
    torch.manual_seed(0)
    B, T, H, Hkv, D, width = 2, 64, 4, 2, 64, 128
    inp, out = (torch.nn.Linear(a, b, bias=False, device=DEV, dtype=torch.bfloat16)
                for a, b in ((width, (H + 2 * Hkv) * D), (H * D, width)))
    weights = [torch.nn.Parameter(torch.ones(D, device=DEV)) for _ in range(2)]
    params = [*inp.parameters(), *out.parameters(), *weights]
    angle = torch.rand(T, D // 2, device=DEV) * 9
    cos, sin = angle.cos(), angle.sin()
    x, y = (torch.randn(B, T, width, device=DEV, dtype=torch.bfloat16) for _ in range(2))

    def backward():
        qkv = inp(x).view(B, T, H + 2 * Hkv, D).transpose(1, 2)
        q, k = smooth_attn.sp2norm_qk_norm_rope(qkv[:, :H], qkv[:, H:H + Hkv], *weights, cos, sin)
        o = smooth_attn.sp2norm_flash_attention(q, k, qkv[:, H + Hkv:])
        loss = ((out(o.transpose(1, 2).reshape(B, T, H * D)) - y) * 0.01).float().square().sum(0)
        loss.backward(torch.ones_like(loss))
        return loss

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            for p in params:
                p.grad = None
            kept = backward()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    want = [p.grad.clone() for p in params]
    for p in params:
        p.grad = None
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        backward()
    for _ in range(3):
        for p in params:
            p.grad.zero_()
        graph.replay()
        torch.cuda.synchronize()
        # (the library's products may sum in another order there: a few bf16 roundings of 2^-8)
        assert all((p.grad - w).norm() <= 2.0 ** -6 * w.norm() for p, w in zip(params, want))
    assert kept.grad_fn is not None
