"""The norm on views whose dims of one element have strides that no row could (GPU)."""
import pytest
import torch

import smooth_attn

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("shape,stride", [
    ((2, 4, 1, 64), (256, 64, 1, 1)), ((2, 4, 1, 64), (512, 128, 8, 1)), ((2, 4, 1, 64), (512, 64, 0, 1)),
    ((1, 4, 5, 64), (3, 320, 64, 1)), ((2, 1, 5, 64), (320, 1, 64, 1)), ((1, 1, 1, 64), (1, 1, 1, 1)),
])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_strides_of_single_elements(shape, stride, dtype):
    g = torch.Generator().manual_seed(1)
    x = torch.randn(2048, generator=g).to(dtype).to(DEV).as_strided(shape, stride)
    B, _, T, D = shape
    angle = (torch.rand(T, D // 2, generator=g) * 9).to(DEV)
    gq, gk = (torch.randn(shape, generator=g).to(dtype).to(DEV) for _ in range(2))
    w = torch.rand(D, generator=g).to(DEV)

    def step(x):
        q, k = (x.detach().requires_grad_(True) for _ in range(2))
        qw = w.clone().requires_grad_(True)
        y = smooth_attn.sp2norm_qk_norm_rope(q, k, qw, None, angle.cos(), angle.sin())
        return [*y, *torch.autograd.grad(y, (q, k, qw), (gq, gk))]

    for a, b in zip(step(x), step(x.clone(memory_format=torch.contiguous_format))):
        assert torch.equal(a, b)
