"""Roundings of the norm's reciprocal root and of its weight gradients (GPU)."""
import pytest
import torch

import smooth_attn

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24


def _one_value(c, D, dtype):
    """Rows [1, 1, len(c), D] with one value each, in changing columns."""
    x = torch.zeros(1, 1, len(c), D)
    x[0, 0, torch.arange(len(c)), torch.arange(len(c)) % D] = c
    return x.to(dtype).to(DEV)


def _turned_by_nothing(T, D):
    return torch.ones(T, D // 2, device=DEV), torch.zeros(T, D // 2, device=DEV)


def test_the_reciprocal_root_is_off_by_a_step_at_most():
    # One value c of 12 significant bits in a row of 64: mean(x^2) = c^2 / 64 exactly, and the output
    # c * r is 8: r off by a step (2^-23 of itself at most), the product by half a one.
    D = 64
    c = torch.cat([(1 + torch.arange(2048) / 2048) * 2.0 ** e for e in (-20, 0, 1, 15)])
    y, _ = smooth_attn.sp2norm_qk_norm_rope(_one_value(c, D, torch.float32), _one_value(-c, D, torch.float32), None, None,
                                            *_turned_by_nothing(len(c), D), eps=0.0)
    got = y.double().sum(-1).cpu()
    assert ((got - 8).abs() <= 8 * 3.01 * U).all(), (got - 8).abs().max() / (8 * U)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_mean_squares_below_the_normal_range(dtype):
    # c^2 / 64 = 2^-148 to 2^-126, exact as denormals; r = 8 / c.  With g = 1 in the row's column, dx is
    # r (g - n mean(g n)) = r (1 - 8 * 8 / 64) = 0 there and r g in a column without a value.
    D = 64
    c = 2.0 ** torch.arange(-71, -59).float()
    q, k = (_one_value(c, D, dtype).requires_grad_(True) for _ in range(2))
    y, yk = smooth_attn.sp2norm_qk_norm_rope(q, k, None, None, *_turned_by_nothing(len(c), D), eps=0.0)
    eight = torch.full((1, 1, len(c)), 8.0, dtype=torch.float64, device=DEV)
    assert torch.equal(y.double().sum(-1), eight) and torch.equal(yk.double().sum(-1), eight)
    own = q.detach() != 0
    dx, = torch.autograd.grad(y, q, torch.ones_like(y))
    assert (dx[own] == 0).all()
    want = (8 / c).to(DEV)[:, None].expand(-1, D)[~own[0, 0]]
    assert torch.equal(dx[~own].float(), want)


def test_a_row_of_zeros_without_eps_is_as_the_formula_says():
    # 0 / sqrt(0)
    x = torch.zeros(1, 1, 3, 64, device=DEV)
    y, _ = smooth_attn.sp2norm_qk_norm_rope(x, x, None, None, *_turned_by_nothing(3, 64), eps=0.0)
    assert torch.isnan(y).all()


def test_a_weight_gradient_of_one_large_term():
    # Rows of ones with gradients of ones: every row's term is 1, but one is 2^34.  A block adds its
    # 128 rows in fp32 and may lose all of them beside the large one; the sum over blocks loses
    # nothing but its last rounding, 2^-24.
    T, H, D = 16384, 8, 64
    q, g = torch.ones(1, H, T, D, device=DEV), torch.ones(1, H, T, D, device=DEV)
    g[0, 0, 0] = 2.0 ** 34
    k = torch.ones(1, 1, T, D, device=DEV)
    w = torch.ones(D, device=DEV, requires_grad=True)
    y, _ = smooth_attn.sp2norm_qk_norm_rope(q, k, w, None, *_turned_by_nothing(T, D), eps=0.0)
    dw = torch.autograd.grad(y, w, g)[0].double().cpu()
    want = 2.0 ** 34 + H * T - 1
    assert ((dw - want).abs() <= 128 + U * want).all(), (dw - want).abs().max()
