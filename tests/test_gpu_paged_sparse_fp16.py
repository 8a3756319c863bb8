"""fp16 weights past the type's range in the attention over listed pages, against the 64-bit form (GPU)."""
import math

import pytest
import torch

import smooth_attn
from oracle import serving

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24


@pytest.mark.parametrize("Hq,Hkv,D,P,lens", [(4, 1, 64, 16, [40, 700]), (6, 2, 128, 8, [333]), (3, 3, 512, 16, [200])])
@pytest.mark.parametrize("every", [1, 5, 97])
def test_weights_past_fp16(Hq, Hkv, D, P, lens, every):
    # Scores of 10 to a few hundred, so weights (about 4 a^2) on both sides of 65504: of every token, of
    # some in every tile, and of single tiles.  Tolerance: a = scale q.k - 1/2 is off by at most
    # da = 2^-24 (D + 2) scale sum|q k| (fp32 sums of exact products), and a weight, with all a above
    # 1, by 2 da / a + 8 steps of 2^-24 of itself; its rounding to fp16 is half a step, 2^-11 (weights of
    # one tile that were scaled down by 2^16 stay normal: y > 4); the output's to bf16 2^-8.
    g = torch.Generator().manual_seed(D + P)
    B, n = len(lens), max(-(-length // P) for length in lens)
    q = (torch.rand(B, Hq, 1, D, generator=g) + 0.5).to(torch.float16)
    shape = (B * n, Hkv, P, D)
    kc = (torch.rand(shape, generator=g) + 0.5) * 0.5
    token = torch.arange(B * n * P).view(B * n, 1, P, 1)
    kc = torch.where(token % every == 0, kc * 16, kc).to(torch.float16)
    vc = torch.randn(shape, generator=g).to(torch.float16)
    table = torch.arange(B * n, dtype=torch.int32).view(B, n)
    ctx = torch.tensor(lens, dtype=torch.int32)
    pages = table.new_tensor(range(n)).expand(B, Hkv, n).contiguous()
    scale = 24.0 / D
    o, bound = serving.sparse_attention(q, kc, vc, table, ctx, pages, scale, P)
    a = scale * torch.einsum("bhd,nkpd->bhnkp", q[:, :, 0].double(), kc.double()) - 0.5
    assert a.min() > 1 and 4 * a.max() ** 2 > 2 * 65504
    da = U * (D + 2) * a.max()
    rel = 2.0 ** -11 + 2 * da / a.min() + 8 * U
    tol = 2.0 ** -8 * o.abs() * (1 + rel) + rel * (bound + o.abs()) * 1.1
    got = smooth_attn.sp2norm_paged_sparse_attention(*(t.to(DEV) for t in (q, kc, vc, table, ctx, pages)), scale=scale,
                                                     block_size=P)
    assert ((got.cpu().double() - o).abs() <= tol).all()
