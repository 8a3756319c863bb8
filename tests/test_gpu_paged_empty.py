"""Bounds, page choice and attention where there are no pages or no table: no token, so zeros (GPU)."""
import pytest
import torch

import smooth_attn

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("n_pages,width", [(0, 4), (5, 0), (0, 0)])
@pytest.mark.parametrize("dtype,cache,D", [(torch.bfloat16, torch.bfloat16, 64), (torch.float16, torch.float16, 128),
                                           (torch.float32, torch.float32, 32), (torch.bfloat16, torch.float8_e4m3fn, 64)])
@pytest.mark.parametrize("top_k", [2, 6])
def test_no_pages_or_no_table(n_pages, width, dtype, cache, D, top_k):
    B, Hq, Hkv, P = 3, 4, 2, 16
    q = torch.ones(B, Hq, 1, D, dtype=dtype, device=DEV)
    kc = torch.ones(n_pages, Hkv, P, D, device=DEV).to(cache)
    table = torch.zeros(B, width, dtype=torch.int32, device=DEV)
    lens = torch.tensor([0, 20, 64], dtype=torch.int32, device=DEV)
    bounds = smooth_attn.sp2norm_paged_key_bounds(kc, table, torch.zeros_like(lens), lens)
    assert bounds.shape == (n_pages, Hkv, 2, D)
    pages = smooth_attn.sp2norm_paged_select_pages(q, bounds, table, lens, top_k)
    assert pages.shape == (B, Hkv, top_k) and (pages == -1).all()
    for listed in (pages, torch.zeros_like(pages), pages[..., :0]):
        o = smooth_attn.sp2norm_paged_sparse_attention(q, kc, kc, table, lens, listed)
        assert o.shape == (B, Hq, D) and o.dtype == torch.bfloat16 and (o == 0).all()
    o = smooth_attn.sp2norm_paged_attention(q, kc, kc, table, lens)
    assert o.shape == (B, Hq, D) and (o == 0).all()
