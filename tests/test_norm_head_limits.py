"""Heads past what a launch of the norm takes are refused before it."""
import pytest
import torch

import smooth_attn

BF = torch.bfloat16
TABLE = torch.zeros(2, 8)


@pytest.mark.parametrize("Hq,Hkv", [(16384, 1), (1, 16384), (70000, 70000)])
def test_too_many_heads(Hq, Hkv):
    q, k = torch.zeros(1, Hq, 2, 16, dtype=BF), torch.zeros(1, Hkv, 2, 16, dtype=BF)
    with pytest.raises(ValueError, match="heads"):
        smooth_attn.sp2norm_qk_norm_rope(q, k, None, None, TABLE, TABLE)
    cache = torch.zeros(1, Hkv, 16, 16, dtype=BF)
    i = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="heads"):
        smooth_attn.sp2norm_paged_qk_norm_rope_append(q[0].transpose(0, 1), k[0].transpose(0, 1), k[0].transpose(0, 1), None,
                                                      None, TABLE, TABLE, i, i, cache, cache)


def test_as_many_as_it_takes_get_to_the_device_check():
    q, k = torch.zeros(1, 16383, 2, 16, dtype=BF), torch.zeros(1, 1, 2, 16, dtype=BF)
    with pytest.raises(ValueError, match="CUDA tensor"):
        smooth_attn.sp2norm_qk_norm_rope(q, k, None, None, TABLE, TABLE)
