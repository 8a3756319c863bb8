"""What a reservation's outputs hold on to (GPU)."""
import pytest
import torch

import smooth_attn

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("native", [True, False])
def test_lengths_do_not_hold_the_token_maps(native):
    B, W, P, N = 5, 8, 16, 100000
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
    table = torch.full((B, W), -1, dtype=torch.int32, device=DEV)
    lens = i32(*[0] * B) if native else torch.zeros(B, dtype=torch.int64, device=DEV)  # (64 bits: the Python path)
    r = smooth_attn.sp2norm_paged_reserve(table, lens, i32(*[3] * B), torch.arange(40, dtype=torch.int32, device=DEV),
                                          i32(40), N, block_size=P)
    assert r.slots.shape == (N,) and r.context_lens.tolist() == [3] * B and r.n_free.tolist() == [35]
    for name in ("starts", "context_lens", "n_free"):
        assert getattr(r, name).untyped_storage().nbytes() < 4 * N, name
