"""A turnover of sequences, captured after a warm-up that is ordered with the
tables' copies (GPU)."""
import pytest
import torch

import smooth_attn
from oracle import serving

pytestmark = pytest.mark.gpu
DEV = "cuda"


def test_a_turnover_replays_in_a_graph_after_an_ordered_warm_up():
    # (the warm-up waits for the copies that make its tables, and the capture for the warm-up)
    B, W, P, n_pages = 40, 12, 16, 600

    def state(seed):
        g = torch.Generator().manual_seed(seed)
        lens = torch.randint(0, W * P // 2, (B,), generator=g).to(torch.int32)
        ids = torch.randperm(n_pages, generator=g).to(torch.int32)
        table, at = torch.full((B, W), -1, dtype=torch.int32), 0
        for b in range(B):
            n = -(-int(lens[b]) // P)
            table[b, :n] = ids[at:at + n]
            at += n
        free = torch.cat([ids[at:], ids[:at]])
        return table, lens, torch.randint(0, 25, (B,), generator=g).to(torch.int32), free, torch.tensor([n_pages - at],
                                                                                                       dtype=torch.int32)

    static = tuple(t.to(DEV) for t in state(1))

    def step():
        t, ln, nw, f, n = static
        ln, n = smooth_attn.sp2norm_paged_release(t, ln, nw > 20, f, n, block_size=P)
        return smooth_attn.sp2norm_paged_reserve(t, ln, nw, f, n, 400, block_size=P)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for seed in range(3):
        fresh = state(20 + seed)
        for d, s in zip(static, fresh):
            d.copy_(s)
        graph.replay()
        torch.cuda.synchronize()
        nw = fresh[2]
        t, f, ln, n = serving.release(fresh[0], fresh[1], nw > 20, fresh[3], fresh[4], P)
        want = serving.reserve(t, ln, nw, f, n, 400, P)
        assert torch.equal(static[0].cpu(), want[0])
        assert all(torch.equal(a.cpu(), b) for a, b in zip(outs[:5], want[1:6])) and outs.n_free.tolist() == [want[6]]
