"""Pages, tables and slot maps on the device against the plain loops (GPU):
whole numbers, equal everywhere."""
import pytest
import torch

import smooth_attn
from oracle import serving

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _state(B, W, P, n_pages, seed, fill=0.5, n_free=None):
    """Sequences that hold random pages of a pool, and the rest of it on the stack."""
    g = torch.Generator().manual_seed(seed)
    lens = (torch.rand(B, generator=g) * fill * W * P).to(torch.int32)
    perm = torch.randperm(n_pages, generator=g).to(torch.int32)
    table = torch.full((B, W), -1, dtype=torch.int32)
    at = 0
    for b in range(B):
        n = min(-(-int(lens[b]) // P), n_pages - at)
        lens[b] = min(int(lens[b]), n * P)
        table[b, :n] = perm[at:at + n]
        at += n
    free = torch.cat([perm[at:], torch.full((at,), -1, dtype=torch.int32)])
    return table, lens, free, torch.tensor([n_pages - at if n_free is None else n_free], dtype=torch.int32)


def _reserve(table, lens, new, free, n_free, n_tokens, P):
    want = serving.reserve(table, lens, new, free, n_free, n_tokens, P)
    t = table.to(DEV)
    free_dev, lens_dev = free.to(DEV), lens.to(DEV)
    got = smooth_attn.sp2norm_paged_reserve(t, lens_dev, new.to(DEV), free_dev, n_free.to(DEV), n_tokens, block_size=P)
    assert torch.equal(t.cpu(), want[0])
    for name, g, w in zip(got._fields, got, want[1:]):
        w = torch.tensor([w], dtype=torch.int32) if isinstance(w, int) else w
        assert g.dtype == torch.int32 and torch.equal(g.cpu(), w), name
    assert torch.equal(free_dev.cpu(), free) and torch.equal(lens_dev.cpu(), lens)
    # the same call again: the same
    again = smooth_attn.sp2norm_paged_reserve(t, lens_dev, new.to(DEV), free_dev, n_free.to(DEV), n_tokens, block_size=P)
    assert torch.equal(t.cpu(), want[0]) and all(torch.equal(a, b) for a, b in zip(got, again))
    return t, got


@pytest.mark.parametrize("B,W,P,most,extra", [
    (1, 4, 16, 1, 0), (1, 8, 16, 100, 5), (3, 7, 16, 1, 0), (64, 40, 16, 1, 3), (65, 12, 8, 40, 0),
    (256, 20, 32, 200, 17), (300, 6, 1, 4, 1), (700, 5, 12, 33, 0), (4096, 3, 16, 2, 100), (5, 30, 64, 1500, 9),
])
def test_reserve(B, W, P, most, extra):
    n_pages = B * W
    table, lens, free, n_free = _state(B, W, P, n_pages, B + W)
    g = torch.Generator().manual_seed(B)
    new = torch.randint(0, most + 1, (B,), generator=g).to(torch.int32)
    new[::7] = 0
    _reserve(table, lens, new, free, n_free, int(new.sum()) + extra, P)


def test_reserve_cuts_where_pages_tables_or_tokens_end():
    P = 4
    table, lens, free, _ = _state(6, 5, P, 40, 1)
    new = torch.tensor([9, 30, 0, 7, 50, 3], dtype=torch.int32)
    for n_free in (0, 1, 2, 3, 5, 8, 1000, -4):  # (more than there is room for, and fewer than none)
        for n_tokens in (0, 1, 10, 38, 99, 120):
            _reserve(table, lens, new, free, torch.tensor([n_free], dtype=torch.int32), n_tokens, P)


def test_reserve_with_bad_lengths_and_pages():
    # lengths below 0 and past the table, pages outside the pool in the table and on the stack
    P = 4
    table, lens, free, n_free = _state(6, 5, P, 40, 2)
    lens[0], lens[1] = -3, 1000
    table[2, 0], table[3] = 77, -9
    lens[2], lens[3] = 2, 6
    free[int(n_free) - 1], free[int(n_free) - 2] = 99, -2
    new = torch.tensor([3, 2, 5, -6, 11, 4], dtype=torch.int32)
    _reserve(table, lens, new, free, n_free, 30, P)


def test_reserve_takes_64_bit_lengths_and_strided_tables():
    P = 16
    table, lens, free, n_free = _state(9, 12, P, 200, 3)
    wide = torch.full((9, 20), 5, dtype=torch.int32, device=DEV)
    view = wide[:, 4:16]
    view.copy_(table)
    new = torch.arange(9) * 3
    got = smooth_attn.sp2norm_paged_reserve(view, lens.long().to(DEV), new.to(DEV), free.to(DEV), n_free.to(DEV), 200)
    want = serving.reserve(table, lens, new, free, n_free, 200, P)
    assert torch.equal(view.cpu(), want[0]) and torch.equal(got.slots.cpu(), want[1])
    assert (wide[:, :4] == 5).all() and (wide[:, 16:] == 5).all()  # the columns beside the table stay


def test_reserve_of_nothing():
    empty = torch.zeros(0, 4, dtype=torch.int32, device=DEV)
    none = torch.zeros(0, dtype=torch.int32, device=DEV)
    free = torch.arange(8, dtype=torch.int32, device=DEV)
    n = torch.tensor([8], dtype=torch.int32, device=DEV)
    r = smooth_attn.sp2norm_paged_reserve(empty, none, none, free, n, 3)
    assert r.slots.tolist() == [-1] * 3 and r.sequences.tolist() == [-1] * 3 and r.starts.tolist() == [0]
    assert r.n_free.tolist() == [8] and r.context_lens.numel() == 0
    r = smooth_attn.sp2norm_paged_reserve(torch.zeros(2, 0, dtype=torch.int32, device=DEV), torch.zeros(2, device=DEV, dtype=torch.int32),
                                          torch.ones(2, device=DEV, dtype=torch.int32), free, n, 2)
    assert r.slots.tolist() == [-1, -1] and r.context_lens.tolist() == [0, 0] and r.n_free.tolist() == [8]
    lens, left = smooth_attn.sp2norm_paged_release(empty, none, none.bool(), free, n)
    assert lens.numel() == 0 and left.tolist() == [8]


@pytest.mark.parametrize("B,W,P,share", [(1, 4, 16, 1.0), (3, 70, 16, 0.5), (64, 200, 16, 0.3), (300, 9, 8, 0.7),
                                         (4096, 2, 4, 0.1), (5, 6, 16, 0.0)])
def test_release(B, W, P, share):
    n_pages = B * W
    table, lens, free, n_free = _state(B, W, P, n_pages, B + W, fill=0.9)
    done = torch.rand(B, generator=torch.Generator().manual_seed(B)) < share
    if B > 2:
        table[B // 2, 0] = -7  # names no page
        lens[0] = min(int(lens[0]) + 1, W * P)
    want = serving.release(table, lens, done, free, n_free, P)
    t, f = table.to(DEV), free.to(DEV)
    got_lens, left = smooth_attn.sp2norm_paged_release(t, lens.to(DEV), done.to(DEV), f, n_free.to(DEV), block_size=P)
    assert torch.equal(t.cpu(), want[0]) and torch.equal(f.cpu(), want[1])
    assert torch.equal(got_lens.cpu(), want[2]) and left.tolist() == [want[3]]
    # given back again: nothing more
    f2 = f.clone()
    _, left2 = smooth_attn.sp2norm_paged_release(t, lens.to(DEV), done.to(DEV), f2, left, block_size=P)
    assert left2.tolist() == left.tolist() and torch.equal(f2, f)


def test_release_never_writes_past_the_stack():
    P = 4
    table, lens, free, n_free = _state(4, 6, P, 24, 5, fill=1.0)
    full = torch.tensor([23], dtype=torch.int32)  # says that there is room for one
    want = serving.release(table, lens, torch.ones(4, dtype=torch.bool), free, full, P)
    room = torch.full((26,), -5, dtype=torch.int32, device=DEV)
    f = room[:24]
    f.copy_(free)
    _, left = smooth_attn.sp2norm_paged_release(table.to(DEV), lens.to(DEV), torch.ones(4, dtype=torch.bool, device=DEV),
                                                f, full.to(DEV), block_size=P)
    assert torch.equal(f.cpu(), want[1]) and left.tolist() == [24] == [want[3]]
    assert (room[24:] == -5).all()


def test_many_steps_keep_every_page_once():
    B, W, P, n_pages = 24, 16, 8, 200
    gen = torch.Generator().manual_seed(9)
    table = torch.full((B, W), -1, dtype=torch.int32, device=DEV)
    lens = torch.zeros(B, dtype=torch.int32, device=DEV)
    free = torch.randperm(n_pages, generator=gen).to(torch.int32).to(DEV)
    n_free = torch.tensor([n_pages], dtype=torch.int32, device=DEV)
    for _ in range(15):
        new = torch.randint(0, 12, (B,), generator=gen).to(torch.int32).to(DEV)
        r = smooth_attn.sp2norm_paged_reserve(table, lens, new, free, n_free, 12 * B, block_size=P)
        lens, n_free = r.context_lens, r.n_free
        used = torch.arange(W, device=DEV) < ((lens + P - 1) // P)[:, None]
        have = torch.cat([table[used], free[:int(n_free)]]).sort().values
        assert torch.equal(have, torch.arange(n_pages, dtype=torch.int32, device=DEV))
        done = (torch.rand(B, generator=gen) < 0.15).to(DEV)
        lens, n_free = smooth_attn.sp2norm_paged_release(table, lens, done, free, n_free, block_size=P)


def test_replays_in_a_graph():
    B, W, P = 40, 12, 16
    table, lens, free, n_free = (t.to(DEV) for t in _state(B, W, P, 600, 11))
    new = torch.ones(B, dtype=torch.int32, device=DEV)
    static = (table.clone(), lens.clone(), new, free.clone(), n_free.clone())

    def step():
        t, ln, nw, f, n = static
        ln, n = smooth_attn.sp2norm_paged_release(t, ln, nw > 20, f, n, block_size=P)
        return smooth_attn.sp2norm_paged_reserve(t, ln, nw, f, n, 400, block_size=P)

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for seed in range(3):
        fresh = _state(B, W, P, 600, 20 + seed)
        nw = torch.randint(0, 25, (B,), generator=torch.Generator().manual_seed(seed)).to(torch.int32)
        for d, s in zip(static, (fresh[0], fresh[1], nw, fresh[2], fresh[3])):
            d.copy_(s)
        graph.replay()
        torch.cuda.synchronize()
        t, f, ln, n = serving.release(fresh[0], fresh[1], nw > 20, fresh[2], fresh[3], P)
        want = serving.reserve(t, ln, nw, f, n, 400, P)
        assert torch.equal(static[0].cpu(), want[0])
        assert all(torch.equal(a.cpu(), b) for a, b in zip(outs[:5], want[1:6])) and outs.n_free.tolist() == [want[6]]
