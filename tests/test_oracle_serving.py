"""The plain forms of the serving operators pinned on the CPU: closed forms,
invariants and the paged attention's own oracle."""
import math

import torch

from oracle import paging, serving


def _g(seed):
    return torch.Generator().manual_seed(seed)


def test_norm_rope_keeps_the_root_mean_square():
    x = torch.randn(3, 5, 64, generator=_g(0), dtype=torch.float64)
    angle = torch.randn(5, 32, generator=_g(1), dtype=torch.float64)
    y = serving.qk_norm_rope(x, None, angle.cos(), angle.sin(), eps=0.0)
    torch.testing.assert_close((y * y).mean(-1), torch.ones(3, 5, dtype=torch.float64))
    # no angle and weight w: w x / rms
    w = torch.rand(64, generator=_g(2), dtype=torch.float64)
    z = serving.qk_norm_rope(x, w, torch.ones(5, 32), torch.zeros(5, 32), eps=0.0)
    torch.testing.assert_close(z, x / (x * x).mean(-1, keepdim=True).sqrt() * w)
    # turning back by the same angle undoes it
    n = serving.qk_norm_rope(y, None, angle.cos(), -angle.sin(), eps=0.0)
    torch.testing.assert_close(n, x / (x * x).mean(-1, keepdim=True).sqrt())


def test_reserve_then_release_keeps_every_page_once():
    P, n_pages, W = 4, 40, 9
    free = torch.randperm(n_pages, generator=_g(3)).to(torch.int32)
    table = torch.full((5, W), -1, dtype=torch.int32)
    lens = torch.zeros(5, dtype=torch.int32)
    n_free = n_pages
    gen = _g(4)
    for step in range(12):
        new = torch.randint(0, 9, (5,), generator=gen)
        before = lens
        table, slots, pos, seq, starts, lens, n_free = serving.reserve(table, lens, new, free, n_free, 40, P)
        held = [int(table[b, j]) for b in range(5) for j in range(-(-int(lens[b]) // P))]
        assert sorted(held + free[:n_free].tolist()) == list(range(n_pages))
        for i in range(40):
            b = int(seq[i])
            if b < 0:
                assert slots[i] == -1
            elif pos[i] < lens[b]:
                assert slots[i] == int(table[b, pos[i] // P]) * P + pos[i] % P
            else:
                assert slots[i] == -1
        assert (lens >= before).all()
        if step % 4 == 3:
            done = torch.tensor([True, False, step == 11, False, True])
            table, free, lens, n_free = serving.release(table, lens, done, free, n_free, P)
    assert n_free > 0


def test_bounds_bound_every_score():
    P, D, Hq, Hkv = 8, 16, 4, 2
    k = torch.randn(1, Hkv, 61, D, generator=_g(5))
    kc, _, table, lens = paging.build_paged_cache(k, k, P, shuffle=True, generator=_g(6))
    bounds = serving.key_bounds(kc, table, torch.zeros(1), lens, torch.zeros(kc.shape[0], Hkv, 2, D), P)
    q = torch.randn(1, Hq, 1, D, generator=_g(7))
    scores = serving.page_scores(q[0, :, 0], bounds, table[0].long())
    for h in range(Hkv):
        s = (q[0, 2 * h:2 * h + 2, 0].double() @ k[0, h].double().t()).sum(0)
        for j in range(8):
            assert s[j * P:(j + 1) * P].max() <= scores[h, j] + 1e-9


def test_sparse_attention_over_all_pages_is_paged_attention():
    P, D, Hq, Hkv, T = 8, 16, 4, 2, 45
    k = torch.randn(2, Hkv, T, D, generator=_g(8))
    v = torch.randn(2, Hkv, T, D, generator=_g(9))
    kc, vc, table, lens = paging.build_paged_cache(k, v, P, shuffle=True, generator=_g(10), context_lens=[45, 17])
    q = torch.randn(2, Hq, 1, D, generator=_g(11))
    pages = serving.select_pages(q, torch.zeros(kc.shape[0], Hkv, 2, D), table, lens, 6, 0, 1, P)
    assert pages[1, 0].tolist() == [0, 1, 2, -1, -1, -1]
    o, _ = serving.sparse_attention(q, kc, vc, table, lens, pages, 1 / math.sqrt(D), P)
    for b, n in enumerate(lens.tolist()):
        for h in range(Hq):
            s = q[b, h, 0].double() @ k[b, h // 2, :n].double().t() / math.sqrt(D)
            arg = 2 * s - 1
            y = (0.5 * (arg + torch.sqrt(arg * arg + 4))) ** 2
            torch.testing.assert_close(o[b, h], y @ v[b, h // 2, :n].double() / y.sum())


def test_select_ties_and_nan():
    P, D = 4, 8
    bounds = torch.zeros(10, 1, 2, D)
    bounds[[2, 5, 7], 0, 1] = 1.0
    table = torch.arange(10, dtype=torch.int32)[None]
    q = torch.ones(1, 1, 1, D)
    lens = torch.tensor([40])
    assert serving.select_pages(q, bounds, table, lens, 3, 0, 1, P).tolist() == [[[2, 5, 9]]]
    assert serving.select_pages(q, bounds, table, lens, 6, 1, 1, P).tolist() == [[[0, 1, 2, 5, 7, 9]]]
    bounds[8, 0, 0, 3] = float("nan")
    assert serving.select_pages(q, bounds, table, lens, 2, 0, 1, P).tolist() == [[[8, 9]]]
