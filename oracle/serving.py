"""Plain restatement of the operators around the paged attention — TEST
INFRASTRUCTURE.  64-bit floating point, Python loops over sequences and tokens,
CPU.  They have no counterpart in the reference.

pinned by: tests/test_oracle_serving.py (closed forms, autograd, invariants).
"""
from __future__ import annotations

import torch

EPS = 1e-12


def qk_norm_rope(x, weight, cos, sin, eps=1e-6):
    """Rows of x [..., D] normed, weighted and turned; cos, sin broadcast against
    [..., D/2].  Differentiable, in x's precision."""
    z = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
    if weight is not None:
        z = z * weight
    half = x.shape[-1] // 2
    a, b = z[..., :half], z[..., half:]
    return torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)


def reserve(table, lens, new, free_pages, n_free, n_tokens, P):
    """(table, slots, positions, sequences, starts, lens, n_free), all new CPU tensors or ints."""
    table = table.clone()
    B, W = table.shape
    n_pages = free_pages.numel()
    left = min(max(int(n_free), 0), n_pages)
    slots, positions, sequences = ([-1] * n_tokens, [0] * n_tokens, [-1] * n_tokens)
    starts, out_lens, i = [0], [], 0
    for b in range(B):
        ctx = min(max(int(lens[b]), 0), W * P)
        had, length = -(-ctx // P), ctx
        fresh = min(max(int(new[b]), 0), n_tokens - i)
        cut = False
        for t in range(fresh):
            pos = ctx + t
            positions[i], sequences[i] = pos, b
            if not cut and pos < W * P:
                pi, row = pos // P, pos % P
                if pi >= had and row == 0:
                    if left == 0:
                        cut = True
                    else:
                        left -= 1
                        table[b, pi] = free_pages[left]
                if not cut:
                    length = pos + 1
                    page = int(table[b, pi])
                    if 0 <= page < n_pages:
                        slots[i] = page * P + row
            i += 1
        starts.append(i)
        out_lens.append(length)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32)  # noqa: E731
    return table, i32(slots), i32(positions), i32(sequences), i32(starts), i32(out_lens), left


def release(table, lens, finished, free_pages, n_free, P):
    """(table, free_pages, lens, n_free), new."""
    table, free_pages, lens = table.clone(), free_pages.clone(), lens.clone().to(torch.int32)
    n_pages = free_pages.numel()
    left = min(max(int(n_free), 0), n_pages)
    for b in range(table.shape[0]):
        if not finished[b]:
            continue
        ctx = min(max(int(lens[b]), 0), table.shape[1] * P)
        for j in range(-(-ctx // P)):
            page = int(table[b, j])
            if 0 <= page < n_pages and left < n_pages:
                free_pages[left] = page
                left += 1
            table[b, j] = -1
        lens[b] = 0
    return table, free_pages, lens, left


def key_bounds(k_cache, table, from_lens, to_lens, bounds, P):
    """bounds (a new tensor) after tokens from_lens .. to_lens - 1 were written."""
    values = k_cache.double()
    out = bounds.double().clone()
    for b in range(table.shape[0]):
        to = min(max(int(to_lens[b]), 0), table.shape[1] * P)
        j = max(int(from_lens[b]), 0) // P
        while j * P < to:
            page = int(table[b, j])
            if 0 <= page < k_cache.shape[0]:
                rows = values[page, :, :min(P, to - j * P)]
                out[page, :, 0], out[page, :, 1] = rows.amin(1), rows.amax(1)
            j += 1
    return out


def page_scores(q, bounds, pages):
    """[Hkv, len(pages)] scores of one sequence's pages; q [Hq, D]."""
    Hkv = bounds.shape[1]
    q = q.double().view(Hkv, -1, q.shape[-1])
    up, down = q.clamp(min=0).sum(1), q.clamp(max=0).sum(1)
    b = bounds[pages].double()  # [n, Hkv, 2, D]
    return ((b[:, :, 1] * up).sum(-1) + (b[:, :, 0] * down).sum(-1)).t()


def select_pages(q, bounds, table, lens, top_k, n_first, n_last, P):
    B, Hkv = q.shape[0], bounds.shape[1]
    out = torch.full((B, Hkv, top_k), -1, dtype=torch.int32)
    for b in range(B):
        np_ = -(-min(max(int(lens[b]), 0), table.shape[1] * P) // P)
        if np_ <= top_k:
            out[b, :, :np_] = torch.arange(np_, dtype=torch.int32)
            continue
        scores = page_scores(q[b, :, 0], bounds, table[b, :np_].long())
        forced = list(range(n_first)) + list(range(np_ - n_last, np_))
        for h in range(Hkv):
            rank = lambda j: (0 if scores[h, j] != scores[h, j] else 1, -float(scores[h, j].nan_to_num()), j)  # noqa: E731
            rest = sorted(range(n_first, np_ - n_last), key=rank)
            mine = sorted(forced + rest[:top_k - len(forced)])
            out[b, h] = torch.tensor(mine, dtype=torch.int32)
    return out


def sparse_attention(q, k_cache, v_cache, table, lens, pages, scale, P):
    """(o, bound): o [B, Hq, D] and the sum of the weights' shares times |v|,
    which the roundings of a kernel scale with."""
    B, Hq, _, D = q.shape
    Hkv = k_cache.shape[1]
    G = Hq // Hkv
    o = torch.zeros(B, Hq, D, dtype=torch.float64)
    bound = torch.zeros_like(o)
    for b in range(B):
        for h in range(Hkv):
            ks, vs = [], []
            for j in pages[b, h].tolist():
                if not 0 <= j < table.shape[1]:
                    continue
                n = min(max(int(lens[b]) - j * P, 0), P)
                if n == 0:
                    continue
                page = min(max(int(table[b, j]), 0), k_cache.shape[0] - 1)
                ks.append(k_cache[page, h, :n].double())
                vs.append(v_cache[page, h, :n].double())
            if not ks:
                continue
            k, v = torch.cat(ks), torch.cat(vs)
            a = q[b, h * G:(h + 1) * G, 0].double() @ k.t() * scale - 0.5
            y = (a + torch.sqrt(a * a + 1)) ** 2
            total = y.sum(-1, keepdim=True) + EPS
            o[b, h * G:(h + 1) * G] = y @ v / total
            bound[b, h * G:(h + 1) * G] = y @ v.abs() / total
    return o, bound
