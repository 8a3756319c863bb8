"""Operators around the attention kernels, as measurable cases: what a training
or serving program calls before and beside them.

Each case is a dict of plain values naming one pass at one size.  ``listed``
holds the fixed ones, ``draw`` makes more of the same ranges, ``prepare`` makes
the tensors that a program has in hand before the pass, ``run`` makes it,
``work`` counts the bytes and operations that it cannot do without, and
``exact`` gives its results in 64 bits.  ``own`` says whether ``run`` calls the
package's operators or computes them in plain torch operations.

Kinds of case:
  norm_rope  RMS norm of each head's q and k rows and rotate-half RoPE, forward
             and, where ``grad`` holds, backward (q, k and the norms' weights)
  append     the same for packed tokens of a serving step, K and V written into
             the paged caches through a slot map
  reserve    pages, slot map and positions of a step's new tokens
  turnover   pages of finished sequences given back, then the same
  bounds     smallest and largest key of every page that a step wrote to
  sparse     pages chosen by the bounds' scores, and one token's attention over them
"""
from __future__ import annotations

import math
import pathlib
import sys

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32, "fp8": torch.float8_e4m3fn}
SIZES = {"bf16": 2, "fp16": 2, "fp32": 4, "fp8": 1}
EPS = 1e-12  # added to the attention's row sums
NORM_EPS = 1e-6  # added to the norms' mean squares
MAX_ROWS = 4 * 64 * 4096  # (head, token) rows of the largest norm case
MAX_CACHE = 64 * 16384 * 8  # (token, KV head) rows of the largest cache
N_POSITIONS = 32768  # rows of the serving rotation tables


def listed():
    return [
        # A small model's training step: 12 heads of 64, short rows.
        {"name": "train_small_d64", "kind": "norm_rope", "dtype": "fp16", "wdtype": "fp16", "B": 4, "Hq": 12,
         "Hkv": 12, "T": 1024, "D": 64, "layout": "bhtd", "grad": True},
        # Fine-tuning with grouped KV heads at an odd length, straight from the projections ([B, T, H, D] buffers).
        {"name": "train_odd_gqa", "kind": "norm_rope", "dtype": "bf16", "wdtype": "bf16", "B": 2, "Hq": 32, "Hkv": 8,
         "T": 1023, "D": 128, "layout": "bthd", "grad": True},
        # The benchmark's attention sizes: training at 4096 tokens, weights of the norms kept in 32 bits.
        {"name": "train_large", "kind": "norm_rope", "dtype": "bf16", "wdtype": "fp32", "B": 4, "Hq": 32, "Hkv": 32,
         "T": 4096, "D": 128, "layout": "bthd", "grad": True},
        # One decode step of 8 sequences: launches and host work count.
        {"name": "append_decode", "kind": "append", "dtype": "bf16", "cache": "bf16", "B": 8, "Hq": 32, "Hkv": 8,
         "D": 128, "page": 16, "lo": 1, "hi": 1},
        # A prefill of ragged prompts, about 8000 tokens, into an 8-bit cache.
        {"name": "append_prefill_fp8", "kind": "append", "dtype": "bf16", "cache": "fp8", "B": 7, "Hq": 32, "Hkv": 8,
         "D": 128, "page": 16, "lo": 300, "hi": 2047},
        # The maps of a decode step of 64 sequences.
        {"name": "reserve_decode", "kind": "reserve", "B": 64, "page": 16, "lo": 512, "hi": 16384, "new_lo": 1,
         "new_hi": 1},
        # Continuous batching: a quarter of 256 sequences is done, new prompts of 64 to 2048 tokens take their rows.
        {"name": "turnover_256", "kind": "turnover", "B": 256, "page": 16, "lo": 512, "hi": 16384, "new_lo": 64,
         "new_hi": 2048},
        # The bounds after a decode step of 64 sequences: one page of each.
        {"name": "bounds_decode", "kind": "bounds", "cache": "bf16", "B": 64, "Hkv": 8, "D": 128, "page": 16,
         "lo": 512, "hi": 16384, "new": 1},
        # The bounds after the prefill of four long prompts.
        {"name": "bounds_prefill", "kind": "bounds", "cache": "bf16", "B": 4, "Hkv": 8, "D": 128, "page": 16,
         "lo": 8192, "hi": 16384, "new": 0},
        # One sequence of up to 16384 tokens, 1024 of them attended to.
        {"name": "sparse_one", "kind": "sparse", "dtype": "bf16", "cache": "bf16", "B": 1, "Hq": 32, "Hkv": 8,
         "D": 128, "page": 16, "lo": 16000, "hi": 16384, "top_k": 64, "n_first": 1, "n_last": 1},
        # The paged benchmark's batch: 64 sequences of 512 to 16384 tokens.
        {"name": "sparse_batch", "kind": "sparse", "dtype": "bf16", "cache": "bf16", "B": 64, "Hq": 32, "Hkv": 8,
         "D": 128, "page": 16, "lo": 512, "hi": 16384, "top_k": 64, "n_first": 1, "n_last": 2},
        # A few very long contexts, 2048 tokens of each attended to.
        {"name": "sparse_long", "kind": "sparse", "dtype": "bf16", "cache": "bf16", "B": 8, "Hq": 32, "Hkv": 8,
         "D": 128, "page": 16, "lo": 65536, "hi": 131072, "top_k": 128, "n_first": 1, "n_last": 2},
    ]


def _log_int(rng, lo, hi):
    """An integer of [lo, hi], spread over its logarithm."""
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    kind = rng.choice(["norm_rope", "norm_rope", "norm_rope", "append", "append", "reserve", "turnover", "bounds",
                       "sparse", "sparse", "sparse"])
    dtype = rng.choice(["bf16", "bf16", "bf16", "fp16", "fp32"])
    Hq, Hkv = rng.choice([(32, 8), (32, 8), (32, 32), (16, 2), (12, 12), (8, 1)])
    D = rng.choice([64, 80, 96, 128, 128, 128, 256])
    page = rng.choice([8, 16, 16, 32, 64])
    if kind == "norm_rope":
        T = _log_int(rng, 1, 8192)
        return {"kind": kind, "dtype": dtype, "wdtype": rng.choice([dtype, "fp32"]),
                "B": _log_int(rng, 1, max(1, min(64, MAX_ROWS * 128 // (D * (Hq + Hkv) * T * (2 if dtype == "fp32" else 1))))),
                "Hq": Hq, "Hkv": Hkv, "T": T, "D": D, "layout": rng.choice(["bhtd", "bthd"]),
                "grad": rng.random() < 0.75}
    if kind in ("reserve", "turnover"):
        hi = _log_int(rng, 1, 16384)
        new = _log_int(rng, 1, 2048)
        return {"kind": kind, "B": _log_int(rng, 1, 256), "page": page, "lo": max(1, hi // 32), "hi": hi,
                "new_lo": max(1, new // 8), "new_hi": new}
    cache = rng.choice([dtype, dtype, "fp8"])
    if cache == "fp8":
        dtype = "bf16"
    if kind == "append":
        hi = _log_int(rng, 1, 2048)
        return {"kind": kind, "dtype": dtype, "cache": cache, "B": _log_int(rng, 1, min(64, max(1, 16384 // hi))),
                "Hq": Hq, "Hkv": Hkv, "D": D, "page": page, "lo": max(1, hi // 8), "hi": hi}
    rows = MAX_CACHE * 128 * 2 // (D * SIZES[cache] * Hkv)  # tokens that fit
    hi = _log_int(rng, 64, min(131072, rows))
    B = _log_int(rng, 1, max(1, min(64, rows // hi)))
    if kind == "bounds":
        return {"kind": kind, "cache": cache, "B": B, "Hkv": Hkv, "D": D, "page": page, "lo": max(1, hi // 32),
                "hi": hi, "new": rng.choice([0, 1, 1, 5])}
    n_first, n_last = rng.choice([0, 1, 2]), rng.choice([1, 1, 2, 4])
    top_k = _log_int(rng, n_first + n_last, max(n_first + n_last, 2048 // page))
    return {"kind": kind, "dtype": dtype, "cache": cache, "B": B, "Hq": Hq, "Hkv": Hkv, "D": D, "page": page,
            "lo": max(1, hi // 32), "hi": hi, "top_k": top_k, "n_first": n_first, "n_last": n_last}


# ---------------------------------------------------------------------------
# Inputs.
# ---------------------------------------------------------------------------
def _randn(gen, shape, dtype):
    """N(0, 1) in dtype (e4m3fn holds the values themselves)."""
    if dtype == torch.float8_e4m3fn:
        return torch.randn(shape, generator=gen, device="cuda", dtype=torch.bfloat16).to(dtype)
    return torch.randn(shape, generator=gen, device="cuda", dtype=dtype)


def _spread(gen, n, lo, hi):
    """n lengths uniform in [lo, hi], one in each of n equal parts of it, in any
    order: every seed has about the same sum."""
    part = (torch.randperm(n, generator=gen, device="cuda") + torch.rand(n, generator=gen, device="cuda")) / n
    return (lo + part * (hi + 1 - lo)).to(torch.int32).clamp_(lo, hi)


def _new_lens(gen, n, lo, hi):
    """n numbers of new tokens over [lo, hi] in any order, and their sum: the
    same ones for every seed, as a program's packed tensors have one size."""
    each = [lo + (hi - lo) * (2 * i + 1) // (2 * n) for i in range(n)]
    order = torch.randperm(n, generator=gen, device="cuda")
    return torch.tensor(each, device="cuda", dtype=torch.int32)[order], sum(each)


def _tables(D, n):
    """cos and sin [n, D / 2] of rotate-half RoPE, angles in 64 bits."""
    inv = 10000.0 ** (-torch.arange(0, D, 2, device="cuda", dtype=torch.float64) / D)
    angle = torch.arange(n, device="cuda", dtype=torch.float64)[:, None] * inv
    return angle.cos().float(), angle.sin().float()


def _weight(gen, D, dtype):
    return (1.0 + 0.1 * torch.randn(D, generator=gen, device="cuda")).to(dtype)


def _width(case):
    """Block table entries of a sequence."""
    return (case["hi"] + max(case.get("new", 0), case.get("new_hi", 0))) // case["page"] + 1


def _keys(gen, shape, dtype):
    """Cached keys: those of a page are alike (a part that they share, and one of their own)."""
    k = _randn(gen, shape, torch.bfloat16 if dtype == torch.float8_e4m3fn else dtype).mul_(0.7)
    k += _randn(gen, (shape[0], shape[1], 1, shape[3]), k.dtype).mul_(0.7)
    return k.to(dtype)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    kind, B = case["kind"], case["B"]
    s = {"case": case}
    if kind == "norm_rope":
        Hq, Hkv, T, D, dt = case["Hq"], case["Hkv"], case["T"], case["D"], DTYPES[case["dtype"]]

        def heads(H, scale):
            shape = (B, T, H, D) if case["layout"] == "bthd" else (B, H, T, D)
            x = _randn(gen, shape, dt).mul_(scale)
            return x.transpose(1, 2) if case["layout"] == "bthd" else x

        s.update(q=heads(Hq, 1.5), k=heads(Hkv, 0.6), qw=_weight(gen, D, DTYPES[case["wdtype"]]),
                 kw=_weight(gen, D, DTYPES[case["wdtype"]]))
        s["cos"], s["sin"] = _tables(D, T)
        if case["grad"]:
            s.update(gq=heads(Hq, 1.0), gk=heads(Hkv, 1.0))
            for n in ("q", "k", "qw", "kw"):
                s[n].requires_grad_(True)
        return s
    P = case["page"]
    if kind == "append":
        Hq, Hkv, D, dt, cdt = case["Hq"], case["Hkv"], case["D"], DTYPES[case["dtype"]], DTYPES[case["cache"]]
        new, _ = _new_lens(gen, B, case["lo"], case["hi"])
        before = _spread(gen, B, 0, 4 * P)  # tokens that each sequence has already
        width = (4 * P + case["hi"]) // P + 1
        table = torch.randperm(B * width, generator=gen, device="cuda").view(B, width)
        seq = torch.repeat_interleave(torch.arange(B, device="cuda"), new)
        starts = new.cumsum(0) - new
        pos = torch.arange(seq.numel(), device="cuda") - starts[seq] + before[seq]
        slots = table[seq, pos // P] * P + pos % P
        fused = _randn(gen, (seq.numel(), (Hq + 2 * Hkv) * D), dt)  # one projection's output
        q, k, v = fused.split([Hq * D, Hkv * D, Hkv * D], dim=1)
        s.update(q=q.unflatten(1, (Hq, D)), k=k.unflatten(1, (Hkv, D)), v=v.unflatten(1, (Hkv, D)),
                 qw=_weight(gen, D, dt), kw=_weight(gen, D, dt), positions=pos.to(torch.int32),
                 slots=slots.to(torch.int32), kc=_randn(gen, (B * width, Hkv, P, D), cdt),
                 vc=_randn(gen, (B * width, Hkv, P, D), cdt))
        s["cos"], s["sin"] = _tables(D, N_POSITIONS)
        return s
    width = _width(case)
    lens = _spread(gen, B, case["lo"], case["hi"])
    perm = torch.randperm(B * width, generator=gen, device="cuda").to(torch.int32)
    used = torch.arange(width, device="cuda") < ((lens + P - 1) // P)[:, None]
    s["table"] = torch.where(used, perm.view(B, width), -1)
    s["lens"] = lens
    if kind in ("reserve", "turnover"):
        total = B * width
        n = B if kind == "reserve" else (B + 3) // 4  # sequences with a prompt; the others get one token
        new, n_tokens = _new_lens(gen, n, case["new_lo"], case["new_hi"])
        if kind == "turnover":
            row = torch.randperm(B, generator=gen, device="cuda")[:n]
            new = torch.ones(B, device="cuda", dtype=torch.int32).index_copy_(0, row, new)
            s["finished"] = torch.zeros(B, device="cuda", dtype=torch.bool).index_fill_(0, row, True)
        # the free pages as a stack: those that no sequence has, and room for the others
        free = torch.cat([perm.view(B, width)[~used], perm.view(B, width)[used]])
        n_free = total - int(used.sum())
        free[n_free:] = -1
        s.update(new=new, free=free, n_free=torch.tensor([n_free], device="cuda", dtype=torch.int32),
                 n_tokens=n_tokens + B)
        return s
    cdt = DTYPES[case["cache"]]
    Hkv, D = case["Hkv"], case["D"]
    s["kc"] = _keys(gen, (B * width, Hkv, P, D), cdt)
    s["bounds"] = torch.zeros(B * width, Hkv, 2, D, device="cuda", dtype=torch.uint8).view(cdt) if cdt == torch.float8_e4m3fn \
        else torch.zeros(B * width, Hkv, 2, D, device="cuda", dtype=cdt)
    if kind == "bounds":
        s["before"] = (lens - case["new"]).clamp_(min=0) if case["new"] else torch.zeros_like(lens)
        return s
    s["vc"] = _randn(gen, (B * width, Hkv, P, D), cdt)
    s["q"] = _randn(gen, (B, case["Hq"], 1, D), DTYPES[case["dtype"]])
    _plain_bounds(s["kc"], s["table"], torch.zeros_like(lens), lens, s["bounds"], P, width)
    return s


# ---------------------------------------------------------------------------
# The plain forms.
# ---------------------------------------------------------------------------
def _raw(t):
    """A tensor that torch indexes whatever its type: 8-bit values as their bytes."""
    return t.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t


def _values(t):
    """8-bit values as the numbers they stand for."""
    return t.to(torch.bfloat16) if t.dtype == torch.float8_e4m3fn else t


def _plain_norm_rope(x, w, cos, sin):
    """(y, n, r) in 32 bits: normed and rotated rows, normed rows, reciprocal root mean squares."""
    x = x.float()
    r = torch.rsqrt((x * x).mean(-1, keepdim=True) + NORM_EPS)
    n = x * r
    a, b = (n * w.float()).chunk(2, dim=-1)
    return torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1), n, r


def _plain_norm_rope_grad(g, n, r, w, cos, sin):
    """Gradients of the rows and of the weight, 32 bits."""
    a, b = g.float().chunk(2, dim=-1)
    dz = torch.cat([a * cos + b * sin, b * cos - a * sin], dim=-1)
    dn = dz * w.float()
    dx = r * (dn - n * (dn * n).mean(-1, keepdim=True))
    return dx, (dz * n).sum((0, 1, 2), dtype=torch.float64)


def _plain_train(s):
    out = {}
    for x, w in (("q", "qw"), ("k", "kw")):
        y, n, r = _plain_norm_rope(s[x].detach(), s[w].detach(), s["cos"], s["sin"])
        out[x] = y.to(s[x].dtype)
        if s["case"]["grad"]:
            dx, dw = _plain_norm_rope_grad(s["g" + x], n, r, s[w].detach(), s["cos"], s["sin"])
            out["d" + x], out["d" + w] = dx.to(s[x].dtype), dw.to(s[w].dtype)
    return out


def _plain_append(s):
    P = s["case"]["page"]
    pos = s["positions"].long()
    cos, sin = s["cos"][pos][:, None], s["sin"][pos][:, None]
    q = _plain_norm_rope(s["q"], s["qw"], cos, sin)[0].to(s["q"].dtype)
    k = _plain_norm_rope(s["k"], s["kw"], cos, sin)[0].to(s["kc"].dtype)
    page, row = s["slots"].long() // P, s["slots"].long() % P
    _raw(s["kc"])[page, :, row] = _raw(k)
    _raw(s["vc"])[page, :, row] = _raw(s["v"].to(s["vc"].dtype))
    return q


def _plain_release(table, lens, finished, free, n_free, P):
    W = table.shape[1]
    j = torch.arange(W, device="cuda")
    n = ((lens.clamp(0, W * P) + P - 1) // P)[:, None]
    mine = finished[:, None] & (j < n)
    back = mine & (table >= 0) & (table < free.numel())
    base = n_free.clamp(0, free.numel()).long()
    at = (base + back.flatten().cumsum(0) - 1).view_as(table)
    at = torch.where(back, at, free.numel()).clamp(max=free.numel())
    grown = torch.cat([free, free.new_zeros(1)]).scatter_(0, at.flatten(), table.flatten())
    free.copy_(grown[:-1])
    table.copy_(torch.where(mine, -1, table))
    return (torch.where(finished, 0, lens).to(torch.int32),
            (base + back.sum()).clamp(max=free.numel()).to(torch.int32))


def _plain_reserve(table, lens, new, free, n_free, n_tokens, P):
    B, W = table.shape
    zero = torch.zeros(1, device="cuda", dtype=torch.int64)
    ctx = lens.long().clamp(0, W * P)
    avail = n_free.long().clamp(0, free.numel())
    starts = torch.cat([zero, new.long().clamp(min=0).cumsum(0)]).clamp(max=n_tokens)
    want = (ctx + starts[1:] - starts[:-1]).clamp(max=W * P)
    had = (ctx + P - 1) // P
    need = (want + P - 1) // P - had
    before = need.cumsum(0) - need
    got = torch.minimum((avail - before).clamp(min=0), need)
    length = torch.minimum(want, (had + got) * P)
    i = torch.arange(n_tokens, device="cuda")
    seq = torch.searchsorted(starts[1:], i, right=True)
    live = seq < B
    b = seq.clamp(max=B - 1)
    pos = torch.where(live, ctx[b] + i - starts[b], 0)
    stored = live & (pos < length[b])
    p = (pos // P).clamp(max=W - 1)
    fresh = p >= had[b]
    taken = free[(avail - 1 - before[b] - (p - had[b])).clamp(0, free.numel() - 1)]
    page = torch.where(fresh, taken, table[b, p])
    stored_at = stored & (page >= 0) & (page < free.numel())
    # (a new page's first token enters it into the table; others write the entry that is there)
    enters = stored & fresh & (pos % P == 0)
    cell = torch.where(enters, b * W + p, B * W)
    grown = torch.cat([table.flatten(), table.new_zeros(1)]).scatter_(0, cell, page.to(torch.int32))
    table.copy_(grown[:-1].view(B, W))
    i32 = torch.int32
    return (torch.where(stored_at, page * P + pos % P, -1).to(i32), pos.to(i32), torch.where(live, b, -1).to(i32),
            starts.to(i32), length.to(i32), (avail - got.sum()).to(i32))


def _plain_bounds(kc, table, before, after, bounds, P, most):
    """``most``: table entries that a sequence's new tokens can lie in."""
    B, W = table.shape
    after = after.long().clamp(0, W * P)[:, None]
    j = (before.long().clamp(min=0) // P)[:, None] + torch.arange(most, device="cuda")
    touched = j * P < after
    page = torch.gather(table, 1, j.clamp(max=W - 1)).long()[touched]
    rows = (after - j * P)[touched]  # rows in use, P or more in a full page
    live = (torch.arange(P, device="cuda") < rows[:, None])[:, None, :, None]
    k = _values(_raw(kc)[page].view(kc.dtype))
    lo = torch.where(live, k, math.inf).amin(2)
    hi = torch.where(live, k, -math.inf).amax(2)
    _raw(bounds)[page] = _raw(torch.stack([lo, hi], dim=2).to(bounds.dtype))
    return bounds


def _plain_select(s):
    case, P, K = s["case"], s["case"]["page"], s["case"]["top_k"]
    Hkv, D = case["Hkv"], case["D"]
    B, W = s["table"].shape
    q = s["q"].double().view(B, Hkv, -1, D)
    up, down = q.clamp(min=0).sum(2), q.clamp(max=0).sum(2)
    j = torch.arange(W, device="cuda")
    n = ((s["lens"].clamp(0, W * P) + P - 1) // P)[:, None]
    page = torch.where(j < n, s["table"], 0).long()
    b = _values(_raw(s["bounds"])[page].view(s["bounds"].dtype)).double()  # [B, W, Hkv, 2, D]
    score = ((b[:, :, :, 1] * up[:, None]).sum(-1) + (b[:, :, :, 0] * down[:, None]).sum(-1)).transpose(1, 2)
    always = (j < case["n_first"]) | (j >= n - case["n_last"])
    score = torch.where(always[:, None], math.inf, score)
    score = torch.where((j < n)[:, None], score, -math.inf)
    order = torch.sort(score, dim=-1, descending=True, stable=True).indices[..., :K]
    order = torch.where(order < n[:, None], order, W).sort(-1).values
    pages = torch.where(order < W, order, -1).to(torch.int32)
    return torch.nn.functional.pad(pages, (0, K - pages.shape[-1]), value=-1)


def _plain_sparse(s, pages):
    case, P = s["case"], s["case"]["page"]
    Hkv, D = case["Hkv"], case["D"]
    B, W = s["table"].shape
    listed_ = pages.long().clamp(min=0)
    phys = torch.gather(s["table"].long().clamp(min=0)[:, None].expand(B, Hkv, W), 2, listed_)
    head = torch.arange(Hkv, device="cuda")[:, None]
    token = listed_[..., None] * P + torch.arange(P, device="cuda")
    live = ((pages >= 0)[..., None] & (token < s["lens"][:, None, None, None])).flatten(2)[:, :, None]
    k = _raw(s["kc"])[phys, head].view(s["kc"].dtype).float().flatten(2, 3)
    v = _raw(s["vc"])[phys, head].view(s["vc"].dtype).float().flatten(2, 3)
    q = s["q"].float().view(B, Hkv, -1, D)
    a = torch.matmul(q, k.transpose(2, 3).contiguous()) * (1.0 / math.sqrt(D)) - 0.5
    y = torch.where(live, (a + torch.sqrt(a * a + 1.0)) ** 2, 0.0)
    v = torch.where(live.transpose(2, 3), v, 0.0)
    return (torch.matmul(y, v) / (y.sum(-1, keepdim=True) + EPS)).view(B, -1, D).to(torch.bfloat16)


# ---------------------------------------------------------------------------
# One pass.
# ---------------------------------------------------------------------------
def _package():
    path = str(pathlib.Path(__file__).resolve().parent.parent / "smooth-attn_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import smooth_attn
    return smooth_attn


def _maps(s, release, reserve):
    """The tables of a step (of copies, where the pass changes what it starts from)."""
    table, lens, free, n_free = s["table"], s["lens"], s["free"], s["n_free"]
    if s["case"]["kind"] == "turnover":
        table, free = table.clone(), free.clone()
        lens, n_free = release(table, lens, s["finished"], free, n_free)
    got = reserve(table, lens, s["new"], free, n_free, s["n_tokens"])
    return {"map": list(got), "table": table, "free": free}


def run(s):
    case = s["case"]
    kind = case["kind"]
    if own:
        sa = _package()
        if kind == "norm_rope":
            q, k = sa.sp2norm_qk_norm_rope(s["q"], s["k"], s["qw"], s["kw"], s["cos"], s["sin"], eps=NORM_EPS)
            if not case["grad"]:
                return {"q": q, "k": k}
            dq, dk, dqw, dkw = torch.autograd.grad((q, k), (s["q"], s["k"], s["qw"], s["kw"]), (s["gq"], s["gk"]))
            return {"q": q.detach(), "k": k.detach(), "dq": dq, "dk": dk, "dqw": dqw, "dkw": dkw}
        P = case["page"]
        if kind == "append":
            q = sa.sp2norm_paged_qk_norm_rope_append(s["q"], s["k"], s["v"], s["qw"], s["kw"], s["cos"], s["sin"],
                                                     s["positions"], s["slots"], s["kc"], s["vc"], eps=NORM_EPS,
                                                     block_size=P)
        elif kind in ("reserve", "turnover"):
            return _maps(s, lambda *a: sa.sp2norm_paged_release(*a, block_size=P),
                         lambda *a: sa.sp2norm_paged_reserve(*a, block_size=P))
        elif kind == "bounds":
            sa.sp2norm_paged_key_bounds(s["kc"], s["table"], s["before"], s["lens"], s["bounds"], block_size=P)
        else:
            pages = sa.sp2norm_paged_select_pages(s["q"], s["bounds"], s["table"], s["lens"], case["top_k"],
                                                  n_first=case["n_first"], n_last=case["n_last"], block_size=P)
            o = sa.sp2norm_paged_sparse_attention(s["q"], s["kc"], s["vc"], s["table"], s["lens"], pages,
                                                  block_size=P)
            return {"pages": pages, "o": o}
    else:
        if kind == "norm_rope":
            return _plain_train(s)
        P = case["page"]
        if kind == "append":
            q = _plain_append(s)
        elif kind in ("reserve", "turnover"):
            return _maps(s, lambda *a: _plain_release(*a, P), lambda *a: _plain_reserve(*a, P))
        elif kind == "bounds":
            _plain_bounds(s["kc"], s["table"], s["before"], s["lens"], s["bounds"], P,
                          (case["new"] + P - 2) // P + 1 if case["new"] else s["table"].shape[1])
        else:
            pages = _plain_select(s)
            return {"pages": pages, "o": _plain_sparse(s, pages)}
    if kind == "append":
        return {"q": q, "kc": _values(s["kc"]), "vc": _values(s["vc"])}
    return _values(s["bounds"])


# ---------------------------------------------------------------------------
# What a pass cannot do without.
# ---------------------------------------------------------------------------
def work(case):
    kind, B = case["kind"], case["B"]
    if kind == "norm_rope":
        e, D = SIZES[case["dtype"]], case["D"]
        n = B * (case["Hq"] + case["Hkv"]) * case["T"] * D
        tables = 4 * case["T"] * D
        if case["grad"]:  # x in, y out; x and dy in, dx out
            return {"bytes": 5 * e * n + tables, "flops": 26 * n}
        return {"bytes": 2 * e * n + tables, "flops": 8 * n}
    P = case["page"]
    mid = (case["lo"] + case["hi"]) / 2
    if kind == "append":
        N, D, e, c = B * mid, case["D"], SIZES[case["dtype"]], SIZES[case["cache"]]
        per = case["Hq"] * D * 2 * e + 2 * case["Hkv"] * D * (e + c) + 8 + 4 * D
        return {"bytes": int(N * per), "flops": int(N * (case["Hq"] + case["Hkv"]) * D * 8)}
    if kind in ("reserve", "turnover"):
        new = (case["new_lo"] + case["new_hi"]) / 2
        tokens = B * new if kind == "reserve" else B / 4 * new + 0.75 * B
        size = 24 * B + 12 * tokens + 8 * tokens / P
        if kind == "turnover":
            size += 12 * B / 4 * mid / P
        return {"bytes": int(size), "flops": int(8 * tokens)}
    c, Hkv, D = SIZES[case["cache"]], case["Hkv"], case["D"]
    if kind == "bounds":
        pages = B * (mid / P if not case["new"] else 1 + (case["new"] - 1) / P)
        rows = B * mid if not case["new"] else B * ((P + 1) / 2 + case["new"] - 1)
        return {"bytes": int(Hkv * D * c * (rows + 2 * pages) + 4 * pages + 8 * B), "flops": int(2 * Hkv * D * rows)}
    pages = B * mid / P
    kept = B * min(case["top_k"], mid / P)
    size = Hkv * D * c * (2 * pages + 2 * P * kept) + 4 * pages + 8 * Hkv * kept + B * case["Hq"] * D * (SIZES[case["dtype"]] + 2)
    return {"bytes": int(size), "flops": int(4 * Hkv * D * pages + 4 * case["Hq"] * D * P * kept)}


# ---------------------------------------------------------------------------
# The same results in 64 bits, sequence by sequence.
# ---------------------------------------------------------------------------
def _turn64(x, c, s):
    """Rows turned by the angles of c and s: each pair (d, d + D / 2) as one complex number."""
    half = x.shape[-1] // 2
    z = torch.complex(x[..., :half], x[..., half:]) * torch.complex(c, s)
    return torch.cat([z.real, z.imag], dim=-1)


def _norm64(x, w):
    x = x.double()
    scale = (x.square().sum(-1, keepdim=True) / x.shape[-1] + NORM_EPS) ** -0.5
    return x * scale * w.double(), scale


def _train64(s):
    out = {}
    c, sn = s["cos"].double(), s["sin"].double()
    for name in ("q", "k"):
        x, w = s[name].detach(), s[name + "w"].detach().double()
        y = torch.empty(x.shape, dtype=torch.float64, device="cuda")
        dx = torch.empty_like(y)
        dw = torch.zeros_like(w)
        for b in range(x.shape[0]):
            z, r = _norm64(x[b], w)
            y[b] = _turn64(z, c, sn)
            if s["case"]["grad"]:
                dz = _turn64(s["g" + name][b].double(), c, -sn)
                xb = x[b].double()
                dw += (dz * xb * r).sum((0, 1))
                h = dz * w
                dx[b] = r * h - xb * r ** 3 * ((h * xb).sum(-1, keepdim=True) / xb.shape[-1])
        out[name] = y
        if s["case"]["grad"]:
            out["d" + name], out["d" + name + "w"] = dx, dw
    return out


def _sparse64(s):
    case, P = s["case"], s["case"]["page"]
    B, Hq, _, D = s["q"].shape
    Hkv, K = case["Hkv"], case["top_k"]
    G = Hq // Hkv
    pages = torch.full((B, Hkv, K), -1, dtype=torch.int32)
    o = torch.zeros(B, Hq, D, dtype=torch.float64, device="cuda")
    bounds, kc, vc = (_raw(s[n]) for n in ("bounds", "kc", "vc"))
    for b, n in enumerate(s["lens"].tolist()):
        np_ = -(-n // P)
        phys = s["table"][b, :np_].long()
        for h in range(Hkv):
            q = s["q"][b, h * G:(h + 1) * G, 0].double()
            bd = bounds[phys, h].view(s["bounds"].dtype).double()
            # each query head's largest product with any key between the bounds, dimension by dimension
            best = sum(torch.maximum(bd[:, 0] * q[g], bd[:, 1] * q[g]).sum(-1) for g in range(G)).tolist()
            forced = set(range(min(case["n_first"], np_))) | set(range(max(0, np_ - case["n_last"]), np_))
            rest = sorted((j for j in range(np_) if j not in forced), key=lambda j: (-best[j], j))
            mine = sorted((sorted(forced) + rest)[:K]) if np_ > K else list(range(np_))
            pages[b, h, :len(mine)] = torch.tensor(mine, dtype=torch.int32)
            at = phys[torch.tensor(mine, device="cuda")]
            rows = torch.cat([torch.arange(j * P, min(j * P + P, n)) - j * P + i * P for i, j in enumerate(mine)]).cuda()
            kk = kc[at, h].view(s["kc"].dtype).double().reshape(-1, D)[rows]
            vv = vc[at, h].view(s["vc"].dtype).double().reshape(-1, D)[rows]
            arg = 2.0 * (q @ kk.t().contiguous()) / math.sqrt(D) - 1.0
            y = (0.5 * (arg + torch.sqrt(arg * arg + 4.0))) ** 2
            o[b, h * G:(h + 1) * G] = (y @ vv) / (y.sum(-1, keepdim=True) + EPS)
    return {"pages": pages.cuda(), "o": o}


@torch.no_grad()
def exact(case, seed):
    kind = case["kind"]
    if kind in ("reserve", "turnover"):
        return None  # whole numbers
    s = prepare(case, seed)
    if kind == "norm_rope":
        return _train64(s)
    P = case["page"]
    if kind == "append":
        pos = s["positions"].long()
        c, sn = s["cos"][pos].double()[:, None], s["sin"][pos].double()[:, None]
        page, row = s["slots"].long().div(P, rounding_mode="floor"), s["slots"].long().remainder(P)
        out = {"q": _turn64(_norm64(s["q"], s["qw"])[0], c, sn)}
        for name, new in (("kc", _turn64(_norm64(s["k"], s["kw"])[0], c, sn)), ("vc", s["v"].double())):
            cache = _values(s[name]).double()
            if s[name].dtype == torch.float8_e4m3fn:
                new = new.to(torch.float8_e4m3fn).double()  # what the cache can hold is the result
            cache[page, :, row] = new
            out[name] = cache
        return out
    if kind == "bounds":
        bounds = _values(s["bounds"]).double()
        after, before = s["lens"].tolist(), s["before"].tolist()
        k = _values(s["kc"])
        for b in range(case["B"]):
            first, full = before[b] // P, after[b] // P
            at = s["table"][b, first:full].long()
            bounds[at] = torch.stack(torch.aminmax(k[at].double(), dim=2), dim=2)
            if after[b] % P:
                at = int(s["table"][b, full])
                bounds[at] = torch.stack(torch.aminmax(k[at, :, :after[b] % P].double(), dim=1), dim=1)
        return bounds
    return _sparse64(s)
