"""Operators of a serving step around the paged attention: pages and slot maps
from lengths, normed and rotated keys into the caches, and attention over chosen
pages.  Everything stays on the device.  No counterpart in the reference.

A step over packed new tokens (one each in decode, whole prompts in prefill):

    r = sp2norm_paged_reserve(table, lens, new_lens, free_pages, n_free, n_tokens)
    q = sp2norm_paged_qk_norm_rope_append(q, k, v, q_weight, k_weight, cos, sin, r.positions, r.slots, kc, vc)
    sp2norm_paged_key_bounds(kc, table, lens, r.context_lens, bounds)
    pages = sp2norm_paged_select_pages(q[:, :, None], bounds, table, r.context_lens, top_k)   # decode
    o = sp2norm_paged_sparse_attention(q[:, :, None], kc, vc, table, r.context_lens, pages)

The caches and tables are plain tensors of the caller's; none of these calls
has a gradient (like the paged attention).
"""
from __future__ import annotations

import math
from typing import NamedTuple

import torch

from . import _lib
from .kernels import (_CACHE_CODE, _DTYPE_CODE, _PAGED_CACHE_DTYPES, _check_paging_args, _check_same_device,
                      _device_of, _flash_operand, _native, _paged_dtype_code, _rope_tables, _stream)
from .qk_norm import MAX_NORM_TOKENS, _check_norm_args, _check_tensors, _int32, _norm_weights, _output_like

__all__ = ["PagedReservation", "sp2norm_paged_key_bounds", "sp2norm_paged_qk_norm_rope_append",
           "sp2norm_paged_release", "sp2norm_paged_reserve", "sp2norm_paged_select_pages",
           "sp2norm_paged_sparse_attention"]

# Sequences of one reservation (their sums lie in a workgroup's shared memory).
MAX_RESERVED_SEQS = 4096


class PagedReservation(NamedTuple):
    """What sp2norm_paged_reserve returns; all int32 on the device.  The three maps
    of tokens may share one allocation, and the others another."""

    slots: torch.Tensor         # [n_tokens] cache slot of each packed token, -1 for none
    positions: torch.Tensor     # [n_tokens] its position in its sequence
    sequences: torch.Tensor     # [n_tokens] its sequence, -1 past the last token
    starts: torch.Tensor        # [B + 1] packed position of each sequence's first new token
    context_lens: torch.Tensor  # [B] lengths with the new tokens that have pages
    n_free: torch.Tensor        # [1] free pages left


def _check_block_size(block_size, n_pages, power_of_two=False):
    if block_size < 1 or (power_of_two and block_size & (block_size - 1)):
        raise ValueError(f"block_size must be {'a power of two' if power_of_two else 'positive'}, got {block_size}")
    if n_pages * block_size >= 1 << 31:
        raise ValueError(f"{n_pages} pages of {block_size} tokens do not fit 32-bit slots")


def _check_maps(block_table, lens, free_pages, n_free, block_size):
    """Arguments that reserve and release share; the table and the stack are
    written in place, so they are taken as they are or refused."""
    if block_table.ndim != 2 or block_table.dtype != torch.int32:
        raise ValueError(f"block_table must be an int32 tensor [B, max_pages], got {block_table.dtype} "
                         f"{tuple(block_table.shape)}")
    B, W = block_table.shape
    if B > MAX_RESERVED_SEQS:
        raise ValueError(f"at most {MAX_RESERVED_SEQS} sequences, got {B}")
    if W and B and (block_table.stride(1) != 1 or (B > 1 and block_table.stride(0) < W)):
        raise ValueError("block_table needs rows of consecutive entries that do not overlap")
    for name, t in lens.items():
        if t.shape != (B,):
            raise ValueError(f"{name} must be [{B}], got {tuple(t.shape)}")
    if free_pages.dtype != torch.int32 or free_pages.ndim != 1 or not free_pages.is_contiguous():
        raise ValueError("free_pages must be a contiguous int32 tensor [n_pages]")
    if n_free.dtype != torch.int32 or n_free.numel() != 1:
        raise ValueError("n_free must be an int32 tensor of one element")
    _check_block_size(block_size, max(free_pages.numel(), W))
    return B, W


def sp2norm_paged_reserve(block_table, context_lens, new_lens, free_pages, n_free, n_tokens, *, block_size=16):
    """Pages for the new tokens of a step, with the maps that the step needs.

    block_table: int32 [B, max_pages], updated in place past the pages that each
    sequence has; context_lens, new_lens: integer [B], tokens that each sequence
    has and gets (0 for none); free_pages: int32 [n_pages], as long as the caches
    have pages (other ids name none), a stack of free page ids of which the first
    n_free (int32, one element) count; n_tokens: room of the packed token tensors
    (an int; tokens past the sum get slot -1).

    A sequence has the first ceil(context_lens[b] / block_size) entries of its
    table row; those past them are taken as empty and overwritten.  So a length
    may not be cut below a page border (rejected tokens, say) before the caller
    has put the pages past it back on the stack: they would be lost to it.

    Sequences are served in their order.  One that finds too few pages, or
    reaches the end of its table row or of the packed tokens, is cut: its
    context_lens in the result says how many tokens have pages, and the others'
    slots are -1.  Returns a PagedReservation; only block_table changes, so
    pass its n_free and context_lens to the next call."""
    out = _native().paged_reserve(block_table, context_lens, new_lens, free_pages, n_free, n_tokens, block_size)
    if out is not None:
        return PagedReservation._make(out)
    _check_tensors(block_table=block_table, context_lens=context_lens, new_lens=new_lens, free_pages=free_pages,
                   n_free=n_free)
    B, W = _check_maps(block_table, {"context_lens": context_lens, "new_lens": new_lens}, free_pages, n_free,
                       block_size)
    n_tokens = int(n_tokens)
    if not 0 <= n_tokens < 1 << 31:
        raise ValueError(f"n_tokens must be in 0..2^31 - 1, got {n_tokens}")
    _check_same_device("block_table", block_table, context_lens=context_lens, new_lens=new_lens,
                       free_pages=free_pages, n_free=n_free)
    ctx, new = _int32("context_lens", context_lens), _int32("new_lens", new_lens)
    empty = lambda n: torch.empty(n, dtype=torch.int32, device=block_table.device)  # noqa: E731
    out = PagedReservation(empty(n_tokens), empty(n_tokens), empty(n_tokens), empty(B + 1), empty(B), empty(1))
    with _device_of(block_table):
        st = _lib.load().sa_paged_reserve(
            block_table.data_ptr(), ctx.data_ptr(), new.data_ptr(), free_pages.data_ptr(), n_free.data_ptr(),
            *(t.data_ptr() for t in out), B, W, block_size, free_pages.numel(), n_tokens,
            max(block_table.stride(0), W), _stream(block_table))
    _lib.check(st, "sa_paged_reserve")
    return out


def sp2norm_paged_release(block_table, context_lens, finished, free_pages, n_free, *, block_size=16):
    """Give the pages of finished sequences (bool [B]) back: they are pushed on
    the stack free_pages in place, in the order of the sequences and their
    tables, and their table entries become -1: the pages of context_lens[b] tokens,
    not entries past them.  A page goes on the stack as often as a finished
    sequence's table names it: one that other sequences still read has to leave the
    table (-1) first.  Returns (context_lens, n_free): lengths
    with 0 for the finished ones, and the new number of free pages."""
    out = _native().paged_release(block_table, context_lens, finished, free_pages, n_free, block_size)
    if out is not None:
        return out
    _check_tensors(block_table=block_table, context_lens=context_lens, finished=finished, free_pages=free_pages,
                   n_free=n_free)
    B, W = _check_maps(block_table, {"context_lens": context_lens, "finished": finished}, free_pages, n_free,
                       block_size)
    if finished.dtype != torch.bool:
        raise ValueError(f"finished must be a bool tensor, got {finished.dtype}")
    _check_same_device("block_table", block_table, context_lens=context_lens, finished=finished,
                       free_pages=free_pages, n_free=n_free)
    ctx, finished = _int32("context_lens", context_lens), finished.contiguous()
    lens, left = torch.empty_like(ctx), torch.empty(1, dtype=torch.int32, device=ctx.device)
    if B == 0:
        return lens, n_free.reshape(1).clone()
    counts = torch.empty_like(ctx)
    with _device_of(block_table):
        st = _lib.load().sa_paged_release(
            block_table.data_ptr(), ctx.data_ptr(), finished.data_ptr(), free_pages.data_ptr(), n_free.data_ptr(),
            lens.data_ptr(), left.data_ptr(), counts.data_ptr(), B, W, block_size, free_pages.numel(),
            max(block_table.stride(0), W), _stream(block_table))
    _lib.check(st, "sa_paged_release")
    return lens, left


def _check_caches(block_size, **caches):
    """Caches that a call writes: 16-byte rows, taken as they are or refused."""
    for name, t in caches.items():
        if t.ndim != 4 or t.shape[2] != block_size:
            raise ValueError(f"{name} must be [n_pages, H_kv, {block_size}, D], got {tuple(t.shape)}")
        if t.dtype not in _PAGED_CACHE_DTYPES:
            raise ValueError("paged caches must be fp32, bf16, fp16 or e4m3fn of one dtype")
        per = 16 // t.element_size()
        if t.numel() and (t.stride(-1) != 1 or any(s % per for s in t.stride()[:-1]) or t.data_ptr() % 16
                          or t.shape[3] % per):
            raise ValueError("paged caches need 16-byte aligned rows with unit stride along D")


def sp2norm_paged_qk_norm_rope_append(q, k, v, q_weight, k_weight, cos, sin, positions, slots, k_cache, v_cache, *,
                                      eps=1e-6, block_size=16):
    """sp2norm_qk_norm_rope of a serving step's packed tokens, with the caches'
    update in the same pass.

    q: [N, Hq, D], k, v: [N, Hkv, D] (any strides: parts of one projection's
    output are read as they lie); positions, slots: integer [N]
    (sp2norm_paged_reserve); k_cache, v_cache: [n_pages, Hkv, block_size, D] of
    one dtype (fp32, bf16, fp16 or e4m3fn).  Token i's key, normed and turned by
    row positions[i] of the tables, and its value go to row slots[i] of the
    caches, each rounded once to their type; a negative slot writes nothing.
    The slots of a call that are not negative must differ.  Returns the normed
    and rotated queries [N, Hq, D] (``[:, :, None]`` of them is a decode's q)."""
    out = _native().paged_norm_append(q, k, v, q_weight, k_weight, cos, sin, positions, slots, k_cache, v_cache, eps,
                                      block_size)
    if out is not None:
        return out
    _check_tensors(q=q, k=k, v=v, q_weight=q_weight, k_weight=k_weight, cos=cos, sin=sin, positions=positions,
                   slots=slots, k_cache=k_cache, v_cache=v_cache)
    if q.ndim != 3 or k.ndim != 3 or v.shape != k.shape or k.shape[0] != q.shape[0] or k.shape[2] != q.shape[2]:
        raise ValueError(f"q must be [N, H_q, D] and k and v [N, H_kv, D], got {tuple(q.shape)}, {tuple(k.shape)}, "
                         f"{tuple(v.shape)}")
    N, Hq, D = q.shape
    Hkv = k.shape[1]
    with torch.no_grad():
        _check_norm_args(("q", "k", "v"), (q, k, v), (q_weight, k_weight), cos, sin, D)
        if N > MAX_NORM_TOKENS:
            raise ValueError(f"the norm takes at most {MAX_NORM_TOKENS} tokens, got {N}")
        _check_caches(block_size, k_cache=k_cache, v_cache=v_cache)
        if v_cache.shape != k_cache.shape or v_cache.dtype != k_cache.dtype or k_cache.shape[1] != Hkv \
                or k_cache.shape[3] != D:
            raise ValueError(f"k_cache and v_cache must both be [n_pages, {Hkv}, {block_size}, {D}] of one dtype")
        _check_block_size(block_size, k_cache.shape[0])
        for name, t in (("positions", positions), ("slots", slots)):
            if t.shape != (N,):
                raise ValueError(f"{name} must be [{N}], got {tuple(t.shape)}")
        if cos.shape[0] == 0 and N > 0:
            raise ValueError("cos and sin have no rows")
        _check_same_device("q", q, k=k, v=v, q_weight=q_weight, k_weight=k_weight, cos=cos, sin=sin, positions=positions,
                           slots=slots, k_cache=k_cache, v_cache=v_cache)
        cos, sin = _rope_tables(cos, sin, N, D)
        positions, slots = _int32("positions", positions), _int32("slots", slots)
        (qw, kw), w_code = _norm_weights(q.dtype, q_weight, k_weight)
        q, k, v = _flash_operand(q), _flash_operand(k), _flash_operand(v)
        q_out = _output_like(q)
        with _device_of(q):
            st = _lib.load().sa_paged_qk_norm_rope_append(
                q.data_ptr(), k.data_ptr(), v.data_ptr(), q_out.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(),
                _lib.ptr(qw), _lib.ptr(kw), cos.data_ptr(), sin.data_ptr(), positions.data_ptr(), slots.data_ptr(),
                N, Hq, Hkv, D, cos.shape[0], block_size, k_cache.shape[0], _lib.strides(q), _lib.strides(k),
                _lib.strides(v), _lib.strides(q_out), _lib.strides(k_cache), _lib.strides(v_cache), float(eps),
                _DTYPE_CODE[q.dtype], w_code, _CACHE_CODE[k_cache.dtype], _stream(q))
        _lib.check(st, "sa_paged_qk_norm_rope_append")
        return q_out


def _check_table(B, block_table, **lens):
    if block_table.ndim != 2 or block_table.shape[0] < B:
        raise ValueError(f"block_table must be [B={B}, max_pages], got {tuple(block_table.shape)}")
    for name, t in lens.items():
        if t.ndim != 1 or t.numel() < B:
            raise ValueError(f"{name} must hold B={B} lengths, got {tuple(t.shape)}")
    table = _int32("block_table", block_table) if block_table.dtype != torch.int32 else block_table
    if table.shape[1] and table.stride(-1) != 1 or table.shape[0] > 1 and table.stride(0) < table.shape[1]:
        table = table.contiguous()
    return table, [_int32(name, t) for name, t in lens.items()]


def _bt_stride(table):
    return max(table.stride(0), table.shape[1])


def _check_paged_head_dim(D, cache_dtype):
    step = 16 if cache_dtype == torch.float8_e4m3fn else 8
    if D % step or not step <= D <= 1024:
        raise ValueError(f"page bounds over {cache_dtype} caches support head dims that are multiples of {step} in "
                         f"{step}..1024, got {D}")


def sp2norm_paged_key_bounds(k_cache, block_table, from_lens, to_lens, bounds=None, *, block_size=16):
    """Smallest and largest value of each key column over the tokens of a page,
    for the pages that hold tokens from_lens[b] .. to_lens[b] - 1 of each
    sequence (the lengths before and after a step).

    bounds: contiguous [n_pages, Hkv, 2, D] of the cache's dtype, updated in
    place and returned (None: a new one, of zeros elsewhere); [:, :, 0] holds the
    smallest values, [:, :, 1] the largest, NaN where a key is.  All of a page's
    tokens below to_lens count, so a page that is filled step by step is right
    after each; one that sequences share must be full in each.  Table entries that
    name no page are skipped."""
    if _native().paged_key_bounds(k_cache, block_table, from_lens, to_lens, bounds, block_size):
        return bounds
    _check_tensors(k_cache=k_cache, block_table=block_table, from_lens=from_lens, to_lens=to_lens, bounds=bounds)
    if k_cache.ndim != 4:
        raise ValueError(f"k_cache must be [n_pages, H_kv, block_size, D], got {tuple(k_cache.shape)}")
    n_pages, Hkv, _, D = k_cache.shape
    if k_cache.shape[2] != block_size or k_cache.dtype not in _PAGED_CACHE_DTYPES:
        raise ValueError(f"k_cache must be [n_pages, H_kv, {block_size}, D] of fp32, bf16, fp16 or e4m3fn")
    _check_block_size(block_size, n_pages, power_of_two=True)
    _check_paged_head_dim(D, k_cache.dtype)
    if block_table.ndim != 2:
        raise ValueError(f"block_table must be [B, max_pages], got {tuple(block_table.shape)}")
    B = block_table.shape[0]
    if bounds is None:
        bounds = torch.zeros(n_pages, Hkv, 2, D * k_cache.element_size(), dtype=torch.uint8,
                             device=k_cache.device).view(k_cache.dtype)
    if bounds.shape != (n_pages, Hkv, 2, D) or bounds.dtype != k_cache.dtype or not bounds.is_contiguous() \
            or bounds.data_ptr() % 16:
        raise ValueError(f"bounds must be a contiguous [{n_pages}, {Hkv}, 2, {D}] tensor of {k_cache.dtype}")
    table, (lo, hi) = _check_table(B, block_table, from_lens=from_lens, to_lens=to_lens)
    _check_same_device("k_cache", k_cache, block_table=block_table, from_lens=from_lens, to_lens=to_lens,
                       bounds=bounds)
    k_cache = _flash_operand(k_cache.detach())
    with _device_of(k_cache):
        st = _lib.load().sa_paged_key_bounds(
            k_cache.data_ptr(), bounds.data_ptr(), table.data_ptr(), lo.data_ptr(), hi.data_ptr(), B, Hkv, D,
            block_size, table.shape[1], n_pages, _lib.strides(k_cache), _bt_stride(table),
            _CACHE_CODE[k_cache.dtype], _stream(k_cache))
    _lib.check(st, "sa_paged_key_bounds")
    return bounds


def sp2norm_paged_select_pages(q, bounds, block_table, context_lens, top_k, *, n_first=0, n_last=1, block_size=16):
    """The pages that one query token of each sequence attends to, by the bounds
    of their keys: int32 [B, Hkv, top_k], indexes into the sequence's table row
    in ascending order, then -1.

    q: [B, Hq, 1, D]; bounds: sp2norm_paged_key_bounds.  A sequence of at most
    top_k pages has them all; else the first n_first, the last n_last, and the
    others with the largest upper bound of the sum over the KV head's query
    heads of q . k, computed in 64 bits (equal bounds: the lower page; NaN above
    all).  With n_last >= 1 the page that is being filled is always there, so
    its bounds may be behind."""
    pages = _native().paged_select_pages(q, bounds, block_table, context_lens, top_k, n_first, n_last, block_size)
    if pages is not None:
        return pages
    _check_tensors(q=q, bounds=bounds, block_table=block_table, context_lens=context_lens)
    if q.ndim != 4 or q.shape[2] != 1:
        raise ValueError(f"q must be [B, H_q, 1, D], got {tuple(q.shape)}")
    B, Hq, _, D = q.shape
    if bounds.ndim != 4 or bounds.shape[2] != 2 or bounds.shape[3] != D or bounds.dtype not in _PAGED_CACHE_DTYPES:
        raise ValueError(f"bounds must be [n_pages, H_kv, 2, {D}] of fp32, bf16, fp16 or e4m3fn, got "
                         f"{bounds.dtype} {tuple(bounds.shape)}")
    n_pages, Hkv = bounds.shape[:2]
    if Hkv == 0 or Hq % Hkv or Hq == 0:
        raise ValueError(f"H_q ({Hq}) must be a multiple of H_kv ({Hkv})")
    _check_block_size(block_size, n_pages, power_of_two=True)
    _check_paged_head_dim(D, bounds.dtype)
    if q.dtype not in _PAGED_CACHE_DTYPES:
        raise ValueError(f"q must be fp32, bf16, fp16 or e4m3fn, got {q.dtype}")
    top_k, n_first, n_last = int(top_k), int(n_first), int(n_last)
    if n_first < 0 or n_last < 0 or not max(1, n_first + n_last) <= top_k < 1 << 24:
        raise ValueError(f"top_k must be at least 1 and n_first + n_last, got {top_k} for {n_first} + {n_last}")
    table, (ctx,) = _check_table(B, block_table, context_lens=context_lens)
    _check_same_device("q", q, bounds=bounds, block_table=block_table, context_lens=context_lens)
    q = q.detach()
    if q.dtype == torch.float8_e4m3fn:
        q = q.float()
    q = _flash_operand(q)
    if not bounds.is_contiguous() or bounds.data_ptr() % 16:
        bounds = bounds.clone(memory_format=torch.contiguous_format)
    pages = torch.empty(B, Hkv, top_k, dtype=torch.int32, device=q.device)
    if B == 0:
        return pages
    lib = _lib.load()
    W = table.shape[1]
    ws = torch.empty(max(8, lib.sa_paged_select_workspace_size(B, Hkv, W) if top_k < W else 0), dtype=torch.uint8,
                     device=q.device)
    with _device_of(q):
        st = lib.sa_paged_select_pages(
            q.data_ptr(), bounds.data_ptr(), table.data_ptr(), ctx.data_ptr(), pages.data_ptr(), B, Hq, Hkv, D,
            block_size, W, n_pages, top_k, n_first, n_last, _lib.strides(q), _bt_stride(table),
            _DTYPE_CODE[q.dtype], _CACHE_CODE[bounds.dtype], ws.data_ptr(), ws.numel(), _stream(q))
    _lib.check(st, "sa_paged_select_pages")
    return pages


def sp2norm_paged_sparse_attention(q, k_cache, v_cache, block_table, context_lens, pages, *, scale=None,
                                   block_size=16):
    """sp2norm_paged_attention over listed pages only (output bf16 [B, Hq, D]).

    pages: integer [B, Hkv, n], indexes into the sequence's table row for each
    KV head (sp2norm_paged_select_pages), in any order; indexes outside the
    table are skipped, of a page the tokens below context_lens[b] count, and a
    page that is listed twice counts twice.  No token at all gives zeros.  The
    other arguments, types and head dims are sp2norm_paged_attention's.  Scores
    (scale q . k) may reach 1023 where q and the caches are fp16."""
    out = _native().paged_sparse(q, k_cache, v_cache, block_table, context_lens, pages, scale, block_size)
    if out is not None:
        return out
    _check_tensors(q=q, k_cache=k_cache, v_cache=v_cache, block_table=block_table, context_lens=context_lens,
                   pages=pages)
    if q.ndim != 4 or q.shape[2] != 1:
        raise ValueError(f"q must be [B, H_q, 1, D], got {tuple(q.shape)}")
    B, Hq, _, D = q.shape
    if k_cache.ndim != 4 or k_cache.shape[2] != block_size:
        raise ValueError(f"k_cache must be [n_pages, H_kv, {block_size}, {D}], got {tuple(k_cache.shape)}")
    Hkv = k_cache.shape[1]
    if Hkv == 0 or Hq == 0 or Hq % Hkv or Hq // Hkv > 32:
        raise ValueError(f"H_q ({Hq}) must be 1 to 32 times H_kv ({Hkv})")
    _check_block_size(block_size, k_cache.shape[0], power_of_two=True)
    code = _paged_dtype_code(q.dtype, k_cache.dtype, v_cache.dtype)
    if D % 8 or not 8 <= D <= 1024 or (k_cache.dtype == torch.float8_e4m3fn and D % 16):
        raise ValueError(f"paged decode over {k_cache.dtype} caches does not support head dim {D}")
    if D > 512 and (k_cache.dtype == torch.float32 or (k_cache.dtype == torch.float16 and q.dtype != torch.float16)):
        raise ValueError(f"paged decode over {k_cache.dtype} caches with a {q.dtype} q supports head dims up to 512, "
                         f"got {D}")
    _check_paging_args(B, D, k_cache, v_cache, block_table, context_lens)
    table, (ctx,) = _check_table(B, block_table, context_lens=context_lens)
    if pages.ndim != 3 or pages.shape[:2] != (B, Hkv):
        raise ValueError(f"pages must be [{B}, {Hkv}, n], got {tuple(pages.shape)}")
    _check_same_device("q", q, k_cache=k_cache, v_cache=v_cache, block_table=block_table, context_lens=context_lens,
                       pages=pages)
    pages = _int32("pages", pages)
    if scale is None:
        scale = 1.0 / math.sqrt(D)
    q = q.detach()
    if (code & 0xFF) == _lib.SA_F32 and q.dtype != torch.float32:
        q = q.float()  # exact
    q, k_cache, v_cache = _flash_operand(q), _flash_operand(k_cache.detach()), _flash_operand(v_cache.detach())
    out = torch.empty(B, Hq, D, device=q.device, dtype=torch.bfloat16)
    lib = _lib.load()
    n = pages.shape[2]
    ws = torch.empty(max(16, lib.sa_paged_sparse_workspace_size(B, Hq, Hkv, D, n, block_size)), dtype=torch.uint8,
                     device=q.device)
    with _device_of(q):
        st = lib.sa_paged_sparse_decode(
            q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), out.data_ptr(), table.data_ptr(), ctx.data_ptr(),
            pages.data_ptr(), B, Hq, Hkv, D, block_size, table.shape[1], k_cache.shape[0], n, _lib.strides(q),
            _lib.strides(k_cache), _lib.strides(v_cache), _lib.strides(out), _bt_stride(table), float(scale), code,
            ws.data_ptr(), ws.numel(), _stream(q))
    _lib.check(st, "sa_paged_sparse_decode")
    return out
