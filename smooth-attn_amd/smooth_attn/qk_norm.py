"""RMS norm of each head's queries and keys with rotate-half RoPE, in one pass
and with its gradients: the step before the fused attention in a model that
norms its queries and keys.  No counterpart in the reference."""
from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from .kernels import _DTYPE_CODE, _check_same_device, _device_of, _flash_operand, _native, _rope_tables, _stream


__all__ = ["sp2norm_qk_norm_rope"]


def _check_tensors(**tensors):
    """Arguments that must be tensors (None: not given)."""
    for name, t in tensors.items():
        if t is not None and not isinstance(t, torch.Tensor):
            raise TypeError(f"{name} must be a torch.Tensor")


def _check_norm_args(names, tensors, weights, cos, sin, D):
    """Types and shapes that the norm's entry points share."""
    first = tensors[0]
    if first.dtype not in _DTYPE_CODE or any(t.dtype != first.dtype for t in tensors):
        raise ValueError(f"the norm expects bf16, fp16 or fp32 {'/'.join(names)} of one dtype, got "
                         f"{'/'.join(str(t.dtype) for t in tensors)}")
    if D % 16 or not 16 <= D <= 512:
        raise ValueError(f"the norm supports head dims that are multiples of 16 in 16..512, got {D}")
    if any(t.shape[1] > MAX_NORM_HEADS for t in tensors):
        raise ValueError(f"the norm takes at most {MAX_NORM_HEADS} heads of {'/'.join(names)}, got "
                         f"{'/'.join(str(t.shape[1]) for t in tensors)}")
    for name, w in zip(("q_weight", "k_weight"), weights):
        if w is not None and (w.shape != (D,) or w.dtype not in (torch.float32, first.dtype)):
            raise ValueError(f"{name} must be [{D}] of {first.dtype} or float32, got {tuple(w.shape)} of {w.dtype}")
    if cos.ndim != 2 or cos.shape[1] != D // 2 or sin.shape != cos.shape:
        raise ValueError(f"cos and sin must both be [positions, {D // 2}], got {tuple(cos.shape)} / {tuple(sin.shape)}")
    if not cos.dtype.is_floating_point or not sin.dtype.is_floating_point:
        raise ValueError("cos and sin must be floating point")
    if torch.is_grad_enabled() and (cos.requires_grad or sin.requires_grad):
        raise ValueError("cos and sin have no gradient: pass them detached")


_INT_DTYPES = (torch.int32, torch.int64, torch.int16, torch.int8, torch.uint8)
# Tokens of one launch (heads and head dims past them make up the rest of 2^32 threads).
MAX_NORM_TOKENS = 1 << 24
# Heads of q or of k (each may be a row of the launch's grid).
MAX_NORM_HEADS = 65535 // 4


def _int32(name, t):
    """A contiguous 32-bit copy or view of an integer tensor; 64-bit values past
    32 bits become the nearest that fit, so none is taken for another."""
    if t.dtype not in _INT_DTYPES:
        raise ValueError(f"{name} must be an integer tensor, got {t.dtype}")
    if t.dtype == torch.int64:
        t = t.clamp(-(1 << 31), (1 << 31) - 1)
    return t.to(torch.int32).contiguous()


def _norm_weights(dtype, *weights):
    """Weights of one type, contiguous and 16-byte aligned, and its code."""
    if all(w is None or w.dtype == dtype for w in weights):
        code = _DTYPE_CODE[dtype]
    else:  # (exact)
        weights = [None if w is None else w.to(torch.float32) for w in weights]
        code = _lib.SA_F32
    fixed = [w if w is None or (w.is_contiguous() and w.data_ptr() % 16 == 0)
             else w.clone(memory_format=torch.contiguous_format) for w in weights]
    return fixed, code


def _output_like(x):
    """A dense tensor in x's order of dims, if that keeps D innermost."""
    y = torch.empty_like(x)
    return y if y.stride(-1) == 1 else torch.empty(x.shape, dtype=x.dtype, device=x.device)


def _positions_arg(positions):
    """(pointer, batch stride) of positions [T] or [B, T] (None: row t)."""
    if positions is None:
        return None, 0
    return positions.data_ptr(), positions.stride(0) if positions.ndim == 2 else 0


def _qk_norm_rope_fwd(q, k, q_weight, k_weight, cos, sin, positions, eps):
    B, Hq, T, D = q.shape
    Hkv = k.shape[1]
    q, k = _flash_operand(q), _flash_operand(k)
    (qw, kw), w_code = _norm_weights(q.dtype, q_weight, k_weight)
    q_out, k_out = _output_like(q), _output_like(k)
    pos, pos_stride = _positions_arg(positions)
    with _device_of(q):
        st = _lib.load().sa_qk_norm_rope_fwd(
            q.data_ptr(), k.data_ptr(), q_out.data_ptr(), k_out.data_ptr(), _lib.ptr(qw), _lib.ptr(kw),
            cos.data_ptr(), sin.data_ptr(), pos, pos_stride, B, Hq, Hkv, T, D, cos.shape[0], _lib.strides(q),
            _lib.strides(k), _lib.strides(q_out), _lib.strides(k_out), float(eps), _DTYPE_CODE[q.dtype], w_code,
            _stream(q))
    _lib.check(st, "sa_qk_norm_rope_fwd")
    return q_out, k_out


def _qk_norm_rope_bwd(q, k, gq, gk, q_weight, k_weight, cos, sin, positions, eps, need_qw, need_kw):
    """(dq, dk, dq_weight, dk_weight); a weight gradient that is not needed is None."""
    _check_same_device("q", q, k=k, gq=gq, gk=gk, q_weight=q_weight, k_weight=k_weight, cos=cos, sin=sin,
                       positions=positions)
    B, Hq, T, D = q.shape
    Hkv = k.shape[1]
    # (saved-tensor hooks may hand back other types, sizes or layouts)
    _check_norm_args(("q", "k"), (q, k), (q_weight, k_weight), cos.detach(), sin.detach(), D)
    if (k.shape != (B, Hkv, T, D) or gq.shape != q.shape or gk.shape != k.shape or cos.shape[0] == 0 < B * T
            or (positions is not None and (positions.dtype != torch.int32 or positions.shape not in ((T,), (B, T))))):
        raise ValueError("the saved tensors of the norm must have the shapes and types that forward saved")
    q, k = _flash_operand(q), _flash_operand(k)
    dq, dk = _output_like(q), _output_like(k)
    dqw = torch.empty_like(q_weight) if need_qw else None
    dkw = torch.empty_like(k_weight) if need_kw else None
    if B * T == 0 or Hq + Hkv == 0:
        return dq, dk, dqw if dqw is None else dqw.zero_(), dkw if dkw is None else dkw.zero_()
    cos, sin = _rope_tables(cos, sin, T, D)
    if positions is not None:
        positions = positions.contiguous()
    gq, gk = _flash_operand(gq.to(q.dtype)), _flash_operand(gk.to(q.dtype))
    (qw, kw), w_code = _norm_weights(q.dtype, q_weight, k_weight)
    w_dtype = next((w.dtype for w in (qw, kw) if w is not None), q.dtype)
    outs = [None if w is None else torch.empty(D, dtype=w_dtype, device=q.device) for w in (dqw, dkw)]
    pos, pos_stride = _positions_arg(positions)
    lib = _lib.load()
    ws = None
    if need_qw or need_kw:
        ws = torch.empty(lib.sa_qk_norm_rope_bwd_workspace_size(B, Hq, Hkv, T, D), dtype=torch.uint8, device=q.device)
    with _device_of(q):
        st = lib.sa_qk_norm_rope_bwd(
            q.data_ptr(), k.data_ptr(), gq.data_ptr(), gk.data_ptr(), dq.data_ptr(), dk.data_ptr(),
            _lib.ptr(outs[0]), _lib.ptr(outs[1]), _lib.ptr(qw), _lib.ptr(kw), cos.data_ptr(), sin.data_ptr(), pos,
            pos_stride, B, Hq, Hkv, T, D, cos.shape[0], _lib.strides(q), _lib.strides(k), _lib.strides(gq),
            _lib.strides(gk), _lib.strides(dq), _lib.strides(dk), float(eps), _DTYPE_CODE[q.dtype], w_code,
            _lib.ptr(ws), 0 if ws is None else ws.numel(), _stream(q))
    _lib.check(st, "sa_qk_norm_rope_bwd")
    return (dq, dk, outs[0] if dqw is None else outs[0].to(dqw.dtype),
            outs[1] if dkw is None else outs[1].to(dkw.dtype))


class _QKNormRopeFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, q_weight, k_weight, cos, sin, positions, eps):
        ctx.save_for_backward(q, k, q_weight, k_weight, cos, sin, positions)
        ctx.eps = eps
        return _qk_norm_rope_fwd(q, k, q_weight, k_weight, cos, sin, positions, eps)

    @staticmethod
    @once_differentiable
    def backward(ctx, gq, gk):
        q, k, q_weight, k_weight, cos, sin, positions = ctx.saved_tensors
        need = ctx.needs_input_grad
        _native().check_capture(q)
        dq, dk, dqw, dkw = _qk_norm_rope_bwd(q, k, gq, gk, q_weight, k_weight, cos, sin, positions, ctx.eps,
                                             need[2], need[3])
        return dq if need[0] else None, dk if need[1] else None, dqw, dkw, None, None, None, None


def sp2norm_qk_norm_rope(q, k, q_weight, k_weight, cos, sin, *, positions=None, eps=1e-6):
    """RMS norm of the query and key rows of each head and rotate-half RoPE, one
    pass, with gradients of q, k and both weights.

    q: [B, Hq, T, D], k: [B, Hkv, T, D], bf16, fp16 or fp32, D a multiple of 16
    up to 512, at most 2^24 tokens and 16383 heads, any strides (those of a
    projection's [B, T, H, D] output are read and written as they lie).  q_weight,
    k_weight: [D] of q's dtype or fp32, or None for ones.  cos, sin: [n_pos, D/2]
    (precompute_rope_cos_sin); row t of the tables turns token t, or row
    positions[t] / positions[b, t] where an integer tensor [T] or [B, T] is given
    (clamped to the tables).

    ``z = x * rsqrt(mean(x^2) + eps) * weight``, then the pair (d, d + D/2) of z
    is turned by its angle; fp32 inside, rounded once.  Returns (q', k') for
    ``sp2norm_flash_attention``.

    Forward and backward can be captured in a HIP graph.  While an autograd graph
    or a hook made on the default stream holds the same leaves, or without the
    native call path, the captured backward raises RuntimeError; made on another
    stream they may live."""
    y = _native().qk_norm_rope(q, k, q_weight, k_weight, cos, sin, positions, eps)
    if y is not None:
        return y
    _check_tensors(q=q, k=k, q_weight=q_weight, k_weight=k_weight, cos=cos, sin=sin, positions=positions)
    if q.ndim != 4 or k.ndim != 4:
        raise ValueError("q and k must be [B, H, T, D] tensors")
    B, _, T, D = q.shape
    if k.shape[0] != B or k.shape[2] != T or k.shape[3] != D:
        raise ValueError(f"k must be [{B}, H_kv, {T}, {D}], got {tuple(k.shape)}")
    _check_norm_args(("q", "k"), (q, k), (q_weight, k_weight), cos, sin, D)
    if B * T > MAX_NORM_TOKENS:
        raise ValueError(f"the norm takes at most {MAX_NORM_TOKENS} tokens, got {B} x {T}")
    if positions is None:
        if cos.shape[0] < T:
            raise ValueError(f"cos and sin must have a row for each of the {T} tokens, got {cos.shape[0]}")
    else:
        if positions.shape != (T,) and positions.shape != (B, T):
            raise ValueError(f"positions must be [{T}] or [{B}, {T}], got {tuple(positions.shape)}")
        positions = _int32("positions", positions)
        if cos.shape[0] == 0 and B * T > 0:
            raise ValueError("cos and sin have no rows")
    _check_same_device("q", q, k=k, q_weight=q_weight, k_weight=k_weight, cos=cos, sin=sin, positions=positions)
    cos, sin = _rope_tables(cos.detach(), sin.detach(), T, D)
    return _QKNormRopeFn.apply(q, k, q_weight, k_weight, cos, sin, positions, eps)
