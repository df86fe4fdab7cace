"""Language-model operators around the routing points, as hand-written kernels.

The dense sublayers of the models whose routing this package runs
(:mod:`kotodama_amd.lmstep`; llama.py:155-192, 300-346) read and write each
query, key and embedding row several times when composed of torch ops.  Here
they are one pass each, differentiable, on the inputs' device and its current
stream, in bf16 or fp32 with fp32 statistics and sums:

* :func:`qk_norm_rope` — RMSNorm of every query and key head and the position
  rotation (``attnres_hip::qk_norm_rope`` / ``qk_norm_rope_bwd``);
* :func:`attention` — causal or full attention of grouped query heads, over
  ragged batches and over a cache (``attnres_hip::attention`` /
  ``attention_bwd``);
* :func:`embedding` — the scaled token lookup (``attnres_hip::embedding`` /
  ``embedding_bwd``).

Inputs may have any strides; one whose last dimension is not contiguous, or
whose rows the attention kernels cannot load in 16-byte pieces, is copied
first.  As everywhere in this package there is no CPU path: CPU tensors raise.
Gradients of gradients and forward-mode derivatives are not provided (the
latter raise :class:`NotImplementedError`).  Results repeat bit for bit: every
sum is taken in a fixed order (the embedding's sort counts tokens with atomics
in LDS, whole numbers whose order does not show).
"""

from __future__ import annotations

import ctypes
import math
import operator
from typing import Optional, Union

import torch
from torch import Tensor
from torch.autograd import forward_ad

from . import _capi
from ._native import native
from .ops import _DeviceStream, _eager_direct, _require_device, dtype_code

MAX_ATTENTION_DIM = 128
MAX_ROPE_DIM = 256
MAX_TOKEN_STRIDE = 32 << 20  # bytes from a token's row to the next that the attention kernels address


def _index_code(name: str, t: Tensor) -> int:
    if t.dtype == torch.int32:
        return _capi.INDEX_I32
    if t.dtype == torch.int64:
        return _capi.INDEX_I64
    raise TypeError(f"{name} must be int32 or int64, got {t.dtype}")


def _same_dtype(op: str, **tensors: Tensor) -> None:
    first = next(iter(tensors.values())).dtype
    dtype_code(first)
    for n, t in tensors.items():
        if t.dtype != first:
            raise TypeError(f"{op}: {n} is {t.dtype}, {next(iter(tensors))} is {first}")


def _check_like(op: str, name: str, t: Optional[Tensor], shape, dtype: Optional[torch.dtype] = None) -> None:
    """A gradient or saved result that the kernels read at the sizes of the inputs."""
    if t is None:
        return
    if t.shape != shape:
        raise ValueError(f"{op}: {name} must be {tuple(shape)}, got {tuple(t.shape)}")
    if dtype is not None and t.dtype != dtype:
        raise TypeError(f"{op}: {name} must be {dtype}, got {t.dtype}")


def _check_sizes(op: str, *tensors: Tensor) -> None:
    """The C calls take most sizes as 32-bit numbers."""
    for t in tensors:
        if max(t.shape, default=0) >= 1 << 31:
            raise ValueError(f"{op}: a size of {max(t.shape)} is over 2^31")


def _no_tangents(op: str, *tensors: Tensor) -> None:
    """Forward mode has no rule here: a tangent would be lost, as the ops see plain tensors."""
    if torch.compiler.is_compiling():
        return
    for t in tensors:
        if forward_ad.unpack_dual(t).tangent is not None:
            raise NotImplementedError(f"{op}: forward-mode differentiation is not provided")


_i64x3 = ctypes.c_int64 * 3


def _strides(t: Tensor):
    return _i64x3(t.stride(0), t.stride(1), t.stride(2))


def _rows(t: Tensor) -> Tensor:
    """``t`` with contiguous rows in its last dimension."""
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _table(t: Tensor) -> Tensor:
    """A 2-D ``t`` with contiguous rows that do not overlap."""
    t = _rows(t)
    return t.contiguous() if t.shape[0] > 1 and t.stride(0) < t.shape[1] else t


def _chunked(t: Tensor) -> Tensor:
    """``t`` with rows that load in 16-byte pieces."""
    m = 16 // t.element_size()
    if t.stride(-1) == 1 and t.data_ptr() % 16 == 0 and all(
            t.stride(i) % m == 0 for i in range(t.dim() - 1) if t.shape[i] > 1) and (
            t.shape[2] <= 1 or t.stride(2) * t.element_size() < MAX_TOKEN_STRIDE):
        return t
    # contiguous() leaves a contiguous tensor at its (unaligned) place
    return t.clone(memory_format=torch.contiguous_format)


def _heads_inside(t: Tensor, shape=None) -> Tensor:
    """An empty (B, H, T, D) tensor over (B, T, H, D) memory: what the projections read and write."""
    b, h, n, d = t.shape if shape is None else shape
    return torch.empty((b, n, h, d), device=t.device, dtype=t.dtype).transpose(1, 2)


def _ptr(t: Optional[Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


def _workspace(nbytes: int, device: torch.device) -> Tensor:
    return torch.empty(max(1, (nbytes + 3) // 4), device=device, dtype=torch.float32)


# ---------------------------------------------------------- qk_norm_rope --


def _check_qk(q: Tensor, k: Tensor, q_weight: Tensor, k_weight: Tensor, cos: Tensor, sin: Tensor,
              positions: Optional[Tensor]) -> None:
    if q.dim() != 4 or k.dim() != 4 or k.shape[0] != q.shape[0] or k.shape[2:] != q.shape[2:]:
        raise ValueError("qk_norm_rope: q and k must be (B, heads, T, D) with the same B, T and D, got "
                         f"{tuple(q.shape)} and {tuple(k.shape)}")
    b, _, t, d = q.shape
    if d % 2 or not 2 <= d <= MAX_ROPE_DIM:
        raise ValueError(f"qk_norm_rope: head size {d} is not even and at most {MAX_ROPE_DIM}")
    _same_dtype("qk_norm_rope", q=q, k=k, q_weight=q_weight, k_weight=k_weight)
    if q_weight.shape != (d,) or k_weight.shape != (d,):
        raise ValueError(f"qk_norm_rope: the weights must be ({d},)")
    if cos.dim() != 2 or cos.shape[1] != d or sin.shape != cos.shape:
        raise ValueError(f"qk_norm_rope: cos and sin must be (rows, {d}), got {tuple(cos.shape)} and {tuple(sin.shape)}")
    if cos.dtype not in (q.dtype, torch.float32) or sin.dtype != cos.dtype:
        raise TypeError(f"qk_norm_rope: cos and sin must both be {q.dtype} or float32, got {cos.dtype} and {sin.dtype}")
    if positions is None:
        if cos.shape[0] < t:
            raise ValueError(f"qk_norm_rope: {t} tokens but the tables have {cos.shape[0]} rows")
    else:
        _index_code("qk_norm_rope: positions", positions)
        if positions.shape not in ((t,), (b, t), (1, t)):
            raise ValueError(f"qk_norm_rope: positions must be ({t},) or ({b}, {t}), got {tuple(positions.shape)}")


def _qk_args(q, k, q_weight, k_weight, cos, sin, positions, eps) -> tuple:
    """The C call's arguments from the first weight to eps."""
    pos_b = pos_t = 0
    code = _capi.INDEX_I64
    if positions is not None:
        code = _index_code("positions", positions)
        pos_t = positions.stride(-1)
        if positions.dim() == 2 and positions.shape[0] > 1:
            pos_b = positions.stride(0)
    return (q_weight.data_ptr(), k_weight.data_ptr(), cos.data_ptr(), cos.stride(0), sin.data_ptr(), sin.stride(0),
            cos.shape[0], dtype_code(cos.dtype), _ptr(positions), code, pos_b, pos_t, float(eps))


def _qk_norm_rope_impl(q, k, q_weight, k_weight, cos, sin, positions, eps) -> tuple[Tensor, Tensor]:
    device = _require_device(q, k, q_weight, k_weight, cos, sin, positions)
    _check_qk(q, k, q_weight, k_weight, cos, sin, positions)
    _check_sizes("qk_norm_rope", q, k)
    q, k, cos, sin = _rows(q), _rows(k), _table(cos), _table(sin)
    q_weight, k_weight = q_weight.contiguous(), k_weight.contiguous()
    b, h, t, d = q.shape
    yq, yk = _heads_inside(q), _heads_inside(k)
    with _DeviceStream(device) as stream:
        _capi.qk_norm_rope_fwd(q.data_ptr(), _strides(q), k.data_ptr(), _strides(k), b, h, k.shape[1], t, d,
                               dtype_code(q.dtype), *_qk_args(q, k, q_weight, k_weight, cos, sin, positions, eps),
                               yq.data_ptr(), _strides(yq), yk.data_ptr(), _strides(yk), stream)
    return yq, yk


@torch.library.custom_op("attnres_hip::qk_norm_rope", mutates_args=())
def qk_norm_rope_op(q: Tensor, k: Tensor, q_weight: Tensor, k_weight: Tensor, cos: Tensor, sin: Tensor,
                    positions: Optional[Tensor], eps: float) -> tuple[Tensor, Tensor]:
    return _qk_norm_rope_impl(q, k, q_weight, k_weight, cos, sin, positions, eps)


@qk_norm_rope_op.register_fake
def _qk_norm_rope_fake(q, k, q_weight, k_weight, cos, sin, positions, eps):
    return _heads_inside(q), _heads_inside(k)


def _qk_norm_rope_bwd_impl(q, k, q_weight, k_weight, cos, sin, positions, eps, grad_q, grad_k):
    device = _require_device(q, k, q_weight, k_weight, cos, sin, positions, grad_q, grad_k)
    _check_qk(q, k, q_weight, k_weight, cos, sin, positions)
    _check_sizes("qk_norm_rope", q, k)
    _check_like("qk_norm_rope_bwd", "grad_q", grad_q, q.shape)
    _check_like("qk_norm_rope_bwd", "grad_k", grad_k, k.shape)
    q, k, cos, sin = _rows(q), _rows(k), _table(cos), _table(sin)
    q_weight, k_weight = q_weight.contiguous(), k_weight.contiguous()
    grad_q, grad_k = _rows(grad_q.to(q.dtype)), _rows(grad_k.to(k.dtype))
    b, h, t, d = q.shape
    dq, dk = _heads_inside(q), _heads_inside(k)
    dwq, dwk = torch.empty_like(q_weight), torch.empty_like(k_weight)
    with _DeviceStream(device) as stream:
        ws = _workspace(_capi.qk_norm_rope_workspace_size(d), device)
        _capi.qk_norm_rope_bwd(q.data_ptr(), _strides(q), k.data_ptr(), _strides(k), grad_q.data_ptr(),
                               _strides(grad_q), grad_k.data_ptr(), _strides(grad_k), b, h, k.shape[1], t, d,
                               dtype_code(q.dtype), *_qk_args(q, k, q_weight, k_weight, cos, sin, positions, eps),
                               dq.data_ptr(), _strides(dq), dk.data_ptr(), _strides(dk), dwq.data_ptr(),
                               dwk.data_ptr(), ws.data_ptr(), ws.numel() * 4, stream)
    return dq, dk, dwq, dwk


@torch.library.custom_op("attnres_hip::qk_norm_rope_bwd", mutates_args=())
def qk_norm_rope_bwd_op(q: Tensor, k: Tensor, q_weight: Tensor, k_weight: Tensor, cos: Tensor, sin: Tensor,
                        positions: Optional[Tensor], eps: float, grad_q: Tensor,
                        grad_k: Tensor) -> tuple[Tensor, Tensor, Tensor, Tensor]:
    """Gradients of q, k and the two weights."""
    return _qk_norm_rope_bwd_impl(q, k, q_weight, k_weight, cos, sin, positions, eps, grad_q, grad_k)


@qk_norm_rope_bwd_op.register_fake
def _qk_norm_rope_bwd_fake(q, k, q_weight, k_weight, cos, sin, positions, eps, grad_q, grad_k):
    return (_heads_inside(q), _heads_inside(k), torch.empty_like(q_weight, memory_format=torch.contiguous_format),
            torch.empty_like(k_weight, memory_format=torch.contiguous_format))


def _qk_setup_context(ctx, inputs, output):
    q, k, q_weight, k_weight, cos, sin, positions, eps = inputs
    ctx.save_for_backward(q, k, q_weight, k_weight, cos, sin, positions)
    ctx.eps = eps


def _qk_backward(ctx, grad_q, grad_k):
    q, k, q_weight, k_weight, cos, sin, positions = ctx.saved_tensors
    dq, dk, dwq, dwk = qk_norm_rope_bwd_op(q, k, q_weight, k_weight, cos, sin, positions, ctx.eps, grad_q, grad_k)
    return dq, dk, dwq, dwk, None, None, None, None


qk_norm_rope_op.register_autograd(_qk_backward, setup_context=_qk_setup_context)


def qk_norm_rope(q: Tensor, k: Tensor, q_weight: Tensor, k_weight: Tensor, cos: Tensor, sin: Tensor, eps: float,
                 positions: Optional[Tensor] = None) -> tuple[Tensor, Tensor]:
    """RMSNorm of every head of ``q`` (B, Hq, T, D) and ``k`` (B, Hk, T, D), then the rotation by position.

    ``n = x * rsqrt(mean(x^2) + eps) * weight`` (llama.py:143-153) and
    ``n * cos + rot(n) * sin`` with the halves rotated (llama.py:155-192), in
    fp32, rounded once.  ``cos`` and ``sin`` are full-width ``(rows, D)``
    tables in q's dtype or fp32.  Token t takes row t, or, with ``positions``
    ((T,) or (B, T) whole numbers on the device: the tokens of a decode step),
    row ``positions[..., t]``; one outside the tables makes the token's
    results NaN (positions stay on the device, so the host cannot refuse it).
    Returns tensors of q's and k's shapes over (B, T, H, D) memory.
    Differentiable in q, k and the weights; the tables have no gradient.
    """
    if not torch.compiler.is_compiling():
        res = native.qk_norm_rope(q, k, q_weight, k_weight, cos, sin, positions, eps)
        if res is not None:
            return res
    _no_tangents("qk_norm_rope", q, k, q_weight, k_weight, cos, sin)
    if torch.is_grad_enabled() and (cos.requires_grad or sin.requires_grad):
        raise NotImplementedError("qk_norm_rope: cos and sin have no gradient; detach them")
    if _eager_direct(q, k, q_weight, k_weight, cos, sin, positions):
        return _qk_norm_rope_impl(q, k, q_weight, k_weight, cos, sin, positions, eps)
    _require_device(q, k, q_weight, k_weight, cos, sin, positions)
    _check_qk(q, k, q_weight, k_weight, cos, sin, positions)
    return qk_norm_rope_op(q, k, q_weight, k_weight, cos, sin, positions, float(eps))


# ------------------------------------------------------------- attention --


def _check_attention(q: Tensor, k: Tensor, v: Tensor, kv_lens: Optional[Tensor], q_start: Optional[Tensor]) -> None:
    if q.dim() != 4 or k.dim() != 4 or v.shape != k.shape or k.shape[0] != q.shape[0] or k.shape[3] != q.shape[3]:
        raise ValueError("attention: q must be (B, heads, Tq, D), k and v (B, kv_heads, Tk, D), got "
                         f"{tuple(q.shape)}, {tuple(k.shape)} and {tuple(v.shape)}")
    b, h, _, d = q.shape
    if k.shape[1] == 0 or h == 0 or h % k.shape[1]:
        raise ValueError(f"attention: {h} query heads are not a multiple of {k.shape[1]} key heads")
    if d % 8 or not 8 <= d <= MAX_ATTENTION_DIM:
        raise ValueError(f"attention: head size {d} is not a multiple of 8 up to {MAX_ATTENTION_DIM}")
    _same_dtype("attention", q=q, k=k, v=v)
    for name, t in (("kv_lens", kv_lens), ("q_start", q_start)):
        if t is not None:
            _index_code(f"attention: {name}", t)
            if t.shape != (b,):
                raise ValueError(f"attention: {name} must be ({b},), got {tuple(t.shape)}")


def _attn_index(kv_lens: Optional[Tensor], q_start: Optional[Tensor]) -> tuple:
    """(kv_lens, q_start, their common index code), contiguous."""
    if kv_lens is not None and q_start is not None and kv_lens.dtype != q_start.dtype:
        kv_lens, q_start = kv_lens.long(), q_start.long()
    kv_lens = None if kv_lens is None else kv_lens.contiguous()
    q_start = None if q_start is None else q_start.contiguous()
    one = kv_lens if kv_lens is not None else q_start
    return kv_lens, q_start, _capi.INDEX_I32 if one is None else _index_code("attention", one)


def _attention_impl(q, k, v, causal, scale, kv_lens, q_start, q_start_value, want_lse=True):
    device = _require_device(q, k, v, kv_lens, q_start)
    _check_attention(q, k, v, kv_lens, q_start)
    _check_sizes("attention", q, k)
    q, k, v = _chunked(q), _chunked(k), _chunked(v)
    kv_lens, q_start, index = _attn_index(kv_lens, q_start)
    b, h, tq, d = q.shape
    hk, tk = k.shape[1], k.shape[2]
    out = _heads_inside(q)
    lse = torch.empty((b, h, tq), device=device, dtype=torch.float32) if want_lse else None
    code = dtype_code(q.dtype)
    with _DeviceStream(device) as stream:
        nbytes = _capi.attention_workspace_size(b, h, hk, tq, tk, d, code, 0)
        ws = _workspace(nbytes, device) if nbytes else None
        _capi.attention_fwd(q.data_ptr(), _strides(q), k.data_ptr(), _strides(k), v.data_ptr(), _strides(v), b, h, hk,
                            tq, tk, d, code, int(causal), float(scale), _ptr(kv_lens), _ptr(q_start), index,
                            q_start_value, out.data_ptr(), _strides(out), _ptr(lse), _ptr(ws), nbytes, stream)
    return out, lse


@torch.library.custom_op("attnres_hip::attention", mutates_args=())
def attention_op(q: Tensor, k: Tensor, v: Tensor, causal: bool, scale: float, kv_lens: Optional[Tensor],
                 q_start: Optional[Tensor], q_start_value: int) -> tuple[Tensor, Tensor]:
    """(out, lse); ``q_start_value`` counts where ``q_start`` is None (the smallest int64: from the end)."""
    return _attention_impl(q, k, v, causal, scale, kv_lens, q_start, q_start_value)


@attention_op.register_fake
def _attention_fake(q, k, v, causal, scale, kv_lens, q_start, q_start_value):
    return _heads_inside(q), q.new_empty(q.shape[:3], dtype=torch.float32)


def _attention_bwd_impl(q, k, v, out, lse, grad_out, grad_lse, causal, scale, kv_lens, q_start, q_start_value):
    device = _require_device(q, k, v, out, lse, grad_out, grad_lse, kv_lens, q_start)
    _check_attention(q, k, v, kv_lens, q_start)
    _check_sizes("attention", q, k)
    _check_like("attention_bwd", "out", out, q.shape, q.dtype)
    _check_like("attention_bwd", "lse", lse, q.shape[:3], torch.float32)
    _check_like("attention_bwd", "grad_out", grad_out, q.shape)
    _check_like("attention_bwd", "grad_lse", grad_lse, q.shape[:3])
    q, k, v, out, grad_out = _chunked(q), _chunked(k), _chunked(v), _chunked(out), _chunked(grad_out.to(q.dtype))
    lse = lse.contiguous()
    grad_lse = None if grad_lse is None else grad_lse.to(torch.float32).contiguous()
    kv_lens, q_start, index = _attn_index(kv_lens, q_start)
    b, h, tq, d = q.shape
    hk, tk = k.shape[1], k.shape[2]
    dq, dk, dv = _heads_inside(q), _heads_inside(k), _heads_inside(k)
    code = dtype_code(q.dtype)
    with _DeviceStream(device) as stream:
        nbytes = _capi.attention_workspace_size(b, h, hk, tq, tk, d, code, 1)
        ws = _workspace(nbytes, device)
        _capi.attention_bwd(q.data_ptr(), _strides(q), k.data_ptr(), _strides(k), v.data_ptr(), _strides(v),
                            out.data_ptr(), _strides(out), grad_out.data_ptr(), _strides(grad_out), lse.data_ptr(),
                            _ptr(grad_lse), b, h, hk, tq, tk, d, code, int(causal), float(scale), _ptr(kv_lens),
                            _ptr(q_start), index, q_start_value, dq.data_ptr(), _strides(dq), dk.data_ptr(),
                            _strides(dk), dv.data_ptr(), _strides(dv), ws.data_ptr(), ws.numel() * 4, stream)
    return dq, dk, dv


@torch.library.custom_op("attnres_hip::attention_bwd", mutates_args=())
def attention_bwd_op(q: Tensor, k: Tensor, v: Tensor, out: Tensor, lse: Tensor, grad_out: Tensor,
                     grad_lse: Optional[Tensor], causal: bool, scale: float, kv_lens: Optional[Tensor],
                     q_start: Optional[Tensor], q_start_value: int) -> tuple[Tensor, Tensor, Tensor]:
    """Gradients of q, k and v."""
    return _attention_bwd_impl(q, k, v, out, lse, grad_out, grad_lse, causal, scale, kv_lens, q_start, q_start_value)


@attention_bwd_op.register_fake
def _attention_bwd_fake(q, k, v, out, lse, grad_out, grad_lse, causal, scale, kv_lens, q_start, q_start_value):
    return _heads_inside(q), _heads_inside(k), _heads_inside(k)


def _attention_setup_context(ctx, inputs, output):
    q, k, v, causal, scale, kv_lens, q_start, q_start_value = inputs
    out, lse = output
    ctx.set_materialize_grads(False)
    ctx.save_for_backward(q, k, v, out, lse, kv_lens, q_start)
    ctx.args = (causal, scale, q_start_value)


def _attention_backward(ctx, grad_out, grad_lse):
    if grad_out is None and grad_lse is None:
        return (None,) * 8
    q, k, v, out, lse, kv_lens, q_start = ctx.saved_tensors
    causal, scale, q_start_value = ctx.args
    if grad_out is None:
        grad_out = torch.zeros_like(out)
    dq, dk, dv = attention_bwd_op(q, k, v, out, lse, grad_out, grad_lse, causal, scale, kv_lens, q_start,
                                  q_start_value)
    return dq, dk, dv, None, None, None, None, None


attention_op.register_autograd(_attention_backward, setup_context=_attention_setup_context)


def attention(q: Tensor, k: Tensor, v: Tensor, *, causal: bool = True, scale: Optional[float] = None,
              kv_lens: Optional[Tensor] = None, q_start: Union[None, int, Tensor] = None, want_lse: bool = False):
    """softmax(scale q k^T) v for ``q`` (B, H, Tq, D) over ``k`` and ``v`` (B, Hk, Tk, D), H a multiple of Hk.

    Query head h reads key head ``h // (H // Hk)``.  ``scale`` (positive) is
    1/sqrt(D) unless given.  ``kv_lens`` ((B,) whole numbers on the device) is how many
    keys of each sequence exist, Tk unless given: a cache's fill, a padded
    batch's lengths.  What the other slots hold, NaN included, is not used.
    Query i is at position ``q_start + i`` of its sequence, ``q_start`` a
    number or a (B,) tensor on the device; by default the last query is at the
    last key (``kv_lens - Tq``: new tokens behind a cache, or whole sequences
    of Tq = Tk).  A padded batch of whole sequences passes ``q_start=0``.

    With ``causal`` a query sees the keys up to its own position, and a query
    whose position lies outside its sequence (padding) sees none.  A row that
    sees no key is zero with lse -inf, and gives and gets no gradient.

    Returns the (B, H, Tq, D) result over (B, Tq, H, D) memory, and with
    ``want_lse`` also the fp32 log-sum-exp of each row's scores (B, H, Tq).
    Differentiable in q, k and v, through both results.  Scores, probabilities,
    sums and statistics are fp32; with bf16 inputs the probabilities and the
    score gradients are rounded to bf16 for the products with v, k, q and the
    output's gradient, and the backward reads the rounded output.  fp32 inputs
    round none of them.  D is a multiple of 8
    up to 128.  A NaN or infinity in a key or value that exists may reach
    every query of its sequence.
    """
    causal = bool(causal)
    scale = 1.0 / math.sqrt(max(1, q.shape[-1])) if scale is None else float(scale)
    if not 0.0 < scale < math.inf:
        raise ValueError(f"attention: scale must be positive and finite, got {scale}")
    if kv_lens is not None and not isinstance(kv_lens, Tensor):
        raise TypeError(f"attention: kv_lens must be a tensor, got {type(kv_lens).__name__}")
    start, value = None, _capi.START_FROM_END
    if isinstance(q_start, Tensor):
        start = q_start
    elif q_start is not None:
        value = operator.index(q_start)
        if abs(value) > 1 << 40:
            raise ValueError(f"attention: q_start {value} is out of range")
    if not torch.compiler.is_compiling():
        res = native.attention(q, k, v, causal, scale, kv_lens, start, value, bool(want_lse))
        if res is not None:
            return res
    _no_tangents("attention", q, k, v)
    if _eager_direct(q, k, v, kv_lens, start):
        out, lse = _attention_impl(q, k, v, causal, scale, kv_lens, start, value, want_lse)
    else:
        _require_device(q, k, v, kv_lens, start)
        _check_attention(q, k, v, kv_lens, start)
        out, lse = attention_op(q, k, v, causal, scale, kv_lens, start, value)
    return (out, lse) if want_lse else out


# ------------------------------------------------------------- embedding --


def _check_embedding(ids: Tensor, weight: Tensor, padding_idx: int) -> None:
    _index_code("embedding: ids", ids)
    if weight.dim() != 2 or weight.shape[1] == 0:
        raise ValueError(f"embedding: weight must be (rows, hidden), got {tuple(weight.shape)}")
    dtype_code(weight.dtype)
    if not -1 <= padding_idx < max(1, weight.shape[0]):
        raise ValueError(f"embedding: padding_idx {padding_idx} is not a row of the table")


def _embedding_impl(ids, weight, scale, padding_idx) -> Tensor:
    device = _require_device(ids, weight)
    _check_embedding(ids, weight, padding_idx)
    _check_sizes("embedding", weight)
    weight, flat = _table(weight), ids.contiguous()
    out = torch.empty((*ids.shape, weight.shape[1]), device=device, dtype=weight.dtype)
    with _DeviceStream(device) as stream:
        _capi.embedding_fwd(flat.data_ptr(), _index_code("ids", ids), flat.numel(), weight.data_ptr(),
                            weight.stride(0), weight.shape[0], weight.shape[1], dtype_code(weight.dtype),
                            float(scale), out.data_ptr(), stream)
    return out


@torch.library.custom_op("attnres_hip::embedding", mutates_args=())
def embedding_op(ids: Tensor, weight: Tensor, scale: float, padding_idx: int) -> Tensor:
    return _embedding_impl(ids, weight, scale, padding_idx)


@embedding_op.register_fake
def _embedding_fake(ids, weight, scale, padding_idx):
    return weight.new_empty((*ids.shape, weight.shape[1]))


def _embedding_bwd_impl(ids, grad_out, rows, scale, padding_idx) -> Tensor:
    device = _require_device(ids, grad_out)
    _index_code("embedding_bwd: ids", ids)
    dtype_code(grad_out.dtype)
    if grad_out.dim() == 0 or grad_out.shape[:-1] != ids.shape or grad_out.shape[-1] == 0:
        raise ValueError(f"embedding_bwd: grad_out must be ({', '.join(map(str, ids.shape))}, hidden), "
                         f"got {tuple(grad_out.shape)}")
    if rows < 0 or not -1 <= padding_idx < max(1, rows):
        raise ValueError(f"embedding_bwd: bad rows {rows} or padding_idx {padding_idx}")
    _check_sizes("embedding", grad_out)
    hidden = grad_out.shape[-1]
    flat = ids.contiguous()
    g = _table(grad_out.reshape(-1, hidden))
    dw = torch.empty((rows, hidden), device=device, dtype=g.dtype)
    with _DeviceStream(device) as stream:
        ws = _workspace(_capi.embedding_workspace_size(flat.numel(), rows, hidden), device)
        _capi.embedding_bwd(flat.data_ptr(), _index_code("ids", ids), flat.numel(), g.data_ptr(), g.stride(0), rows,
                            hidden, dtype_code(g.dtype), float(scale), padding_idx, dw.data_ptr(), ws.data_ptr(),
                            ws.numel() * 4, stream)
    return dw


@torch.library.custom_op("attnres_hip::embedding_bwd", mutates_args=())
def embedding_bwd_op(ids: Tensor, grad_out: Tensor, rows: int, scale: float, padding_idx: int) -> Tensor:
    """The gradient of the (rows, hidden) table, in grad_out's dtype."""
    return _embedding_bwd_impl(ids, grad_out, rows, scale, padding_idx)


@embedding_bwd_op.register_fake
def _embedding_bwd_fake(ids, grad_out, rows, scale, padding_idx):
    return grad_out.new_empty((rows, grad_out.shape[-1]))


def _embedding_setup_context(ctx, inputs, output):
    ids, weight, scale, padding_idx = inputs
    ctx.save_for_backward(ids)
    ctx.args = (weight.shape[0], scale, padding_idx, weight.dtype)


def _embedding_backward(ctx, grad_out):
    (ids,) = ctx.saved_tensors
    rows, scale, padding_idx, dtype = ctx.args
    return None, embedding_bwd_op(ids, grad_out.to(dtype), rows, scale, padding_idx), None, None


embedding_op.register_autograd(_embedding_backward, setup_context=_embedding_setup_context)


def embedding(ids: Tensor, weight: Tensor, scale: float = 1.0, padding_idx: Optional[int] = None) -> Tensor:
    """``scale * weight[ids]`` for whole numbers ``ids`` of any shape and a (rows, hidden) table.

    The table's gradient is dense: the tokens are sorted by row, stably, and
    each row's gradients added in that order in fp32, so it repeats bit for
    bit whatever the batch.  Tokens equal to ``padding_idx`` (a negative one
    counts from the end) give no gradient.  An id outside the table gives a
    row of NaN and no gradient (ids stay on the device, so the host cannot
    refuse it).
    """
    pad = -1
    if padding_idx is not None:
        pad = operator.index(padding_idx)
        rows = weight.shape[0] if weight.dim() == 2 else 0
        if not -rows <= pad < rows:
            raise ValueError(f"embedding: padding_idx {pad} is not a row of the table")
        pad %= rows
    if not torch.compiler.is_compiling():
        out = native.embedding(ids, weight, scale, pad)
        if out is not None:
            return out
    _no_tangents("embedding", weight)
    if _eager_direct(ids, weight):
        return _embedding_impl(ids, weight, scale, pad)
    _require_device(ids, weight)
    _check_embedding(ids, weight, pad)
    return embedding_op(ids, weight, float(scale), pad)


__all__ = ["attention", "embedding", "qk_norm_rope"]
