"""Serving from a paged cache, as hand-written kernels.

The reference's KV-cache engine (llama.py:718-763) concatenates every layer's
keys and values anew for each token.  Here they lie in pages that sequences
take as they grow, and one call serves prompts in chunks, single tokens and
drafted ones of many sequences together:

* :func:`paged_slots` / :func:`paged_release` — block tables, slot maps and the
  free list, from the requests' lengths (``attnres_hip::paged_slots`` /
  ``paged_release``);
* :func:`paged_write` — new keys and values into their slots
  (``attnres_hip::paged_write``);
* :func:`paged_attention` — attention of the new tokens over the pages
  (``attnres_hip::paged_attention``);
* :func:`verify_drafts` — drafted tokens against the model's logits, and the
  token behind the last that stays (``attnres_hip::verify_drafts``).

:class:`PagedCache` keeps what a model needs of it, and
:meth:`kotodama_amd.lmstep.LanguageModel.logits_paged` / ``step_paged`` run on it.

Lengths, tables and slots are whole numbers on the device and stay there: no
call waits for the GPU, and all can be captured into a graph.  The host cannot refuse what they hold,
so the kernels take lengths into what the tensors have and read or write
nothing outside them.  As everywhere in this package there is no CPU path: CPU
tensors raise.  These are inference operators: a call that autograd would record, or
with a forward-mode tangent, raises :class:`NotImplementedError`.  Results
repeat bit for bit.
"""

from __future__ import annotations

import ctypes
import math
import operator
from typing import NamedTuple, Optional

import torch
from torch import Tensor
from torch.autograd.graph import increment_version

from . import _capi
from ._native import native
from .lmops import (MAX_ATTENTION_DIM, _check_sizes, _index_code, _no_tangents, _ptr, _rows, _same_dtype, _table,
                    _workspace)
from .ops import _DeviceStream, _eager_direct, _require_device, dtype_code

MIN_PAGE = 16  # rows
MAX_PAGE = 1 << 16
MAX_VOCAB = 1 << 21  # of verify_drafts

_i64x2 = ctypes.c_int64 * 2
_i64x3 = ctypes.c_int64 * 3


def _no_grad(op: str, *tensors: Optional[Tensor]) -> None:
    some = [t for t in tensors if t is not None]
    _no_tangents(op, *(t for t in some if t.is_floating_point()))
    if torch.is_grad_enabled() and any(t.requires_grad for t in some):
        raise NotImplementedError(f"{op}: no gradient is provided; detach the inputs or call it under torch.no_grad()")


def _check_page(op: str, page_size: int) -> int:
    page = operator.index(page_size)
    if not MIN_PAGE <= page <= MAX_PAGE or page & (page - 1):
        raise ValueError(f"{op}: page size {page} is not a power of two from {MIN_PAGE} to {MAX_PAGE}")
    return page


def _check_lengths(op: str, name: str, t: Tensor, n: int) -> None:
    _index_code(f"{op}: {name}", t)
    if t.shape != (n,):
        raise ValueError(f"{op}: {name} must be ({n},), got {tuple(t.shape)}")


def _check_int32(op: str, name: str, t: Tensor) -> None:
    if t.dtype != torch.int32:
        raise TypeError(f"{op}: {name} must be int32, got {t.dtype}")


def _aligned(t: Tensor) -> bool:
    """Rows that load in 16-byte pieces."""
    m = 16 // t.element_size()
    return (t.stride(-1) == 1 or t.shape[-1] == 1) and t.data_ptr() % 16 == 0 and all(
        t.stride(i) % m == 0 and t.stride(i) >= 0 for i in range(t.dim() - 1) if t.shape[i] > 1)


def _pieces(t: Tensor) -> Tensor:
    return t if _aligned(t) else t.clone(memory_format=torch.contiguous_format)


# ----------------------------------------------------------------- slots --


class PagedSlots(NamedTuple):
    """What :func:`paged_slots` gives, int32 on the device."""

    slots: Tensor  #: (num_tokens,) ``page * page_size + row`` of each new token; -1 for padding and refused sequences
    positions: Tensor  #: (num_tokens,) its place in its sequence; 0 for padding
    q_starts: Tensor  #: (B + 1,) where each sequence's new tokens begin
    kv_lens: Tensor  #: (B,) tokens held with the new ones; 0 for a refused sequence
    free_count: Tensor  #: (1,) pages that stay free


def _check_slots(op: str, block_table: Tensor, held: Tensor, change_name: str, change: Tensor, free_pages: Tensor,
                 free_count: Tensor, page_size: int) -> None:
    if block_table.dim() != 2:
        raise ValueError(f"{op}: block_table must be (sequences, pages), got {tuple(block_table.shape)}")
    b, m = block_table.shape
    for name, t in (("block_table", block_table), ("free_pages", free_pages), ("free_count", free_count)):
        _check_int32(op, name, t)
    if (m > 1 and block_table.stride(1) != 1) or (b > 1 and block_table.stride(0) < m):
        raise ValueError(f"{op}: block_table's rows must be contiguous and apart, got strides {block_table.stride()}")
    _check_lengths(op, "held", held, b)
    _check_lengths(op, change_name, change, b)
    if free_pages.dim() != 1 or not free_pages.is_contiguous():
        raise ValueError(f"{op}: free_pages must be one contiguous dimension, got {tuple(free_pages.shape)}")
    if free_count.numel() != 1:
        raise ValueError(f"{op}: free_count must have one element, got {tuple(free_count.shape)}")
    if m * _check_page(op, page_size) > 1 << 30:
        raise ValueError(f"{op}: a row of the table is over 2^30 tokens")
    _check_sizes(op, block_table, free_pages)


def _lengths(t: Tensor) -> tuple[Tensor, int]:
    return t.contiguous(), _index_code("lengths", t)


def _paged_slots_impl(block_table, held, new, free_pages, free_count, page_size, num_tokens) -> tuple:
    device = _require_device(block_table, held, new, free_pages, free_count)
    _check_slots("paged_slots", block_table, held, "new", new, free_pages, free_count, page_size)
    b, m = block_table.shape
    held, held_code = _lengths(held)
    new, new_code = _lengths(new)
    slots, positions, q_starts, kv_lens, count = _paged_slots_fake(block_table, held, new, free_pages, free_count,
                                                                   page_size, num_tokens)
    with _DeviceStream(device) as stream:
        _capi.paged_slots(block_table.data_ptr(), block_table.stride(0), b, m, held.data_ptr(), held_code,
                          new.data_ptr(), new_code, free_pages.data_ptr(), free_pages.shape[0], free_count.data_ptr(),
                          page_size, num_tokens, slots.data_ptr(), positions.data_ptr(), q_starts.data_ptr(),
                          kv_lens.data_ptr(), count.data_ptr(), stream)
    return slots, positions, q_starts, kv_lens, count


@torch.library.custom_op("attnres_hip::paged_slots", mutates_args=("block_table",))
def paged_slots_op(block_table: Tensor, held: Tensor, new: Tensor, free_pages: Tensor, free_count: Tensor,
                   page_size: int, num_tokens: int) -> tuple[Tensor, Tensor, Tensor, Tensor, Tensor]:
    return _paged_slots_impl(block_table, held, new, free_pages, free_count, page_size, num_tokens)


@paged_slots_op.register_fake
def _paged_slots_fake(block_table, held, new, free_pages, free_count, page_size, num_tokens):
    b = block_table.shape[0]
    return tuple(block_table.new_empty((n,), dtype=torch.int32) for n in (num_tokens, num_tokens, b + 1, b, 1))


def paged_slots(block_table: Tensor, held: Tensor, new: Tensor, free_pages: Tensor, free_count: Tensor, page_size: int,
                num_tokens: int) -> PagedSlots:
    """Pages and slots for new tokens: sequence b holds ``held[b]`` tokens and adds ``new[b]``.

    ``block_table`` (B, M) int32 names each sequence's pages in order; the
    pages that sequences need on top of the ``ceil(held / page_size)`` they have are
    written into it.  They come from the end of ``free_pages[:free_count]``, in the
    sequences' order: a sequence gets all it needs where the needs of the
    sequences up to it are at most ``free_count`` pages, and is refused
    otherwise, as is one whose tokens do not fit its row of the table, or end behind the
    ``num_tokens`` of the packed batch (as all behind it do), or whose lengths are
    negative or over 2^30.  ``num_tokens`` (a number on the host) may be more than the sum of ``new``: the rows behind
    are padding.  ``held`` and ``new`` are (B,) whole numbers on the device,
    ``page_size`` a power of two from 16 to 65536.

    ``free_pages`` and ``free_count`` stay as they are: the count that is left comes
    back in the result, and the same call again gives the same.
    """
    num_tokens = operator.index(num_tokens)
    if not 0 <= num_tokens <= 1 << 30:
        raise ValueError(f"paged_slots: num_tokens {num_tokens} is not from 0 to 2^30")
    if not torch.compiler.is_compiling():
        res = native.paged_slots(block_table, held, new, free_pages, free_count, page_size, num_tokens)
        if res is not None:
            return PagedSlots(*res)
    page_size = _check_page("paged_slots", page_size)
    if _eager_direct(block_table, held, new, free_pages, free_count):
        res = _paged_slots_impl(block_table, held, new, free_pages, free_count, page_size, num_tokens)
        increment_version(block_table)
        return PagedSlots(*res)
    _require_device(block_table, held, new, free_pages, free_count)
    _check_slots("paged_slots", block_table, held, "new", new, free_pages, free_count, page_size)
    return PagedSlots(*paged_slots_op(block_table, held, new, free_pages, free_count, page_size, num_tokens))


def _paged_release_impl(block_table, held, kept, free_pages, free_count, page_size) -> Tensor:
    device = _require_device(block_table, held, kept, free_pages, free_count)
    _check_slots("paged_release", block_table, held, "kept", kept, free_pages, free_count, page_size)
    b, m = block_table.shape
    held, held_code = _lengths(held)
    kept, kept_code = _lengths(kept)
    count = free_count.new_empty((1,))
    with _DeviceStream(device) as stream:
        _capi.paged_release(block_table.data_ptr(), block_table.stride(0), b, m, held.data_ptr(), held_code,
                            kept.data_ptr(), kept_code, free_pages.data_ptr(), free_pages.shape[0],
                            free_count.data_ptr(), page_size, count.data_ptr(), stream)
    return count


@torch.library.custom_op("attnres_hip::paged_release", mutates_args=("free_pages",))
def paged_release_op(block_table: Tensor, held: Tensor, kept: Tensor, free_pages: Tensor, free_count: Tensor,
                     page_size: int) -> Tensor:
    return _paged_release_impl(block_table, held, kept, free_pages, free_count, page_size)


@paged_release_op.register_fake
def _paged_release_fake(block_table, held, kept, free_pages, free_count, page_size):
    return free_count.new_empty((1,))


def paged_release(block_table: Tensor, held: Tensor, kept: Tensor, free_pages: Tensor, free_count: Tensor,
                  page_size: int) -> Tensor:
    """Gives back pages: sequence b, which holds ``held[b]`` tokens, keeps the first ``kept[b]`` (0: it ends).

    The pages behind those are written into ``free_pages`` from
    ``free_count`` on, sequence by sequence, a sequence's last page first (so
    that the next to be taken is the one that continues it).  Returns the new
    count, (1,) int32; ``free_count`` stays as it is.  ``kept`` is taken into
    [0, held].  The table keeps the pages' numbers, which then mean nothing.
    """
    if not torch.compiler.is_compiling():
        res = native.paged_release(block_table, held, kept, free_pages, free_count, page_size)
        if res is not None:
            return res
    page_size = _check_page("paged_release", page_size)
    if _eager_direct(block_table, held, kept, free_pages, free_count):
        res = _paged_release_impl(block_table, held, kept, free_pages, free_count, page_size)
        increment_version(free_pages)
        return res
    _require_device(block_table, held, kept, free_pages, free_count)
    _check_slots("paged_release", block_table, held, "kept", kept, free_pages, free_count, page_size)
    return paged_release_op(block_table, held, kept, free_pages, free_count, page_size)


# ----------------------------------------------------------------- write --


def _check_cache(op: str, k_cache: Tensor, v_cache: Tensor) -> None:
    if k_cache.dim() != 4 or v_cache.shape != k_cache.shape:
        raise ValueError(f"{op}: k_cache and v_cache must be (pages, kv_heads, page_size, D), got "
                         f"{tuple(k_cache.shape)} and {tuple(v_cache.shape)}")
    _, hk, page, d = k_cache.shape
    if hk == 0:
        raise ValueError(f"{op}: the cache has no heads")
    if d % 8 or not 8 <= d <= MAX_ATTENTION_DIM:
        raise ValueError(f"{op}: head size {d} is not a multiple of 8 up to {MAX_ATTENTION_DIM}")
    _check_page(op, page)
    _same_dtype(op, k_cache=k_cache, v_cache=v_cache)
    _check_sizes(op, k_cache)


def _rows_apart(t: Tensor) -> bool:
    """Strides that each lead past all that the smaller ones reach: no two elements lie on one another."""
    reach = 0
    for stride, size in sorted((st, n) for st, n in zip(t.stride(), t.shape) if n > 1):
        if stride <= reach:
            return False
        reach += stride * (size - 1)
    return True


def _check_cache_memory(op: str, k_cache: Tensor, v_cache: Tensor, written: bool = False) -> None:
    # a cache is written in place and read by its pages: not copied
    for name, t in (("k_cache", k_cache), ("v_cache", v_cache)):
        if t.numel() and not _aligned(t):
            raise ValueError(f"{op}: {name} must lie in 16-byte pieces, got strides {t.stride()}")
        apart = t.stride(0) if t.shape[0] > 1 else 0
        if t.numel() and max(t.stride(2) * t.shape[2], apart) * t.element_size() >= 1 << 31:
            raise ValueError(f"{op}: {name}: a head's rows of a page span 2^31 bytes, or its pages lie so far apart")
        if written and t.numel() and not _rows_apart(t):
            raise ValueError(f"{op}: rows of {name} lie on one another, got strides {t.stride()}")


def _check_write(k: Tensor, v: Tensor, k_cache: Tensor, v_cache: Tensor, slots: Tensor) -> None:
    _check_cache("paged_write", k_cache, v_cache)
    _same_dtype("paged_write", k_cache=k_cache, k=k, v=v)
    if k.dim() != 3 or v.shape != k.shape or k.shape[1:] != (k_cache.shape[1], k_cache.shape[3]):
        raise ValueError(f"paged_write: k and v must be (N, {k_cache.shape[1]}, {k_cache.shape[3]}), got "
                         f"{tuple(k.shape)} and {tuple(v.shape)}")
    _check_lengths("paged_write", "slots", slots, k.shape[0])
    _check_sizes("paged_write", k)


def _cache_strides(t: Tensor):
    return _i64x3(t.stride(0), t.stride(1), t.stride(2))


def _paged_write_impl(k, v, k_cache, v_cache, slots) -> None:
    device = _require_device(k, v, k_cache, v_cache, slots)
    _check_write(k, v, k_cache, v_cache, slots)
    _check_cache_memory("paged_write", k_cache, v_cache, written=True)
    k, v = _pieces(k), _pieces(v)
    slots, code = _lengths(slots)
    n, hk, d = k.shape
    with _DeviceStream(device) as stream:
        _capi.paged_write(k.data_ptr(), _i64x2(k.stride(0), k.stride(1)), v.data_ptr(),
                          _i64x2(v.stride(0), v.stride(1)), n, hk, d, dtype_code(k.dtype), k_cache.data_ptr(),
                          _cache_strides(k_cache), v_cache.data_ptr(), _cache_strides(v_cache), k_cache.shape[0],
                          k_cache.shape[2], slots.data_ptr(), code, stream)


@torch.library.custom_op("attnres_hip::paged_write", mutates_args=("k_cache", "v_cache"))
def paged_write_op(k: Tensor, v: Tensor, k_cache: Tensor, v_cache: Tensor, slots: Tensor) -> None:
    _paged_write_impl(k, v, k_cache, v_cache, slots)


@paged_write_op.register_fake
def _paged_write_fake(k, v, k_cache, v_cache, slots):
    return None


def paged_write(k: Tensor, v: Tensor, k_cache: Tensor, v_cache: Tensor, slots: Tensor) -> None:
    """Writes keys and values ``k`` and ``v`` (N, Hk, D) into rows ``slots`` of the caches (pages, Hk, page_size, D).

    ``slots`` ((N,) whole numbers on the device, as :func:`paged_slots` gives
    them) are ``page * page_size + row``; one outside the cache (-1: padding,
    a refused sequence) is skipped.  No slot may be named twice: which of its
    tokens a row then holds, and whether whole, is not said.  ``k`` and ``v``
    may have any strides, the caches any whose rows lie in 16-byte pieces and that each lead past all that
    the smaller ones reach: rows that lie on one another, as in an overlapping view, are refused.  The
    host does not see it where ``k_cache`` and ``v_cache`` share rows, or a cache shares memory
    with ``k`` or ``v``: what stands there afterwards is not said either.
    """
    if not torch.compiler.is_compiling() and native.paged_write(k, v, k_cache, v_cache, slots):
        return
    _no_grad("paged_write", k, v, k_cache, v_cache)
    if _eager_direct(k, v, k_cache, v_cache, slots):
        _paged_write_impl(k, v, k_cache, v_cache, slots)
        increment_version((k_cache, v_cache))
        return
    _require_device(k, v, k_cache, v_cache, slots)
    _check_write(k, v, k_cache, v_cache, slots)
    paged_write_op(k, v, k_cache, v_cache, slots)


# ------------------------------------------------------------- attention --


def _check_paged_attention(q: Tensor, k_cache: Tensor, v_cache: Tensor, block_table: Tensor, kv_lens: Tensor,
                           q_starts: Optional[Tensor]) -> None:
    op = "paged_attention"
    _check_cache(op, k_cache, v_cache)
    _same_dtype(op, q=q, k_cache=k_cache)
    hk, page, d = k_cache.shape[1:]
    if q.dim() != 3 or q.shape[2] != d:
        raise ValueError(f"{op}: q must be (N, heads, {d}), got {tuple(q.shape)}")
    if q.shape[1] == 0 or q.shape[1] % hk:
        raise ValueError(f"{op}: {q.shape[1]} query heads are not a multiple of {hk} key heads")
    _check_int32(op, "block_table", block_table)
    if block_table.dim() != 2:
        raise ValueError(f"{op}: block_table must be (sequences, pages), got {tuple(block_table.shape)}")
    b, m = block_table.shape
    if m * page > 1 << 30:
        raise ValueError(f"{op}: a row of the table is over 2^30 tokens")
    _check_lengths(op, "kv_lens", kv_lens, b)
    if q_starts is not None:
        _check_lengths(op, "q_starts", q_starts, b + 1)
    elif q.shape[0] != b:
        raise ValueError(f"{op}: without q_starts every sequence has one new token, got {q.shape[0]} for {b}")
    _check_sizes(op, q, block_table)


def _paged_attention_impl(q, k_cache, v_cache, block_table, kv_lens, q_starts, scale, want_lse=True):
    device = _require_device(q, k_cache, v_cache, block_table, kv_lens, q_starts)
    _check_paged_attention(q, k_cache, v_cache, block_table, kv_lens, q_starts)
    _check_cache_memory("paged_attention", k_cache, v_cache)
    q, block_table = _pieces(q), _table(block_table)
    kv_lens, lens_code = _lengths(kv_lens)
    starts_code = _capi.INDEX_I32
    if q_starts is not None:
        q_starts, starts_code = _lengths(q_starts)
    n, h, d = q.shape
    pages, hk, page, _ = k_cache.shape
    b, m = block_table.shape
    out = torch.empty((n, h, d), device=device, dtype=q.dtype)
    lse = torch.empty((n, h), device=device, dtype=torch.float32) if want_lse else None
    code = dtype_code(q.dtype)
    with _DeviceStream(device) as stream:
        nbytes = _capi.paged_attention_workspace_size(n, b, h, hk, d, code, m, page)
        ws = _workspace(nbytes, device) if nbytes else None
        _capi.paged_attention_fwd(q.data_ptr(), _i64x2(q.stride(0), q.stride(1)), k_cache.data_ptr(),
                                  _cache_strides(k_cache), v_cache.data_ptr(), _cache_strides(v_cache), n, b, h, hk, d,
                                  code, pages, page, block_table.data_ptr(), block_table.stride(0), m,
                                  kv_lens.data_ptr(), lens_code, _ptr(q_starts), starts_code, float(scale),
                                  out.data_ptr(), _i64x2(h * d, d), _ptr(lse), _ptr(ws), nbytes, stream)
    return out, lse


@torch.library.custom_op("attnres_hip::paged_attention", mutates_args=())
def paged_attention_op(q: Tensor, k_cache: Tensor, v_cache: Tensor, block_table: Tensor, kv_lens: Tensor,
                       q_starts: Optional[Tensor], scale: float) -> tuple[Tensor, Tensor]:
    """(out, lse)"""
    return _paged_attention_impl(q, k_cache, v_cache, block_table, kv_lens, q_starts, scale)


@paged_attention_op.register_fake
def _paged_attention_fake(q, k_cache, v_cache, block_table, kv_lens, q_starts, scale):
    return q.new_empty(q.shape), q.new_empty(q.shape[:2], dtype=torch.float32)


def paged_attention(q: Tensor, k_cache: Tensor, v_cache: Tensor, block_table: Tensor, kv_lens: Tensor,
                    q_starts: Optional[Tensor] = None, *, scale: Optional[float] = None, want_lse: bool = False):
    """Causal attention of packed new tokens ``q`` (N, H, D) over their sequences' pages.

    ``k_cache`` and ``v_cache`` (pages, Hk, page_size, D) hold the keys and
    values, the new tokens' own among them; H is a multiple of Hk, and query
    head h reads key head ``h // (H // Hk)``.  Key t of sequence b is row
    ``t % page_size`` of page ``block_table[b, t // page_size]`` ((B, M)
    int32).  ``kv_lens`` ((B,)) is how many keys each sequence has and
    ``q_starts`` ((B + 1,), rising from 0) where its new tokens begin among the N,
    whole numbers on the device; without ``q_starts`` each sequence has one.
    Token i of a sequence's n is at position ``kv_lens - n + i`` and sees the
    keys up to it.  Chunks of prompts, drafts and single tokens may be mixed.

    Returns (N, H, D), and with ``want_lse`` the fp32 log-sum-exp (N, H) too.
    Rows that see no key (of an empty sequence, at negative positions, behind the last
    sequence) are zero with lse -inf.  ``scale`` (positive) is 1/sqrt(D) unless
    given.  What the pages hold behind a sequence's length, NaN included, is
    not used; a NaN or infinity in a key or value that exists, and a
    table entry outside the cache, may reach every row of its sequence (the latter
    as NaN).  Lengths are taken into what the table has.

    Scores, probabilities, sums and statistics are fp32; with bf16 inputs the
    probabilities are rounded to bf16 for their product with v.  D is a
    multiple of 8 up to 128, page_size a power of two from 16 to 65536.  The
    caches may have any strides whose rows lie in 16-byte pieces.
    """
    scale = 1.0 / math.sqrt(max(1, q.shape[-1] if q.dim() else 1)) if scale is None else float(scale)
    if not 0.0 < scale < math.inf:
        raise ValueError(f"paged_attention: scale must be positive and finite, got {scale}")
    if not torch.compiler.is_compiling():
        res = native.paged_attention(q, k_cache, v_cache, block_table, kv_lens, q_starts, scale, bool(want_lse))
        if res is not None:
            return res
    _no_grad("paged_attention", q, k_cache, v_cache)
    if _eager_direct(q, k_cache, v_cache, block_table, kv_lens, q_starts):
        out, lse = _paged_attention_impl(q, k_cache, v_cache, block_table, kv_lens, q_starts, scale, want_lse)
    else:
        _require_device(q, k_cache, v_cache, block_table, kv_lens, q_starts)
        _check_paged_attention(q, k_cache, v_cache, block_table, kv_lens, q_starts)
        out, lse = paged_attention_op(q, k_cache, v_cache, block_table, kv_lens, q_starts, scale)
    return (out, lse) if want_lse else out


# ---------------------------------------------------------------- verify --


def _check_verify(logits: Tensor, ids: Tensor, q_starts: Tensor, uniforms: Tensor, draft_probs: Optional[Tensor],
                  temperature: float) -> None:
    op = "verify_drafts"
    if logits.dim() != 2 or logits.shape[1] == 0:
        raise ValueError(f"{op}: logits must be (N, vocabulary), got {tuple(logits.shape)}")
    n, v = logits.shape
    if v > MAX_VOCAB or n > 1 << 24:
        raise ValueError(f"{op}: {n} rows or a vocabulary of {v} are over 2^24 and 2^21")
    dtype_code(logits.dtype)
    _check_lengths(op, "ids", ids, n)
    _index_code(f"{op}: q_starts", q_starts)
    if q_starts.dim() != 1 or q_starts.shape[0] < 1:
        raise ValueError(f"{op}: q_starts must be (sequences + 1,), got {tuple(q_starts.shape)}")
    if uniforms.dtype != torch.float32:
        raise TypeError(f"{op}: uniforms must be float32, got {uniforms.dtype}")
    if uniforms.shape != (n, 2):
        raise ValueError(f"{op}: uniforms must be ({n}, 2), got {tuple(uniforms.shape)}")
    if draft_probs is not None:
        dtype_code(draft_probs.dtype)
        if draft_probs.shape != logits.shape:
            raise ValueError(f"{op}: draft_probs must be {tuple(logits.shape)}, got {tuple(draft_probs.shape)}")
    if temperature != 0.0 and not 1e-6 <= temperature < 1e38:
        raise ValueError(f"{op}: temperature must be 0 or from 1e-6 up, got {temperature}")


def _verify_drafts_impl(logits, ids, q_starts, uniforms, draft_probs, temperature) -> tuple[Tensor, Tensor]:
    device = _require_device(logits, ids, q_starts, uniforms, draft_probs)
    _check_verify(logits, ids, q_starts, uniforms, draft_probs, temperature)
    logits, uniforms = _table(logits), uniforms.contiguous()
    ids, ids_code = _lengths(ids)
    q_starts, starts_code = _lengths(q_starts)
    n, v = logits.shape
    tokens, counts = torch.empty_like(ids), ids.new_empty((q_starts.shape[0] - 1,), dtype=torch.int32)
    draft_args = (None, 0, _capi.DTYPE_F32)
    if draft_probs is not None:
        draft_probs = _table(draft_probs)
        draft_args = (draft_probs.data_ptr(), draft_probs.stride(0), dtype_code(draft_probs.dtype))
    with _DeviceStream(device) as stream:
        nbytes = _capi.verify_drafts_workspace_size(n, q_starts.shape[0] - 1, v)
        ws = _workspace(nbytes, device)
        _capi.verify_drafts(logits.data_ptr(), logits.stride(0), dtype_code(logits.dtype), *draft_args, n, v,
                            ids.data_ptr(), ids_code, q_starts.data_ptr(), starts_code, q_starts.shape[0] - 1,
                            uniforms.data_ptr(), float(temperature), tokens.data_ptr(), counts.data_ptr(),
                            ws.data_ptr(), nbytes, stream)
    return tokens, counts


@torch.library.custom_op("attnres_hip::verify_drafts", mutates_args=())
def verify_drafts_op(logits: Tensor, ids: Tensor, q_starts: Tensor, uniforms: Tensor, draft_probs: Optional[Tensor],
                     temperature: float) -> tuple[Tensor, Tensor]:
    return _verify_drafts_impl(logits, ids, q_starts, uniforms, draft_probs, temperature)


@verify_drafts_op.register_fake
def _verify_drafts_fake(logits, ids, q_starts, uniforms, draft_probs, temperature):
    return (ids.new_empty(ids.shape), ids.new_empty((q_starts.shape[0] - 1,), dtype=torch.int32))


def verify_drafts(logits: Tensor, ids: Tensor, q_starts: Tensor, uniforms: Tensor,
                  draft_probs: Optional[Tensor] = None, temperature: float = 1.0) -> tuple[Tensor, Tensor]:
    """Which drafted tokens stay, and the token behind them: speculative sampling's rule.

    Sequence b's rows ``q_starts[b] .. q_starts[b + 1] - 1`` (whole numbers rising from 0, the rows from the
    last on padding) are the packed input of a model's step: ``ids`` its last token and the drafts behind it,
    ``logits`` (N, V) the model's for each.  With p = softmax(logits /
    temperature) of row r and q the distribution that the draft ``ids[r + 1]``
    was drawn from (``draft_probs[r]``; none given: the draft is certain), the
    draft stays if ``uniforms[r, 0] * q < p`` at it.  The first that does not
    is replaced by a token from max(p - q, 0) (from p where that is all zero);
    behind drafts that all stay comes one from the last row's p.  It is the
    first j whose running sum is over ``uniforms[r, 1]`` times the whole.  So the tokens
    are distributed as if drawn from the model one by one; sequences of one row are plainly sampled.
    ``temperature`` is 0 (greedy: p is 1 at the largest logit, the lowest index of
    several; draft_probs are not read) or from 1e-6 up, and taken as fp32.

    Returns ``tokens`` (N,), of ids' type: row r the token behind ``ids[r]``, -1
    behind the last and in padding; and ``counts`` (B,) int32: how many tokens each sequence
    gets, at least 1 where it has rows (so many of its rows stand in the cache).  A row with
    a NaN or +infinity, or nothing but -infinity, gives no token: -1, not counted.
    ``uniforms`` (N, 2) fp32 are from [0, 1); ``logits`` and ``draft_probs`` bf16
    or fp32, V up to 2^21.  Sums that decide are taken in 64 bits.
    """
    temperature = float(temperature)
    if not torch.compiler.is_compiling():
        res = native.verify_drafts(logits, ids, q_starts, uniforms, draft_probs, temperature)
        if res is not None:
            return res
    _no_grad("verify_drafts", logits, draft_probs, uniforms)
    if _eager_direct(logits, ids, q_starts, uniforms, draft_probs):
        return _verify_drafts_impl(logits, ids, q_starts, uniforms, draft_probs, temperature)
    _require_device(logits, ids, q_starts, uniforms, draft_probs)
    _check_verify(logits, ids, q_starts, uniforms, draft_probs, temperature)
    return verify_drafts_op(logits, ids, q_starts, uniforms, draft_probs, temperature)


# ----------------------------------------------------------------- cache --


class PagedLayer(NamedTuple):
    """One layer's part in a step: what an attention sublayer writes and reads."""

    k: Tensor  #: (pages, kv_heads, page_size, head_dim)
    v: Tensor
    block_table: Tensor
    step: PagedSlots


class PagedCache:
    """Every layer's keys and values in pages, and which sequence holds which.

    ``pages`` pages of ``page_size`` tokens serve up to ``sequences`` sequences of up to
    ``max_tokens`` (whole pages) each.  All state (``block_table``, ``lens``, ``free_pages``,
    ``free_count``, the pages) is on the device and changed in place, so that a
    captured step runs on from where the last one ended.
    """

    def __init__(self, layers: int, pages: int, page_size: int, kv_heads: int, head_dim: int, sequences: int,
                 max_tokens: int, dtype: torch.dtype, device) -> None:
        self.page_size = _check_page("PagedCache", page_size)
        if max_tokens < page_size or max_tokens % page_size:
            raise ValueError(f"PagedCache: {max_tokens} tokens are not whole pages of {page_size}")
        shape = (layers, 2, pages, kv_heads, page_size, head_dim)
        self.kv = torch.empty(shape, dtype=dtype, device=device)
        i32 = dict(dtype=torch.int32, device=device)
        self.block_table = torch.zeros((sequences, max_tokens // page_size), **i32)
        self.lens = torch.zeros(sequences, **i32)  # tokens that each sequence holds
        self.free_pages = torch.arange(pages - 1, -1, -1, **i32)
        self.free_count = torch.full((1,), pages, **i32)

    @torch.no_grad()
    def extend(self, new: Tensor, num_tokens: int) -> PagedSlots:
        """Takes pages and slots for ``new`` ((B,)) tokens; a refused sequence (kv_lens 0) keeps what it has."""
        step = paged_slots(self.block_table, self.lens, new, self.free_pages, self.free_count, self.page_size,
                           num_tokens)
        self.lens.copy_(torch.where(step.kv_lens > 0, step.kv_lens, self.lens))
        self.free_count.copy_(step.free_count)
        return step

    @torch.no_grad()
    def keep(self, kept: Tensor) -> None:
        """Shortens every sequence to its first ``kept`` ((B,)) tokens; the pages behind are free again."""
        self.free_count.copy_(paged_release(self.block_table, self.lens, kept, self.free_pages, self.free_count,
                                            self.page_size))
        self.lens.copy_(torch.minimum(self.lens, kept.clamp(min=0)))

    def layers(self, step: PagedSlots) -> list:
        """The layers' parts in a step."""
        return [PagedLayer(k, v, self.block_table, step) for k, v in self.kv]


__all__ = ["PagedCache", "PagedLayer", "PagedSlots", "paged_attention", "paged_release", "paged_slots", "paged_write",
           "verify_drafts"]
