"""Latent attention: every cached token is one vector that all heads share.

A latent layer projects a token to a small vector ``c`` (``latent_dim`` values) and a rotated key part
``k_r`` (64 values), and caches only those: ``[c | k_r]``, 1,152 bytes a token at latent_dim 512 in 16
bits whatever the number of heads. Head ``h`` has the key ``[c @ Wk_h | k_r]`` and the value ``c @ Wv_h``.
Two forms give the same attention:

* absorbed: ``q_nope . (c @ Wk_h) = (q_nope @ Wk_h^T) . c``, so the query moves into the latent space and
  attends over the cached vectors themselves; ``Wv_h`` is applied to the result. Little to read, many
  operations per key: for decoding (``latent_decode_paged_fn``).
* expanded: keys and values of every head are computed once per token and attended over as usual, a third
  of the operations per (query, key) pair: for prefill chunks (``latent_prefill_fn``).

``latent_rope_append`` is the input side: it normalises the latent, rotates the key part and the queries'
rotated parts, and writes the cache rows.

The cache is laid out as the paged cache of one KV head, ``[num_blocks, block_size, 1, latent_dim + 64]``
(``engine.kv_layout.allocate_latent_cache``), so block tables, slot mappings, ``copy_blocks`` and
``swap_blocks`` apply to it as they are. The reference has no latent layers; these functions stand beside
its ``store_kvcache``, ``gqa_decode_paged_fn`` and varlen prefill.

Both attention forms hold scores, softmax statistics and sums in 32 bits and round the softmax weights to the
operands' type for the matrix unit, half a step of each weight, as the paged GQA kernels do (fp16 weights are
lifted by 2^7 first, so that those far below their row's greatest keep their bits); the result is rounded
once more.

All run on the current stream, allocate through torch's caching allocator only, read no device value on
the host, and can be captured in a graph.
"""
from __future__ import annotations

import ctypes
import functools

import torch

from .. import _lib
from .qknorm_rope import _cos_sin

__all__ = ["latent_rope_append", "latent_decode_paged_fn", "latent_prefill_fn"]

ROPE_DIM = 64
LATENT_DIMS = (256, 512)


def _vec_rows(t: torch.Tensor) -> bool:
    """Unit element stride, 16-byte aligned rows."""
    return (t.stride(-1) == 1 and t.data_ptr() % 16 == 0
            and all(s % 8 == 0 for s in t.stride()[:-1]))


def _as_rows(t: torch.Tensor) -> torch.Tensor:
    return t if _vec_rows(t) else t.clone(memory_format=torch.contiguous_format)


def _scale(scale: float) -> float:
    scale = float(scale)
    if not 0 < scale <= 1e30:
        raise ValueError(f"scale {scale} must be positive and at most 1e30")
    return scale


def latent_rope_append(q_rope: torch.Tensor | None, latent: torch.Tensor, key_rope: torch.Tensor,
                       weight: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor,
                       latent_cache: torch.Tensor, slot_mapping: torch.Tensor, eps: float = 1e-5, *,
                       weight_offset: float = 1.0, q_out: torch.Tensor | None = None):
    """Input side of one step of a latent layer in one launch; returns the rotated ``q_rope``.

    q_rope ``[T, H, 64]`` (the queries' rotated parts, None for none), latent ``[T, L]`` as projected,
    key_rope ``[T, 64]`` (any strides: both may be slices of one projection), weight ``[L]``, cos/sin
    ``[T, 64]``, ``[1, 64]`` or ``[64]`` (the first 32 columns serve both halves); ``latent_cache`` the
    cache rows ``[num_slots, L + 64]``; ``slot_mapping`` ``[T]`` int32 (slots < 0 or >= num_slots are
    skipped, duplicates unsupported). The row written is ``[RMSNorm(latent) * (weight_offset + weight) |
    rotate(key_rope)]``, the rotation pairing ``i`` with ``i + 32`` (weights trained with neighbours ``2 i`` and
    ``2 i + 1`` as pairs: the columns ``0, 2, .. 62, 1, 3, .. 63`` of both rotated parts' projections, once, give the
    same scores); ``weight_offset`` is 1 as in ``qknorm_rope``, 0 for weights that are the whole factor. ``q_out``
    ``[T, H, 64]`` receives the rotated parts, for instance the last 64 columns of ``latent_decode_paged_fn``'s
    queries; it may be ``q_rope`` itself.
    """
    # The call in its common form is checked and made in native code; None: another form, or one to refuse.
    stream = None if q_out is not None else _lib.native(latent)
    if stream is not None:
        r = _lib.result(_lib.calls().latent_append(q_rope, latent, key_rope, weight, cos, sin, latent_cache,
                                                   slot_mapping, eps, weight_offset, stream))
        if r is not None:
            return None if r is True else r
    if latent.dim() != 2 or key_rope.dim() != 2:
        raise ValueError("latent must be [T, L] and key_rope [T, 64]")
    t, dim = latent.shape
    dev, dt = latent.device, latent.dtype
    code = _lib.dtype_code(dt)
    if dev.type != "cuda":
        raise ValueError("latent_rope_append runs on the GPU; latent is on " + str(dev))
    if dim not in LATENT_DIMS:
        raise ValueError(f"latent_dim {dim} must be one of {LATENT_DIMS}")
    if key_rope.shape != (t, ROPE_DIM):
        raise ValueError(f"key_rope must be [{t}, {ROPE_DIM}], got {tuple(key_rope.shape)}")
    heads = 0
    if q_rope is not None:
        if q_rope.dim() != 3 or q_rope.shape[0] != t or q_rope.shape[2] != ROPE_DIM:
            raise ValueError(f"q_rope must be [{t}, H, {ROPE_DIM}], got {tuple(q_rope.shape)}")
        heads = q_rope.shape[1]
    elif q_out is not None:
        raise ValueError("q_out without q_rope")
    if weight.shape != (dim,):
        raise ValueError(f"weight must be [{dim}], got {tuple(weight.shape)}")
    if latent_cache.dim() != 2 or latent_cache.shape[1] != dim + ROPE_DIM:
        raise ValueError(f"latent_cache must be [num_slots, {dim + ROPE_DIM}] rows, got "
                         f"{tuple(latent_cache.shape)}")
    if not _vec_rows(latent_cache) or latent_cache.stride(0) < dim + ROPE_DIM:
        raise ValueError("latent_cache rows must be contiguous, apart and 16-byte aligned (the cache is "
                         "never copied)")
    for name, x in (("key_rope", key_rope), ("q_rope", q_rope), ("weight", weight),
                    ("latent_cache", latent_cache)):
        if x is not None and (x.dtype != dt or x.device != dev):
            raise ValueError(f"{name} must be {dt} on {dev}")
    if slot_mapping.dtype != torch.int32 or slot_mapping.shape != (t,) or slot_mapping.device != dev:
        raise ValueError(f"slot_mapping must be [{t}] int32 on {dev}")
    cos, sin, rd, cs_stride = _cos_sin(cos, sin, t, dt, dev)
    if rd != ROPE_DIM:
        raise ValueError(f"cos/sin must have {ROPE_DIM} columns, got {rd}")
    if cs_stride % 8 or cos.data_ptr() % 16 or sin.data_ptr() % 16:
        cos, sin = cos.clone(memory_format=torch.contiguous_format), sin.clone(
            memory_format=torch.contiguous_format)
        cs_stride = 0 if cs_stride == 0 else cos.stride(0)
    if q_rope is not None:
        if q_out is None:
            q_out = torch.empty((t, heads, ROPE_DIM), dtype=dt, device=dev)
        elif (q_out.shape != q_rope.shape or q_out.dtype != dt or q_out.device != dev
              or not _vec_rows(q_out)):
            raise ValueError("q_out must be a [T, H, 64] tensor of q_rope's dtype and device with 16-byte "
                             "aligned rows")
        q_rope = _as_rows(q_rope)
    if t == 0:
        return q_out
    latent, key_rope = _as_rows(latent), _as_rows(key_rope)
    weight, slot_mapping = _as_rows(weight), slot_mapping.contiguous()
    q = (q_rope.data_ptr(), q_rope.stride(0), q_rope.stride(1), q_out.data_ptr(), q_out.stride(0),
         q_out.stride(1)) if heads else (None, 0, 0, None, 0, 0)
    with _lib.on(dev):
        _lib.check(_lib.load().ti_latent_rope_append(
            *q, latent.data_ptr(), latent.stride(0), key_rope.data_ptr(), key_rope.stride(0),
            weight.data_ptr(), float(weight_offset), cos.data_ptr(), sin.data_ptr(), cs_stride,
            latent_cache.data_ptr(), latent_cache.stride(0), latent_cache.shape[0],
            slot_mapping.data_ptr(), t, heads, dim, ROPE_DIM, float(eps), code,
            _lib.stream_handle(dev)))
    return q_out


@functools.lru_cache(maxsize=256)
def _decode_workspace(batch: int, new: int, heads: int, latent: int, device: int) -> int:
    """Bytes for these sizes on this GPU (its number of CUs counts)."""
    nbytes = ctypes.c_int64(0)
    _lib.check(_lib.load().ti_latent_decode_workspace_bytes(batch, new, heads, latent,
                                                            ctypes.byref(nbytes)))
    return nbytes.value


def latent_decode_paged_fn(q: torch.Tensor, latent_cache: torch.Tensor, block_table: torch.Tensor,
                           seqlen_kv: torch.Tensor, page_size: int = 16, *, scale: float,
                           out: torch.Tensor | None = None) -> torch.Tensor:
    """Latent attention on the cache pages, absorbed form: a decode step, or a few tokens a sequence.

    Args:
        q: ``[B, H, L + 64]`` for one new token a sequence, or ``[B, N, H, L + 64]`` for its last ``N``
            (drafted tokens, a short chunk): ``[q_nope @ Wk^T | rotated part]``; B N H below 2^24
        latent_cache: ``[num_blocks, block_size, 1, L + 64]``, contiguous; the new tokens' rows are in it
        block_table: ``[B, W]`` int32 (-1 padding allowed past each sequence)
        seqlen_kv: ``[B]`` int32 context lengths, the new tokens included
        page_size: tokens per page of the flattened cache (any)
        scale: factor of the scores, ``(nope_dim + 64) ** -0.5`` of the expanded heads
        out: preallocated contiguous result
    Returns:
        ``[B, H, L]`` or ``[B, N, H, L]`` in q's dtype: the weighted latents, to which the caller applies
        each head's ``Wv``. Query ``i`` of ``N`` sees the keys ``j <= seqlen_kv - N + i``; one that sees
        nothing gives zeros. Block ids outside the cache below ``seqlen_kv`` are treated as absent. A cached
        value that is not finite also reaches the queries of ``N`` that come before its token (a weight of
        zero times it); what lies behind ``seqlen_kv`` reaches none.
    """
    # The call in its common form is checked and made in native code; None: another form, or one to refuse.
    stream = None if out is not None else _lib.native(q)
    if stream is not None:
        r = _lib.result(_lib.calls().latent_decode(q, latent_cache, block_table, seqlen_kv, page_size, scale,
                                                   stream))
        if r is not None:
            return r
    if q.dim() not in (3, 4):
        raise ValueError(f"q must be [B, H, L + 64] or [B, N, H, L + 64], got {tuple(q.shape)}")
    q4 = q.unsqueeze(1) if q.dim() == 3 else q
    b, new, h, row = q4.shape
    dim = row - ROPE_DIM
    dev, dt = q.device, q.dtype
    code = _lib.dtype_code(dt)
    if dev.type != "cuda":
        raise ValueError("latent_decode_paged_fn runs on the GPU; q is on " + str(dev))
    if dim not in LATENT_DIMS:
        raise ValueError(f"q's last dimension {row} must be latent_dim + 64 with latent_dim in {LATENT_DIMS}")
    if h == 0 or new == 0:
        raise ValueError(f"q {tuple(q.shape)} has no heads or no tokens")
    if latent_cache.dim() != 4 or latent_cache.shape[2] != 1 or latent_cache.shape[3] != row:
        raise ValueError(f"latent_cache must be [num_blocks, block_size, 1, {row}], got "
                         f"{tuple(latent_cache.shape)}")
    if not latent_cache.is_contiguous() or latent_cache.data_ptr() % 16:
        raise ValueError("latent_cache must be contiguous and 16-byte aligned (the cache is never copied)")
    if latent_cache.dtype != dt:
        raise TypeError(f"dtype mismatch: q {dt}, latent_cache {latent_cache.dtype}")
    block_table, seqlen_kv, rows, page_size = _paged_args(block_table, seqlen_kv, latent_cache, page_size,
                                                          b, dev)
    scale = _scale(scale)
    shape = (b, h, dim) if q.dim() == 3 else (b, new, h, dim)
    if out is None:
        out = torch.empty(shape, dtype=dt, device=dev)
    elif (out.shape != shape or out.dtype != dt or out.device != dev or not out.is_contiguous()
          or out.data_ptr() % 16):
        raise ValueError(f"out must be a contiguous {list(shape)} tensor of q's dtype and device")
    if b == 0:
        return out
    q4 = _as_rows(q4)
    with _lib.on(dev):
        nbytes = _decode_workspace(b, new, h, dim, torch.cuda.current_device())
        ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
        _lib.check(_lib.load().ti_latent_decode_paged(
            q4.data_ptr(), q4.stride(0), q4.stride(1), q4.stride(2), latent_cache.data_ptr(),
            block_table.data_ptr(), block_table.stride(0), seqlen_kv.data_ptr(), out.data_ptr(),
            ws.data_ptr(), nbytes, b, new, h, dim, ROPE_DIM, page_size, rows // page_size,
            block_table.shape[1], scale, code, _lib.stream_handle(dev)))
    return out


def _paged_args(block_table, seqlen_kv, cache, page_size, b, dev):
    """The block table, lengths and page size of a call on ``cache``, checked."""
    if block_table.dtype != torch.int32 or seqlen_kv.dtype != torch.int32:
        raise TypeError(f"block_table/seqlen_kv must be int32, got {block_table.dtype}/{seqlen_kv.dtype}")
    if block_table.dim() != 2 or block_table.shape[0] != b:
        raise ValueError(f"block_table must be [{b}, W], got {tuple(block_table.shape)}")
    if seqlen_kv.shape != (b,):
        raise ValueError(f"seqlen_kv must be [{b}], got {tuple(seqlen_kv.shape)}")
    page_size = int(page_size)
    rows = cache.shape[0] * cache.shape[1]
    if page_size <= 0 or rows % page_size != 0:
        raise ValueError(f"page_size {page_size} does not tile the cache's {rows} rows")
    for name, t in (("cache", cache), ("block_table", block_table), ("seqlen_kv", seqlen_kv)):
        if t.device != dev:
            raise ValueError(f"{name} is on {t.device}, q on {dev}")
    if block_table.stride(-1) != 1:
        block_table = block_table.contiguous()
    return block_table, seqlen_kv.contiguous(), rows, page_size


@functools.lru_cache(maxsize=256)
def _prefill_workspace(batch: int, total_q: int, total_k: int, heads: int, d: int, device: int) -> int:
    """Bytes for these sizes on this GPU (its number of CUs counts)."""
    nbytes = ctypes.c_int64(0)
    _lib.check(_lib.load().ti_latent_prefill_workspace_bytes(batch, total_q, total_k, heads, d,
                                                             ctypes.byref(nbytes)))
    return nbytes.value


def latent_prefill_fn(q: torch.Tensor, kv: torch.Tensor, key_rope: torch.Tensor,
                      cu_seqlens_q: torch.Tensor, cu_seqlens_k: torch.Tensor, max_seqlen_q: int, *,
                      causal: bool = True, scale: float | None = None,
                      out: torch.Tensor | None = None) -> torch.Tensor:
    """Latent attention over packed chunks, expanded form.

    Args:
        q: ``[total_q, H, D + 64]``, ``[q_nope | rotated part]``, D 128 or 64
        kv: ``[total_k, H, 2 D]``, ``[c @ Wk | c @ Wv]`` of every key token: a chunk's own and, for a
            continuation, the cached ones before it, whose rows the caller gathers from the pages
        key_rope: ``[total_k, 64]`` the rotated key parts, shared by the heads (any row stride: for
            instance the last columns of cache rows)
        cu_seqlens_q, cu_seqlens_k: ``[B + 1]`` int32 offsets of each sequence's queries and keys
        max_seqlen_q: host int, at least the longest chunk
        causal: query ``i`` sees the keys ``j <= k_len - q_len + i`` (False: all of its sequence's)
        scale: factor of the scores, ``(D + 64) ** -0.5`` by default
    Returns:
        ``[total_q, H, D]`` in q's dtype; rows that see no key are zero, rows of no sequence are not
        written. A value (kv's second half) that is not finite can reach queries that do not see its key (a
        weight of zero times it): those that share their 32 queries, counted from the chunk's start, with one
        that sees any of its 64 keys, counted from the sequence's start. Keys that are not finite and not
        seen reach none.
    """
    if q.dim() != 3 or kv.dim() != 3 or key_rope.dim() != 2:
        raise ValueError("q and kv must be [tokens, H, dims] and key_rope [tokens, 64]")
    total_q, h, row = q.shape
    d = row - ROPE_DIM
    dev, dt = q.device, q.dtype
    code = _lib.dtype_code(dt)
    if dev.type != "cuda":
        raise ValueError("latent_prefill_fn runs on the GPU; q is on " + str(dev))
    if d not in (64, 128):
        raise ValueError(f"q's last dimension {row} must be 128 + 64 or 64 + 64")
    total_k = kv.shape[0]
    if kv.shape[1:] != (h, 2 * d) or h == 0:
        raise ValueError(f"kv must be [total_k, {h}, {2 * d}], got {tuple(kv.shape)}")
    if key_rope.shape != (total_k, ROPE_DIM):
        raise ValueError(f"key_rope must be [{total_k}, {ROPE_DIM}], got {tuple(key_rope.shape)}")
    for name, t in (("kv", kv), ("key_rope", key_rope)):
        if t.dtype != dt or t.device != dev:
            raise ValueError(f"{name} must be {dt} on {dev}")
    if cu_seqlens_q.dim() != 1 or cu_seqlens_q.shape != cu_seqlens_k.shape or cu_seqlens_q.shape[0] < 1:
        raise ValueError("cu_seqlens_q and cu_seqlens_k must both be [B + 1]")
    for name, t in (("cu_seqlens_q", cu_seqlens_q), ("cu_seqlens_k", cu_seqlens_k)):
        if t.dtype != torch.int32:
            raise TypeError(f"{name} must be int32, got {t.dtype}")
        if t.device != dev:
            raise ValueError(f"{name} is on {t.device}, q on {dev}")
    b = cu_seqlens_q.shape[0] - 1
    max_seqlen_q = int(max_seqlen_q)
    if max_seqlen_q < 0:
        raise ValueError(f"max_seqlen_q {max_seqlen_q} is negative")
    max_seqlen_q = min(max_seqlen_q, _lib.INT32_MAX)  # no chunk is longer
    scale = _scale(row ** -0.5 if scale is None else scale)
    if out is None:
        out = torch.empty((total_q, h, d), dtype=dt, device=dev)
    elif out.shape != (total_q, h, d) or out.dtype != dt or out.device != dev or not _vec_rows(out):
        raise ValueError(f"out must be a [{total_q}, {h}, {d}] tensor of q's dtype and device with 16-byte "
                         "aligned rows")
    if total_q == 0 or b == 0:
        return out
    q, kv, key_rope = _as_rows(q), _as_rows(kv), _as_rows(key_rope)
    # Held until the launch: a copy freed before it is handed out again, for instance to the next copy.
    cu_seqlens_q, cu_seqlens_k = cu_seqlens_q.contiguous(), cu_seqlens_k.contiguous()
    with _lib.on(dev):
        nbytes = _prefill_workspace(b, total_q, total_k, h, d, torch.cuda.current_device())
        ws = torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None
        _lib.check(_lib.load().ti_latent_prefill(
            q.data_ptr(), q.stride(0), q.stride(1), kv.data_ptr(), kv.stride(0), kv.stride(1),
            key_rope.data_ptr(), key_rope.stride(0), cu_seqlens_q.data_ptr(),
            cu_seqlens_k.data_ptr(), out.data_ptr(), out.stride(0), out.stride(1),
            None if ws is None else ws.data_ptr(), nbytes, b, total_q,
            total_k, max_seqlen_q, h, d, ROPE_DIM, int(bool(causal)), scale, code,
            _lib.stream_handle(dev)))
    return out
