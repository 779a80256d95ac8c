"""Paged prefill with shaped scores: capped by a tanh, biased by distance, masked by an interval of keys a query.

``gqa_prefill_shaped_fn`` is ``gqa_prefill_paged_fn`` for layers whose scores or masks are not the plain causal ones:

* ``softcap``: scores become ``softcap * tanh(score / softcap)``;
* ``slopes``: every head's scores lose its slope times the distance;
* ``window``: a query sees the last ``window`` tokens up to itself;
* ``first_key``: the first token that each query sees, for instance the first of its document where several are
  packed into one sequence;
* ``last_key``: the last token that each query sees, in place of its own position, for instance the end of a
  prefix or of an image whose tokens see each other.

Any of them may be combined. ``gqa_tree_paged_fn`` is the decode step (and the verification of drafts) of such layers.
Scores, softmax statistics and sums are held in 32 bits; the softmax weights are rounded to the cache's type for the
matrix unit, half a step of each weight, as in the paged GQA kernels (fp16 weights lifted by 2^7 first), and the result
is rounded once more. The reference has the causal mask only (kernels/gqa_varlen.py:40-185).

The call runs on the current stream, allocates through torch's caching allocator only, reads no device value on the
host (with ``max_seqlen_q`` given), and can be captured in a graph.
"""
from __future__ import annotations

import ctypes
import functools

import torch

from .. import _lib
from .draft_tree import _caches, _slopes, _softcap, _window
from .latent_attention import _as_rows, _paged_args, _scale, _vec_rows

__all__ = ["gqa_prefill_shaped_fn"]


@functools.lru_cache(maxsize=256)
def _shaped_workspace(batch: int, total_q: int, max_q: int, hq: int, hkv: int, d: int, max_k: int, device: int) -> int:
    """Bytes for these sizes on this GPU (its number of CUs counts)."""
    nbytes = ctypes.c_int64(0)
    _lib.check(_lib.load().ti_gqa_prefill_shaped_workspace_bytes(batch, total_q, max_q, hq, hkv, d, max_k,
                                                                 ctypes.byref(nbytes)))
    return nbytes.value


def gqa_prefill_shaped_fn(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_table: torch.Tensor,
                          cu_seqlens_q: torch.Tensor, seqlen_k: torch.Tensor, max_seqlen_q: int | None = None,
                          page_size: int = 16, *, causal: bool = True, scale: float | None = None,
                          softcap: float | None = None, slopes: torch.Tensor | None = None,
                          window: int | None = None, first_key: torch.Tensor | None = None,
                          last_key: torch.Tensor | None = None, max_seqlen_k: int | None = None,
                          out: torch.Tensor | None = None) -> torch.Tensor:
    """Varlen GQA of packed queries over paged K/V with shaped scores.

    Args:
        q: ``[total_q, H_q, D]`` packed query rows, D 128 or 256
        k_cache, v_cache: ``[num_blocks, block_size, H_kv, D]``, contiguous; the chunks' own rows are in them
        block_table: ``[B, W]`` int32 (-1 padding allowed past each sequence)
        cu_seqlens_q: ``[B + 1]`` int32 query row offsets
        seqlen_k: ``[B]`` int32 cached tokens per sequence, the chunk included; query ``i`` of a chunk sits at the
            position ``seqlen_k - q_len + i``
        max_seqlen_q: host bound on every query length; None reads it from ``cu_seqlens_q`` (one device-to-host copy)
        page_size: tokens per page of the flattened cache (any)
        causal: a query sees the keys up to its own position (False: all of its sequence's); ``last_key`` goes before it
        scale: factor of the scores, ``D ** -0.5`` by default; positive
        softcap: 1e-3 to 1e4
        slopes: ``[H_q]`` float32; scores lose ``slopes[h] * |position - key|`` (after the cap)
        window: keys with ``position - key >= window`` are not seen
        first_key, last_key: ``[total_q]`` int32 positions in the query's sequence, both seen themselves
        max_seqlen_k: host bound on every ``seqlen_k``; only used to choose the schedule (without it the block table's
            width)
        out: preallocated ``[total_q, H_q, D]`` with 16-byte aligned rows
    Returns:
        ``[total_q, H_q, D]`` in q's dtype; rows that see no key are zero, rows of no sequence are not written. Block
        ids outside the cache below ``seqlen_k`` are treated as absent. A cached value (V) that is not finite can reach
        queries that do not see its token (a weight of zero times it), those whose rows share a workgroup with one that
        sees a token of its tile; keys that are not seen reach none.
    """
    # The call in its common form is checked and made in native code; None: another form, or one to refuse.
    stream = None if out is not None else _lib.native(q)
    if stream is not None and q.dim() == 3 and q.shape[-1] > 0:
        r = _lib.result(_lib.calls().shaped(q, k_cache, v_cache, block_table, cu_seqlens_q, seqlen_k, max_seqlen_q,
                                            page_size, causal, q.shape[-1] ** -0.5 if scale is None else scale, softcap,
                                            slopes, window, first_key, last_key, max_seqlen_k, stream))
        if r is not None:
            return r
    if q.dim() != 3:
        raise ValueError(f"q must be [total_q, H_q, D], got {tuple(q.shape)}")
    total_q, hq, d = q.shape
    dev, dt = q.device, q.dtype
    code = _lib.dtype_code(dt)
    if dev.type != "cuda":
        raise ValueError("gqa_prefill_shaped_fn runs on the GPU; q is on " + str(dev))
    _caches(k_cache, v_cache, hq, d, dt)
    hkv = k_cache.shape[2]
    if block_table.dim() != 2:
        raise ValueError(f"block_table must be [B, W], got {tuple(block_table.shape)}")
    b = block_table.shape[0]
    block_table, seqlen_k, rows, page_size = _paged_args(block_table, seqlen_k, k_cache, page_size, b, dev)
    if cu_seqlens_q.dtype != torch.int32:
        raise TypeError(f"cu_seqlens_q must be int32, got {cu_seqlens_q.dtype}")
    if cu_seqlens_q.shape != (b + 1,) or cu_seqlens_q.device != dev:
        raise ValueError(f"cu_seqlens_q must be [{b + 1}] on {dev}, got {tuple(cu_seqlens_q.shape)}")
    cu_seqlens_q = cu_seqlens_q.contiguous()
    for name, x in (("first_key", first_key), ("last_key", last_key)):
        if x is not None and (x.dtype != torch.int32 or x.shape != (total_q,) or x.device != dev):
            raise ValueError(f"{name} must be [{total_q}] int32 on {dev}")
    # Held until the launch: a copy freed before it is handed out again, for instance to the next copy.
    first_key = None if first_key is None else first_key.contiguous()
    last_key = None if last_key is None else last_key.contiguous()
    scale = _scale(d ** -0.5 if scale is None else scale)
    softcap, window, slopes = _softcap(softcap), _window(window), _slopes(slopes, hq, dev)
    if max_seqlen_q is None:
        max_seqlen_q = int((cu_seqlens_q[1:] - cu_seqlens_q[:-1]).max().item()) if b else 0
    max_seqlen_q = int(max_seqlen_q)
    if max_seqlen_q < 0:
        raise ValueError(f"max_seqlen_q must be >= 0, got {max_seqlen_q}")
    max_seqlen_q = min(max_seqlen_q, total_q)  # no chunk is longer
    bound = block_table.shape[1] * page_size
    if max_seqlen_k is not None:
        if int(max_seqlen_k) < 0:
            raise ValueError(f"max_seqlen_k must be >= 0, got {max_seqlen_k}")
        bound = min(bound, int(max_seqlen_k))
    if out is None:
        out = torch.empty((total_q, hq, d), dtype=dt, device=dev)
    elif out.shape != q.shape or out.dtype != dt or out.device != dev or not _vec_rows(out):
        raise ValueError("out must be a [total_q, H_q, D] tensor of q's dtype and device with 16-byte aligned rows")
    if b == 0 or total_q == 0:
        return out
    q = _as_rows(q)
    with _lib.on(dev):
        nbytes = _shaped_workspace(b, total_q, max_seqlen_q, hq, hkv, d, bound, torch.cuda.current_device())
        ws = torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None
        _lib.check(_lib.load().ti_gqa_prefill_shaped(
            q.data_ptr(), q.stride(0), q.stride(1), k_cache.data_ptr(), v_cache.data_ptr(), block_table.data_ptr(),
            block_table.stride(0), cu_seqlens_q.data_ptr(), seqlen_k.data_ptr(),
            None if first_key is None else first_key.data_ptr(), None if last_key is None else last_key.data_ptr(),
            None if slopes is None else slopes.data_ptr(), out.data_ptr(), out.stride(0), out.stride(1),
            None if ws is None else ws.data_ptr(), nbytes, b, total_q, max_seqlen_q, hq, hkv, d, page_size,
            rows // page_size, block_table.shape[1], bound, int(bool(causal)), scale, softcap, window, code,
            _lib.stream_handle(dev)))
    return out
