"""Drafted trees on the paged cache: attention of the drafts, and the accepted path's rows put in place.

A speculative step drafts up to 64 tokens for every sequence as a tree: the last certain token as its root, then
continuations of which several may share a beginning. All of them are appended to the cache in the order in which
they are listed (``rope_axes_append`` at the positions ``context + depth``), and ``gqa_tree_paged_fn`` gives each
its attention: over the context, and over those drafts that lie on its own path. Once the model's choices have
accepted one path, ``keep_drafts`` moves that path's rows behind the context in every layer at once, and the
sequence goes on from the returned length.

``gqa_tree_paged_fn`` with one token a sequence is a decode step whose scores may be shaped: capped by
``softcap tanh(s / softcap)``, less a slope times the distance, cut to a window (``gqa_prefill_shaped_fn`` is the
prefill of such layers). Scores, softmax statistics and sums are held in 32 bits; the softmax weights are rounded to
the cache's type for the matrix unit, half a step of each weight, as in the paged GQA kernels (fp16 weights lifted by
2^7 first), and the result is rounded once more. The reference drafts nothing; these functions stand beside its
``gqa_decode_paged_fn`` and ``store_kvcache`` and take the same caches, tables and lengths.

All run on the current stream, allocate through torch's caching allocator only, read no device value on the host,
and can be captured in a graph.
"""
from __future__ import annotations

import ctypes
import functools

import torch

from .. import _lib
from .latent_attention import _as_rows, _paged_args, _scale

__all__ = ["gqa_tree_paged_fn", "keep_drafts", "tree_masks"]

MAX_DRAFTS = 64


def _softcap(softcap: float | None) -> float:
    """The cap as the library takes it, 0 for none."""
    if softcap is None:
        return 0.0
    softcap = float(softcap)
    if not 1e-3 <= softcap <= 1e4:
        raise ValueError(f"softcap {softcap} must be 1e-3 to 1e4 (None: no cap)")
    return softcap


def _window(window: int | None) -> int:
    """The window as the library takes it, 0 for none."""
    if window is None:
        return 0
    window = int(window)
    if window < 1:
        raise ValueError(f"window {window} must be positive (None: no window)")
    return min(window, _lib.INT32_MAX)


def _slopes(slopes: torch.Tensor | None, heads: int, dev) -> torch.Tensor | None:
    if slopes is None:
        return None
    if slopes.shape != (heads,) or slopes.dtype != torch.float32 or slopes.device != dev:
        raise ValueError(f"slopes must be [{heads}] float32 on {dev}")
    return slopes.contiguous()


def _caches(k_cache: torch.Tensor, v_cache: torch.Tensor, hq: int, d: int, dt) -> None:
    if k_cache.dim() != 4 or v_cache.shape != k_cache.shape:
        raise ValueError(f"caches must both be [num_blocks, block_size, H_kv, D], got {tuple(k_cache.shape)} and "
                         f"{tuple(v_cache.shape)}")
    hkv, d2 = k_cache.shape[2:]
    if d2 != d:
        raise ValueError(f"head_dim mismatch: q {d}, cache {d2}")
    if d not in (128, 256):
        raise ValueError(f"head_dim {d} must be 128 or 256")
    if hkv <= 0 or hq == 0 or hq % hkv:
        raise ValueError(f"H_q={hq} is not a multiple of H_kv={hkv}")
    for name, c in (("k_cache", k_cache), ("v_cache", v_cache)):
        if not c.is_contiguous() or c.data_ptr() % 16:
            raise ValueError(f"{name} must be contiguous and 16-byte aligned (a copy of the cache is never made)")
        if c.dtype != dt:
            raise TypeError(f"dtype mismatch: q {dt}, {name} {c.dtype}")
    if v_cache.device != k_cache.device:
        raise ValueError(f"k_cache is on {k_cache.device}, v_cache on {v_cache.device}")


def tree_masks(parents) -> torch.Tensor:
    """Masks of a tree given as the parent of every draft (-1: none), int64 ``[N]`` or ``[B, N]`` on the CPU.

    Bit ``j`` of entry ``i``: draft ``j`` is draft ``i`` or one of its ancestors. Parents come before their children.
    """
    rows = torch.as_tensor(parents, dtype=torch.int64, device="cpu")
    if rows.dim() not in (1, 2) or not 1 <= rows.shape[-1] <= MAX_DRAFTS:
        raise ValueError(f"parents must be [N] or [B, N] with N from 1 to {MAX_DRAFTS}, got {tuple(rows.shape)}")
    if bool(((rows >= torch.arange(rows.shape[-1])) | (rows < -1)).any()):
        raise ValueError("a draft's parent must come before it, or be -1")
    out = []
    for row in rows.reshape(-1, rows.shape[-1]).tolist():
        masks = []
        for i, p in enumerate(row):
            masks.append((masks[p] if p >= 0 else 0) | 1 << i)
        out.append([m - (1 << 64) if m >> 63 else m for m in masks])
    return torch.tensor(out, dtype=torch.int64).reshape(rows.shape)


@functools.lru_cache(maxsize=256)
def _tree_workspace(batch: int, drafts: int, hq: int, hkv: int, d: int, device: int) -> int:
    """Bytes for these sizes on this GPU (its number of CUs counts)."""
    nbytes = ctypes.c_int64(0)
    _lib.check(_lib.load().ti_gqa_tree_workspace_bytes(batch, drafts, hq, hkv, d, ctypes.byref(nbytes)))
    return nbytes.value


def gqa_tree_paged_fn(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_table: torch.Tensor,
                      seqlen_kv: torch.Tensor, tree_mask: torch.Tensor | None = None, page_size: int = 16, *,
                      scale: float | None = None, softcap: float | None = None,
                      slopes: torch.Tensor | None = None, window: int | None = None,
                      out: torch.Tensor | None = None) -> torch.Tensor:
    """GQA of every sequence's last N tokens, a drafted tree, over its cache pages.

    Args:
        q: ``[B, N, H_q, D]``, N 1 to 64 drafts in the order of their cache rows, or ``[B, H_q, D]`` for one; D 128
            or 256; ``B N H_q`` below 2^24
        k_cache, v_cache: ``[num_blocks, block_size, H_kv, D]``, contiguous; the drafts' rows are in them
        block_table: ``[B, W]`` int32 (-1 padding allowed past each sequence)
        seqlen_kv: ``[B]`` int32 cached tokens, the drafts included: the context is ``C = seqlen_kv - N``
        tree_mask: ``[N]`` (one tree for all sequences) or ``[B, N]`` int64: draft ``i`` sees draft ``j`` where bit
            ``j`` of entry ``i`` is set (``tree_masks``; its own bit is not implied, bits from N on are ignored).
            None: the drafts ``j <= i``, a chain
        page_size: tokens per page of the flattened cache (any)
        scale: factor of the scores, ``D ** -0.5`` by default; positive
        softcap: scores become ``softcap * tanh(score / softcap)``; 1e-3 to 1e4
        slopes: ``[H_q]`` float32; scores lose ``slopes[h] * |p_i - p_j|`` (after the cap)
        window: keys with ``p_i - p_j >= window`` are not seen
        out: preallocated contiguous result
    Positions: token ``j`` of the context is at ``j``, draft ``i`` at ``C`` plus the number of other drafts that it
    sees, its depth in the tree.
    Returns:
        q's shape and dtype. A draft that sees nothing gives zeros; block ids outside the cache below ``seqlen_kv``
        are treated as absent; where ``seqlen_kv < N`` (graph padding) the drafts before token 0 do not exist as
        keys. A cached value (V) that is not finite also reaches the drafts that do not see its token (a weight of
        zero times it); keys that are not seen, and what lies behind ``seqlen_kv``, reach none.
    """
    # The call in its common form is checked and made in native code; None: another form, or one to refuse.
    stream = None if out is not None else _lib.native(q)
    if stream is not None and q.dim() > 0 and q.shape[-1] > 0:
        r = _lib.result(_lib.calls().tree(q, k_cache, v_cache, block_table, seqlen_kv, tree_mask, page_size,
                                          q.shape[-1] ** -0.5 if scale is None else scale, softcap, slopes, window, stream))
        if r is not None:
            return r
    if q.dim() not in (3, 4):
        raise ValueError(f"q must be [B, H_q, D] or [B, N, H_q, D], got {tuple(q.shape)}")
    q4 = q.unsqueeze(1) if q.dim() == 3 else q
    b, n, hq, d = q4.shape
    dev, dt = q.device, q.dtype
    code = _lib.dtype_code(dt)
    if dev.type != "cuda":
        raise ValueError("gqa_tree_paged_fn runs on the GPU; q is on " + str(dev))
    if not 1 <= n <= MAX_DRAFTS:
        raise ValueError(f"{n} drafts must be 1 to {MAX_DRAFTS}")
    _caches(k_cache, v_cache, hq, d, dt)
    hkv = k_cache.shape[2]
    block_table, seqlen_kv, rows, page_size = _paged_args(block_table, seqlen_kv, k_cache, page_size, b, dev)
    mask_stride = 0
    if tree_mask is not None:
        if tree_mask.dtype != torch.int64 or tree_mask.device != dev or tree_mask.shape not in ((n,), (b, n)):
            raise ValueError(f"tree_mask must be [{n}] or [{b}, {n}] int64 on {dev}, got {tuple(tree_mask.shape)} "
                             f"{tree_mask.dtype} on {tree_mask.device}")
        if tree_mask.stride(-1) != 1:
            tree_mask = tree_mask.contiguous()
        mask_stride = tree_mask.stride(0) if tree_mask.dim() == 2 else 0
    scale = _scale(d ** -0.5 if scale is None else scale)
    softcap, window, slopes = _softcap(softcap), _window(window), _slopes(slopes, hq, dev)
    if out is None:
        out = torch.empty(q.shape, dtype=dt, device=dev)
    elif (out.shape != q.shape or out.dtype != dt or out.device != dev or not out.is_contiguous()
          or out.data_ptr() % 16):
        raise ValueError(f"out must be a contiguous {list(q.shape)} tensor of q's dtype and device")
    if b == 0:
        return out
    q4 = _as_rows(q4)
    with _lib.on(dev):
        nbytes = _tree_workspace(b, n, hq, hkv, d, torch.cuda.current_device())
        ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
        _lib.check(_lib.load().ti_gqa_tree_paged(
            q4.data_ptr(), q4.stride(0), q4.stride(1), q4.stride(2), k_cache.data_ptr(), v_cache.data_ptr(),
            block_table.data_ptr(), block_table.stride(0), seqlen_kv.data_ptr(),
            None if tree_mask is None else tree_mask.data_ptr(), mask_stride,
            None if slopes is None else slopes.data_ptr(), out.data_ptr(), ws.data_ptr(),
            nbytes, b, n, hq, hkv, d,
            page_size, rows // page_size, block_table.shape[1], scale, softcap, window, code,
            _lib.stream_handle(dev)))
    return out


def keep_drafts(cache: torch.Tensor, block_table: torch.Tensor, seqlen_kv: torch.Tensor, accepted: torch.Tensor,
                page_size: int = 16, *, num_drafts: int) -> torch.Tensor:
    """Move the accepted drafts' cache rows behind the context, in place; returns the new lengths.

    Args:
        cache: ``[..., num_blocks, block_size, H_kv, D]``, contiguous: all layers' keys and values at once (for
            instance ``allocate_kv_cache``'s ``[2, layers, num_blocks, block_size, H_kv, D]``), one layer's, or a
            latent cache; 16-bit
        block_table: ``[B, W]`` int32, as the attention took it
        seqlen_kv: ``[B]`` int32 cached tokens, the drafts included
        accepted: ``[B, M]`` int32: the accepted drafts of every sequence, ascending (a path of the tree from its
            root), -1 behind the last. The list ends at its first entry that does not ascend or is no draft
        page_size: tokens per page of the flattened cache (any)
        num_drafts: N of the step, 1 to 64
    Returns:
        ``[B]`` int32: ``C + accepted drafts`` with ``C = seqlen_kv - num_drafts``. Token ``C + j`` of every plane holds
        what token ``C + accepted[j]`` held; what lies behind the new lengths is not defined. A sequence with
        ``seqlen_kv < num_drafts`` (graph padding) keeps its rows and length. Blocks outside the cache are skipped. The
        drafts' blocks belong to one sequence each.
    """
    # The call in its common form is checked and made in native code; None: another form, or one to refuse.
    stream = _lib.native(cache)
    if stream is not None:
        r = _lib.result(_lib.calls().keep(cache, block_table, seqlen_kv, accepted, page_size, num_drafts, stream))
        if r is not None:
            return r
    if cache.dim() < 4:
        raise ValueError(f"cache must be [..., num_blocks, block_size, H_kv, D], got {tuple(cache.shape)}")
    dev = cache.device
    _lib.dtype_code(cache.dtype)
    if dev.type != "cuda":
        raise ValueError("keep_drafts runs on the GPU; cache is on " + str(dev))
    if not cache.is_contiguous() or cache.data_ptr() % 16:
        raise ValueError("cache must be contiguous and 16-byte aligned (a copy of the cache is never made)")
    nb, bs, hkv, d = cache.shape[-4:]
    if hkv * d == 0 or hkv * d % 8:
        raise ValueError(f"cache rows of {hkv} x {d} values must be a multiple of 8")
    num_drafts = int(num_drafts)
    if not 1 <= num_drafts <= MAX_DRAFTS:
        raise ValueError(f"num_drafts {num_drafts} must be 1 to {MAX_DRAFTS}")
    if block_table.dim() != 2:
        raise ValueError(f"block_table must be [B, W], got {tuple(block_table.shape)}")
    b = block_table.shape[0]
    if accepted.dtype != torch.int32 or accepted.device != dev:
        raise ValueError(f"accepted must be int32 on {dev}")
    if accepted.dim() != 2 or accepted.shape[0] != b:
        raise ValueError(f"accepted must be [{b}, M], got {tuple(accepted.shape)}")
    if cache.numel() == 0:
        raise ValueError(f"cache {tuple(cache.shape)} has no rows")
    planes = cache.view(-1, nb, bs, hkv, d)
    block_table, seqlen_kv, rows, page_size = _paged_args(block_table, seqlen_kv, planes[0], page_size, b, dev)
    if accepted.stride(1) != 1:
        accepted = accepted.contiguous()
    seqlen = torch.empty(b, dtype=torch.int32, device=dev)
    if b == 0:
        return seqlen
    with _lib.on(dev):
        _lib.check(_lib.load().ti_keep_drafts(
            cache.data_ptr(), block_table.data_ptr(), block_table.stride(0), seqlen_kv.data_ptr(),
            accepted.data_ptr(), accepted.stride(0), seqlen.data_ptr(), b, num_drafts, accepted.shape[1], planes.shape[0],
            hkv * d, page_size, rows // page_size, block_table.shape[1], _lib.stream_handle(dev)))
    return seqlen
