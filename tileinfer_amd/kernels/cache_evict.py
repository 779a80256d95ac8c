"""Eviction from the paged cache by accumulated attention weight.

``cache_attention_mass`` adds up, for every cached token and KV head, the softmax weight that the last
queries of its sequence give it: those of one decode step, step after step, or of a window at the end of a
prompt. ``evict_kvcache`` keeps the heaviest tokens of every (sequence, KV head), with the first and the most
recent ones always among them, and copies their rows to the blocks of a new, shorter table. The old table's
blocks are untouched, so blocks shared with other sequences (prefix caching) stay valid; the caller takes the
new blocks from its block manager and releases the old table afterwards.

Both take the KV cache of one attention layer, or a latent cache as its one KV head with ``v_cache=None``.
Keys are cached after their rotation, so a token keeps its position's angle wherever its row moves; the
queries' positions go on counting the evicted tokens, the cache's length does not. ``engine.Sequence`` has one
count for both, so a cut sequence's slots, tables and lengths are the caller's to make: from the new table and
the returned lengths, not from ``engine.kv_layout``, ``DeviceBlockTables`` or ``PagedKVManager``, and its table is
no prefix of its token ids (never recorded in a prefix cache).

All run on the current stream, allocate through torch's caching allocator only, read no device value on
the host, and can be captured in a graph. The reference never drops cached tokens.
"""
from __future__ import annotations

import ctypes
import functools

import torch

from .. import _lib
from .latent_attention import _as_rows, _paged_args, _scale

__all__ = ["cache_attention_mass", "evict_kvcache"]

HEAD_DIMS = (128, 256, 320, 576)


@functools.lru_cache(maxsize=256)
def _mass_workspace(batch: int, new: int, hq: int, hkv: int, d: int, page_size: int, width: int) -> int:
    nbytes = ctypes.c_int64(0)
    _lib.check(_lib.load().ti_cache_mass_workspace_bytes(batch, new, hq, hkv, d, page_size, width,
                                                         ctypes.byref(nbytes)))
    return nbytes.value


def _cache_ok(name: str, cache: torch.Tensor) -> None:
    if cache.dim() != 4:
        raise ValueError(f"{name} must be [num_blocks, block_size, H_kv, D], got {tuple(cache.shape)}")
    if not cache.is_contiguous() or cache.data_ptr() % 16:
        raise ValueError(f"{name} must be contiguous and 16-byte aligned (a copy of the cache is never made)")


def _mass_ok(mass: torch.Tensor, b: int, hkv: int, tokens: int, dev) -> None:
    if mass.dtype != torch.float32:
        raise TypeError(f"mass must be float32, got {mass.dtype}")
    if mass.dim() != 3 or mass.shape[:2] != (b, hkv) or mass.shape[2] < tokens:
        raise ValueError(f"mass must be [{b}, {hkv}, >= {tokens}] (block table width x page_size), got "
                         f"{tuple(mass.shape)}")
    if mass.device != dev:
        raise ValueError(f"mass is on {mass.device}, the cache on {dev}")
    if mass.numel() and (mass.stride(2) != 1 or mass.stride(1) < mass.shape[2]
                         or (b > 1 and mass.stride(0) < hkv * mass.stride(1))):
        raise ValueError(f"mass rows must be contiguous and apart (stride {mass.stride()})")


def cache_attention_mass(q: torch.Tensor, k_cache: torch.Tensor, block_table: torch.Tensor,
                         seqlen_kv: torch.Tensor, page_size: int = 16, *, scale: float | None = None,
                         mass: torch.Tensor | None = None) -> torch.Tensor:
    """Attention weight of every cached token from its sequence's last queries.

    Args:
        q: ``[B, H_q, D]`` (a decode step's queries) or ``[B, N, H_q, D]`` (the last ``N`` tokens'), as the
            attention gets them
        k_cache: ``[num_blocks, block_size, H_kv, D]``, contiguous, the new tokens' keys in it; D 128 or
            256, or a latent cache's 320 or 576 (H_kv 1)
        block_table, seqlen_kv, page_size: as ``gqa_decode_paged_fn`` takes them (any page size)
        scale: factor of the scores, ``D ** -0.5`` by default
        mass: running sums ``[B, H_kv, capacity >= W * page_size]`` float32, added to in place; None for
            new ones, zero elsewhere
    Returns:
        ``mass``: ``mass[b, g, t] += sum over queries i and heads h of group g of softmax_t(scale * q . K)``,
        query ``i`` of ``N`` seeing ``t <= seqlen_kv - N + i``. Values from ``seqlen_kv`` on are not touched.
        The same call gives the same bits.
    """
    # The call in its common form is checked and made in native code; None: another form, or one to refuse.
    stream = _lib.native(q)
    if stream is not None and q.dim() > 0 and q.shape[-1] > 0:
        r = _lib.result(_lib.calls().cache_mass(q, k_cache, block_table, seqlen_kv, page_size,
                                                q.shape[-1] ** -0.5 if scale is None else scale, mass, stream))
        if r is not None:
            return r
    if q.dim() not in (3, 4):
        raise ValueError(f"q must be [B, H_q, D] or [B, N, H_q, D], got {tuple(q.shape)}")
    q4 = q.unsqueeze(1) if q.dim() == 3 else q
    b, new, hq, d = q4.shape
    dev, dt = q.device, q.dtype
    code = _lib.dtype_code(dt)
    if dev.type != "cuda":
        raise ValueError("cache_attention_mass runs on the GPU; q is on " + str(dev))
    _cache_ok("k_cache", k_cache)
    hkv = k_cache.shape[2]
    if k_cache.shape[3] != d:
        raise ValueError(f"head_dim mismatch: q {d}, cache {k_cache.shape[3]}")
    if d not in HEAD_DIMS:
        raise ValueError(f"head_dim {d} must be one of {HEAD_DIMS}")
    if hkv <= 0 or hq == 0 or hq % hkv != 0 or new == 0:
        raise ValueError(f"q {tuple(q.shape)} does not match {hkv} KV heads")
    if k_cache.dtype != dt:
        raise TypeError(f"dtype mismatch: q {dt}, k_cache {k_cache.dtype}")
    block_table, seqlen_kv, rows, page_size = _paged_args(block_table, seqlen_kv, k_cache, page_size, b, dev)
    width = block_table.shape[1]
    scale = _scale(d ** -0.5 if scale is None else scale)
    if mass is None:
        mass = torch.zeros((b, hkv, width * page_size), dtype=torch.float32, device=dev)
    else:
        _mass_ok(mass, b, hkv, width * page_size, dev)
    if b == 0 or width == 0:
        return mass
    q4 = _as_rows(q4)
    nbytes = _mass_workspace(b, new, hq, hkv, d, page_size, width)
    with _lib.on(dev):
        ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
        _lib.check(_lib.load().ti_cache_mass(
            q4.data_ptr(), q4.stride(0), q4.stride(1), q4.stride(2), k_cache.data_ptr(),
            block_table.data_ptr(), block_table.stride(0), seqlen_kv.data_ptr(), mass.data_ptr(),
            mass.stride(0), mass.stride(1), ws.data_ptr(), nbytes, b, new, hq, hkv, d, page_size,
            rows // page_size, width, scale, code,
            _lib.stream_handle(dev)))
    return mass


def evict_kvcache(k_cache: torch.Tensor, v_cache: torch.Tensor | None, mass: torch.Tensor,
                  block_table: torch.Tensor, seqlen_kv: torch.Tensor, new_block_table: torch.Tensor,
                  budget: int, page_size: int = 16, *, sinks: int = 0, recent: int = 0):
    """Keep at most ``budget`` tokens of every (sequence, KV head) and move them to a new block table.

    A sequence of ``n <= budget`` tokens keeps all of them. Otherwise the first ``sinks`` and the last
    ``recent`` tokens stay and the rest of the budget goes to the tokens of the greatest ``mass``, ties to
    the lowest position (NaN counts as least). Kept tokens keep their order. Heads of a sequence keep
    different tokens, all the same number.

    Args:
        k_cache, v_cache: one layer's ``[num_blocks, block_size, H_kv, D]`` caches, contiguous, updated in
            place; ``v_cache`` None for a latent cache
        mass: ``[B, H_kv, capacity >= W * page_size]`` float32, as ``cache_attention_mass`` makes it
        block_table: ``[B, W]`` int32, every block below ``seqlen_kv`` in the cache
        seqlen_kv: ``[B]`` int32
        new_block_table: ``[B, W2]`` int32 with room for ``min(budget, W * page_size)`` tokens where a
            sequence has them (-1 beyond a sequence's kept tokens). Its blocks must be fresh: in no table
            that is still used, this call's ``block_table`` among them.
        budget, sinks, recent: host ints, ``sinks + recent <= budget < 2^31``
    Returns:
        ``(seqlen, kept, mass)``: the new lengths ``[B]`` int32, the kept positions ``[B, H_kv, budget]`` int32
        (ascending, -1 behind the last) and their masses ``[B, H_kv, capacity]`` (0 behind the last).
    """
    # The call in its common form is checked and made in native code; None: another form, or one to refuse.
    stream = _lib.native(k_cache)
    if stream is not None:
        r = _lib.result(_lib.calls().evict(k_cache, v_cache, mass, block_table, seqlen_kv, new_block_table, budget,
                                           page_size, sinks, recent, stream))
        if r is not None:
            return r
    _cache_ok("k_cache", k_cache)
    dev, dt = k_cache.device, k_cache.dtype
    code = _lib.dtype_code(dt)
    if dev.type != "cuda":
        raise ValueError("evict_kvcache runs on the GPU; k_cache is on " + str(dev))
    _, _, hkv, d = k_cache.shape
    if hkv == 0 or d == 0 or d % 8:
        raise ValueError(f"k_cache {tuple(k_cache.shape)}: needs heads of a multiple of 8 values")
    if v_cache is not None:
        _cache_ok("v_cache", v_cache)
        if v_cache.shape != k_cache.shape or v_cache.dtype != dt or v_cache.device != dev:
            raise ValueError("v_cache must have k_cache's shape, dtype and device")
    budget, sinks, recent = int(budget), int(sinks), int(recent)
    if not 0 < budget <= _lib.INT32_MAX or sinks < 0 or recent < 0 or sinks + recent > budget:
        raise ValueError(f"budget {budget} must be positive, below 2^31 and hold sinks {sinks} and recent {recent}")
    if block_table.dim() != 2:
        raise ValueError(f"block_table must be [B, W], got {tuple(block_table.shape)}")
    b = block_table.shape[0]
    block_table, seqlen_kv, rows, page_size = _paged_args(block_table, seqlen_kv, k_cache, page_size, b, dev)
    width = block_table.shape[1]
    if new_block_table.dtype != torch.int32 or new_block_table.device != dev:
        raise ValueError(f"new_block_table must be int32 on {dev}")
    if new_block_table.dim() != 2 or new_block_table.shape[0] != b:
        raise ValueError(f"new_block_table must be [{b}, W], got {tuple(new_block_table.shape)}")
    if new_block_table.stride(-1) != 1:
        new_block_table = new_block_table.contiguous()
    _mass_ok(mass, b, hkv, width * page_size, dev)
    capacity = mass.shape[2]
    kept = torch.empty((b, hkv, budget), dtype=torch.int32, device=dev)
    new_seqlen = torch.empty(b, dtype=torch.int32, device=dev)
    new_mass = torch.empty((b, hkv, capacity), dtype=torch.float32, device=dev)
    if b == 0:
        return new_seqlen, kept, new_mass
    with _lib.on(dev):
        _lib.check(_lib.load().ti_evict_kvcache(
            k_cache.data_ptr(), None if v_cache is None else v_cache.data_ptr(), mass.data_ptr(),
            mass.stride(0), mass.stride(1), capacity, block_table.data_ptr(), block_table.stride(0),
            seqlen_kv.data_ptr(), new_block_table.data_ptr(), new_block_table.stride(0), kept.data_ptr(),
            new_seqlen.data_ptr(), new_mass.data_ptr(), b, hkv, d, page_size, rows // page_size, width,
            new_block_table.shape[1], budget, sinks, recent, code, _lib.stream_handle(dev)))
    return new_seqlen, kept, new_mass
