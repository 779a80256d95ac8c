"""Positions of several axes: the input side of a step of image, video and drafted tokens.

A token of an image or a video has a time, a height and a width; its rotation takes every frequency's angle
from one of them. ``rope_axes_append`` forms the angles from the integer positions themselves (no cos/sin tables
to build and read), normalises queries and keys where weights are given, rotates them, and writes keys and values
into the paged cache, in one launch. One axis is the ordinary case: positions that need no table, for instance
those of a drafted tree, whose tokens sit at the context's length plus their depth.

It stands beside ``qknorm_rope_append`` (cos/sin given, one position a token), with which it shares the layout of
its operands; unlike that call, which rounds the normalised row as the reference's fused kernel does, every value
here is rounded once. The reference has no positions of several axes.

The call runs on the current stream, allocates through torch's caching allocator only, reads no device value on
the host, and can be captured in a graph.
"""
from __future__ import annotations

import torch

from .. import _lib
from .latent_attention import _as_rows, _vec_rows

__all__ = ["rope_axes", "rope_axes_append"]

MAX_AXES = 4


def rope_axes(sections, *, interleaved: bool = False, device=None) -> torch.Tensor:
    """Axis of every frequency, int32 ``[sum(sections)]``, for ``rope_axes_append``.

    ``sections``: how many frequencies each axis has (for instance ``(24, 20, 20)`` for time, height and width).
    Plain: the first ``sections[0]`` belong to axis 0, the next to axis 1, and so on. ``interleaved``: of ``A``
    axes, axis ``a > 0`` has the frequencies ``a, a + A, a + 2 A, ..``, ``sections[a]`` of them; axis 0 has the rest.
    """
    sections = [int(n) for n in sections]
    if not 1 <= len(sections) <= MAX_AXES or min(sections) < 0:
        raise ValueError(f"sections must be 1 to {MAX_AXES} counts, got {sections}")
    total = sum(sections)
    if not interleaved:
        axes = [a for a, n in enumerate(sections) for _ in range(n)]
    else:
        axes = [0] * total
        for a, n in enumerate(sections[1:], 1):
            at = list(range(a, a + n * len(sections), len(sections)))
            if at and at[-1] >= total:
                raise ValueError(f"sections {sections} do not interleave: axis {a} needs frequency {at[-1]} of {total}")
            for i in at:
                axes[i] = a
    return torch.tensor(axes, dtype=torch.int32, device=device)


def rope_axes_append(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, positions: torch.Tensor,
                     inv_freq: torch.Tensor, axes: torch.Tensor | None, k_cache: torch.Tensor,
                     v_cache: torch.Tensor, slot_mapping: torch.Tensor, *, q_weight: torch.Tensor | None = None,
                     k_weight: torch.Tensor | None = None, eps: float = 1e-5, weight_offset: float = 1.0,
                     q_out: torch.Tensor | None = None) -> torch.Tensor:
    """Input side of one step in one launch; returns the (normalised and) rotated ``q``.

    Args:
        q: ``[T, H_q, D]``, k, v ``[T, H_kv, D]``, D 128 or 256, any strides (for instance slices of one
            projection)
        positions: ``[A, T]`` (A 1 to 4) or ``[T]``, int32 or int64
        inv_freq: ``[rotary_dim / 2]`` float32; rotary_dim a multiple of 16, at most D. Frequency ``i``
            turns the pair ``(i, i + rotary_dim / 2)`` of every query and key head
        axes: ``[rotary_dim / 2]`` int32, the axis of every frequency (``rope_axes``; entries outside ``0 .. A - 1``
            are clamped); None: axis 0
        k_cache, v_cache: the layer's cache rows ``[num_slots, H_kv * D]`` (the views ``store_kvcache`` takes),
            16-byte aligned
        slot_mapping: ``[T]`` int32, slots outside the cache are skipped, duplicates unsupported
        q_weight, k_weight: ``[D]``, both or neither: RMSNorm of every head, factor ``weight_offset + weight``
            (1 as in ``qknorm_rope``, 0 for weights that are the whole factor)
        q_out: ``[T, H_q, D]`` for the result; it may be ``q`` itself
    Angles are formed in 64 bits: position 10^6 is as exact as position 10. Values past rotary_dim are only
    normalised.
    """
    # The call in its common form is checked and made in native code; None: another form, or one to refuse.
    stream = None if q_out is not None else _lib.native(q)
    if stream is not None:
        r = _lib.result(_lib.calls().rope_axes_append(q, k, v, positions, inv_freq, axes, k_cache, v_cache, slot_mapping,
                                                      q_weight, k_weight, eps, weight_offset, stream))
        if r is not None:
            return r
    if q.dim() != 3 or k.dim() != 3 or v.dim() != 3:
        raise ValueError("q, k, v must be [T, heads, D]")
    t, hq, d = q.shape
    dev, dt = q.device, q.dtype
    code = _lib.dtype_code(dt)
    if dev.type != "cuda":
        raise ValueError("rope_axes_append runs on the GPU; q is on " + str(dev))
    if k.shape[0] != t or v.shape != k.shape or k.shape[2] != d:
        raise ValueError(f"k {tuple(k.shape)} / v {tuple(v.shape)} do not match q {tuple(q.shape)}")
    hkv = k.shape[1]
    if d not in (128, 256):
        raise ValueError(f"head_dim {d} must be 128 or 256")
    if hq == 0 or hkv == 0:
        raise ValueError(f"q {tuple(q.shape)} / k {tuple(k.shape)} have no heads")
    if inv_freq.dim() != 1 or inv_freq.dtype != torch.float32:
        raise ValueError(f"inv_freq must be [rotary_dim / 2] float32, got {tuple(inv_freq.shape)} {inv_freq.dtype}")
    half = inv_freq.shape[0]
    if half % 8 or 2 * half > d:
        raise ValueError(f"rotary_dim {2 * half} must be a multiple of 16 and at most {d}")
    if positions.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"positions must be int32 or int64, got {positions.dtype}")
    if positions.dim() == 1:
        positions = positions[None]
    if positions.dim() != 2 or positions.shape[1] != t or not 1 <= positions.shape[0] <= MAX_AXES:
        raise ValueError(f"positions must be [{t}] or [1 .. {MAX_AXES}, {t}], got {tuple(positions.shape)}")
    if axes is not None and (axes.shape != (half,) or axes.dtype != torch.int32):
        raise ValueError(f"axes must be [{half}] int32, got {tuple(axes.shape)} {axes.dtype}")
    if (q_weight is None) != (k_weight is None):
        raise ValueError("q_weight and k_weight are given both or not at all")
    for name, w in (("q_weight", q_weight), ("k_weight", k_weight)):
        if w is not None and (w.shape != (d,) or w.dtype != dt):
            raise ValueError(f"{name} must be [{d}] {dt}")
    if k_cache.dim() != 2 or v_cache.shape != k_cache.shape or k_cache.shape[1] != hkv * d:
        raise ValueError(f"caches must be [num_slots, {hkv * d}] rows")
    if v_cache.stride() != k_cache.stride() or k_cache.stride(0) < hkv * d or not (
            _vec_rows(k_cache) and _vec_rows(v_cache)):
        raise ValueError("k_cache and v_cache rows must be contiguous, apart, 16-byte aligned and at the same strides (a "
                         "cache is never copied)")
    if slot_mapping.dtype != torch.int32 or slot_mapping.shape != (t,):
        raise ValueError(f"slot_mapping must be [{t}] int32")
    for name, x in (("k", k), ("v", v), ("k_cache", k_cache), ("v_cache", v_cache)):
        if x.dtype != dt:
            raise TypeError(f"dtype mismatch: q {dt}, {name} {x.dtype}")
    for name, x in (("k", k), ("v", v), ("positions", positions), ("inv_freq", inv_freq), ("axes", axes),
                    ("q_weight", q_weight), ("k_weight", k_weight), ("k_cache", k_cache), ("v_cache", v_cache),
                    ("slot_mapping", slot_mapping)):
        if x is not None and x.device != dev:
            raise ValueError(f"{name} is on {x.device}, q on {dev}")
    if q_out is None:
        q_out = torch.empty((t, hq, d), dtype=dt, device=dev)
    elif q_out.shape != q.shape or q_out.dtype != dt or q_out.device != dev or not _vec_rows(q_out):
        raise ValueError("q_out must be a [T, H_q, D] tensor of q's dtype and device with 16-byte aligned rows")
    if t == 0:
        return q_out
    # Held until the launch: a copy freed before it is handed out again, for instance to the next copy.
    q, k, v = _as_rows(q), _as_rows(k), _as_rows(v)
    if positions.stride(1) != 1:
        positions = positions.contiguous()
    inv_freq, slot_mapping = inv_freq.contiguous(), slot_mapping.contiguous()
    axes = None if axes is None else axes.contiguous()
    if q_weight is not None:
        q_weight, k_weight = _as_rows(q_weight), _as_rows(k_weight)
    with _lib.on(dev):
        _lib.check(_lib.load().ti_rope_axes_append(
            q.data_ptr(), q.stride(0), q.stride(1), k.data_ptr(), k.stride(0), k.stride(1), v.data_ptr(),
            v.stride(0), v.stride(1), positions.data_ptr(), positions.stride(0), positions.element_size() * 8,
            inv_freq.data_ptr(), None if axes is None else axes.data_ptr(),
            None if q_weight is None else q_weight.data_ptr(), None if k_weight is None else k_weight.data_ptr(),
            float(weight_offset), q_out.data_ptr(), q_out.stride(0), q_out.stride(1), k_cache.data_ptr(),
            v_cache.data_ptr(), k_cache.stride(0), k_cache.shape[0], slot_mapping.data_ptr(), t, positions.shape[0],
            hq, hkv, d, 2 * half, float(eps), code, _lib.stream_handle(dev)))
    return q_out
