"""Plain 64-bit forms of rotation by several position axes, of attention with shaped scores (drafted trees, capped,
biased and masked prefill) and of moving accepted drafts, from their formulas, with elementwise limits on how far a
kernel may be off that count its roundings."""
from __future__ import annotations

import torch

from .ref_latent import half_step, rows_of


def rope_axes(x, positions, inv_freq, axes, weight=None, eps: float = 1e-5, offset: float = 1.0):
    """(rows, limit) of x [T, H, D]: norm where there is a weight, rotation of the pairs (i, i + half). positions
    [A, T]. The limit: statistics, factor and rotation in 32 bits (a dozen roundings of terms no larger than the row's
    pair; the sine and cosine of a fraction of a turn rounded to 32 bits are off by 2 pi 2^-25 and their own last bits,
    2^-22 together), one rounding to x's type."""
    half = inv_freq.numel()
    y = x.double()
    if weight is not None:
        y = y / torch.sqrt(y.square().mean(-1, keepdim=True) + eps) * (offset + weight.double())
    axes = [0] * half if axes is None else [min(max(int(a), 0), positions.shape[0] - 1) for a in axes]
    angle = torch.stack([positions[a].double() for a in axes], 1) * inv_freq.double() if half else torch.zeros(
        x.shape[0], 0).double()
    c, s = angle.cos()[:, None], angle.sin()[:, None]
    a, b = y[..., :half], y[..., half:2 * half]
    out = torch.cat([a * c - b * s, b * c + a * s, y[..., 2 * half:]], -1)
    size = torch.cat([a.abs() + b.abs(), a.abs() + b.abs(), y[..., 2 * half:].abs()], -1)
    # Statistics of D squares in 32 bits: relative D 2^-24 of a sum, half of it in its root.
    rel = 2.0 ** -21 + (x.shape[-1] * 2.0 ** -24 if weight is not None else 0.0)
    return out, rel * size + half_step(x.dtype) * out.abs() + torch.finfo(x.dtype).smallest_normal * half_step(x.dtype) * 2


def attend(q, k, v, seen, dist, scale: float, cap: float, slope: float, dtype):
    """(output, limit) [R, D] of one head: q [R, D], k, v [n, D], seen, dist [R, n].

    A score may be off by its sum of D products and its scaling in 32 bits, a capped one by the last bits of an
    exponential and a reciprocal (cap 2^-20), a biased one by the slope's, the product's and the sum's rounding and
    that of the exponential's argument (2^-21 of the bias); the weights are rounded to ``dtype`` before the product with
    v, their 32-bit sums over n keys are off likewise, and the output is rounded once."""
    q, k = q.double(), k.double()
    any_seen = seen.any(0)[:, None]
    k = torch.where(any_seen, k, torch.zeros_like(k))
    s = q @ k.t() * scale
    off = (q.shape[1] + 4) * 2.0 ** -24 * ((q.abs() @ k.abs().t()) * scale)
    if cap:
        s = cap * torch.tanh(s / cap)
        off = off + cap * 2.0 ** -20
    if slope:
        bias = slope * dist.double().abs()
        s = s - bias
        off = off + bias.abs() * 2.0 ** -21
    p = torch.softmax(s.masked_fill(~seen, -torch.inf), -1).nan_to_num(0.0)
    # Keys that weigh nothing cannot move the others: their scores' errors do not count.
    off = torch.where(seen & (p > 2.0 ** -60), off, torch.zeros_like(off)).amax(-1, keepdim=True) if k.shape[0] else \
        torch.zeros(q.shape[0], 1).double()
    v = torch.where(any_seen, v.double(), torch.zeros_like(v.double()))
    out, size = p @ v, p @ v.abs()
    h = half_step(dtype)
    rel = h + 2 * off + (k.shape[0] + 16) * 2.0 ** -23
    small = 2.0 ** -24 if dtype == torch.float16 else 0.0  # fp16 weights below 2^-14, of a row whose greatest is at least 1
    return out, rel * size + h * out.abs() + small * v.abs().sum(0) + torch.finfo(dtype).smallest_normal


def _cached(cache, table, n: int, page: int):
    """(rows [n, H, D] with zeros where absent, existing [n]) of a sequence's first n tokens."""
    flat = cache.reshape(-1, *cache.shape[2:])
    rows, there = rows_of(table.tolist(), page, flat.shape[0] // page, n)
    x = flat[rows].double()
    return torch.where(there[:, None, None], x, torch.zeros_like(x)), there


def tree(q, k_cache, v_cache, table, lens, masks, page: int, scale: float, cap: float = 0.0, slopes=None,
         window: int = 0):
    """(output, limit) [B, N, Hq, D]. masks: [B][N] Python ints, or None for chains."""
    b, n, hq, d = q.shape
    group = hq // k_cache.shape[2]
    out, limit = torch.zeros(q.shape).double(), torch.zeros(q.shape).double()
    for i in range(b):
        m = max(0, min(int(lens[i]), table.shape[1] * page))
        k, there = _cached(k_cache, table[i], m, page)
        v, _ = _cached(v_cache, table[i], m, page)
        context = m - n
        row = [(1 << (j + 1)) - 1 for j in range(n)] if masks is None else [int(x) & ((1 << n) - 1) for x in masks[i]]
        depth = [bin(x & ~(1 << j)).count("1") for j, x in enumerate(row)]
        seen, dist = torch.zeros(n, m, dtype=torch.bool), torch.zeros(n, m, dtype=torch.long)
        for j in range(n):
            t = torch.arange(m)
            draft = t - context
            at = torch.where(draft < 0, t, context + torch.tensor(depth)[draft.clamp(0, n - 1)])
            dist[j] = context + depth[j] - at
            bits = torch.tensor([(row[j] >> x) & 1 for x in range(n)], dtype=torch.bool)
            seen[j] = there & ((draft < 0) | bits[draft.clamp(0, n - 1)])
            if window:
                seen[j] &= dist[j] < window
        for h in range(hq):
            out[i, :, h], limit[i, :, h] = attend(q[i, :, h], k[:, h // group], v[:, h // group], seen, dist, scale, cap,
                                                  0.0 if slopes is None else float(slopes[h]), q.dtype)
    return out, limit


def prefill(q, k_cache, v_cache, table, cu_q, lens, page: int, scale: float, causal: bool = True, cap: float = 0.0,
            slopes=None, window: int = 0, first=None, last=None):
    """(output, limit) [total_q, Hq, D]."""
    group = q.shape[1] // k_cache.shape[2]
    out, limit = torch.zeros(q.shape).double(), torch.zeros(q.shape).double()
    for i in range(len(cu_q) - 1):
        a, e = int(cu_q[i]), int(cu_q[i + 1])
        m = max(0, min(int(lens[i]), table.shape[1] * page))
        k, there = _cached(k_cache, table[i], m, page)
        v, _ = _cached(v_cache, table[i], m, page)
        position = (m - (e - a) + torch.arange(e - a))[:, None]
        key = torch.arange(m)[None]
        dist = position - key
        end = last[a:e].long()[:, None] if last is not None else position if causal else torch.full_like(position, m)
        seen = there[None] & (key <= end)
        if first is not None:
            seen &= key >= first[a:e].long()[:, None]
        if window:
            seen &= dist < window
        for h in range(q.shape[1]):
            out[a:e, h], limit[a:e, h] = attend(q[a:e, h], k[:, h // group], v[:, h // group], seen, dist, scale, cap,
                                                0.0 if slopes is None else float(slopes[h]), q.dtype)
    return out, limit


def keep(cache, table, lens, accepted, page: int, drafts: int):
    """(cache [planes, rows, ...] after the moves, new lengths)."""
    planes = cache.reshape(-1, cache.shape[-4] * cache.shape[-3], *cache.shape[-2:]).clone()
    rows = planes.shape[1]
    new = []
    for b, n in enumerate(lens.tolist()):
        context = n - drafts
        if context < 0:
            new.append(n)
            continue
        path, before = [], -1
        for a in accepted[b].tolist():
            if not before < a < drafts:
                break
            path.append(a)
            before = a

        def row(t):
            block = int(table[b, t // page]) if t // page < table.shape[1] else -1
            return block * page + t % page if 0 <= block < rows // page else None

        old = {a: planes[:, row(context + a)].clone() for a in path if row(context + a) is not None}
        for j, a in enumerate(path):
            if a in old and row(context + j) is not None:
                planes[:, row(context + j)] = old[a]
        new.append(context + len(path))
    return planes.reshape(cache.shape), torch.tensor(new, dtype=torch.int32)
