"""Plain 64-bit forms of latent attention, of the attention weight of cached tokens and of eviction, from
their formulas, with elementwise limits on how far a kernel may be off that count its roundings."""
from __future__ import annotations

import torch


def half_step(dtype: torch.dtype) -> float:
    """The largest relative error of one rounding to ``dtype``."""
    return torch.finfo(dtype).eps / 2


def rows_of(table, page: int, num_blocks: int, n: int):
    """(cache rows, existing) of a sequence's tokens 0 .. n - 1; a token whose block id is outside the cache
    does not exist."""
    rows, there = [], []
    for t in range(n):
        j = t // page
        block = int(table[j]) if j < len(table) else -1
        ok = 0 <= block < num_blocks
        rows.append(block * page + t % page if ok else 0)
        there.append(ok)
    return torch.tensor(rows, dtype=torch.long), torch.tensor(there, dtype=torch.bool)


def softmax_rows(q, k, scale: float, seen):
    """(weights, score error) of queries [R, E] over keys [n, E] in 64 bits. ``seen`` [R, n]. Rows that see
    nothing are zero. The error bounds a score that sums its E products and scales them in 32 bits."""
    q, k = q.double(), k.double()
    k = torch.where(seen.any(0)[:, None], k, torch.zeros_like(k))
    s = q @ k.t() * scale
    off = (q.shape[1] + 4) * 2.0 ** -24 * ((q.abs() @ k.abs().t()) * abs(scale))
    s = s.masked_fill(~seen, -torch.inf)
    p = torch.softmax(s, -1).nan_to_num(0.0)
    off = torch.where(seen, off, torch.zeros_like(off))
    return p, off.amax(-1, keepdim=True) if k.shape[0] else off.new_zeros((q.shape[0], 1))


def attend(q, k, v, scale: float, seen, dtype):
    """(output, limit) [R, Dv]: the weights are rounded to ``dtype`` before the product with v, each score may
    be off by its 32-bit sum (in the numerator and in the sum of the weights), the 32-bit sums over n keys
    likewise, and the output is rounded to ``dtype`` once."""
    p, off = softmax_rows(q, k, scale, seen)
    v = torch.where(seen.any(0)[:, None], v.double(), torch.zeros_like(v.double()))
    out, size = p @ v, p @ v.abs()
    h = half_step(dtype)
    tiny = torch.finfo(dtype).smallest_normal  # a weight below it has steps of its own
    rel = h + 2 * off + (k.shape[0] + 16) * 2.0 ** -23
    small = 2.0 ** -24 if dtype == torch.float16 else 0.0  # fp16 weights below 2^-14, of a row whose greatest is at least 1
    return out, rel * size + h * out.abs() + small * v.abs().sum(0) + tiny


def causal(q_len: int, k_len: int, there=None, is_causal: bool = True):
    """[q_len, k_len]: query i sees the existing keys j <= k_len - q_len + i."""
    j = torch.arange(k_len)
    seen = j[None] <= (k_len - q_len + torch.arange(q_len))[:, None] if is_causal else torch.ones(
        (q_len, k_len), dtype=torch.bool)
    return seen if there is None else seen & there[None]


def rotate(x, cos, sin):
    """Rotation of pairs (i, i + half) by each token's angle."""
    half = x.shape[-1] // 2
    x, c, s = x.double(), cos.double()[..., :half], sin.double()[..., :half]
    return torch.cat([x[..., :half] * c - x[..., half:] * s, x[..., half:] * c + x[..., :half] * s], -1)


def latent_rows(latent, key_rope, weight, cos, sin, eps: float, offset: float):
    """[T, L + R]: the cache rows of a latent layer's input side."""
    x = latent.double()
    x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps) * (offset + weight.double())
    return torch.cat([x, rotate(key_rope, cos, sin)], -1)


def latent_decode(q, cache, table, lens, page: int, scale: float):
    """(output, limit) [B, N, H, L] of the absorbed form. q [B, N, H, E], cache [nb, bs, 1, E]."""
    b, new, h, e = q.shape
    flat = cache.reshape(-1, e)
    blocks = flat.shape[0] // page
    out, limit = torch.zeros(b, new, h, e - 64).double(), torch.zeros(b, new, h, e - 64).double()
    for i in range(b):
        n = max(0, min(int(lens[i]), table.shape[1] * page))
        rows, there = rows_of(table[i].tolist(), page, blocks, n)
        k = torch.where(there[:, None], flat[rows].double(), torch.zeros(1).double())
        seen = causal(new, n, there)
        for x in range(h):
            out[i, :, x], limit[i, :, x] = attend(q[i, :, x], k, k[:, :e - 64], scale, seen, q.dtype)
    return out, limit


def latent_prefill(q, kv, key_rope, cu_q, cu_k, scale: float, is_causal: bool = True):
    """(output, limit) [total_q, H, D] of the expanded form."""
    d = q.shape[2] - 64
    out, limit = torch.zeros(q.shape[0], q.shape[1], d).double(), torch.zeros(q.shape[0], q.shape[1], d).double()
    for i in range(len(cu_q) - 1):
        a, b, c, e = int(cu_q[i]), int(cu_q[i + 1]), int(cu_k[i]), int(cu_k[i + 1])
        seen = causal(b - a, e - c, None, is_causal)
        for h in range(q.shape[1]):
            k = torch.cat([kv[c:e, h, :d], key_rope[c:e]], -1)
            out[a:b, h], limit[a:b, h] = attend(q[a:b, h], k, kv[c:e, h, d:], scale, seen, q.dtype)
    return out, limit


def attention_mass(q, k_cache, table, lens, page: int, scale: float):
    """(mass, limit) [B, H_kv, W * page]: summed softmax weights. Each weight is off by its score (and the
    sum's), 32-bit sums over n keys and the rows."""
    b, new, hq, d = q.shape
    hkv = k_cache.shape[2]
    flat = k_cache.reshape(-1, hkv, d)
    blocks = flat.shape[0] // page
    mass = torch.zeros(b, hkv, table.shape[1] * page).double()
    limit = torch.zeros_like(mass)
    for i in range(b):
        n = max(0, min(int(lens[i]), table.shape[1] * page))
        rows, there = rows_of(table[i].tolist(), page, blocks, n)
        seen = causal(new, n, there)
        for h in range(hq):
            g = h // (hq // hkv)
            k = torch.where(there[:, None], flat[rows, g].double(), torch.zeros(1).double())
            p, off = softmax_rows(q[i, :, h], k, scale, seen)
            mass[i, g, :n] += p.sum(0)
            limit[i, g, :n] += (p * (2 * off + (n + new * hq + 32) * 2.0 ** -23)).sum(0)
    return mass, limit + 2.0 ** -120


def evict(mass, lens, budget: int, sinks: int, recent: int):
    """(kept [B, H, budget] with -1 behind, new lengths) from their definition."""
    b, hkv, cap = mass.shape
    kept = torch.full((b, hkv, budget), -1, dtype=torch.int32)
    new = []
    for i in range(b):
        n = max(0, min(int(lens[i]), cap))
        new.append(min(n, budget))
        for h in range(hkv):
            def rank(t):
                always = t < sinks or t >= n - recent
                x = float(mass[i, h, t])
                return (0 if always else 1, 0 if always or x == x else 1, 0.0 if always or x != x else -x, t)
            keep = sorted(sorted(range(n), key=rank)[:budget]) if n > budget else list(range(n))
            kept[i, h, :len(keep)] = torch.tensor(keep, dtype=torch.int32)
    return kept, torch.tensor(new, dtype=torch.int32)
