"""What a program does around the latent and eviction calls: a chunk over cached tokens from the pages, weights whose
rotation pairs neighbours, and decoding on after a cut with positions and cached rows counted apart."""
import pytest
import torch

from helpers import say
from oracle import ref_latent as ref
from tileinfer_amd.engine.kv_layout import allocate_latent_cache, latent_layer_views
from tileinfer_amd.kernels import (cache_attention_mass, evict_kvcache, gqa_decode_paged_fn, latent_prefill_fn,
                                   latent_rope_append, qknorm_rope_append)

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def test_chunks_over_cached_tokens_from_the_pages(dev):
    """Packed keys and values of several sequences from their cached rows: one gather, one product, one call."""
    say("latent chunk over cached tokens")
    heads, d, latent = 6, 128, 512
    q_lens, k_lens = [37, 1, 130], [100, 33, 130]
    cache = allocate_latent_cache(2, 40, 16, latent, device=dev)
    cache.copy_(torch.randn(cache.shape, generator=_gen(1)))
    rows, _ = latent_layer_views(cache, 1)
    tables = torch.randperm(40, generator=_gen(2))[:27].view(3, 9).to(torch.int32).to(dev)
    w_kv = (torch.randn(latent, heads * 2 * d, generator=_gen(3)) * latent ** -0.5).to(BF16).to(dev)
    q = torch.randn(sum(q_lens), heads, d + 64, generator=_gen(4)).to(BF16).to(dev)
    cu_q, cu_k = (torch.tensor([0] + x, device=dev).cumsum(0).to(torch.int32) for x in (q_lens, k_lens))

    pos = torch.cat([torch.arange(n, device=dev) for n in k_lens])
    seq = torch.arange(3, device=dev).repeat_interleave(torch.tensor(k_lens, device=dev))
    cached = rows[tables[seq, pos // 16].long() * 16 + pos % 16]
    kv = (cached[:, :latent] @ w_kv).view(-1, heads, 2 * d)
    out = latent_prefill_fn(q, kv, cached[:, latent:], cu_q, cu_k, max(q_lens))

    every = []
    for b, n in enumerate(k_lens):
        every += [cache[1, tables[b, t // 16], t % 16, 0] for t in range(n)]
    assert torch.equal(cached, torch.stack(every))
    exact, limit = ref.latent_prefill(q.cpu(), kv.cpu(), cached[:, latent:].cpu(), cu_q.tolist(), cu_k.tolist(), 192 ** -0.5)
    assert ((out.double().cpu() - exact).abs() <= limit).all()


def test_weights_whose_rotation_pairs_neighbours(dev):
    """Columns in the order 0, 2, .. 62, 1, 3, .. 63 of the rotated parts' projections turn neighbours into the halves
    that the call rotates; the scores are those of the neighbours' rotation."""
    say("latent rotation of neighbours")
    t, heads = 7, 5
    pairs = torch.cat([torch.arange(0, 64, 2), torch.arange(1, 64, 2)])
    q = torch.randn(t, heads, 64, generator=_gen(5)).to(BF16)
    k = torch.randn(t, 64, generator=_gen(6)).to(BF16)
    angle = torch.rand(t, 32, generator=_gen(7)) * 6.28
    cos, sin = angle.cos().to(BF16), angle.sin().to(BF16)

    def neighbours(x, c, s):
        a, b, c, s = x[..., 0::2].double(), x[..., 1::2].double(), c.double(), s.double()
        return torch.stack([a * c - b * s, b * c + a * s], -1).flatten(-2)

    want = torch.einsum("thd,sd->ths", neighbours(q, cos[:, None], sin[:, None]), neighbours(k, cos, sin))
    cache = torch.zeros(t, 320, dtype=BF16, device=dev)
    both = [torch.cat([x, x], -1).to(dev) for x in (cos, sin)]
    got_q = latent_rope_append(q[..., pairs].to(dev), torch.zeros(t, 256, dtype=BF16, device=dev), k[:, pairs].to(dev),
                               torch.zeros(256, dtype=BF16, device=dev), *both, cache,
                               torch.arange(t, dtype=torch.int32, device=dev)).double().cpu()
    got = torch.einsum("thd,sd->ths", got_q, cache[:, 256:].double().cpu())
    # each rotated value is rounded once, 2^-8 of it at most: 2^-7 (and its square) of the sum of the products' sizes
    size = torch.einsum("thd,sd->ths", got_q.abs(), cache[:, 256:].double().abs().cpu())
    assert ((got - want).abs() <= 2.02 * 2.0 ** -8 * size).all()


def test_decoding_goes_on_after_two_cuts(dev):
    """The rotation counts every token seen, slots and lengths count the cached rows; running sums stay with their rows."""
    say("decode over two cuts")
    b, hq, hkv, d, page, budget = 2, 8, 2, 128, 16, 40
    blocks = 40
    k, v = (torch.randn(blocks, page, hkv, d, generator=_gen(i)).to(BF16).to(dev) for i in (8, 9))
    free = list(range(blocks))

    def take(n):
        return [[free.pop() for _ in range(n)] for _ in range(b)]

    tables = torch.tensor(take(5), dtype=torch.int32, device=dev)
    lens = torch.tensor([70, 33], dtype=torch.int32, device=dev)
    positions = lens.clone()
    ones = torch.zeros(d, dtype=BF16, device=dev)
    freq = 1e4 ** (-torch.arange(32, device=dev) / 32)
    g = _gen(10)
    # What is cached, host side: (K, V, sum) of every row in order, for each (sequence, head).
    rows = lambda i, h, n, x: x[tables[i, torch.arange(n, device=dev) // page].long(), torch.arange(n, device=dev) % page, h]  # noqa: E731
    held = {(i, h): (rows(i, h, int(lens[i]), k).cpu(), rows(i, h, int(lens[i]), v).cpu(), torch.zeros(int(lens[i])).double())
            for i in range(b) for h in range(hkv)}
    mass = torch.zeros(b, hkv, 6 * page, device=dev)
    spread = 0.0  # a step's weights are off by their 32-bit scores: twice (D + 4) 2^-24 of |q| |k| scale, up to about 14
    for step in range(24):
        if step in (4, 19):
            new_tables = torch.tensor(take(4), dtype=torch.int32, device=dev)
            lens, kept, mass = evict_kvcache(k, v, mass, tables, lens, new_tables, budget, page, sinks=2, recent=6)
            assert lens.tolist() == [min(budget, len(held[i, 0][0])) for i in range(b)]
            for (i, h), x in held.items():
                at = kept[i, h, :int(lens[i])].cpu().long()
                held[i, h] = tuple(y[at] for y in x)
            tables = new_tables
        lens = lens + 1
        angle = positions[:, None] * freq
        cos, sin = (torch.cat([f(angle)] * 2, -1).to(BF16) for f in (torch.cos, torch.sin))
        slots = tables.gather(1, ((lens - 1) // page).long()[:, None])[:, 0] * page + (lens - 1) % page
        q, k1, v1 = (torch.randn(b, n, d, generator=g).to(BF16).to(dev) for n in (hq, hkv, hkv))
        q = qknorm_rope_append(q, k1, v1, ones, ones, cos, sin, k.view(-1, hkv * d), v.view(-1, hkv * d), slots)
        positions = positions + 1
        out = gqa_decode_paged_fn(q, k, v, tables, lens, page).double().cpu()
        mass = cache_attention_mass(q, k, tables, lens, page, mass=mass)
        spread += 2.0 ** -12
        for (i, h), x in held.items():
            at = slots[i].item()
            kk = torch.cat([x[0], k.view(-1, hkv, d)[at, h][None].cpu()])
            vv = torch.cat([x[1], v.view(-1, hkv, d)[at, h][None].cpu()])
            assert torch.equal(vv[-1], v1[i, h].cpu())
            mine = q[i, h * (hq // hkv):(h + 1) * (hq // hkv)].cpu()
            seen = torch.ones(hq // hkv, len(kk), dtype=torch.bool)
            exact, limit = ref.attend(mine, kk, vv, d ** -0.5, seen, BF16)
            assert ((out[i, h * (hq // hkv):(h + 1) * (hq // hkv)] - exact).abs() <= limit).all(), step
            p, _ = ref.softmax_rows(mine, kk, d ** -0.5, seen)
            sums = torch.cat([x[2], torch.zeros(1).double()]) + p.sum(0)
            held[i, h] = (kk, vv, sums)
            n = int(lens[i])
            assert n == len(kk) and (mass[i, h, n:] == 0).all()
            torch.testing.assert_close(mass[i, h, :n].double().cpu(), sums, rtol=spread, atol=1e-7)
    assert positions.tolist() == [94, 57]
