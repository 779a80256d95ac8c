"""Latent, mass and eviction calls on caches and operands whose offsets pass 2^31 elements (4 GiB and more), against the
same call on a small cache that holds the same rows."""
import pytest
import torch

from helpers import bits, say
from oracle import ref_latent as ref
from tileinfer_amd.kernels import (cache_attention_mass, evict_kvcache, latent_decode_paged_fn, latent_prefill_fn,
                                   latent_rope_append)

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def _randn(dev, *shape, seed=0):
    return torch.randn(*shape, device=dev, generator=torch.Generator(dev).manual_seed(seed)).to(BF16)


def _pool(dev, heads, d, held):
    """(blocks of a cache whose last ones lie behind 2^31 elements, the ids of `held` of them at its end)."""
    blocks = 2 ** 31 // (16 * heads * d) + 40 + held
    pool = torch.empty(blocks, 16, heads, d, dtype=BF16, device=dev)
    ids = torch.arange(blocks - held, blocks, dtype=torch.int32, device=dev).flip(0)
    assert int(ids.min()) * 16 * heads * d > 2 ** 31
    return pool, ids


@pytest.mark.parametrize("latent", [256, 512])
def test_a_latent_cache_behind_2_31_elements(latent, dev):
    say(f"latent large pool L={latent}")
    row = latent + 64
    pool, ids = _pool(dev, 1, row, 40)
    small = _randn(dev, 40, 16, 1, row)
    pool[ids.long()] = small
    table = torch.arange(30, dtype=torch.int32, device=dev).view(3, 10)
    new = torch.arange(30, 36, dtype=torch.int32, device=dev).view(3, 2)
    big, big_new = ids[table.long()], ids[new.long()]
    lens = torch.tensor([160, 31, 100], dtype=torch.int32, device=dev)
    slots = torch.tensor([9 * 16 + 15, 39 * 16, 38 * 16 + 7], device=dev)
    big_slots = (ids[slots // 16].long() * 16 + slots % 16).to(torch.int32)
    c, kr, w, angle = _randn(dev, 3, latent), _randn(dev, 3, 64, seed=1), _randn(dev, latent, seed=2), _randn(dev, 3, 64, seed=3)
    latent_rope_append(None, c, kr, w, angle, angle, small.view(-1, row), slots.to(torch.int32))
    latent_rope_append(None, c, kr, w, angle, angle, pool.view(-1, row), big_slots)
    assert torch.equal(bits(pool[ids.long()]), bits(small))
    q = _randn(dev, 3, 2, 24, row, seed=4)
    assert torch.equal(bits(latent_decode_paged_fn(q, pool, big, lens, scale=0.05)),
                       bits(latent_decode_paged_fn(q, small, table, lens, scale=0.05)))
    mass = cache_attention_mass(q, small, table, lens, scale=0.05)
    assert torch.equal(cache_attention_mass(q, pool, big, lens, scale=0.05), mass)
    one = q[:, 0, :16]
    assert torch.equal(cache_attention_mass(one, pool, big, lens, scale=0.05),
                       cache_attention_mass(one, small, table, lens, scale=0.05))
    for a, b in zip(evict_kvcache(pool, None, mass, big, lens, big_new, 32, sinks=2, recent=3),
                    evict_kvcache(small, None, mass, table, lens, new, 32, sinks=2, recent=3)):
        assert torch.equal(a, b)
    assert torch.equal(bits(pool[ids.long()]), bits(small))


def test_a_kv_cache_behind_2_31_elements(dev):
    """Rows move from behind 2^31 elements to the front, by running sums whose sequences lie as far apart."""
    say("mass and eviction, large pool")
    pool, ids = _pool(dev, 4, 256, 16)
    values = torch.empty_like(pool)
    k, v = _randn(dev, 20, 16, 4, 256), _randn(dev, 20, 16, 4, 256, seed=1)
    pool[ids.long()], values[ids.long()] = k[:16], v[:16]
    table, new = torch.arange(16, dtype=torch.int32, device=dev).view(2, 8), torch.tensor([[16, 17], [18, 19]], dtype=torch.int32, device=dev)
    big, big_new = ids[table.long()], new - 16
    lens = torch.tensor([128, 77], dtype=torch.int32, device=dev)
    far = torch.empty(2 ** 31 + 1024, dtype=torch.float32, device=dev)
    sums = far.as_strided((2, 4, 128), (2 ** 31, 128, 1)).zero_()
    for n in (1, 5):
        q = _randn(dev, 2, n, 24, 256, seed=n)
        near = torch.zeros(2, 4, 128, device=dev)
        sums.zero_()
        cache_attention_mass(q, k, table, lens, mass=near)
        cache_attention_mass(q, pool, big, lens, mass=sums)
        assert torch.equal(sums, near)
    for a, b in zip(evict_kvcache(pool, values, sums, big, lens, big_new, 32, recent=3),
                    evict_kvcache(k, v, near, table, lens, new, 32, recent=3)):
        assert torch.equal(a, b)
    assert torch.equal(bits(pool[:4]), bits(k[16:])) and torch.equal(bits(values[:4]), bits(v[16:]))


def test_prefill_operands_behind_2_31_elements(dev):
    say("latent prefill, large operands")
    heads, d, total_q, total_k, n, m = 128, 128, 100000, 70000, 300, 1000
    q = torch.empty(total_q, heads, d + 64, dtype=BF16, device=dev)
    kv = torch.empty(total_k, heads, 2 * d, dtype=BF16, device=dev)
    kr = torch.empty(total_k, 64, dtype=BF16, device=dev)
    q[-n:], kv[-m:], kr[-m:] = _randn(dev, n, heads, d + 64), _randn(dev, m, heads, 2 * d, seed=1), _randn(dev, m, 64, seed=2)
    cu_q = torch.tensor([0, total_q - n, total_q - n, total_q], dtype=torch.int32, device=dev)
    cu_k = torch.tensor([0, 0, total_k - m, total_k], dtype=torch.int32, device=dev)
    out = latent_prefill_fn(q, kv, kr, cu_q, cu_k, total_q - n)
    assert out.numel() > 1.5 * 2 ** 30 and q.numel() > 2 ** 31 and kv.numel() > 2 ** 31
    assert not out[:-n].any()
    some = [0, 50, 127]
    exact, limit = ref.latent_prefill(q[-n:, some].cpu(), kv[-m:, some].cpu(), kr[-m:].cpu(), [0, n], [0, m], 192 ** -0.5)
    got = out[-n:, some].double().cpu()
    assert torch.isfinite(got).all() and ((got - exact).abs() <= limit).all()
