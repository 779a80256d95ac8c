"""Latent and eviction calls as a serving loop mixes them: on two streams, captured, swapped, evicted and resumed."""
import pytest
import torch

from oracle import ref_latent as ref
from tileinfer_amd.engine.kv_layout import allocate_latent_cache, latent_layer_views
from tileinfer_amd.kernels import (cache_attention_mass, copy_blocks, evict_kvcache, latent_decode_paged_fn,
                                   latent_prefill_fn, latent_rope_append)

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


@pytest.fixture
def dev():
    return torch.device("cuda:0")


def _state(dev, seed, batch=3, blocks=64, latent=512, heads=24):
    g = torch.Generator().manual_seed(seed)
    cache = torch.randn(blocks, 16, 1, latent + 64, generator=g).to(BF16).to(dev)
    width = blocks // (2 * batch)
    table = torch.randperm(blocks, generator=g)[:batch * width].reshape(batch, width).to(torch.int32).to(dev)
    lens = torch.randint(1, width * 16 + 1, (batch,), generator=g).to(torch.int32).to(dev)
    q = torch.randn(batch, heads, latent + 64, generator=g).to(BF16).to(dev)
    return q, cache, table, lens


def test_two_streams_at_once(dev):
    """Calls that overlap on two streams have workspaces of their own."""
    states = [_state(dev, 1), _state(dev, 2, batch=5, latent=256, heads=32)]
    alone = []
    for q, cache, table, lens in states:
        alone.append((latent_decode_paged_fn(q, cache, table, lens, scale=0.06),
                      cache_attention_mass(q, cache, table, lens, scale=0.06)))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(8):
        got = []
        for s, (q, cache, table, lens) in zip(streams, states):
            with torch.cuda.stream(s):
                got.append((latent_decode_paged_fn(q, cache, table, lens, scale=0.06),
                            cache_attention_mass(q, cache, table, lens, scale=0.06)))
        torch.cuda.synchronize()
        for a, b in zip(alone, got):
            assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_two_graphs_of_one_step(dev):
    """Two captured steps (append, decode, mass) replayed in turn, with eager calls and changed inputs between."""
    heads, latent = 24, 512
    q, cache, table, lens = _state(dev, 3)
    rows = cache.view(-1, latent + 64)
    g = torch.Generator().manual_seed(4)
    new = torch.randn(3, latent + 64, generator=g).to(BF16).to(dev)
    angle = torch.randn(3, 32, generator=g)
    cos, sin = (torch.cat((f(angle), f(angle)), -1).to(BF16).to(dev) for f in (torch.cos, torch.sin))
    weight = torch.zeros(latent, dtype=BF16, device=dev)

    def step(at):
        slots = torch.gather(table, 1, ((lens - 1) // 16).long()[:, None])[:, 0] * 16 + (lens - 1) % 16
        latent_rope_append(None, new[:, :latent], new[:, latent:], weight, cos, sin, rows, slots)
        return latent_decode_paged_fn(q + at, cache, table, lens, scale=0.05), cache_attention_mass(
            q + at, cache, table, lens, scale=0.05)

    step(0.0)
    graphs = []
    for at in (0.0, 1.0):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            graphs.append((graph, step(at), at))
    for i in range(3):
        for graph, out, at in graphs:
            new.copy_(torch.randn(3, latent + 64, generator=g))
            graph.replay()
            torch.cuda.synchronize()
            kept = [x.clone() for x in out]
            for a, b in zip(kept, step(at)):
                assert torch.equal(a, b), (i, at)


def test_two_graphs_of_a_first_chunk(dev):
    """Captured prefills of every schedule (a unit each, two key groups, cut units) repeat the eager call."""
    g = torch.Generator().manual_seed(5)
    for tokens, heads in ((300, 2), (1100, 40), (300, 200)):
        q = torch.randn(tokens, heads, 128, generator=g).to(BF16).to(dev)
        kv = torch.randn(tokens, heads, 128, generator=g).to(BF16).to(dev)
        kr = torch.randn(tokens, 64, generator=g).to(BF16).to(dev)
        cu = torch.tensor([0, tokens], dtype=torch.int32, device=dev)
        graphs = []
        for _ in range(2):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                graphs.append((graph, latent_prefill_fn(q, kv, kr, cu, cu, tokens)))
        for _ in range(3):
            q.copy_(torch.randn(q.shape, generator=g))
            for graph, out in graphs:
                graph.replay()
                torch.cuda.synchronize()
                kept = out.clone()
                assert torch.equal(kept, latent_prefill_fn(q, kv, kr, cu, cu, tokens)), (tokens, heads)


def test_a_swapped_latent_cache_decodes_the_same(dev):
    """Blocks of a latent slab go to pinned memory and back to other blocks."""
    layers, blocks = 2, 24
    cache = allocate_latent_cache(layers, blocks, 16, 256, device=dev)
    cache.copy_(torch.randn(cache.shape, generator=torch.Generator().manual_seed(6)))
    table = torch.tensor([[3, 1, 7], [2, 9, 4]], dtype=torch.int32, device=dev)
    lens = torch.tensor([37, 48], dtype=torch.int32, device=dev)
    q = torch.randn(2, 16, 320, generator=torch.Generator().manual_seed(7)).to(BF16).to(dev)
    before = [latent_decode_paged_fn(q, latent_layer_views(cache, i)[1], table, lens, scale=0.1)
              for i in range(layers)]
    host = torch.empty((layers, 6, 16, 1, 320), dtype=BF16, pin_memory=True)
    old = table.reshape(-1).long()
    new = torch.tensor([20, 11, 15, 12, 23, 0], device=dev)
    there = torch.arange(6, device=dev)
    copy_blocks(cache, host, torch.stack((old, there), 1))
    torch.cuda.synchronize()
    cache[:, old] = 0
    copy_blocks(host, cache, torch.stack((there, new), 1))
    moved = new.to(torch.int32).reshape(2, 3)
    for i in range(layers):
        after = latent_decode_paged_fn(q, latent_layer_views(cache, i)[1], moved, lens, scale=0.1)
        assert torch.equal(after, before[i])


@pytest.mark.parametrize("latent", [256, 512])
def test_a_cut_latent_cache_goes_on(latent, dev):
    """Mass over a window, cut, append to the cut sequence, decode: the formula over the kept rows and the new one."""
    q, cache, table, lens = _state(dev, 8, batch=2, blocks=80, latent=latent)
    lens = torch.tensor([200, 9], dtype=torch.int32, device=dev)
    window = torch.randn(2, 4, 24, latent + 64, generator=torch.Generator().manual_seed(9)).to(BF16).to(dev)
    mass = cache_attention_mass(window, cache, table, lens, scale=0.05)
    used = set(table.reshape(-1).tolist())
    free = [i for i in range(80) if i not in used][:10]
    new_table = torch.tensor(free, dtype=torch.int32, device=dev).reshape(2, 5)
    n, kept, left = evict_kvcache(cache, None, mass, table, lens, new_table, 64, sinks=2, recent=4)
    assert n.tolist() == [64, 9]
    rows = cache.view(-1, latent + 64)
    for b in range(2):
        at = kept[b, 0, :n[b]].long()
        old = rows[table[b, at // 16].long() * 16 + at % 16]
        here = torch.arange(int(n[b]), device=dev)
        assert torch.equal(rows[new_table[b, here // 16].long() * 16 + here % 16], old)
        assert torch.equal(left[b, 0, :n[b]], mass[b, 0, at])
    n = n + 1
    slots = torch.gather(new_table, 1, ((n - 1) // 16).long()[:, None])[:, 0] * 16 + (n - 1) % 16
    token = torch.randn(2, latent + 64, generator=torch.Generator().manual_seed(10)).to(BF16).to(dev)
    one, none = torch.ones(64, dtype=BF16, device=dev), torch.zeros(64, dtype=BF16, device=dev)
    latent_rope_append(None, token[:, :latent], token[:, latent:], torch.zeros(latent, dtype=BF16, device=dev),
                       one, none, rows, slots)
    assert torch.equal(rows[slots.long(), latent:], token[:, latent:])
    out = latent_decode_paged_fn(q, cache, new_table, n, scale=0.05)
    exact, limit = ref.latent_decode(q[:, None].cpu(), cache.cpu(), new_table.cpu(), n.cpu(), 16, 0.05)
    assert ((out.double().cpu()[:, None] - exact).abs() <= limit).all()
