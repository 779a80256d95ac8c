"""Attention weight of cached tokens and eviction by it, against their 64-bit forms."""
import pytest
import torch

from helpers import bits, say
from oracle import ref_latent as ref
from tileinfer_amd.kernels import cache_attention_mass, evict_kvcache, gqa_decode_paged_fn

pytestmark = pytest.mark.gpu
BF16, F16 = torch.bfloat16, torch.float16


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _paged(lens, page, heads, d, dtype, seed, extra=3, width=None):
    """Caches whose unused rows are NaN, and tables of shuffled blocks with -1 behind."""
    g = _gen(seed)
    counts = [-(-max(n, 0) // page) for n in lens]
    blocks = sum(counts) + extra
    perm = torch.randperm(blocks, generator=g).tolist()
    width = width or max(max(counts), 1)
    table = torch.full((len(lens), width), -1, dtype=torch.int32)
    k = torch.full((blocks, page, heads, d), torch.nan).to(dtype)
    v = k.clone()
    at = 0
    for i, (n, c) in enumerate(zip(lens, counts)):
        table[i, :c] = torch.tensor(perm[at:at + c], dtype=torch.int32)
        at += c
        pos = torch.arange(n)
        for x in (k, v):
            x[table[i].long()[pos // page], pos % page] = torch.randn(n, heads, d, generator=g).to(dtype)
    return k, v, table, torch.tensor(lens, dtype=torch.int32), perm[at:]


def _close(out, exact, limit):
    out = out.double().cpu()
    assert torch.isfinite(out).all()
    worst = ((out - exact).abs() / limit).max().item()
    say(f"  worst error is {worst:.3f} of its limit")
    assert worst <= 1.0


MASSES = [
    # query heads, KV heads, head_dim, new tokens, page, dtype, lengths
    (24, 4, 256, 1, 16, BF16, [1, 130, 0, 700]),
    (32, 8, 128, 1, 8, F16, [1000, 3]),
    (4, 4, 256, 1, 1, BF16, [65]),
    (16, 1, 576, 1, 16, BF16, [300, 31]),
    (24, 1, 576, 2, 16, F16, [1, 150]),
    (32, 1, 320, 33, 24, BF16, [400, 20]),
    (12, 2, 256, 32, 16, BF16, [31, 32, 33, 600]),
    (32, 8, 128, 5, 4, F16, [257, 4]),
    (8, 8, 128, 17, 32, BF16, [64]),
]


@pytest.mark.parametrize("hq,hkv,d,new,page,dtype,lens", MASSES)
def test_mass_matches_formula(hq, hkv, d, new, page, dtype, lens, dev):
    say(f"mass {hq}/{hkv} D={d} N={new} page={page} {dtype} {lens}")
    k, _, table, n, _ = _paged(lens, page, hkv, d, dtype, 1)
    q = torch.randn(len(lens), new, hq, d, generator=_gen(2)).to(dtype)
    exact, limit = ref.attention_mass(q, k, table, n, page, d ** -0.5)
    args = [x.to(dev) for x in (q, k, table, n)]
    mass = cache_attention_mass(*args, page)
    assert mass.dtype == torch.float32 and mass.shape == (len(lens), hkv, table.shape[1] * page)
    _close(mass, exact, limit)
    for i, length in enumerate(lens):
        assert (mass[i, :, length:] == 0).all()
        seen = sum(1 for t in range(new) if length - new + t >= 0)
        total = mass[i].double().sum(-1).cpu()
        torch.testing.assert_close(total, torch.full_like(total, seen * hq / hkv), rtol=1e-4, atol=1e-6)
    assert torch.equal(mass, cache_attention_mass(*args, page))  # the same bits
    if new == 1:
        assert torch.equal(mass, cache_attention_mass(args[0][:, 0], *args[1:], page))


def test_mass_adds_to_running_sums(dev):
    """In place, in a larger strided buffer, what lies behind a sequence untouched; a captured call adds
    once per replay."""
    say("mass in place")
    k, _, table, n, _ = _paged([50, 7], 16, 2, 128, BF16, 3, width=5)
    q = torch.randn(2, 1, 8, 128, generator=_gen(4)).to(BF16)
    exact, limit = ref.attention_mass(q, k, table, n, 16, 0.3)
    buf = torch.full((2, 3, 100), 2.0, device=dev)
    mass = buf[:, :2]
    args = [x.to(dev) for x in (q, k, table, n)]
    r = cache_attention_mass(*args, 16, scale=0.3, mass=mass)
    assert r is mass
    _close(mass[..., :80] - 2.0, exact, limit + 2.0 ** -22)
    assert (buf[:, 2] == 2).all() and (mass[0, :, 50:] == 2).all() and (mass[1, :, 7:] == 2).all()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache_attention_mass(*args, 16, scale=0.3, mass=mass)
    eager = mass.clone()
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        cache_attention_mass(*args, 16, scale=0.3, mass=eager)
        assert torch.equal(eager, mass)


@pytest.mark.parametrize("new", [1, 9])
def test_mass_absent_blocks(new, dev):
    say(f"mass absent blocks N={new}")
    k, _, table, n, _ = _paged([70, 40], 8, 4, 128, BF16, 5, width=12)
    table[0, 3], table[0, 0] = -1, 10 ** 6
    table[1, :5] = -1
    q = (40 * torch.randn(2, new, 8, 128, generator=_gen(6))).to(BF16)
    exact, limit = ref.attention_mass(q, k, table, n, 8, 128 ** -0.5)
    mass = cache_attention_mass(*(x.to(dev) for x in (q, k, table, n)), 8)
    _close(mass, exact, limit)
    assert (mass[1] == 0).all()


EVICTS = [
    # KV heads, head_dim, page, dtype, lengths, budget, sinks, recent, latent
    (4, 256, 16, BF16, [1, 100, 0, 64, 65], 64, 4, 8, False),
    (8, 128, 8, F16, [300, 10], 33, 0, 0, False),
    (1, 576, 16, BF16, [6001], 100, 4, 32, True),
    (1, 320, 24, F16, [500, 99], 100, 50, 50, True),
    (2, 128, 1, BF16, [2500], 1, 0, 0, False),
    (2, 128, 16, BF16, [1500], 1, 1, 0, False),
    (2, 128, 16, BF16, [40, 41], 1000, 4, 4, False),
]


def _masses(shape, seed):
    """Few distinct values, so that ties cross the border; among them zeros of both signs and infinities."""
    m = (torch.rand(shape, generator=_gen(seed)).pow(6) * 40).round() / 8
    m.view(-1)[::7] *= -0.0
    m.view(-1)[3::101] = torch.inf
    return m


@pytest.mark.parametrize("hkv,d,page,dtype,lens,budget,sinks,recent,latent", EVICTS)
def test_evict_keeps_the_heaviest(hkv, d, page, dtype, lens, budget, sinks, recent, latent, dev):
    say(f"evict {hkv}x{d} page={page} {lens} -> {budget} ({sinks}, {recent})")
    most = max(min(n, budget) for n in lens)
    need = [-(-min(n, budget) // page) for n in lens]
    k, v, table, n, free = _paged(lens, page, hkv, d, dtype, 7, extra=sum(need) + 2)
    new_table = torch.full((len(lens), -(-min(budget, table.shape[1] * page) // page)), -1, dtype=torch.int32)
    at = 0
    for i, c in enumerate(need):
        new_table[i, :c] = torch.tensor(free[at:at + c], dtype=torch.int32)
        at += c
    mass = _masses((len(lens), hkv, table.shape[1] * page + 5), 8)
    kept, seqlen = ref.evict(mass[..., :table.shape[1] * page], n, budget, sinks, recent)
    kd, vd = k.to(dev), None if latent else v.to(dev)
    got_len, got_kept, got_mass = evict_kvcache(kd, vd, mass.to(dev), table.to(dev), n.to(dev), new_table.to(dev),
                                                budget, page, sinks=sinks, recent=recent)
    assert torch.equal(got_len.cpu(), seqlen)
    assert torch.equal(got_kept.cpu(), kept)
    for old, cache in ((k, kd), (v, vd)):
        if cache is None:
            continue
        want = old.clone()
        for i in range(len(lens)):
            c = int(seqlen[i])
            j = torch.arange(c)
            into = new_table[i].long()[j // page], j % page
            for h in range(hkv):
                t = kept[i, h, :c].long()
                want[into[0], into[1], h] = old[table[i].long()[t // page], t % page, h]
        assert torch.equal(bits(cache.cpu()), bits(want))  # the kept rows, and every other row as it was
    for i in range(len(lens)):
        c = int(seqlen[i])
        assert torch.equal(got_mass[i, :, :c].cpu(), mass[i].gather(-1, kept[i, :, :c].long()))
        assert (got_mass[i, :, c:] == 0).all()
    assert most >= 0


def test_evict_ranks_nan_last_and_takes_any_sign(dev):
    say("evict nan")
    k, v, table, n, free = _paged([40], 8, 1, 128, BF16, 9, extra=4)
    mass = torch.linspace(-3, 3, 40).view(1, 1, 40).clone()
    mass[0, 0, 20:] = torch.nan
    mass[0, 0, 5] = -torch.inf
    new_table = torch.tensor([free[:3]], dtype=torch.int32)
    kept, _ = ref.evict(mass, n, 22, 0, 0)
    _, got, _ = evict_kvcache(k.to(dev), v.to(dev), mass.to(dev), table.to(dev), n.to(dev), new_table.to(dev), 22, 8)
    assert torch.equal(got.cpu(), kept)


def test_evict_long_sequence_and_graph(dev):
    """A selection over 70,000 tokens of all-different and of all-equal masses; a captured call repeats."""
    say("evict long")
    g = _gen(10)
    page, n, budget = 16, 70000, 5001
    blocks = n // page
    k = torch.randn(blocks + 313, page, 1, 128, generator=g).to(BF16).to(dev)
    table = torch.arange(blocks, dtype=torch.int32, device=dev)[None]
    new_table = torch.arange(blocks, blocks + 313, dtype=torch.int32, device=dev)[None]
    lens = torch.tensor([n], dtype=torch.int32, device=dev)
    mass = torch.rand(1, 1, n, generator=g).to(dev)
    order = torch.sort(mass[0, 0], descending=True, stable=True).indices[:budget].sort().values
    _, kept, _ = evict_kvcache(k, None, mass, table, lens, new_table, budget, page)
    assert torch.equal(kept[0, 0].long(), order)
    rows = k.view(-1, 128)
    assert torch.equal(bits(rows[n:n + budget]), bits(rows[order]))
    _, kept, _ = evict_kvcache(k, None, torch.ones_like(mass), table, lens, new_table, budget, page, recent=10)
    want = torch.cat([torch.arange(budget - 10), torch.arange(n - 10, n)])
    assert torch.equal(kept[0, 0].cpu().long(), want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        _, g_kept, g_mass = evict_kvcache(k, None, mass, table, lens, new_table, budget, page)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(g_kept[0, 0].long(), order)
        assert torch.equal(g_mass[0, 0, :budget], mass[0, 0, order])


def test_decode_goes_on_over_the_kept_tokens(dev):
    """Steps that accumulate weight, an eviction, and the decode over the shorter table: the attention over
    exactly the kept tokens of each head."""
    say("evict and decode")
    page, hq, hkv, d, budget = 16, 24, 4, 256, 48
    lens = [200, 75]
    k, v, table, n, free = _paged(lens, page, hkv, d, BF16, 12, extra=6)
    kd, vd, td, nd = (x.to(dev) for x in (k, v, table, n))
    mass = None
    for step in range(3):
        q = (3 * torch.randn(2, hq, d, generator=_gen(20 + step))).to(BF16).to(dev)
        mass = cache_attention_mass(q, kd, td, nd, page, mass=mass)
    new_table = torch.tensor([free[:3], free[3:6]], dtype=torch.int32, device=dev)
    lens2, kept, _ = evict_kvcache(kd, vd, mass, td, nd, new_table, budget, page, sinks=2, recent=8)
    assert lens2.tolist() == [48, 48]
    q = torch.randn(2, hq, d, generator=_gen(30)).to(BF16)
    out = gqa_decode_paged_fn(q.to(dev), kd, vd, new_table, lens2, page).double().cpu()
    for i in range(2):
        for h in range(hq):
            g = h // (hq // hkv)
            t = kept[i, g].cpu().long()
            rows = table[i].long()[t // page], t % page
            seen = torch.ones(1, budget, dtype=torch.bool)
            exact, limit = ref.attend(q[i, h][None], k[rows[0], rows[1], g], v[rows[0], rows[1], g], d ** -0.5, seen, BF16)
            assert ((out[i, h] - exact[0]).abs() <= limit[0]).all()
