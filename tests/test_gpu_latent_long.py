"""Latent attention and attention mass at lengths that take more than one round of their inner loops: runs whose block
ids do not fit at once, rows with many parts, queries that fill every stage again."""
import pytest
import torch

from helpers import say
from oracle import ref_latent as ref
from tileinfer_amd.kernels import cache_attention_mass, latent_decode_paged_fn

pytestmark = pytest.mark.gpu
BF16, F16 = torch.bfloat16, torch.float16


def _pool(lens, page, heads, d, dtype, seed, dev, extra=3, width=None):
    """Random cache rows, tables of shuffled blocks with -1 behind, lengths; on the GPU."""
    g = torch.Generator(dev).manual_seed(seed)
    counts = [-(-n // page) for n in lens]
    blocks = sum(counts) + extra
    cache = torch.empty(blocks, page, heads, d, dtype=dtype, device=dev).normal_(generator=g)
    perm = torch.randperm(blocks, generator=g, device=dev, dtype=torch.int32)
    table = torch.full((len(lens), width or max(counts)), -1, dtype=torch.int32, device=dev)
    at = 0
    for i, c in enumerate(counts):
        table[i, :c] = perm[at:at + c]
        at += c
    return cache, table, torch.tensor(lens, dtype=torch.int32, device=dev)


def _check(got, exact, limit, what):
    got = got.double().cpu()
    assert torch.isfinite(got).all(), what
    worst = ((got - exact).abs() / limit).max().item()
    say(f"  {what}: worst error is {worst:.3f} of its limit")
    assert worst <= 1.0


PIECES = [
    # pages, latent, heads, dtype, lengths, sequences and heads compared. A run's ids come 510 at a time: 15 tiles at pages
    # of 1, 47 at pages of 3 (1,504 tokens: pieces start inside a page), 255 at pages of 16.
    (1, 256, 128, BF16, [7000, 1, 6500, 90, 0, 8001, 7777, 9000], [0, 3, 5], [0, 33, 127]),
    (1, 512, 97, F16, [12000, 10001, 13999], [1, 2], [0, 95, 96]),
    (3, 256, 128, F16, [33000, 31001, 35999, 17], [1, 3], [5, 64]),
    (3, 512, 24, BF16, [3001] * 135, [0, 77, 134], [0, 23]),
    (16, 256, 128, BF16, [32800] * 16, [0, 15], [31, 96]),
]


@pytest.mark.parametrize("page,latent,heads,dtype,lens,seqs,some", PIECES)
def test_decode_runs_of_many_pieces(page, latent, heads, dtype, lens, seqs, some, dev):
    say(f"latent decode pieces page={page} L={latent} H={heads} {dtype} {len(lens)} x {max(lens)}")
    cache, table, n = _pool(lens, page, 1, latent + 64, dtype, 61, dev, width=-(-max(lens) // page) + 2)
    if page == 3:
        table[seqs[0], 400:410] = -1  # absent blocks inside a piece
        table[seqs[0], 700] = 2 ** 30
    q = torch.randn(len(lens), 1, heads, latent + 64, device=dev, generator=torch.Generator(dev).manual_seed(62)).to(dtype)
    tiles = sum(-(-x // 32) for x in lens) * -(-heads // 32)
    runs = torch.cuda.get_device_properties(dev).multi_processor_count
    assert tiles // runs > 510 * page // 32, "the sizes do not reach a second piece"
    out = latent_decode_paged_fn(q, cache, table, n, page, scale=0.05)
    again = latent_decode_paged_fn(q, cache, table, n, page, scale=0.05)
    assert torch.equal(out, again)
    cache, table, n, q, out = (x.cpu() for x in (cache, table, n, q, out))
    for i in seqs:
        exact, limit = ref.latent_decode(q[i:i + 1][:, :, some], cache, table[i:i + 1], n[i:i + 1], page, 0.05)
        _check(out[i:i + 1][:, :, some], exact, limit, f"sequence {i}")
    for i in (i for i, x in enumerate(lens) if x == 0):
        assert (out[i] == 0).all()


MASSES = [
    # query heads, KV heads, head_dim, new tokens, page, dtype, lengths
    (24, 4, 256, 1, 16, BF16, [9100, 1, 700]),       # more than 64 parts of 128 tokens, nine ranges of 1,024
    (16, 1, 576, 1, 8, F16, [8321, 8192]),
    (32, 8, 128, 4, 16, F16, [17000, 5]),            # 16 rows, more than two rounds of parts
    (32, 8, 128, 32, 16, BF16, [8705, 300]),         # a window: 128 rows, statistics joined over 69 parts
    (24, 1, 576, 5, 16, BF16, [4500, 3, 4161]),      # 120 rows in four blocks through two stages, 71 parts of 64
    (97, 1, 576, 1, 3, F16, [4200, 129]),            # four blocks, the last of one row
    (40, 1, 320, 4, 16, F16, [8300, 64]),            # five blocks through three stages
    (12, 2, 256, 33, 16, BF16, [9000, 20]),          # 198 rows: seven blocks, the last of six rows
]


@pytest.mark.parametrize("hq,hkv,d,new,page,dtype,lens", MASSES)
def test_mass_of_long_sequences(hq, hkv, d, new, page, dtype, lens, dev):
    say(f"mass {hq}/{hkv} D={d} N={new} page={page} {dtype} {lens}")
    k, table, n = _pool(lens, page, hkv, d, dtype, 63, dev, width=-(-max(lens) // page) + 1)
    table[0, 100], table[0, 7] = -1, 10 ** 6  # absent
    q = (2 * torch.randn(len(lens), new, hq, d, device=dev, generator=torch.Generator(dev).manual_seed(64))).to(dtype)
    got = cache_attention_mass(q, k, table, n, page)
    assert torch.equal(got, cache_attention_mass(q, k, table, n, page))
    exact, limit = ref.attention_mass(q.cpu(), k.cpu(), table.cpu(), n.cpu(), page, d ** -0.5)
    _check(got, exact, limit, "mass")
    for i, x in enumerate(lens):
        assert (got[i, :, x:] == 0).all()
    sums = torch.full_like(got, 0.5)
    cache_attention_mass(q, k, table, n, page, mass=sums)
    _check(sums - 0.5, exact, limit + 2.0 ** -24 * (exact.abs() + 0.5) * 2, "added")
