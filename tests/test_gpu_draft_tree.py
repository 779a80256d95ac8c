"""Attention of drafted trees over the paged cache, and the accepted rows put in place, against their 64-bit forms."""
import pytest
import torch

from helpers import bits, say
from oracle import ref_shaped as ref
from tileinfer_amd.kernels import gqa_tree_paged_fn, keep_drafts, tree_masks

pytestmark = pytest.mark.gpu
BF16, F16 = torch.bfloat16, torch.float16


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def within(out, exact, limit, what=""):
    out = out.double().cpu()
    assert torch.isfinite(out).all(), f"{what}: values that are not finite"
    worst = ((out - exact).abs() / limit).max().item() if out.numel() else 0.0
    say(f"  {what}: worst error is {worst:.3f} of its limit")
    assert worst <= 1.0


def paged(lens, page, hkv, d, dtype, seed, extra=3, width=None):
    """Key and value caches whose unused rows are NaN, and tables of shuffled blocks with -1 behind."""
    g = _gen(seed)
    counts = [-(-max(n, 0) // page) for n in lens]
    blocks = sum(counts) + extra
    perm = torch.randperm(blocks, generator=g).to(torch.int32)
    width = width or max(max(counts), 1)
    table = torch.full((len(lens), width), -1, dtype=torch.int32)
    caches = [torch.full((blocks, page, hkv, d), torch.nan).to(dtype) for _ in range(2)]
    at = 0
    for i, (n, c) in enumerate(zip(lens, counts)):
        table[i, :c] = perm[at:at + c]
        at += c
        t = torch.arange(n)
        rows = table[i, t // page].long() * page + t % page
        for cache in caches:
            cache.view(-1, hkv, d)[rows] = torch.randn(n, hkv, d, generator=g).to(dtype)
    return caches[0], caches[1], table, torch.tensor(lens, dtype=torch.int32)


def random_tree(n, g):
    """Parents of n drafts, some of them roots."""
    return [-1 if i == 0 or torch.rand((), generator=g) < 0.05 else
            int(torch.randint(max(0, i - 4), i, (), generator=g)) for i in range(n)]


def slopes_of(hq):
    return 2.0 ** (-8.0 * torch.arange(1, hq + 1, dtype=torch.float32) / hq)


TREES = [
    # heads, D, drafts, page, dtype, lengths, cap, slopes, window
    (24, 4, 256, 1, 16, BF16, [1, 31, 32, 33, 700, 0], 0.0, False, 0),
    (24, 4, 256, 1, 16, BF16, [1, 2, 64, 300], 30.0, True, 40),
    (24, 4, 256, 2, 16, F16, [2, 31, 65, 500], 0.0, True, 0),
    (24, 4, 256, 4, 8, BF16, [4, 5, 36, 257, 0], 50.0, False, 0),
    (24, 4, 256, 7, 16, F16, [7, 20, 39, 400], 20.0, True, 16),
    (24, 4, 256, 16, 24, BF16, [16, 17, 48, 333], 0.0, True, 0),
    (24, 4, 256, 64, 16, BF16, [64, 65, 100, 290], 50.0, False, 0),
    (6, 1, 256, 33, 4, F16, [33, 70, 129], 0.0, False, 5),
    (2, 2, 256, 5, 1, BF16, [5, 77, 200], 0.0, True, 0),
    (32, 8, 128, 1, 16, BF16, [1, 63, 64, 65, 900], 30.0, False, 0),
    (32, 8, 128, 3, 8, F16, [3, 66, 128, 511], 0.0, True, 100),
    (32, 8, 128, 8, 16, BF16, [8, 71, 72, 640], 0.0, False, 0),
    (32, 8, 128, 17, 32, F16, [17, 81, 300], 15.0, True, 0),
    (32, 8, 128, 64, 16, BF16, [64, 127, 128, 400], 0.0, True, 30),
    (16, 16, 128, 20, 2, BF16, [20, 84, 150], 50.0, True, 0),
    (20, 2, 128, 6, 48, F16, [6, 100, 260], 0.0, False, 0),
    (24, 4, 256, 3, 16, BF16, [3, 35] * 40, 0.0, False, 0),
]


@pytest.mark.parametrize("hq,hkv,d,n,page,dtype,lens,cap,slopes,window", TREES)
def test_tree_matches_formula(hq, hkv, d, n, page, dtype, lens, cap, slopes, window, dev):
    say(f"tree {hq}/{hkv} D={d} N={n} page={page} {dtype} lens={lens[:6]} cap={cap} slopes={slopes} window={window}")
    k, v, table, lens_t = paged(lens, page, hkv, d, dtype, 21)
    g = _gen(22)
    q = (2 * torch.randn(len(lens), n, hq, d, generator=g)).to(dtype)
    parents = [random_tree(n, g) for _ in lens]
    masks = tree_masks(parents)
    sl = slopes_of(hq) if slopes else None
    scale = d ** -0.5
    call = dict(softcap=cap or None, slopes=None if sl is None else sl.to(dev), window=window or None)
    args = (k.to(dev), v.to(dev), table.to(dev), lens_t.to(dev))
    for mask in (masks, masks[0], None):
        rows = None if mask is None else (mask if mask.dim() == 2 else mask[None].expand(len(lens), n)).tolist()
        exact, limit = ref.tree(q, k, v, table, lens_t, rows, page, scale, cap, sl, window)
        out = gqa_tree_paged_fn(q.to(dev), *args, None if mask is None else mask.to(dev), page, **call)
        assert out.shape == q.shape and out.dtype == dtype
        within(out, exact, limit, "tree")
    if n == 1:
        one = gqa_tree_paged_fn(q[:, 0].to(dev), *args, None, page, **call)
        assert one.shape == (len(lens), hq, d) and torch.equal(bits(one), bits(out[:, 0]))


@pytest.mark.parametrize("hq,hkv,d,n,length,window", [(24, 4, 256, 1, 9000, 0), (24, 4, 256, 9, 6001, 0),
                                                      (32, 8, 128, 16, 7000, 3000), (32, 8, 128, 1, 20000, 0)])
def test_tree_long_sequences_cut_into_runs(hq, hkv, d, n, length, window, dev):
    say(f"tree long {hq}/{hkv} D={d} N={n} n={length} window={window}")
    lens = [length, n + 16, length // 2, n, 2 * n]
    k, v, table, lens_t = paged(lens, 16, hkv, d, BF16, 31, width=-(-length // 16) + 5)
    g = _gen(32)
    q = (2 * torch.randn(len(lens), n, hq, d, generator=g)).to(BF16)
    masks = tree_masks([random_tree(n, g) for _ in lens])
    exact, limit = ref.tree(q, k, v, table, lens_t, masks.tolist(), 16, 0.07, 30.0, None, window)
    out = gqa_tree_paged_fn(q.to(dev), k.to(dev), v.to(dev), table.to(dev), lens_t.to(dev), masks.to(dev), scale=0.07,
                            softcap=30.0, window=window or None)
    within(out, exact, limit, "tree")


def test_masks_that_leave_rows_empty_and_any_bits(dev):
    """A mask without its own bit, without any, with bits of no draft; sequences shorter than their drafts; blocks
    outside the cache; scores of +-10^4."""
    say("tree: masks of any bits, short sequences, absent blocks")
    n, hq, hkv, d = 5, 8, 2, 128
    lens = [n, 3, 1, 0, 40, 90, 33]
    k, v, table, lens_t = paged(lens, 8, hkv, d, BF16, 41, width=13)
    table[4, 1], table[4, 3], table[5, 0], table[6] = -1, 10 ** 6, -7, -1
    g = _gen(42)
    q = torch.randn(len(lens), n, hq, d, generator=g).to(BF16)
    q[5] *= 80
    masks = torch.randint(-2 ** 62, 2 ** 62, (len(lens), n), generator=g)
    masks[0, 2] = 0
    masks[5, 1] = -1
    for cap, window in ((0.0, 0), (10.0, 3)):
        exact, limit = ref.tree(q, k, v, table, lens_t, masks.tolist(), 8, 0.1, cap, slopes_of(hq), window)
        out = gqa_tree_paged_fn(q.to(dev), k.to(dev), v.to(dev), table.to(dev), lens_t.to(dev), masks.to(dev), 8,
                                scale=0.1, softcap=cap or None, slopes=slopes_of(hq).to(dev), window=window or None)
        within(out, exact, limit, "tree")
        assert (out[0, 2] == 0).all() and (out[3] == 0).all() and (out[6] == 0).all()


def test_keys_that_are_not_seen_may_be_anything(dev):
    say("tree: unseen keys that are not finite")
    n, hq, hkv, d = 6, 24, 4, 256
    lens = [50, 100]
    k, v, table, lens_t = paged(lens, 16, hkv, d, BF16, 51)
    masks = tree_masks([[-1, 0, 0, 1, 2, 4]] * 2)
    q = torch.randn(2, n, hq, d, generator=_gen(52)).to(BF16)
    call = (table.to(dev), lens_t.to(dev), masks.to(dev))
    base = gqa_tree_paged_fn(q.to(dev), k.to(dev), v.to(dev), *call, softcap=20.0)
    for bad in (torch.nan, torch.inf, -torch.inf):
        k2 = k.clone()
        for b, m in enumerate(lens):  # draft 3 is seen by itself alone
            t = m - n + 3
            k2[table[b, t // 16], t % 16] = bad
        out = gqa_tree_paged_fn(q.to(dev), k2.to(dev), v.to(dev), *call, softcap=20.0)
        others = [0, 1, 2, 4, 5]
        assert torch.equal(bits(out[:, others].contiguous()), bits(base[:, others].contiguous()))


KEEPS = [
    # planes, D of a row, heads, drafts, page, dtype, lengths
    ((2, 3), 256, 4, 8, 16, BF16, [8, 9, 20, 100]),
    ((2, 16), 128, 2, 64, 8, F16, [64, 65, 300, 3, 0]),
    ((), 576, 1, 33, 16, BF16, [40, 33, 90]),
    ((5,), 64, 3, 2, 1, BF16, [2, 3, 50]),
    ((2,), 128, 8, 1, 32, F16, [1, 40]),
    ((1,), 8, 1, 17, 24, BF16, [17, 30, 41] * 30),
]


@pytest.mark.parametrize("planes,d,heads,n,page,dtype,lens", KEEPS)
def test_keep_moves_the_accepted_rows(planes, d, heads, n, page, dtype, lens, dev):
    say(f"keep planes={planes} row={heads}x{d} N={n} page={page} lens={lens[:5]}")
    g = _gen(61)
    counts = [-(-m // page) for m in lens]
    blocks = sum(counts) + 2
    cache = torch.randn(*planes, blocks, page, heads, d, generator=g).to(dtype)
    perm = torch.randperm(blocks, generator=g).to(torch.int32)
    table = torch.full((len(lens), max(max(counts), 1)), -1, dtype=torch.int32)
    at = 0
    for i, c in enumerate(counts):
        table[i, :c] = perm[at:at + c]
        at += c
    lens_t = torch.tensor(lens, dtype=torch.int32)
    for trial in range(4):
        accepted = torch.full((len(lens), (n, n + 3, max(1, n // 2), 70)[trial]), -1, dtype=torch.int32)
        for i in range(len(lens)):
            path = [j for j in range(n) if torch.rand((), generator=g) < (0.3, 1.0, 0.7, 0.5)[trial]]
            path = path[:accepted.shape[1]]
            accepted[i, :len(path)] = torch.tensor(path, dtype=torch.int32)
        if trial == 2 and len(lens) > 1:  # lists that do not ascend end there
            accepted[0] = torch.randint(-2, n + 2, accepted[0].shape, generator=g).to(torch.int32)
        want, new = ref.keep(cache, table, lens_t, accepted, page, n)
        got = cache.to(dev)
        lens_out = keep_drafts(got, table.to(dev), lens_t.to(dev), accepted.to(dev), page, num_drafts=n)
        assert torch.equal(lens_out.cpu(), new)
        assert torch.equal(bits(got.cpu()), bits(want))


def test_keep_skips_blocks_outside_the_cache(dev):
    say("keep: absent blocks")
    n, page = 6, 2
    cache = torch.randn(2, 9, page, 1, 16, generator=_gen(71)).to(BF16)
    table = torch.tensor([[0, 1, -1, 3], [4, 99, 6, 7]], dtype=torch.int32)
    lens = torch.tensor([8, 9], dtype=torch.int32)  # the second's last token lies behind its table
    accepted = torch.tensor([[0, 2, 3, 4, 5], [1, 2, 4, 5, -1]], dtype=torch.int32)
    want, new = ref.keep(cache, table, lens, accepted, page, n)
    got = cache.to(dev)
    lens_out = keep_drafts(got, table.to(dev), lens.to(dev), accepted.to(dev), page, num_drafts=n)
    assert torch.equal(lens_out.cpu(), new) and torch.equal(bits(got.cpu()), bits(want))
