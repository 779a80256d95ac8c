"""Paged prefill with capped, biased and interval-masked scores against its 64-bit form."""
import pytest
import torch

from helpers import bits, say
from oracle import ref_shaped as ref
from test_gpu_draft_tree import paged, slopes_of, within
from tileinfer_amd.kernels import gqa_prefill_paged_fn, gqa_prefill_shaped_fn

pytestmark = pytest.mark.gpu
BF16, F16 = torch.bfloat16, torch.float16


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def inputs(hq, hkv, d, q_lens, lens, page, dtype, seed=3):
    k, v, table, lens_t = paged(lens, page, hkv, d, dtype, seed)
    q = (2 * torch.randn(sum(q_lens), hq, d, generator=_gen(seed + 1))).to(dtype)
    cu = torch.tensor([0] + list(torch.tensor(q_lens).cumsum(0)), dtype=torch.int32)
    return q, k, v, table, cu, lens_t


def documents(q_lens, lens, mean, g):
    """First key of every query: the start of its document."""
    out = []
    for n, m in zip(q_lens, lens):
        starts = torch.zeros(max(m, n), dtype=torch.int32)
        at = 0
        while at < m:
            size = int(torch.randint(1, 2 * mean, (), generator=g))
            starts[at:at + size] = at
            at += size
        out.append(starts[max(m, n) - n:] if n else starts[:0])
    return torch.cat(out)


CASES = [
    # heads, D, chunks, cached with the chunk, page, dtype, causal, cap, slopes, window, first, last
    (24, 4, 256, [1, 33, 64, 0, 130], [1, 33, 70, 5, 300], 16, BF16, True, 0.0, False, 0, None, None),
    (24, 4, 256, [50, 7], [50, 400], 16, BF16, True, 30.0, True, 60, None, None),
    (6, 1, 256, [100, 20], [260, 20], 8, F16, True, 50.0, False, 0, "docs", None),
    (6, 1, 256, [200], [200], 16, BF16, True, 0.0, True, 0, None, "spans"),
    (8, 2, 256, [90, 40], [150, 40], 1, BF16, False, 20.0, True, 0, "docs", "docs"),
    (2, 2, 256, [300], [650], 32, F16, True, 0.0, False, 100, None, "prefix"),
    (32, 8, 128, [1, 65, 129, 200], [64, 65, 129, 513], 16, BF16, True, 50.0, False, 0, None, None),
    (32, 8, 128, [40, 3], [128, 700], 24, F16, True, 0.0, True, 33, None, None),
    (16, 16, 128, [150, 70], [190, 333], 16, F16, True, 15.0, True, 0, "docs", "spans"),
    (20, 2, 128, [77], [177], 4, BF16, False, 0.0, False, 0, None, None),
    (4, 4, 128, [200], [200], 16, BF16, True, 0.0, False, 1, None, None),
    (8, 1, 128, [5] * 50, [5, 9, 100, 64, 300] * 10, 16, BF16, True, 0.0, True, 0, "docs", None),
    (6, 2, 128, [30, 5], [10, 3], 2, BF16, True, 10.0, False, 0, None, None),  # more queries than keys
]


@pytest.mark.parametrize("hq,hkv,d,q_lens,lens,page,dtype,causal,cap,slopes,window,first,last", CASES)
def test_matches_formula(hq, hkv, d, q_lens, lens, page, dtype, causal, cap, slopes, window, first, last, dev):
    say(f"shaped {hq}/{hkv} D={d} q={q_lens[:4]} k={lens[:4]} page={page} {dtype} {causal} {cap} {slopes} {window} {first} {last}")
    q, k, v, table, cu, lens_t = inputs(hq, hkv, d, q_lens, lens, page, dtype)
    g = _gen(9)
    firsts = documents(q_lens, lens, 40, g) if first else None
    ends = None
    if last:
        position = torch.cat([torch.arange(m - n, m) for n, m in zip(q_lens, lens)])
        if last == "prefix":
            ends = position.clamp_min(120)
        elif last == "spans":  # some spans end inside, at and behind the sequence
            ends = position + torch.randint(0, 50, position.shape, generator=g)
        else:
            ends = position + torch.randint(-30, 30, position.shape, generator=g)
        ends = ends.to(torch.int32)
    sl = slopes_of(hq) if slopes else None
    exact, limit = ref.prefill(q, k, v, table, cu, lens_t, page, d ** -0.5, causal, cap, sl, window, firsts, ends)
    to = lambda x: None if x is None else x.to(dev)  # noqa: E731
    out = gqa_prefill_shaped_fn(*map(to, (q, k, v, table, cu, lens_t)), max(q_lens), page, causal=causal,
                                softcap=cap or None, slopes=to(sl), window=window or None, first_key=to(firsts),
                                last_key=to(ends))
    assert out.shape == q.shape and out.dtype == dtype
    within(out, exact, limit, "shaped prefill")


@pytest.mark.parametrize("hq,hkv,d,n,length,window", [(6, 1, 256, 40, 5000, 0), (4, 1, 128, 100, 9000, 2500),
                                                      (8, 2, 128, 1, 3000, 0)])
def test_keys_cut_between_workgroups(hq, hkv, d, n, length, window, dev):
    say(f"shaped splits {hq}/{hkv} D={d} q={n} k={length}")
    q_lens, lens = [n, 3, n // 2], [length, 900, 40 + n]
    q, k, v, table, cu, lens_t = inputs(hq, hkv, d, q_lens, lens, 16, BF16)
    exact, limit = ref.prefill(q, k, v, table, cu, lens_t, 16, 0.05, True, 25.0, None, window)
    to = lambda x: x.to(dev)  # noqa: E731
    for bound in (length, None):
        out = gqa_prefill_shaped_fn(*map(to, (q, k, v, table, cu, lens_t)), n, scale=0.05, softcap=25.0,
                                    window=window or None, max_seqlen_k=bound)
        within(out, exact, limit, "shaped prefill")


def test_plain_scores_are_the_paged_prefills(dev):
    """Without any shape the call is gqa_prefill_paged_fn, up to both kernels' limits."""
    say("shaped: plain")
    q, k, v, table, cu, lens_t = (x.to(dev) for x in inputs(24, 4, 256, [200, 31], [700, 31], 16, BF16))
    a = gqa_prefill_shaped_fn(q, k, v, table, cu, lens_t, 200)
    b = gqa_prefill_paged_fn(q, k.nan_to_num(0.0), v.nan_to_num(0.0), table, cu, lens_t, 200)
    exact, limit = ref.prefill(q.cpu(), k.cpu(), v.cpu(), table.cpu(), cu.cpu(), lens_t.cpu(), 16, 256 ** -0.5)
    within(a, exact, limit, "shaped")
    within(b, exact, limit, "paged")


def test_empty_intervals_absent_blocks_and_rows_of_no_sequence(dev):
    say("shaped: empty intervals, absent blocks")
    hq, hkv, d = 6, 2, 128
    q, k, v, table, cu, lens_t = inputs(hq, hkv, d, [70, 20], [150, 100], 8, BF16)
    table[0, 3], table[0, 9], table[1, :5] = -1, 10 ** 6, -9
    q = torch.cat([q, q[:7]])  # rows behind the last sequence
    g = _gen(11)
    first = torch.randint(-20, 160, (97,), generator=g).to(torch.int32)
    last = torch.randint(-20, 200, (97,), generator=g).to(torch.int32)
    first[5], last[5] = 2 ** 31 - 1, -2 ** 31
    first[6], last[6] = -2 ** 31, 2 ** 31 - 1
    exact, limit = ref.prefill(q[:90], k, v, table, cu, lens_t, 8, 0.1, True, 8.0, slopes_of(hq), 0, first[:90], last[:90])
    out = torch.full((97, hq, d), 5.0, dtype=BF16, device=dev)
    to = lambda x: x.to(dev)  # noqa: E731
    gqa_prefill_shaped_fn(*map(to, (q, k, v, table, cu, lens_t)), 70, 8, scale=0.1, softcap=8.0,
                          slopes=slopes_of(hq).to(dev), first_key=to(first), last_key=to(last), out=out)
    within(out[:90], exact, limit, "shaped prefill")
    assert (out[5] == 0).all() and (out[90:] == 5).all()


def test_keys_that_are_not_seen_may_be_anything(dev):
    say("shaped: unseen keys that are not finite")
    q, k, v, table, cu, lens_t = inputs(8, 2, 128, [64], [200], 16, BF16)
    last = torch.arange(136, 200, dtype=torch.int32).clamp_max(170)
    first = torch.full((64,), 20, dtype=torch.int32)
    to = lambda x: x.to(dev)  # noqa: E731
    call = dict(softcap=9.0, first_key=to(first), last_key=to(last))
    base = gqa_prefill_shaped_fn(*map(to, (q, k, v, table, cu, lens_t)), 64, **call)
    for bad in (torch.nan, torch.inf, -torch.inf):
        k2 = k.clone()
        for t in [*range(20), *range(171, 200)]:
            k2[table[0, t // 16], t % 16] = bad
        out = gqa_prefill_shaped_fn(*map(to, (q, k2, v, table, cu, lens_t)), 64, **call)
        assert torch.equal(bits(out), bits(base))
