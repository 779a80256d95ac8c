"""Several position axes, drafted trees, kept drafts and shaped prefill as programs call them: both forms of each call,
captured and replayed, on another stream, behind 2^31 elements, over many pages, with operands of any strides, with wrong
ones, and one after the other."""
import pytest
import torch

from helpers import bits, say
from oracle import ref_shaped as ref
from test_gpu_draft_tree import paged, random_tree, slopes_of, within
from test_native_calls import _FORMS, both
from tileinfer_amd.kernels import (gqa_prefill_shaped_fn, gqa_tree_paged_fn, keep_drafts, rope_axes, rope_axes_append,
                                   tree_masks)

pytestmark = pytest.mark.gpu
BF16, F16 = torch.bfloat16, torch.float16


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _randn(dev, *shape, seed=0):
    return torch.randn(*shape, device=dev, generator=torch.Generator(dev).manual_seed(seed)).to(BF16)


def _ints(dev, values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device=dev)


# Both forms of a call

@pytest.mark.parametrize("form", list(_FORMS))
@pytest.mark.parametrize("which", ["q", "k", "positions", "inv_freq", "axes", "slots", "weight"])
def test_forms_of_rope(which, form, dev, monkeypatch):
    say(f"rope forms {which} {form}")
    if form == "transposed" and which in ("inv_freq", "axes", "slots", "weight"):
        pytest.skip("no such form")
    if form == "wide" and which == "positions":
        pytest.skip("float positions are tested with the refusals")
    if form == "short" and which == "positions":
        pytest.skip("positions of fewer axes are positions")
    f = lambda name, t: _FORMS[form](t) if which == name else t  # noqa: E731
    n = 6
    weight = f("weight", _randn(dev, 128, seed=4))

    def call():
        caches = [torch.zeros(9, 256, dtype=BF16, device=dev) for _ in range(2)]
        pos = _ints(dev, [[3, 4, 5, 6, 7, 8], [1, 1, 1, 2, 2, 2]])
        q = rope_axes_append(f("q", _randn(dev, n, 4, 128)), f("k", _randn(dev, n, 2, 128, seed=1)), _randn(dev, n, 2, 128, seed=2),
                             f("positions", pos), f("inv_freq", torch.rand(32, device=dev, generator=torch.Generator(dev).manual_seed(3))),
                             f("axes", _ints(dev, [0, 1] * 16)), *caches, f("slots", _ints(dev, [4, -1, 0, 7, 8, 2])),
                             q_weight=weight, k_weight=weight, eps=1e-6)
        return [q, *caches]

    refused = both(monkeypatch, call, True if form == "plain" else None)
    if form == "parameter" and which in ("positions", "axes", "slots"):
        return
    assert (refused is not None) == (form in ("short", "wide")) or form == "odd"


@pytest.mark.parametrize("drafts", [3, 40])  # either kernel
@pytest.mark.parametrize("form", list(_FORMS))
@pytest.mark.parametrize("which", ["q", "cache", "table", "lens", "mask", "slopes"])
def test_forms_of_tree(which, form, drafts, dev, monkeypatch):
    say(f"tree forms {which} {form} {drafts}")
    if form == "transposed" and which in ("lens", "cache", "slopes") or form == "parameter" and which in ("table", "lens", "mask"):
        pytest.skip("no such form")
    if which == "cache" and form in ("short", "strided", "odd"):
        pytest.skip("another cache, or one that is never copied")
    f = lambda name, t: _FORMS[form](t) if which == name else t  # noqa: E731
    cache = _randn(dev, 16, 16, 2, 128, seed=5)
    masks = tree_masks([random_tree(drafts, _gen(6)) for _ in range(3)]).to(dev)

    def call():
        return [gqa_tree_paged_fn(f("q", _randn(dev, 3, drafts, 6, 128)), f("cache", cache), cache + 1,
                                  f("table", _ints(dev, [[1, 2, 3, 4, 5], [6, 7, 8, 9, 10], [11, 12, 13, 14, 15]])),
                                  f("lens", _ints(dev, [80, 41, 60])), f("mask", masks), slopes=f("slopes", slopes_of(6).to(dev)),
                                  softcap=20.0, window=30)]

    refused = both(monkeypatch, call, True if form == "plain" else None)
    assert (refused is not None) == (form in ("short", "wide")) or form == "odd"


@pytest.mark.parametrize("form", list(_FORMS))
@pytest.mark.parametrize("which", ["table", "lens", "accepted"])
def test_forms_of_keep(which, form, dev, monkeypatch):
    say(f"keep forms {which} {form}")
    if form == "transposed" and which == "lens" or form == "parameter":
        pytest.skip("no such form")
    f = lambda name, t: _FORMS[form](t) if which == name else t  # noqa: E731

    def call():
        cache = _randn(dev, 2, 3, 8, 4, 1, 64, seed=7)
        lens = keep_drafts(cache, f("table", _ints(dev, [[1, 2, 3], [4, 5, 6]])), f("lens", _ints(dev, [11, 9])),
                           f("accepted", _ints(dev, [[0, 2, 5, -1], [1, 3, 4, 6]])), 4, num_drafts=7)
        return [cache, lens.to(torch.int16)]

    refused = both(monkeypatch, call, True if form == "plain" else None)
    assert (refused is not None) == (form in ("short", "wide")) or form == "odd"


@pytest.mark.parametrize("form", list(_FORMS))
@pytest.mark.parametrize("which", ["q", "cache", "table", "cu", "lens", "first", "last", "slopes"])
def test_forms_of_shaped(which, form, dev, monkeypatch):
    say(f"shaped forms {which} {form}")
    if form == "transposed" and which not in ("q", "table") or form == "parameter" and which not in ("q", "cache", "slopes"):
        pytest.skip("no such form")
    if which == "cache" and form in ("short", "strided", "odd"):
        pytest.skip("another cache, or one that is never copied")
    f = lambda name, t: _FORMS[form](t) if which == name else t  # noqa: E731
    cache = _randn(dev, 16, 16, 2, 128, seed=5)

    def call():
        return [gqa_prefill_shaped_fn(
            f("q", _randn(dev, 30, 6, 128)), f("cache", cache), cache + 1,
            f("table", _ints(dev, [[1, 2, 3, 4, 5], [6, 7, 8, 9, 10]])), f("cu", _ints(dev, [0, 13, 30])),
            f("lens", _ints(dev, [80, 41])), 17, softcap=20.0, slopes=f("slopes", slopes_of(6).to(dev)), window=30,
            first_key=f("first", torch.arange(30, dtype=torch.int32, device=dev)),
            last_key=f("last", torch.arange(20, 80, 2, dtype=torch.int32, device=dev)), max_seqlen_k=80)]

    refused = both(monkeypatch, call, True if form == "plain" else None)
    assert (refused is not None) == (form in ("short", "wide")) or form == "odd"


def test_refusals(dev):
    """Wrong types, sizes, devices and numbers raise before anything is launched."""
    say("shaped refusals")
    cache = _randn(dev, 8, 16, 2, 128)
    table, lens, q = _ints(dev, [[1, 2, 3]]), _ints(dev, [40]), _randn(dev, 1, 2, 4, 128)
    mask = _ints(dev, [1, 3], torch.int64)
    ok = dict(softcap=30.0, window=8, slopes=slopes_of(4).to(dev))
    gqa_tree_paged_fn(q, cache, cache, table, lens, mask, **ok)
    for change in (dict(softcap=0.0), dict(softcap=float("nan")), dict(window=0), dict(window=-3), dict(scale=0.0), dict(scale=1e31),
                   dict(slopes=slopes_of(3).to(dev)), dict(slopes=slopes_of(4)), dict(slopes=slopes_of(4).half().to(dev)),
                   dict(out=torch.empty(1, 2, 4, 64, dtype=BF16, device=dev))):
        with pytest.raises((ValueError, TypeError)):
            gqa_tree_paged_fn(q, cache, cache, table, lens, mask, **{**ok, **change})
    for args in ((q[..., :64], cache, cache, table, lens, mask), (q, cache[..., :64], cache, table, lens, mask),
                 (q, cache, cache[:-1], table, lens, mask), (q, cache.half(), cache.half(), table, lens, mask),
                 (q, cache, cache, table.long(), lens, mask), (q, cache, cache, table, lens.long(), mask),
                 (q, cache, cache, table, lens, mask.int()), (q, cache, cache, table, lens, mask[:1]),
                 (q, cache, cache, table, lens, mask.cpu()), (q, cache, cache, table.cpu(), lens, mask),
                 (q.cpu(), cache, cache, table, lens, mask), (q[:, :, :3], cache, cache, table, lens, mask),
                 (q[0, 0, 0], cache, cache, table, lens, mask), (q.expand(1, 2, 4, 128).repeat(1, 33, 1, 1), cache, cache, table, lens, None),
                 (q, cache.transpose(1, 2), cache.transpose(1, 2), table, lens, mask)):
        with pytest.raises((ValueError, TypeError)):
            gqa_tree_paged_fn(*args)
    with pytest.raises(ValueError):
        gqa_tree_paged_fn(q, cache, cache, table, lens, mask, 7)
    accepted = _ints(dev, [[0, 1]])
    for args, kw in (((cache[0], table, lens, accepted), dict(num_drafts=2)), ((cache.float(), table, lens, accepted), dict(num_drafts=2)),
                     ((cache, table, lens, accepted.long()), dict(num_drafts=2)), ((cache, table, lens, accepted[0]), dict(num_drafts=2)),
                     ((cache, table, lens, accepted), dict(num_drafts=0)), ((cache, table, lens, accepted), dict(num_drafts=65)),
                     ((cache, table, lens, accepted, 7), dict(num_drafts=2)), ((cache[:0], table, lens, accepted), dict(num_drafts=2)),
                     ((cache.cpu(), table, lens, accepted), dict(num_drafts=2)), ((cache.transpose(0, 1), table, lens, accepted), dict(num_drafts=2))):
        with pytest.raises((ValueError, TypeError)):
            keep_drafts(*args, **kw)
    q3, cu = q[0], _ints(dev, [0, 2])
    gqa_prefill_shaped_fn(q3, cache, cache, table, cu, lens, 2, **ok)
    for kw in (dict(first_key=_ints(dev, [1])), dict(last_key=_ints(dev, [1, 2], torch.int64)), dict(first_key=torch.tensor([1, 2], dtype=torch.int32)),
               dict(max_seqlen_q=-1), dict(max_seqlen_k=-1), dict(softcap=1e5), dict(window=0), dict(scale=-1.0),
               dict(out=torch.empty(2, 4, 128, dtype=F16, device=dev))):
        with pytest.raises((ValueError, TypeError)):
            gqa_prefill_shaped_fn(q3, cache, cache, table, cu, lens, **{"max_seqlen_q": 2, **kw})
    with pytest.raises((ValueError, TypeError)):
        gqa_prefill_shaped_fn(q3, cache, cache, table, cu.long(), lens, 2)
    rows = cache.view(-1, 256)
    k = _randn(dev, 2, 2, 128)
    pos, inv, slots = _ints(dev, [1, 2]), torch.rand(32, device=dev), _ints(dev, [0, 1])
    good = dict(q=q3, k=k, v=k, positions=pos, inv_freq=inv, axes=None, k_cache=rows, v_cache=rows.clone(), slot_mapping=slots)
    rope_axes_append(**good)
    for kw in (dict(positions=pos.float()), dict(positions=pos[:1]), dict(positions=pos.expand(5, 2)), dict(inv_freq=inv.double()),
               dict(inv_freq=inv[:30]), dict(inv_freq=torch.rand(72, device=dev)), dict(axes=_ints(dev, [0] * 31)), dict(axes=torch.zeros(32, device=dev)),
               dict(k=k[:1]), dict(v=k.half()), dict(k_cache=rows[:, :128]), dict(k_cache=rows[1:]), dict(slot_mapping=slots.long()),
               dict(slot_mapping=slots.cpu()), dict(q_weight=_randn(dev, 128)), dict(q=q3[..., :64], k=k[..., :64], v=k[..., :64]),
               dict(q_out=torch.empty(2, 4, 64, dtype=BF16, device=dev))):
        with pytest.raises((ValueError, TypeError)):
            rope_axes_append(**{**good, **kw})


def test_no_tokens_and_no_sequences(dev):
    say("shaped: empty calls")
    cache = _randn(dev, 8, 16, 2, 128)
    e = lambda *s: torch.empty(*s, dtype=BF16, device=dev)  # noqa: E731
    assert gqa_tree_paged_fn(e(0, 3, 4, 128), cache, cache, _ints(dev, []).view(0, 2), _ints(dev, [])).shape == (0, 3, 4, 128)
    assert gqa_prefill_shaped_fn(e(0, 4, 128), cache, cache, _ints(dev, [[1]]), _ints(dev, [0, 0]), _ints(dev, [5]), 0).shape == (0, 4, 128)
    assert keep_drafts(cache, _ints(dev, []).view(0, 2), _ints(dev, []), _ints(dev, []).view(0, 4), num_drafts=3).shape == (0,)
    assert keep_drafts(cache, _ints(dev, [[1]]), _ints(dev, [9]), _ints(dev, []).view(1, 0), num_drafts=3).tolist() == [6]
    q = rope_axes_append(e(0, 4, 128), e(0, 2, 128), e(0, 2, 128), _ints(dev, []), torch.rand(8, device=dev), None,
                         cache.view(-1, 256), cache.view(-1, 256).clone(), _ints(dev, []))
    assert q.shape == (0, 4, 128)
    none = torch.empty(3, 0, dtype=torch.int32, device=dev)  # tables without a column
    for n in (1, 33):
        out = gqa_tree_paged_fn(_randn(dev, 3, n, 4, 128), cache, cache, none, _ints(dev, [5, 0, 70]))
        assert (out == 0).all()
    out = gqa_prefill_shaped_fn(_randn(dev, 6, 4, 128), cache, cache, none, _ints(dev, [0, 2, 4, 6]), _ints(dev, [5, 0, 70]), 2)
    assert (out == 0).all()


# Streams and graphs

def _step(dev, drafts=9, heads=(24, 4), d=256, seed=3):
    lens = [drafts + 3, 700 + drafts, 300, 2500]
    k, v, table, lens_t = (x.nan_to_num(0.0).to(dev) if x.is_floating_point() else x.to(dev)
                           for x in paged(lens, 16, heads[1], d, BF16, seed))
    masks = tree_masks([random_tree(drafts, _gen(seed + i)) for i in range(4)]).to(dev)
    return k, v, table, lens_t, masks


@pytest.mark.parametrize("drafts", [1, 9, 40])
def test_two_graphs_of_a_verification(drafts, dev):
    """Two captured steps replayed in turn with eager ones and changed inputs between them."""
    say(f"graphs of a verification, {drafts} drafts")
    k, v, table, lens, masks = _step(dev, drafts)
    t = 4 * drafts
    qkv = _randn(dev, t, 32, 256, seed=8)
    inv = torch.rand(32, device=dev)
    first = torch.arange(drafts, dtype=torch.int32, device=dev)
    accepted = torch.full((4, drafts), -1, dtype=torch.int32, device=dev)
    accepted[:, 0] = drafts - 1
    slab = torch.stack([k, v])

    def step(cap):
        pos = ((lens - drafts)[:, None] + first).reshape(-1)
        at = pos.view(4, drafts)
        slots = (table.gather(1, (at // 16).long()) * 16 + at % 16).reshape(-1)
        kc, vc = slab[0], slab[1]
        q = rope_axes_append(qkv[:, :24], qkv[:, 24:28], qkv[:, 28:], pos, inv, None, kc.view(-1, 1024), vc.view(-1, 1024), slots)
        out = gqa_tree_paged_fn(q.view(4, drafts, 24, 256), kc, vc, table, lens, masks, softcap=cap)
        new = keep_drafts(slab, table, lens, accepted, num_drafts=drafts)
        return out, new, slab.clone()

    start = slab.clone()
    step(None)
    graphs = []
    for cap in (None, 30.0):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            graphs.append((graph, step(cap), cap))
    for i in range(3):
        qkv.copy_(_randn(dev, t, 32, 256, seed=20 + i))
        for graph, out, cap in graphs:
            slab.copy_(start)
            graph.replay()
            torch.cuda.synchronize()
            kept = [x.clone() for x in out]
            slab.copy_(start)
            for a, b in zip(kept, step(cap)):
                assert torch.equal(a, b), (i, cap)


@pytest.mark.parametrize("tokens,heads", [(300, (4, 1)), (900, (24, 4))])  # cut units, one workgroup a unit
def test_two_graphs_of_a_chunk(tokens, heads, dev):
    say(f"graphs of a shaped chunk {tokens} {heads}")
    k, v, table, lens = (x.nan_to_num(0.0).to(dev) if x.is_floating_point() else x.to(dev)
                         for x in paged([tokens + 3000], 16, heads[1], 128, BF16, 4))
    q = _randn(dev, tokens, heads[0], 128)
    cu = _ints(dev, [0, tokens])
    graphs = []
    for cap in (None, 20.0):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            graphs.append((graph, gqa_prefill_shaped_fn(q, k, v, table, cu, lens, tokens, softcap=cap), cap))
    for i in range(3):
        q.copy_(_randn(dev, *q.shape, seed=30 + i))
        for graph, out, cap in graphs:
            graph.replay()
            torch.cuda.synchronize()
            kept = out.clone()
            assert torch.equal(kept, gqa_prefill_shaped_fn(q, k, v, table, cu, lens, tokens, softcap=cap))


def test_calls_on_two_streams_at_once(dev):
    """The same calls on two other streams, without waiting between them."""
    say("shaped calls on two streams")
    k, v, table, lens, masks = _step(dev, 40)
    q = _randn(dev, 4, 40, 24, 256, seed=9)
    cu = _ints(dev, [0, 40, 80, 120, 160])
    want = gqa_tree_paged_fn(q, k, v, table, lens, masks), gqa_prefill_shaped_fn(q.view(160, 24, 256), k, v, table, cu, lens, 40, window=50)
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], []
    for _ in range(4):
        for s in streams:
            with torch.cuda.stream(s):
                got.append((gqa_tree_paged_fn(q, k, v, table, lens, masks),
                            gqa_prefill_shaped_fn(q.view(160, 24, 256), k, v, table, cu, lens, 40, window=50)))
    torch.cuda.synchronize()
    for a in got:
        assert all(torch.equal(bits(x), bits(y)) for x, y in zip(a, want))


# Sizes

@pytest.mark.parametrize("heads,d", [((24, 4), 256), ((32, 8), 128)])
def test_behind_2_31_elements(heads, d, dev):
    say(f"shaped large pool D={d}")
    hq, hkv = heads
    held = 24
    blocks = 2 ** 31 // (16 * hkv * d) + 20 + held
    small = _randn(dev, 2, held, 16, hkv, d)
    slab = torch.empty(2, blocks, 16, hkv, d, dtype=BF16, device=dev)
    ids = torch.arange(blocks - held, blocks, dtype=torch.int32, device=dev).flip(0)
    slab[:, ids.long()] = small
    table = torch.arange(24, dtype=torch.int32, device=dev).view(2, 12)
    big = ids[table.long()]
    lens = _ints(dev, [170, 100])
    for n in (2, 33):
        q = _randn(dev, 2, n, hq, d, seed=n)
        a = gqa_tree_paged_fn(q, small[0], small[1], table, lens, softcap=30.0)
        b = gqa_tree_paged_fn(q, slab[0], slab[1], big, lens, softcap=30.0)
        assert torch.equal(bits(a), bits(b))
    cu = _ints(dev, [0, 60, 80])
    q = _randn(dev, 80, hq, d, seed=1)
    a = gqa_prefill_shaped_fn(q, small[0], small[1], table, cu, lens, 60, window=70)
    b = gqa_prefill_shaped_fn(q, slab[0], slab[1], big, cu, lens, 60, window=70)
    assert torch.equal(bits(a), bits(b))
    slots = torch.arange(5, 160, 31, device=dev)
    t = slots.numel()
    args = (_randn(dev, t, hq, d), _randn(dev, t, hkv, d, seed=2), _randn(dev, t, hkv, d, seed=3), slots.int(),
            torch.rand(32, device=dev), None)
    far = (ids[slots // 16].long() * 16 + slots % 16).int()
    rope_axes_append(*args, small[0].view(-1, hkv * d), small[1].view(-1, hkv * d), slots.int())
    rope_axes_append(*args, slab[0].view(-1, hkv * d), slab[1].view(-1, hkv * d), far)
    accepted = _ints(dev, [[1, 5, 6], [0, 2, -1]])
    assert torch.equal(keep_drafts(small, table, lens, accepted, num_drafts=8), keep_drafts(slab, big, lens, accepted, num_drafts=8))
    assert torch.equal(bits(slab[:, ids.long()]), bits(small))


@pytest.mark.parametrize("d,hq,hkv", [(256, 6, 1), (128, 4, 1)])
@pytest.mark.parametrize("n", [1, 12, 40])
def test_more_pages_than_are_staged_at_once(d, hq, hkv, n, dev):
    """Pages of one token: a run's block ids are staged in several pieces."""
    say(f"shaped pieces D={d} N={n}")
    lens = [1300, n, 700]
    k, v, table, lens_t = paged(lens, 1, hkv, d, BF16, 13)
    q = torch.randn(3, n, hq, d, generator=_gen(14)).to(BF16)
    masks = tree_masks([random_tree(n, _gen(15 + i)) for i in range(3)])
    exact, limit = ref.tree(q, k, v, table, lens_t, masks.tolist(), 1, 0.1, 0.0, slopes_of(hq), 900)
    out = gqa_tree_paged_fn(*(x.to(dev) for x in (q, k, v, table, lens_t, masks)), 1, scale=0.1, slopes=slopes_of(hq).to(dev), window=900)
    within(out, exact, limit, "tree")
    if n == 12:
        cu = torch.tensor([0, 12, 24, 36], dtype=torch.int32)
        exact, limit = ref.prefill(q.view(36, hq, d), k, v, table, cu, lens_t, 1, 0.1, True, 20.0)
        out = gqa_prefill_shaped_fn(*(x.to(dev) for x in (q.view(36, hq, d), k, v, table, cu, lens_t)), 12, 1, scale=0.1, softcap=20.0)
        within(out, exact, limit, "prefill")


@pytest.mark.parametrize("n,hq,hkv,d", [(16, 24, 4, 256), (33, 8, 2, 128), (2, 32, 8, 128)])
def test_many_short_sequences(n, hq, hkv, d, dev):
    """More than 64 sequences (the lists are scanned 64 at a time), lengths of zero among them."""
    say(f"tree of 90 sequences N={n}")
    lens = [(37 * i) % 91 if i % 7 else 0 for i in range(90)]
    k, v, table, lens_t = paged(lens, 16, hkv, d, BF16, 17)
    q = torch.randn(90, n, hq, d, generator=_gen(18)).to(BF16)
    mask = tree_masks(random_tree(n, _gen(19)))
    exact, limit = ref.tree(q, k, v, table, lens_t, [mask.tolist()] * 90, 16, 0.1)
    out = gqa_tree_paged_fn(*(x.to(dev) for x in (q, k, v, table, lens_t, mask)), scale=0.1)
    within(out, exact, limit, "tree")


def test_long_lists_that_are_streamed(dev):
    """Enough tiles for the streaming policy, with and without two sequences that share their first block."""
    say("tree: streamed")
    lens = [9000] * 20
    counts = 563
    k, v = (_randn(dev, counts * 20, 16, 8, 128, seed=s) for s in (1, 2))
    table = torch.randperm(counts * 20, generator=_gen(3)).to(torch.int32).view(20, counts)
    shared = table.clone()
    shared[1, :40] = shared[0, :40]
    q = _randn(dev, 20, 2, 32, 128, seed=5)
    for t in (table, shared):
        out = gqa_tree_paged_fn(q, k, v, t.to(dev), _ints(dev, lens), softcap=30.0)
        some = [0, 1, 19]
        for b in some:
            exact, limit = ref.tree(q[b:b + 1].cpu(), k.cpu(), v.cpu(), t[b:b + 1], torch.tensor([9000]), None, 16, 128 ** -0.5, 30.0)
            within(out[b:b + 1], exact, limit, f"sequence {b}")


def test_offsets_that_go_back_or_beyond(dev):
    """cu_seqlens_q beyond the rows are cut off, a sequence whose end lies before its start is empty, rows past
    max_seqlen_q blocks and rows of no sequence are left as they were."""
    say("shaped: offsets")
    k, v, table, lens = paged([90, 60, 50], 16, 2, 128, BF16, 23)
    q = torch.randn(40, 4, 128, generator=_gen(24)).to(BF16)
    cu = torch.tensor([2, 25, 20, 99], dtype=torch.int32)
    out = torch.full((40, 4, 128), 3.0, dtype=BF16, device=dev)
    gqa_prefill_shaped_fn(*(x.to(dev) for x in (q, k, v, table, cu, lens)), 40, out=out)
    want, limit = ref.prefill(q[2:25], k, v, table[:1], torch.tensor([0, 23]), lens[:1], 16, 128 ** -0.5)
    last, limit2 = ref.prefill(q[20:], k, v, table[2:], torch.tensor([0, 20]), lens[2:], 16, 128 ** -0.5)
    within(out[2:20], want[:18], limit[:18], "first")
    within(out[25:], last[5:], limit2[5:], "last")
    assert (out[:2] == 3).all()


# One after the other

@pytest.mark.parametrize("heads,d,cap,slopes", [((24, 4), 256, 30.0, False), ((8, 2), 128, None, True)])
def test_speculative_steps_of_a_sequence(heads, d, cap, slopes, dev):
    """A prompt with an image goes in by chunks; then trees are drafted, verified and kept. What the accepted drafts saw is
    what a prefill of the accepted tokens sees, and the cache is that prefill's."""
    say(f"speculative steps {heads} D={d}")
    hq, hkv = heads
    layers, page, width = 2, 16, 20
    g = _gen(33)
    slab = torch.zeros(2, layers, 64, page, hkv, d, dtype=BF16, device=dev)
    plain = torch.zeros_like(slab)
    table = torch.randperm(64, generator=g)[:width].to(torch.int32).to(dev)[None]
    inv = (1e4 ** (-torch.arange(32).double() / 32)).float().to(dev)
    axes = rope_axes((12, 10, 10), device=dev)
    sl = slopes_of(hq).to(dev) if slopes else None
    shape = dict(softcap=cap, slopes=sl)

    def slots_of(at):
        return table[0, (at // page).long()] * page + at % page

    def append(cache, x, pos, slots):
        for layer in range(layers):
            q = rope_axes_append(x[:, :hq] + layer, x[:, hq:hq + hkv] + layer, x[:, hq + hkv:] + layer, pos, inv, axes,
                                 cache[0, layer].view(-1, hkv * d), cache[1, layer].view(-1, hkv * d), slots)
        return q  # of the last layer

    new = lambda n: torch.randn(n, hq + 2 * hkv, d, generator=g).to(BF16).to(dev)  # noqa: E731
    prompt = 60
    at = torch.arange(prompt, dtype=torch.int32, device=dev)
    image = (at >= 20) & (at < 36)
    pos = torch.stack([torch.where(image, 20, at), torch.where(image, 20 + (at - 20) // 4, at), torch.where(image, 20 + at % 4, at)])
    last = torch.where(image, 35, at).int()
    x = new(prompt)
    q = append(slab, x, pos.int(), slots_of(at))
    append(plain, x, pos.int(), slots_of(at))
    lens = _ints(dev, [prompt])
    out = gqa_prefill_shaped_fn(q, slab[0, 1], slab[1, 1], table, _ints(dev, [0, prompt]), lens, prompt, last_key=last, **shape)
    exact, limit = ref.prefill(q.cpu(), slab[0, 1].cpu(), slab[1, 1].cpu(), table.cpu(), torch.tensor([0, prompt]), lens.cpu(), page,
                               d ** -0.5, True, cap or 0.0, None if sl is None else sl.cpu(), 0, None, last.cpu())
    within(out, exact, limit, "prompt")
    for step in range(3):
        n = (12, 5, 33)[step]
        parents = random_tree(n, g)
        parents[1:] = [max(p, 0) for p in parents[1:]]
        masks = tree_masks(parents).to(dev)
        depth = torch.tensor([bin(m & (2 ** 64 - 1)).count("1") - 1 for m in masks.tolist()], dtype=torch.int32, device=dev)
        context = int(lens[0])
        x = new(n)
        q = append(slab, x, (context + depth).expand(3, n), slots_of(context + torch.arange(n, dtype=torch.int32, device=dev)))
        out = gqa_tree_paged_fn(q[None], slab[0, 1], slab[1, 1], table, lens + n, masks, **shape)
        path, node = [], n - 1 - step
        while node >= 0:
            path.append(node)
            node = parents[node]
        path = path[::-1]
        accepted = torch.full((1, n), -1, dtype=torch.int32, device=dev)
        accepted[0, :len(path)] = _ints(dev, path)
        lens = keep_drafts(slab, table, lens + n, accepted, num_drafts=n)
        assert int(lens[0]) == context + len(path)
        # The accepted tokens by themselves
        at = context + torch.arange(len(path), dtype=torch.int32, device=dev)
        qp = append(plain, x[path], at.expand(3, len(path)), slots_of(at))
        assert torch.equal(bits(qp), bits(q[path]))
        rows = slots_of(torch.arange(int(lens[0]), dtype=torch.int32, device=dev)).long()
        flat = lambda c: c.view(2, layers, -1, hkv, d)[:, :, rows]  # noqa: E731
        assert torch.equal(bits(flat(slab)), bits(flat(plain)))
        ref_out, limit = ref.prefill(qp.cpu(), plain[0, 1].cpu(), plain[1, 1].cpu(), table.cpu(), torch.tensor([0, len(path)]), lens.cpu(),
                                     page, d ** -0.5, True, cap or 0.0, None if sl is None else sl.cpu())
        within(out[0, path], ref_out, limit, f"step {step}")
