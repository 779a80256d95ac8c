"""Latent attention (input side, absorbed decode on the pages, expanded prefill) against its 64-bit form."""
import pytest
import torch

from helpers import bits, say
from oracle import ref_latent as ref
from tileinfer_amd.kernels import latent_decode_paged_fn, latent_prefill_fn, latent_rope_append

pytestmark = pytest.mark.gpu
BF16, F16 = torch.bfloat16, torch.float16
SCALE = 192 ** -0.5


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _within(out, exact, limit, what=""):
    out = out.double().cpu()
    assert torch.isfinite(out).all(), f"{what}: values that are not finite"
    worst = ((out - exact).abs() / limit).max().item() if out.numel() else 0.0
    say(f"  {what}: worst error is {worst:.3f} of its limit")
    assert worst <= 1.0


def _paged(lens, page, row, dtype, seed, extra=3, width=None):
    """A cache whose unused rows are NaN, and tables of shuffled blocks with -1 behind."""
    g = _gen(seed)
    counts = [-(-max(n, 0) // page) for n in lens]
    blocks = sum(counts) + extra
    perm = torch.randperm(blocks, generator=g).tolist()
    width = width or max(max(counts), 1)
    table = torch.full((len(lens), width), -1, dtype=torch.int32)
    cache = torch.full((blocks, page, 1, row), torch.nan).to(dtype)
    at = 0
    for i, (n, c) in enumerate(zip(lens, counts)):
        table[i, :c] = torch.tensor(perm[at:at + c], dtype=torch.int32)
        at += c
        for t in range(n):
            cache[table[i, t // page], t % page, 0] = torch.randn(row, generator=g).to(dtype)
    return cache, table, torch.tensor(lens, dtype=torch.int32)


DECODES = [
    # heads, new tokens, latent, page, dtype, lengths
    (24, 1, 512, 16, BF16, [1, 31, 32, 33, 700, 0]),
    (32, 1, 512, 8, F16, [65, 2, 1000]),
    (1, 1, 512, 16, BF16, [100]),
    (16, 1, 256, 32, BF16, [5, 64, 257]),
    (17, 1, 256, 1, F16, [40, 1100]),
    (6, 3, 512, 4, BF16, [2, 3, 4, 90]),
    (24, 3, 512, 16, F16, [1, 500, 34]),
    (32, 4, 256, 24, BF16, [3, 130, 40]),
    (128, 1, 512, 16, BF16, [77, 300]),
    (128, 2, 256, 64, F16, [1, 150]),
    (12, 1, 512, 2, BF16, [33] * 70 + [0, 1]),
]


@pytest.mark.parametrize("heads,new,latent,page,dtype,lens", DECODES)
def test_decode_matches_formula(heads, new, latent, page, dtype, lens, dev):
    say(f"latent decode H={heads} N={new} L={latent} page={page} {dtype} lens={lens[:6]}")
    cache, table, n = _paged(lens, page, latent + 64, dtype, 11)
    q = torch.randn(len(lens), new, heads, latent + 64, generator=_gen(12)).to(dtype)
    exact, limit = ref.latent_decode(q, cache, table, n, page, SCALE)
    out = latent_decode_paged_fn(q.to(dev), cache.to(dev), table.to(dev), n.to(dev), page, scale=SCALE)
    assert out.shape == (len(lens), new, heads, latent) and out.dtype == dtype
    _within(out, exact, limit, "decode")
    if new == 1:
        again = latent_decode_paged_fn(q[:, 0].to(dev), cache.to(dev), table.to(dev), n.to(dev), page, scale=SCALE)
        assert again.shape == (len(lens), heads, latent)
        assert torch.equal(bits(again), bits(out[:, 0]))


@pytest.mark.parametrize("latent,heads,length", [(512, 24, 5000), (256, 32, 9001)])
def test_decode_long_sequences_cut_into_runs(latent, heads, length, dev):
    say(f"latent decode long L={latent} H={heads} n={length}")
    g = _gen(3)
    page, dtype = 16, BF16
    lens = [length, 17, length // 2, 0, 1]
    counts = [-(-n // page) for n in lens]
    cache = torch.randn(sum(counts), page, 1, latent + 64, generator=g).to(dtype)
    perm = torch.randperm(sum(counts), generator=g)
    table = torch.full((len(lens), max(counts) + 5), -1, dtype=torch.int32)
    at = 0
    for i, c in enumerate(counts):
        table[i, :c] = perm[at:at + c]
        at += c
    n = torch.tensor(lens, dtype=torch.int32)
    q = torch.randn(len(lens), 1, heads, latent + 64, generator=g).to(dtype)
    exact, limit = ref.latent_decode(q, cache, table, n, page, 0.2)
    out = latent_decode_paged_fn(q.to(dev), cache.to(dev), table.to(dev), n.to(dev), page, scale=0.2)
    _within(out, exact, limit, "decode")


def test_decode_absent_blocks_and_scores_of_any_size(dev):
    """Block ids outside the cache are masked, a row that sees nothing is zero, scores of +-10^4 and equal
    ones stay finite."""
    say("latent decode absent blocks")
    cache, table, n = _paged([70, 40, 33], 8, 576, BF16, 5, width=12)
    table[0, 3], table[0, 0], table[1, 4] = -1, 10 ** 6, -7
    table[2, :5] = -1
    q = torch.randn(3, 2, 24, 576, generator=_gen(6)).to(BF16)
    q[1] *= 60
    q[0, 0] = 0
    exact, limit = ref.latent_decode(q, cache, table, n, 8, SCALE)
    out = latent_decode_paged_fn(q.to(dev), cache.to(dev), table.to(dev), n.to(dev), 8, scale=SCALE)
    _within(out, exact, limit, "decode")
    assert (out[2] == 0).all()


def test_decode_strided_queries_out_and_graph(dev):
    """Queries and results in larger buffers, a captured call replayed with other lengths."""
    say("latent decode strides and graph")
    cache, table, n = _paged([300, 45], 16, 576, BF16, 8, width=30)
    big = torch.randn(2, 30, 600, generator=_gen(9)).to(BF16).to(dev)
    q = big[:, 3:27, 8:584]
    out = torch.empty(2, 24, 512, dtype=BF16, device=dev)
    c, t, l = cache.to(dev), table.to(dev), n.to(dev)
    r = latent_decode_paged_fn(q, c, t, l, 16, scale=SCALE, out=out)
    assert r is out
    exact, limit = ref.latent_decode(q.cpu().unsqueeze(1), cache, table, n, 16, SCALE)
    _within(out, exact[:, 0], limit[:, 0], "strided")
    odd = big[:, 3:27, 4:580]  # rows that are not 16-byte aligned: copied
    e2, l2 = ref.latent_decode(odd.cpu().unsqueeze(1), cache, table, n, 16, SCALE)
    _within(latent_decode_paged_fn(odd, c, t, l, 16, scale=SCALE), e2[:, 0], l2[:, 0], "odd")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        latent_decode_paged_fn(q, c, t, l, 16, scale=SCALE)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        g_out = latent_decode_paged_fn(q, c, t, l, 16, scale=SCALE)
    for lens in ([300, 45], [1, 44], [299, 0], [300, 45]):
        l.copy_(torch.tensor(lens, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        eager = latent_decode_paged_fn(q, c, t, l, 16, scale=SCALE)
        assert torch.equal(bits(g_out), bits(eager)), lens


def test_decode_of_an_empty_batch_and_empty_sequences(dev):
    say("latent decode empty")
    cache, table, n = _paged([20], 16, 576, BF16, 8)
    c, t, l = cache.to(dev), table.to(dev), n.to(dev)
    q = torch.randn(1, 24, 576, generator=_gen(2)).to(BF16).to(dev)
    assert latent_decode_paged_fn(q[:0], c, t[:0], l[:0], 16, scale=SCALE).shape == (0, 24, 512)
    assert (latent_decode_paged_fn(q, c, t, l * 0, 16, scale=SCALE) == 0).all()
    assert (latent_decode_paged_fn(q, c, t, l - 100, 16, scale=SCALE) == 0).all()
    assert (latent_decode_paged_fn(q, c, t[:, :0], l, 16, scale=SCALE) == 0).all()
    # a length beyond the table counts as the table's
    over = latent_decode_paged_fn(q, c, t[:, :1], l + 10 ** 9, 16, scale=SCALE)
    exact, limit = ref.latent_decode(q.cpu().unsqueeze(1), cache, table[:, :1], n, 16, SCALE)
    _within(over, exact[:, 0], limit[:, 0], "over")


PREFILLS = [
    # heads, dim, dtype, (query, key) lengths, causal
    (3, 128, BF16, [(1, 1)], True),
    (4, 128, BF16, [(130, 130), (1, 77), (0, 5), (64, 64), (33, 300)], True),
    (2, 64, F16, [(200, 200), (17, 17), (128, 1000)], True),
    (8, 64, BF16, [(5, 3), (70, 65), (129, 0)], True),
    (2, 128, F16, [(257, 640)], False),
    (1, 64, BF16, [(31, 63), (65, 66)], False),
    # more units than CUs: one workgroup each
    (48, 64, BF16, [(700, 700), (1, 9), (50, 130)], True),
    (33, 128, F16, [(1100, 1100)], True),
    # sequences in the order of their keys, equal and empty ones among them
    (33, 64, BF16, [(300, 1500), (0, 900), (300, 1500), (1, 3000), (130, 131), (0, 0), (200, 2100)], True),
    (40, 128, F16, [(200, 1100), (700, 1300), (129, 1100)], False),
    # long first chunks of few units: two key groups
    (40, 128, BF16, [(1100, 1100)], True),
    (20, 64, F16, [(1030, 1050), (1301, 1281)], True),
    (14, 128, F16, [(1, 1), (2500, 2499), (600, 601)], True),
    # cut units: few heads over long keys, blocks that see nothing, empty sequences between others
    (2, 128, BF16, [(300, 2500), (0, 0), (0, 40), (400, 130), (1, 1999)], True),
    (1, 64, F16, [(129, 3001)] + [(3, 70)] * 70, True),
]


@pytest.mark.parametrize("heads,dim,dtype,lens,is_causal", PREFILLS)
def test_prefill_matches_formula(heads, dim, dtype, lens, is_causal, dev):
    say(f"latent prefill H={heads} D={dim} {dtype} {lens} causal={is_causal}")
    g = _gen(21)
    cu_q = torch.tensor([0] + [a for a, _ in lens]).cumsum(0).to(torch.int32)
    cu_k = torch.tensor([0] + [b for _, b in lens]).cumsum(0).to(torch.int32)
    tq, tk = int(cu_q[-1]), int(cu_k[-1])
    q = torch.randn(tq, heads, dim + 64, generator=g).to(dtype)
    kv = torch.randn(tk, heads, 2 * dim, generator=g).to(dtype)
    wide = torch.randn(tk, 512 + 64, generator=g).to(dtype)
    scale = (dim + 64) ** -0.5
    exact, limit = ref.latent_prefill(q, kv, wide[:, 512:], cu_q, cu_k, scale, is_causal)
    out = latent_prefill_fn(q.to(dev), kv.to(dev), wide.to(dev)[:, 512:], cu_q.to(dev), cu_k.to(dev),
                            max(a for a, _ in lens), causal=is_causal)
    assert out.shape == (tq, heads, dim) and out.dtype == dtype
    _within(out, exact, limit, "prefill")


def test_prefill_keeps_to_its_rows(dev):
    """Rows behind the last sequence stay as they were, what lies behind the last key is not read, a longer
    bound changes nothing, and a captured call repeats."""
    say("latent prefill rows")
    g = _gen(22)
    lens = [(40, 100), (3, 3)]
    cu_q = torch.tensor([0, 40, 43], dtype=torch.int32)
    cu_k = torch.tensor([0, 100, 103], dtype=torch.int32)
    q = torch.full((60, 4, 192), torch.nan).to(BF16)
    kv, kr = torch.full((200, 4, 256), torch.nan).to(BF16), torch.full((200, 64), torch.nan).to(BF16)
    q[:43] = torch.randn(43, 4, 192, generator=g)
    kv[:103] = torch.randn(103, 4, 256, generator=g)
    kr[:103] = torch.randn(103, 64, generator=g)
    exact, limit = ref.latent_prefill(q[:43], kv, kr, cu_q, cu_k, 0.1)
    out = torch.full((60, 4, 128), 7.0, dtype=BF16, device=dev)
    args = [x.to(dev) for x in (q, kv, kr, cu_q, cu_k)]
    latent_prefill_fn(*args, 40, scale=0.1, out=out)
    _within(out[:43], exact, limit, "prefill")
    assert (out[43:] == 7.0).all()
    assert torch.equal(bits(latent_prefill_fn(*args, 60, scale=0.1)[:43]), bits(out[:43]))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        r = latent_prefill_fn(*args, 40, scale=0.1)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(bits(r[:43]), bits(out[:43]))


APPENDS = [(1, 24, 512, BF16, 0), (33, 24, 512, BF16, 3), (257, 5, 256, F16, 0), (70, 0, 256, BF16, 0),
           (19, 1, 512, F16, 1)]


@pytest.mark.parametrize("tokens,heads,latent,dtype,skipped", APPENDS)
def test_append_matches_formula(tokens, heads, latent, dtype, skipped, dev):
    say(f"latent append T={tokens} H={heads} L={latent} {dtype}")
    g = _gen(31)
    both = torch.randn(tokens, latent + 64, generator=g).to(dtype)  # one projection's output
    c, kr = 3 * both[:, :latent], both[:, latent:]
    qr = torch.randn(tokens, heads, 64, generator=g).to(dtype) if heads else None
    w = (0.2 * torch.randn(latent, generator=g)).to(dtype)
    angle = torch.rand(tokens, 32, generator=g) * 6.28
    cos, sin = (torch.cat([f(angle)] * 2, -1).to(dtype) for f in (torch.cos, torch.sin))
    slots = torch.randperm(tokens + 40, generator=g)[:tokens].to(torch.int32)
    if skipped:
        slots[:skipped] = torch.tensor([-1, 10 ** 6, -5])[:skipped]
    cache = torch.full((tokens + 40, latent + 64), 5.0).to(dtype).to(dev)
    c = c.to(dtype)
    got = latent_rope_append(None if qr is None else qr.to(dev), c.to(dev), kr.to(dev), w.to(dev), cos.to(dev),
                             sin.to(dev), cache, slots.to(dev), 1e-6)
    h = ref.half_step(dtype)
    rows = ref.latent_rows(c, kr, w, cos, sin, 1e-6, 1.0)
    live = (slots >= 0) & (slots < tokens + 40)
    # one rounding of the value, 32-bit arithmetic on the way; a rotation's two terms may cancel
    size = torch.cat([rows[:, :latent].abs(), (kr.double().abs() + kr.double().abs().roll(32, -1))], -1)
    _within(cache.cpu()[slots[live].long()], rows[live], (h * rows.abs() + 2.0 ** -18 * size + 2.0 ** -24)[live], "rows")
    rest = torch.ones(tokens + 40, dtype=torch.bool)
    rest[slots[live].long()] = False
    assert (cache.cpu()[rest] == 5.0).all()
    if heads:
        exact = ref.rotate(qr, cos[:, None], sin[:, None])
        size = qr.double().abs() + qr.double().abs().roll(32, -1)
        _within(got, exact, h * exact.abs() + 2.0 ** -20 * size + 2.0 ** -24, "q")
    else:
        assert got is None


def test_append_into_the_queries_and_plain_weights(dev):
    """The rotated parts land in the last columns of the queries, in place too; a weight that is the whole
    factor; one cos / sin row for all tokens; operands whose rows are not aligned."""
    say("latent append q_out")
    g = _gen(32)
    t, h = 9, 6
    q = torch.randn(t, h, 576, generator=g).to(BF16).to(dev)
    before = q.clone()
    c, kr = (torch.randn(t, n, generator=g).to(BF16).to(dev) for n in (512, 64))
    w = torch.rand(512, generator=g).to(BF16).to(dev)
    cos, sin = torch.rand(64, generator=g).to(BF16).to(dev), torch.rand(64, generator=g).to(BF16).to(dev)
    cache = torch.zeros(20, 576, dtype=BF16, device=dev)
    slots = torch.arange(t, dtype=torch.int32, device=dev)
    r = latent_rope_append(q[..., 512:], c, kr, w, cos, sin, cache, slots, weight_offset=0.0, q_out=q[..., 512:])
    assert r.data_ptr() == q[..., 512:].data_ptr()
    assert torch.equal(bits(q[..., :512]), bits(before[..., :512]))
    plain = latent_rope_append(before[..., 512:], c, kr, w, cos[None].expand(t, 64), sin[None].expand(t, 64),
                               cache.clone(), slots, weight_offset=0.0)
    assert torch.equal(bits(plain), bits(q[..., 512:]))
    rows = ref.latent_rows(c.cpu(), kr.cpu(), w.cpu(), cos.cpu()[None], sin.cpu()[None], 1e-5, 0.0)
    _within(cache[:t], rows, 2.0 ** -8 * rows.abs() + 2.0 ** -16, "rows")
    shifted = torch.zeros(t * 512 + 4, dtype=BF16, device=dev)[4:].view(t, 512).copy_(c)
    other = torch.zeros_like(cache)
    latent_rope_append(None, shifted, kr, w, cos, sin, other, slots, weight_offset=0.0)
    assert torch.equal(bits(other), bits(cache))


def test_a_latent_layer_end_to_end(dev):
    """A prompt prefilled in two chunks with the expanded form, then decoded with the absorbed one: both give
    the attention over the same cached latents, step by step."""
    say("latent layer end to end")
    g = _gen(41)
    h, dim, latent, page, dtype = 6, 128, 512, 16, BF16
    wk = (torch.randn(h, latent, dim, generator=g) * latent ** -0.5).to(dev)
    wv = (torch.randn(h, latent, dim, generator=g) * latent ** -0.5).to(dev)
    norm_w = torch.zeros(latent, dtype=dtype, device=dev)
    cache = torch.zeros(12, page, 1, latent + 64, dtype=dtype, device=dev)
    table = torch.tensor([[3, 1, 7, 0, 9, 11]], dtype=torch.int32, device=dev)
    flat = cache.view(-1, latent + 64)
    scale = (dim + 64) ** -0.5
    done = 0
    for chunk in (40, 23, 1, 1):
        c = torch.randn(chunk, latent, generator=g).to(dtype).to(dev)
        kr = torch.randn(chunk, 64, generator=g).to(dtype).to(dev)
        q_nope = torch.randn(chunk, h, dim, generator=g).to(dtype).to(dev)
        q_rope = torch.randn(chunk, h, 64, generator=g).to(dtype).to(dev)
        pos = torch.arange(done, done + chunk, device=dev)
        angle = pos[:, None] * 1e4 ** (-torch.arange(32, device=dev) / 32)
        cos, sin = (torch.cat([f(angle)] * 2, -1).to(dtype) for f in (torch.cos, torch.sin))
        slots = (table[0, pos // page] * page + pos % page).to(torch.int32)
        q_rot = latent_rope_append(q_rope, c, kr, norm_w, cos, sin, flat, slots)
        done += chunk
        every = torch.arange(done, device=dev)
        rows = flat[(table[0, every // page] * page + every % page).long()]
        kv = torch.cat([torch.einsum("tl,hld->thd", rows[:, :latent].float(), w) for w in (wk, wv)], -1).to(dtype)
        expanded = latent_prefill_fn(
            torch.cat([q_nope, q_rot], -1), kv, rows[:, latent:],
            torch.tensor([0, chunk], dtype=torch.int32, device=dev),
            torch.tensor([0, done], dtype=torch.int32, device=dev), chunk)
        q_abs = torch.cat([torch.einsum("thd,hld->thl", q_nope.float(), wk).to(dtype), q_rot], -1)
        o = latent_decode_paged_fn(q_abs[None], cache, table, torch.tensor([done], dtype=torch.int32, device=dev),
                                   page, scale=scale)[0]
        absorbed = torch.einsum("thl,hld->thd", o.float(), wv)
        # Both round kv or q and o to 16 bits (2^-8 each of terms of about one) and P twice.
        torch.testing.assert_close(expanded.float(), absorbed, atol=6 * 2.0 ** -8, rtol=2.0 ** -6)


@pytest.mark.parametrize("shared", [False, True])
def test_decode_of_many_tiles_streams_or_keeps_shared_pages(shared, dev):
    """Enough tiles for the streaming loads, with private pages and with a prefix that half of the batch shares:
    the same values through either table."""
    say(f"latent decode many tiles shared={shared}")
    g = torch.Generator(device=dev).manual_seed(51)
    page, b, width = 16, 40, 130
    lens = torch.randint(1500, width * page + 1, (b,), generator=g, device=dev, dtype=torch.int32)
    pool = torch.randn(b * width, page, 1, 576, generator=g, device=dev).to(BF16)
    table = torch.randperm(b * width, generator=g, device=dev).to(torch.int32).view(b, width)
    if shared:
        for i in range(1, b // 2):
            pool[table[i, :50].long()] = pool[table[0, :50].long()]
    q = torch.randn(b, 24, 576, generator=g, device=dev).to(BF16)
    out = latent_decode_paged_fn(q, pool, table, lens, page, scale=SCALE)
    if shared:
        one = table.clone()
        one[1:b // 2, :50] = table[0, :50]
        assert torch.equal(bits(latent_decode_paged_fn(q, pool, one, lens, page, scale=SCALE)), bits(out))
    for i in (0, b // 2, b - 1):
        exact, limit = ref.latent_decode(q[i:i + 1, None].cpu(), pool.cpu(), table[i:i + 1].cpu(), lens[i:i + 1].cpu(),
                                         page, SCALE)
        _within(out[i:i + 1, None], exact, limit, f"sequence {i}")
