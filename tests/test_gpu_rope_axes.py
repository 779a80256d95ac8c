"""Rotation by several position axes, with and without norms, into the paged cache, against its 64-bit form."""
import pytest
import torch

from helpers import bits, say
from oracle import ref_shaped as ref
from test_gpu_draft_tree import within
from tileinfer_amd.kernels import rope_axes_append

pytestmark = pytest.mark.gpu
BF16, F16 = torch.bfloat16, torch.float16
CASES = [
    # tokens, heads, D, rotary, axes, norm, dtype, position type, far
    (1, 24, 4, 256, 64, 3, True, BF16, torch.int64, 10),
    (5, 24, 4, 256, 64, 3, True, F16, torch.int32, 10 ** 6),
    (33, 24, 4, 256, 64, 1, False, BF16, torch.int32, 131072),
    (7, 1, 1, 256, 128, 2, True, BF16, torch.int64, 2 ** 31 - 1),
    (9, 3, 1, 256, 16, 4, True, F16, torch.int32, 999),
    (6, 5, 2, 256, 0, 1, True, BF16, torch.int32, 5),
    (300, 24, 4, 256, 64, 3, True, BF16, torch.int64, 40000),
    (1031, 32, 8, 128, 128, 3, False, F16, torch.int32, 2 ** 30),
    (40, 32, 8, 128, 128, 3, True, BF16, torch.int64, 250000),
    (3, 20, 2, 128, 48, 3, False, BF16, torch.int32, 77),
    (17, 7, 7, 128, 32, 2, True, F16, torch.int64, -5000),
]


def _inputs(t, hq, hkv, d, rotary, na, norm, dtype, pdt, far, seed=5):
    g = torch.Generator().manual_seed(seed)
    q, k, v = (torch.randn(t, h, d, generator=g).to(dtype) for h in (hq, hkv, hkv))
    pos = torch.randint(min(far, 0), max(far, 1), (na, t), generator=g).to(pdt)
    pos[:, 0] = far
    half = rotary // 2
    inv = (1e6 ** (-torch.arange(half, dtype=torch.float64) / max(half, 1))).float()
    axes = torch.randint(-1, na + 1, (half,), generator=g).to(torch.int32) if na > 1 else None
    weights = [(0.2 * torch.randn(d, generator=g)).to(dtype) for _ in range(2)] if norm else [None, None]
    slots = torch.randperm(t + 9, generator=g)[:t].to(torch.int32)
    slots[::7] = -1
    if t > 2:
        slots[2] = t + 9
    return q, k, v, pos, inv, axes, weights, slots


@pytest.mark.parametrize("case", CASES)
def test_matches_formula(case, dev):
    t, hq, hkv, d, rotary, na, norm, dtype, pdt, far = case
    say(f"rope axes {case}")
    q, k, v, pos, inv, axes, (qw, kw), slots = _inputs(*case)
    to = lambda x: None if x is None else x.to(dev)  # noqa: E731
    for offset in (1.0, 0.0) if norm else (1.0,):
        caches = [torch.full((t + 9, hkv * d), 7.0, dtype=dtype, device=dev) for _ in range(2)]
        out = rope_axes_append(*map(to, (q, k, v, pos, inv, axes)), *caches, to(slots), q_weight=to(qw), k_weight=to(kw),
                               eps=1e-6, weight_offset=offset)
        exact, limit = ref.rope_axes(q, pos, inv, axes, qw, 1e-6, offset)
        within(out, exact, limit, "q")
        exact, limit = ref.rope_axes(k, pos, inv, axes, kw, 1e-6, offset)
        there = (slots >= 0) & (slots < t + 9)
        rows = slots[there].long()
        got = [c.cpu().view(-1, hkv, d) for c in caches]
        within(got[0][rows], exact[there], limit[there], "k")
        assert torch.equal(bits(got[1][rows]), bits(v[there]))
        rest = torch.ones(t + 9, dtype=torch.bool)
        rest[rows] = False
        assert all((c[rest] == 7).all() for c in got)


def test_both_launch_shapes_give_the_same_bits(dev):
    """A token's result does not depend on how many there are."""
    say("rope axes: few and many tokens")
    q, k, v, pos, inv, axes, (qw, kw), slots = [x if isinstance(x, list) or x is None else x.to(dev) for x in
                                                _inputs(1500, 24, 4, 256, 64, 3, True, BF16, torch.int32, 9999)]
    qw, kw = qw.to(dev), kw.to(dev)
    runs = []
    for n in (1500, 20):
        caches = [torch.zeros(1509, 1024, dtype=BF16, device=dev) for _ in range(2)]
        o = rope_axes_append(q[:n], k[:n], v[:n], pos[:, :n], inv, axes, *caches, slots[:n], q_weight=qw, k_weight=kw)
        at = slots[:20][(slots[:20] >= 0) & (slots[:20] < 1509)].long()
        runs.append([o[:20], caches[0][at], caches[1][at]])
    for a, b in zip(*runs):
        assert torch.equal(bits(a), bits(b))


def test_strided_operands_and_q_in_place(dev):
    """Slices of one projection, positions of which one axis is used twice, unaligned rows, the result over q."""
    say("rope axes: strides")
    q, k, v, pos, inv, axes, (qw, kw), slots = _inputs(12, 4, 2, 128, 128, 3, True, BF16, torch.int64, 500)
    to = lambda x: x.to(dev)  # noqa: E731
    want = [torch.zeros(21, 256, dtype=BF16, device=dev) for _ in range(2)]
    o = rope_axes_append(*map(to, (q, k, v, pos, inv, axes)), *want, to(slots), q_weight=to(qw), k_weight=to(kw))
    for form in ("projection", "odd", "transposed"):
        if form == "projection":
            both = torch.cat([q, k, v], 1).to(dev)
            a, b, c = both[:, :4], both[:, 4:6], both[:, 6:]
        elif form == "odd":
            a, b, c = (torch.cat([x.new_zeros(12, x.shape[1], 1), x], 2).to(dev)[..., 1:] for x in (q, k, v))
        else:
            a, b, c = (x.transpose(0, 1).contiguous().to(dev).transpose(0, 1) for x in (q, k, v))
        p = pos.t().contiguous().to(dev).t() if form == "odd" else pos.to(dev)
        got = [torch.zeros(21, 256, dtype=BF16, device=dev) for _ in range(2)]
        r = rope_axes_append(a, b, c, p, to(inv), to(axes), *got, to(slots), q_weight=to(qw), k_weight=to(kw),
                             q_out=a if form == "projection" else None)
        assert torch.equal(bits(r.contiguous()), bits(o))
        assert all(torch.equal(bits(x), bits(y)) for x, y in zip(got, want))
