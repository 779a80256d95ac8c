"""Rotation by several position axes of more than 128 values of a head of 256, the whole head among them."""
import pytest
import torch

from helpers import bits, say
from oracle import ref_shaped as ref
from test_gpu_draft_tree import within
from test_gpu_rope_axes import BF16, F16, _inputs
from tileinfer_amd.kernels import rope_axes_append

pytestmark = pytest.mark.gpu
CASES = [
    # tokens, heads, D, rotary, axes, norm, dtype, position type, far
    (1, 24, 4, 256, 256, 1, True, BF16, torch.int64, 10),
    (9, 24, 4, 256, 256, 3, False, F16, torch.int32, 10 ** 6),
    (33, 5, 1, 256, 144, 3, True, BF16, torch.int32, 131072),
    (6, 8, 2, 256, 240, 4, False, BF16, torch.int64, -5000),
    (1031, 24, 4, 256, 256, 2, True, F16, torch.int32, 40000),
    (1500, 16, 8, 256, 192, 1, False, BF16, torch.int64, 250000),
]


@pytest.mark.parametrize("case", CASES)
def test_matches_formula(case, dev):
    t, hq, hkv, d, rotary, na, norm, dtype, pdt, far = case
    say(f"rope of a whole head {case}")
    q, k, v, pos, inv, axes, (qw, kw), slots = _inputs(*case)
    to = lambda x: None if x is None else x.to(dev)  # noqa: E731
    caches = [torch.full((t + 9, hkv * d), 7.0, dtype=dtype, device=dev) for _ in range(2)]
    args = [*map(to, (q, k, v, pos, inv, axes)), *caches, to(slots)]
    out = rope_axes_append(*args, q_weight=to(qw), k_weight=to(kw), eps=1e-6)
    within(out, *ref.rope_axes(q, pos, inv, axes, qw, 1e-6, 1.0), "q")
    exact, limit = ref.rope_axes(k, pos, inv, axes, kw, 1e-6, 1.0)
    there = (slots >= 0) & (slots < t + 9)
    rows = slots[there].long()
    got = [c.cpu().view(-1, hkv, d) for c in caches]
    within(got[0][rows], exact[there], limit[there], "k")
    assert torch.equal(bits(got[1][rows]), bits(v[there]))
    # The other form of the call (the result's tensor given), over the queries themselves.
    again = args[0].clone()
    rope_axes_append(again, *args[1:], q_weight=to(qw), k_weight=to(kw), eps=1e-6, q_out=again)
    assert torch.equal(bits(again), bits(out))
