"""Operands of the latent and eviction calls in forms that their documentation allows: columns of wider tables, rows off
their alignment, host numbers of any size."""
import pytest
import torch

from helpers import bits, say
from oracle import ref_latent as ref
from tileinfer_amd.kernels import (evict_kvcache, gqa_prefill_paged_fn, latent_decode_paged_fn,
                                   latent_prefill_fn)

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def _randn(dev, *shape, seed=0, dtype=BF16):
    return torch.randn(*shape, device=dev, generator=torch.Generator(dev).manual_seed(seed)).to(dtype)


@pytest.mark.parametrize("heads", [2, 150])
def test_prefill_offsets_as_columns_of_one_table(heads, dev):
    """Both offsets strided, with as many bytes each and different values: their copies live until the launch."""
    say(f"latent prefill, offsets as columns, H={heads}")
    both = torch.tensor([[0, 0], [40, 100], [75, 175], [90, 400]], dtype=torch.int32, device=dev)
    q, kv, kr = _randn(dev, 90, heads, 128), _randn(dev, 400, heads, 128, seed=1), _randn(dev, 400, 64, seed=2)
    want = latent_prefill_fn(q, kv, kr, both[:, 0].contiguous(), both[:, 1].contiguous(), 40)
    torch.cuda.synchronize()
    for _ in range(3):
        got = latent_prefill_fn(q, kv, kr, both[:, 0], both[:, 1], 40, out=torch.zeros_like(want))
        assert torch.equal(bits(got), bits(want))


def _right(got, exact, limit):
    got = got.double().cpu()
    assert torch.isfinite(got).all() and ((got - exact).abs() <= limit).all()


@pytest.mark.parametrize("heads,q_len,k_len,at", [
    (2, 200, 240, 70), (2, 200, 240, 130), (2, 200, 205, 191), (150, 200, 240, 130),  # cut units; one workgroup a unit
    (16, 2500, 2500, 70), (16, 2500, 2500, 2431)])                                    # two key groups
@pytest.mark.parametrize("what", ["inf", "nan"])
def test_prefill_reach_of_a_value_that_is_not_finite(heads, q_len, k_len, at, what, dev):
    """Queries whose 32 see no key of the value's 64 are right; a key that is not finite reaches only those that see it."""
    say(f"latent prefill, {what} at {at}, H={heads} {q_len}/{k_len}")
    q, kv, kr = _randn(dev, q_len, heads, 128), _randn(dev, k_len, heads, 128, seed=1), _randn(dev, k_len, 64, seed=2)
    cu_q, cu_k = (torch.tensor([0, n], dtype=torch.int32, device=dev) for n in (q_len, k_len))
    offset = k_len - q_len
    group = next(g for g in range(q_len) if offset + min(32 * g + 31, q_len - 1) >= at // 64 * 64)
    n = min(32 * group, 96)  # rows compared
    exact, limit = ref.latent_prefill(q[:n].cpu(), kv.cpu(), kr.cpu(), [0, n], [0, offset + n], 128 ** -0.5)
    bad = kv.clone()
    bad[at, :, 64:] = float(what)
    out = latent_prefill_fn(q, bad, kr, cu_q, cu_k, q_len)
    assert torch.isfinite(out[:32 * group]).all()
    _right(out[:n], exact, limit)
    assert not torch.isfinite(out[max(0, at - offset):]).any()
    plain = latent_prefill_fn(q, kv, kr, cu_q, cu_k, q_len)
    bad = kv.clone()
    bad[at, :, :64] = float("nan")
    out = latent_prefill_fn(q, bad, kr, cu_q, cu_k, q_len)
    first = max(0, at - offset)
    assert torch.equal(bits(out[:first]), bits(plain[:first])) and torch.isnan(out[first:]).all()


def test_decode_reach_of_a_row_that_is_not_finite(dev):
    """It stays in its sequence; its rotated part reaches only the queries that see it."""
    say("latent decode, rows that are not finite")
    cache = _randn(dev, 12, 16, 1, 320)
    table = torch.arange(12, dtype=torch.int32, device=dev).view(3, 4)
    lens = torch.tensor([40, 50, 64], dtype=torch.int32, device=dev)
    q = _randn(dev, 3, 3, 24, 320, seed=1)
    plain = latent_decode_paged_fn(q, cache, table, lens, scale=0.05)
    for part in (slice(0, 256), slice(256, 320)):
        bad = cache.clone()
        bad[7, 1, 0, part] = float("nan")  # token 49 of sequence 1, its last one
        out = latent_decode_paged_fn(q, bad, table, lens, scale=0.05)
        assert torch.equal(bits(out[[0, 2]]), bits(plain[[0, 2]])) and torch.isnan(out[1, 2]).all()
        if part.start:
            assert torch.equal(bits(out[1, :2]), bits(plain[1, :2]))


def test_host_numbers_beyond_32_bits(dev):
    """A bound on the chunks' length may be any number; a budget that does not fit the call is refused."""
    say("host numbers beyond 32 bits")
    cu = torch.tensor([0, 40, 90], dtype=torch.int32, device=dev)
    q, kv, kr = _randn(dev, 90, 3, 192), _randn(dev, 90, 3, 256, seed=1), _randn(dev, 90, 64, seed=2)
    want = latent_prefill_fn(q, kv, kr, cu, cu, 50)
    for bound in (2 ** 31 - 1, 2 ** 31, 2 ** 32, 2 ** 33 + 7, 2 ** 70):
        assert torch.equal(bits(latent_prefill_fn(q, kv, kr, cu, cu, bound, out=torch.zeros_like(want))), bits(want))
    k, v = _randn(dev, 8, 16, 2, 128), _randn(dev, 8, 16, 2, 128, seed=1)
    table = torch.arange(8, dtype=torch.int32, device=dev).view(2, 4)
    q, lens = _randn(dev, 90, 4, 128), torch.tensor([40, 60], dtype=torch.int32, device=dev)
    want = gqa_prefill_paged_fn(q, k, v, table, cu, lens, 50)
    for bound in (2 ** 31, 2 ** 32, 2 ** 70):
        got = gqa_prefill_paged_fn(q, k, v, table, cu, lens, bound, out=torch.zeros_like(want))
        assert torch.equal(bits(got), bits(want))
    mass = torch.rand(2, 2, 32, device=dev)
    for budget in (2 ** 31, 2 ** 32 + 16, 2 ** 70):
        with pytest.raises(ValueError, match="budget"):
            evict_kvcache(k, v, mass, table[:, :2], lens, table[:, 2:], budget, 16)


@pytest.mark.parametrize("heads", [2, 150])
def test_prefill_offsets_that_go_back(heads, dev):
    """A sequence whose end lies before its start is empty, one that starts inside another has its own keys; offsets stay
    within the tensors. Rows that two sequences claim get either result."""
    say(f"latent prefill offsets that go back, H={heads}")
    q, kv, kr = _randn(dev, 300, heads, 128), _randn(dev, 500, heads, 128, seed=1), _randn(dev, 500, 64, seed=2)
    i = lambda *x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    out = latent_prefill_fn(q, kv, kr, i(-5, 200, 100, 2 ** 31 - 1), i(0, 320, 40, 2 ** 31 - 1), 300)
    first = latent_prefill_fn(q[:200], kv[:320], kr[:320], i(0, 200), i(0, 320), 200, out=torch.empty_like(out[:200]))
    last = latent_prefill_fn(q[100:], kv[40:], kr[40:], i(0, 200), i(0, 460), 200)
    near = dict(rtol=2.0 ** -6, atol=2.0 ** -7)  # other cuts: P and the output rounded apart
    torch.testing.assert_close(out[:100], first[:100], **near)
    torch.testing.assert_close(out[200:], last[100:], **near)
    assert torch.isfinite(out[100:200]).all()
