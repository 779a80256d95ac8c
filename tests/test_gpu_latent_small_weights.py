"""Many weights far below their row's greatest, as behind a first token that takes most of the attention and has a
small value: what they sum to is not lost to the 16-bit weights of the second product."""
import math

import pytest
import torch

from helpers import say
from tileinfer_amd.kernels import latent_decode_paged_fn, latent_prefill_fn

pytestmark = pytest.mark.gpu
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def _limit(exact, n, dtype, score, dims):
    """Of an output whose n - 1 small weights stand beside values of one: the weights' and the output's half steps, a 32-bit
    score's error in the weight and in the sum, 32-bit sums; fp16 weights have steps of 2^-24 once lifted by 2^7."""
    small = n * 2.0 ** -32 if dtype == torch.float16 else 0.0
    return exact * (2 * HALF[dtype] + 2 * (dims + 4) * 2.0 ** -24 * score + (n + 16) * 2.0 ** -23) + small


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("bits", [20.5, 25.6])
@pytest.mark.parametrize("heads", [300, 2])
def test_prefill(dtype, bits, heads, dev):
    """One workgroup a unit, and cut units."""
    n = 60000
    say(f"latent prefill small weights {dtype} 2^-{bits} H={heads}")
    q = torch.zeros(1, heads, 128, dtype=dtype, device=dev)
    q[..., 64] = 1
    kv = torch.zeros(n, 1, 128, dtype=dtype, device=dev)
    kv[1:, :, 64:] = 1
    kr = torch.zeros(n, 64, dtype=dtype, device=dev)
    kr[0, 0] = 8
    scale = bits * math.log(2) / 8
    cu_q, cu_k = (torch.tensor([0, x], dtype=torch.int32, device=dev) for x in (1, n))
    out = latent_prefill_fn(q, kv.expand(n, heads, 128), kr, cu_q, cu_k, 1, scale=scale).double()
    exact = (n - 1) * 2.0 ** -bits / (1 + (n - 1) * 2.0 ** -bits)
    limit = _limit(exact, n, dtype, bits, 128)
    say(f"  {exact:.3e}: off by {(out - exact).abs().max().item() / exact:.2e} of it, limit {limit / exact:.2e}")
    assert ((out - exact).abs() <= limit).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("bits", [20.5, 25.6])
@pytest.mark.parametrize("latent", [256, 512])
def test_decode(dtype, bits, latent, dev):
    """64 sequences, so that a run holds whole ones."""
    n, b, heads = 8192, 64, 24
    say(f"latent decode small weights {dtype} 2^-{bits} L={latent}")
    q = torch.zeros(b, heads, latent + 64, dtype=dtype, device=dev)
    q[..., latent] = 1
    cache = torch.zeros(n // 16 + 1, 16, 1, latent + 64, dtype=dtype, device=dev)
    cache[..., :latent] = 1
    cache[0, 0, 0, :latent], cache[0, 0, 0, latent] = 0, 8
    table = torch.arange(n // 16, dtype=torch.int32, device=dev).expand(b, n // 16).contiguous()
    lens = torch.full((b,), n, dtype=torch.int32, device=dev)
    out = latent_decode_paged_fn(q, cache, table, lens, scale=bits * math.log(2) / 8).double()
    exact = (n - 1) * 2.0 ** -bits / (1 + (n - 1) * 2.0 ** -bits)
    limit = _limit(exact, n, dtype, bits, latent + 64)
    say(f"  {exact:.3e}: off by {(out - exact).abs().max().item() / exact:.2e} of it, limit {limit / exact:.2e}")
    assert ((out - exact).abs() <= limit).all()
