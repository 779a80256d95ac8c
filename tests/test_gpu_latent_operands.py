"""Operands of the latent and eviction calls in forms that their documentation allows: columns of wider tables, rows off
their alignment, host numbers of any size."""
import pytest
import torch

from helpers import bits, say
from tileinfer_amd.kernels import latent_prefill_fn

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
