"""First chunks around the sizes at which the expanded prefill shares a tile's keys between two groups of waves, against
the 64-bit form."""
import pytest
import torch

from helpers import say
from oracle import ref_latent as ref
from tileinfer_amd.kernels import latent_prefill_fn

pytestmark = pytest.mark.gpu
BF16, F16 = torch.bfloat16, torch.float16

CHUNKS = [
    # heads, dim, dtype, (query, key) lengths: as many keys as queries in all
    (40, 128, F16, [(1027, 1027)]),
    (20, 128, BF16, [(1030, 1050), (1301, 1281)]),
    (30, 128, F16, [(2050, 2051), (1, 0)]),
    (40, 64, BF16, [(1155, 1155)]),
    (33, 64, F16, [(1024, 1024)]),
    # more sequences than share them
    (20, 64, BF16, [(1030, 1050), (1301, 1281)]),
    (14, 128, F16, [(1100, 1100), (1099, 1101), (1302, 1300)]),
    (40, 64, F16, [(0, 0), (1155, 1155)]),
]


@pytest.mark.parametrize("heads,dim,dtype,lens", CHUNKS)
def test_first_chunks_of_few_units(heads, dim, dtype, lens, dev):
    say(f"latent prefill key groups H={heads} D={dim} {dtype} {lens}")
    g = torch.Generator().manual_seed(71)
    cu_q, cu_k = (torch.tensor([0] + [x[i] for x in lens]).cumsum(0).to(torch.int32) for i in (0, 1))
    total = int(cu_q[-1])
    assert total == int(cu_k[-1])
    units = -(-total // 128) * heads
    cus = torch.cuda.get_device_properties(dev).multi_processor_count
    assert cus < units <= 2 * cus
    q = torch.randn(total, heads, dim + 64, generator=g).to(dtype)
    kv = torch.randn(total, heads, 2 * dim, generator=g).to(dtype)
    kr = torch.randn(total, 64, generator=g).to(dtype)
    some = [0, heads // 2, heads - 1]
    exact, limit = ref.latent_prefill(q[:, some], kv[:, some], kr, cu_q, cu_k, (dim + 64) ** -0.5)
    args = [x.to(dev) for x in (q, kv, kr, cu_q, cu_k)]
    out = latent_prefill_fn(*args, max(a for a, _ in lens))
    assert torch.equal(out, latent_prefill_fn(*args, max(a for a, _ in lens)))
    got = out[:, some].double().cpu()
    worst = ((got - exact).abs() / limit).max().item()
    say(f"  worst error is {worst:.3f} of its limit")
    assert torch.isfinite(got).all() and worst <= 1.0
