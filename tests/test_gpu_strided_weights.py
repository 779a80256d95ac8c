"""The input side's two norm weights as columns of one table."""
import pytest
import torch

from helpers import bits, say
from tileinfer_amd.kernels import qknorm_rope_append

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def test_qknorm_append_weights_as_columns_of_one_table(dev):
    """Both weights strided, with as many bytes each and different values: their copies live until the launch."""
    say("qknorm append, weights as columns")
    g = torch.Generator(dev).manual_seed(3)
    t, hq, hkv, d = 5, 4, 2, 256
    r = lambda *s: torch.randn(*s, device=dev, generator=g).to(BF16)  # noqa: E731
    q, k, v, both, cos, sin = r(t, hq, d), r(t, hkv, d), r(t, hkv, d), r(d, 2), r(t, 64), r(t, 64)
    slots = torch.arange(t, dtype=torch.int32, device=dev)

    def call(q_weight, k_weight):
        kc, vc = torch.zeros(8, hkv * d, dtype=BF16, device=dev), torch.zeros(8, hkv * d, dtype=BF16, device=dev)
        return qknorm_rope_append(q, k, v, q_weight, k_weight, cos, sin, kc, vc, slots), kc, vc

    want = call(both[:, 0].contiguous(), both[:, 1].contiguous())
    torch.cuda.synchronize()
    for _ in range(3):
        for x, y in zip(call(both[:, 0], both[:, 1]), want):
            assert torch.equal(bits(x), bits(y))
