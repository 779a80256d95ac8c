"""Caps far above the scores: the capped score of a small one is as exact as the score itself, for every cap that the
calls take, on each of their kernels."""
import pytest
import torch

from helpers import say
from oracle import ref_shaped as ref
from test_gpu_draft_tree import paged, slopes_of, within
from tileinfer_amd.kernels import gqa_prefill_shaped_fn, gqa_tree_paged_fn

pytestmark = pytest.mark.gpu
BF16, F16 = torch.bfloat16, torch.float16


def _two_keys(d, dtype, lens, seed):
    """Caches of which tokens 0 and 1 have the values +1 and -1, so that a row over both is the difference of their
    weights, where an error of their scores shows whole."""
    k, v, table, lens_t = paged(lens, 16, 2, d, dtype, seed)
    for b in range(len(lens)):
        block = int(table[b, 0])
        v[block, 0], v[block, 1] = 1.0, -1.0
    return k, v, table, lens_t


def _limit(q, k, scale, plain):
    """The limit of a call without a cap, which counts the roundings of the score and of the weights, and that of the cap:
    a dozen roundings of the capped score at most (2^-20 of it, which the uncapped one bounds), of two weights whose sum
    is one and whose values are one."""
    most = scale * q.double().abs().amax((0, 1, 2))[None].mul(k[:, :2].double().nan_to_num(0.0).abs().amax((0, 1, 2))).sum()
    return plain + 2 * 2.0 ** -20 * min(float(most), 1e4)


@pytest.mark.parametrize("cap", [257.0, 1000.0, 1e4])
@pytest.mark.parametrize("d,dtype", [(128, F16), (256, F16), (128, BF16)])
@pytest.mark.parametrize("drafts", [3, 40])  # either kernel
@pytest.mark.parametrize("slopes", [False, True])
@pytest.mark.parametrize("size", [1.0, 0.3])  # of the scores, times 1 or (the cap's curve) a third of the cap
def test_tree(cap, d, dtype, drafts, slopes, size, dev):
    say(f"tree, cap {cap} D={d} {dtype} N={drafts} slopes={slopes} {size}")
    lens = [drafts + 2] * 24
    k, v, table, lens_t = _two_keys(d, dtype, lens, 3)
    q = torch.randn(len(lens), drafts, 4, d, generator=torch.Generator().manual_seed(4)).to(dtype)
    scale = d ** -0.5 * (1.0 if size == 1.0 else size * cap)
    masks = torch.zeros(drafts, dtype=torch.int64)  # the drafts see the context alone
    sl = slopes_of(4) if slopes else None
    rows = [masks.tolist()] * len(lens)
    exact, _ = ref.tree(q, k, v, table, lens_t, rows, 16, scale, cap, sl)
    _, plain = ref.tree(q, k, v, table, lens_t, rows, 16, scale, 0.0, sl)
    out = gqa_tree_paged_fn(*(x.to(dev) for x in (q, k, v, table, lens_t, masks)), scale=scale, softcap=cap,
                            slopes=None if sl is None else sl.to(dev))
    within(out, exact, _limit(q, k[table[:, 0].long()], scale, plain), "tree")


@pytest.mark.parametrize("cap", [257.0, 1000.0, 1e4])
@pytest.mark.parametrize("d,dtype", [(128, F16), (256, F16), (256, BF16)])
@pytest.mark.parametrize("slopes", [False, True])
@pytest.mark.parametrize("size", [1.0, 0.3])
def test_prefill(cap, d, dtype, slopes, size, dev):
    say(f"prefill, cap {cap} D={d} {dtype} slopes={slopes} {size}")
    n, lens = 60, [62, 70, 64]
    k, v, table, lens_t = _two_keys(d, dtype, lens, 5)
    q = torch.randn(3 * n, 6, d, generator=torch.Generator().manual_seed(6)).to(dtype)
    cu = torch.tensor([0, n, 2 * n, 3 * n], dtype=torch.int32)
    last = torch.ones(3 * n, dtype=torch.int32)
    scale = d ** -0.5 * (1.0 if size == 1.0 else size * cap)
    sl = slopes_of(6) if slopes else None
    exact, _ = ref.prefill(q, k, v, table, cu, lens_t, 16, scale, True, cap, sl, 0, None, last)
    _, plain = ref.prefill(q, k, v, table, cu, lens_t, 16, scale, True, 0.0, sl, 0, None, last)
    out = gqa_prefill_shaped_fn(*(x.to(dev) for x in (q, k, v, table, cu, lens_t)), n, scale=scale, softcap=cap,
                                slopes=None if sl is None else sl.to(dev), last_key=last.to(dev))
    within(out, exact, _limit(q[None], k[table[:, 0].long()], scale, plain), "prefill")
