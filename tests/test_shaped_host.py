"""Drafted trees, several position axes and shaped scores without a GPU: helpers on the host, the 64-bit forms against
simpler spellings, and refusals before the first launch."""
import ctypes

import pytest
import torch

from oracle import ref_shaped as ref
from test_latent_host import _addr, _refused
from tileinfer_amd import _lib
from tileinfer_amd.kernels import rope_axes, tree_masks
from tileinfer_amd.kernels.draft_tree import _softcap, _window


def test_axes_of_sections():
    assert rope_axes((2, 1, 3)).tolist() == [0, 0, 1, 2, 2, 2]
    assert rope_axes((4, 2, 2), interleaved=True).tolist() == [0, 1, 2, 0, 1, 2, 0, 0]
    assert rope_axes((3,)).tolist() == [0, 0, 0]
    for bad in ((), (1,) * 5, (-1, 3)):
        with pytest.raises(ValueError):
            rope_axes(bad)
    with pytest.raises(ValueError):
        rope_axes((1, 3, 1), interleaved=True)


def test_masks_of_parents():
    assert tree_masks([-1, 0, 0, 1]).tolist() == [1, 3, 5, 11]
    assert tree_masks([[-1, -1], [-1, 0]]).tolist() == [[1, 2], [1, 3]]
    chain = tree_masks(list(range(-1, 63)))
    assert chain[63].item() == -1 and chain[62].item() == 2 ** 63 - 1
    for bad in ([0], [-1, 1], [-2], list(range(-1, 64)), [[[-1]]], []):
        with pytest.raises(ValueError):
            tree_masks(bad)


def test_host_numbers_of_a_shape():
    assert _softcap(None) == 0 and _softcap(30) == 30.0 and _window(None) == 0 and _window(2 ** 40) == 2 ** 31 - 1
    for bad in (0, -1.0, 1e5, float("nan"), float("inf")):
        with pytest.raises(ValueError):
            _softcap(bad)
    for bad in (0, -5):
        with pytest.raises(ValueError):
            _window(bad)


def test_forms_against_closed_ones():
    """One visible key gives its value; equal scores the mean; a capped score saturates; slope and window by hand."""
    g = torch.Generator().manual_seed(1)
    k, v = (torch.randn(3, 4, 1, 128, generator=g) for _ in range(2))
    table, lens = torch.tensor([[2, 0, 1]], dtype=torch.int32), torch.tensor([10])
    rows = torch.tensor([8, 9, 10, 11, 0, 1, 2, 3, 4, 5])
    vs = v.view(-1, 128)[rows].double()
    q = torch.zeros(1, 2, 1, 128)
    out, _ = ref.tree(q, k, v, table, lens, [[1, 2]], 4, 0.1)
    assert torch.allclose(out[0, 0, 0], vs[:9].mean(0)) and torch.allclose(out[0, 1, 0], vs[[*range(8), 9]].mean(0))
    out, _ = ref.tree(q, k, v, table, lens, [[0, 2]], 4, 0.1, window=1)
    assert (out[0, 0, 0] == 0).all() and torch.allclose(out[0, 1, 0], vs[9])  # a draft without its bit sees nothing nearer than 1
    out, _ = ref.tree(q, k, v, table, lens, [[1, 3]], 4, 0.1, slopes=torch.tensor([0.5]))
    w = torch.exp(-0.5 * torch.arange(9, -1, -1).double())
    assert torch.allclose(out[0, 1, 0], (w[:, None] * vs).sum(0) / w.sum())
    first, last = torch.tensor([3, 9]), torch.tensor([3, 5])
    out, _ = ref.prefill(q[0], k, v, table, [0, 2], lens, 4, 0.1, first=first, last=last)
    assert torch.allclose(out[0, 0], vs[3]) and (out[1] == 0).all()
    big = 1e4 * torch.ones(1, 1, 1, 128)
    capped, _ = ref.tree(big, big.expand(1, 4, 1, 128), v[:1], torch.tensor([[0]]), torch.tensor([4]), None, 4, 1.0, cap=3.0)
    assert torch.allclose(capped[0, 0, 0], v.view(-1, 128)[:4].double().mean(0))


def test_keep_by_hand():
    cache = torch.arange(12.0).view(1, 6, 2, 1, 1).repeat(2, 1, 1, 1, 1)
    table = torch.tensor([[4, 1, 0]], dtype=torch.int32)  # tokens 0 .. 5 are rows 8, 9, 2, 3, 0, 1
    got, lens = ref.keep(cache, table, torch.tensor([6]), torch.tensor([[1, 3, -1]]), 2, 4)  # drafts: tokens 2 .. 5
    assert lens.tolist() == [4] and got.view(2, 12)[1].tolist() == [0, 1, 3, 1, 4, 5, 6, 7, 8, 9, 10, 11]


def test_rope_axes_refusals():
    p = _addr()
    good = [p, 512, 128, p, 256, 128, p, 256, 128, p, 8, 32, p, p, p, p, 1.0, p, 512, 128, p, p, 256, 20, p, 8, 3, 4, 2, 128,
            64, 1e-6, 0, None]
    _refused("ti_rope_axes_append", good,
             [(0, None), (3, None), (6, None), (9, None), (12, None), (14, None), (15, None), (17, None), (20, None),
              (21, None), (24, None), (0, p + 8), (1, 100), (22, 248), (22, 257), (23, -1), (25, -1), (25, 1 << 28), (26, 0),
              (26, 5), (27, 0), (28, 0)], _lib.TI_EINVAL)
    _refused("ti_rope_axes_append", good, [(29, 64), (30, 24), (30, 144), (30, -16), (11, 16), (32, 4)], _lib.TI_EUNSUPPORTED)
    good[25] = 0
    assert _lib.load().ti_rope_axes_append(*good) == _lib.TI_OK


@pytest.mark.parametrize("drafts", [4, 64])  # either kernel
def test_tree_refusals(drafts):
    p, lib, n = _addr(), _lib.load(), ctypes.c_int64()
    assert lib.ti_gqa_tree_workspace_bytes(2, drafts, 8, 2, 128, ctypes.byref(n)) == 0 and n.value > 0
    good = [p, 1024 * drafts, 1024, 128, p, p, p, 4, p, p, drafts, p, p, p, n.value, 2, drafts, 8, 2, 128, 16, 8, 4, 0.1, 30.0,
            0, 0, None]
    _refused("ti_gqa_tree_paged", good,
             [(0, None), (4, None), (5, None), (6, None), (8, None), (12, None), (13, None), (0, p + 8), (4, p + 8), (3, 100),
              (14, n.value - 16), (15, -1), (17, 7), (18, 0), (20, 0), (21, -1), (21, 1 << 28), (22, -1), (22, 1 << 28),
              (23, 0.0), (23, 1e31), (23, float("nan")), (24, -1.0), (24, 1e-4), (24, 1e5), (24, float("nan")), (25, -1),
              (15, 1 << 24)], _lib.TI_EINVAL)
    _refused("ti_gqa_tree_paged", good, [(19, 64), (16, 0), (16, 65), (26, 3)], _lib.TI_EUNSUPPORTED)
    good[15] = 0
    assert lib.ti_gqa_tree_paged(*good) == _lib.TI_OK
    assert lib.ti_gqa_tree_workspace_bytes(2, drafts, 8, 2, 128, None) == _lib.TI_EINVAL
    assert lib.ti_gqa_tree_workspace_bytes(2, 65, 8, 2, 128, ctypes.byref(n)) == _lib.TI_EUNSUPPORTED


def test_keep_refusals():
    p = _addr()
    good = [p, p, 4, p, p, 8, p, 2, 8, 8, 4, 512, 16, 8, 4, None]
    _refused("ti_keep_drafts", good,
             [(0, None), (1, None), (3, None), (4, None), (6, None), (0, p + 8), (7, -1), (9, -1), (10, -1), (11, 0), (11, 12),
              (11, 1 << 32), (12, 0), (13, -1), (13, 1 << 28), (14, -1), (14, 1 << 28), (7, 1 << 26)], _lib.TI_EINVAL)
    _refused("ti_keep_drafts", good, [(8, 0), (8, 65)], _lib.TI_EUNSUPPORTED)
    good[7] = 0
    assert _lib.load().ti_keep_drafts(*good) == _lib.TI_OK


def test_shaped_prefill_refusals():
    p, lib, n = _addr(), _lib.load(), ctypes.c_int64()
    assert lib.ti_gqa_prefill_shaped_workspace_bytes(1, 10, 10, 8, 2, 128, 4000, ctypes.byref(n)) == 0 and n.value > 0
    good = [p, 1024, 128, p, p, p, 250, p, p, p, p, p, p, 1024, 128, p, n.value, 1, 10, 10, 8, 2, 128, 16, 300, 250, 4000, 1,
            0.1, 0.0, 0, 0, None]
    _refused("ti_gqa_prefill_shaped", good,
             [(0, None), (3, None), (4, None), (5, None), (7, None), (8, None), (12, None), (0, p + 8), (2, 100), (12, p + 2),
              (16, n.value - 16), (15, p + 8), (17, -1), (17, 1 << 17), (18, -1), (19, -1), (20, 7), (21, 0), (23, 0), (24, -1),
              (24, 1 << 28), (25, -1), (25, 1 << 28), (26, -1), (28, 0.0), (28, 1e31), (29, 1e-4), (29, 1e5), (30, -1)],
             _lib.TI_EINVAL)
    _refused("ti_gqa_prefill_shaped", good, [(22, 64), (31, 9)], _lib.TI_EUNSUPPORTED)
    for at in (17, 18, 19):
        args = list(good)
        args[at] = 0
        assert lib.ti_gqa_prefill_shaped(*args) == _lib.TI_OK
    assert lib.ti_gqa_prefill_shaped_workspace_bytes(1, 10, 10, 8, 2, 128, 4000, None) == _lib.TI_EINVAL
    # More workgroups than a launch counts are refused before the first one.
    big = ctypes.c_int64()
    args = list(good)
    args[17], args[18], args[19], args[15], args[16] = 65535, 1 << 22, 1 << 22, None, 0
    assert lib.ti_gqa_prefill_shaped(*args) == _lib.TI_EINVAL
    assert lib.ti_gqa_prefill_shaped_workspace_bytes(65535, 1 << 22, 1 << 22, 8, 2, 128, 4000, ctypes.byref(big)) == 0


def test_native_form_declines_what_is_not_its_form():
    c, t = _lib.calls(), torch.zeros(1, 1, 256)
    for f, n in ((c.rope_axes_append, 14), (c.tree, 12), (c.keep, 7), (c.shaped, 17)):
        for x in (t, None, 3):
            assert f(*[x] * n) is None
        with pytest.raises(TypeError):
            f(t)
