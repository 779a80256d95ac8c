"""Drafted trees, position axes and shaped scores without a GPU: operands that must be apart, sizes of workspaces and of
rotations."""
import ctypes

from test_latent_host import _addr, _refused
from tileinfer_amd import _lib


def test_keep_refuses_lengths_in_place():
    """A sequence's workgroups read its old length while one of them stores the new one: the two are apart."""
    p = _addr()
    old = _addr()
    good = [p, p, 4, old, p, 8, old + 8, 2, 8, 8, 4, 512, 16, 8, 4, None]  # two lengths, the new ones right behind
    _refused("ti_keep_drafts", good, [(6, old), (6, old + 4), (6, old - 4)], _lib.TI_EINVAL)
    good[6], good[7] = old, 0
    assert _lib.load().ti_keep_drafts(*good) == _lib.TI_OK


def test_shaped_workspace_is_that_of_the_units_there_are():
    """A padded batch has blocks that do not exist: they get no parts. 512 units of 128 rows of 128 32-bit values (256 of
    256) are what the GPU takes at once, and their statistics."""
    lib, n = _lib.load(), ctypes.c_int64()
    for batch, total, longest, hq, hkv, d in ((32, 631, 600, 8, 1, 128), (32, 1031, 1000, 8, 1, 256), (100, 3000, 2000, 8, 1, 128),
                                              (7, 343, 300, 8, 2, 128), (1, 300, 300, 24, 4, 256), (60, 60, 1, 24, 4, 256)):
        assert lib.ti_gqa_prefill_shaped_workspace_bytes(batch, total, longest, hq, hkv, d, 1 << 17, ctypes.byref(n)) == 0
        assert n.value <= 512 * 128 * (128 + 2) * 4, (batch, total, longest, n.value)
