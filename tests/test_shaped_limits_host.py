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
