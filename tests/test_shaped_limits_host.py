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


def test_rope_turns_whole_heads():
    """Heads of 256 may be turned whole, as qknorm_rope_append turns them; no head past its end."""
    p, lib = _addr(), _lib.load()
    good = [p, 512, 256, p, 512, 256, p, 512, 256, p, 8, 32, p, p, p, p, 1.0, p, 512, 256, p, p, 512, 20, p, 0, 3, 2, 2, 256,
            256, 1e-6, 0, None]  # no tokens: checked, not launched
    for head_dim, rotary in ((256, 256), (256, 240), (256, 144), (256, 0), (128, 128)):
        good[29], good[30] = head_dim, rotary
        assert lib.ti_rope_axes_append(*good) == _lib.TI_OK, (head_dim, rotary, lib.ti_last_error())
    _refused("ti_rope_axes_append", good, [(30, 144), (30, 256), (30, 136)], _lib.TI_EUNSUPPORTED)
    good[29] = 256
    _refused("ti_rope_axes_append", good, [(30, 272), (30, 200)], _lib.TI_EUNSUPPORTED)
