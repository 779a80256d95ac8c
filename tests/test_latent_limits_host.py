"""Sizes that no launch of the latent and eviction entry points takes are refused before the first one (no GPU needed)."""
import ctypes

import pytest

from test_latent_host import _addr
from tileinfer_amd import _lib
from tileinfer_amd.kernels.latent_attention import _scale


def test_more_work_items_than_a_launch_counts():
    """A launch counts its work items along x in 32 bits, 2^24 workgroups of 256: where a call's second launch has more, its
    first one must not run either, and where its first one has, the second must not add up what nothing wrote."""
    lib, n, p = _lib.load(), ctypes.c_int64(), _addr()
    assert lib.ti_latent_decode_workspace_bytes(1 << 14, 7, 128, 512, ctypes.byref(n)) == _lib.TI_OK
    assert lib.ti_latent_decode_workspace_bytes(1 << 14, 8, 128, 512, ctypes.byref(n)) == _lib.TI_EINVAL
    assert lib.ti_latent_decode_paged(p, 8 * 576, 576, 576, p, p, 4, p, p, p, 1 << 40, 1 << 14, 8, 128, 512, 64, 16, 8, 4,
                                      0.1, 0, None) == _lib.TI_EINVAL
    assert b"2^24" in lib.ti_last_error()
    assert lib.ti_cache_mass_workspace_bytes(1, 1, 8, 1, 128, 16, 1 << 26, ctypes.byref(n)) == _lib.TI_OK
    assert lib.ti_cache_mass_workspace_bytes(1, 1, 8, 8, 128, 16, 1 << 26, ctypes.byref(n)) == _lib.TI_EINVAL
    assert lib.ti_cache_mass_workspace_bytes(1, 17, 1, 1, 576, 16, 1 << 26, ctypes.byref(n)) == _lib.TI_EINVAL
    assert lib.ti_cache_mass(p, 1024, 1024, 128, p, p, 4, p, p, 1 << 33, 1 << 30, p, 1 << 60, 1, 1, 8, 8, 128, 16, 8, 1 << 26,
                             0.1, 0, None) == _lib.TI_EINVAL
    assert lib.ti_latent_rope_append(p, 192, 64, p, 192, 64, p, 512, p, 64, p, 1.0, p, p, 64, p, 576, 8, p, 1 << 25, 24, 512,
                                     64, 1e-6, 0, None) == _lib.TI_EINVAL


def test_a_list_of_tiles_that_offsets_could_make_too_long_is_not_cut():
    """Cut units are counted in 32 bits; offsets that go back could give each of 65,535 sequences all 8 blocks and 1,024
    tiles of 16 heads."""
    lib, n = _lib.load(), ctypes.c_int64(1)
    assert lib.ti_latent_prefill_workspace_bytes(65535, 1024, 65536, 16, 128, ctypes.byref(n)) == _lib.TI_OK
    assert n.value == 0
    assert lib.ti_latent_prefill_workspace_bytes(2 ** 31 - 1, 1, 2 ** 31 - 1, 2, 128, ctypes.byref(n)) == _lib.TI_OK
    assert n.value == 0  # more sequences than a call takes
    assert lib.ti_latent_prefill_workspace_bytes(24, 2048, 400000, 16, 128, ctypes.byref(n)) == _lib.TI_OK
    assert n.value > 0


@pytest.mark.parametrize("scale", [1e31, 1e39, float("inf"), 0.0, 1e-60])
def test_scales_that_32_bits_do_not_hold(scale):
    """A host double beyond 32 bits arrives as infinity (or zero), which would make every output a NaN."""
    lib, n, p = _lib.load(), ctypes.c_int64(), _addr()
    if scale != 1e-60:  # a positive double, which the library refuses
        with pytest.raises(ValueError, match="scale"):
            _scale(scale)
    decode = [p, 24 * 576, 24 * 576, 576, p, p, 4, p, p, p, 1 << 40, 2, 1, 24, 512, 64, 16, 8, 4, scale, 0, None]
    assert lib.ti_latent_decode_paged(*decode) == _lib.TI_EINVAL and b"scale" in lib.ti_last_error()
    prefill = [p, 768, 192, p, 1024, 256, p, 64, p, p, p, 512, 128, p, 1 << 40, 1, 100, 100, 100, 4, 128, 64, 1, scale, 0,
               None]
    assert lib.ti_latent_prefill(*prefill) == _lib.TI_EINVAL and b"scale" in lib.ti_last_error()
    mass = [p, 1024, 1024, 128, p, p, 4, p, p, 128, 64, p, 1 << 40, 2, 1, 8, 2, 128, 16, 8, 4, scale, 0, None]
    assert lib.ti_cache_mass(*mass) == _lib.TI_EINVAL and b"scale" in lib.ti_last_error()
