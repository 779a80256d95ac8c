"""Latent attention and cache eviction without a GPU: their 64-bit forms against other ways to compute the same,
the cache layout, and what the entry points refuse before they touch a device."""
import ctypes

import pytest
import torch

from oracle import ref_latent as ref
from tileinfer_amd import _lib
from tileinfer_amd.engine import kv_layout
from tileinfer_amd.kernels import (cache_attention_mass, evict_kvcache, latent_decode_paged_fn,
                                   latent_prefill_fn, latent_rope_append)

BF16 = torch.bfloat16


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def test_absorbed_and_expanded_forms_agree():
    """The identity behind the two kernels, in 64 bits: q_nope . (c Wk) = (q_nope Wk^T) . c, o = (p c) Wv."""
    g = _gen(1)
    n, new, h, d, latent = 37, 5, 3, 64, 256
    rows = torch.randn(n, latent + 64, generator=g).double()
    wk, wv = (torch.randn(h, latent, d, generator=g).double() for _ in range(2))
    q_nope, q_rot = torch.randn(new, h, d, generator=g).double(), torch.randn(new, h, 64, generator=g).double()
    kv = torch.cat([torch.einsum("tl,hld->thd", rows[:, :latent], w) for w in (wk, wv)], -1)
    cu = lambda m: torch.tensor([0, m])  # noqa: E731
    scale = 1e-2
    q = torch.cat([q_nope, q_rot], -1).to(torch.float64)
    seen = ref.causal(new, n)
    for x in range(h):
        p, _ = ref.softmax_rows(q[:, x], torch.cat([kv[:, x, :d], rows[:, latent:]], -1), scale, seen)
        expanded = p @ kv[:, x, d:]
        qa = torch.cat([q_nope[:, x] @ wk[x].t(), q_rot[:, x]], -1)
        pa, _ = ref.softmax_rows(qa, rows, scale, seen)
        torch.testing.assert_close(pa @ rows[:, :latent] @ wv[x], expanded, rtol=1e-9, atol=1e-9)
    assert cu(3).tolist() == [0, 3]


def test_evict_definition():
    mass = torch.tensor([[[1.0, 5.0, float("nan"), 5.0, 0.0, 2.0, -0.0, 7.0]]])
    kept, lens = ref.evict(mass, [8], 3, 0, 0)
    assert kept.tolist() == [[[1, 3, 7]]] and lens.tolist() == [3]
    kept, _ = ref.evict(mass, [8], 4, 1, 1)
    assert kept.tolist() == [[[0, 1, 3, 7]]]
    kept, _ = ref.evict(mass, [8], 7, 0, 0)  # the NaN goes first
    assert kept.tolist() == [[[0, 1, 3, 4, 5, 6, 7]]]
    kept, lens = ref.evict(mass, [2], 3, 0, 0)
    assert kept.tolist() == [[[0, 1, -1]]] and lens.tolist() == [2]


def test_rows_that_see_nothing_are_zero():
    out, limit = ref.latent_prefill(torch.randn(3, 1, 128).to(BF16), torch.randn(1, 1, 128).to(BF16),
                                    torch.randn(1, 64).to(BF16), [0, 3], [0, 1], 0.1)
    assert (out[:2] == 0).all() and (out[2] != 0).any() and (limit > 0).all()


def test_latent_cache_layout():
    shape = kv_layout.latent_cache_shape(3, 10, 16, 512)
    assert shape == (3, 10, 16, 1, 576)
    assert kv_layout.latent_block_bytes(16, 512, 3) == 16 * 576 * 2 * 3
    cache = kv_layout.allocate_latent_cache(3, 10, 16, 256, device="cpu")
    rows, paged = kv_layout.latent_layer_views(cache, 1)
    assert rows.shape == (160, 320) and paged.shape == (10, 16, 1, 320) and paged.is_contiguous()
    rows[17] = 1
    assert (cache[1, 1, 1] == 1).all() and cache.sum() == 320


def _args():
    """CPU operands of the right shapes: every function refuses them for their device alone."""
    t = lambda *s: torch.zeros(*s, dtype=BF16)  # noqa: E731
    i = lambda *s: torch.zeros(*s, dtype=torch.int32)  # noqa: E731
    return t, i


def test_functions_run_on_the_gpu_only():
    t, i = _args()
    for call in (
        lambda: latent_rope_append(t(2, 3, 64), t(2, 512), t(2, 64), t(512), t(2, 64), t(2, 64), t(9, 576), i(2)),
        lambda: latent_decode_paged_fn(t(2, 3, 576), t(4, 16, 1, 576), i(2, 2), i(2), 16, scale=0.1),
        lambda: latent_prefill_fn(t(2, 3, 192), t(2, 3, 256), t(2, 64), i(2), i(2), 2),
        lambda: cache_attention_mass(t(2, 4, 128), t(4, 16, 2, 128), i(2, 2), i(2), 16),
        lambda: evict_kvcache(t(4, 16, 2, 128), None, torch.zeros(2, 2, 32), i(2, 2), i(2), i(2, 1), 4, 16),
    ):
        with pytest.raises(ValueError, match="GPU"):
            call()


def _addr(n=1 << 16):
    """A 16-byte aligned host address that no refused call reads."""
    buf = ctypes.create_string_buffer(n + 16)
    _addr.kept.append(buf)
    a = ctypes.addressof(buf)
    return a + (-a) % 16


_addr.kept = []


def _refused(name, good, changes, code):
    """Each change of the call's good arguments is refused with `code` and a text that names the function."""
    lib = _lib.load()
    for at, value in changes:
        args = list(good)
        args[at] = value
        assert getattr(lib, name)(*args) == code, (name, at, value)
        assert name.encode() in lib.ti_last_error(), (name, at, value, lib.ti_last_error())


def test_append_refusals():
    p = _addr()
    good = [p, 192, 64, p, 192, 64, p, 512, p, 64, p, 1.0, p, p, 64, p, 576, 8, p, 4, 3, 512, 64, 1e-6, 0, None]
    _refused("ti_latent_rope_append", good,
             [(3, None), (6, None), (8, None), (18, None), (15, None), (6, p + 2), (1, 190), (14, 4), (16, 575),
              (16, 568), (17, -1), (19, -1), (20, -1), (19, 1 << 30)], _lib.TI_EINVAL)
    _refused("ti_latent_rope_append", good, [(21, 384), (22, 32), (24, 2)], _lib.TI_EUNSUPPORTED)
    good[19] = 0
    assert _lib.load().ti_latent_rope_append(*good) == _lib.TI_OK  # no tokens: nothing to do


def test_decode_refusals():
    p, lib = _addr(), _lib.load()
    n = ctypes.c_int64()
    assert lib.ti_latent_decode_workspace_bytes(2, 1, 24, 512, ctypes.byref(n)) == 0 and n.value > 0
    good = [p, 24 * 576, 24 * 576, 576, p, p, 4, p, p, p, n.value, 2, 1, 24, 512, 64, 16, 8, 4, 0.1, 0, None]
    _refused("ti_latent_decode_paged", good,
             [(0, None), (4, None), (5, None), (7, None), (8, None), (9, None), (0, p + 8), (3, 577), (10, n.value - 16),
              (11, -1), (12, 0), (13, 0), (16, 0), (17, -1), (18, -1), (19, 0.0), (19, -1.0), (19, float("nan")),
              (17, 1 << 28), (18, 1 << 28), (12, 1 << 24)], _lib.TI_EINVAL)
    _refused("ti_latent_decode_paged", good, [(14, 128), (15, 32), (20, 7)], _lib.TI_EUNSUPPORTED)
    good[11] = 0
    assert lib.ti_latent_decode_paged(*good) == _lib.TI_OK
    assert lib.ti_latent_decode_workspace_bytes(2, 1, 24, 512, None) == _lib.TI_EINVAL
    assert lib.ti_latent_decode_workspace_bytes(2, 1, 24, 500, ctypes.byref(n)) == _lib.TI_EUNSUPPORTED


def test_prefill_refusals():
    p, lib = _addr(), _lib.load()
    n = ctypes.c_int64()
    assert lib.ti_latent_prefill_workspace_bytes(1, 100, 100, 4, 128, ctypes.byref(n)) == 0 and n.value > 0
    big = ctypes.c_int64(1)
    assert lib.ti_latent_prefill_workspace_bytes(1, 1 << 20, 1 << 20, 64, 128, ctypes.byref(big)) == 0
    assert big.value == 0  # units enough for every CU: one workgroup each
    good = [p, 4 * 192, 192, p, 4 * 256, 256, p, 64, p, p, p, 512, 128, p, n.value, 1, 100, 100, 100, 4, 128, 64, 1,
            0.1, 0, None]
    _refused("ti_latent_prefill", good,
             [(0, None), (3, None), (6, None), (8, None), (9, None), (10, None), (0, p + 2), (5, 250), (7, 60),
              (12, 127), (14, n.value - 16), (13, p + 8), (15, -1), (16, -1), (17, -1), (18, -1), (19, 0), (23, 0.0),
              (4, 1 << 24), (7, -8), (15, 70000)], _lib.TI_EINVAL)
    _refused("ti_latent_prefill", good, [(20, 96), (21, 128), (24, 5)], _lib.TI_EUNSUPPORTED)
    good[16] = 0
    assert lib.ti_latent_prefill(*good) == _lib.TI_OK


def test_mass_refusals():
    p, lib = _addr(), _lib.load()
    n = ctypes.c_int64()
    assert lib.ti_cache_mass_workspace_bytes(2, 1, 8, 2, 128, 16, 4, ctypes.byref(n)) == 0 and n.value > 0
    good = [p, 1024, 1024, 128, p, p, 4, p, p, 128, 64, p, n.value, 2, 1, 8, 2, 128, 16, 8, 4, 0.1, 0, None]
    _refused("ti_cache_mass", good,
             [(0, None), (4, None), (5, None), (7, None), (8, None), (11, None), (0, p + 2), (3, 100), (10, 63),
              (12, n.value - 16), (13, -1), (14, 0), (15, 7), (16, 0), (18, 0), (19, -1), (20, -1), (21, 0.0),
              (13, 70000)], _lib.TI_EINVAL)
    _refused("ti_cache_mass", good, [(17, 64), (22, 3)], _lib.TI_EUNSUPPORTED)
    good[13] = 0
    assert lib.ti_cache_mass(*good) == _lib.TI_OK


def test_evict_refusals():
    p, lib = _addr(), _lib.load()
    good = [p, p, p, 128, 64, 64, p, 4, p, p, 1, p, p, p, 2, 2, 128, 16, 8, 4, 1, 16, 2, 4, 0, None]
    _refused("ti_evict_kvcache", good,
             [(0, None), (2, None), (6, None), (8, None), (9, None), (11, None), (12, None), (13, None), (0, p + 2),
              (1, p + 2), (4, 63), (5, 63), (14, -1), (15, 0), (16, 12), (17, 0), (18, -1), (20, 0), (21, 0), (21, -3),
              (21, 17), (22, -1), (23, 15), (19, 1 << 28)], _lib.TI_EINVAL)
    _refused("ti_evict_kvcache", good, [(24, 9)], _lib.TI_EUNSUPPORTED)
    good[14] = 0
    assert lib.ti_evict_kvcache(*good) == _lib.TI_OK
