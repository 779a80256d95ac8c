"""The native form of the latent and eviction entry points against their Python form: over operands plain, strided,
off their alignment, transposed, wrong in size or type, the same bits or the same refusal."""
import pytest
import torch

from helpers import say
from test_native_calls import _FORMS, _Watched, both
from tileinfer_amd import _lib
from tileinfer_amd.kernels import (cache_attention_mass, evict_kvcache, latent_decode_paged_fn,
                                   latent_rope_append)

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def _randn(dev, *shape, dtype=BF16):
    return torch.randn(*shape, device=dev, generator=torch.Generator(dev).manual_seed(sum(shape))).to(dtype)


def _as16(*tensors):
    """Tensors for a bitwise comparison as 16-bit payloads."""
    return [t.contiguous().view(torch.int16) if t.dtype != BF16 else t for t in tensors]


def _form(form, which, name, t):
    return _FORMS[form](t) if which == name else t


@pytest.mark.parametrize("form", list(_FORMS))
@pytest.mark.parametrize("which", ["q_rope", "latent", "key_rope", "weight", "cos", "slots"])
def test_append(which, form, dev, monkeypatch):
    say(f"native latent append {which} {form}")
    if form == "transposed" and which in ("weight", "slots"):
        pytest.skip("no such form")
    n = 5
    f = lambda name, t: _form(form, which, name, t)  # noqa: E731
    args = [f("q_rope", _randn(dev, n, 3, 64)), f("latent", _randn(dev, n, 512)), f("key_rope", _randn(dev, n, 64)),
            f("weight", _randn(dev, 512)), f("cos", _randn(dev, n, 64)), _randn(dev, n, 64)]
    slots = f("slots", torch.tensor([4, -1, 0, 7, 30], dtype=torch.int32, device=dev))

    def call():
        cache = torch.zeros(9, 576, dtype=BF16, device=dev)
        q = latent_rope_append(*args, cache, slots, 1e-6)
        return [q, cache]

    refused = both(monkeypatch, call, True if form == "plain" else None)
    assert (refused is not None) == (form in ("short", "wide")) or form == "odd"


@pytest.mark.parametrize("form", list(_FORMS))
@pytest.mark.parametrize("which", ["q", "table", "lens", "cache"])
def test_decode_and_mass(which, form, dev, monkeypatch):
    say(f"native latent decode and mass {which} {form}")
    if form == "transposed" and which in ("lens", "cache"):
        pytest.skip("no such form")
    if which == "cache" and form == "short":
        pytest.skip("a cache of fewer blocks is a cache")
    f = lambda name, t: _form(form, which, name, t)  # noqa: E731
    q = f("q", _randn(dev, 3, 6, 320))
    cache = f("cache", _randn(dev, 12, 16, 1, 320))
    table = f("table", torch.randperm(12, device=dev, dtype=torch.int64).to(torch.int32).view(3, 4))
    lens = f("lens", torch.tensor([1, 40, 64], dtype=torch.int32, device=dev))
    bad = form in ("short", "wide")
    for call in (lambda: [latent_decode_paged_fn(q, cache, table, lens, 16, scale=0.1)],
                 lambda: _as16(cache_attention_mass(q, cache, table, lens, 16, scale=0.1)),
                 lambda: _as16(cache_attention_mass(q, cache, table, lens, 16, scale=0.1,
                                                    mass=torch.ones(3, 1, 70, device=dev)))):
        refused = both(monkeypatch, call, True if form == "plain" else None)
        # The cache is never copied: contiguous and aligned, or refused.
        want = bad or which == "cache" and form in ("strided", "odd")
        assert (refused is not None) == want or form == "odd"


@pytest.mark.parametrize("form", list(_FORMS))
@pytest.mark.parametrize("which", ["k", "v", "mass", "table", "lens", "new_table"])
def test_evict(which, form, dev, monkeypatch):
    say(f"native evict {which} {form}")
    if form == "transposed" and which in ("lens", "k", "v"):
        pytest.skip("no such form")
    if which == "k" and form == "short":
        pytest.skip("a cache of fewer blocks is a cache")
    f = lambda name, t: _form(form, which, name, t)  # noqa: E731
    mass = f("mass", torch.rand(2, 2, 48, device=dev))
    ids = torch.arange(8, device=dev, dtype=torch.int32)
    table, new_table = f("table", ids[:6].view(2, 3)), f("new_table", ids[6:].view(2, 1))
    lens = f("lens", torch.tensor([48, 20], dtype=torch.int32, device=dev))

    def call():
        k, v = f("k", _randn(dev, 8, 16, 2, 128)), f("v", _randn(dev, 8, 16, 2, 128))
        return _as16(*evict_kvcache(k, v, mass, table, lens, new_table, 16, 16, sinks=1, recent=2), k.contiguous(), v.contiguous())

    refused = both(monkeypatch, call, True if form == "plain" else None)
    if form in ("short", "wide") or which in ("k", "v") and form == "strided":
        assert refused is not None
    elif form in ("plain", "parameter"):
        assert refused is None


def test_other_forms_go_to_python(dev, monkeypatch):
    """Given outputs, default scales of integers, no queries: what the native form declines gives the same."""
    say("native latent declines")
    q, cache = _randn(dev, 2, 4, 320), _randn(dev, 4, 16, 1, 320)
    table = torch.arange(4, dtype=torch.int32, device=dev).view(2, 2)
    lens = torch.tensor([5, 32], dtype=torch.int32, device=dev)
    taken = []
    with monkeypatch.context() as m:
        w = _Watched(taken)
        m.setattr(_lib, "calls", lambda: w)
        a = latent_decode_paged_fn(q, cache, table, lens, 16, scale=1.0)
        b = latent_decode_paged_fn(q, cache, table, lens, 16, scale=1)
        c = latent_decode_paged_fn(q, cache, table, lens, 16, scale=1.0, out=torch.empty_like(a))
        none = latent_rope_append(None, _randn(dev, 2, 256), _randn(dev, 2, 64), _randn(dev, 256), _randn(dev, 2, 64),
                                  _randn(dev, 2, 64), cache.view(64, 320), lens)
    assert taken == [True, False, True] and none is None
    assert torch.equal(a, b) and torch.equal(a, c)
    for bad in (0.0, -1.0, float("inf"), float("nan")):
        with pytest.raises(ValueError, match="scale"):
            latent_decode_paged_fn(q, cache, table, lens, 16, scale=bad)
        with pytest.raises(ValueError, match="scale"):
            cache_attention_mass(q, cache, table, lens, 16, scale=bad)
