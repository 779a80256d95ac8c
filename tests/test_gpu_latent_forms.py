"""Operands of the latent and eviction calls as every second row of a larger tensor, off a 16-byte boundary, or with their
last axes swapped in memory: copied where a copy is documented, which gives the bits of plain ones, or refused."""
import pytest
import torch

from helpers import say
from test_native_calls import _odd, _strided, _transposed
from tileinfer_amd.kernels import (cache_attention_mass, evict_kvcache, latent_decode_paged_fn, latent_prefill_fn,
                                   latent_rope_append)

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16
FORMS = {"strided": _strided, "odd": _odd, "transposed": _transposed}


def _randn(dev, *shape, seed=0):
    return torch.randn(*shape, device=dev, generator=torch.Generator(dev).manual_seed(seed)).to(BF16)


def _ints(dev, *values):
    return torch.tensor(values, dtype=torch.int32, device=dev)


def _append(dev):
    ops = dict(q_rope=_randn(dev, 5, 3, 64), latent=_randn(dev, 5, 512, seed=1), key_rope=_randn(dev, 5, 64, seed=2),
               weight=_randn(dev, 512, seed=3), cos=_randn(dev, 5, 64, seed=4), sin=_randn(dev, 5, 64, seed=5),
               slots=_ints(dev, 4, -1, 0, 7, 30))

    def call(o):
        cache = torch.zeros(9, 576, dtype=BF16, device=dev)
        return latent_rope_append(o["q_rope"], o["latent"], o["key_rope"], o["weight"], o["cos"], o["sin"], cache, o["slots"],
                                  1e-6), cache
    return ops, call


def _paged(dev):
    return dict(q=_randn(dev, 3, 6, 320), cache=_randn(dev, 12, 16, 1, 320, seed=1),
                table=torch.randperm(12, generator=torch.Generator().manual_seed(6)).to(torch.int32).view(3, 4).to(dev),
                lens=_ints(dev, 1, 40, 64))


def _decode(dev):
    return _paged(dev), lambda o: [latent_decode_paged_fn(o["q"], o["cache"], o["table"], o["lens"], 16, scale=0.1)]


def _mass(dev):
    ops = dict(_paged(dev), mass=_randn(dev, 3, 1, 70, seed=7).float())
    return ops, lambda o: [cache_attention_mass(o["q"], o["cache"], o["table"], o["lens"], 16, scale=0.1, mass=m)
                           for m in (None, o["mass"])]


def _prefill(dev):
    ops = dict(q=_randn(dev, 90, 3, 192), kv=_randn(dev, 400, 3, 256, seed=1), key_rope=_randn(dev, 400, 64, seed=2),
               cu_q=_ints(dev, 0, 40, 75, 90), cu_k=_ints(dev, 0, 100, 175, 400))
    return ops, lambda o: [latent_prefill_fn(o["q"], o["kv"], o["key_rope"], o["cu_q"], o["cu_k"], 40)]


def _evict(dev):
    ids = torch.arange(8, device=dev, dtype=torch.int32)
    ops = dict(k=_randn(dev, 8, 16, 2, 128), v=_randn(dev, 8, 16, 2, 128, seed=1), mass=_randn(dev, 2, 2, 48, seed=7).float(),
               table=ids[:6].view(2, 3), new_table=ids[6:].view(2, 1), lens=_ints(dev, 48, 20))

    return ops, lambda o: (*evict_kvcache(o["k"], o["v"], o["mass"], o["table"], o["lens"], o["new_table"], 16, 16, sinks=1,
                                          recent=2), o["k"], o["v"])


REFUSED = {("decode", "cache"), ("mass", "cache"), ("evict", "k"), ("evict", "v")}
CALLS = {"append": _append, "decode": _decode, "mass": _mass, "prefill": _prefill, "evict": _evict}
CASES = [(name, which) for name, which in (
    [("append", w) for w in ("q_rope", "latent", "key_rope", "weight", "cos", "sin", "slots")]
    + [(n, w) for n in ("decode", "mass") for w in ("q", "cache", "table", "lens")] + [("mass", "mass")]
    + [("prefill", w) for w in ("q", "kv", "key_rope", "cu_q", "cu_k")]
    + [("evict", w) for w in ("k", "v", "mass", "table", "new_table", "lens")])]


@pytest.mark.parametrize("form", list(FORMS))
@pytest.mark.parametrize("name,which", CASES)
def test_form(name, which, form, dev):
    say(f"{name} {which} {form}")
    ops, call = CALLS[name](dev)
    if form == "transposed" and (ops[which].dim() == 1 or which == "cache" or (name, which) == ("mass", "mass")):
        pytest.skip("no such form: one axis, or one of size one")
    want = [x.clone() for x in call(ops)]
    ops, call = CALLS[name](dev)  # the call may update its operands
    ops[which] = FORMS[form](ops[which])
    # A cache is updated in place or too large to copy, running sums are rows: contiguous (and aligned), or refused.
    if (name, which) in REFUSED or (which == "mass" and form == "transposed"):
        before = ops[which].clone()
        with pytest.raises(ValueError):
            call(ops)
        assert torch.equal(ops[which], before)
        return
    for a, b in zip(call(ops), want, strict=True):
        assert torch.equal(a, b)
