"""The calls that make the paged cache smaller, as measurable cases: latent attention (one shared vector
a token in place of every KV head's key and value) and eviction by accumulated attention weight.

Kinds of case (the `kind` entry):
  append   latent_rope_append: the input side of a latent layer (norm, rotation, cache rows)
  decode   latent_decode_paged_fn: the absorbed form on the pages, one or a few new tokens a sequence
  prefill  latent_prefill_fn: the expanded form on packed chunks (first chunks, or over cached tokens)
  mass     cache_attention_mass: softmax weights of a sequence's last queries, summed for each cached token
  evict    evict_kvcache: the heaviest tokens of each (sequence, KV head) move to the blocks of a new table

Sizes are those of the repository's workloads and tests (24, 32, 12, 16 query heads, 4 or 8 KV heads of
256 or 128, a rotated part of 64, pages of 8, 16 and 32 tokens, one short sequence up to 64 long ones)
with latent vectors of 512 or 256.
"""
import math
import random

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
ROTARY = 64  # rotated dimensions beside a latent vector
EPS = 1e-6


def _case(name, kind, **kw):
    case = {"kind": kind, "dtype": "bf16", "page": 16, "lens": 1, **kw}
    return {"name": name, **case} if name else case


def listed():
    return [
        # A decode step's input side, padded to a captured batch: a few rows, launch bound.
        _case("append_33", "append", tokens=33, pad=3, heads=24, latent=512),
        # The input side of a prefill layer: a long chunk.
        _case("append_8191", "append", tokens=8191, pad=0, heads=24, latent=512),
        # One short interactive session: launch and latency bound.
        _case("decode_1x700", "decode", batch=1, lo=700, hi=700, new=1, heads=24, latent=512),
        # An ordinary serving batch of mixed lengths.
        _case("decode_16_mixed", "decode", batch=16, lo=512, hi=8192, new=1, heads=24, latent=512,
              lens=2),
        # Draft tokens verified three at a time, another model's sizes, small pages.
        _case("decode_24_draft3", "decode", batch=24, lo=1, hi=6000, new=3, heads=32, latent=256,
              page=8, dtype="fp16", lens=3),
        # Long contexts, a full batch: the cache's bytes are everything.
        _case("decode_64x16k", "decode", batch=64, lo=16384, hi=16384, new=1, heads=32, latent=512),
        # The first chunk of a prompt.
        _case("prefill_first_2048", "prefill", seqs=1, q_lo=2048, q_hi=2048, c_lo=0, c_hi=0, heads=24,
              dim=128),
        # Chunks of several prompts, some with cached context expanded before the call.
        _case("prefill_12_ragged", "prefill", seqs=12, q_lo=17, q_hi=700, c_lo=0, c_hi=4000, heads=32,
              dim=64, dtype="fp16", lens=5),
        # A decode step's weights added to the running sums.
        _case("mass_16_step", "mass", batch=16, lo=512, hi=8192, new=1, hq=24, hkv=4, d=256, fresh=False,
              lens=2),
        # The last 32 queries of long prompts decide what stays.
        _case("mass_4_window32", "mass", batch=4, lo=2000, hi=16000, new=32, hq=32, hkv=8, d=128,
              fresh=True, dtype="fp16", lens=6),
        # One latent-attention sequence cut to a small budget.
        _case("evict_1_latent", "evict", batch=1, lo=6001, hi=6001, budget=1024, hkv=1, d=576, sinks=4,
              recent=32),
        # A batch of long sequences, one of them possibly within the budget.
        _case("evict_8x32k", "evict", batch=8, lo=3000, hi=32768, budget=4096, hkv=4, d=256, sinks=4,
              recent=128, lens=7),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    common = {"dtype": rng.choice(["bf16", "bf16", "fp16"]), "page": rng.choice([16, 16, 16, 8, 32]),
              "lens": rng.randrange(1 << 20)}
    kind = rng.choice(["append", "decode", "decode", "decode", "prefill", "prefill", "mass", "mass",
                       "evict", "evict"])
    heads, latent = rng.choice([24, 24, 32, 16, 12, 6]), rng.choice([512, 512, 256])
    while True:
        if kind == "append":
            tokens = _log_int(rng, 1, 16384)
            case = _case(None, kind, tokens=tokens, pad=rng.choice([0, 0, tokens // 8]), heads=heads,
                         latent=latent, **common)
        elif kind == "decode":
            hi = _log_int(rng, 64, 32768)
            case = _case(None, kind, batch=_log_int(rng, 1, 128), lo=rng.choice([1, max(1, hi // 16), hi]),
                         hi=hi, new=rng.choice([1, 1, 1, 2, 4, 7]), heads=heads, latent=latent, **common)
        elif kind == "prefill":
            q_hi = _log_int(rng, 16, 4000)
            c_hi = rng.choice([0, 0, _log_int(rng, 64, 8000)])
            case = _case(None, kind, seqs=_log_int(rng, 1, 32), q_lo=rng.choice([q_hi, max(1, q_hi // 20)]),
                         q_hi=q_hi, c_lo=rng.choice([0, c_hi]), c_hi=c_hi, heads=heads,
                         dim=rng.choice([128, 128, 64]), **common)
        else:
            hq, hkv, d = rng.choice([(24, 4, 256), (24, 4, 256), (12, 2, 256), (32, 8, 128),
                                     (heads, 1, latent + ROTARY)])
            hi = _log_int(rng, 64, 32768)
            sizes = {"batch": _log_int(rng, 1, 64), "lo": rng.choice([1, max(1, hi // 16), hi]), "hi": hi,
                     "hkv": hkv, "d": d}
            if kind == "mass":
                case = _case(None, kind, hq=hq, new=rng.choice([1, 1, 1, 8, 32, 33]),
                             fresh=rng.random() < 0.5, **sizes, **common)
            else:
                budget = _log_int(rng, 16, 8192)
                case = _case(None, kind, budget=budget, sinks=rng.choice([0, 4]),
                             recent=rng.choice([0, min(32, budget - 4)]), **sizes, **common)
        w = work(case)
        if max(w["bytes"], w["flops"] / 50) <= 1.2e9 and _held(case) <= 8e9:
            return case


def _lens(case):
    """(query tokens, context tokens) of every sequence; a function of the case alone."""
    rng = random.Random(case["lens"])
    kind = case["kind"]
    if kind == "append":
        return [case["tokens"]], [case["tokens"]]
    if kind == "prefill":
        q = [rng.randint(case["q_lo"], case["q_hi"]) for _ in range(case["seqs"])]
        return q, [n + rng.randint(case["c_lo"], case["c_hi"]) for n in q]
    ctx = [rng.randint(case["lo"], case["hi"]) for _ in range(case["batch"])]
    return [case.get("new", 1)] * len(ctx), ctx


def _held(case):
    """Bytes that the plain form holds at once, about: the scores of a padded prefill, the padded rows."""
    q, ctx = _lens(case)
    if case["kind"] == "prefill":
        return 12 * len(q) * case["heads"] * max(q) * max(ctx)
    if case["kind"] == "mass":
        return len(ctx) * max(ctx) * (4 * case["hkv"] * case["d"] + 12 * case["hq"] * case["new"])
    if case["kind"] == "decode":
        return len(ctx) * max(ctx) * (4 * (case["latent"] + ROTARY) + 12 * case["heads"] * case["new"])
    return 0


def _pages(case):
    return [-(-c // case["page"]) for c in _lens(case)[1]]


def _kept(case):
    return [min(n, case["budget"]) for n in _lens(case)[1]]


def _visible(q_len, kv_len):
    """(query, key) pairs of the last q_len of kv_len tokens, each seeing itself and those before it."""
    return sum(max(0, kv_len - q_len + 1 + i) for i in range(q_len))


def work(case):
    q_lens, ctx = _lens(case)
    kind, pages = case["kind"], sum(_pages(case))
    if kind == "append":
        n, row = case["tokens"], case["latent"] + ROTARY
        return {"bytes": n * (4 * row + 4 * case["heads"] * ROTARY + 4 * ROTARY + 4),
                "flops": n * (4 * case["latent"] + 3 * (case["heads"] + 1) * ROTARY)}
    if kind == "prefill":
        h, dim = case["heads"], case["dim"]
        nbytes = 2 * sum(q_lens) * h * (2 * dim + ROTARY) + 2 * sum(ctx) * (h * 2 * dim + ROTARY)
        return {"bytes": nbytes + 8 * len(ctx),
                "flops": 2 * h * (2 * dim + ROTARY) * sum(map(_visible, q_lens, ctx))}
    pairs = sum(map(_visible, q_lens, ctx))
    if kind == "decode":
        h, row = case["heads"], case["latent"] + ROTARY
        return {"bytes": 2 * row * sum(ctx) + 2 * sum(q_lens) * h * (row + case["latent"]) + 4 * pages + 4 * len(ctx),
                "flops": 2 * h * (row + case["latent"]) * pairs}
    hkv, d = case["hkv"], case["d"]
    if kind == "mass":
        sums = 4 * hkv * sum(ctx) * (1 if case["fresh"] else 2)
        return {"bytes": 2 * hkv * d * sum(ctx) + sums + 2 * sum(q_lens) * case["hq"] * d + 4 * pages + 4 * len(ctx),
                "flops": (2 * d + 4) * case["hq"] * pairs}
    kept, rows = sum(_kept(case)), 1 if case["d"] % 128 else 2  # a latent cache has one row a token
    return {"bytes": 4 * hkv * sum(ctx) + 2 * rows * 2 * hkv * d * kept + 8 * hkv * kept + 4 * pages,
            "flops": 0}


def _randn(shape, gen, dt):
    return torch.empty(shape, dtype=dt, device="cuda").normal_(generator=gen)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _offsets(lens):
    at = [0]
    for n in lens:
        at.append(at[-1] + n)
    return _ints(at)


def _tables(counts, perm, first=0):
    """Block tables of `counts` blocks each, -1 behind, from the blocks of `perm`."""
    rows = []
    width, at = max(counts), first
    for n in counts:
        rows.append(torch.cat([perm[at:at + n], torch.full((width - n,), -1, dtype=torch.int32, device="cuda")]))
        at += n
    return torch.stack(rows).contiguous(), at


def _angles(pos, dt):
    freq = 1e6 ** (-torch.arange(0, ROTARY, 2, device="cuda", dtype=torch.float64) / ROTARY)
    angle = pos.double()[:, None] * torch.cat([freq, freq])[None]
    return angle.cos().to(dt), angle.sin().to(dt)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    dt, page, kind = DTYPES[case["dtype"]], case["page"], case["kind"]
    q_lens, ctx = _lens(case)
    st = {"case": case, "max_len": max(ctx)}
    if kind == "prefill":
        # The chunks' queries, and keys and values expanded from the latent rows (one product in the
        # caller's program); the rotated keys are those rows' last columns.
        h, dim = case["heads"], case["dim"]
        st["q"] = _randn((sum(q_lens), h, dim + ROTARY), gen, dt)
        st["kv"] = _randn((sum(ctx), h, 2 * dim), gen, dt)
        st["key_rope"] = _randn((sum(ctx), 512 + ROTARY), gen, dt)[:, 512:]
        st["cu_q"], st["cu_k"] = _offsets(q_lens), _offsets(ctx)
        st["max_q"] = max(q_lens)
        return st
    counts = _pages(case)
    new_counts = [-(-n // page) for n in _kept(case)] if kind == "evict" else [0]
    pool = math.ceil(1.25 * sum(counts)) + sum(new_counts)
    perm = torch.randperm(pool, generator=gen, device="cuda", dtype=torch.int32)
    st["table"], at = _tables(counts, perm)
    st["seqlen"] = _ints(ctx)
    # A cache is a pool of blocks; the one behind its last stands for slots that are not written.
    hkv, d = (case["hkv"], case["d"]) if "hkv" in case else (1, case["latent"] + ROTARY)
    st["k_pool"] = _randn((pool + 1, page, hkv, d), gen, dt)
    st["k_cache"] = st["k_pool"][:-1]
    if kind == "append":
        n, h, latent = case["tokens"], case["heads"], case["latent"]
        st["latent"] = 2 * _randn((n, latent), gen, dt)
        st["key_rope"], st["q_rope"] = _randn((n, ROTARY), gen, dt), _randn((n, h, ROTARY), gen, dt)
        st["weight"] = 0.1 * _randn((latent,), gen, dt)
        pos = torch.arange(n, device="cuda")
        st["cos"], st["sin"] = _angles(pos, dt)
        st["slots"] = (st["table"][0, pos // page].long() * page + pos % page).to(torch.int32)
        st["slots"][n - case["pad"]:] = -1
    elif kind == "decode":
        st["q"] = _randn((len(ctx), case["new"], case["heads"], d), gen, dt)
        st["scale"] = (128 + ROTARY) ** -0.5
    elif kind == "mass":
        st["q"] = _randn((len(ctx), case["new"], case["hq"], d), gen, dt)
        st["scale"] = d ** -0.5
        if not case["fresh"]:
            st["mass"] = torch.rand((len(ctx), hkv, st["table"].shape[1] * page), generator=gen, device="cuda")
    else:
        if d % 128 == 0:
            st["v_pool"] = _randn((pool + 1, page, hkv, d), gen, dt)
            st["v_cache"] = st["v_pool"][:-1]
        st["new_table"], _ = _tables(new_counts, perm, at)
        # Summed softmax weights: a few tokens hold most, many are alike, some are exactly equal.
        mass = torch.rand((len(ctx), hkv, st["table"].shape[1] * page), generator=gen, device="cuda")
        st["mass"] = (mass.pow(8) * 64).mul(4096).round().div(4096)
    return st


def _rotated(x, cos, sin):
    """Rotation of the last axis' halves by each token's angles."""
    half = x.shape[-1] // 2
    c, s, a, b = cos[..., :half], sin[..., :half], x[..., :half], x[..., half:]
    return torch.cat([a * c - b * s, b * c + a * s], -1)


def _token_rows(table, page, n):
    """Cache rows of each sequence's tokens 0 .. n - 1 (row 0 where the table has no block)."""
    pos = torch.arange(n, device="cuda")
    return (table[:, pos // page].long() * page + pos % page).clamp_min(0)


def _softmax(s):
    """Softmax weights over the last axis; rows with nothing left (-inf everywhere) are zero."""
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    return p / torch.where(total > 0, total, torch.ones_like(total))


def _plain_append(st):
    n, dt = st["latent"].shape[0], st["latent"].dtype
    x, cos, sin = st["latent"].float(), st["cos"].float(), st["sin"].float()
    x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * (1 + st["weight"].float())
    rows = torch.cat([x, _rotated(st["key_rope"].float(), cos, sin)], -1).to(dt)
    st["k_pool"].view(-1, rows.shape[1])[st["slots"].long()] = rows  # slot -1: the row behind the cache
    q = _rotated(st["q_rope"].float(), cos[:, None], sin[:, None]).to(dt)
    return {"q": q, "cache": st["k_cache"]}


def _plain_decode(st):
    case, q = st["case"], st["q"]
    b, new, h, row = q.shape
    n = st["max_len"]
    rows = st["k_cache"].reshape(-1, row)[_token_rows(st["table"], case["page"], n)].float()
    s = torch.matmul(q.reshape(b, new * h, row).float(), rows.transpose(1, 2)).view(b, new, h, n) * st["scale"]
    last = st["seqlen"][:, None] - new + torch.arange(new, device="cuda")
    seen = torch.arange(n, device="cuda") <= last[..., None]
    p = _softmax(s.masked_fill(~seen[:, :, None], -math.inf)).view(b, new * h, n)
    out = torch.matmul(p, rows[..., :case["latent"]])
    return {"out": out.view(b, new, h, case["latent"]).to(q.dtype)}


def _plain_prefill(st):
    case = st["case"]
    dim, q, cu_q, cu_k = case["dim"], st["q"], st["cu_q"].long(), st["cu_k"].long()
    iq, ik = torch.arange(st["max_q"], device="cuda"), torch.arange(st["max_len"], device="cuda")
    lq, lk = (cu_q[1:] - cu_q[:-1])[:, None], (cu_k[1:] - cu_k[:-1])[:, None]
    at_q = torch.where(iq < lq, cu_q[:-1, None] + iq, 0)
    at_k = torch.where(ik < lk, cu_k[:-1, None] + ik, 0)
    qs, kv = q[at_q].float().transpose(1, 2), st["kv"][at_k].float().transpose(1, 2)
    kr = st["key_rope"][at_k].float()[:, None]
    s = torch.matmul(qs[..., :dim], kv[..., :dim].transpose(2, 3))
    s = (s + torch.matmul(qs[..., dim:], kr.transpose(2, 3))) * (dim + ROTARY) ** -0.5
    seen = ik <= (lk - lq + iq)[..., None]
    out = torch.matmul(_softmax(s.masked_fill(~seen[:, None], -math.inf)), kv[..., dim:])
    token = torch.arange(q.shape[0], device="cuda")
    seq = torch.searchsorted(cu_q, token, right=True) - 1
    return {"out": out.transpose(1, 2)[seq, token - cu_q[seq]].to(q.dtype)}


def _plain_mass(st):
    case, q = st["case"], st["q"]
    b, new, hq, d = q.shape
    n, hkv = st["max_len"], case["hkv"]
    k = st["k_cache"].reshape(-1, hkv, d)[_token_rows(st["table"], case["page"], n)].float()
    qs = q.float().view(b, new, hkv, hq // hkv, d).transpose(1, 2).reshape(b, hkv, -1, d)
    s = torch.matmul(qs, k.permute(0, 2, 3, 1)).view(b, hkv, new, hq // hkv, n) * st["scale"]
    last = st["seqlen"][:, None] - new + torch.arange(new, device="cuda")
    seen = torch.arange(n, device="cuda") <= last[..., None]
    weight = _softmax(s.masked_fill(~seen[:, None, :, None], -math.inf)).sum((2, 3))
    mass = st.get("mass")
    if mass is None:
        mass = torch.zeros((b, hkv, st["table"].shape[1] * case["page"]), device="cuda")
    mass[..., :n] += weight
    return {"mass": mass}


def _plain_evict(st):
    case, mass, lens = st["case"], st["mass"], st["seqlen"].long()[:, None, None]
    page, budget = case["page"], case["budget"]
    b, hkv, cap = mass.shape
    at = torch.arange(cap, device="cuda")
    held = (at < case["sinks"]) | (at >= lens - case["recent"])
    key = torch.where(at < lens, torch.where(held, math.inf, mass), -math.inf)
    order = torch.sort(key, dim=-1, descending=True, stable=True).indices
    count = lens.clamp_max(budget)
    place = torch.arange(budget, device="cuda")
    kept = torch.nn.functional.pad(order, (0, max(0, budget - cap)))[..., :budget]
    kept = torch.where(place < count, kept, cap).sort(-1).values
    there = kept < cap
    kept = torch.where(there, kept, -1)
    seq, head = torch.arange(b, device="cuda")[:, None, None], torch.arange(hkv, device="cuda")[:, None]
    source = st["table"].long()[seq, kept.clamp_min(0) // page] * page + kept.clamp_min(0) % page
    width = st["new_table"].shape[1]
    into = st["new_table"].long()[seq, (place // page).clamp_max(width - 1)] * page + place % page
    into = torch.where(there, into, -1)  # the row behind the cache
    out = {"kept": kept.to(torch.int32), "seqlen": count.view(-1).to(torch.int32),
           "mass": torch.zeros_like(mass)}
    out["mass"][..., :budget] = torch.where(there, mass.gather(-1, kept.clamp_min(0)), 0.0)[..., :cap]
    for name in ("k", "v"):
        if name + "_pool" in st:
            rows = st[name + "_pool"].view(-1, hkv, case["d"])
            rows[into, head] = rows[source, head]
            out[name + "_cache"] = st[name + "_cache"]
    return out


def _own_append(st):
    from tileinfer_amd.kernels import latent_rope_append

    cache = st["k_cache"].view(-1, st["k_cache"].shape[-1])
    q = latent_rope_append(st["q_rope"], st["latent"], st["key_rope"], st["weight"], st["cos"], st["sin"],
                           cache, st["slots"], EPS)
    return {"q": q, "cache": st["k_cache"]}


def _own_decode(st):
    from tileinfer_amd.kernels import latent_decode_paged_fn

    return {"out": latent_decode_paged_fn(st["q"], st["k_cache"], st["table"], st["seqlen"],
                                          st["case"]["page"], scale=st["scale"])}


def _own_prefill(st):
    from tileinfer_amd.kernels import latent_prefill_fn

    return {"out": latent_prefill_fn(st["q"], st["kv"], st["key_rope"], st["cu_q"], st["cu_k"], st["max_q"])}


def _own_mass(st):
    from tileinfer_amd.kernels import cache_attention_mass

    return {"mass": cache_attention_mass(st["q"], st["k_cache"], st["table"], st["seqlen"],
                                         st["case"]["page"], scale=st["scale"], mass=st.get("mass"))}


def _own_evict(st):
    from tileinfer_amd.kernels import evict_kvcache

    case = st["case"]
    seqlen, kept, mass = evict_kvcache(
        st["k_cache"], st.get("v_cache"), st["mass"], st["table"], st["seqlen"], st["new_table"],
        case["budget"], case["page"], sinks=case["sinks"], recent=case["recent"])
    out = {"kept": kept, "seqlen": seqlen, "mass": mass}
    return {**out, **{n: st[n] for n in ("k_cache", "v_cache") if n in st}}


def run(st):
    kind = st["case"]["kind"]
    if own:
        return {"append": _own_append, "decode": _own_decode, "prefill": _own_prefill, "mass": _own_mass,
                "evict": _own_evict}[kind](st)
    return {"append": _plain_append, "decode": _plain_decode, "prefill": _plain_prefill,
            "mass": _plain_mass, "evict": _plain_evict}[kind](st)


def _history(st, b, length):
    """Cache rows of one sequence's tokens, in order."""
    blocks = st["table"][b].tolist()
    page = st["case"]["page"]
    rows = [blocks[t // page] * page + t % page for t in range(length)]
    return torch.tensor(rows, device="cuda", dtype=torch.int64)


def _weights64(q, k, scale, first):
    """Softmax weights, in 64 bits, of queries whose first sits at position `first` over keys from 0."""
    s = (q.double() @ k.double().t().contiguous()) * scale
    hidden = torch.ones_like(s, dtype=torch.bool).tril(first).logical_not()
    p = torch.softmax(s.masked_fill(hidden, -math.inf), -1)
    return p.nan_to_num(0.0)  # rows that see nothing


def exact(case, seed):
    st = prepare(case, seed)
    kind, dim = case["kind"], case.get("dim")
    q_lens, ctx = _lens(case)
    if kind == "append":
        x = st["latent"].double()
        x = x / torch.sqrt((x * x).sum(-1, keepdim=True) / x.shape[1] + EPS) * (1 + st["weight"].double())
        turn = torch.complex(st["cos"].double(), st["sin"].double())[:, :ROTARY // 2]
        out = []
        for t, w in ((st["key_rope"].double(), turn), (st["q_rope"].double(), turn[:, None])):
            z = torch.complex(t[..., :ROTARY // 2].contiguous(), t[..., ROTARY // 2:].contiguous()) * w
            out.append(torch.cat([z.real, z.imag], -1))
        cache = st["k_cache"].double()
        real = case["tokens"] - case["pad"]
        cache.view(-1, x.shape[1] + ROTARY)[st["slots"][:real].long()] = torch.cat([x, out[0]], -1)[:real]
        return {"q": out[1], "cache": cache}
    if kind == "evict":
        return _exact_evict(st)
    if kind == "prefill":
        out = torch.empty(st["q"].shape[:2] + (dim,), dtype=torch.float64, device="cuda")
        a = c = 0
        for n, m in zip(q_lens, ctx):
            for h in range(case["heads"]):
                k = torch.cat([st["kv"][c:c + m, h, :dim], st["key_rope"][c:c + m]], -1)
                p = _weights64(st["q"][a:a + n, h], k, (dim + ROTARY) ** -0.5, m - n)
                out[a:a + n, h] = p @ st["kv"][c:c + m, h, dim:].double()
            a, c = a + n, c + m
        return {"out": out}
    new = case["new"]
    if kind == "decode":
        out = torch.empty(st["q"].shape[:3] + (case["latent"],), dtype=torch.float64, device="cuda")
        for b, m in enumerate(ctx):
            k = st["k_cache"].reshape(-1, st["q"].shape[-1])[_history(st, b, m)]
            for h in range(case["heads"]):
                out[b, :, h] = _weights64(st["q"][b, :, h], k, st["scale"], m - new) @ k[:, :case["latent"]].double()
        return {"out": out}
    group = case["hq"] // case["hkv"]
    mass = torch.zeros((len(ctx), case["hkv"], st["table"].shape[1] * case["page"]), dtype=torch.float64,
                       device="cuda")
    if not case["fresh"]:
        mass += st["mass"]
    for b, m in enumerate(ctx):
        k = st["k_cache"].reshape(-1, case["hkv"], case["d"])[_history(st, b, m)]
        for h in range(case["hq"]):
            mass[b, h // group, :m] += _weights64(st["q"][b, :, h], k[:, h // group], st["scale"], m - new).sum(0)
    return {"mass": mass}


def _exact_evict(st):
    case, page = st["case"], st["case"]["page"]
    b, hkv, cap = st["mass"].shape
    budget, ctx = case["budget"], _lens(case)[1]
    kept = np.full((b, hkv, budget), -1, dtype=np.int32)
    mass, values = np.zeros((b, hkv, cap)), st["mass"].cpu().numpy()
    tables, new_tables = st["table"].cpu().numpy(), st["new_table"].cpu().numpy()
    moves = []
    for i, n in enumerate(ctx):
        at = np.arange(n)
        always = (at < case["sinks"]) | (at >= n - case["recent"])
        for h in range(hkv):
            best = np.lexsort((at, -values[i, h, :n], ~always))  # the last key counts first
            keep = np.sort(best[:min(n, budget)])
            kept[i, h, :len(keep)] = keep
            mass[i, h, :len(keep)] = values[i, h, keep]
            j = np.arange(len(keep))
            moves.append(np.stack([np.full(len(keep), h), tables[i, keep // page] * page + keep % page,
                                   new_tables[i, j // page] * page + j % page]))
    head, source, into = torch.from_numpy(np.concatenate(moves, 1)).cuda()
    out = {"kept": torch.from_numpy(kept).cuda(), "seqlen": _ints([min(n, budget) for n in ctx]),
           "mass": torch.from_numpy(mass).cuda()}
    for name in ("k_cache", "v_cache"):
        if name in st:
            rows = st[name].reshape(-1, hkv, case["d"]).double()
            rows[into, head] = rows[source, head]
            out[name] = rows.view(st[name].shape)
    return out
