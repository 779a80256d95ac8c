"""Drafted trees and shaped scores on the paged cache, as measurable cases: the input side with several
position axes, the attention of a tree of drafts, the rows of an accepted path moved into place, and prefill
with capped, biased and interval-masked scores.

Kinds of case (the `kind` entry):
  rope     rope_axes_append: norms, rotation by one or three position axes, cache rows, one launch
  tree     gqa_tree_paged_fn: the last tokens of every sequence are a tree of drafts (one: a decode step)
  keep     keep_drafts: accepted drafts' rows move behind the context, in all layers at once
  prefill  gqa_prefill_shaped_fn: packed chunks over their cached context

Sizes are those of the repository's workloads and tests (24/4 heads of 256, 32/8 of 128, pages of 8,
16 and 32 tokens, one short sequence up to batches of long ones, chunks of 2,048 over 8,192 keys), with
trees of up to 64 drafts.
"""
import math
import random

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
EPS = 1e-6


def _case(name, kind, **kw):
    case = {"kind": kind, "dtype": "bf16", "page": 16, "lens": 1, "hq": 24, "hkv": 4, "d": 256, **kw}
    return {"name": name, **case} if name else case


def _shape(cap=0.0, slopes=False, window=0):
    return {"cap": cap, "slopes": slopes, "window": window}


def listed():
    return [
        # The input side of a small verification step, padded to a captured batch: launch bound.
        _case("rope_48", "rope", tokens=48, pad=6, axes=3, norm=True),
        # A long chunk of image and text tokens.
        _case("rope_8191", "rope", tokens=8191, pad=0, axes=3, norm=True),
        # A model without QK-norm, one axis.
        _case("rope_2080_plain", "rope", tokens=2080, pad=32, axes=1, norm=False, hq=32, hkv=8, d=128, dtype="fp16"),
        # One interactive session, a small tree: latency bound.
        _case("tree_1x700", "tree", batch=1, lo=700, hi=700, new=8, shared=True, **_shape()),
        # An ordinary serving batch, each sequence with a tree of its own, capped scores.
        _case("tree_16_mixed", "tree", batch=16, lo=512, hi=8192, new=16, shared=False, lens=2, **_shape(cap=50.0)),
        # Wide trees, slopes, small pages: as much arithmetic as memory.
        _case("tree_24_wide", "tree", batch=24, lo=64, hi=6000, new=64, shared=False, page=8, lens=3, hq=32, hkv=8, d=128,
              dtype="fp16", **_shape(slopes=True)),
        # A plain decode step of a model with capped scores, long contexts: the cache's bytes are everything.
        _case("step_32x16k", "tree", batch=32, lo=16384, hi=16384, new=1, shared=True, hq=32, hkv=8, d=128,
              **_shape(cap=30.0)),
        # After a verification step: four sequences, the sixteen attention layers' keys and values.
        _case("keep_4", "keep", batch=4, lo=200, hi=900, new=8, planes=32, lens=4),
        # A full batch with wide trees.
        _case("keep_64", "keep", batch=64, lo=64, hi=400, new=32, planes=32, lens=5),
        # The first chunk of a prompt, capped scores.
        _case("first_2048_cap", "prefill", seqs=1, q_lo=2048, q_hi=2048, c_lo=0, c_hi=0, docs=0, spans=0,
              **_shape(cap=50.0)),
        # A continuation over a long context, capped, every query within its window.
        _case("chunk_2048_window", "prefill", seqs=1, q_lo=2048, q_hi=2048, c_lo=8192, c_hi=8192, docs=0, spans=0,
              **_shape(cap=50.0, window=4096)),
        # Packed documents and image spans, some with cached context, slopes.
        _case("prefill_12_docs", "prefill", seqs=12, q_lo=17, q_hi=1200, c_lo=0, c_hi=2000, docs=400, spans=150,
              hq=32, hkv=8, d=128, dtype="fp16", lens=6, **_shape(slopes=True)),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


HEADS = [(24, 4, 256), (24, 4, 256), (8, 2, 256), (6, 1, 256), (32, 8, 128), (32, 8, 128), (16, 16, 128), (20, 2, 128)]


def draw(rng):
    while True:
        hq, hkv, d = rng.choice(HEADS)
        common = {"dtype": rng.choice(["bf16", "bf16", "fp16"]), "page": rng.choice([16, 16, 16, 8, 32]),
                  "lens": rng.randrange(1 << 20), "hq": hq, "hkv": hkv, "d": d}
        kind = rng.choice(["rope", "tree", "tree", "tree", "keep", "prefill", "prefill", "prefill"])
        hi = _log_int(rng, 64, 32768)
        lengths = {"lo": rng.choice([1, max(1, hi // 16), hi]), "hi": hi}
        shape = _shape(cap=rng.choice([0.0, 30.0, 50.0]), slopes=rng.random() < 0.4,
                       window=rng.choice([0, 0, _log_int(rng, 16, 8192)]))
        if kind == "rope":
            tokens = _log_int(rng, 1, 16384)
            case = _case(None, kind, tokens=tokens, pad=rng.choice([0, 0, tokens // 8]), axes=rng.choice([1, 3, 3]),
                         norm=rng.random() < 0.6, **common)
        elif kind == "tree":
            case = _case(None, kind, batch=_log_int(rng, 1, 128), new=rng.choice([1, 1, 4, 8, 17, 32, 64]),
                         shared=rng.random() < 0.4, **lengths, **shape, **common)
        elif kind == "keep":
            case = _case(None, kind, batch=_log_int(rng, 1, 128), new=rng.choice([2, 8, 16, 33, 64]),
                         planes=rng.choice([2, 8, 32, 32]), **lengths, **common)
        else:
            q_hi = _log_int(rng, 16, 4000)
            c_hi = rng.choice([0, 0, _log_int(rng, 64, 12000)])
            case = _case(None, kind, seqs=_log_int(rng, 1, 32), q_lo=rng.choice([q_hi, max(1, q_hi // 20)]), q_hi=q_hi,
                         c_lo=rng.choice([0, c_hi]), c_hi=c_hi, docs=rng.choice([0, 0, _log_int(rng, 20, 2000)]),
                         spans=rng.choice([0, 0, _log_int(rng, 10, 600)]), **shape, **common)
        w = work(case)
        if w["bytes"] + w["flops"] / 200 <= 2.1e9 and _held(case) <= 8e9:
            return case


def _lens(case):
    """(query tokens, context tokens) of every sequence; a function of the case alone."""
    rng = random.Random(case["lens"])
    kind = case["kind"]
    if kind == "rope":
        return [case["tokens"]], [case["tokens"]]
    if kind == "prefill":
        q = [rng.randint(case["q_lo"], case["q_hi"]) for _ in range(case["seqs"])]
        return q, [n + rng.randint(case["c_lo"], case["c_hi"]) for n in q]
    ctx = [rng.randint(case["lo"], case["hi"]) + case["new"] - 1 for _ in range(case["batch"])]
    return [case["new"]] * len(ctx), ctx


def _cuts(rng, n, mean):
    """Lengths that add up to n, about `mean` each."""
    out = []
    while n > 0:
        out.append(min(n, rng.randint(max(1, mean // 2), max(1, 3 * mean // 2))))
        n -= out[-1]
    return out


def _intervals(case):
    """Per sequence (first key, last key) of every query of a prefill: within its document, to the end of its
    image span (each document's spans alternate with text) or to itself."""
    rng = random.Random(case["lens"] + 1)
    out = []
    for n, m in zip(*_lens(case)):
        first, last = np.zeros(m, dtype=np.int64), np.arange(m)
        at = 0
        for size in _cuts(rng, m, case["docs"] or m):
            if case["docs"]:
                first[at:at + size] = at
            if case["spans"]:
                begin, image = at, False
                for part in _cuts(rng, size, case["spans"]):
                    if image:
                        last[begin:begin + part] = begin + part - 1
                    begin, image = begin + part, not image
            at += size
        out.append((first[m - n:], last[m - n:]))
    return out


def _seen(case):
    """(pairs, keys): (query, key) pairs that attend, and cached tokens that some query sees."""
    pairs = keys = 0
    window = case["window"]
    if case["kind"] == "prefill":
        for (n, m), (first, last) in zip(zip(*_lens(case)), _intervals(case)):
            if window:
                first = np.maximum(first, np.arange(m - n, m) - window + 1)
            pairs += int(np.maximum(last - first + 1, 0).sum())
            keys += int(last.max() - first.min() + 1)
        return pairs, keys
    new = case["new"]
    for b, m in enumerate(_lens(case)[1]):
        bits, depth = _tree(case, b)
        context = m - new
        near = np.minimum(context, np.maximum(window - depth, 0)) if window else np.full(new, context)
        drafts = bits if not window else bits & (depth[:, None] - depth < window)
        pairs += int(near.sum() + drafts.sum())
        keys += int(near.max() + drafts.any(0).sum())
    return pairs, keys


def _parents(case, b):
    """A tree of drafts behind its root (the last token that is certain): parents[i] < i."""
    rng = random.Random(1000 * case["lens"] + (0 if case.get("shared") else b))
    return [-1] + [max(0, i - rng.choice([1, 1, 1, 2, 3, 5])) for i in range(1, case["new"])]


def _tree(case, b):
    """bits[i, j]: draft i sees draft j (itself and those before it on its path); depth of every draft."""
    parents, n = _parents(case, b), case["new"]
    bits = np.zeros((n, n), dtype=bool)
    for i, p in enumerate(parents):
        if p >= 0:
            bits[i] = bits[p]
        bits[i, i] = True
    return bits, bits.sum(1) - 1


def _paths(case):
    """Accepted drafts of every sequence: the path to a random draft."""
    rng = random.Random(case["lens"] + 2)
    out = []
    for b in range(case["batch"]):
        parents, at, path = _parents(case, b), rng.randrange(case["new"]), []
        while at >= 0:
            path.append(at)
            at = parents[at]
        out.append(path[::-1])
    return out


def _held(case):
    """Bytes that the plain form holds at once, about: padded scores and rows."""
    q, ctx = _lens(case)
    if case["kind"] in ("tree", "prefill"):
        return len(ctx) * max(ctx) * (8 * case["hkv"] * case["d"] + 12 * case["hq"] * max(q))
    if case["kind"] == "keep":
        return 8 * sum(_pages(case)) * case["page"] * case["planes"] * case["hkv"] * case["d"]
    return 0


def _pages(case):
    return [-(-c // case["page"]) for c in _lens(case)[1]]


def work(case):
    q_lens, ctx = _lens(case)
    kind, hq, hkv, d = case["kind"], case["hq"], case["hkv"], case["d"]
    if kind == "rope":
        n = case["tokens"]
        return {"bytes": n * (4 * (hq + 2 * hkv) * d + 4 * case["axes"] + 4),
                "flops": n * (hq + hkv) * ((4 * d if case["norm"] else 0) + 3 * _rotary(case))}
    if kind == "keep":
        moved = sum(sum(1 for j, a in enumerate(p) if a != j) for p in _paths(case))
        return {"bytes": 4 * moved * case["planes"] * hkv * d + 4 * sum(map(len, _paths(case))) + 8 * len(ctx), "flops": 0}
    pairs, keys = _seen(case)
    return {"bytes": 4 * keys * hkv * d + 4 * sum(q_lens) * hq * d + 4 * sum(_pages(case)) + 4 * len(ctx),
            "flops": 4 * d * hq * pairs}


def _rotary(case):
    return 64 if case["d"] == 256 else case["d"]


def _randn(shape, gen, dt):
    return torch.empty(shape, dtype=dt, device="cuda").normal_(generator=gen)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _offsets(lens):
    return _ints(np.concatenate([[0], np.cumsum(lens)]).tolist())


def _tables(counts, perm):
    """Block tables of `counts` blocks each, -1 behind, from the blocks of `perm`."""
    rows, width, at = [], max(counts), 0
    for n in counts:
        rows.append(torch.cat([perm[at:at + n], torch.full((width - n,), -1, dtype=torch.int32, device="cuda")]))
        at += n
    return torch.stack(rows).contiguous()


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    dt, page, kind = DTYPES[case["dtype"]], case["page"], case["kind"]
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    q_lens, ctx = _lens(case)
    st = {"case": case, "max_len": max(ctx)}
    counts = _pages(case)
    pool = math.ceil(1.25 * sum(counts))
    perm = torch.randperm(pool, generator=gen, device="cuda", dtype=torch.int32)
    st["table"], st["seqlen"] = _tables(counts, perm), _ints(ctx)
    if kind == "keep":
        st["cache"] = _randn((2, case["planes"] // 2, pool, page, hkv, d), gen, dt)
        paths = _paths(case)
        st["accepted"] = _ints([p + [-1] * (case["new"] - len(p)) for p in paths])
        return st
    # A cache is a pool of blocks; the one behind its last stands for slots that are not written.
    for name in ("k", "v"):
        st[name + "_pool"] = _randn((pool + 1, page, hkv, d), gen, dt)
        st[name + "_cache"] = st[name + "_pool"][:-1]
    if kind == "rope":
        n, half = case["tokens"], _rotary(case) // 2
        qkv = _randn((n, hq + 2 * hkv, d), gen, dt)  # one projection's output
        st["q"], st["k"], st["v"] = qkv[:, :hq], qkv[:, hq:hq + hkv], qkv[:, hq + hkv:]
        if case["norm"]:
            st["q_weight"], st["k_weight"] = 0.1 * _randn((d,), gen, dt), 0.1 * _randn((d,), gen, dt)
        st["inv_freq"] = (1e6 ** (-torch.arange(half, device="cuda", dtype=torch.float64) / half)).float()
        pos = torch.arange(n, device="cuda", dtype=torch.int32) + int(case["lens"]) % 200000
        st["positions"] = pos[None]
        if case["axes"] == 3:  # runs of 256 text tokens and images of 16 x 16 in turn
            image, at = (pos // 256) % 2 == 1, pos % 256
            st["positions"] = torch.stack([torch.where(image, pos - at, pos), torch.where(image, pos - at + at // 16, pos),
                                           torch.where(image, pos - at + at % 16, pos)])
            third = half // 3
            st["axes"] = _ints([0] * (half - 2 * third) + [1] * third + [2] * third)
        at = torch.arange(n, device="cuda")
        st["slots"] = (st["table"][0, at // page].long() * page + at % page).to(torch.int32)
        st["slots"][n - case["pad"]:] = -1
        return st
    st["scale"] = d ** -0.5
    st["cap"], st["window"] = case["cap"] or None, case["window"] or None
    st["slopes"] = None
    if case["slopes"]:
        st["slopes"] = 2.0 ** (-8.0 * torch.arange(1, hq + 1, device="cuda", dtype=torch.float32) / hq)
    if kind == "tree":
        # Queries and keys as an attention's norms leave them: some keys stand out.
        st["q"] = 2 * _randn((len(ctx), case["new"], hq, d), gen, dt)
        masks = [[sum(1 << j for j in range(case["new"]) if row[j]) for row in _tree(case, b)[0]]
                 for b in range(1 if case["shared"] else len(ctx))]
        masks = [[m - (1 << 64) if m >> 63 else m for m in row] for row in masks]
        st["mask"] = torch.tensor(masks[0] if case["shared"] else masks, dtype=torch.int64, device="cuda")
        return st
    st["q"] = 2 * _randn((sum(q_lens), hq, d), gen, dt)
    st["cu_q"], st["max_q"] = _offsets(q_lens), max(q_lens)
    spans = _intervals(case)
    st["first"] = _ints(np.concatenate([f for f, _ in spans]).tolist()) if case["docs"] else None
    st["last"] = _ints(np.concatenate([e for _, e in spans]).tolist()) if case["spans"] else None
    return st


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


def _plain_rope(st):
    case, dt = st["case"], st["q"].dtype
    half = _rotary(case) // 2
    axes = st["axes"].long() if "axes" in st else torch.zeros(half, dtype=torch.int64, device="cuda")
    angle = st["positions"].double()[axes].t() * st["inv_freq"].double()
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]

    def rows(x, weight):
        x = x.float()
        if weight is not None:
            x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * (1 + weight.float())
        a, b = x[..., :half], x[..., half:2 * half]
        return torch.cat([a * cos - b * sin, b * cos + a * sin, x[..., 2 * half:]], -1).to(dt)

    slots = st["slots"].long()  # slot -1: the row behind the cache
    row = (case["hkv"], case["d"])
    st["k_pool"].view(-1, *row)[slots] = rows(st["k"], st.get("k_weight"))
    st["v_pool"].view(-1, *row)[slots] = st["v"]
    return {"q": rows(st["q"], st.get("q_weight")), "k_cache": st["k_cache"], "v_cache": st["v_cache"]}


def _grouped(x, hkv):
    """[B, N, Hq, D] -> [B, Hkv, N * group, D] in 32 bits."""
    b, n, hq, d = x.shape
    return x.float().view(b, n, hkv, hq // hkv, d).transpose(1, 2).reshape(b, hkv, -1, d)


def _plain_attention(st, q, seen, dist):
    """q [B, N, Hq, D] over each sequence's cached tokens; seen, dist [B, N, tokens]."""
    case = st["case"]
    b, new, hq, d = q.shape
    hkv, n = case["hkv"], seen.shape[-1]
    rows = _token_rows(st["table"], case["page"], n)
    k = st["k_cache"].reshape(-1, hkv, d)[rows].float().permute(0, 2, 3, 1).contiguous()
    s = torch.matmul(_grouped(q, hkv), k).view(b, hkv, new, hq // hkv, n) * st["scale"]
    if st["cap"]:
        s = st["cap"] * torch.tanh(s / st["cap"])
    if st["slopes"] is not None:
        s = s - st["slopes"].view(1, hkv, 1, -1, 1) * dist.abs().float()[:, None, :, None]
    s.masked_fill_(~seen[:, None, :, None], -math.inf)
    p = _softmax(s).view(b, hkv, -1, n)
    v = st["v_cache"].reshape(-1, hkv, d)[rows].float().transpose(1, 2).contiguous()
    out = torch.matmul(p, v).view(b, hkv, new, hq // hkv, d)
    return out.transpose(1, 2).reshape(b, new, hq, d).to(q.dtype)


def _plain_tree(st):
    q, n = st["q"], st["max_len"]
    b, new = q.shape[:2]
    at = torch.arange(new, device="cuda")
    bits = ((st["mask"].view(-1, new, 1) >> at) & 1).bool().expand(b, new, new)
    depth = bits.sum(-1) - bits.diagonal(dim1=1, dim2=2).long()
    first = st["seqlen"].long()[:, None] - new  # position of the tree's root
    draft = torch.arange(n, device="cuda") - first  # which draft a cached token is; negative: context
    index = draft.clamp(0, new - 1)
    seen = (draft < 0)[:, None] | ((draft < new)[:, None] & bits.gather(2, index[:, None].expand(b, new, n)))
    position = torch.where(draft < 0, torch.arange(n, device="cuda"), first + depth.gather(1, index))
    dist = (first + depth)[..., None] - position[:, None]
    if st["window"]:
        seen = seen & (dist < st["window"])
    return {"out": _plain_attention(st, q, seen, dist)}


def _plain_keep(st):
    case = st["case"]
    page, new = case["page"], case["new"]
    accepted, first = st["accepted"].long(), st["seqlen"].long()[:, None] - new
    there = accepted >= 0
    j = torch.arange(new, device="cuda")
    table = st["table"].long()

    def rows(position):
        return table.gather(1, position // page) * page + position % page

    source, into = rows(first + accepted.clamp_min(0))[there], rows(first + j.expand_as(accepted))[there]
    flat = st["cache"].view(case["planes"], -1, case["hkv"], case["d"])
    flat[:, into] = flat[:, source]
    return {"seqlen": (first[:, 0] + there.sum(1)).to(torch.int32), "cache": st["cache"]}


def _plain_prefill(st):
    case, q, cu = st["case"], st["q"], st["cu_q"].long()
    i = torch.arange(st["max_q"], device="cuda")
    lens, total = cu[1:] - cu[:-1], st["seqlen"].long()
    at = torch.where(i < lens[:, None], cu[:-1, None] + i, 0)
    position = (total - lens)[:, None] + i
    first = torch.zeros_like(position) if st["first"] is None else st["first"].long()[at]
    last = position if st["last"] is None else st["last"].long()[at]
    if st["window"]:
        first = torch.maximum(first, position - st["window"] + 1)
    key = torch.arange(st["max_len"], device="cuda")
    seen = (key >= first[..., None]) & (key <= last[..., None]) & (key < total[:, None, None])
    out = _plain_attention(st, q[at], seen, position[..., None] - key)
    token = torch.arange(q.shape[0], device="cuda")
    seq = torch.searchsorted(cu, token, right=True) - 1
    return {"out": out[seq, token - cu[seq]]}


def _own_rope(st):
    from tileinfer_amd.kernels import rope_axes_append

    row = st["case"]["hkv"] * st["case"]["d"]
    q = rope_axes_append(st["q"], st["k"], st["v"], st["positions"], st["inv_freq"], st.get("axes"),
                         st["k_cache"].view(-1, row), st["v_cache"].view(-1, row), st["slots"],
                         q_weight=st.get("q_weight"), k_weight=st.get("k_weight"), eps=EPS)
    return {"q": q, "k_cache": st["k_cache"], "v_cache": st["v_cache"]}


def _own_tree(st):
    from tileinfer_amd.kernels import gqa_tree_paged_fn

    return {"out": gqa_tree_paged_fn(st["q"], st["k_cache"], st["v_cache"], st["table"], st["seqlen"], st["mask"],
                                     st["case"]["page"], scale=st["scale"], softcap=st["cap"], slopes=st["slopes"],
                                     window=st["window"])}


def _own_keep(st):
    from tileinfer_amd.kernels import keep_drafts

    seqlen = keep_drafts(st["cache"], st["table"], st["seqlen"], st["accepted"], st["case"]["page"],
                         num_drafts=st["case"]["new"])
    return {"seqlen": seqlen, "cache": st["cache"]}


def _own_prefill(st):
    from tileinfer_amd.kernels import gqa_prefill_shaped_fn

    return {"out": gqa_prefill_shaped_fn(
        st["q"], st["k_cache"], st["v_cache"], st["table"], st["cu_q"], st["seqlen"], st["max_q"], st["case"]["page"],
        scale=st["scale"], softcap=st["cap"], slopes=st["slopes"], window=st["window"], first_key=st["first"],
        last_key=st["last"], max_seqlen_k=st["max_len"])}


def run(st):
    kind = st["case"]["kind"]
    if own:
        return {"rope": _own_rope, "tree": _own_tree, "keep": _own_keep, "prefill": _own_prefill}[kind](st)
    return {"rope": _plain_rope, "tree": _plain_tree, "keep": _plain_keep, "prefill": _plain_prefill}[kind](st)


def _history(st, b, length):
    """Cache rows of one sequence's tokens, in order."""
    blocks = st["table"][b].tolist()
    page = st["case"]["page"]
    return torch.tensor([blocks[t // page] * page + t % page for t in range(length)], device="cuda", dtype=torch.int64)


def _exact_rows(st, b, length, q, seen, dist):
    """Attention, in 64 bits, of q [N, Hq, D] over sequence b's first `length` tokens, one head after the other."""
    case = st["case"]
    rows = _history(st, b, length)
    out = torch.empty(q.shape, dtype=torch.float64, device="cuda")
    for h in range(case["hq"]):
        g = h // (case["hq"] // case["hkv"])
        k = st["k_cache"].reshape(-1, case["hkv"], case["d"])[rows, g].double()
        v = st["v_cache"].reshape(-1, case["hkv"], case["d"])[rows, g].double()
        s = (q[:, h].double() @ k.t().contiguous()) * st["scale"]
        if case["cap"]:
            s = torch.tanh(s / case["cap"]) * case["cap"]
        if case["slopes"]:
            s = s - float(st["slopes"][h]) * dist.abs()
        s = s.masked_fill(~seen, -math.inf)
        out[:, h] = torch.softmax(s, -1).nan_to_num(0.0) @ v  # rows that see nothing
    return out


def exact(case, seed):
    kind, window = case["kind"], case.get("window")
    q_lens, ctx = _lens(case)
    if kind == "keep" and _held(case) > 24e9:
        return None
    st = prepare(case, seed)
    if kind == "rope":
        return _exact_rope(st)
    if kind == "keep":
        return _exact_keep(st)
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device="cuda")
    if kind == "tree":
        new = case["new"]
        for b, m in enumerate(ctx):
            bits, depth = _tree(case, b)
            seen = np.concatenate([np.ones((new, m - new), dtype=bool), bits], 1)
            dist = m - new + depth[:, None] - np.concatenate([np.arange(m - new), m - new + depth])
            if window:
                seen &= dist < window
            out[b] = _exact_rows(st, b, m, st["q"][b], torch.from_numpy(seen).cuda(), torch.from_numpy(dist).cuda())
        return {"out": out}
    at = 0
    for b, (n, m, (first, last)) in enumerate(zip(q_lens, ctx, _intervals(case))):
        key, position = torch.arange(m, device="cuda"), torch.arange(m - n, m, device="cuda")[:, None]
        seen = (key >= torch.from_numpy(first).cuda()[:, None]) & (key <= torch.from_numpy(last).cuda()[:, None])
        if window:
            seen &= position - key < window
        out[at:at + n] = _exact_rows(st, b, m, st["q"][at:at + n], seen, position - key)
        at += n
    return {"out": out}


def _exact_rope(st):
    case = st["case"]
    half, real = _rotary(case) // 2, case["tokens"] - case["pad"]
    axes = st["axes"].tolist() if "axes" in st else [0] * half
    angle = torch.stack([st["positions"][a].double() for a in axes], 1) * st["inv_freq"].double()
    turn = torch.polar(torch.ones_like(angle), angle)[:, None]
    out = []
    for name in ("q", "k"):
        x = st[name].double()
        if case["norm"]:
            x = x / torch.sqrt((x * x).sum(-1, keepdim=True) / x.shape[-1] + EPS) * (1 + st[name + "_weight"].double())
        z = torch.complex(x[..., :half].contiguous(), x[..., half:2 * half].contiguous()) * turn
        out.append(torch.cat([z.real, z.imag, x[..., 2 * half:]], -1))
    caches = []
    for cache, rows in ((st["k_cache"], out[1]), (st["v_cache"], st["v"].double())):
        cache = cache.double()
        cache.view(-1, case["hkv"], case["d"])[st["slots"][:real].long()] = rows[:real]
        caches.append(cache)
    return {"q": out[0], "k_cache": caches[0], "v_cache": caches[1]}


def _exact_keep(st):
    case, page, new = st["case"], st["case"]["page"], st["case"]["new"]
    tables, moves, lens = st["table"].tolist(), [], []
    for b, (m, path) in enumerate(zip(_lens(case)[1], _paths(case))):
        first = m - new
        lens.append(first + len(path))
        for j, a in enumerate(path):
            moves.append([tables[b][(first + i) // page] * page + (first + i) % page for i in (a, j)])
    source, into = torch.tensor(moves, device="cuda").t()
    cache = st["cache"].double()
    flat = cache.view(case["planes"], -1, case["hkv"], case["d"])
    flat[:, into] = flat[:, source]
    return {"seqlen": _ints(lens), "cache": cache}
