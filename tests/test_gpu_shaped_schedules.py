"""How the shaped prefill hands out its work: every unit whole, the last partial round cut, all cut, and batches of which few
units exist; each against the 64-bit form, replayed from a graph, and within its workspace."""
import ctypes

import pytest
import torch

from helpers import bits, say
from oracle import ref_shaped as ref
from test_gpu_draft_tree import paged, slopes_of, within
from tileinfer_amd import _lib
from tileinfer_amd.kernels import gqa_prefill_shaped_fn

pytestmark = pytest.mark.gpu
BF16, F16 = torch.bfloat16, torch.float16
GUARD = 4096  # bytes behind a workspace


def _inputs(hq, hkv, d, dtype, q_lens, lens, seed, dev):
    k, v, table, lens_t = paged(lens, 16, hkv, d, dtype, seed)
    q = (2 * torch.randn(sum(q_lens), hq, d, generator=torch.Generator().manual_seed(seed + 1))).to(dtype)
    cu = torch.tensor([0] + list(torch.tensor(q_lens).cumsum(0)), dtype=torch.int32)
    cpu = q, k, v, table, cu, lens_t
    return cpu, [x.to(dev) for x in cpu]


def _bytes(args, max_q, max_k):
    q, k, _, table, _, _ = args
    n = ctypes.c_int64(-1)
    _lib.check(_lib.load().ti_gqa_prefill_shaped_workspace_bytes(
        table.shape[0], q.shape[0], max_q, q.shape[1], k.shape[2], q.shape[2], max_k, ctypes.byref(n)))
    return n.value


def _call(args, max_q, max_k, cap=0.0, slopes=None, workspace=True):
    """The C call with a workspace of just its size (or none); the bytes behind it stay as they were."""
    q, k, v, table, cu, lens = args
    out = torch.empty_like(q)
    size = _bytes(args, max_q, max_k) if workspace else 0
    ws = torch.full((size + GUARD,), 0xA5, dtype=torch.uint8, device=q.device)
    _lib.check(_lib.load().ti_gqa_prefill_shaped(
        q.data_ptr(), q.stride(0), q.stride(1), k.data_ptr(), v.data_ptr(), table.data_ptr(), table.stride(0), cu.data_ptr(),
        lens.data_ptr(), None, None, None if slopes is None else slopes.data_ptr(), out.data_ptr(), out.stride(0), out.stride(1),
        ws.data_ptr() if workspace else None, size, table.shape[0], q.shape[0], max_q, q.shape[1], k.shape[2], q.shape[2], 16,
        k.shape[0] * k.shape[1] // 16, table.shape[1], max_k, 1, q.shape[2] ** -0.5, cap, 0, _lib.dtype_code(q.dtype),
        _lib.stream_handle(q.device)))
    torch.cuda.synchronize()
    assert (ws[size:] == 0xA5).all()
    return out


def _rows(cpu, a, e, cap, slopes):
    """(output, limit) of the queries a .. e - 1 of one causal chunk: a chunk by themselves over the keys up to theirs."""
    q, k, v, table, cu, lens = cpu
    return ref.prefill(q[a:e], k, v, table, [0, e - a], [int(lens[0]) - q.shape[0] + e], 16, q.shape[2] ** -0.5, True, cap, slopes)


ONE = [
    # heads, D, type, queries, keys, cap, slopes: the GPU holds 256 units of head_dim 256, 512 of 128
    (24, 4, 256, BF16, 1500, 3100, 30.0, False),  # 284 units: 256 whole, 28 cut in 9
    (24, 4, 256, F16, 1500, 3100, 0.0, True),
    (32, 8, 128, BF16, 2100, 4300, 30.0, True),   # 528: 512 whole, 16 cut in 16
    (32, 8, 128, F16, 2100, 4300, 0.0, False),
    (24, 4, 256, BF16, 1400, 1400, 0.0, False),   # 264, of a first chunk: all whole
    (24, 4, 256, BF16, 300, 2000, 30.0, False),   # 60: all cut
]


@pytest.mark.parametrize("hq,hkv,d,dtype,n,m,cap,slopes", ONE)
def test_one_chunk(hq, hkv, d, dtype, n, m, cap, slopes, dev):
    say(f"schedule of {hq}/{hkv} D={d} {dtype} {n} of {m} cap={cap} slopes={slopes}")
    cpu, args = _inputs(hq, hkv, d, dtype, [n], [m], 3, dev)
    sl = slopes_of(hq) if slopes else None
    dsl = None if sl is None else sl.to(dev)
    out = _call(args, n, m, cap, dsl)
    plain = _call(args, n, m, cap, dsl, workspace=False)
    same = gqa_prefill_shaped_fn(*args, n, softcap=cap or None, slopes=dsl, max_seqlen_k=m)
    assert torch.equal(bits(out), bits(same))
    edge = 128 // (hq // hkv)
    for a, e in ((0, 8 * edge + 30), (n - 50, n)):  # the first blocks of rows, the cut ones among them, and the last
        exact, limit = _rows(cpu, a, e, cap, sl)
        within(out[a:e], exact, limit, f"rows {a} to {e}")
        within(plain[a:e], exact, limit, "without a workspace")
    if n * (hq // hkv) > 128 * 64:  # whole units give what they give without a workspace
        assert torch.equal(bits(out[n // 2:]), bits(plain[n // 2:]))


BATCHES = [
    # heads, D, type, chunks, cached with the chunk, cap, slopes
    (8, 1, 128, BF16, [600] + [1] * 31, [3000] + [900, 70, 1, 2500] * 7 + [5, 6, 7], 30.0, False),
    (8, 2, 128, F16, [1, 0, 300, 1, 40, 0, 1], [3000, 50, 4000, 1, 2000, 0, 700], 0.0, True),
    (6, 1, 256, BF16, [3] * 70 + [200, 1], [40 * i % 1500 + 3 for i in range(70)] + [3000, 2000], 0.0, False),
    (6, 1, 256, F16, [90, 1, 1, 60], [2500, 2000, 300, 1800], 20.0, True),
]


@pytest.mark.parametrize("hq,hkv,d,dtype,q_lens,lens,cap,slopes", BATCHES)
def test_batches_of_unlike_chunks(hq, hkv, d, dtype, q_lens, lens, cap, slopes, dev):
    """One long chunk among short ones: most blocks of the padded batch do not exist, and the parts of those that do lie side
    by side."""
    say(f"schedule of {hq}/{hkv} D={d} {dtype} chunks {q_lens[:3]}.. of {len(q_lens)}")
    cpu, args = _inputs(hq, hkv, d, dtype, q_lens, lens, 5, dev)
    sl = slopes_of(hq) if slopes else None
    exact, limit = ref.prefill(*cpu, 16, d ** -0.5, True, cap, sl)
    assert _bytes(args, max(q_lens), max(lens)) > 0
    for workspace in (True, False):
        out = _call(args, max(q_lens), max(lens), cap, None if sl is None else sl.to(dev), workspace)
        within(out, exact, limit, f"workspace {workspace}")


def test_offsets_that_go_back_over_all_rows(dev):
    """Offsets that name the same rows twice have more units than the rows, and than the workspace has parts for."""
    say("schedule: offsets that go back")
    n, hq, d = 900, 4, 128
    cpu, args = _inputs(hq, 1, d, BF16, [n], [2500], 7, dev)
    q, k, v, table, _, lens = args
    again = [q, k, v, table.expand(5, -1).contiguous(), torch.tensor([0, n, 0, n, 0, n], dtype=torch.int32, device=dev),
             lens.expand(5).contiguous()]
    exact, limit = _rows(cpu, 0, n, 0.0, None)
    within(_call(again, n, 2500), exact, limit, "rows")


@pytest.mark.parametrize("n,m", [(1400, 1400), (1500, 3100)])  # all units whole; the last round cut
def test_two_graphs(n, m, dev):
    say(f"schedule: graphs of {n} of {m}")
    _, args = _inputs(24, 4, 256, BF16, [n], [m], 9, dev)
    args[1:3] = [x.nan_to_num(0.0) for x in args[1:3]]
    q, graphs = args[0], []
    call = lambda cap: gqa_prefill_shaped_fn(*args, n, softcap=cap, max_seqlen_k=m)  # noqa: E731
    call(None)
    for cap in (None, 20.0):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            graphs.append((graph, call(cap), cap))
    for i in range(3):
        q.copy_(torch.randn(q.shape, device=dev, generator=torch.Generator(dev).manual_seed(i)).to(BF16))
        for graph, out, cap in graphs:
            graph.replay()
            torch.cuda.synchronize()
            kept = out.clone()
            assert torch.equal(bits(kept), bits(call(cap)))
