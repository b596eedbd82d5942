"""The tcgen05 kernel of the sliding-window chunks, at sizes that go to it: head layouts, windows,
edges of the buffers, split items. Each call is checked to have launched it."""
import ctypes as C

import numpy as np
import pytest
import torch

import dendrite_b200 as dd
from dendrite_b200 import _lib
from tests.test_gpu_window import KVD, Dev, _ints
from tests.window_ref import PAGE, Batch, check_attention

pytestmark = pytest.mark.gpu

# What a weight is off by: two bf16 terms, both cut off after 8 bits (what the first leaves is below
# 2^-7 of the weight, what the second leaves below 2^-7 of that); one f16 term, rounded.
WEIGHTS = {"bf16": 2.0 ** -14, "mxfp8": 2.0 ** -14, "e4m3": 2.0 ** -11}
FMTS = ["bf16", "e4m3", "mxfp8"]
TOKENS, NEW = [500, 90, 700, 5, 33, 40], [400, 90, 520, 5, 1, 0]


def chunk_kernel(call, launches=1):
    """call(), which launches the chunk kernel that many times and no other attention kernel."""
    _lib.profile_enable(True)
    try:
        _lib.profile_read()
        res = call()
        torch.cuda.synchronize()
        seen = _lib.profile_read()
    finally:
        _lib.profile_enable(False)
    assert (seen["attn_tc"][1], seen["attn_mma"][1]) == (launches, 0), "not the chunk kernel"
    return res


SHAPES = [(32, 8, 128, True), (8, 8, 64, False), (8, 1, 128, True), (12, 2, 128, False), (40, 2, 64, True),
          (64, 1, 128, False)]


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: f"{s[0]}-{s[1]}-{s[2]}-{'g' if s[3] else 't'}")
@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 0), (33, 37), (300, 4)])
def test_layouts(cuda, fmt, shape, window, sinks):
    b = Batch(70 + window, TOKENS, NEW, *shape[:3], fmt, shape[3], window, sinks, dead=10 ** 6)
    d = Dev(b, cuda, strided=window == 33)
    out, lse = chunk_kernel(d.prefill)
    check_attention(out, lse, b.attention(), f"{fmt} {shape} {window}", WEIGHTS[fmt])


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("shape", [(160, 1, 64, True), (100, 1, 128, False), (128, 1, 128, True), (66, 2, 64, True)], ids=str)
def test_wide_groups(cuda, fmt, shape):
    """Groups of as many heads as a tile has rows, and of sizes that leave rows over; more go elsewhere."""
    b = Batch(71, [300, 90, 260], [131, 90, 63], *shape[:3], fmt, shape[3], 100, 3)
    d = Dev(b, cuda)
    out, lse = chunk_kernel(d.prefill) if shape[0] <= 128 * shape[1] else d.prefill()
    check_attention(out, lse, b.attention(), f"{shape} {fmt}", WEIGHTS[fmt])


@pytest.mark.parametrize("fmt", FMTS)
def test_zeros_and_tiny_rows(cuda, fmt):
    b = Batch(72, TOKENS, NEW, 8, 2, 128, fmt, True, 40, 3, magnitude=1e-7)
    b.q[::2] = 0
    b.q[1::4] *= 1e-36
    out, lse = chunk_kernel(Dev(b, cuda).prefill)
    check_attention(out, lse, b.attention(), fmt, WEIGHTS[fmt])


@pytest.mark.parametrize("fmt", FMTS)
def test_large_scores(cuda, fmt):
    b = Batch(73, TOKENS, NEW, 8, 2, 128, fmt, True, 50, 4, magnitude=30.0)
    out, lse = chunk_kernel(Dev(b, cuda).prefill)
    check_attention(out, lse, b.attention(), fmt, WEIGHTS[fmt])


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("window", [0, 8])
def test_rows_before_the_first_token(cuda, fmt, window):
    b = Batch(74, [300, 0, 500, 1], [620, 40, 500, 9], 8, 2, 128, fmt, True, window, 2)
    out, lse = chunk_kernel(Dev(b, cuda).prefill)
    check_attention(out, lse, b.attention(), f"{fmt} {window}", WEIGHTS[fmt])


@pytest.mark.parametrize("fmt", FMTS)
def test_rows_of_nobody(cuda, fmt):
    """Rows before the first sequence and behind the last stay as they are."""
    b = Batch(75, TOKENS, NEW, 8, 2, 128, fmt, True, 100, 3)
    d = Dev(b, cuda)
    front, back = 161, 37
    pad = [torch.full((n, 8, 128), float("nan"), dtype=d.q.dtype, device=cuda) for n in (front, back)]
    d.q, d.q_indptr = torch.cat([pad[0], d.q, pad[1]]), d.q_indptr + front
    out = torch.full(d.q.shape, 7.0, dtype=d.q.dtype, device=cuda)
    lse = torch.full(d.q.shape[:2], 7.0, device=cuda)
    chunk_kernel(lambda: d.prefill(out=out, lse=lse))
    for x in (out, lse):
        assert x[:front].eq(7).all() and x[front + b.rows:].eq(7).all()
    mine = slice(front, front + b.rows)
    check_attention(out[mine], lse[mine], b.attention(), fmt, WEIGHTS[fmt])


@pytest.mark.parametrize("fmt", FMTS)
def test_rows_without_any_token(cuda, fmt):
    b = Batch(76, [5], [2], 8, 2, 128, fmt, True, 8, 2)
    d = Dev(b, cuda)
    q = d.q[:1].expand(3000, 8, 128).contiguous()
    out, lse = chunk_kernel(lambda: dd.prefill_paged_window(
        d.cfg, q, d.pool, _ints([0, 2999, 3000], cuda), _ints([0, 0, 0], cuda),
        torch.empty(0, dtype=torch.int32, device=cuda), _ints([0, 0], cuda), 8, kv_scales=d.scales))
    assert out.eq(0).all() and lse.isneginf().all()


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("window,sinks", [(2 ** 31 - 1, 0), (2 ** 31 - 1, 2 ** 31 - 1), (20, 2 ** 31 - 1), (20, 255)])
def test_windows_longer_than_any_sequence(cuda, fmt, window, sinks):
    b = Batch(77, TOKENS, NEW, 8, 2, 128, fmt, True, window, sinks)
    d = Dev(b, cuda)
    out, lse = chunk_kernel(lambda: d.prefill(max_pages=44))
    check_attention(out, lse, b.attention(), f"{fmt} {window} {sinks}", WEIGHTS[fmt])


@pytest.mark.parametrize("fmt", FMTS)
def test_borders_of_the_buffers(cuda, fmt):
    """q, out, the pool and MXFP8's exponents on 16-byte, not 32-byte, borders; 4-byte ones for the rest; no lse."""
    b = Batch(78, TOKENS, NEW, 16, 2, 64, fmt, True, 100, 3)
    d = Dev(b, cuda)

    def moved(t, by=16):
        n = by // t.element_size()
        y = torch.empty(t.numel() + n, dtype=t.dtype, device=cuda)[n:].view(t.shape)
        y.copy_(t)
        assert y.data_ptr() % 32 == by
        return y

    want = chunk_kernel(d.prefill)
    check_attention(*want, b.attention(), fmt, WEIGHTS[fmt])
    d.q, d.pool = moved(d.q), moved(d.pool)
    if d.scales is not None:
        d.scales = moved(d.scales, 16 if fmt == "mxfp8" else 4)
    d.indptr, d.ids, d.tokens, d.q_indptr = (moved(x, 4) for x in (d.indptr, d.ids, d.tokens, d.q_indptr))
    out, lse = moved(torch.empty_like(want[0])), moved(torch.empty_like(want[1]), 4)
    chunk_kernel(lambda: d.prefill(out=out, lse=lse))
    assert torch.equal(out, want[0]) and torch.equal(lse, want[1])
    out.zero_()
    rc = chunk_kernel(lambda: _lib.lib.dd_prefill_paged_window(
        C.byref(d.cfg), len(NEW), b.rows, 0, 100, 3, d.q.data_ptr(), 16 * 64, d.pool.data_ptr(),
        None if d.scales is None else d.scales.data_ptr(), d.q_indptr.data_ptr(), d.indptr.data_ptr(), d.ids.data_ptr(),
        d.tokens.data_ptr(), out.data_ptr(), None, None, torch.cuda.current_stream().cuda_stream))
    assert rc == 0 and torch.equal(out, want[0])


@pytest.mark.parametrize("fmt", FMTS)
def test_missing_pages(cuda, fmt):
    b = Batch(79, TOKENS, NEW, 8, 2, 128, fmt, True, 0, 0)
    good = b.ids[3]
    b.ids[3] = b.P + 5
    d = Dev(b, cuda)
    status = torch.zeros(2, dtype=torch.int32, device=cuda)
    out, lse = chunk_kernel(lambda: d.prefill(status=status))
    assert status.tolist() == [1, b.P + 5]
    check_attention(out, lse, b.attention(), "bad id", WEIGHTS[fmt])
    b.ids[3] = good
    short = b.indptr[3] - 1                # the third table ends a page early
    b.ids[short] = -1
    d = Dev(b, cuda)
    d.indptr = torch.cat([d.indptr[:3], d.indptr[3:] - 1])
    d.ids = torch.cat([d.ids[:short], d.ids[short + 1:]])
    status.zero_()
    out, lse = chunk_kernel(lambda: d.prefill(status=status))
    assert status.tolist() == [1, b.tokens[2] // PAGE]
    check_attention(out, lse, b.attention(), "short table", WEIGHTS[fmt])


@pytest.mark.parametrize("fmt", FMTS)
def test_pages_past_32_bits(cuda, fmt):
    """The batch's pages at the end of a pool of more than 2^32 bytes."""
    Hkv, D = 16, 128
    b = Batch(80, [700, 90], [500, 70], 16, Hkv, D, fmt, True, 100, 3)
    P = 2 ** 32 // (2 * Hkv * PAGE * D * (2 if fmt == "bf16" else 1)) + 200
    d = Dev(b, cuda)
    pool = torch.empty((P,) + d.pool.shape[1:], dtype=d.pool.dtype, device=cuda)
    pool[P - b.P:] = d.pool
    if fmt == "mxfp8":
        scales = torch.empty((P,) + d.scales.shape[1:], dtype=torch.uint8, device=cuda)
        scales[P - b.P:] = d.scales
        d.scales = scales
    d.pool, d.ids = pool, d.ids + (P - b.P)
    d.cfg = dd.make_config(16, Hkv, D, P, kv_dtype=KVD[fmt], gqa_map=_lib.GQA_GROUPED)
    out, lse = chunk_kernel(d.prefill)
    check_attention(out, lse, b.attention(), fmt, WEIGHTS[fmt])


@pytest.mark.parametrize("shape", [(8, 2, 128, True), (16, 2, 64, False), (12, 1, 128, True)], ids=str)
@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("window,sinks", [(0, 0), (8000, 900)])
def test_items_that_are_shared_out(cuda, shape, fmt, window, sinks):
    """Few rows over many tokens: an item's tokens are split over a cluster and joined; missing pages there."""
    b = Batch(81, [15000], [300], *shape[:3], fmt, shape[3], window, sinks, dead=10 ** 6)
    d = Dev(b, cuda)
    status = torch.zeros(2, dtype=torch.int32, device=cuda)
    out, lse = chunk_kernel(lambda: d.prefill(max_pages=938, status=status))
    assert status.tolist() == [0, 0]
    check_attention(out, lse, b.attention(), f"{shape} {fmt}", WEIGHTS[fmt])
    again, _ = chunk_kernel(lambda: d.prefill(max_pages=938))
    assert torch.equal(out, again)
    for i in (580, 700, 937):
        b.ids[i] = b.P + 7
    d = Dev(b, cuda)
    out, lse = chunk_kernel(lambda: d.prefill(max_pages=938, status=status))
    assert status.tolist() == [1, b.P + 7]
    check_attention(out, lse, b.attention(), f"{shape} {fmt} missing", WEIGHTS[fmt])


@pytest.mark.parametrize("fmt", FMTS)
def test_captured_and_replayed(cuda, fmt):
    """A captured chunk follows the arrays' contents; two graphs at once share nothing."""
    batches = [Batch(82 + i, n, [400, 3, 520], 8, 2, 128, fmt, True, 64, 4, spare=80) for i, n in
               enumerate(([500, 64, 700], [401, 200, 521], [899, 3, 640]))]
    P, N = max(b.P for b in batches), max(len(b.ids) for b in batches)
    devs = [Dev(b, cuda) for b in batches]
    cfg = dd.make_config(8, 2, 128, P, kv_dtype=KVD[fmt], gqa_map=_lib.GQA_GROUPED)

    def pad(t, n):
        return torch.cat([t, torch.zeros((n - t.shape[0],) + t.shape[1:], dtype=t.dtype, device=cuda)])

    ins = [dict(q=d.q.clone(), pool=pad(d.pool, P), indptr=d.indptr, ids=pad(d.ids, N), tokens=d.tokens) for d in devs]
    for i, d in zip(ins, devs):
        if fmt != "bf16":
            i["scales"] = pad(d.scales, P) if fmt == "mxfp8" else d.scales
    graphs = []
    for _ in range(2):
        buf = {k: v.clone() for k, v in ins[0].items()}
        out, lse = torch.empty_like(buf["q"]), torch.empty(buf["q"].shape[:2], device=cuda)

        def call():
            dd.prefill_paged_window(cfg, buf["q"], buf["pool"], devs[0].q_indptr, buf["indptr"], buf["ids"], buf["tokens"],
                                    64, 4, kv_scales=buf.get("scales"), out=out, lse=lse)
        chunk_kernel(call)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            call()
        graphs.append((graph, buf, out, lse))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    wants = [b.attention() for b in batches]
    for i in (1, 2, 0):
        for j, (graph, buf, out, lse) in enumerate(graphs):
            for k, v in ins[(i + j) % 3].items():
                buf[k].copy_(v)
            out.fill_(float("nan"))
        torch.cuda.synchronize()
        for st, (graph, *_) in zip(streams, graphs):
            with torch.cuda.stream(st):
                graph.replay()
        torch.cuda.synchronize()
        for j, (graph, buf, out, lse) in enumerate(graphs):
            check_attention(out, lse, wants[(i + j) % 3], f"{fmt} {i} {j}", WEIGHTS[fmt])


@pytest.mark.parametrize("fmt", FMTS)
def test_through_the_cache(cuda, fmt):
    """A long prompt as chunks of a PagedKVCache is the prompt at once."""
    g = torch.Generator().manual_seed(83)
    n, cut = 1500, 700
    x = torch.randn(n, 12, 128, generator=g).to(torch.bfloat16).to(cuda)
    q, k, v = x[:, :8], x[:, 8:10], x[:, 10:]
    table = torch.randperm(96, generator=g).tolist()
    outs = []
    for cuts in ([0, n], [0, cut, n]):
        cache = dd.PagedKVCache(1, 96, 8, 2, 128, kv_dtype=fmt, device=cuda, windows=[(200, 3)],
                                e4m3_scales=[torch.full((2, 2), 0.02)] if fmt == "e4m3" else None)
        res = []
        for a, e in zip(cuts, cuts[1:]):
            cache.begin_chunks([0, 96], table, [e], [e - a])
            res.append(chunk_kernel(lambda: cache.layer_chunk(0, q[a:e], k[a:e], v[a:e])))
        cache.check()
        outs.append(torch.cat(res).float())
    kk, vv = (t.double().cpu() for t in cache.read_tokens(0, [0, 96], table, [0], [n], torch.float32))
    b = Batch.__new__(Batch)
    b.tokens, b.new, b.Hq, b.Hkv, b.D, b.fmt, b.grouped = [n], [n], 8, 2, 128, "f64", True
    b.window, b.sinks, b.rows, b.q_indptr = 200, 3, n, [0, n]
    b.P = -(-n // PAGE)
    b.indptr, b.ids = [0, b.P], list(range(b.P))
    pool = np.zeros((b.P, 2, 2, PAGE, 128))
    for j in range(n):
        pool[j // PAGE, 0, :, j % PAGE], pool[j // PAGE, 1, :, j % PAGE] = kk[j], vv[j]
    b.values = lambda: pool
    want = b.attention(q.cpu())
    for o in outs:
        check_attention(o.to(torch.bfloat16), torch.tensor(want[1]), want, fmt, WEIGHTS[fmt])
