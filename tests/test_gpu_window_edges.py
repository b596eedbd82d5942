"""Sliding-window attention, append and read-back at the edges of what their
documentation allows, against tests/window_ref.py in 64 bits."""
import ctypes as C

import numpy as np
import pytest
import torch

import dendrite_b200 as dd
from dendrite_b200 import _lib
from tests.test_gpu_window import KVD, WEIGHTS, Dev, _ints
from tests.window_ref import PAGE, Batch, check_attention

pytestmark = pytest.mark.gpu

FORMS = [("decode", [1, 1, 1]), ("prefill", [3, 1, 2]), ("prefill", [200, 90, 130])]
FORM_IDS = ["decode", "few", "many"]


def _run(d, form, **kw):
    out, lse = getattr(d, form)(**kw)
    torch.cuda.synchronize()
    return out, lse


@pytest.mark.parametrize("form,new", FORMS, ids=FORM_IDS)
@pytest.mark.parametrize("fmt", ["bf16", "e4m3", "mxfp8"])
def test_rows_of_zeros_and_tiny_rows(cuda, form, new, fmt):
    """Scores of zero, or nearly: the mean of the visible V, also under tiny K scales."""
    b = Batch(30, [300, 90, 260], new, 8, 2, 128, fmt, True, 40, 3, magnitude=1e-7)
    b.q[::2] = 0
    b.q[1::4] *= 1e-36
    d = Dev(b, cuda)
    out, lse = _run(d, form)
    check_attention(out, lse, b.attention(), f"{form} {fmt}", WEIGHTS[form])


@pytest.mark.parametrize("form,new", FORMS, ids=FORM_IDS)
@pytest.mark.parametrize("fmt", ["bf16", "e4m3", "mxfp8", "f32"])
def test_buffers_on_16_bytes(cuda, form, new, fmt):
    """q, out, the pool and MXFP8's exponents on 16-byte, not 32-byte, borders; 4-byte ones for the rest."""
    b = Batch(31, [300, 90, 260], new, 8, 2, 64, fmt, True, 100, 3)
    d = Dev(b, cuda, torch.float32 if fmt == "f32" else torch.bfloat16)

    def moved(t, by=16):
        n = by // t.element_size()
        buf = torch.empty(t.numel() + n, dtype=t.dtype, device=cuda)
        y = buf[n:].view(t.shape)
        y.copy_(t)
        assert y.data_ptr() % 32 == by
        return y

    want = _run(d, form)
    d.q, d.pool = moved(d.q), moved(d.pool)
    if d.scales is not None:
        d.scales = moved(d.scales, 16 if fmt == "mxfp8" else 4)
    d.indptr, d.ids, d.tokens, d.q_indptr = (moved(x, 4) for x in (d.indptr, d.ids, d.tokens, d.q_indptr))
    out, lse = moved(torch.empty_like(want[0])), moved(torch.empty_like(want[1]), 4)
    _run(d, form, out=out, lse=lse)
    assert torch.equal(out, want[0]) and torch.equal(lse, want[1])
    check_attention(out, lse, b.attention(), f"{form} {fmt}", WEIGHTS[form])


@pytest.mark.parametrize("new", [[3, 1, 2], [200, 90, 130]], ids=["few", "many"])
@pytest.mark.parametrize("fmt", ["bf16", "e4m3", "f32"])
def test_rows_before_the_first_sequence(cuda, new, fmt):
    """q_indptr[0] > 0: the rows before it belong to nobody and stay as they are."""
    b = Batch(32, [300, 90, 260], new, 8, 2, 128, fmt, True, 100, 3)
    d = Dev(b, cuda, torch.float32 if fmt == "f32" else torch.bfloat16)
    front = 161
    d.q = torch.cat([torch.full((front, 8, 128), float("nan"), dtype=d.q.dtype, device=cuda), d.q])
    d.q_indptr = d.q_indptr + front
    out = torch.full((front + b.rows, 8, 128), 7.0, dtype=d.q.dtype, device=cuda)
    lse = torch.full((front + b.rows, 8), 7.0, device=cuda)
    _run(d, "prefill", out=out, lse=lse)
    assert out[:front].eq(7).all() and lse[:front].eq(7).all()
    check_attention(out[front:], lse[front:], b.attention(), fmt, WEIGHTS["prefill"])


@pytest.mark.parametrize("form,new", FORMS, ids=FORM_IDS)
@pytest.mark.parametrize("window,sinks", [(2 ** 31 - 1, 0), (2 ** 31 - 1, 2 ** 31 - 1), (20, 2 ** 31 - 1), (20, 255)])
def test_windows_longer_than_any_sequence(cuda, form, new, window, sinks):
    for fmt in ("bf16", "mxfp8"):
        b = Batch(33, [300, 90, 260], new, 8, 2, 128, fmt, True, window, sinks)
        d = Dev(b, cuda)
        out, lse = _run(d, form)
        check_attention(out, lse, b.attention(), f"{form} {fmt}", WEIGHTS[form])


@pytest.mark.parametrize("fmt", ["bf16", "e4m3", "mxfp8", "f32"])
def test_batches_without_anything(cuda, fmt):
    """No sequences, no rows, no tokens, no pages in any table."""
    b = Batch(34, [5], [2], 8, 2, 128, fmt, True, 8, 2)
    d = Dev(b, cuda, torch.float32 if fmt == "f32" else torch.bfloat16)
    q = d.q
    empty = torch.empty(0, dtype=torch.int32, device=cuda)
    kw = dict(kv_scales=d.scales)
    out, _ = dd.decode_paged_window(d.cfg, q[:0], d.pool, _ints([0], cuda), empty, empty, 8, 2, **kw)
    assert out.shape == (0, 8, 128)
    out, _ = dd.prefill_paged_window(d.cfg, q[:0], d.pool, _ints([0], cuda), _ints([0], cuda), empty, empty, 8, **kw)
    assert out.shape == (0, 8, 128)
    # Rows behind the (no) last sequence, in sequences without rows, and rows of sequences without tokens.
    keep = torch.full_like(q, 7)
    dd.prefill_paged_window(d.cfg, q, d.pool, _ints([0], cuda), _ints([0], cuda), empty, empty, 8, out=keep, **kw)
    dd.prefill_paged_window(d.cfg, q, d.pool, _ints([0, 0, 0], cuda), _ints([0, 0, 0], cuda), empty,
                            _ints([0, 0], cuda), 8, out=keep, **kw)
    assert keep.eq(7).all()
    for rows in (2, 700):
        big = q[:1].expand(rows, 8, 128).contiguous()
        out, lse = dd.prefill_paged_window(d.cfg, big, d.pool, _ints([0, rows - 1, rows], cuda), _ints([0, 0, 0], cuda),
                                           empty, _ints([0, 0], cuda), 8, **kw)
        assert out.eq(0).all() and lse.isneginf().all()
        out, lse = dd.decode_paged_window(d.cfg, big, d.pool, torch.zeros(rows + 1, dtype=torch.int32, device=cuda), empty,
                                          torch.zeros(rows, dtype=torch.int32, device=cuda), 8, **kw)
        assert out.eq(0).all() and lse.isneginf().all()
    before = d.pool.clone()
    k = torch.ones(3, 2, 128, dtype=torch.bfloat16, device=cuda)
    dd.append_kv_paged(d.cfg, d.pool, d.scales, _ints([0], cuda), _ints([0], cuda), empty, empty, k, k)
    dd.append_kv_paged(d.cfg, d.pool, d.scales, _ints([0, 3], cuda), _ints([0, 0], cuda), empty, _ints([3], cuda), k, k)
    assert torch.equal(d.pool.view(torch.uint8), before.view(torch.uint8))
    ko, vo = dd.gather_kv_paged(d.cfg, d.pool, d.scales, _ints([0, 3], cuda), None, _ints([0, 0], cuda), empty, 3)
    assert ko.eq(0).all() and vo.eq(0).all()


@pytest.mark.parametrize("shape", [(160, 1, 64, True), (100, 1, 128, False), (128, 1, 128, True), (66, 2, 64, True),
                                   (16, 2, 256, True)], ids=str)
@pytest.mark.parametrize("fmt", ["bf16", "e4m3", "mxfp8"])
def test_groups_and_dims_of_chunks(cuda, shape, fmt):
    """Groups of more heads than a tile has rows, of as many, and of sizes that leave rows over."""
    Hq, Hkv, D, grouped = shape
    b = Batch(35, [300, 90, 260], [131, 90, 63], Hq, Hkv, D, fmt, grouped, 100, 3, dead=10 ** 6)
    d = Dev(b, cuda)
    out, lse = _run(d, "prefill")
    check_attention(out, lse, b.attention(), f"{shape} {fmt}", WEIGHTS["prefill"])


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("fmt", ["bf16", "e4m3", "mxfp8"])
def test_two_calls_at_once(cuda, D, fmt):
    """Chunk and decode calls of two batches on three streams: each its own results."""
    ds = [Dev(Batch(36 + i, n, m, 16, 8, D, fmt, True, 200, 4), cuda) for i, (n, m) in
          enumerate([([900, 700], [600, 500]), ([800, 900], [700, 333]), ([500] * 6, [1] * 6)])]
    forms = ["prefill", "prefill", "decode"]
    want = [getattr(d, f)() for d, f in zip(ds, forms)]
    for d, (out, lse), f in zip(ds, want, forms):
        check_attention(out, lse, d.b.attention(), f, WEIGHTS[f])
    bufs = [[(torch.zeros_like(o), torch.zeros_like(l)) for o, l in want] for _ in range(6)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in ds]
    for turn in bufs:
        for d, f, st, (o, l) in zip(ds, forms, streams, turn):
            getattr(d, f)(out=o, lse=l, stream=st)
    torch.cuda.synchronize()
    for turn in bufs:
        for (o, l), (wo, wl) in zip(turn, want):
            assert torch.equal(o, wo) and torch.equal(l, wl)


@pytest.mark.parametrize("fmt", ["bf16", "e4m3"])
def test_many_sequences_with_few_rows(cuda, fmt):
    """Thousands of sequences, most of them without a row; unsigned indices; a wrong max_pages."""
    tokens, new = [3] * 4000, [0] * 4000
    for s, (n, m) in {0: (40, 2), 1999: (70, 1), 2500: (33, 33), 3999: (20, 3)}.items():
        tokens[s], new[s] = n, m
    b = Batch(37, tokens, new, 8, 2, 64, fmt, True, 16, 3)
    d = Dev(b, cuda)
    d.indptr, d.ids, d.tokens, d.q_indptr = (x.view(torch.uint32) for x in (d.indptr, d.ids, d.tokens, d.q_indptr))
    for mp in (0, 1, 5000):
        out, lse = _run(d, "prefill", max_pages=mp)
        check_attention(out, lse, b.attention(), f"{fmt} {mp}", WEIGHTS["prefill"])


@pytest.mark.parametrize("form,new", [("decode", [1] * 40), ("prefill", [2] * 40), ("prefill", [30] * 40)], ids=FORM_IDS)
@pytest.mark.parametrize("fmt", ["bf16", "mxfp8"])
def test_sequences_that_share_pages(cuda, form, new, fmt):
    """Forks of one sequence: the same pages in every table."""
    b = Batch(38, [200] + [0] * 39, [new[0]] + [0] * 39, 8, 2, 128, fmt, True, 150, 20)
    ids = b.ids[:13]
    b.tokens, b.new, b.ids = [200] * 40, list(new), ids * 40
    b.indptr = [13 * i for i in range(41)]
    b.rows, b.q_indptr = sum(new), np.concatenate([[0], np.cumsum(new)]).tolist()
    b.q = torch.randn(b.rows, 8, 128, generator=b.g)
    d = Dev(b, cuda)
    out, lse = _run(d, form)
    check_attention(out, lse, b.attention(), f"{form} {fmt}", WEIGHTS[form])


@pytest.mark.parametrize("fmt", ["bf16", "e4m3", "mxfp8"])
def test_pages_past_32_bits(cuda, fmt):
    """The batch's pages at the end of a pool of more than 2^32 bytes: the four calls."""
    Hkv, D = 16, 128
    per_page = 2 * Hkv * PAGE * D * (2 if fmt == "bf16" else 1)
    P = 2 ** 32 // per_page + 200
    shape5 = (P, 2, Hkv, PAGE, D)
    pool = torch.empty(shape5, dtype=torch.bfloat16 if fmt == "bf16" else torch.uint8, device=cuda)
    scales = None if fmt == "bf16" else torch.empty(shape5[:-1] + (D // 32,), dtype=torch.uint8, device=cuda)
    for form, new in (("decode", [1, 1]), ("prefill", [150, 70])):
        b = Batch(39, [300, 90], new, 16, Hkv, D, fmt, True, 100, 3)
        d = Dev(b, cuda)
        pool[P - b.P:] = d.pool
        if fmt == "mxfp8":
            scales[P - b.P:] = d.scales
        if fmt == "e4m3":
            scales = d.scales
        d.pool, d.scales, d.ids = pool, scales, d.ids + (P - b.P)
        d.cfg = dd.make_config(16, Hkv, D, P, kv_dtype=KVD[fmt], gqa_map=_lib.GQA_GROUPED)
        out, lse = _run(d, form)
        check_attention(out, lse, b.attention(), f"{form} {fmt}", WEIGHTS[form])
    g = torch.Generator().manual_seed(40)
    k = torch.randn(20, Hkv, D, generator=g).to(torch.bfloat16).to(cuda)
    small = dd.make_config(Hkv, Hkv, D, 2, kv_dtype=KVD[fmt])
    sp = torch.zeros((2,) + shape5[1:], dtype=pool.dtype, device=cuda)
    ss = scales if fmt == "e4m3" else None if scales is None else torch.zeros((2,) + scales.shape[1:], dtype=torch.uint8, device=cuda)
    got = []
    for cfg, pl, sc, ids in ((small, sp, ss, [0, 1]), (d.cfg, pool, scales, [P - 1, P - 2])):
        t = (_ints([0, 20], cuda), _ints([0, 2], cuda), _ints(ids, cuda))
        dd.append_kv_paged(cfg, pl, sc, *t, _ints([20], cuda), k, -k)
        got.append(dd.gather_kv_paged(cfg, pl, sc, t[0], None, *t[1:], 20))
    assert torch.equal(got[0][0], got[1][0]) and torch.equal(got[0][1], got[1][1])
    assert got[0][0].float().abs().sum() > 0


@pytest.mark.parametrize("form,new", FORMS, ids=FORM_IDS)
@pytest.mark.parametrize("fmt", ["bf16", "mxfp8", "f32"])
def test_without_an_lse(cuda, form, new, fmt):
    """lse may be NULL at the C entry."""
    b = Batch(41, [300, 90, 260], new, 8, 2, 128, fmt, True, 40, 3)
    d = Dev(b, cuda, torch.float32 if fmt == "f32" else torch.bfloat16)
    want, _ = _run(d, form)
    out = torch.zeros_like(want)
    stream = torch.cuda.current_stream().cuda_stream
    head = (C.byref(d.cfg), 3) if form == "decode" else (C.byref(d.cfg), 3, b.rows)
    args = head + (0, 40, 3, d.q.data_ptr(), 8 * 128, d.pool.data_ptr(), None if d.scales is None else d.scales.data_ptr())
    if form == "prefill":
        args += (d.q_indptr.data_ptr(),)
    rc = getattr(_lib.lib, f"dd_{form}_paged_window")(*args, d.indptr.data_ptr(), d.ids.data_ptr(), d.tokens.data_ptr(),
                                                      out.data_ptr(), None, None, stream)
    torch.cuda.synchronize()
    assert rc == 0 and torch.equal(out, want)


def test_prompt_between_the_chunks_of_a_batch(cuda):
    """layer_prefill of another sequence leaves the batch of begin_chunks alone; rows behind the batch go nowhere."""
    g = torch.Generator().manual_seed(42)
    x = torch.randn(60, 12, 128, generator=g).to(torch.bfloat16).to(cuda)
    q, k, v = x[:, :8], x[:, 8:10], x[:, 10:]
    res = []
    for between in (False, True):
        cache = dd.PagedKVCache(1, 8, 8, 2, 128, device=cuda, windows=[(24, 3)])
        cache.begin_chunks([0, 2, 4], [0, 1, 2, 3], [20, 30], [20, 30])
        if between:
            cache.layer_prefill(0, q[:17], k[:17], v[:17], [6, 7], 0)
        res.append(cache.layer_chunk(0, q, k, v)[:50])
    assert torch.equal(*res)


@pytest.mark.parametrize("shape", [(8, 2, 128, True), (16, 2, 64, False), (12, 1, 128, True)], ids=str)
@pytest.mark.parametrize("fmt", ["bf16", "e4m3", "mxfp8"])
@pytest.mark.parametrize("window,sinks", [(0, 0), (4096, 4), (3000, 900), (64, 5000)])
def test_chunks_over_long_sequences(cuda, shape, fmt, window, sinks):
    """Few rows over many tokens: the tokens are split and joined. One sequence, two, one whose shares are empty for some rows."""
    Hq, Hkv, D, grouped = shape
    for tokens, new in (([9001], [100]), ([7000, 5003], [131, 77]), ([6000, 1, 40], [90, 1, 0]), ([130], [130])):
        b = Batch(43, tokens, new, Hq, Hkv, D, fmt, grouped, window, sinks, dead=10 ** 6)
        d = Dev(b, cuda)
        want = b.attention()
        for mp in (0, 563):
            status = torch.zeros(2, dtype=torch.int32, device=cuda)
            out, lse = _run(d, "prefill", max_pages=mp, status=status)
            assert status.tolist() == [0, 0]
            check_attention(out, lse, want, f"{shape} {fmt} {new} {mp}", WEIGHTS["prefill"])
            again, _ = _run(d, "prefill", max_pages=mp)
            assert torch.equal(out, again)


def test_bad_pages_of_a_split_chunk(cuda):
    for fmt in ("bf16", "e4m3", "mxfp8"):
        b = Batch(44, [8000], [120], 8, 2, 128, fmt, True, 0, 0)
        for i in (3, 250, 490):
            b.ids[i] = b.P + 7
        d = Dev(b, cuda)
        status = torch.zeros(2, dtype=torch.int32, device=cuda)
        out, lse = _run(d, "prefill", status=status)
        assert status.tolist() == [1, b.P + 7]
        check_attention(out, lse, b.attention(), fmt, WEIGHTS["prefill"])
