"""Sliding-window attention over the paged cache (decode and chunk forms),
ragged append and read-back, against tests/window_ref.py in 64 bits."""
import numpy as np
import pytest
import torch

import dendrite_b200 as dd
from dendrite_b200 import _lib
from tests.window_ref import PAGE, Batch, check_attention, encode

pytestmark = pytest.mark.gpu

KVD = {"f32": _lib.DTYPE_F32, "bf16": _lib.DTYPE_BF16, "e4m3": _lib.DTYPE_E4M3, "mxfp8": _lib.DTYPE_MXFP8}
# Rounding of the softmax weights (half a step): one bf16 term in the chunk kernel at worst.
WEIGHTS = {"decode": 2.0 ** -11, "prefill": 2.0 ** -8}


def _ints(v, dev):
    return torch.tensor(v, dtype=torch.int32, device=dev)


class Dev:
    """A Batch on the device, with what the calls take."""

    def __init__(self, b: Batch, dev, q_dtype=torch.bfloat16, strided=False):
        self.b = b
        self.cfg = dd.make_config(b.Hq, b.Hkv, b.D, b.P, kv_dtype=KVD[b.fmt],
                                  q_dtype=_lib.DTYPE_F32 if q_dtype == torch.float32 else _lib.DTYPE_BF16,
                                  gqa_map=_lib.GQA_GROUPED if b.grouped else _lib.GQA_TILED)
        self.pool = b.pool.to(dev)
        self.scales = None if b.scales is None else b.scales.to(dev)
        self.indptr, self.ids, self.tokens = _ints(b.indptr, dev), _ints(b.ids, dev), _ints(b.tokens, dev)
        self.q_indptr = _ints(b.q_indptr, dev)
        b.q = b.q.to(q_dtype)
        self.q = b.q.to(dev)
        if strided:  # inside a wider row, as a fused projection leaves it
            wide = torch.full((b.rows, b.Hq + 3, b.D), float("nan"), dtype=q_dtype, device=dev)
            wide[:, 1:1 + b.Hq] = self.q
            self.q = wide[:, 1:1 + b.Hq]

    def decode(self, **kw):
        return dd.decode_paged_window(self.cfg, self.q, self.pool, self.indptr, self.ids, self.tokens,
                                      self.b.window, self.b.sinks, kv_scales=self.scales, **kw)

    def prefill(self, **kw):
        return dd.prefill_paged_window(self.cfg, self.q, self.pool, self.q_indptr, self.indptr, self.ids,
                                       self.tokens, self.b.window, self.b.sinks, kv_scales=self.scales, **kw)


LENGTHS = [1, 2, 15, 16, 17, 33, 100, 257, 400, 0]
SHAPES = [(32, 8, 128, True), (8, 8, 64, False), (8, 1, 128, True), (12, 2, 128, False), (40, 2, 64, True),
          (64, 1, 128, False), (6, 3, 256, True)]


@pytest.mark.parametrize("fmt", ["bf16", "e4m3", "mxfp8", "f32"])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: f"{s[0]}-{s[1]}-{s[2]}-{'g' if s[3] else 't'}")
@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 0), (16, 4), (33, 37), (128, 1), (500, 16)])
def test_decode(cuda, fmt, shape, window, sinks):
    Hq, Hkv, D, grouped = shape
    b = Batch(1 + window, LENGTHS, [1] * len(LENGTHS), Hq, Hkv, D, fmt, grouped, window, sinks)
    for q_dtype in ((torch.bfloat16,) if fmt != "f32" else (torch.bfloat16, torch.float32)):
        d = Dev(b, cuda, q_dtype, strided=window == 16)
        out, lse = d.decode(max_pages=0 if window == 33 else 26)
        torch.cuda.synchronize()
        check_attention(out, lse, b.attention(), f"{fmt} {shape} {window} {sinks}", WEIGHTS["decode"])


@pytest.mark.parametrize("fmt", ["bf16", "e4m3", "mxfp8", "f32"])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: f"{s[0]}-{s[1]}-{s[2]}-{'g' if s[3] else 't'}")
@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 0), (16, 4), (33, 37), (128, 1), (500, 16)])
@pytest.mark.parametrize("new", ["few", "many"])
def test_prefill(cuda, fmt, shape, window, sinks, new):
    Hq, Hkv, D, grouped = shape
    tokens = [1, 16, 30, 77, 5, 300, 200]
    counts = [1, 3, 2, 5, 0, 4, 1] if new == "few" else [1, 16, 17, 70, 5, 131, 0]
    b = Batch(2 + window, tokens, counts, Hq, Hkv, D, fmt, grouped, window, sinks, dead=10 ** 6)
    d = Dev(b, cuda, torch.float32 if fmt == "f32" else torch.bfloat16, strided=window == 16)
    out, lse = d.prefill()
    torch.cuda.synchronize()
    check_attention(out, lse, b.attention(), f"{fmt} {shape} {window} {sinks}", WEIGHTS["prefill"])


def test_long_sequences(cuda):
    """Work split over a long axis: one sequence, many pages, windows of all sizes."""
    for fmt, window, sinks, n in (("bf16", 0, 0, 9001), ("bf16", 4096, 4, 9001), ("e4m3", 8000, 100, 9005),
                                  ("mxfp8", 0, 0, 8191), ("mxfp8", 5000, 16, 8193)):
        b = Batch(n, [n], [1], 8, 2, 128, fmt, True, window, sinks)
        d = Dev(b, cuda)
        for mp in (0, 600):
            out, lse = d.decode(max_pages=mp)
            check_attention(out, lse, b.attention(), f"{fmt} {window}", WEIGHTS["decode"])


def test_rows_before_the_first_token(cuda):
    """More rows than tokens: the first rows stand for no token and see nothing."""
    for fmt, window in (("bf16", 0), ("mxfp8", 8), ("f32", 8)):
        b = Batch(5, [3, 0, 20], [6, 4, 20], 8, 2, 128, fmt, True, window, 2)
        d = Dev(b, cuda, torch.float32 if fmt == "f32" else torch.bfloat16)
        out, lse = d.prefill()
        check_attention(out, lse, b.attention(), fmt, WEIGHTS["prefill"])


@pytest.mark.parametrize("rows", ["few", "many"])
def test_rows_behind_the_last_sequence(cuda, rows):
    n = [4, 2] if rows == "few" else [300, 150]
    b = Batch(6, [400, 160], n, 8, 2, 128, "bf16", True, 64, 4)
    d = Dev(b, cuda)
    pad = 37
    d.q = torch.cat([d.q, torch.full((pad, 8, 128), float("nan"), dtype=d.q.dtype, device=cuda)])
    out = torch.full((b.rows + pad, 8, 128), 7.0, dtype=torch.bfloat16, device=cuda)
    lse = torch.full((b.rows + pad, 8), 7.0, device=cuda)
    d.prefill(out=out, lse=lse)
    torch.cuda.synchronize()
    assert out[b.rows:].eq(7).all() and lse[b.rows:].eq(7).all()
    check_attention(out[:b.rows], lse[:b.rows], b.attention(), rows, WEIGHTS["prefill"])


def test_bad_pages_are_skipped_and_reported(cuda):
    for new in ([1, 1], [40, 90]):
        b = Batch(7, [200, 200], new, 8, 2, 128, "bf16", True, 0, 0)
        bad = b.ids[3]
        b.ids[3] = b.P + 5
        d = Dev(b, cuda)
        status = torch.zeros(2, dtype=torch.int32, device=cuda)
        out, lse = d.prefill(status=status)
        assert status.tolist() == [1, b.P + 5]
        check_attention(out, lse, b.attention(), "bad id", WEIGHTS["prefill"])
        b.ids[3] = bad
        # A table that ends before the sequence does: the last page is missing.
        b.indptr[2] -= 1
        b.ids[-1] = -1
        d = Dev(b, cuda)
        d.ids[-1] = 0
        status.zero_()
        out, lse = d.prefill(status=status)
        assert status.tolist() == [1, 12]
        check_attention(out, lse, b.attention(), "short table", WEIGHTS["prefill"])


def test_infinite_and_nan_scores(cuda):
    """A visible NaN reaches its own sequence and no other; an invisible one nobody."""
    b = Batch(8, [50, 50], [1, 1], 8, 2, 128, "bf16", True, 16, 2)
    page1, slot1 = b.place(1, 33)        # outside the window, in the window's first page
    b.pool[page1, :, :, slot1] = float("nan")
    d = Dev(b, cuda)
    out, lse = d.decode()
    check_attention(out, lse, b.attention(), "invisible", WEIGHTS["decode"])
    page, slot = b.place(0, 40)
    b.pool[page, :, 0, slot] = float("nan")
    d = Dev(b, cuda)
    out, lse = d.decode()
    o = out.float().cpu()
    assert o[0, :4].isnan().all() and lse[0, :4].isnan().all()
    assert o[0, 4:].isfinite().all() and o[1].isfinite().all()


def test_large_scores(cuda):
    """Scores far apart: one token takes nearly everything, whichever it is."""
    for fmt in ("bf16", "e4m3", "mxfp8"):
        for new in ([1] * 4, [60] * 4):
            b = Batch(9, [61, 300, 150, 77], new, 8, 2, 128, fmt, True, 50, 4, magnitude=30.0)
            d = Dev(b, cuda)
            out, lse = d.prefill()
            check_attention(out, lse, b.attention(), f"{fmt} {new[0]}", WEIGHTS["prefill"])


def test_mxfp8_scales_far_apart(cuda):
    """Blocks of one dim range whose exponents differ by up to 20 from token to token."""
    for new in ([1, 1], [9, 70]):
        b = Batch(10, [90, 300], new, 8, 2, 128, "mxfp8", True, 64, 4)
        r = torch.randint(-10, 11, b.scales.shape, generator=b.g)
        r[:, 0] = r[:, 0].clamp(-2, 0)   # K: keep the scores moderate
        live = b.scales != 0xFF
        b.scales = torch.where(live, (b.scales.int() + r).to(torch.uint8), b.scales)
        d = Dev(b, cuda)
        out, lse = d.prefill()
        check_attention(out, lse, b.attention(), str(new), WEIGHTS["prefill"])


@pytest.mark.parametrize("fmt", ["bf16", "e4m3", "mxfp8"])
def test_forms_agree_and_repeat(cuda, fmt):
    """Decode is the chunk form of one row; the same call gives the same bits."""
    b = Batch(11, [70, 500, 33, 900], [1] * 4, 16, 4, 128, fmt, True, 256, 4)
    d = Dev(b, cuda)
    o1, l1 = d.decode()
    o2, l2 = d.decode()
    o3, l3 = d.prefill()
    assert torch.equal(o1, o2) and torch.equal(l1, l2)
    assert torch.equal(o1, o3) and torch.equal(l1, l3)
    b = Batch(12, [700, 500], [300, 41], 16, 4, 128, fmt, True, 256, 4)
    d = Dev(b, cuda)
    o1, l1 = d.prefill()
    o2, l2 = d.prefill()
    assert torch.equal(o1, o2) and torch.equal(l1, l2)


def test_matches_the_cascade_without_a_window(cuda):
    """window = 0 is the attention of the framework's plans (both are within their bounds of the same sums)."""
    b = Batch(13, [300, 77], [64, 20], 8, 2, 128, "bf16", True, 0, 0, junk=0.0)
    d = Dev(b, cuda)
    out, lse = d.prefill()
    plan = dd.CascadePlan.prefill(d.cfg, b.indptr, np.array(b.ids, np.uint32),
                                  [n - m for n, m in zip(b.tokens, b.new)], b.new)
    ref, ref_lse = dd.cascade_decode(d.cfg, plan, d.q.contiguous(), d.pool)
    want = b.attention()
    check_attention(out, lse, want, "window form", WEIGHTS["prefill"])
    check_attention(ref, ref_lse, want, "cascade", WEIGHTS["prefill"])


@pytest.mark.parametrize("form", ["decode", "prefill"])
def test_captured_and_replayed(cuda, form):
    """A captured call follows the arrays' contents: lengths, tables, values; two graphs share nothing."""
    new = [1] * 3 if form == "decode" else [100, 3, 40]
    batches = [Batch(20 + i, n, new, 8, 2, 128, "mxfp8", True, 64, 4, spare=40 - 0) for i, n in
               enumerate(([130, 64, 300], [101, 200, 41], [299, 3, 256]))]
    P = max(b.P for b in batches)
    N = max(len(b.ids) for b in batches)
    devs = [Dev(b, cuda) for b in batches]
    cfg = dd.make_config(8, 2, 128, P, kv_dtype=KVD["mxfp8"], gqa_map=_lib.GQA_GROUPED)

    def pad(t, n):
        return torch.cat([t, torch.zeros((n - t.shape[0],) + t.shape[1:], dtype=t.dtype, device=t.device)])

    ins = [dict(q=d.q.clone(), pool=pad(d.pool, P), scales=pad(d.scales, P), indptr=d.indptr, ids=pad(d.ids, N),
                tokens=d.tokens) for d in devs]
    graphs = []
    for _ in range(2):
        buf = {k: v.clone() for k, v in ins[0].items()}
        out, lse = torch.empty_like(buf["q"]), torch.empty(buf["q"].shape[:2], device=cuda)

        def call(stream=None):
            if form == "decode":
                dd.decode_paged_window(cfg, buf["q"], buf["pool"], buf["indptr"], buf["ids"], buf["tokens"], 64, 4,
                                       kv_scales=buf["scales"], out=out, lse=lse)
            else:
                dd.prefill_paged_window(cfg, buf["q"], buf["pool"], devs[0].q_indptr, buf["indptr"], buf["ids"],
                                        buf["tokens"], 64, 4, kv_scales=buf["scales"], out=out, lse=lse)
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            call()
        torch.cuda.current_stream().wait_stream(s)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            call()
        graphs.append((graph, buf, out, lse))
    for i in (1, 2, 0):
        other = (i + 1) % 3
        for j, (graph, buf, out, lse) in enumerate(graphs):
            for k, v in ins[i if j == 0 else other].items():
                buf[k].copy_(v)
            out.fill_(float("nan"))
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream(), torch.cuda.Stream()]
        for st, (graph, *_) in zip(streams, graphs):
            with torch.cuda.stream(st):
                graph.replay()
        torch.cuda.synchronize()
        for j, (graph, buf, out, lse) in enumerate(graphs):
            b = batches[i if j == 0 else other]
            check_attention(out, lse, b.attention(), f"replay {i} graph {j}", WEIGHTS["prefill"])


def test_on_another_stream(cuda):
    b = Batch(14, [800] * 3, [200] * 3, 8, 2, 128, "bf16", True, 128, 4)
    d = Dev(b, cuda)
    want = d.prefill()[0]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    got = d.prefill(stream=s)[0]
    s.synchronize()
    assert torch.equal(got, want)


# ---------------------------------------------------------- append / read-back
IO_SHAPES = [(8, 128), (1, 64), (3, 256), (2, 128)]


def _tables(rng, tokens):
    """Page tables over a shuffled pool with spare pages; returns (indptr, ids, pages)."""
    need = [-(-n // PAGE) for n in tokens]
    order = rng.permutation(sum(need) + 3)
    indptr = np.concatenate([[0], np.cumsum(need)]).astype(int)
    return indptr.tolist(), order[:indptr[-1]].tolist(), len(order)


@pytest.mark.parametrize("fmt", ["bf16", "e4m3", "mxfp8", "f32"])
@pytest.mark.parametrize("shape", IO_SHAPES, ids=str)
@pytest.mark.parametrize("src", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
def test_append_and_gather(cuda, fmt, shape, src):
    Hkv, D = shape
    rng = np.random.default_rng(3)
    g = torch.Generator().manual_seed(4)
    tokens, new = [40, 1, 16, 100, 7, 333], [3, 1, 16, 50, 0, 333]
    indptr, ids, P = _tables(rng, tokens)
    rows = sum(new)
    new_indptr = np.concatenate([[0], np.cumsum(new)]).tolist()
    wide = (torch.randn(rows + 5, 2 * Hkv + 1, D, generator=g) * 3).to(src)
    wide[::13] *= 90                     # outliers: saturating codes
    wide[1::29] = 0
    wide[2::31, :, 5] *= 1e-6
    dw = wide.to(cuda)
    k, v = dw[:, :Hkv], dw[:, Hkv:2 * Hkv]
    cfg = dd.make_config(Hkv, Hkv, D, P, kv_dtype=KVD[fmt])
    shape5 = (P, 2, Hkv, PAGE, D)
    scales = None
    if fmt in ("bf16", "f32"):
        pool = torch.randn(shape5, generator=g).to(torch.bfloat16 if fmt == "bf16" else torch.float32)
    else:
        pool = torch.randint(0, 120, shape5, generator=g).to(torch.uint8)
        scales = torch.rand(2, Hkv, generator=g) * 0.05 + 0.01 if fmt == "e4m3" else \
            torch.randint(100, 140, shape5[:-1] + (D // 32,), generator=g).to(torch.uint8)
    want, want_s = pool.clone(), None if scales is None else scales.clone()
    for s in range(len(tokens)):
        for i in range(new[s]):
            pos, r = tokens[s] - new[s] + i, new_indptr[s] + i
            page, slot = ids[indptr[s] + pos // PAGE], pos % PAGE
            for which, x in ((0, wide[r, :Hkv]), (1, wide[r, Hkv:2 * Hkv])):
                if fmt in ("bf16", "f32"):
                    want[page, which, :, slot] = x.to(want.dtype)
                else:
                    c, e = encode(x.float(), fmt, scales[which][:, None] if fmt == "e4m3" else None)
                    want[page, which, :, slot] = c
                    if e is not None:
                        want_s[page, which, :, slot] = e
    dp, ds = pool.to(cuda), None if scales is None else scales.to(cuda)
    status = torch.zeros(2, dtype=torch.int32, device=cuda)
    dd.append_kv_paged(cfg, dp, ds, _ints(new_indptr, cuda), _ints(indptr, cuda), _ints(ids, cuda),
                       _ints(tokens, cuda), k, v, status=status)
    torch.cuda.synchronize()
    assert status.tolist() == [0, 0]
    as_bits = (lambda t: t.view(torch.int16)) if fmt == "bf16" else (lambda t: t)
    assert torch.equal(as_bits(dp.cpu()), as_bits(want))
    if ds is not None:
        assert torch.equal(ds.cpu(), want_s)

    # Read back: ragged ranges, the whole of one sequence among them.
    first, count = [5, 0, 3, 90, 0, 0], [30, 1, 0, 10, 7, 333]
    out_indptr = np.concatenate([[0], np.cumsum(count)]).tolist()
    vals = want.double()
    if fmt != "bf16" and fmt != "f32":
        vals = want.view(torch.float8_e4m3fn).double()
        sc = want_s.double()[None, :, :, None, None] if fmt == "e4m3" else \
            torch.exp2(want_s.double() - 127).repeat_interleave(32, -1)
        vals = vals * sc
    for out_dtype in (torch.bfloat16, torch.float32):
        n = out_indptr[-1]
        ko = torch.full((n + 2, Hkv, D), 7.0, dtype=out_dtype, device=cuda)
        vo = ko.clone()
        dd.gather_kv_paged(cfg, dp, ds, _ints(out_indptr, cuda), _ints(first, cuda), _ints(indptr, cuda),
                           _ints(ids, cuda), n + 2, out_dtype, k=ko, v=vo, status=status)
        torch.cuda.synchronize()
        assert status.tolist() == [0, 0] and ko[n:].eq(7).all() and vo[n:].eq(7).all()
        for s in range(len(tokens)):
            for i in range(count[s]):
                pos, r = first[s] + i, out_indptr[s] + i
                page, slot = ids[indptr[s] + pos // PAGE], pos % PAGE
                # code * scale has 28 significant bits at most in E4M3 and is rounded to f32 first.
                assert torch.equal(ko[r].cpu(), vals[page, 0, :, slot].float().to(out_dtype))
                assert torch.equal(vo[r].cpu(), vals[page, 1, :, slot].float().to(out_dtype))


def test_append_gather_bad_pages(cuda):
    Hkv, D, P = 2, 128, 9
    cfg = dd.make_config(Hkv, Hkv, D, P)
    pool = torch.zeros(P, 2, Hkv, PAGE, D, dtype=torch.bfloat16, device=cuda)
    k = torch.ones(40, Hkv, D, dtype=torch.bfloat16, device=cuda)
    # sequence 0: 20 tokens, its second page is outside the pool; sequence 1: 20 tokens, one page only
    indptr, ids = _ints([0, 2, 3], cuda), _ints([4, P, 6], cuda)
    status = torch.zeros(2, dtype=torch.int32, device=cuda)
    dd.append_kv_paged(cfg, pool, None, _ints([0, 20, 40], cuda), indptr, ids, _ints([20, 20], cuda), k, k,
                       status=status)
    st = status.tolist()
    assert st[0] == 1 and st[1] in list(range(16, 20)) + list(range(36, 40))
    assert pool[4].eq(1).all() and pool[6].eq(1).all()
    assert pool.float().sum().item() == 2 * 2 * Hkv * PAGE * D
    status.zero_()
    ko, vo = dd.gather_kv_paged(cfg, pool, None, _ints([0, 20, 40], cuda), None, indptr, ids, 40, status=status)
    st = status.tolist()
    assert st[0] == 1 and st[1] in list(range(16, 20)) + list(range(36, 40))
    for t in (ko, vo):
        assert t[:16].eq(1).all() and t[20:36].eq(1).all() and t[16:20].eq(0).all() and t[36:].eq(0).all()
    # A token before the sequence's first one (more new rows than tokens) goes nowhere.
    pool.zero_()
    dd.append_kv_paged(cfg, pool, None, _ints([0, 3], cuda), _ints([0, 1], cuda), _ints([2], cuda),
                       _ints([2], cuda), k[:3], k[:3])
    assert pool[2, :, :, :2].eq(1).all() and pool.float().sum().item() == 2 * 2 * Hkv * D


def test_append_one_token_per_sequence(cuda):
    """new_indptr None: row s is the last token of sequence s."""
    Hkv, D, P = 2, 64, 6
    cfg = dd.make_config(Hkv, Hkv, D, P)
    pool = torch.zeros(P, 2, Hkv, PAGE, D, dtype=torch.bfloat16, device=cuda)
    k = torch.arange(1, 4, device=cuda).to(torch.bfloat16)[:, None, None].expand(3, Hkv, D).contiguous()
    dd.append_kv_paged(cfg, pool, None, None, _ints([0, 2, 3, 4], cuda), _ints([5, 0, 1, 3], cuda),
                       _ints([17, 4, 16], cuda), k, -k)
    for page, slot, x in ((0, 0, 1), (1, 3, 2), (3, 15, 3)):
        assert pool[page, 0, :, slot].eq(x).all() and pool[page, 1, :, slot].eq(-x).all()
    assert pool.float().abs().sum().item() == 2 * Hkv * D * 6


def test_append_e4m3_at_the_borders_of_codes(cuda):
    """x / scale rounded to f32 and then to E4M3: x within a few steps of every
    border between two codes, and where the quotient leaves f32's middle range,
    under scales of all kinds. The codes are those of torch's f32 division."""
    Hkv, D = 1, 256
    codes = torch.arange(0, 127, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    borders = torch.cat([(codes[1:] + codes[:-1]) / 2, codes, torch.tensor([464.0, 480.0, 1e3, 2.0 ** -21, 2.0 ** 11])])
    g = torch.Generator().manual_seed(9)
    scales = torch.cat([torch.rand(20, generator=g) * 0.1, torch.exp2(torch.randint(-60, 60, (12,), generator=g).float()),
                        torch.rand(12, generator=g) * 2.0 ** -60, torch.tensor([1.0, 2.0 ** -70, 2.0 ** 80, 2.0 ** -126])])
    scales = torch.where(scales > 0, scales, torch.tensor(1.0)).float()
    cfg = dd.make_config(Hkv, Hkv, D, 8, kv_dtype=KVD["e4m3"])
    for s in scales:
        x = (borders * s.double()).float()
        ulp = torch.nextafter(x, torch.tensor(float("inf"))) - x
        x = torch.cat([x + i * ulp for i in range(-4, 5)])
        x = torch.cat([x, -x, torch.tensor([0.0, -0.0, float("inf"), -float("inf"), 1e-40, -1e-40, 3e38, float("nan")])])
        rows = -(-x.numel() // D)
        x = torch.cat([x, torch.zeros(rows * D - x.numel())]).view(rows, Hkv, D)
        assert rows <= 16 * 8
        pool = torch.zeros(8, 2, Hkv, PAGE, D, dtype=torch.uint8, device=cuda)
        sc = torch.stack([s, s]).view(2, 1).to(cuda)
        dd.append_kv_paged(cfg, pool, sc, _ints([0, rows], cuda), _ints([0, 8], cuda), _ints(list(range(8)), cuda),
                           _ints([rows], cuda), x.to(cuda), x.to(cuda))
        q = x / s
        want = torch.where(q.isnan(), torch.tensor(0x7F, dtype=torch.uint8), encode(x, "e4m3", s)[0])
        for which in (0, 1):
            got = pool[:, which].permute(0, 2, 1, 3).reshape(-1, Hkv, D)[:rows].cpu()
            ok = (got == want) | (q.isnan() & (got & 0x7F == 0x7F))
            assert ok.all(), (s.item(), x[~ok][:4], got[~ok][:4], want[~ok][:4])
