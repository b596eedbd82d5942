"""Refusals of the sliding-window operators, and their reference against a
second formulation (no GPU)."""
import ctypes as C

import numpy as np
import pytest
import torch

import dendrite_b200 as dd
from dendrite_b200 import _lib
from tests.window_ref import Batch, encode, visible

HQ, HKV, D, P = 8, 2, 64, 4
FAKE = 1 << 20  # never dereferenced: every refusal comes before a launch


def _args(**kw):
    cfg = dd.make_config(HQ, HKV, D, P, kv_dtype=kw.pop("kv_dtype", _lib.DTYPE_BF16))
    a = dict(q=torch.zeros(3, HQ, D, dtype=torch.bfloat16),
             kv_pages=torch.zeros(P, 2, HKV, 16, D, dtype=torch.bfloat16),
             q_indptr=torch.tensor([0, 1, 3], dtype=torch.int32), page_indptr=torch.tensor([0, 1, 2, 3], dtype=torch.int32),
             page_indices=torch.zeros(3, dtype=torch.int32), num_tokens=torch.ones(3, dtype=torch.int32),
             window=4, sinks=1)
    a.update(kw)
    return cfg, a


BAD = [
    (dict(q=torch.zeros(3, HQ, D)), "q_dtype"),
    (dict(q=torch.zeros(3, HQ, D + 64, dtype=torch.bfloat16)), "dense rows"),
    (dict(q=torch.zeros(3, HQ, 2 * D, dtype=torch.bfloat16)[:, :, ::2]), "dense rows"),
    (dict(q=torch.zeros(HQ, 3, D, dtype=torch.bfloat16).transpose(0, 1)), "dense rows"),
    (dict(kv_pages=torch.zeros(P, 2, HKV, 16, D)), "kv_pages"),
    (dict(kv_pages=torch.zeros(P - 1, 2, HKV, 16, D, dtype=torch.bfloat16)), "kv_pages"),
    (dict(kv_pages=torch.zeros(P, 2, 16, HKV, D, dtype=torch.bfloat16).transpose(2, 3)), "kv_pages"),
    (dict(page_indptr=torch.zeros(2, dtype=torch.int32)), "page_indptr"),
    (dict(page_indptr=torch.zeros(4, dtype=torch.int64)), "page_indptr"),
    (dict(page_indices=torch.zeros(6, dtype=torch.int32)[::2]), "page_indices"),
    (dict(num_tokens=torch.zeros(1, dtype=torch.int32)), "num_tokens"),
    (dict(num_tokens=torch.zeros(3)), "num_tokens"),
    (dict(out=torch.zeros(3, HQ, D)), "out"),
    (dict(out=torch.zeros(2, HQ, D, dtype=torch.bfloat16)), "out"),
    (dict(lse=torch.zeros(3, HQ, dtype=torch.float64)), "lse"),
    (dict(status=torch.zeros(1, dtype=torch.int32)), "status"),
    (dict(), "CUDA device"),
]


@pytest.mark.parametrize("bad,msg", BAD, ids=lambda x: x if isinstance(x, str) else None)
def test_attention_refusals(bad, msg):
    cfg, a = _args(**bad)
    with pytest.raises(dd.InvalidArgument, match=msg):
        dd.prefill_paged_window(cfg, **a)
    a.pop("q_indptr")
    with pytest.raises(dd.InvalidArgument, match=msg):
        dd.decode_paged_window(cfg, **a)


def test_prefill_needs_its_rows():
    cfg, a = _args(q_indptr=None)
    with pytest.raises(dd.InvalidArgument, match="q_indptr"):
        dd.prefill_paged_window(cfg, **a)
    cfg, a = _args(q_indptr=torch.zeros(0, dtype=torch.int32))
    with pytest.raises(dd.InvalidArgument, match="q_indptr"):
        dd.prefill_paged_window(cfg, **a)


@pytest.mark.parametrize("kvd,good", [
    (_lib.DTYPE_E4M3, torch.zeros(2, HKV)), (_lib.DTYPE_MXFP8, torch.zeros(P, 2, HKV, 16, D // 32, dtype=torch.uint8))])
def test_fp8_pools_need_their_scales(kvd, good):
    pool = torch.zeros(P, 2, HKV, 16, D, dtype=torch.uint8)
    for bad in (None, good[:1], good.double()):
        cfg, a = _args(kv_dtype=kvd, kv_pages=pool, kv_scales=bad)
        with pytest.raises(dd.InvalidArgument, match="kv_scales"):
            dd.prefill_paged_window(cfg, **a)
    cfg, a = _args(kv_dtype=kvd, kv_pages=pool, kv_scales=good)
    with pytest.raises(dd.InvalidArgument, match="CUDA device"):
        dd.prefill_paged_window(cfg, **a)


def _c_attend(form="prefill", **kw):
    a = dict(cfg=dd.make_config(HQ, HKV, D, P), seqs=2, rows=3, max_pages=0, window=4, sinks=1, q=FAKE,
             q_stride=HQ * D, kv=FAKE, scales=None, q_indptr=FAKE, page_indptr=FAKE, page_indices=FAKE,
             num_tokens=FAKE, out=FAKE)
    a.update(kw)
    head = (C.byref(a["cfg"]) if a["cfg"] is not None else None, a["seqs"])
    rest = (a["max_pages"], a["window"], a["sinks"], a["q"], a["q_stride"], a["kv"], a["scales"])
    tables = (a["page_indptr"], a["page_indices"], a["num_tokens"], a["out"], None, None, None)
    if form == "decode":
        return _lib.lib.dd_decode_paged_window(*head, *rest, *tables)
    return _lib.lib.dd_prefill_paged_window(*head, a["rows"], *rest, a["q_indptr"], *tables)


@pytest.mark.parametrize("form", ["decode", "prefill"])
@pytest.mark.parametrize("kw,rc", [
    (dict(cfg=None), 1), (dict(cfg=dd.make_config(8, 3, 64, 4)), 1), (dict(cfg=dd.make_config(8, 2, 96, 4)), 1),
    (dict(cfg=dd.make_config(8, 2, 64, 4, kv_dtype=_lib.DTYPE_F16)), 3),
    (dict(cfg=dd.make_config(8, 2, 64, 4, kv_dtype=_lib.DTYPE_E4M3)), 1),
    (dict(cfg=dd.make_config(8, 2, 64, 4, kv_dtype=_lib.DTYPE_MXFP8), scales=FAKE + 4), 1),
    (dict(seqs=-1), 1), (dict(window=-1), 1), (dict(sinks=-1), 1), (dict(max_pages=-1), 1),
    (dict(q=None), 1), (dict(out=None), 1), (dict(kv=None), 1), (dict(page_indptr=None), 1), (dict(num_tokens=None), 1),
    (dict(q=FAKE + 2), 1), (dict(out=FAKE + 8), 1), (dict(kv=FAKE + 1), 1),
    (dict(q_stride=HQ * D - 8), 1), (dict(q_stride=HQ * D + 1), 1), (dict(q_stride=0), 1), (dict(q_stride=-4096), 1),
    (dict(seqs=0), 0),
])
def test_c_refusals(form, kw, rc):
    assert _c_attend(form, **kw) == rc
    if rc:
        assert _lib.lib.dd_last_error()


def test_c_refusals_of_the_chunk_form():
    assert _c_attend(rows=-1) == 1
    assert _c_attend(q_indptr=None) == 1
    assert _c_attend(rows=0, q_indptr=None) == 0


def _c_append(**kw):
    a = dict(cfg=dd.make_config(HQ, HKV, D, P), kv=FAKE, scales=None, seqs=2, rows=3, indptr=FAKE, page_indptr=FAKE,
             ids=FAKE, tokens=FAKE, k=FAKE, ks=HKV * D, v=FAKE, vs=HKV * D, src=_lib.DTYPE_BF16)
    a.update(kw)
    return _lib.lib.dd_append_kv_paged(C.byref(a["cfg"]), a["kv"], a["scales"], a["seqs"], a["rows"], a["indptr"],
                                       a["page_indptr"], a["ids"], a["tokens"], a["k"], a["ks"], a["v"], a["vs"],
                                       a["src"], None, None)


def _c_gather(**kw):
    a = dict(cfg=dd.make_config(HQ, HKV, D, P), kv=FAKE, scales=None, seqs=2, rows=3, indptr=FAKE, page_indptr=FAKE,
             ids=FAKE, tokens=FAKE, k=FAKE, v=FAKE, src=_lib.DTYPE_BF16)
    a.update(kw)
    return _lib.lib.dd_gather_kv_paged(C.byref(a["cfg"]), a["kv"], a["scales"], a["seqs"], a["rows"], a["indptr"],
                                       a["tokens"], a["page_indptr"], a["ids"], a["k"], a["v"], a["src"], None, None)


@pytest.mark.parametrize("kw,rc", [
    (dict(kv=None), 1), (dict(k=None), 1), (dict(v=None), 1), (dict(page_indptr=None), 1), (dict(seqs=-1), 1),
    (dict(rows=-1), 1), (dict(src=_lib.DTYPE_E4M3), 1), (dict(src=_lib.DTYPE_F16), 1), (dict(k=FAKE + 2), 1),
    (dict(kv=FAKE + 8), 1), (dict(cfg=dd.make_config(8, 2, 64, 4, kv_dtype=_lib.DTYPE_MXFP8)), 1),
    (dict(cfg=dd.make_config(8, 2, 64, 4, kv_dtype=_lib.DTYPE_E4M3), scales=FAKE + 2), 1), (dict(seqs=0), 0),
    (dict(rows=0), 0)])
def test_c_refusals_of_append_and_gather(kw, rc):
    assert _c_append(**kw) == rc
    assert _c_gather(**kw) == rc


def test_c_refusals_of_append():
    assert _c_append(tokens=None) == 1
    assert _c_append(indptr=None) == 1          # 3 rows, 2 sequences
    assert _c_append(ks=HKV * D - 8) == 1 and _c_append(vs=HKV * D + 4) == 1
    assert _c_gather(indptr=None) == 1


def test_append_gather_refusals():
    cfg = dd.make_config(HQ, HKV, D, P)
    pool = torch.zeros(P, 2, HKV, 16, D, dtype=torch.bfloat16)
    ip = torch.tensor([0, 1], dtype=torch.int32)
    one = torch.ones(1, dtype=torch.int32)
    k = torch.zeros(1, HKV, D, dtype=torch.bfloat16)
    for bad in (dict(k=k.float()), dict(k=k.half(), v=k.half()), dict(v=torch.zeros(2, HKV, D, dtype=torch.bfloat16)),
                dict(k=torch.zeros(1, HQ, D, dtype=torch.bfloat16)), dict(num_tokens=one.long()),
                dict(new_indptr=ip.float()), dict(kv_pages=pool[:2]), dict()):
        a = dict(kv_pages=pool, kv_scales=None, new_indptr=ip, page_indptr=ip, page_indices=one, num_tokens=one, k=k, v=k)
        a.update(bad)
        with pytest.raises(dd.InvalidArgument):
            dd.append_kv_paged(cfg, **a)
    for bad in (dict(out_dtype=torch.float16), dict(num_rows=-1), dict(first_token=one.long()), dict(k=k[:, :1]), dict()):
        a = dict(kv_pages=pool, kv_scales=None, out_indptr=ip, first_token=None, page_indptr=ip, page_indices=one, num_rows=1)
        a.update(bad)
        with pytest.raises(dd.InvalidArgument):
            dd.gather_kv_paged(cfg, **a)


# -------------------------------------------------------------- the reference
@pytest.mark.parametrize("fmt", ["f32", "bf16", "e4m3", "mxfp8"])
@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 0), (7, 3), (40, 16)])
def test_reference_against_a_loop(fmt, window, sinks):
    b = Batch(1, [5, 33, 0, 50], [5, 3, 2, 1], 4, 2, 64, fmt, False, window, sinks)
    out, lse, _, _, _ = b.attention()
    vals, row = b.values(), 0
    for s, (n, m) in enumerate(zip(b.tokens, b.new)):
        for i in range(m):
            for h in range(4):
                tot, acc = 0.0, np.zeros(64)
                for j in visible(n - m + i, window, sinks):
                    page, slot = b.place(s, j)
                    k, v = vals[page, 0, h % 2, slot], vals[page, 1, h % 2, slot]
                    w = np.exp(float(b.q[row, h].double().numpy() @ k) / 8.0)
                    tot, acc = tot + w, acc + w * v
                if tot:
                    assert np.allclose(acc / tot, out[row, h], rtol=1e-9, atol=1e-12)
                    assert np.isclose(np.log(tot), lse[row, h], rtol=1e-10, atol=1e-12)
                else:
                    assert np.isneginf(lse[row, h]) and not out[row, h].any()
            row += 1


def test_reference_codes_match_the_oracle():
    import oracle

    x = torch.randn(6, 4, 64, generator=torch.Generator().manual_seed(2)) * 5
    x[0] = 0
    x[1] *= 1e-30
    c, e = encode(x, "mxfp8")
    oc, oe = oracle.quantize_mx(x.numpy().reshape(24, 1, 1, 1, 64))
    assert np.array_equal(c.numpy().reshape(-1), oc.reshape(-1)) and np.array_equal(e.numpy().reshape(-1), oe.reshape(-1))
    c, _ = encode(x, "e4m3", torch.tensor(0.017))
    assert np.array_equal(c.numpy(), oracle.e4m3_encode(x.numpy() / np.float32(0.017)))


def test_paged_cache_refusals():
    with pytest.raises(dd.InvalidArgument, match="windows"):
        dd.PagedKVCache(2, 4, HQ, HKV, D, device="cpu", windows=[(4, 0)])
    for bad in ((0, 1), (4, -1), (4,)):
        with pytest.raises(dd.InvalidArgument, match="windows"):
            dd.PagedKVCache(1, 4, HQ, HKV, D, device="cpu", windows=[bad])
    cache = dd.PagedKVCache(1, 4, HQ, HKV, D, device="cpu", windows=[(4, 1)])
    k = torch.zeros(1, HKV, D, dtype=torch.bfloat16)
    with pytest.raises(dd.InvalidArgument, match="begin_chunks"):
        cache.layer_chunk(0, torch.zeros(1, HQ, D, dtype=torch.bfloat16), k, k)
    for args in (([0, 1], [0], [17], [1]), ([0, 1], [0], [3], [4]), ([0, 1], [0], [3, 3], [1, 1]), ([0, 2], [0], [3], [1]),
                 ([0, 1], [0], [3], [-1])):
        with pytest.raises(dd.InvalidArgument, match="fit together"):
            cache.begin_chunks(*args)
    for args in (([0, 1], [0], [10], [7]), ([0, 1], [0], [-1], [1]), ([0, 1], [0], [0], [-1]), ([0, 2], [0], [0], [1])):
        with pytest.raises(dd.InvalidArgument, match="fit together"):
            cache.read_tokens(0, *args)


@pytest.mark.parametrize("kw", [dict(window=1 << 31), dict(window=1 << 32), dict(window=-1), dict(sinks=1 << 32),
                                dict(sinks=-1), dict(max_pages=1 << 32), dict(max_pages=-1)], ids=str)
def test_sizes_that_32_bits_do_not_hold(kw):
    cfg, a = _args(**kw)
    with pytest.raises(dd.InvalidArgument, match="2.31"):
        dd.prefill_paged_window(cfg, **a)
    a.pop("q_indptr")
    with pytest.raises(dd.InvalidArgument, match="2.31"):
        dd.decode_paged_window(cfg, **a)


def test_paged_cache_tables_that_reach_outside():
    cache = dd.PagedKVCache(1, 4, HQ, HKV, D, device="cpu", windows=[(4, 1)])
    for indptr in ([-1, 0], [0, 2, 1], [0, 1, 3]):
        n = len(indptr) - 1
        with pytest.raises(dd.InvalidArgument, match="fit together"):
            cache.begin_chunks(indptr, [0, 1], [0] * n, [0] * n)
        with pytest.raises(dd.InvalidArgument, match="fit together"):
            cache.read_tokens(0, indptr, [0, 1], [0] * n, [0] * n)


def test_paged_cache_chunks_need_their_rows():
    cache = dd.PagedKVCache(1, 4, HQ, HKV, D, device="cpu", windows=[(4, 1)])
    cache.begin_chunks([0, 1], [0], [5], [5])
    def rows(n, heads):
        return torch.zeros(n, heads, D, dtype=torch.bfloat16)
    for nq, nk in ((4, 4), (5, 4), (4, 5), (6, 5)):
        with pytest.raises(dd.InvalidArgument, match="5 rows"):
            cache.layer_chunk(0, rows(nq, HQ), rows(nk, HKV), rows(nk, HKV))
