"""AttentionConfig.sliding_window through the backend's prefill and decode, against 64 bits over
the values that its pages hold."""
import numpy as np
import pytest
import torch

import dendrite_b200 as dd
from dendrite_b200._lib import GQA_GROUPED, GQA_TILED
from tests.window_ref import HALF, kv_head, visible

pytestmark = pytest.mark.gpu

HKV, D, P = 2, 128, 40


def _values(be):
    kv, sc = be._kv()
    if sc is None:
        return kv.double().cpu().numpy()
    return dd.dequantize_kv_pages(kv, sc, be.kv_dtype, torch.float32).double().cpu().numpy()


def _check(got, q, vals, table, positions, Hq, grouped, window, what):
    """Half a step of the output, and the weights' and scores' roundings against sum w |v|: 11 bits
    of a weight at worst (E4M3), and of a score D 2^-24 of |q| |k|."""
    ids = np.array(table.blocks())
    g, q = got.double().cpu().numpy(), q.double().cpu().numpy()
    for i, p in enumerate(positions):
        j = visible(p, window, 0)
        page, slot = ids[j // 16], j % 16
        for h in range(Hq):
            c = kv_head(h, Hq, HKV, grouped)
            k, v = vals[page, 0, c, slot], vals[page, 1, c, slot]
            x = k @ q[i, h] / np.sqrt(D)
            w = np.exp(x - x.max())
            w /= w.sum()
            reach = (np.abs(k) @ np.abs(q[i, h])).max() / np.sqrt(D)
            want, size = w @ v, w @ np.abs(v)
            tol = HALF[got.dtype] * np.abs(want) + (2.0 ** -11 + 2 * D * 2.0 ** -24 * reach + 2.0 ** -16) * size * 1.01
            assert np.all(np.abs(g[i, h] - want) <= tol), (what, i, h, np.max(np.abs(g[i, h] - want) / tol))


@pytest.mark.parametrize("fmt", ["f32", "bf16", "e4m3", "mxfp8"])
@pytest.mark.parametrize("grouped", [False, True], ids=["tiled", "grouped"])
@pytest.mark.parametrize("window", [1, 20, 1000, 2 ** 40])
def test_prefill_and_decode(cuda, fmt, grouped, window):
    Hq, dt = 8, torch.float32 if fmt == "f32" else torch.bfloat16
    g = torch.Generator().manual_seed(3)
    be = dd.B200Backend(P, HKV, D, "f32" if fmt == "f32" else "bf16", cuda, GQA_GROUPED if grouped else GQA_TILED)
    order = torch.randperm(P, generator=g).tolist()
    cfg = dd.AttentionConfig(Hq, HKV, D, sliding_window=window)

    def rand(heads, n):
        return torch.randn(1, heads, n, D, generator=g).to(cuda, dt)

    tables = [dd.BlockTable(blocks=order[:4]), dd.BlockTable(blocks=order[4:24])]
    for table, n in zip(tables, (37, 300)):
        table.set_num_tokens(n)
        q = rand(Hq, n)
        out = be.prefill(q, rand(HKV, n), rand(HKV, n), table, cfg)
        assert out.shape == q.shape and out.dtype == q.dtype
        _check(out[0].transpose(0, 1), q[0].transpose(0, 1), _values(be), table, range(n), Hq, grouped, window, "prefill")
    if fmt in ("e4m3", "mxfp8"):
        be.quantize(fmt)
        table = tables[0]
        table.add_tokens(11)             # a second chunk behind tokens that are there
        q = rand(Hq, 11)
        out = be.prefill(q, rand(HKV, 11), rand(HKV, 11), table, cfg)
        _check(out[0].transpose(0, 1), q[0].transpose(0, 1), _values(be), table, range(37, 48), Hq, grouped, window, "chunk")
    empty = dd.BlockTable()
    qs = [rand(Hq, 1) for _ in range(3)]
    outs = be.decode_batch(qs, [tables[0], empty, tables[1]], cfg)
    assert outs[1].eq(0).all()
    for out, q, table in ((outs[0], qs[0], tables[0]), (outs[2], qs[2], tables[1])):
        _check(out[0].transpose(0, 1), q[0].transpose(0, 1), _values(be), table, [table.num_tokens() - 1], Hq, grouped, window, "decode")
    one = be.decode(qs[2], tables[1], cfg)
    assert one.shape == qs[2].shape


def test_refusals(cuda):
    be = dd.B200Backend(P, HKV, D, "bf16", cuda)
    q, kv = torch.zeros(1, 4, 1, D, device=cuda), torch.ones(1, HKV, 1, D, device=cuda, dtype=torch.bfloat16)
    for bad in (0, -3):
        cfg = dd.AttentionConfig(4, HKV, D, sliding_window=bad)
        with pytest.raises(dd.InvalidArgument, match="sliding_window"):
            be.decode(q, dd.BlockTable(blocks=[1], num_tokens=1), cfg)
        with pytest.raises(dd.InvalidArgument, match="sliding_window"):
            be.prefill(q, kv, kv, dd.BlockTable(blocks=[1], num_tokens=1), cfg)
    assert be.pages.eq(0).all()          # nothing was stored before the refusal
    cfg = dd.AttentionConfig(4, HKV, D, sliding_window=8)
    for blocks, n in (([1], 17), ([], 1), ([P], 3), ([-1], 3)):
        with pytest.raises(dd.InvalidArgument):
            be.decode(q, dd.BlockTable(blocks=blocks, num_tokens=n), cfg)
        with pytest.raises(dd.InvalidArgument):
            be.prefill(q, kv, kv, dd.BlockTable(blocks=blocks, num_tokens=n), cfg)
    assert be.pages.eq(0).all()
    with pytest.raises(dd.InvalidArgument):
        be.decode_batch([q, q], [dd.BlockTable(blocks=[1], num_tokens=1)], cfg)
