"""FP8 pages at head dims 64 and 256 through the plans, paged decode and the backend, against 64 bits."""
import numpy as np
import pytest
import torch

import dendrite_b200 as dd
from tests.test_gpu_window import Dev
from tests.window_ref import Batch, check_attention

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fmt", ["e4m3", "mxfp8"])
@pytest.mark.parametrize("shape", [(8, 2, 64, True), (32, 4, 64, False), (6, 3, 256, True)], ids=str)
@pytest.mark.parametrize("form", ["decode", "prefill", "flat"])
def test_plans(cuda, fmt, shape, form):
    tokens = [300, 77, 16, 1]
    new = [20, 5, 16, 1] if form == "prefill" else [1] * 4
    b = Batch(90, tokens, new, *shape[:3], fmt, shape[3], 0, 0, junk=None)
    d = Dev(b, cuda)
    if form == "flat":
        out, lse = dd.decode_paged(d.cfg, d.q, d.pool, d.indptr, d.ids, d.tokens, 19, d.scales)
    else:
        plan = dd.CascadePlan(d.cfg, b.indptr, np.array(b.ids), b.tokens) if form == "decode" else \
            dd.CascadePlan.prefill(d.cfg, b.indptr, np.array(b.ids), [n - m for n, m in zip(tokens, new)], new)
        out, lse = dd.cascade_decode(d.cfg, plan, d.q, d.pool, d.scales)
    # E4M3: code * scale is rounded to bf16, so V is off by 2^-8 and so, times reach, are the scores
    # (D 2^-24 2^10 >= 2^-8); MXFP8's code * 2^e is exact. The weights stay in f32.
    want, weights = b.attention(), 2.0 ** -14
    if fmt == "e4m3":
        weights, want = weights + 2.0 ** -8, (*want[:3], want[3] * 2.0 ** 10, want[4])
    got_lse = torch.tensor(want[1]) if fmt == "e4m3" else lse
    check_attention(out, got_lse, want, f"{fmt} {shape} {form}", weights)


@pytest.mark.parametrize("fmt", ["e4m3", "mxfp8"])
def test_backend(cuda, fmt):
    g = torch.Generator().manual_seed(91)
    be = dd.B200Backend(8, 2, 64, "bf16", cuda)
    rand = lambda h, n: torch.randn(1, h, n, 64, generator=g).to(cuda, torch.bfloat16)  # noqa: E731
    table = dd.BlockTable(blocks=[3, 1, 6], num_tokens=40)
    cfg = dd.AttentionConfig(8, 2, 64)
    q, k, v = rand(8, 40), rand(2, 40), rand(2, 40)
    be.prefill(q, k, v, table, cfg)
    be.quantize(fmt)
    out = be.decode(q[:, :, -1:], table, cfg)
    vals = dd.dequantize_kv_pages(*be._kv(), fmt, torch.bfloat16)[[3, 1, 6]].double()
    kk, vv = (vals[:, i].transpose(1, 2).reshape(48, 2, 64)[:40] for i in (0, 1))
    for h in range(8):
        w = torch.softmax(kk[:, h % 2] @ q[0, h, -1].double() / 8, 0)
        want, size = w @ vv[:, h % 2], w @ vv[:, h % 2].abs()
        assert ((out[0, h, 0].double() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -13 * size).all()
