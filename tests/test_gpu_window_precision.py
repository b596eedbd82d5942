"""What the sliding-window kernels hold: weights of 16 bits (E4M3 pages: 11) in every form."""
import pytest
import torch

from tests.test_gpu_window import Dev
from tests.window_ref import Batch, check_attention

pytestmark = pytest.mark.gpu

# (form, tokens, new): one token each; a few; chunks for the tcgen05 kernel; a chunk whose tiles are shared out.
FORMS = [("decode", [90, 300, 17, 700], [1] * 4), ("few", [90, 300, 17, 700], [3, 2, 5, 1]),
         ("many", [90, 300, 700], [33, 140, 260]), ("split", [2500], [130])]
FORM_IDS = [f[0] for f in FORMS]
# What a weight is off by: two bf16 terms, both cut off after 8 bits (what the first leaves is below
# 2^-7 of the weight, what the second leaves below 2^-7 of that); one f16 term, rounded.
WEIGHTS = {"bf16": 2.0 ** -14, "mxfp8": 2.0 ** -14, "e4m3": 2.0 ** -11}


def _run(b, form, dev, **kw):
    d = Dev(b, dev)
    return (d.decode if form == "decode" else d.prefill)(**kw)


SHAPES = [(8, 2, 128, True), (16, 2, 64, False), (6, 3, 256, True)]


@pytest.mark.parametrize("fmt", ["bf16", "e4m3"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("form,tokens,new", FORMS, ids=FORM_IDS)
@pytest.mark.parametrize("window,sinks", [(0, 0), (100, 4)])
def test_weights(cuda, fmt, shape, form, tokens, new, window, sinks):
    b = Batch(40 + window, tokens, new, *shape[:3], fmt, shape[3], window, sinks)
    out, lse = _run(b, form, cuda)
    check_attention(out, lse, b.attention(), f"{fmt} {shape} {form} {window}", WEIGHTS[fmt])


@pytest.mark.parametrize("fmt", ["bf16", "e4m3", "mxfp8"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("form,tokens,new", FORMS, ids=FORM_IDS)
@pytest.mark.parametrize("window", [0, 1])
def test_a_row_of_one_token_is_its_value(cuda, fmt, shape, form, tokens, new, window):
    """Its weight is 1: the output is V, bit for bit (V is exact in bf16: codes times powers of two)."""
    Hq, Hkv, D, grouped = shape
    tokens = tokens if window else new    # without a window the first row of a new sequence
    b = Batch(41, tokens, new, Hq, Hkv, D, fmt, grouped, window, 0)
    if fmt == "e4m3":
        b.scales = torch.exp2(torch.randint(-9, -3, (2, Hkv), generator=b.g).float())
    out, lse = _run(b, form, cuda)
    vals = torch.from_numpy(b.values()).to(torch.bfloat16)
    for s, (n, m) in enumerate(zip(tokens, new)):
        for i in range(m if window else 1):
            page, slot = b.place(s, n - m + i)
            v = vals[int(page), 1, :, int(slot)]
            want = v.repeat_interleave(Hq // Hkv, 0) if grouped else v.repeat(Hq // Hkv, 1)
            assert torch.equal(out[b.q_indptr[s] + i].cpu(), want), (s, i)
