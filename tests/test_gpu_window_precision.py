"""What the sliding-window kernels hold: weights of 16 bits (E4M3 pages: 11) in
every form, whatever the pages' exponents and the signs of their scales."""
import numpy as np
import pytest
import torch

from tests.test_gpu_window import Dev
from tests.test_gpu_window_chunk_kernel import WEIGHTS, chunk_kernel
from tests.window_ref import HALF, Batch, check_attention

pytestmark = pytest.mark.gpu

# (form, tokens, new): one token each; a few; chunks for the tcgen05 kernel; without a window, one whose tiles are shared out.
FORMS = [("decode", [90, 300, 17, 700], [1] * 4), ("few", [90, 300, 17, 700], [3, 2, 5, 1]),
         ("many", [90, 400, 1100], [33, 240, 900]), ("split", [9000], [900])]
FORM_IDS = [f[0] for f in FORMS]
def _run(b, form, dev, **kw):
    d = Dev(b, dev)
    if form == "decode":
        return d.decode(**kw)
    return chunk_kernel(d.prefill) if form in ("many", "split") and b.D <= 128 else d.prefill(**kw)


def _check(got, lse, want, weights, what):
    """check_attention's bound without its terms for tiny weights and for exponents: nothing
    but each token's own w |v| counts, and what f32 does not hold of a weight (2^-125)."""
    out, want_lse, size, reach, mass = want
    g, gl = got.cpu().double().numpy(), lse.cpu().double().numpy()
    score = out.shape[-1] * 2.0 ** -24 * reach
    assert np.isfinite(g).all(), f"{what}: not finite"
    assert np.all(np.abs(gl - want_lse) <= score + 2.0 ** -18 * (1 + np.abs(want_lse))), f"{what}: lse"
    tol = HALF[got.dtype] * np.abs(out) + (2 * score[..., None] + weights + 2.0 ** -16) * size * (1 + 2.0 ** -8) \
        + 2.0 ** -125 * mass
    err = np.abs(g - out)
    assert np.all(err <= tol), f"{what}: worst error / bound {np.max(err / tol):.2f}"


SHAPES = [(8, 2, 128, True), (16, 2, 64, False), (6, 3, 256, True)]


@pytest.mark.parametrize("fmt", ["bf16", "e4m3", "mxfp8"])
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


@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("form,tokens,new", FORMS, ids=FORM_IDS)
@pytest.mark.parametrize("up", [12, 24, 32, 60])
def test_mxfp8_one_large_value(cuda, shape, form, tokens, new, up):
    """V of some tokens is 2^up larger than the others': tokens of next to no weight (their scores are
    some 2^-(up + 8) of the others'), and in the chunk forms tokens that only later rows see."""
    Hq, Hkv, D, grouped = shape
    b = Batch(30 + up, tokens, new, Hq, Hkv, D, "mxfp8", grouped, 64, 4, junk=None)
    low = 0.7 * (up + 8) * D ** 0.5          # what the scores of the heavy tokens lose, before the scale
    b.q[..., 0] = 8.0
    heavy = [(s, j) for s, n in enumerate(tokens) for j in {0, max(n - 20, 0), n - 2} if n > 2]
    codes, exps = b.pool.view(torch.float8_e4m3fn).float(), b.scales.int()
    codes[:, 0, :, :, 0] = 0.0
    for s, j in heavy:
        page, slot = (int(x) for x in b.place(s, j))
        exps[page, 1, :, slot] += up
        exps[page, 0, :, slot, 0] = 127
        codes[page, 0, :, slot, :32] = 0.0
        codes[page, 0, :, slot, 0] = -low / 8.0
    b.pool, b.scales = codes.to(torch.float8_e4m3fn).view(torch.uint8), exps.to(torch.uint8)
    out, lse = _run(b, form, cuda)
    want = b.attention()
    # mass without the exponents' part: what a weight loses below f32's range, times |v|
    mass = np.full_like(want[0], np.abs(b.values()[:, 1]).max() * max(tokens))
    _check(out, lse, (*want[:4], mass), WEIGHTS["mxfp8"], f"{shape} {form} {up}")


@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("form,tokens,new", FORMS, ids=FORM_IDS)
def test_mxfp8_smallest_exponents(cuda, shape, form, tokens, new):
    """V around 2^-120, exponent bytes from 0 on. Below 2^-126, where f32 and bf16 have fewer bits, a
    value may be off by half of bf16's smallest step (2^-134 each), and so may the sums' roundings."""
    b = Batch(50, tokens, new, *shape[:3], "mxfp8", shape[3], 64, 4, junk=None)
    b.scales[:, 1] = torch.randint(0, 5, b.scales[:, 1].shape, generator=b.g).to(torch.uint8)
    out, lse = _run(b, form, cuda)
    want = b.attention()
    assert np.abs(want[0]).max() > 2.0 ** -121
    tol = 2.0 ** -8 * np.abs(want[0]) + 2.0 ** -10 * want[2] + 2.0 ** -132
    err = np.abs(out.cpu().double().numpy() - want[0])
    assert np.all(err <= tol), f"worst error / bound {np.max(err / tol):.2f}"


@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("form,tokens,new", FORMS, ids=FORM_IDS)
def test_mxfp8_nan_exponents(cuda, shape, form, tokens, new):
    """The NaN exponent of one block of V makes that block of its head NaN, in the rows that see the
    token, and no other block or head; one of K makes the rows of its head NaN."""
    Hq, Hkv, D, grouped = shape
    b = Batch(51, tokens, new, Hq, Hkv, D, "mxfp8", grouped, 0, 0, junk=None)
    page, slot = (int(x) for x in b.place(0, 3))
    b.scales[page, 1, 0, slot, 1] = 255
    out, lse = _run(b, form, cuda)
    heads = [h for h in range(Hq) if (h // (Hq // Hkv) if grouped else h % Hkv) == 0]
    rows = list(range(b.q_indptr[1]))
    bad = torch.zeros(out.shape, dtype=torch.bool)
    for h in heads:
        bad[rows, h, 32:64] = True
    assert torch.equal(out.isnan().cpu(), bad) and lse.isfinite().all()
    b.scales[page, 1, 0, slot, 1] = 127
    b.scales[page, 0, 0, slot, 1] = 255
    out, lse = _run(b, form, cuda)
    bad[:] = False
    for h in heads:
        bad[rows, h] = True
    assert torch.equal(out.isnan().cpu(), bad)
    assert torch.equal(lse.isnan().cpu(), bad[..., 0])


@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("form,tokens,new", FORMS, ids=FORM_IDS)
@pytest.mark.parametrize("window,sinks", [(0, 0), (100, 4)])
def test_e4m3_scales_of_either_sign(cuda, shape, form, tokens, new, window, sinks):
    b = Batch(60 + window, tokens, new, *shape[:3], "e4m3", shape[3], window, sinks)
    b.scales[0, ::2] *= -1
    b.scales[1, 1::2] *= -1
    out, lse = _run(b, form, cuda)
    check_attention(out, lse, b.attention(), f"{shape} {form} {window}", WEIGHTS["e4m3"])


@pytest.mark.parametrize("which", [0, 1], ids=["K", "V"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("form,tokens,new", FORMS + [("decode", [0, 20, 0], [1] * 3), ("many", [5, 0, 1000], [40, 7, 960])])
def test_e4m3_nan_scales(cuda, which, shape, form, tokens, new):
    """A NaN scale makes its head's rows NaN; rows that see nothing stay zeros, and other heads what they are."""
    Hq, Hkv, D, grouped = shape
    b = Batch(61, tokens, new, Hq, Hkv, D, "e4m3", grouped, 100, 4)
    good, good_lse = _run(b, form, cuda)
    b.scales[which, 0] = float("nan")
    out, lse = _run(b, form, cuda)
    sees = torch.tensor([n - m + i >= 0 for n, m in zip(tokens, new) for i in range(m)])
    bad = torch.zeros(out.shape[:2], dtype=torch.bool)
    for h in range(Hq):
        if (h // (Hq // Hkv) if grouped else h % Hkv) == 0:
            bad[:, h] = sees
    bad = bad.to(cuda)
    assert out[bad].isnan().all() and torch.equal(out[~bad], good[~bad])
    assert torch.equal(lse[~bad], good_lse[~bad])
    if which == 0:
        assert lse[bad].isnan().all()
    else:
        assert torch.equal(lse, good_lse)
