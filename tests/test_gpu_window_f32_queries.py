"""f32 queries over pools of every type: the CUDA-core form of the sliding-window calls."""
import pytest
import torch

from tests.test_gpu_window import Dev
from tests.window_ref import Batch, check_attention

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fmt", ["bf16", "e4m3", "mxfp8"])
@pytest.mark.parametrize("shape", [(8, 2, 64, False), (6, 3, 128, True), (4, 1, 256, True)], ids=str)
@pytest.mark.parametrize("form,new", [("decode", [1, 1, 1, 1]), ("prefill", [3, 40, 0, 130])], ids=["decode", "prefill"])
@pytest.mark.parametrize("window,sinks", [(0, 0), (33, 5)])
def test_f32_queries(cuda, fmt, shape, form, new, window, sinks):
    b = Batch(95, [3, 90, 17, 300], new, *shape[:3], fmt, shape[3], window, sinks)
    if fmt == "e4m3":
        b.scales[0, 0] *= -1
    d = Dev(b, cuda, torch.float32, strided=window > 0)
    out, lse = getattr(d, form)()
    assert out.dtype == torch.float32
    check_attention(out, lse, b.attention(), f"{fmt} {shape} {form}")
