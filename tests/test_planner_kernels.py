"""Which kernel the plans give work to, by head dim and types: only one that is built for them."""
import numpy as np
import pytest

import dendrite_b200 as dd
from dendrite_b200 import _lib

SIMPLE, MMA = 0, 1
KV = {"f32": _lib.DTYPE_F32, "bf16": _lib.DTYPE_BF16, "e4m3": _lib.DTYPE_E4M3, "mxfp8": _lib.DTYPE_MXFP8}
# Of the streaming tensor-core kernel: bf16 pages at head dims 64 and 128, FP8 pages at 128.
BUILT = {("bf16", 64), ("bf16", 128), ("e4m3", 128), ("mxfp8", 128)}


@pytest.mark.parametrize("q", [_lib.DTYPE_BF16, _lib.DTYPE_F32], ids=["bf16 q", "f32 q"])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("fmt", list(KV))
def test_kernel_of_a_plan(fmt, D, q):
    cfg = dd.make_config(8, 2, D, 64, kv_dtype=KV[fmt], q_dtype=q)
    table = np.arange(40, dtype=np.uint32)
    for plan in (dd.CascadePlan(cfg, [0, 20, 40], table, [300, 320]),
                 dd.CascadePlan.prefill(cfg, [0, 20, 40], table, [290, 0], [9, 20])):
        tokens = list(plan.info().kv_tokens_by_kernel)
        want = MMA if (fmt, D) in BUILT and q == _lib.DTYPE_BF16 else SIMPLE
        assert tokens[want] > 0 and sum(tokens) == tokens[want], tokens
