"""PagedKVCache takes q, k and v as a model leaves them: parts of one projection, heads before rows,
odd alignment; windowed and full layers alike, with the results of dense tensors."""
import pytest
import torch

import dendrite_b200 as dd

pytestmark = pytest.mark.gpu

HQ, HKV, D = 8, 2, 64


def _dense(x):
    return x


def _heads_first(x):
    return x.transpose(0, 1).contiguous().transpose(0, 1)


def _shifted(x):
    y = torch.empty(x.numel() + 1, dtype=x.dtype, device=x.device)[1:].view(x.shape)
    return y.copy_(x)


def _odd_rows(x):
    y = torch.empty(x.shape[0], x.shape[1] * D + 3, dtype=x.dtype, device=x.device)[:, :x.shape[1] * D]
    y.copy_(x.flatten(1))
    return y.unflatten(1, (x.shape[1], D))


def _wide_rows(x):
    y = torch.empty(x.shape[0], x.shape[1] + 5, D, dtype=x.dtype, device=x.device)[:, 2:2 + x.shape[1]]
    return y.copy_(x)


def _one_row_for_all(x):
    return x[:1].expand(x.shape)


@pytest.mark.parametrize("fmt", ["bf16", "mxfp8"])
@pytest.mark.parametrize("window", [None, (24, 3)], ids=["full", "windowed"])
@pytest.mark.parametrize("src", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("lay", [_heads_first, _shifted, _odd_rows, _wide_rows, _one_row_for_all])
def test_layouts(cuda, fmt, window, src, lay):
    g = torch.Generator().manual_seed(1)

    def run(lay):
        g.manual_seed(2)
        cache = dd.PagedKVCache(1, 16, HQ, HKV, D, kv_dtype=fmt, device=cuda, windows=[window])

        def qkv(n):
            return [lay(x) for x in torch.randn(n, HQ + 2 * HKV, D, generator=g).to(cuda, src)
                    .split([HQ, HKV, HKV], 1)]

        outs = [cache.layer_prefill(0, *qkv(37), [4, 2, 9], 0)]
        if window:
            cache.begin_chunks([0, 3, 6], [4, 2, 9, 1, 5, 7], [40, 33], [3, 33])
            outs.append(cache.layer_chunk(0, *qkv(36)))
        for n in (40, 41):
            cache.begin_step([0, 3, 6], [4, 2, 9, 1, 5, 7], [n, n - 7])
            outs.append(cache.layer_step(0, *qkv(2)))
        cache.begin_step([0, 3], [4, 2, 9], [42])
        outs.append(cache.layer_step(0, *qkv(1)))
        cache.check()
        return outs, cache

    if lay is _one_row_for_all:
        want, a = run(lambda x: lay(x).contiguous())
    else:
        want, a = run(lambda x: x.contiguous())
    got, b = run(lay)
    for x, y in zip(got, want):
        assert torch.equal(x, y)
    assert torch.equal(a.pools[0], b.pools[0])
