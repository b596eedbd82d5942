"""A page that is not there: skipped on the device, and found by PagedKVCache.check()."""
import pytest
import torch

import dendrite_b200 as dd

pytestmark = pytest.mark.gpu

HQ, HKV, D = 8, 2, 128


@pytest.mark.parametrize("fmt", ["bf16", "mxfp8"])
@pytest.mark.parametrize("gone", [-1, 0, 300], ids=["-1", "the first behind the pool", "far behind it"])
@pytest.mark.parametrize("new", [3, 200])   # a few rows, and a chunk for the tcgen05 kernel
def test_a_page_given_back_too_early(cuda, fmt, gone, new):
    pages = -(-(20 + new) // 16)
    gone = gone if gone < 0 else pages + gone
    cache = dd.PagedKVCache(1, pages, HQ, HKV, D, kv_dtype=fmt, device=cuda, windows=[(40, 2)])
    table = list(range(pages))
    first_gone, second_gone = [gone] + table[1:], table[:1] + [gone] + table[2:]

    def qkv(n):
        x = torch.randn(n, HQ + 2 * HKV, D, device=cuda).to(torch.bfloat16)
        return x[:, :HQ], x[:, HQ:HQ + HKV], x[:, HQ + HKV:]

    def found():
        with pytest.raises(dd.InvalidArgument, match="outside the pool"):
            cache.check()
        cache.check()

    cache.begin_chunks([0, pages], table, [20], [20])
    cache.layer_chunk(0, *qkv(20))
    cache.check()
    cache.begin_chunks([0, pages], first_gone, [20 + new], [new])   # the page of the first tokens
    cache.layer_chunk(0, *qkv(new))
    found()
    cache.begin_step([0, pages], first_gone, [20])
    cache.layer_step(0, *qkv(1))
    found()
    cache.begin_step([0, pages], second_gone, [20])                 # the page that the token goes to
    cache.layer_step(0, *qkv(1))
    found()
    k, v = cache.read_tokens(0, [0, pages], first_gone, [14], [4])
    assert k[:2].eq(0).all() and v[:2].eq(0).all()
    found()
    cache.begin_step([0, pages], table, [20])
    cache.layer_step(0, *qkv(1))
    cache.read_tokens(0, [0, pages], table, [14], [4])
    cache.check()
