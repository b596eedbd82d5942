"""PagedKVCache's own checks and bookkeeping, without a GPU (no kernel runs)."""
import numpy as np
import pytest
import torch

import dendrite_b200 as dd

HQ, HKV, D, P = 4, 2, 64, 8


def _cache(windows):
    return dd.PagedKVCache(len(windows), P, HQ, HKV, D, device="cpu", windows=windows)


@pytest.mark.parametrize("windows", [[None], [(20, 2)], [(20, 2), None]], ids=["full", "windowed", "both"])
@pytest.mark.parametrize("indptr,ids,positions", [
    ([0, 1, 2], [3, 5], [16, 0]),            # past the first table: the place is the second sequence's
    ([0, 1, 2], [3, 5], [0, 16]),            # past the last one
    ([0, 1, 2], [3, 5], [0, -1]),            # before the first token
    ([0, 1, 2], [3, 5], [0, 2 ** 32]),       # a position that 32 bits would cut off to 0
    ([0, 0, 1], [3], [0, 0]),                # a sequence without a page
    ([0, 1, 2], [3, 5], [0]),                # fewer positions than tables
    ([0, 1, 3], [3, 5], [0, 20]),            # tables past the ids
    ([0, 2, 1], [3, 5], [0, 0]),
    ([-1, 1, 2], [3, 5], [0, 0]),
    ([], [], []),
], ids=str)
def test_a_step_outside_its_tables_is_refused(windows, indptr, ids, positions):
    with pytest.raises(dd.InvalidArgument, match="fit together"):
        _cache(windows).begin_step(np.array(indptr, np.int32), np.array(ids, np.uint32), positions)


def test_a_step_stores_at_its_positions():
    cache = _cache([(20, 2)])
    assert cache.begin_step([0, 2, 2 + 1], [3, 5, 1], [17, 15]) is False
    assert cache._page_ids.tolist() == [5, 1] and cache._slots.tolist() == [1, 15]
    ip, ids, ntok, longest = cache._step
    assert (ip.tolist(), ids.tolist(), ntok.tolist(), longest) == ([0, 2, 3], [3, 5, 1], [18, 16], 2)


@pytest.mark.parametrize("ids", [[-1, 4], np.array([-1, 4]), np.array([-1, 4], np.int32),
                                 np.array([2 ** 32 - 1, 4], np.uint32)], ids=["list", "int64", "int32", "uint32"])
def test_a_step_over_pages_given_back(ids):
    """A table entry of a page that no window reaches any more may be -1, in whatever type the ids come."""
    cache = _cache([(4, 0)])
    cache.begin_step([0, 2], ids, [30])
    assert cache._page_ids.tolist() == [4] and cache._slots.tolist() == [14]
    assert cache._step[1].tolist() == [-1, 4]


def test_a_refused_step_leaves_the_last_one(monkeypatch):
    """When the plan refuses a step, nothing of it stays: the pages that the layers write, the tables
    that windowed layers read and the plan are those of the last step, and the next one goes on from it."""
    uploads = []
    monkeypatch.setattr(dd.CascadePlan, "upload", lambda plan, device=None, stream=None: uploads.append(plan.batch_size))
    cache = _cache([(20, 2), None])
    cache.begin_step([0, 1, 2], [3, 5], [4, 7])
    nodes = {k: v.tolist() for k, v in cache.plan.nodes().items()}
    with pytest.raises(dd.InvalidArgument):
        cache.begin_step([0, 1], [P + 92], [9])         # no such page
    assert cache._page_ids.tolist() == [3, 5] and cache._slots.tolist() == [4, 7]
    assert cache._step[1].tolist() == [3, 5] and cache._step[2].tolist() == [5, 8]
    assert cache.plan.batch_size == 2 and {k: v.tolist() for k, v in cache.plan.nodes().items()} == nodes
    assert cache.begin_step([0, 1, 2], [3, 5], [5, 8]) is True
    assert uploads == [2, 2, 2]
    cache = _cache([(20, 2), None])
    with pytest.raises(dd.InvalidArgument):
        cache.begin_step([0, 1], [P + 92], [9])
    assert cache.plan is None and cache._step is None and cache._page_ids is None


def _rows(n, heads):
    return torch.zeros(n, heads, D, dtype=torch.bfloat16)


@pytest.mark.parametrize("windows", [[None], [(20, 2)]], ids=["full", "windowed"])
@pytest.mark.parametrize("nq,nk,nv", [(2, 3, 3), (3, 2, 2), (2, 2, 1), (2, 1, 2), (3, 3, 3), (1, 1, 1)], ids=str)
def test_rows_that_are_not_the_steps(monkeypatch, windows, nq, nk, nv):
    """The append reads a page and a slot for each row of K: more rows than the step has would read past them."""
    monkeypatch.setattr(dd.CascadePlan, "upload", lambda plan, device=None, stream=None: None)
    cache = _cache(windows)
    with pytest.raises(dd.InvalidArgument, match="begin_step"):
        cache.layer_step(0, _rows(2, HQ), _rows(2, HKV), _rows(2, HKV))
    cache.begin_step([0, 1, 2], [3, 5], [4, 7])
    with pytest.raises(dd.InvalidArgument, match="2 rows"):
        cache.layer_step(0, _rows(nq, HQ), _rows(nk, HKV), _rows(nv, HKV))


@pytest.mark.parametrize("windows", [[None], [(20, 2)]], ids=["full", "windowed"])
@pytest.mark.parametrize("nk,nv", [(3, 3), (1, 1), (2, 1), (1, 2)], ids=str)
def test_rows_that_are_not_the_prompts(windows, nk, nv):
    with pytest.raises(dd.InvalidArgument, match="2 rows"):
        _cache(windows).layer_prefill(0, _rows(2, HQ), _rows(nk, HKV), _rows(nv, HKV), [3], 4)


@pytest.mark.parametrize("windows", [[None], [(20, 2)]], ids=["full", "windowed"])
@pytest.mark.parametrize("table,prefix", [([3], 15), ([3], -1), ([], 0)], ids=str)
def test_a_prompt_outside_its_table(windows, table, prefix):
    """Position -1 would be the last slot of the table's last page."""
    with pytest.raises(dd.InvalidArgument, match="fit together"):
        _cache(windows).layer_prefill(0, _rows(2, HQ), _rows(2, HKV), _rows(2, HKV), table, prefix)


def test_check_raises_once():
    cache = _cache([(20, 2)])
    cache.check()
    for status, error in (([1, -2], dd.InvalidArgument), ([2, 0], dd.CudaError)):
        cache._status[:] = torch.tensor(status, dtype=torch.int32)
        with pytest.raises(error):
            cache.check()
        cache.check()


def test_every_call_reports_to_the_cache(monkeypatch):
    import dendrite_b200.paged_cache as pc

    cache, seen = _cache([(20, 2), None]), []

    def call(name, result):
        def fake(*args, status=None, **kw):
            assert status is cache._status, name
            seen.append(name)
            return result
        monkeypatch.setattr(pc, name, fake)

    out = _rows(1, HQ)
    for name, result in (("append_kv_batch", None), ("append_kv_paged", None), ("decode_paged_window", (out, None)),
                         ("prefill_paged_window", (out, None)), ("gather_kv_paged", (out, out))):
        call(name, result)
    monkeypatch.setattr(pc, "cascade_decode", lambda *args, **kw: (out, None))
    monkeypatch.setattr(dd.CascadePlan, "upload", lambda plan, device=None, stream=None: None)
    qkv = (_rows(1, HQ), _rows(1, HKV), _rows(1, HKV))
    cache.begin_step([0, 1], [3], [4])
    cache.begin_chunks([0, 1], [3], [6], [1])
    for layer in (0, 1):
        cache.layer_step(layer, *qkv)
        cache.layer_chunk(layer, *qkv)
        cache.layer_prefill(layer, *qkv, [3], 6)
        cache.read_tokens(layer, [0, 1], [3], [0], [7])
    assert sorted(set(seen)) == ["append_kv_batch", "append_kv_paged", "decode_paged_window", "gather_kv_paged",
                                 "prefill_paged_window"] and len(seen) == 7 + 5
