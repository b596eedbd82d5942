"""Paged KV cache for a model's decode loop: the attention step of
TransformerLayer::forward_with_cache
(crates/dendrite-core/src/model/layer.rs:374-416) over a page pool per layer
instead of the contiguous LayerCache, with one cascade plan per step for all
layers.

forward_with_cache appends the step's RoPE'd K/V to the layer's cache
(`cache.append`, :392-393) and attends with `compute_attention` (:276-318):
scale 1/sqrt(head_dim), GQA by `repeat_kv` (:321-340), an unsqueeze-expand-
reshape that gives query head h the KV head h // (Hq / Hkv) (the grouped
map). Here a step of B sequences (the leaves of a tree) is:

* ``begin_step(tables, positions)``: the sequences' block tables (CSR) and
  the position of each one's new token. The plan is advanced in place when
  every sequence only grew by that token (``CascadePlan.advance``, a new block
  read from its table when the token starts one) and re-planned otherwise
  (first step, a fork, a copy-on-write); it is uploaded once for all layers.
* ``layer_step(layer, q, k, v)``: stores the new token's K/V of that layer
  into its pool at (table[pos // 16], pos % 16) — quantised for FP8 pools —
  and runs the cascade decode of q [B, Hq, D] over the pool with the shared
  plan; returns the attention output [B, Hq, D] (what compute_attention
  returns before the output projection).

Prompts go in through ``layer_prefill`` (the causal prefill plan of the new
tokens over their sequence, ReferenceBackend::prefill's attention when the
sequence starts empty).

Layers whose tokens attend to a sliding window and a few first tokens are named
in ``windows`` (``(window, sinks)`` per layer, None for full attention); they
run without a plan, on device copies of the tables that ``begin_step`` makes,
and never read the table entries of pages that no window reaches any more.

A ragged batch of chunks (several sequences, any number of new tokens each,
prompts in flight or tokens to be checked) goes in through

* ``begin_chunks(tables, num_tokens, new_tokens)``: the batch, once for all
  layers;
* ``layer_chunk(layer, q, k, v)``: stores the layer's new K/V (quantised for
  FP8 pools) and returns the causal attention, windowed or full;

and ``read_tokens`` takes token ranges back out, dequantised.

A page id that is not in the pool stops no kernel: it is skipped and noted on
the device, and ``check()`` raises for it (after a step, or every few).
"""
from __future__ import annotations

import numpy as np
import torch

from . import _lib
from .backend import (PAGE_SIZE, CascadePlan, _alloc_ws, append_kv_batch, cascade_decode,
                      make_config)
from .paged_window import (append_kv_paged, decode_paged_window, gather_kv_paged,
                           prefill_paged_window)

_KV = {"bf16": _lib.DTYPE_BF16, "e4m3": _lib.DTYPE_E4M3, "mxfp8": _lib.DTYPE_MXFP8}


def _rows_in_place(t: torch.Tensor) -> torch.Tensor:
    """[rows, heads, dim] as the window kernels take it: itself where its heads are dense and its rows
    lie on 16 bytes (part of a wider projection), else a dense copy."""
    width = t.shape[1] * t.shape[2]
    if t.data_ptr() % 16 == 0 and t.stride(2) == 1 and (t.shape[1] == 1 or t.stride(1) == t.shape[2]) and \
            (t.shape[0] <= 1 or (t.stride(0) >= width and t.stride(0) * t.element_size() % 16 == 0)):
        return t
    return t.clone(memory_format=torch.contiguous_format)


class PagedKVCache:
    """Page pools of `num_layers` layers ([num_pages][2][Hkv][16][D] each) and
    the step's cascade plan, shared by the layers."""

    def __init__(self, num_layers: int, num_pages: int, num_heads: int, num_kv_heads: int,
                 head_dim: int, kv_dtype: str = "bf16", e4m3_scales=None,
                 device: str | torch.device = "cuda", windows=None):
        if kv_dtype not in _KV:
            raise _lib.InvalidArgument("kv_dtype must be bf16, e4m3 or mxfp8")
        self.windows = [None] * num_layers if windows is None else list(windows)
        if len(self.windows) != num_layers or any(
                w is not None and (len(w) != 2 or w[0] < 1 or w[1] < 0) for w in self.windows):
            raise _lib.InvalidArgument("windows must be one (window >= 1, sinks >= 0) or None per layer")
        self.device = torch.device(device)
        self.Hq, self.Hkv, self.D, self.num_pages = num_heads, num_kv_heads, head_dim, num_pages
        self.kv_dtype = kv_dtype
        self.cfg = make_config(num_heads, num_kv_heads, head_dim, num_pages, kv_dtype=_KV[kv_dtype],
                               gqa_map=_lib.GQA_GROUPED)
        shape = (num_pages, 2, num_kv_heads, PAGE_SIZE, head_dim)
        if kv_dtype == "bf16":
            self.pools = [torch.zeros(shape, dtype=torch.bfloat16, device=self.device)
                          for _ in range(num_layers)]
            self.scales = [None] * num_layers
        else:
            self.pools = [torch.zeros(shape, dtype=torch.uint8, device=self.device)
                          for _ in range(num_layers)]
            if kv_dtype == "mxfp8":
                self.scales = [torch.zeros(shape[:-1] + (head_dim // 32,), dtype=torch.uint8,
                                           device=self.device) for _ in range(num_layers)]
            else:
                if e4m3_scales is None:
                    raise _lib.InvalidArgument("per-head E4M3 pages need e4m3_scales ([2][Hkv] per layer)")
                self.scales = [torch.as_tensor(s, dtype=torch.float32).reshape(2, num_kv_heads)
                               .contiguous().to(self.device) for s in e4m3_scales]
        self.plan: CascadePlan | None = None
        self._ntok = None
        self._tables = None
        self._ws: dict = {}
        self._page_ids = self._slots = None
        self._step = self._chunks = None  # device tables of the step / of the chunks
        self._status = torch.zeros(2, dtype=torch.int32, device=self.device)  # of every call, until check()

    # -- per step ---------------------------------------------------------
    def _only_grew(self, indptr, block_ids) -> bool:
        """Every table is the previous step's, with at most one block appended."""
        pi, pb = self._tables
        old_len, new_len = np.diff(pi), np.diff(indptr)
        if len(old_len) != len(new_len) or np.any((new_len < old_len) | (new_len > old_len + 1)):
            return False
        idx = np.repeat(indptr[:-1], old_len) + (np.arange(int(pi[-1])) - np.repeat(pi[:-1], old_len))
        return bool(np.array_equal(block_ids[idx], pb[:int(pi[-1])]))

    def begin_step(self, indptr, block_ids, positions, tree_grew_only: bool | None = None) -> bool:
        """Plan the step. positions[b]: the new token's index in sequence b
        (so it holds positions[b] + 1 tokens after the step). The plan is
        advanced in place when every sequence only gained this token (and
        maybe a block for it) since the last step — checked against the
        previous tables unless the caller says so with tree_grew_only=True —
        and re-planned otherwise. Returns True when advanced."""
        indptr = np.ascontiguousarray(indptr, dtype=np.int32)
        block_ids = np.ascontiguousarray(np.asarray(block_ids).astype(np.uint32))  # -1: a page given back
        pos = np.ascontiguousarray(positions, dtype=np.int64)
        # The plan checks the lengths against the tables; a step of windowed layers has none.
        self._check_tables(indptr, block_ids)
        if len(pos) != len(indptr) - 1 or np.any(pos < 0) or \
                np.any(pos >= np.diff(indptr).astype(np.int64) * PAGE_SIZE):
            raise _lib.InvalidArgument("the tables and the positions do not fit together")
        ntok = (pos + 1).astype(np.int32)
        blk = block_ids[indptr[:-1] + pos // PAGE_SIZE]
        advanced = False
        if not all(self.windows):  # else nothing needs the plan
            if self.plan is not None and self._ntok is not None and len(self._ntok) == len(ntok) \
                    and np.array_equal(self._ntok + 1, ntok) \
                    and (tree_grew_only or (tree_grew_only is None and self._only_grew(indptr, block_ids))):
                advanced = self.plan.advance(np.ones(len(ntok), np.int32), blk)
            if not advanced:
                if self.plan is None:
                    self.plan = CascadePlan(self.cfg, indptr, block_ids, ntok)
                else:
                    try:
                        self.plan.rebuild(indptr, block_ids, ntok)
                    except _lib.InvalidArgument:  # which empties the plan
                        self.plan.rebuild(*self._tables, self._ntok)
                        self.plan.upload(self.device)
                        raise
            self.plan.upload(self.device)
            self._ntok = ntok
            self._tables = (indptr.copy(), block_ids.copy())
        # Only now: a step that the plan refuses leaves the last one as it was.
        if any(self.windows):
            self._step = self._device_tables(indptr, block_ids, ntok)
        self._page_ids = torch.from_numpy(blk.astype(np.int32)).to(self.device)
        self._slots = torch.from_numpy((pos % PAGE_SIZE).astype(np.int32)).to(self.device)
        return advanced

    @staticmethod
    def _check_tables(indptr, block_ids) -> None:
        if len(indptr) < 1 or indptr[0] < 0 or np.any(np.diff(indptr) < 0) or indptr[-1] > len(block_ids):
            raise _lib.InvalidArgument("the tables and the block ids do not fit together")

    def _device_tables(self, indptr, block_ids, ntok):
        """(page_indptr, page_indices, num_tokens on the device, pages of the longest table)."""
        self._check_tables(indptr, block_ids)
        dev = [torch.from_numpy(np.ascontiguousarray(x).view(np.int32)).to(self.device)
               for x in (indptr, block_ids, ntok)]
        return (*dev, int(np.diff(indptr).max(initial=0)))

    @staticmethod
    def _check_rows(q, k, v, rows) -> None:
        """The append takes a page and a slot for each row of K."""
        if not q.shape[0] == k.shape[0] == v.shape[0] == rows:
            raise _lib.InvalidArgument(f"q, k and v must have the batch's {rows} rows")

    def layer_step(self, layer: int, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor) -> torch.Tensor:
        """Store layer `layer`'s new K/V [B, Hkv, D] and attend with q [B, Hq, D]."""
        if self._page_ids is None:
            raise _lib.InvalidArgument("begin_step first")
        self._check_rows(q, k, v, len(self._page_ids))
        q = _rows_in_place(q.to(torch.bfloat16))
        if self.windows[layer]:
            ip, ids, ntok, longest = self._step
            append_kv_paged(self.cfg, self.pools[layer], self.scales[layer], None, ip, ids, ntok, _rows_in_place(k),
                            _rows_in_place(v), status=self._status)
            out, _ = decode_paged_window(self.cfg, q, self.pools[layer], ip, ids, ntok, *self.windows[layer],
                                         max_pages=longest, kv_scales=self.scales[layer], status=self._status)
            return out
        append_kv_batch(self.cfg, self.pools[layer], self.scales[layer], self._page_ids, self._slots,
                        k.contiguous(), v.contiguous(), status=self._status)
        ws = _alloc_ws(self.plan.info().workspace_bytes, self.device, self._ws)
        out, _ = cascade_decode(self.cfg, self.plan, q.contiguous(), self.pools[layer], self.scales[layer],
                                workspace=ws)
        return out

    # -- prompts ------------------------------------------------------------
    def layer_prefill(self, layer: int, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                      table, prefix_len: int) -> torch.Tensor:
        """One sequence's S new tokens: store their K/V [S, Hkv, D] at
        positions prefix_len .. prefix_len + S of `table` and return the
        causal attention of q [S, Hq, D] (new token i sees tokens
        0 .. prefix_len + i)."""
        S = q.shape[0]
        self._check_rows(q, k, v, S)
        if prefix_len < 0 or prefix_len + S > len(table) * PAGE_SIZE:
            raise _lib.InvalidArgument("the table, prefix_len and the rows do not fit together")
        if self.windows[layer]:
            tbl = np.asarray(table).astype(np.uint32)
            return self._chunk(layer, self._chunk_tables([0, len(tbl)], tbl, [prefix_len + S], [S]), q, k, v)
        pos = np.arange(prefix_len, prefix_len + S)
        tbl = np.asarray(table, dtype=np.uint32)
        page_ids = torch.from_numpy(tbl[pos // PAGE_SIZE].astype(np.int32)).to(self.device)
        slots = torch.from_numpy((pos % PAGE_SIZE).astype(np.int32)).to(self.device)
        append_kv_batch(self.cfg, self.pools[layer], self.scales[layer], page_ids, slots,
                        k.contiguous(), v.contiguous(), status=self._status)
        plan = CascadePlan.prefill(self.cfg, [0, len(tbl)], tbl, [prefix_len], [S])
        plan.upload(self.device)
        out, _ = cascade_decode(self.cfg, plan, _rows_in_place(q.to(torch.bfloat16)).contiguous(), self.pools[layer],
                                self.scales[layer])
        return out

    # -- chunks of several sequences ------------------------------------------
    def begin_chunks(self, indptr, block_ids, num_tokens, new_tokens) -> None:
        """A ragged batch: sequence s (table block_ids[indptr[s]:indptr[s + 1]])
        will hold num_tokens[s] tokens, the last new_tokens[s] of them new."""
        self._chunks = self._chunk_tables(indptr, block_ids, num_tokens, new_tokens)

    def _chunk_tables(self, indptr, block_ids, num_tokens, new_tokens):
        """_device_tables of a ragged batch, its rows' borders on the device, and its rows."""
        indptr = np.ascontiguousarray(indptr, dtype=np.int32)
        ids = np.ascontiguousarray(np.asarray(block_ids).astype(np.uint32))
        ntok = np.ascontiguousarray(num_tokens, dtype=np.int32)
        new = np.ascontiguousarray(new_tokens, dtype=np.int32)
        if len(indptr) != len(ntok) + 1 or len(new) != len(ntok) or np.any(new < 0) or np.any(new > ntok) or \
                np.any(ntok > np.diff(indptr).astype(np.int64) * PAGE_SIZE):
            raise _lib.InvalidArgument("tables, num_tokens and new_tokens do not fit together")
        rows = np.concatenate([[0], np.cumsum(new, dtype=np.int64)]).astype(np.int32)
        return self._device_tables(indptr, ids, ntok) + (torch.from_numpy(rows).to(self.device), int(rows[-1]))

    def layer_chunk(self, layer: int, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor) -> torch.Tensor:
        """Store layer `layer`'s new K/V [rows, Hkv, D] of the batch of
        begin_chunks and attend with q [rows, Hq, D] (rows sequence by
        sequence; all three may be parts of a wider projection, and have more
        rows than the batch, whose outputs then are not set)."""
        if self._chunks is None:
            raise _lib.InvalidArgument("begin_chunks first")
        return self._chunk(layer, self._chunks, q, k, v)

    def _chunk(self, layer, tables, q, k, v):
        ip, ids, ntok, longest, borders, rows = tables
        if not q.shape[0] == k.shape[0] == v.shape[0] >= rows:
            raise _lib.InvalidArgument(f"q, k and v must have the batch's {rows} rows")
        append_kv_paged(self.cfg, self.pools[layer], self.scales[layer], borders, ip, ids, ntok, _rows_in_place(k),
                        _rows_in_place(v), status=self._status)
        window, sinks = self.windows[layer] or (0, 0)
        out, _ = prefill_paged_window(self.cfg, _rows_in_place(q.to(torch.bfloat16)), self.pools[layer], borders, ip,
                                      ids, ntok, window, sinks, max_pages=longest, kv_scales=self.scales[layer],
                                      status=self._status)
        return out

    def read_tokens(self, layer: int, indptr, block_ids, first, count, out_dtype=torch.bfloat16):
        """K and V [sum(count), Hkv, D] of tokens first[s] .. first[s] + count[s]
        of each sequence, dequantised."""
        indptr = np.ascontiguousarray(indptr, dtype=np.int32)
        ids = np.ascontiguousarray(np.asarray(block_ids).astype(np.uint32))
        first = np.ascontiguousarray(first, dtype=np.int32)
        count = np.ascontiguousarray(count, dtype=np.int32)
        if len(indptr) != len(first) + 1 or len(count) != len(first) or np.any(first < 0) or np.any(count < 0) or \
                np.any(first.astype(np.int64) + count > np.diff(indptr).astype(np.int64) * PAGE_SIZE):
            raise _lib.InvalidArgument("tables, first and count do not fit together")
        ip, pages, start, _ = self._device_tables(indptr, ids, first)
        rows = np.concatenate([[0], np.cumsum(count, dtype=np.int64)]).astype(np.int32)
        return gather_kv_paged(self.cfg, self.pools[layer], self.scales[layer], torch.from_numpy(rows).to(self.device),
                               start, ip, pages, int(rows[-1]), out_dtype, status=self._status)

    # -- what went wrong on the device ----------------------------------------
    def check(self) -> None:
        """Raise if an append, a windowed attention or a read-back since the last
        check met a page outside the pool or the table (it skipped the page, or
        read zeros), or gave up a wait. Waits for the current stream; a page
        that the engine gave back one step too early is found here."""
        code, where = self._status.tolist()
        if not code:
            return
        self._status.zero_()
        if code == 1:
            raise _lib.InvalidArgument("a page outside the pool, or a missing one, was skipped "
                                       f"(the page, or the row that it was for: {where & 0xffffffff})")
        raise _lib.CudaError(f"a kernel gave up a wait (status {code}, {where & 0xffffffff}): its outputs are not valid")

