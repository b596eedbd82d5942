"""Sliding-window layers over the paged cache: the append of a ragged batch of
new tokens, attention of one token or of a chunk of tokens per sequence over
the last `window` tokens and the first `sinks` ones, and the read-back of
token ranges.

All four take the batch as device arrays (CSR page tables, token counts), so
nothing of it is planned or copied on the host and a call can be captured into
a CUDA graph. Sequence s holds num_tokens[s] tokens, the new ones included;
its page table is page_indices[page_indptr[s]:page_indptr[s + 1]] (int32 or
uint32). Table entries of pages that no window reaches any more are not read
and may hold anything. See include/dendrite_b200.h for the exact rules.

`status` (2 x int32 or uint32 on the device, cleared by the caller) receives
the first bad page; without it bad pages are skipped silently.
"""
from __future__ import annotations

import ctypes as C

import torch

from ._lib import DTYPE_BF16, DTYPE_E4M3, DTYPE_F32, DTYPE_MXFP8, AttnConfig, InvalidArgument, check, lib

_INDEX = (torch.int32, torch.uint32)
_POOL = {DTYPE_BF16: (torch.bfloat16,), DTYPE_F32: (torch.float32,),
         DTYPE_E4M3: (torch.uint8, torch.float8_e4m3fn), DTYPE_MXFP8: (torch.uint8, torch.float8_e4m3fn)}


def _fail(msg: str):
    raise InvalidArgument(msg)


def _check_pool(cfg: AttnConfig, kv_pages, kv_scales) -> None:
    kvd = cfg.kv_dtype
    if kv_pages is None:
        _fail("kv_pages is None")
    if kv_pages.dtype not in _POOL.get(kvd, ()) or not kv_pages.is_contiguous() or \
            kv_pages.shape != (cfg.num_pages, 2, cfg.num_kv_heads, cfg.page_size, cfg.head_dim):
        _fail("kv_pages must be a dense [num_pages][2][Hkv][16][D] pool of the config's kv_dtype")
    if kvd == DTYPE_E4M3:
        if kv_scales is None or kv_scales.dtype != torch.float32 or not kv_scales.is_contiguous() or \
                kv_scales.numel() != 2 * cfg.num_kv_heads:
            _fail("E4M3 pages need dense f32 kv_scales [2][Hkv]")
    elif kvd == DTYPE_MXFP8:
        if kv_scales is None or kv_scales.dtype != torch.uint8 or not kv_scales.is_contiguous() or \
                kv_scales.numel() * 32 != kv_pages.numel():
            _fail("MXFP8 pages need dense uint8 kv_scales [num_pages][2][Hkv][16][D/32]")


def _check_index(name: str, t, n: int) -> None:
    if t.dtype not in _INDEX or not t.is_contiguous() or t.dim() != 1 or t.numel() < n:
        _fail(f"{name} must be a dense int32 vector of at least {n}")


def _check_rows(name: str, t, heads: int, dim: int) -> int:
    """[rows][heads][dim], the heads dense behind one another, any row stride.
    Returns the row stride; that of a single row may be anything and is not used."""
    shape, stride = t.shape, t.stride()
    if len(shape) != 3 or shape[1] != heads or shape[2] != dim or stride[2] != 1 or \
            (heads > 1 and stride[1] != dim):
        _fail(f"{name} must be [rows][{heads}][{dim}] with dense rows")
    return stride[0] if shape[0] > 1 else heads * dim


def _device(*tensors) -> int:
    dev = tensors[0].get_device()  # -1 on the host
    for t in tensors:
        if t is not None and t.get_device() != dev:
            _fail("all tensors must be on one device")
    if dev < 0:
        _fail("the tensors must be on a CUDA device")
    return dev


def _status_ptr(status):
    if status is None:
        return None
    if status.dtype not in _INDEX or not status.is_contiguous() or status.numel() < 2:
        _fail("status must be a dense int32 vector of 2")
    return status.data_ptr()


def _call(dev: int, fn, name: str, args, stream) -> None:
    """The C call with the tensors' device current, on `stream` or that device's current one."""
    handle = torch._C._cuda_getCurrentRawStream(dev) if stream is None else stream.cuda_stream
    if torch.cuda.current_device() == dev:
        check(fn(*args, handle), name)
    else:
        with torch.cuda.device(dev):
            check(fn(*args, handle), name)


def _attend(cfg, q, kv_pages, q_indptr, page_indptr, page_indices, num_tokens, window, sinks, max_pages,
            kv_scales, out, lse, status, stream):
    if not (0 <= window < 1 << 31 and 0 <= sinks < 1 << 31 and 0 <= max_pages < 1 << 31):
        _fail("window, sinks and max_pages must be >= 0 and below 2^31")  # ctypes would cut them off
    heads, dim = cfg.num_qo_heads, cfg.head_dim
    stride = _check_rows("q", q, heads, dim)
    if q.dtype != (torch.float32 if cfg.q_dtype == DTYPE_F32 else torch.bfloat16):
        _fail("q does not have the config's q_dtype")
    _check_pool(cfg, kv_pages, kv_scales)
    rows = q.shape[0]
    if q_indptr is None:
        seqs = rows
    else:
        _check_index("q_indptr", q_indptr, 1)
        seqs = q_indptr.numel() - 1
    _check_index("page_indptr", page_indptr, seqs + 1)
    _check_index("page_indices", page_indices, 0)
    _check_index("num_tokens", num_tokens, seqs)
    shape = (rows, heads, dim)
    if out is not None and (out.dtype != q.dtype or out.shape != shape or not out.is_contiguous()):
        _fail("out must be dense, of q's shape and type")
    if lse is not None and (lse.dtype != torch.float32 or lse.shape != shape[:2] or not lse.is_contiguous()):
        _fail("lse must be dense f32 [rows][Hq]")
    st = _status_ptr(status)
    dev = _device(q, kv_pages, kv_scales, q_indptr, page_indptr, page_indices, num_tokens, out, lse, status)
    if out is None:
        out = q.new_empty(shape)
    if lse is None:
        lse = q.new_empty(shape[:2], dtype=torch.float32)
    head = (C.byref(cfg), seqs) if q_indptr is None else (C.byref(cfg), seqs, rows)
    tables = (page_indptr.data_ptr(), page_indices.data_ptr(), num_tokens.data_ptr())
    args = head + (max_pages, window, sinks, q.data_ptr(), stride, kv_pages.data_ptr(),
                   None if kv_scales is None else kv_scales.data_ptr())
    if q_indptr is None:
        _call(dev, lib.dd_decode_paged_window, "dd_decode_paged_window",
              args + tables + (out.data_ptr(), lse.data_ptr(), st), stream)
    else:
        _call(dev, lib.dd_prefill_paged_window, "dd_prefill_paged_window",
              args + (q_indptr.data_ptr(),) + tables + (out.data_ptr(), lse.data_ptr(), st), stream)
    return out, lse


def decode_paged_window(cfg: AttnConfig, q: torch.Tensor, kv_pages: torch.Tensor, page_indptr: torch.Tensor,
                        page_indices: torch.Tensor, num_tokens: torch.Tensor, window: int, sinks: int = 0,
                        max_pages: int = 0, kv_scales: torch.Tensor | None = None,
                        out: torch.Tensor | None = None, lse: torch.Tensor | None = None,
                        status: torch.Tensor | None = None, stream=None):
    """One new token per sequence: q [B, Hq, D] (any row stride), its token
    already stored, over the last `window` tokens (0: all) and the first
    `sinks`. max_pages (pages of the longest table, 0: unknown) only guides how
    the work is divided. Returns (out [B, Hq, D], lse [B, Hq])."""
    return _attend(cfg, q, kv_pages, None, page_indptr, page_indices, num_tokens, window, sinks, max_pages,
                   kv_scales, out, lse, status, stream)


def prefill_paged_window(cfg: AttnConfig, q: torch.Tensor, kv_pages: torch.Tensor, q_indptr: torch.Tensor,
                         page_indptr: torch.Tensor, page_indices: torch.Tensor, num_tokens: torch.Tensor,
                         window: int, sinks: int = 0, max_pages: int = 0,
                         kv_scales: torch.Tensor | None = None, out: torch.Tensor | None = None,
                         lse: torch.Tensor | None = None, status: torch.Tensor | None = None, stream=None):
    """A chunk of new tokens per sequence, causally: rows q_indptr[s]:q_indptr[s+1]
    of q [rows, Hq, D] are the last tokens of sequence s, already stored.
    Rows behind q_indptr[-1] are left as they are. Returns (out, lse)."""
    if q_indptr is None:
        _fail("q_indptr is None")
    return _attend(cfg, q, kv_pages, q_indptr, page_indptr, page_indices, num_tokens, window, sinks,
                   max_pages, kv_scales, out, lse, status, stream)


def append_kv_paged(cfg: AttnConfig, kv_pages: torch.Tensor, kv_scales: torch.Tensor | None,
                    new_indptr: torch.Tensor | None, page_indptr: torch.Tensor, page_indices: torch.Tensor,
                    num_tokens: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                    status: torch.Tensor | None = None, stream=None) -> None:
    """Store rows new_indptr[s]:new_indptr[s+1] of k, v [rows, Hkv, D] (bf16 or
    f32, any row stride) as the last tokens of sequence s, quantising for FP8
    pools. num_tokens counts them already; new_indptr None: one per sequence."""
    _check_pool(cfg, kv_pages, kv_scales)
    k_stride = _check_rows("k", k, cfg.num_kv_heads, cfg.head_dim)
    v_stride = _check_rows("v", v, cfg.num_kv_heads, cfg.head_dim)
    if k.dtype != v.dtype or k.dtype not in (torch.bfloat16, torch.float32) or k.shape[0] != v.shape[0]:
        _fail("k and v must both be bf16 or f32, of as many rows")
    rows = k.shape[0]
    if new_indptr is None:
        seqs = rows
    else:
        _check_index("new_indptr", new_indptr, 1)
        seqs = new_indptr.numel() - 1
    _check_index("page_indptr", page_indptr, seqs + 1)
    _check_index("page_indices", page_indices, 0)
    _check_index("num_tokens", num_tokens, seqs)
    st = _status_ptr(status)
    dev = _device(kv_pages, kv_scales, new_indptr, page_indptr, page_indices, num_tokens, k, v, status)
    _call(dev, lib.dd_append_kv_paged, "dd_append_kv_paged",
          (C.byref(cfg), kv_pages.data_ptr(), None if kv_scales is None else kv_scales.data_ptr(), seqs, rows,
           None if new_indptr is None else new_indptr.data_ptr(), page_indptr.data_ptr(), page_indices.data_ptr(),
           num_tokens.data_ptr(), k.data_ptr(), k_stride, v.data_ptr(), v_stride,
           DTYPE_F32 if k.dtype == torch.float32 else DTYPE_BF16, st), stream)


def gather_kv_paged(cfg: AttnConfig, kv_pages: torch.Tensor, kv_scales: torch.Tensor | None,
                    out_indptr: torch.Tensor, first_token: torch.Tensor | None, page_indptr: torch.Tensor,
                    page_indices: torch.Tensor, num_rows: int, out_dtype: torch.dtype = torch.bfloat16,
                    k: torch.Tensor | None = None, v: torch.Tensor | None = None,
                    status: torch.Tensor | None = None, stream=None):
    """Read token first_token[s] + i (first_token None: i) of sequence s back
    into row out_indptr[s] + i of k, v [num_rows, Hkv, D], dequantised and
    rounded once to out_dtype (bf16 or f32). Returns (k, v)."""
    _check_pool(cfg, kv_pages, kv_scales)
    if out_dtype not in (torch.bfloat16, torch.float32):
        _fail("out_dtype must be bf16 or f32")
    if not 0 <= num_rows < 1 << 31:
        _fail("num_rows must be >= 0 and below 2^31")
    _check_index("out_indptr", out_indptr, 1)
    seqs = out_indptr.numel() - 1
    _check_index("page_indptr", page_indptr, seqs + 1)
    _check_index("page_indices", page_indices, 0)
    if first_token is not None:
        _check_index("first_token", first_token, seqs)
    shape = (num_rows, cfg.num_kv_heads, cfg.head_dim)
    for name, t in (("k", k), ("v", v)):
        if t is not None and (t.dtype != out_dtype or t.shape != shape or not t.is_contiguous()):
            _fail(f"{name} must be dense [num_rows][Hkv][D] of out_dtype")
    st = _status_ptr(status)
    dev = _device(kv_pages, kv_scales, out_indptr, first_token, page_indptr, page_indices, k, v, status)
    if k is None:
        k = kv_pages.new_empty(shape, dtype=out_dtype)
    if v is None:
        v = kv_pages.new_empty(shape, dtype=out_dtype)
    _call(dev, lib.dd_gather_kv_paged, "dd_gather_kv_paged",
          (C.byref(cfg), kv_pages.data_ptr(), None if kv_scales is None else kv_scales.data_ptr(), seqs, num_rows,
           out_indptr.data_ptr(), None if first_token is None else first_token.data_ptr(), page_indptr.data_ptr(),
           page_indices.data_ptr(), k.data_ptr(), v.data_ptr(),
           DTYPE_F32 if out_dtype == torch.float32 else DTYPE_BF16, st), stream)
    return k, v
