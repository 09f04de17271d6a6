"""Operators over tensors in device memory (the mk_k_*_dev entry points), for serving many continuations of one prompt.

Unlike the wrappers of ``ops``, which move host arrays to the device and back, these take CUDA tensors as they are, enqueue their kernels on
the current stream of the tensors' device and return without waiting; they may be captured into a CUDA graph (sizes, pointers, Python
numbers and strides are fixed then, contents are not).  Index tensors are int32.  ``status`` is an optional int32 tensor of one element into
which the kernels OR what they met (``BAD_PAGE``, ``WAIT_GAVE_UP``, ``BAD_RANGE``, ``BAD_ROW``); ``check_status`` reads it.  Arguments that can be judged by shape, type and
stride are refused with ValueError before anything is launched, what the entry points themselves refuse (a head size, a length, an alignment, rows that overlap) with MkError, also before.
"""
from __future__ import annotations

import ctypes as C
import functools

import torch

from . import _capi as capi

BAD_PAGE, WAIT_GAVE_UP, BAD_RANGE, BAD_ROW = 1, 2, 4, 8

_TYPES = {torch.float32: capi.TYPE_F32, torch.float16: capi.TYPE_F16, torch.bfloat16: capi.TYPE_BF16}
_I32, _F32 = torch.int32, torch.float32
_current_device, _raw_stream = torch._C._cuda_getDevice, torch._C._cuda_getCurrentRawStream


# A call's host time counts in ticks of a few microseconds, so shapes, types, strides and places are compared in line and a message is only put together for a refusal.

def _dense(t, dtype, shape, device, what: str) -> int:
    """Address of a contiguous tensor."""
    if t.dtype is not dtype or t.shape != shape or t.get_device() != device or not t.is_contiguous():
        raise ValueError(f"{what} is a contiguous {dtype} tensor of shape {tuple(shape)} on the device of the others: got {t.dtype} {tuple(t.shape)} on {t.device}")
    return t.data_ptr()


def _rows(t, lanes, device, what: str):
    """Address, row distance and width of an int32 tensor [lanes, width] whose rows are dense."""
    shape = t.shape
    if t.dtype is not _I32 or len(shape) != 2 or shape[0] != lanes or t.get_device() != device or (shape[1] > 1 and t.stride(1) != 1):
        raise ValueError(f"{what} is an int32 tensor [{lanes}, ...] with dense rows on the device of the others: got {t.dtype} {tuple(shape)} on {t.device}")
    return t.data_ptr(), t.stride(0) if lanes > 1 else max(shape[1], 1), shape[1]


def _run(device: int, fn, *args) -> None:
    """fn(..., the device's current stream), with that device current."""
    if device < 0:
        raise ValueError("tensors are on a CUDA device")
    if _current_device() == device:
        code = fn(*args, _raw_stream(device))
    else:
        with torch.cuda.device(device):
            code = fn(*args, _raw_stream(device))
    if code:
        capi.check(code)


@functools.lru_cache(maxsize=4096)
def _attention_workspace(*sizes) -> int:
    need = C.c_int64()
    capi.check(capi.lib().mk_k_shared_attention_workspace(*sizes, C.byref(need)))
    return need.value


@functools.lru_cache(maxsize=4096)
def _verify_workspace(*sizes) -> int:
    need = C.c_int64()
    capi.check(capi.lib().mk_k_verify_drafts_workspace(*sizes, C.byref(need)))
    return need.value


def check_status(status) -> None:
    """Reads a status tensor (waits for the current stream) and raises what it tells of; clears it."""
    bits = int(status.item())
    if bits:
        status.zero_()
        told = [text for bit, text in ((BAD_PAGE, "a page number outside the pool"), (WAIT_GAVE_UP, "a bounded wait inside a kernel gave up"),
                                       (BAD_RANGE, "a length, count, position or setting out of range"), (BAD_ROW, "a row of logits that is no distribution")) if bits & bit]
        raise capi.MkError("; ".join(told))


def shared_attention(q, k_pool, v_pool, tables, lengths, shared_len: int, *, scale: float, cu_seqlens=None, max_rows: int = 0, softcap: float = 0.0, window: int = 0,
                     out=None, status=None):
    """Attention of a batch whose lanes share their first ``shared_len`` tokens (whole pages), which are read once for all lanes.

    q [total, q_heads, head_dim]; k_pool / v_pool [pages, kv_heads, block_tokens, head_dim], one layer, f16 or bf16 like q (pages may be further apart than
    they are long); tables [lanes, width] page numbers; lengths [lanes] tokens of each lane, its rows of q being the last of them.  Without cu_seqlens
    [lanes + 1] every lane has total / lanes rows; with it, ``max_rows`` is the most that a lane has.  Returns [total, q_heads, head_dim]; rows outside
    cu_seqlens are left as ``out`` had them."""
    dtype, device, shape, pool, strides, v_strides = q.dtype, q.get_device(), q.shape, k_pool.shape, k_pool.stride(), v_pool.stride()
    if len(shape) != 3 or (dtype is not torch.float16 and dtype is not torch.bfloat16):
        raise ValueError("q is a float16 or bfloat16 tensor [rows, heads, head size]")
    total, heads, dim = shape
    if (len(pool) != 4 or pool[3] != dim or v_pool.shape != pool or (v_strides != strides and any(x != y and n != 1 for n, x, y in zip(pool, strides, v_strides))) or k_pool.dtype is not dtype or v_pool.dtype is not dtype
            or k_pool.get_device() != device or v_pool.get_device() != device):
        raise ValueError("k_pool and v_pool are [pages, kv heads, tokens of a page, head size] of q's type and head size, strided alike, on its device")
    pages, kv_heads, page, _ = pool
    if strides[1:] != (page * dim, dim, 1) and (kv_heads != 1 or strides[2:] != (dim, 1)):
        raise ValueError("pages are dense")
    lanes = tables.shape[0] if tables.dim() == 2 else -1
    table, table_stride, width = _rows(tables, lanes, device, "tables")
    if cu_seqlens is None:
        rows, cu = total // lanes if lanes else 0, None
        if rows * lanes != total:
            raise ValueError("without cu_seqlens every lane has the same number of rows")
    else:
        rows, cu = max_rows, _dense(cu_seqlens, _I32, (lanes + 1,), device, "cu_seqlens")
        if max_rows <= 0 and total:
            raise ValueError("with cu_seqlens, max_rows says how many rows a lane has at most")
    q_strides = q.stride()
    if total and q_strides[1:] != (dim, 1) and (heads != 1 or q_strides[2] != 1):
        raise ValueError("the heads of a row are dense")
    if out is None:
        out, out_stride = torch.empty_like(q), heads * dim   # dense, since the heads of a row are
    else:
        out_strides = out.stride()
        if (out.shape != shape or out.dtype is not dtype or out.get_device() != device
                or (total and out_strides[1:] != (dim, 1) and (heads != 1 or out_strides[2] != 1))):
            raise ValueError("out is like q, the heads of a row dense")
        out_stride = out_strides[0] if total > 1 else heads * dim
    need = _attention_workspace(heads, kv_heads, dim, page, width, lanes, rows, total, shared_len, window)
    space = q.new_empty(need // 2) if need else None
    _run(device, capi.lib().mk_k_shared_attention_dev, _TYPES[dtype], q.data_ptr(), q_strides[0] if total > 1 else heads * dim, k_pool.data_ptr(), v_pool.data_ptr(), pages,
         strides[0] if pages > 1 else kv_heads * page * dim, heads, kv_heads, dim, page, table, table_stride, width, _dense(lengths, _I32, (lanes,), device, "lengths"), cu, lanes, rows,
         total, shared_len, scale, softcap, window, out.data_ptr(), out_stride, space.data_ptr() if need else None, need,
         None if status is None else _dense(status, _I32, (1,), device, "status"))
    return out


def verify_drafts(logits, drafts, u, *, temperature, top_k, top_p, draft_probs=None, tokens=None, accepted=None, status=None):
    """Keeps the drafted tokens that the target's distribution bears out and draws the one behind them, from given random numbers.

    logits [lanes, drafts + 1, vocab] f32, f16 or bf16 (rows may be further apart); drafts [lanes, drafts], a negative one ends a lane's; u [lanes, drafts + 1] f32 in
    [0, 1); temperature, top_k, top_p [lanes] as of the sampler (temperature 0: greedy, top_k 0: the whole vocabulary); draft_probs [lanes, drafts, vocab] f32, or None for
    drafts that were looked up.  As of the sampler too, top_k goes up to 1024 and top_p below 1 needs a top_k: a lane with another setting gets token -1, no drafts and
    BAD_RANGE, and one that reaches a row that is no distribution token -1 and BAD_ROW.  Returns (tokens [lanes, drafts + 1]: kept drafts, the token behind them, -1 behind that; accepted [lanes])."""
    dtype, device, shape = logits.dtype, logits.get_device(), logits.shape
    if len(shape) != 3 or dtype not in _TYPES or shape[1] < 1 or shape[2] < 1:
        raise ValueError("logits is a float32, float16 or bfloat16 tensor [lanes, drafts + 1, vocabulary]")
    lanes, n, vocab = shape
    strides = logits.stride()
    ld = strides[1] if n > 1 else (strides[0] if lanes > 1 else vocab)
    if lanes and ((vocab > 1 and strides[2] != 1) or (n > 1 and lanes > 1 and strides[0] != n * ld)):
        raise ValueError("rows of logits are dense and evenly apart")
    need = _verify_workspace(_TYPES[dtype], lanes, n - 1, vocab)
    of_lane, of_row = (lanes,), (lanes, n)
    n -= 1
    given = _dense(drafts, _I32, (lanes, n), device, "drafts")
    if tokens is None:
        tokens = torch.empty_like(u, dtype=_I32)
    if accepted is None:
        accepted = torch.empty_like(top_k)
    space = logits.new_empty(need // logits.element_size() + 1)
    _run(device, capi.lib().mk_k_verify_drafts_dev, _TYPES[dtype], logits.data_ptr(), ld, lanes, n, vocab, given,
         None if draft_probs is None else _dense(draft_probs, _F32, (lanes, n, vocab), device, "draft_probs"), _dense(u, _F32, of_row, device, "u"),
         _dense(temperature, _F32, of_lane, device, "temperature"), _dense(top_k, _I32, of_lane, device, "top_k"), _dense(top_p, _F32, of_lane, device, "top_p"),
         _dense(tokens, _I32, of_row, device, "tokens"), _dense(accepted, _I32, of_lane, device, "accepted"), space.data_ptr(), need,
         None if status is None else _dense(status, _I32, (1,), device, "status"))
    return tokens, accepted


def _pools(k_pool, v_pool):
    shape, dtype = k_pool.shape, k_pool.dtype
    if (len(shape) != 5 or v_pool.shape != shape or v_pool.dtype is not dtype or dtype not in _TYPES or v_pool.get_device() != k_pool.get_device()
            or not k_pool.is_contiguous() or not v_pool.is_contiguous()):
        raise ValueError("k_pool and v_pool are contiguous [layers, pages, kv heads, tokens of a page, head size] of one shape and type (float32, float16 or bfloat16), on one device")
    layers, pages, heads, page, dim = shape
    return k_pool.data_ptr(), v_pool.data_ptr(), layers, pages, heads, page, dim * dtype.itemsize


def copy_pages(k_pool, v_pool, copies, *, status=None) -> None:
    """Copies the first ``rows`` tokens of pages to other pages, in every layer: copies [n, 3] of (from page, to page, rows).  No page is written twice, or
    written by one copy and read by another."""
    if copies.dim() != 2:
        raise ValueError("copies is [n, 3]")
    device, n = k_pool.get_device(), copies.shape[0]
    _run(device, capi.lib().mk_k_copy_pages_dev, *_pools(k_pool, v_pool), _dense(copies, _I32, (n, 3), device, "copies"), n,
         None if status is None else _dense(status, _I32, (1,), device, "status"))


def gather_tokens(k_pool, v_pool, from_tables, keep, counts, to_tables, first, *, status=None) -> None:
    """Moves kept tokens of lanes together, in every layer: token keep[i, j] of the pages from_tables[i] becomes token first[i] + j of the pages to_tables[i], for
    j < counts[i].  keep ascends; the tables name the same pages (then first[i] <= keep[i, 0] and no token is kept twice), or pages that nothing else here reads or writes."""
    if keep.dim() != 2:
        raise ValueError("keep is [lanes, kept tokens]")
    device, lanes = k_pool.get_device(), keep.shape[0]
    _run(device, capi.lib().mk_k_gather_tokens_dev, *_pools(k_pool, v_pool), *_rows(from_tables, lanes, device, "from_tables"), *_rows(keep, lanes, device, "keep"),
         _dense(counts, _I32, (lanes,), device, "counts"), *_rows(to_tables, lanes, device, "to_tables"), _dense(first, _I32, (lanes,), device, "first"), lanes,
         None if status is None else _dense(status, _I32, (1,), device, "status"))
