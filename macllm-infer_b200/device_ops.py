"""Operators over tensors in device memory (the mk_k_*_dev entry points), for serving many continuations of one prompt.

Unlike the wrappers of ``ops``, which move host arrays to the device and back, these take CUDA tensors as they are, enqueue their kernels on
the current stream of the tensors' device and return without waiting; they may be captured into a CUDA graph (sizes, pointers, Python
numbers and strides are fixed then, contents are not).  Index tensors are int32.  ``status`` is an optional int32 tensor of one element into
which the kernels OR what they met (``BAD_PAGE``, ``WAIT_GAVE_UP``, ``BAD_RANGE``, ``BAD_ROW``); ``check_status`` reads it.  Arguments that can be judged by shape, type and
stride are refused with ValueError before anything is launched.
"""
from __future__ import annotations

import ctypes as C

import torch

from . import _capi as capi

BAD_PAGE, WAIT_GAVE_UP, BAD_RANGE, BAD_ROW = 1, 2, 4, 8

_TYPES = {torch.float32: capi.TYPE_F32, torch.float16: capi.TYPE_F16, torch.bfloat16: capi.TYPE_BF16}


def _ask(ok: bool, what: str) -> None:
    if not ok:
        raise ValueError(what)


def _index(t, shape, device, what: str) -> int:
    """Address of an int32 tensor of that shape, its last dimension dense; rows may be further apart (see _stride)."""
    if t.dtype is not torch.int32 or t.shape != shape or t.device != device or (t.numel() > 1 and t.shape[-1] > 1 and t.stride(-1) != 1):
        raise ValueError(f"{what} is an int32 tensor of shape {tuple(shape)} on {device}, dense in its last dimension: got {t.dtype} {tuple(t.shape)} on {t.device}")
    return t.data_ptr()


def _dense(t, dtype, shape, device, what: str) -> int:
    if t.dtype is not dtype or t.shape != shape or t.device != device or not t.is_contiguous():
        raise ValueError(f"{what} is a contiguous {dtype} tensor of shape {tuple(shape)} on {device}: got {t.dtype} {tuple(t.shape)} on {t.device}")
    return t.data_ptr()


def _row_stride(t) -> int:
    """Distance of the rows of a two-dimensional tensor."""
    return t.stride(0) if t.shape[0] > 1 else max(t.shape[1], 1)


def _status(status, device):
    return None if status is None else _dense(status, torch.int32, (1,), device, "status")


def _call(device, fn, *args) -> None:
    """fn(..., the device's current stream), with that device current."""
    if device.type != "cuda":
        raise ValueError(f"tensors are on a CUDA device: got {device}")
    if torch.cuda.current_device() == device.index:
        code = fn(*args, torch._C._cuda_getCurrentRawStream(device.index))
    else:
        with torch.cuda.device(device):
            code = fn(*args, torch._C._cuda_getCurrentRawStream(device.index))
    if code:
        capi.check(code)


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
    device = q.device
    _ask(q.dim() == 3 and q.dtype in (torch.float16, torch.bfloat16), "q is a float16 or bfloat16 tensor [rows, heads, head size]")
    total, heads, dim = q.shape
    _ask(k_pool.dim() == 4 and k_pool.shape[3] == dim and k_pool.shape == v_pool.shape and k_pool.stride() == v_pool.stride() and k_pool.dtype is q.dtype and v_pool.dtype is q.dtype
         and k_pool.device == device and v_pool.device == device, "k_pool and v_pool are [pages, kv heads, tokens of a page, head size] of q's type and head size, strided alike")
    pages, kv_heads, page, _ = k_pool.shape
    _ask(k_pool.stride()[1:] == (page * dim, dim, 1), "pages are dense")
    _ask(tables.dim() == 2, "tables is [lanes, pages]")
    lanes, width = tables.shape
    if cu_seqlens is None:
        rows = total // lanes if lanes else 0
        _ask(rows * lanes == total, "without cu_seqlens every lane has the same number of rows")
        cu = None
    else:
        rows, cu = max_rows, _dense(cu_seqlens, torch.int32, (lanes + 1,), device, "cu_seqlens")
        _ask(max_rows > 0 or total == 0, "with cu_seqlens, max_rows says how many rows a lane has at most")
    if out is None:
        out = torch.empty((total, heads, dim), dtype=q.dtype, device=device)
    else:
        _ask(out.shape == q.shape and out.dtype is q.dtype and out.device == device, "out is like q")
    for t in (q, out):
        _ask(total == 0 or t.stride()[1:] == (dim, 1), "the heads of a row are dense")
    need = C.c_int64()
    lib = capi.lib()
    capi.check(lib.mk_k_shared_attention_workspace(heads, kv_heads, dim, page, width, lanes, rows, total, shared_len, C.byref(need)))
    space = torch.empty(need.value, dtype=torch.uint8, device=device) if need.value else None
    _call(device, lib.mk_k_shared_attention_dev, _TYPES[q.dtype], q.data_ptr(), q.stride(0) if total > 1 else heads * dim, k_pool.data_ptr(), v_pool.data_ptr(), pages,
          k_pool.stride(0) if pages > 1 else kv_heads * page * dim, heads, kv_heads, dim, page, _index(tables, (lanes, width), device, "tables"), _row_stride(tables), width,
          _dense(lengths, torch.int32, (lanes,), device, "lengths"), cu, lanes, rows, total, shared_len, scale, softcap, window, out.data_ptr(),
          out.stride(0) if total > 1 else heads * dim, None if space is None else space.data_ptr(), need.value, _status(status, device))
    return out


def verify_drafts(logits, drafts, u, *, temperature, top_k, top_p, draft_probs=None, tokens=None, accepted=None, status=None):
    """Keeps the drafted tokens that the target's distribution bears out and draws the one behind them, from given random numbers.

    logits [lanes, drafts + 1, vocab] f32, f16 or bf16 (rows may be further apart); drafts [lanes, drafts], a negative one ends a lane's; u [lanes, drafts + 1] f32 in
    [0, 1); temperature, top_k, top_p [lanes] as of the sampler (temperature 0: greedy, top_k 0: the whole vocabulary); draft_probs [lanes, drafts, vocab] f32, or None for
    drafts that were looked up.  Returns (tokens [lanes, drafts + 1]: kept drafts, the token behind them, -1 behind that; accepted [lanes])."""
    device = logits.device
    _ask(logits.dim() == 3 and logits.dtype in _TYPES and logits.shape[1] > 0 and logits.shape[2] > 0, "logits is a float32, float16 or bfloat16 tensor [lanes, drafts + 1, vocabulary]")
    lanes, n, vocab = logits.shape
    ld = logits.stride(1) if n > 1 else (logits.stride(0) if lanes > 1 else vocab)
    _ask(lanes == 0 or ((vocab == 1 or logits.stride(2) == 1) and (n == 1 or lanes == 1 or logits.stride(0) == n * ld)), "rows of logits are dense and evenly apart")
    n -= 1
    if tokens is None:
        tokens = torch.empty((lanes, n + 1), dtype=torch.int32, device=device)
    if accepted is None:
        accepted = torch.empty((lanes,), dtype=torch.int32, device=device)
    need = C.c_int64()
    lib = capi.lib()
    code = lib.mk_k_verify_drafts_workspace(_TYPES[logits.dtype], lanes, n, vocab, C.byref(need))
    if code:
        capi.check(code)
    size = need.value
    space = torch.empty(size, dtype=torch.uint8, device=device)
    _call(device, lib.mk_k_verify_drafts_dev, _TYPES[logits.dtype], logits.data_ptr(), ld, lanes, n, vocab, _dense(drafts, torch.int32, (lanes, n), device, "drafts"),
          None if draft_probs is None else _dense(draft_probs, torch.float32, (lanes, n, vocab), device, "draft_probs"), _dense(u, torch.float32, (lanes, n + 1), device, "u"),
          _dense(temperature, torch.float32, (lanes,), device, "temperature"), _dense(top_k, torch.int32, (lanes,), device, "top_k"),
          _dense(top_p, torch.float32, (lanes,), device, "top_p"), _dense(tokens, torch.int32, (lanes, n + 1), device, "tokens"),
          _dense(accepted, torch.int32, (lanes,), device, "accepted"), space.data_ptr(), size, _status(status, device))
    return tokens, accepted


def _pools(k_pool, v_pool):
    _ask(k_pool.dim() == 5 and k_pool.shape == v_pool.shape and k_pool.dtype is v_pool.dtype and k_pool.dtype in _TYPES and k_pool.device == v_pool.device
         and k_pool.is_contiguous() and v_pool.is_contiguous(),
         "k_pool and v_pool are contiguous [layers, pages, kv heads, tokens of a page, head size] of one shape and type (float32, float16 or bfloat16)")
    layers, pages, heads, page, dim = k_pool.shape
    return k_pool.data_ptr(), v_pool.data_ptr(), layers, pages, heads, page, dim * k_pool.element_size()


def copy_pages(k_pool, v_pool, copies, *, status=None) -> None:
    """Copies the first ``rows`` tokens of pages to other pages, in every layer: copies [n, 3] of (from page, to page, rows).  No page is written twice, or
    written by one copy and read by another."""
    _ask(copies.dim() == 2 and copies.shape[1] == 3, "copies is [n, 3]: from page, to page, rows")
    device = k_pool.device
    _call(device, capi.lib().mk_k_copy_pages_dev, *_pools(k_pool, v_pool), _dense(copies, torch.int32, copies.shape, device, "copies"), copies.shape[0], _status(status, device))


def gather_tokens(k_pool, v_pool, from_tables, keep, counts, to_tables, first, *, status=None) -> None:
    """Moves kept tokens of lanes together, in every layer: token keep[i, j] of the pages from_tables[i] becomes token first[i] + j of the pages to_tables[i], for
    j < counts[i].  keep ascends; the tables name the same pages, or pages that nothing else here reads or writes."""
    _ask(from_tables.dim() == 2 and keep.dim() == 2 and to_tables.dim() == 2, "from_tables, keep and to_tables are [lanes, ...]")
    device, lanes = k_pool.device, keep.shape[0]
    tables = [(_index(t, (lanes, t.shape[1]), device, name), _row_stride(t), t.shape[1]) for t, name in ((from_tables, "from_tables"), (keep, "keep"), (to_tables, "to_tables"))]
    _call(device, capi.lib().mk_k_gather_tokens_dev, *_pools(k_pool, v_pool), *tables[0], *tables[1], _dense(counts, torch.int32, (lanes,), device, "counts"), *tables[2],
          _dense(first, torch.int32, (lanes,), device, "first"), lanes, _status(status, device))
