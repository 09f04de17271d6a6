"""Operators over tensors in device memory (the mk_k_*_dev entry points), for serving many continuations of one prompt, for caches of keys and values
in 4 or 8 bits, and for scoring given tokens.

Unlike the wrappers of ``ops``, which move host arrays to the device and back, these take CUDA tensors as they are, enqueue their kernels on
the current stream of the tensors' device and return without waiting; they may be captured into a CUDA graph (sizes, pointers, Python
numbers and strides are fixed then, contents are not).  Index tensors are int32.  ``status`` is an optional int32 tensor of one element into
which the kernels OR what they met (``BAD_PAGE``, ``WAIT_GAVE_UP``, ``BAD_RANGE``, ``BAD_ROW``); ``check_status`` reads it.  Arguments that can be judged by shape, type and
stride are refused with ValueError before anything is launched, what the entry points themselves refuse (a head size, a length, an alignment, rows that overlap) with MkError, also before.
"""
from __future__ import annotations

import ctypes as C
import functools
from typing import NamedTuple

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


def _int(n: int, what: str) -> int:
    """n as the entry points take it: a larger number would lose its upper bits on the way."""
    if n > 0x7fffffff:
        raise ValueError(f"{what} is at most 2^31 - 1: got {n}")
    return n


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
    need = _attention_workspace(heads, kv_heads, dim, page, width, lanes, _int(rows, "max_rows"), total, _int(shared_len, "shared_len"), _int(window, "window"))
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
    if (len(shape) != 5 or v_pool.shape != shape or v_pool.dtype is not dtype or (dtype not in _TYPES and dtype is not torch.uint8) or v_pool.get_device() != k_pool.get_device()
            or not k_pool.is_contiguous() or not v_pool.is_contiguous()):
        raise ValueError("k_pool and v_pool are contiguous [layers, pages, kv heads, tokens of a page, head size] of one shape and type (float32, float16, bfloat16, or uint8 for codes), on one device")
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


# ---- caches in 4 or 8 bits -----------------------------------------------------------------------------------------------------------------------------------------

_GROUP = 64


class QuantizedPools(NamedTuple):
    """One layer's keys and values in 4 or 8 bits: codes [pages, kv_heads, block_tokens, head_dim * bits / 8] uint8 (the lower four bits of a byte come first), and for each
    group of 64 neighbouring values of a row a pair (step, lowest value) [pages, kv_heads, block_tokens, head_dim / 64, 2] of the rows' type; code c stands for
    lowest + step * c.  Where a call takes pools, any tuple of four such tensors will do; pages may be further apart than they are long, all at the same distances."""
    k_codes: torch.Tensor
    v_codes: torch.Tensor
    k_scales: torch.Tensor
    v_scales: torch.Tensor


def quantized_pools(pages: int, kv_heads: int, block_tokens: int, head_dim: int, *, bits: int = 4, dtype=torch.float16, device="cuda") -> QuantizedPools:
    """Empty pools for one layer, of 4.5 or 8.5 bits a value."""
    if bits not in (4, 8) or head_dim not in (64, 128, 256) or dtype not in (torch.float16, torch.bfloat16):
        raise ValueError("a cache has 4 or 8 bits, heads of 64, 128 or 256 values and float16 or bfloat16 rows")
    codes = [torch.zeros(pages, kv_heads, block_tokens, head_dim * bits // 8, dtype=torch.uint8, device=device) for _ in range(2)]
    scales = [torch.zeros(pages, kv_heads, block_tokens, head_dim // _GROUP, 2, dtype=dtype, device=device) for _ in range(2)]
    return QuantizedPools(*codes, *scales)


def _quantized(pools, device):
    """The pools' arguments of an entry point; head size, type and KV heads beside them."""
    k_codes, v_codes, k_scales, v_scales = pools
    shape, of_scales, dtype = k_codes.shape, k_scales.shape, k_scales.dtype
    if len(shape) != 4 or len(of_scales) != 5 or of_scales[:3] != shape[:3] or of_scales[4] != 2 or (dtype is not torch.float16 and dtype is not torch.bfloat16):
        raise ValueError("pools are codes [pages, kv heads, tokens of a page, bytes] and scales [pages, kv heads, tokens of a page, groups, 2], float16 or bfloat16")
    pages, heads, page, row = shape
    groups = of_scales[3]
    dim = groups * _GROUP
    if (v_codes.shape != shape or v_scales.shape != of_scales or k_codes.dtype is not torch.uint8 or v_codes.dtype is not torch.uint8 or v_scales.dtype is not dtype
            or (2 * row != dim and row != dim) or not k_codes.get_device() == v_codes.get_device() == k_scales.get_device() == v_scales.get_device() == device):
        raise ValueError("codes are uint8, half a byte or a byte for each value of 64 to a scale, keys and values alike, on the device of the others")
    strides, of_strides = k_codes.stride(), k_scales.stride()
    if v_codes.stride() != strides or v_scales.stride() != of_strides or strides[1:] != (page * row, row, 1) or of_strides[1:] != (page * groups * 2, groups * 2, 2, 1):
        # a dimension of one element may have any stride
        if pages > 1 and (v_codes.stride(0) != strides[0] or v_scales.stride(0) != of_strides[0]):
            raise ValueError("pages of keys and of values are equally far apart")
        if pages and not (k_codes[0].is_contiguous() and v_codes[0].is_contiguous() and k_scales[0].is_contiguous() and v_scales[0].is_contiguous()):
            raise ValueError("pages are dense")
    return dim, dtype, heads, (_TYPES[dtype], 8 * row // dim, k_codes.data_ptr(), v_codes.data_ptr(), k_scales.data_ptr(), v_scales.data_ptr(), pages,
                               strides[0] if pages > 1 else heads * page * row, of_strides[0] if pages > 1 else heads * page * groups * 2, heads, dim, page)


def _lanes(tables, lengths, cu_seqlens, device):
    lanes = tables.shape[0] if tables.dim() == 2 else -1
    return lanes, (*_rows(tables, lanes, device, "tables"), _dense(lengths, _I32, (lanes,), device, "lengths"),
                   None if cu_seqlens is None else _dense(cu_seqlens, _I32, (lanes + 1,), device, "cu_seqlens"), lanes)


def _head_rows(t, shape, dtype, device, what: str):
    """Address and strides of rows [total, kv heads, head size] whose heads are dense."""
    if t.shape != shape or t.dtype is not dtype or t.get_device() != device or (t.stride()[2] != 1 and shape[0]):
        raise ValueError(f"{what} is a {dtype} tensor of shape {tuple(shape)} with dense heads on the device of the others: got {t.dtype} {tuple(t.shape)} on {t.device}")
    row, head, _ = t.stride()
    return t.data_ptr(), row if shape[0] > 1 else shape[1] * shape[2], head if shape[1] > 1 else shape[2]


def _word(status, device):
    return None if status is None else _dense(status, _I32, (1,), device, "status")


def quantize_rows(k, v, pools, tables, lengths, *, cu_seqlens=None, status=None) -> None:
    """Writes rows of keys and values [total, kv_heads, head_dim] into the pages of ``pools``, as codes and scales.

    tables [lanes, width] page numbers; lengths [lanes] tokens of each lane, the last of which are its rows (cu_seqlens [lanes + 1], or total / lanes rows each): rows and
    heads may be strided.  Rows in front of a lane's first token are left out.  A group with a value that is not finite reads as NaN."""
    device = k.get_device()
    dim, dtype, heads, cache = _quantized(pools, device)
    _, where = _lanes(tables, lengths, cu_seqlens, device)
    shape = (_int(k.shape[0], "the number of rows") if k.dim() else 0, heads, dim)
    _run(device, capi.lib().mk_k_quantize_rows_dev, *_head_rows(k, shape, dtype, device, "k"), *_head_rows(v, shape, dtype, device, "v"), *cache, *where, shape[0],
         _word(status, device))


def dequantize_rows(pools, tables, lengths, total: int, *, cu_seqlens=None, k=None, v=None, status=None):
    """Reads the tokens that ``quantize_rows`` with the same tables, lengths and cu_seqlens writes back into rows.

    Returns (k, v) [total, kv_heads, head_dim] of the scales' type.  Rows in front of a lane's first token are zeros, and rows outside cu_seqlens left as ``k`` and ``v`` had them."""
    device = pools[0].get_device()
    dim, dtype, heads, cache = _quantized(pools, device)
    _, where = _lanes(tables, lengths, cu_seqlens, device)
    if total < 0:
        raise ValueError("total is not negative")
    shape, row = (_int(total, "total"), heads, dim), heads * dim
    if k is None and v is None:
        k, v = pools[2].new_empty((2, total, heads, dim)).unbind()
        to_k, to_v = (k.data_ptr(), row, dim), (v.data_ptr(), row, dim)
    else:
        if k is None:
            k = pools[2].new_empty(shape)
        if v is None:
            v = pools[2].new_empty(shape)
        to_k, to_v = _head_rows(k, shape, dtype, device, "k"), _head_rows(v, shape, dtype, device, "v")
    _run(device, capi.lib().mk_k_dequantize_rows_dev, *cache, *where, total, *to_k, *to_v, _word(status, device))
    return k, v


@functools.lru_cache(maxsize=4096)
def _quantized_workspace(*sizes) -> int:
    need = C.c_int64()
    capi.check(capi.lib().mk_k_quantized_attention_workspace(*sizes, C.byref(need)))
    return need.value


def quantized_attention(q, pools, tables, lengths, *, scale: float, cu_seqlens=None, max_rows: int = 0, softcap: float = 0.0, window: int = 0, out=None, status=None):
    """Attention of a ragged batch over a cache in 4 or 8 bits, read as it is.

    q [total, q_heads, head_dim] of the scales' type; tables, lengths, cu_seqlens and ``max_rows`` as of ``shared_attention``: a lane's rows are the last of its tokens, whose
    keys and values are in the pages already.  Pages wholly in front of every row's window need not be there.  Returns [total, q_heads, head_dim]; a row that sees nothing becomes zeros,
    rows outside cu_seqlens are left as ``out`` had them."""
    device, shape = q.get_device(), q.shape
    dim, dtype, _, cache = _quantized(pools, device)
    if len(shape) != 3 or q.dtype is not dtype or shape[2] != dim:
        raise ValueError(f"q is a {dtype} tensor [rows, heads, {dim}], as the pools are")
    total, heads, _ = shape
    lanes, where = _lanes(tables, lengths, cu_seqlens, device)
    if cu_seqlens is None:
        rows = total // lanes if lanes else 0
        if rows * lanes != total:
            raise ValueError("without cu_seqlens every lane has the same number of rows")
    else:
        rows = max_rows
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
    need = _quantized_workspace(cache[1], heads, *cache[9:], where[2], lanes, _int(rows, "max_rows"), total, _int(window, "window"))
    space = q.new_empty(need // 2) if need else None
    _run(device, capi.lib().mk_k_quantized_attention_dev, q.data_ptr(), q_strides[0] if total > 1 else heads * dim, heads, *cache, *where, rows, total, scale, softcap, window,
         out.data_ptr(), out_stride, space.data_ptr() if need else None, need, _word(status, device))
    return out


# ---- scoring -------------------------------------------------------------------------------------------------------------------------------------------------------


class TokenLogprobs(NamedTuple):
    logprobs: torch.Tensor       # [rows] f32
    entropy: torch.Tensor        # [rows] f32
    ranks: torch.Tensor          # [rows] int32, 1 is the likeliest
    top_tokens: torch.Tensor     # [rows, top] int32
    top_logprobs: torch.Tensor   # [rows, top] f32


def token_logprobs(logits, tokens, *, top: int = 0, status=None) -> TokenLogprobs:
    """Log probabilities (natural) of given tokens, with the entropy of their distributions, their ranks and the ``top`` likeliest tokens, at most 64.

    logits [rows, vocab] f32, f16 or bf16 (rows may be further apart; -inf is a token that cannot be); tokens [rows] int32.  Equal logits are ranked by rising token.  A
    negative token asks for none (log probability 0, rank 0), one beyond the vocabulary gets NaN and BAD_RANGE; a row that is no distribution NaN, rank 0, tokens -1 and BAD_ROW."""
    dtype, device, shape = logits.dtype, logits.get_device(), logits.shape
    if len(shape) != 2 or dtype not in _TYPES or shape[1] < 1:
        raise ValueError("logits is a float32, float16 or bfloat16 tensor [rows, vocabulary]")
    rows, vocab = shape
    strides = logits.stride()
    if rows and vocab > 1 and strides[1] != 1:
        raise ValueError("rows of logits are dense")
    given = _dense(tokens, _I32, (rows,), device, "tokens")
    if not 0 <= top <= min(64, vocab):
        raise ValueError("top is at most 64 and at most the vocabulary")
    likeliest = (rows, top)
    out = TokenLogprobs(torch.empty_like(tokens, dtype=_F32), torch.empty_like(tokens, dtype=_F32), torch.empty_like(tokens), tokens.new_empty(likeliest), tokens.new_empty(likeliest, dtype=_F32))
    logprobs, entropy, ranks, top_tokens, top_logprobs = out
    _run(device, capi.lib().mk_k_token_logprobs_dev, _TYPES[dtype], logits.data_ptr(), strides[0] if rows > 1 else vocab, rows, vocab, given, top, logprobs.data_ptr(),
         entropy.data_ptr(), ranks.data_ptr(), top_tokens.data_ptr(), top_logprobs.data_ptr(), _word(status, device))
    return out
