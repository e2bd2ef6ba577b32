"""The operators with which a frozen packed model answers token by token.

Every function hands raw device pointers to the C ABI (include/ue5m3_fp4.h) on the caller's current
CUDA stream, never synchronises and may be captured into a CUDA graph: sizes that live on the device
(lengths, settings per row) are read there.  They have no gradients.  None of them has a counterpart
in the reference, which evaluates frozen models by whole forward passes.
"""

from __future__ import annotations

import ctypes
import functools

import torch
from torch import Tensor

from ue5m3_fp4 import _native
from ue5m3_fp4.backends import b200

_PAGE_SIZES = (16, 32, 64, 128, 256)
_BF16 = torch.bfloat16


def _require_cuda(tensor: Tensor, name: str) -> None:
    if not isinstance(tensor, Tensor) or not tensor.is_cuda:
        b200._require_cuda(tensor, name)


def _no_gradient(*tensors: Tensor | None) -> None:
    if torch.is_grad_enabled():
        for tensor in tensors:
            if tensor is not None and tensor.requires_grad:
                raise RuntimeError("serving operators have no gradients; call them under torch.no_grad() or on "
                                   "detached tensors")


def _call(function, name: str, launches: int, index: int, *arguments) -> None:
    """The library call on the current stream of the device ``index``, with that device current."""

    if index == torch._C._cuda_getDevice():
        status = function(*arguments, _native.raw_stream(index))
    else:
        with torch.cuda.device(index):
            status = function(*arguments, _native.raw_stream(index))
    _native.check(status, name, launches)


def decode_factor(tensor_amax: float, scale_target: float) -> float:
    """The tensor-scale decode factor in the quantizer's own fp32 steps: 1 / min(fl(6T) / amax, FLT_MAX), and 1
    where amax is 0 (formats.py:394-408 of the reference)."""

    import numpy as np

    amax, six_t = np.float32(tensor_amax), np.float32(6.0 * scale_target)
    if amax == 0:
        return 1.0
    with np.errstate(over="ignore", divide="ignore"):
        encode = min(six_t / amax, np.finfo(np.float32).max)
        return 1.0 if encode == 0 else float(np.float32(1.0) / np.float32(encode))


@functools.lru_cache(maxsize=4096)
def _matvec_workspace_bytes(*sizes: int) -> int:
    return _native.load().ue5m3_packed_matvec_workspace_bytes(*sizes)


@functools.lru_cache(maxsize=4096)
def _checked_factor(tensor_amax: float, scale_target: float) -> float:
    if not 0 <= tensor_amax < float("inf"):
        raise ValueError("tensor_amax must be finite and not negative")
    if not 0 < scale_target < float("inf"):
        raise ValueError("scale_target must be positive and finite")
    return decode_factor(tensor_amax, scale_target)


def packed_matvec(
    x: Tensor,
    codes: Tensor,
    scales: Tensor,
    *,
    rows: int,
    cols: int,
    block_size: int,
    two_dimensional: bool,
    tensor_amax: float,
    scale_target: float = 448.0,
    bias: Tensor | None = None,
    out_dtype: torch.dtype | None = None,
) -> Tensor:
    """``x [..., cols] @ W.T + bias`` with a packed weight W [rows, cols] (E2M1 ``codes`` and UE5M3
    ``scales`` as ``quantize_packed`` and ``PackedFP4Tensor`` hold them) for a few rows of bf16 or
    fp32 activations, which are not quantized.  Sums are fp32; the result is rounded once, to
    ``out_dtype`` (default: that of ``x``).  Any ``rows`` and ``cols``; the last axis of ``x`` must be
    contiguous.  Eight rows are read at the cost of one; the weight is read and decoded once for every 64 rows
    of bf16 ``x`` and every 32 of fp32, so that whole prompts run at no more than about 250 TFLOP/s.
    At most 2^24 rows of ``x``, 2^30 ``rows`` and 2^22 ``cols``."""

    _require_cuda(x, "x")
    _no_gradient(x, bias)
    index = x.get_device()  # the operands' devices are compared by number: device objects cost host time
    if block_size != 16 and block_size != 32:
        raise ValueError("block_size must be 16 or 32")
    if x.ndim == 0 or x.shape[-1] != cols or cols <= 0:
        raise ValueError(f"x must have {cols} columns, at least one")
    scale_rows = (rows + block_size - 1) // block_size if two_dimensional else rows
    if (codes.dtype is not torch.uint8 or codes.shape != (rows, (cols + 1) // 2) or not codes.is_contiguous()
            or codes.get_device() != index):
        raise ValueError("codes must be contiguous uint8 [rows, ceil(cols/2)] on the operand's device")
    if (scales.dtype is not torch.uint8 or scales.shape != (scale_rows, (cols + block_size - 1) // block_size)
            or not scales.is_contiguous() or scales.get_device() != index):
        raise ValueError("scales must be contiguous uint8 with one byte per block, on the operand's device")
    x_code = _native.dtype_code(x.dtype)
    if out_dtype is None:
        out_dtype, out_code = x.dtype, x_code
    else:
        out_code = _native.dtype_code(out_dtype)
    bias_code, bias_pointer = 0, None
    if bias is not None:
        if bias.shape != (rows,) or not bias.is_contiguous() or bias.get_device() != index:
            raise ValueError("bias must be contiguous [rows] on the operand's device")
        bias_code, bias_pointer = _native.dtype_code(bias.dtype), bias.data_ptr()
    factor = _checked_factor(float(tensor_amax), float(scale_target))
    flat = x if x.ndim == 2 else x.reshape(-1, cols)
    tokens = flat.shape[0]
    out = x.new_empty((tokens, rows), dtype=out_dtype)
    if tokens and rows:
        ldx, step = flat.stride()
        if tokens == 1:
            ldx = cols
        if (step != 1 and cols > 1) or ldx < cols:
            raise ValueError("the last axis of x must be contiguous and its rows must not overlap")
        # more than eight rows: prepared once, in memory of the current stream's pool for this call alone
        library = _native.load()
        need = _matvec_workspace_bytes(x_code, tokens, cols) if tokens > 8 else 0
        workspace = x.new_empty(need, dtype=torch.uint8) if need else None
        _call(library.ue5m3_packed_matvec, "ue5m3_packed_matvec", 2 if need else 1, index, flat.data_ptr(), x_code, tokens, ldx,
              codes.data_ptr(), scales.data_ptr(), rows, cols, block_size, two_dimensional, factor, bias_pointer,
              bias_code, out.data_ptr(), out_code, rows, None if workspace is None else workspace.data_ptr(), need)
    return out if x.ndim == 2 else out.view(*x.shape[:-1], rows)


def _strides(name: str, tensor: Tensor) -> tuple[int, ...]:
    """Strides of all axes but the channels', for the library: that of an axis with one element is immaterial."""

    if tensor.is_contiguous():  # channels are 64 or 128: every stride is a multiple of 8
        shape = tensor.shape
        row = shape[-2] * shape[-1]
        return (row, shape[-1]) if len(shape) == 3 else (shape[1] * row, row, shape[-1])
    strides = tensor.stride()
    if strides[-1] != 1:
        raise ValueError(f"{name} must have contiguous channels")
    if tensor.ndim == 4 and any(stride == 0 and size > 1 for size, stride in zip(tensor.shape, strides)):
        raise ValueError(f"{name} must not be expanded: every key and value has a place of its own")
    if 1 in tensor.shape[:-1]:
        strides = tuple(0 if size == 1 else stride for size, stride in zip(tensor.shape, strides))
        if tensor.ndim == 4:  # the tensor map of the pages takes no zero strides
            shape = tensor.shape
            dense = (shape[1] * shape[2] * shape[3], shape[2] * shape[3], shape[3])
            strides = tuple(stride or full for stride, full in zip(strides, dense))
    for stride in strides[:tensor.ndim - 1]:
        if stride % 8 or stride < 0:
            raise ValueError(f"the strides of {name} must be multiples of 8 elements")
    return strides[:tensor.ndim - 1]


@functools.lru_cache(maxsize=4096)
def _workspace_bytes(index: int, *sizes: int) -> int:
    """Asked for once per device and sizes: into how many parts sequences are split depends on the device's SMs."""

    function = _native.load().ue5m3_paged_attention_workspace_bytes
    if index == torch._C._cuda_getDevice():
        return function(*sizes)
    with torch.cuda.device(index):
        return function(*sizes)


def paged_attention(
    q: Tensor,
    k_pages: Tensor,
    v_pages: Tensor,
    page_table: Tensor,
    kv_lengths: Tensor,
    query_starts: Tensor,
    *,
    max_query_length: int,
    max_kv_length: int | None = None,
    scale: float | None = None,
    new_k: Tensor | None = None,
    new_v: Tensor | None = None,
    out: Tensor | None = None,
) -> Tensor:
    """Attention of a chunk of new tokens per sequence over a paged key/value cache.

    ``q`` bf16 [tokens, heads, head_dim] holds the new tokens of all sequences one behind the other,
    those of sequence b in rows ``query_starts[b] : query_starts[b + 1]`` (int32 [sequences + 1]).
    ``k_pages`` / ``v_pages`` bf16 [pages, page_size, kv_heads, head_dim]; entry j of row b of
    ``page_table`` (int32 [sequences, width]) is the page of that sequence's keys ``j * page_size``
    onwards; entries behind its last page are not looked at.  ``kv_lengths`` (int32 [sequences])
    counts a sequence's keys with the new tokens' own: of L keys and n new tokens, token i sees keys
    ``0 ... L - n + i``, and gets zeros where that is none.  ``new_k`` / ``new_v`` [tokens, kv_heads,
    head_dim], when given, are first written to the new tokens' places in the pages.

    ``max_query_length`` and ``max_kv_length`` are bounds from which the launch is sized (default for
    the latter: what the table has room for); larger actual lengths are right, only slower.  Rows of
    ``q`` behind the last sequence are padding: the result is zero there, or, with ``out`` given, as
    ``out`` was.  A page outside the cache is not touched; rows that need it are NaN.
    head_dim is 64 or 128, page_size 16, 32, 64, 128 or 256; heads is a multiple of kv_heads."""

    _require_cuda(q, "q")
    _no_gradient(q, new_k, new_v, k_pages, v_pages)
    index = q.get_device()
    if q.ndim != 3 or k_pages.ndim != 4 or page_table.ndim != 2 or v_pages.shape != k_pages.shape:
        raise ValueError("q must be [tokens, heads, head_dim], the pages [pages, page_size, kv_heads, head_dim], the "
                         "table rank 2")
    tokens, heads, head_dim = q.shape
    pages, page_size, kv_heads, width = k_pages.shape
    if q.dtype is not _BF16 or k_pages.dtype is not _BF16 or v_pages.dtype is not _BF16:
        raise ValueError("q, k_pages and v_pages must be bfloat16")
    if k_pages.get_device() != index or v_pages.get_device() != index or page_table.get_device() != index:
        raise ValueError("the cache must be on the operand's device")
    if head_dim != width or (head_dim != 64 and head_dim != 128):
        raise ValueError("head_dim must be 64 or 128, and that of the pages")
    if page_size not in _PAGE_SIZES:
        raise ValueError("page_size must be 16, 32, 64, 128 or 256")
    if kv_heads == 0 or heads == 0 or heads % kv_heads:
        raise ValueError("heads must be a multiple of kv_heads")
    sequences, width = page_table.shape
    table_stride, step = page_table.stride()
    if page_table.dtype is not torch.int32 or (step != 1 and width > 1) or (table_stride < width and sequences > 1):
        raise ValueError("page_table must be int32 with contiguous rows")
    if (kv_lengths.dtype is not torch.int32 or kv_lengths.shape != (sequences,) or kv_lengths.get_device() != index
            or not kv_lengths.is_contiguous()):
        raise ValueError("kv_lengths must be contiguous int32 [sequences] on the operand's device")
    if (query_starts.dtype is not torch.int32 or query_starts.shape != (sequences + 1,) or query_starts.get_device() != index
            or not query_starts.is_contiguous()):
        raise ValueError("query_starts must be contiguous int32 [sequences + 1] on the operand's device")
    if max_query_length <= 0 or (max_kv_length is not None and max_kv_length <= 0):
        raise ValueError("max_query_length and max_kv_length must be positive")
    if scale is None:
        scale = head_dim ** -0.5
    elif not 0 < scale <= 2.0 ** 126:  # times log2(e), in fp32
        raise ValueError("scale must be positive and no larger than 2^126")
    zero_tail = out is None
    if zero_tail:
        out = q.new_empty((tokens, heads, head_dim))
    elif out.dtype is not _BF16 or out.shape != q.shape or not out.is_contiguous() or out.get_device() != index:
        raise ValueError("out must be contiguous bfloat16 of q's shape on its device")
    k_pointer = v_pointer = None
    k_strides = v_strides = (0, 0)
    if new_k is not None or new_v is not None:
        if new_k is None or new_v is None:
            raise ValueError("new_k and new_v come together")
        for name, tensor in (("new_k", new_k), ("new_v", new_v)):
            if tensor.dtype is not _BF16 or tensor.shape != (tokens, kv_heads, head_dim) or tensor.get_device() != index:
                raise ValueError(f"{name} must be bfloat16 [tokens, kv_heads, head_dim] on the operand's device")
        k_pointer, v_pointer = new_k.data_ptr(), new_v.data_ptr()
        k_strides, v_strides = _strides("new_k", new_k), _strides("new_v", new_v)
    if tokens == 0:
        return out
    if sequences == 0:
        return out.zero_() if zero_tail else out
    if pages == 0 or width == 0:
        raise ValueError("the cache has no pages, or its table no columns")
    room = width * page_size
    max_kv_length = room if max_kv_length is None else min(int(max_kv_length), room)
    max_query_length = min(int(max_query_length), tokens)
    cache = _native.PagedCache(
        k_pages.data_ptr(), v_pages.data_ptr(), *_strides("k_pages", k_pages), *_strides("v_pages", v_pages), pages,
        page_size, kv_heads, head_dim, page_table.data_ptr(), sequences, width,
        table_stride if sequences > 1 else width)
    need = _workspace_bytes(index, tokens, sequences, heads, kv_heads, head_dim, max_query_length, max_kv_length)
    # from the current stream's pool, for this call alone: calls and captured graphs share nothing
    workspace = q.new_empty(need // 2) if need else None
    # kernels: attention, the rows of split sequences, new keys ahead of the kernel for many rows
    launches = 1 + (need > 0) + (k_pointer is not None and max_query_length * (heads // kv_heads) > 32)
    _call(_native.load().ue5m3_paged_attention, "ue5m3_paged_attention", launches, index, q.data_ptr(),
          *_strides("q", q), tokens, heads, ctypes.byref(cache), kv_lengths.data_ptr(), query_starts.data_ptr(),
          max_query_length, max_kv_length, scale, k_pointer, *k_strides, v_pointer, *v_strides, out.data_ptr(),
          zero_tail, None if workspace is None else workspace.data_ptr(), need, b200.gemm_status(q.device).data_ptr())
    return out


def _setting(name: str, value, rows: int, dtype: torch.dtype, index: int):
    """(device pointer or None, value) of a setting given as a number or as one number per row."""

    if not isinstance(value, Tensor):
        return None, value
    if value.dtype is not dtype or value.shape != (rows,) or not value.is_contiguous() or value.get_device() != index:
        raise ValueError(f"{name} must be a number or a contiguous {dtype} tensor [rows] on the operand's device")
    return value.data_ptr(), 0


def sample_tokens(
    logits: Tensor,
    uniforms: Tensor,
    *,
    temperature: float | Tensor = 1.0,
    top_k: int | Tensor = 0,
    top_p: float | Tensor = 1.0,
    min_p: float | Tensor = 0.0,
) -> tuple[Tensor, Tensor]:
    """The next token (int64) of every row of ``logits`` [rows, vocabulary] (bf16 or fp32) and the log
    of its probability (fp32) under the distribution it was drawn from, from one uniform number of
    [0, 1) per row (``uniforms``, fp32 [rows]).

    With weights exp((l - max) / temperature), kept are the ``top_k`` largest (equal logits: lowest
    index first; 0: all), of these the shortest prefix in descending order whose weight reaches
    ``top_p`` of theirs (1: all), of these the tokens with at least ``min_p`` of the largest weight.
    The token is the first kept one, in vocabulary order, whose running weight exceeds
    ``uniform * (weight of all kept)``.  temperature 0 takes the largest logit.  Each setting is a
    number or a tensor with one per row (int32 for ``top_k``, fp32 otherwise; there a value outside its
    range counts as the nearest in it, a NaN ``temperature`` as 0, a NaN ``top_p`` or ``min_p`` as none, and a NaN
    in ``uniforms`` as 0).  Minus infinity masks a
    token; a row with a NaN, or with every token masked, gives token -1 and NaN.  Sums are exact: the
    same inputs give the same tokens, whatever the launch."""

    _require_cuda(logits, "logits")
    _no_gradient(logits)
    index = logits.get_device()
    if logits.ndim != 2:
        raise ValueError("logits must be [rows, vocabulary]")
    rows, vocabulary = logits.shape
    code = _native.dtype_code(logits.dtype)
    if (uniforms.dtype is not torch.float32 or uniforms.shape != (rows,) or not uniforms.is_contiguous()
            or uniforms.get_device() != index):
        raise ValueError("uniforms must be contiguous float32 [rows] on the operand's device")
    if not 0 < vocabulary <= 1 << 18:
        raise ValueError("the vocabulary must have between 1 and 2^18 tokens")
    ld, step = logits.stride()
    if rows <= 1:
        ld = vocabulary
    if (step != 1 and vocabulary > 1) or ld < vocabulary:
        raise ValueError("the rows of logits must be contiguous and must not overlap")
    heat = _setting("temperature", temperature, rows, torch.float32, index)
    k = _setting("top_k", top_k, rows, torch.int32, index)
    p = _setting("top_p", top_p, rows, torch.float32, index)
    least = _setting("min_p", min_p, rows, torch.float32, index)
    if not heat[1] >= 0:
        raise ValueError("temperature must not be negative")
    if not k[1] >= 0:
        raise ValueError("top_k must not be negative")
    if p[0] is None and not 0 < p[1] <= 1:
        raise ValueError("top_p must be in (0, 1]")
    if not 0 <= least[1] <= 1:
        raise ValueError("min_p must be in [0, 1]")
    if k[1] > vocabulary:
        k = (None, vocabulary)
    tokens = uniforms.new_empty(rows, dtype=torch.int64)
    logprobs = uniforms.new_empty(rows)
    if rows:
        _call(_native.load().ue5m3_sample_tokens, "ue5m3_sample_tokens", 1, index, logits.data_ptr(), code, rows,
              vocabulary, ld, uniforms.data_ptr(), *heat, *k, *p, *least, tokens.data_ptr(), logprobs.data_ptr())
    return tokens, logprobs


__all__ = ["packed_matvec", "paged_attention", "sample_tokens"]
