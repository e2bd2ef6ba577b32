"""The operators with which a frozen packed model answers token by token.

Every function hands raw device pointers to the C ABI (include/ue5m3_fp4.h) on the caller's current
CUDA stream, never synchronises and may be captured into a CUDA graph: sizes that live on the device
(lengths, settings per row) are read there.  They have no gradients.  None of them has a counterpart
in the reference, which evaluates frozen models by whole forward passes.
"""

from __future__ import annotations

import contextlib
import ctypes

import torch
from torch import Tensor

from ue5m3_fp4 import _native
from ue5m3_fp4.backends import b200

_HEAD_DIMS = (64, 128)
_PAGE_SIZES = (16, 32, 64, 128, 256)


def _on(device: torch.device):
    """The device of the operands as the current one, at no cost where it is already."""

    if device.index == torch.cuda.current_device():
        return contextlib.nullcontext()
    return torch.cuda.device(device)


def _require(condition: bool, message: str) -> None:
    if not condition:
        raise ValueError(message)


def _no_gradient(*tensors: Tensor | None) -> None:
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise RuntimeError("serving operators have no gradients; call them under torch.no_grad() or on detached tensors")


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


_factors: dict[tuple[float, float], float] = {}


def _cached_factor(tensor_amax: float, scale_target: float) -> float:
    key = (tensor_amax, scale_target)
    factor = _factors.get(key)
    if factor is None:
        if not (tensor_amax >= 0 and tensor_amax != float("inf")):
            raise ValueError("tensor_amax must be finite and not negative")
        if not 0 < scale_target < float("inf"):
            raise ValueError("scale_target must be positive and finite")
        if len(_factors) > 4096:
            _factors.clear()
        factor = _factors[key] = decode_factor(tensor_amax, scale_target)
    return factor


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
    contiguous.  The cost grows with every 32 rows of bf16 ``x`` (8 rows are read at the cost of one):
    for whole prompts use the GEMM."""

    b200._require_cuda(x, "x")
    _no_gradient(x, bias)
    device = x.device
    _require(block_size in (16, 32), "block_size must be 16 or 32")
    _require(x.ndim >= 1 and x.shape[-1] == cols, f"x must have {cols} columns")
    scale_rows = (rows + block_size - 1) // block_size if two_dimensional else rows
    _require(codes.dtype is torch.uint8 and tuple(codes.shape) == (rows, (cols + 1) // 2) and codes.is_contiguous()
             and codes.device == device, "codes must be contiguous uint8 [rows, ceil(cols/2)] on the operand's device")
    _require(scales.dtype is torch.uint8 and tuple(scales.shape) == (scale_rows, (cols + block_size - 1) // block_size)
             and scales.is_contiguous() and scales.device == device,
             "scales must be contiguous uint8 with one byte per block, on the operand's device")
    x_code = _native.dtype_code(x.dtype)
    out_dtype = out_dtype or x.dtype
    out_code = _native.dtype_code(out_dtype)
    bias_code = 0
    if bias is not None:
        bias_code = _native.dtype_code(bias.dtype)
        _require(tuple(bias.shape) == (rows,) and bias.is_contiguous() and bias.device == device,
                 "bias must be contiguous [rows] on the operand's device")
    factor = _cached_factor(float(tensor_amax), float(scale_target))
    shape = x.shape[:-1]
    flat = x if x.ndim == 2 else x.reshape(-1, cols)
    tokens = flat.shape[0]
    out = torch.empty((tokens, rows), dtype=out_dtype, device=device)
    if tokens == 0 or rows == 0:
        return out.view(*shape, rows)
    _require(cols > 0, "cols must be positive")
    ldx = flat.stride(0) if tokens > 1 else cols
    if (cols > 1 and flat.stride(1) != 1) or ldx < cols:
        raise ValueError("the last axis of x must be contiguous and its rows must not overlap")
    with _on(device):
        status = _native.load().ue5m3_packed_matvec(
            flat.data_ptr(), x_code, tokens, ldx, codes.data_ptr(), scales.data_ptr(), rows, cols, block_size,
            int(two_dimensional), factor, None if bias is None else bias.data_ptr(), bias_code, out.data_ptr(),
            out_code, rows, _native.stream_ptr(device))
    _native.check(status, "ue5m3_packed_matvec")
    return out if x.ndim == 2 else out.view(*shape, rows)


def _page_strides(pages: Tensor) -> tuple[int, int, int]:
    """Strides of page, slot and head; that of an axis with one element is immaterial."""

    contiguous = (pages.shape[1] * pages.shape[2] * pages.shape[3], pages.shape[2] * pages.shape[3], pages.shape[3])
    return tuple(pages.stride(i) if pages.shape[i] > 1 else contiguous[i] for i in range(3))


def _check_lengths(name: str, tensor: Tensor, count: int, device: torch.device) -> None:
    _require(tensor.dtype is torch.int32 and tensor.device == device and tuple(tensor.shape) == (count,)
             and tensor.is_contiguous(), f"{name} must be contiguous int32 [{count}] on the operand's device")


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

    b200._require_cuda(q, "q")
    _no_gradient(q, new_k, new_v, k_pages, v_pages)
    device = q.device
    _require(q.ndim == 3 and k_pages.ndim == 4 and v_pages.shape == k_pages.shape and page_table.ndim == 2,
             "q must be [tokens, heads, head_dim], the pages [pages, page_size, kv_heads, head_dim], the table rank 2")
    tokens, heads, head_dim = q.shape
    pages, page_size, kv_heads, _ = k_pages.shape
    sequences, width = page_table.shape
    for name, tensor in (("q", q), ("k_pages", k_pages), ("v_pages", v_pages)):
        _require(tensor.dtype is torch.bfloat16, f"{name} must be bfloat16")
        _require(tensor.device == device and tensor.shape[-1] == head_dim and tensor.stride(-1) == 1,
                 f"{name} must be on the operand's device with contiguous channels of q's width")
    _require(head_dim in _HEAD_DIMS, "head_dim must be 64 or 128")
    _require(page_size in _PAGE_SIZES, "page_size must be 16, 32, 64, 128 or 256")
    _require(kv_heads > 0 and heads % kv_heads == 0 and heads > 0, "heads must be a multiple of kv_heads")
    _require(page_table.dtype is torch.int32 and page_table.device == device
             and (width <= 1 or page_table.stride(1) == 1), "page_table must be int32 on the operand's device, rows contiguous")
    _check_lengths("kv_lengths", kv_lengths, sequences, device)
    _check_lengths("query_starts", query_starts, sequences + 1, device)
    _require(max_query_length > 0, "max_query_length must be positive")
    if scale is None:
        scale = head_dim ** -0.5
    _require(0 < scale < float("inf"), "scale must be positive and finite")
    if (new_k is None) != (new_v is None):
        raise ValueError("new_k and new_v come together")
    for name, tensor in (("new_k", new_k), ("new_v", new_v)):
        if tensor is not None:
            _require(tensor.dtype is torch.bfloat16 and tuple(tensor.shape) == (tokens, kv_heads, head_dim)
                     and tensor.device == device and tensor.stride(2) == 1,
                     f"{name} must be bfloat16 [tokens, kv_heads, head_dim] with contiguous channels")
    zero_tail = out is None
    if out is None:
        out = torch.empty((tokens, heads, head_dim), dtype=torch.bfloat16, device=device)
    else:
        _require(out.dtype is torch.bfloat16 and out.shape == q.shape and out.is_contiguous() and out.device == device,
                 "out must be contiguous bfloat16 of q's shape on its device")
    if tokens == 0:
        return out
    if sequences == 0:
        return out.zero_() if zero_tail else out
    _require(pages > 0 and width > 0, "the cache has no pages, or its table no columns")
    if max_kv_length is None:
        max_kv_length = width * page_size
    _require(max_kv_length > 0, "max_kv_length must be positive")
    k_strides, v_strides = _page_strides(k_pages), _page_strides(v_pages)
    for stride in (*k_strides, *v_strides, *(t.stride(i) for t in (q, new_k, new_v) if t is not None
                                             for i in range(2) if t.shape[i] > 1)):
        _require(stride % 8 == 0, "strides must be multiples of 8 elements")
    cache = _native.PagedCache(
        k_pages.data_ptr(), v_pages.data_ptr(), *k_strides, *v_strides, pages, page_size, kv_heads, head_dim,
        page_table.data_ptr(), sequences, width, page_table.stride(0) if sequences > 1 else width)
    lib = _native.load()
    max_query_length = min(int(max_query_length), tokens)
    max_kv_length = min(int(max_kv_length), width * page_size)
    with _on(device):
        need = lib.ue5m3_paged_attention_workspace_bytes(tokens, sequences, heads, kv_heads, head_dim, max_query_length,
                                                         max_kv_length)
        # from the current stream's pool, for this call alone: calls and captured graphs share nothing
        workspace = torch.empty(need, dtype=torch.uint8, device=device) if need else None
        strides = [(t.stride(0) if tokens > 1 else 0, t.stride(1) if t.shape[1] > 1 else 0) if t is not None else (0, 0)
                   for t in (q, new_k, new_v)]
        status = lib.ue5m3_paged_attention(
            q.data_ptr(), *strides[0], tokens, heads, ctypes.byref(cache), kv_lengths.data_ptr(),
            query_starts.data_ptr(), max_query_length, max_kv_length, float(scale),
            None if new_k is None else new_k.data_ptr(), *strides[1], None if new_v is None else new_v.data_ptr(),
            *strides[2], out.data_ptr(), int(zero_tail), None if workspace is None else workspace.data_ptr(), need,
            b200.gemm_status(device).data_ptr(), _native.stream_ptr(device))
    _native.check(status, "ue5m3_paged_attention")
    return out


def _setting(name: str, value, rows: int, dtype: torch.dtype, device: torch.device):
    """(device pointer or None, value) of a setting given as a number or as one number per row."""

    if isinstance(value, Tensor):
        _require(value.dtype is dtype and tuple(value.shape) == (rows,) and value.is_contiguous()
                 and value.device == device, f"{name} must be a number or a contiguous {dtype} tensor [rows]")
        return value.data_ptr(), 0
    return None, value


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
    number or a tensor with one per row (int32 for ``top_k``, fp32 otherwise).  Minus infinity masks a
    token; a row with a NaN, or with every token masked, gives token -1 and NaN.  Sums are exact: the
    same inputs give the same tokens, whatever the launch."""

    b200._require_cuda(logits, "logits")
    _no_gradient(logits)
    device = logits.device
    _require(logits.ndim == 2, "logits must be [rows, vocabulary]")
    rows, vocabulary = logits.shape
    code = _native.dtype_code(logits.dtype)
    _require(uniforms.dtype is torch.float32 and tuple(uniforms.shape) == (rows,) and uniforms.is_contiguous()
             and uniforms.device == device, "uniforms must be contiguous float32 [rows] on the operand's device")
    _require(0 < vocabulary <= 1 << 18, "the vocabulary must have between 1 and 2^18 tokens")
    _require(vocabulary == 1 or logits.stride(1) == 1, "the rows of logits must be contiguous")
    ld = logits.stride(0) if rows > 1 else vocabulary
    _require(ld >= vocabulary, "the rows of logits must not overlap")
    if not isinstance(temperature, Tensor):
        _require(temperature >= 0, "temperature must not be negative")
    if not isinstance(top_k, Tensor):
        _require(top_k >= 0, "top_k must not be negative")
        top_k = min(int(top_k), vocabulary)
    if not isinstance(top_p, Tensor):
        _require(0 < top_p <= 1, "top_p must be in (0, 1]")
    if not isinstance(min_p, Tensor):
        _require(0 <= min_p <= 1, "min_p must be in [0, 1]")
    heat = _setting("temperature", temperature, rows, torch.float32, device)
    k = _setting("top_k", top_k, rows, torch.int32, device)
    p = _setting("top_p", top_p, rows, torch.float32, device)
    least = _setting("min_p", min_p, rows, torch.float32, device)
    tokens = torch.empty(rows, dtype=torch.int64, device=device)
    logprobs = torch.empty(rows, dtype=torch.float32, device=device)
    if rows:
        with _on(device):
            status = _native.load().ue5m3_sample_tokens(
                logits.data_ptr(), code, rows, vocabulary, ld, uniforms.data_ptr(), *heat, *k, *p, *least,
                tokens.data_ptr(), logprobs.data_ptr(), _native.stream_ptr(device))
        _native.check(status, "ue5m3_sample_tokens")
    return tokens, logprobs


__all__ = ["packed_matvec", "paged_attention", "sample_tokens"]
