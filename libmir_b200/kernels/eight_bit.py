"""Launchers of the operators for serving in 8 bits (csrc/store_8bit.cu, attention_8bit*.cu, linear_8bit*.cu).

The 8-bit cache holds e4m3 numbers (torch.float8_e4m3fn) in pages, [pages * page_size, kv_heads, head_dim], and one float32
scale per page and kv head for the keys and one for the values, [pages, kv_heads], powers of two: an element stands for its
number times its page's scale.  store_kv_8bit writes it, decode_attention_8bit and prefill_attention_8bit read it; they stand
beside qk_rope_store, decode_attention and prefill_attention over pages of the activations' dtype.  linear_8bit stands beside
linear.  All of them run on torch's current stream and device, on tensors of that device."""

from __future__ import annotations

import ctypes
from typing import Callable, Optional

import torch

from ..errors import KernelError
from . import _check, _ptr, _raw_device, _stream, library

E4M3 = torch.float8_e4m3fn
BLOCK = 128                 # rows and columns of a weight that share a scale, and columns of a row of activations
MOST_KEYS = (1 << 31) - 256      # of a context, as 32-bit positions have it


# (The checks run at every call: conditions are tested in place and messages put together only where one fails.)
def _on_this_device(what: str, *tensors) -> None:
    here = _current_device()
    for tensor in tensors:
        if tensor is not None and tensor.get_device() != here:
            if not tensor.is_cuda:
                raise KernelError("kernels take CUDA tensors only: there is no CPU path")
            raise KernelError(f"{what}: a tensor is on {tensor.device}, the current device is cuda:{here}")


def _current_device() -> int:
    return _raw_device() if _raw_device is not None and torch.cuda.is_initialized() else (
        torch.cuda.current_device() if torch.cuda.is_available() else 0)


def _cache(what: str, k_pages, v_pages, k_scales, v_scales, page_size: int, kv_heads: int, head_dim: int) -> int:
    """Checks the four tensors of an 8-bit cache; how many pages it has."""
    if page_size <= 0 or kv_heads <= 0 or head_dim not in (64, 128):
        raise KernelError(f"{what}: takes head_dim 64 or 128, got {head_dim} (page {page_size}, {kv_heads} kv heads)")
    shape = k_pages.shape
    if not (len(shape) == 3 and shape[1] == kv_heads and shape[2] == head_dim and v_pages.shape == shape and shape[0] > 0
            and shape[0] % page_size == 0 and k_pages.dtype is E4M3 and v_pages.dtype is E4M3 and k_pages.is_contiguous()
            and v_pages.is_contiguous()):
        raise KernelError(f"{what}: the pages are contiguous float8_e4m3fn [pages * {page_size}, {kv_heads}, {head_dim}]")
    pages = shape[0] // page_size
    shape = k_scales.shape
    if not (len(shape) == 2 and shape[0] == pages and shape[1] == kv_heads and v_scales.shape == shape and k_scales.dtype is torch.float32
            and v_scales.dtype is torch.float32 and k_scales.is_contiguous() and v_scales.is_contiguous()):
        raise KernelError(f"{what}: the scales are contiguous float32 [{pages}, {kv_heads}]")
    return pages


def _attention(what: str, qkv, out, block_table, heads: int, kv_heads: int, head_dim: int, rows: int, sinks, scratch) -> None:
    if heads <= 0 or heads % kv_heads:
        raise KernelError(f"{what}: {heads} heads do not divide over {kv_heads} kv heads")
    width, given, result = heads * head_dim, qkv.shape, out.shape
    if not (qkv.dtype is torch.bfloat16 and out.dtype is torch.bfloat16 and len(given) == 2 and len(result) == 2 and given[1] >= width
            and result[1] == width and given[0] >= result[0] and qkv.stride(1) == 1 and out.is_contiguous()):
        raise KernelError(f"{what}: bfloat16 rows that begin with {heads} heads of {head_dim} are needed, and out [rows, heads * head_dim]")
    table = block_table.shape
    if not (block_table.dtype is torch.int32 and len(table) == 2 and table[0] >= rows and (table[1] > 0 or rows == 0)
            and block_table.is_contiguous()):
        raise KernelError(f"{what}: the block table is contiguous int32 [rows, blocks]")
    if sinks is not None and not (sinks.dtype is torch.float32 and sinks.numel() == heads and sinks.is_contiguous()):
        raise KernelError(f"{what}: sinks are float32 [heads]")
    if scratch is not None and not (scratch.dtype is torch.float32 and scratch.is_contiguous()):
        raise KernelError(f"{what}: scratch must be float32")


def store_kv_8bit(qkv: torch.Tensor, slot_mapping: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                  k_scales: torch.Tensor, v_scales: torch.Tensor, page_size: int, heads: int, kv_heads: int, head_dim: int) -> None:
    """Keys and values of a step into an 8-bit cache.  `qkv`: packed bfloat16 rows, `heads` query heads, then kv_heads keys
    (normed and rotated: qk_rope_store with keys_in_place) and kv_heads values; `slot_mapping` [rows] int32, below 0: no slot.

    A page's scale for a head is the least power of two (2^-118 or more) with which all that was written into the page since
    it was begun fits in 448; where it grows, the page's other rows are taken to the new scale.  A token at a page's first
    place begins the page: what the page held counts for nothing from then on.  Infinities are held as 448 times the scale
    and, like NaN (held as NaN), do not count for it.  The tokens of a page stand side by side in `qkv` (a page is one
    request's), and a slot occurs once; otherwise the page's contents are undefined."""
    _on_this_device("store_kv_8bit", qkv, slot_mapping, k_pages, v_pages, k_scales, v_scales)
    pages = _cache("store_kv_8bit", k_pages, v_pages, k_scales, v_scales, page_size, kv_heads, head_dim)
    if not (heads >= 0 and qkv.dtype is torch.bfloat16 and qkv.dim() == 2 and qkv.stride(1) == 1 and qkv.shape[1] >= (heads + 2 * kv_heads) * head_dim):
        raise KernelError("store_kv_8bit: qkv is bfloat16 [rows, (heads + 2 kv_heads) * head_dim]")
    if not (slot_mapping.dtype is torch.int32 and slot_mapping.is_contiguous() and slot_mapping.numel() >= qkv.shape[0]):
        raise KernelError("store_kv_8bit: one int32 slot for each row is needed")
    lib = library("eight_bit")
    _check(lib, lib.mir_store_8bit(qkv.data_ptr(), qkv.stride(0), slot_mapping.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(),
                                   k_scales.data_ptr(), v_scales.data_ptr(), qkv.shape[0], page_size, pages, heads, kv_heads, head_dim,
                                   _stream()))


def decode_attention_8bit_plan(rows: int, heads: int, kv_heads: int, head_dim: int, page_size: int, max_context: int) -> tuple:
    """(partition, num_partitions, floats of scratch) for decode_attention_8bit of `rows` single tokens whose longest context is
    max_context keys.  Sizes that the tcgen05 kernel takes (head_dim 128, pages of 8 to 128 keys that divide 128): partition 0,
    and the CTAs over which it shares all requests' keys out evenly, by the positions it finds on the device, however long
    the contexts are by then.  Others: keys per partition, and as many partitions as cover the longest context."""
    keys, count, floats = ctypes.c_int(), ctypes.c_int(), ctypes.c_longlong()
    lib = library("eight_bit")
    _check(lib, lib.mir_decode_attention_8bit_plan(rows, heads, kv_heads, head_dim, page_size, max_context, ctypes.byref(keys),
                                                   ctypes.byref(count), ctypes.byref(floats)))
    return keys.value, count.value, floats.value


def decode_attention_8bit(qkv: torch.Tensor, out: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                          k_scales: torch.Tensor, v_scales: torch.Tensor, block_table: torch.Tensor, positions: torch.Tensor,
                          page_size: int, heads: int, kv_heads: int, head_dim: int, scale: float, window: Optional[int],
                          partition: int, num_partitions: int, scratch: Optional[torch.Tensor],
                          sinks: Optional[torch.Tensor] = None) -> None:
    """decode_attention over an 8-bit cache: row r of qkv is one token of request r at positions[r], and sees the keys up to
    its own (inside the window).  A position below 0 is a padding row: its row of `out` is left as it is.  Keys whose page the
    block table does not have (an entry below 0 or beyond the pool, or a block behind its last column) are not seen; a row
    that sees none gets zeros.  `partition`, `num_partitions`: decode_attention_8bit_plan's; where partition is not 0, keys behind
    partition * num_partitions are not seen either.  `scratch`: float32, the plan's size, on a 16-byte boundary; calls that
    may run at the same time, or graphs, take one each.  `sinks`: one number per query head in the softmax's denominator.  A key's
    weight is rounded on its way into the product with the values, by at most 2^-8 of itself (where partition is 0: down to
    2^-56 of the largest among 128 keys, times their pages' scales, and by 2^-67 of that below)."""
    what = "decode_attention_8bit"
    _on_this_device(what, qkv, out, k_pages, v_pages, k_scales, v_scales, block_table, positions, scratch, sinks)
    rows = out.shape[0]
    pages = _cache(what, k_pages, v_pages, k_scales, v_scales, page_size, kv_heads, head_dim)
    _attention(what, qkv, out, block_table, heads, kv_heads, head_dim, rows, sinks, scratch)
    if not (positions.dtype is torch.int32 and positions.is_contiguous() and positions.numel() >= rows):
        raise KernelError(f"{what}: bad positions")
    lib = library("eight_bit")
    _check(lib, lib.mir_decode_attention_8bit(
        qkv.data_ptr(), qkv.stride(0), out.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), k_scales.data_ptr(),
        v_scales.data_ptr(), pages, block_table.data_ptr(), block_table.shape[1], positions.data_ptr(), rows, page_size, heads,
        kv_heads, head_dim, scale, int(window or 0), partition, num_partitions, _ptr(scratch),
        0 if scratch is None else scratch.numel(), _ptr(sinks), _stream()))


def prefill_attention_8bit(qkv: torch.Tensor, out: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                           k_scales: torch.Tensor, v_scales: torch.Tensor, block_table: torch.Tensor, query_starts: torch.Tensor,
                           context_lens: torch.Tensor, page_size: int, heads: int, kv_heads: int, head_dim: int, scale: float,
                           window: Optional[int], sinks: Optional[torch.Tensor] = None, max_context: Optional[int] = None,
                           alloc: Optional[Callable] = None) -> None:
    """prefill_attention over an 8-bit cache, causal: request r has the tokens query_starts[r] .. query_starts[r + 1] - 1 of
    qkv and out, and its context_lens[r] cached tokens include them.  Rows that no request has are left as they are; missing
    pages and rows without a visible key as in decode_attention_8bit.  `max_context`: the longest context, where the caller
    knows it better than the block table's width says (keys from there on need not be seen); `alloc(shape, dtype)`: where scratch comes from (torch's caching
    allocator by default), on a 16-byte boundary."""
    what = "prefill_attention_8bit"
    _on_this_device(what, qkv, out, k_pages, v_pages, k_scales, v_scales, block_table, query_starts, context_lens, sinks)
    rows, tokens = context_lens.numel(), out.shape[0]
    pages = _cache(what, k_pages, v_pages, k_scales, v_scales, page_size, kv_heads, head_dim)
    _attention(what, qkv, out, block_table, heads, kv_heads, head_dim, rows, sinks, None)
    if not (query_starts.dtype is torch.int32 and context_lens.dtype is torch.int32 and query_starts.numel() == rows + 1
            and query_starts.is_contiguous() and context_lens.is_contiguous()):
        raise KernelError(f"{what}: query_starts is int32 [requests + 1], context_lens int32 [requests]")
    longest = min(block_table.shape[1] * page_size, MOST_KEYS)
    if max_context is not None:
        longest = min(longest, max_context)
    lib = library("eight_bit")
    keys, parts, floats = ctypes.c_int(), ctypes.c_int(), ctypes.c_longlong()
    _check(lib, lib.mir_prefill_attention_8bit_plan(rows, tokens, heads, kv_heads, head_dim, page_size, longest, ctypes.byref(keys),
                                                    ctypes.byref(parts), ctypes.byref(floats)))
    partition, count, scratch = keys.value, parts.value, None
    if floats.value:
        scratch = alloc((floats.value,), torch.float32) if alloc is not None else \
            torch.empty((floats.value,), dtype=torch.float32, device=out.device)
    _check(lib, lib.mir_prefill_attention_8bit(
        qkv.data_ptr(), qkv.stride(0), out.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), k_scales.data_ptr(),
        v_scales.data_ptr(), pages, block_table.data_ptr(), block_table.shape[1], query_starts.data_ptr(), context_lens.data_ptr(),
        rows, tokens, page_size, heads, kv_heads, head_dim, scale, int(window or 0), partition, count, _ptr(scratch),
        0 if scratch is None else scratch.numel(), _ptr(sinks), _stream()))


_ERRORS = ("mir_decode_attention_8bit_error", "mir_prefill_attention_8bit_error", "mir_linear_8bit_tiles_error", "mir_linear_8bit_few_error")


def eight_bit_error(reset: bool = False) -> int:
    """0 unless a bounded wait of one of the tcgen05 kernels ran out on the current device (waits for all its streams).  The calls
    return before their kernels run, so that this alone says it: whoever relies on results asks at times, as after a step.  The
    results of the call whose wait ran out are undefined (of linear_8bit: as they were, or right, element by element), and that
    kernel stores nothing more from then on, until `reset` lets it work again."""
    lib = library("eight_bit")
    found = [getattr(lib, name)(0 if reset else -1) for name in _ERRORS]
    return next((error for error in found if error), 0)


def quantize_weight_8bit(weight: torch.Tensor) -> tuple:
    """(values, scales) of a float32 or bfloat16 weight [N, K] for linear_8bit: e4m3 [N, K] and float32 [ceil(N / 128),
    ceil(K / 128)], a block's scale its largest magnitude / 448 (infinities do not count and are held as 448 times it)."""
    _on_this_device("quantize_weight_8bit", weight)
    if not (weight.dim() == 2 and weight.is_contiguous() and weight.dtype in (torch.float32, torch.bfloat16) and weight.numel() > 0):
        raise KernelError("quantize_weight_8bit: a contiguous float32 or bfloat16 [rows, columns] is needed")
    rows, columns = weight.shape
    values = torch.empty((rows, columns), dtype=E4M3, device=weight.device)
    scales = torch.empty((-(-rows // BLOCK), -(-columns // BLOCK)), dtype=torch.float32, device=weight.device)
    lib = library("eight_bit")
    _check(lib, lib.mir_quantize_weight_8bit(int(weight.dtype is torch.bfloat16), weight.data_ptr(), values.data_ptr(),
                                             scales.data_ptr(), rows, columns, _stream()))
    return values, scales


def set_linear_8bit_splits(splits: int) -> None:
    """For measurements: over how many CTAs a product of up to 128 rows cuts K (1, 2, 4 or 8; 0: the launcher's rule)."""
    lib = library("eight_bit")
    _check(lib, lib.mir_linear_8bit_few_set_splits(int(splits)))


def linear_8bit(x: torch.Tensor, weight: torch.Tensor, scales: torch.Tensor, out: torch.Tensor,
                bias: Optional[torch.Tensor] = None, accumulate: bool = False, alloc: Optional[Callable] = None) -> None:
    """out = (out if accumulate) + x . w^T (+ bias), w = weight[n, k] * scales[n // 128, k // 128].

    `weight`: e4m3 [N, K] with K a multiple of 16, `scales`: any float32 [ceil(N / 128), ceil(K / 128)] (quantize_weight_8bit
    makes both, and checkpoints bring them).  `x`: bfloat16 [M, K]; every row's runs of 128 columns are rounded to e4m3 with
    the least power of two as their scale (2^-118 or more) that keeps them within 448; infinities are taken as 448 times it.
    Sums are 32-bit, and so is the product of a block's two scales (below 2^-126 it loses bits).  `out`: bfloat16 or, the only one that accumulates, float32; `bias` has out's dtype.  x and out may be
    row-strided views; x's rows begin on 8-byte boundaries.  `alloc(shape, dtype)`: where the workspace comes from (torch's caching allocator by default)."""
    _on_this_device("linear_8bit", x, weight, scales, out, bias)
    if not (x.dim() == 2 and weight.dim() == 2 and x.dtype is torch.bfloat16 and weight.dtype is E4M3):
        raise KernelError("linear_8bit: x is bfloat16 [M, K], weight float8_e4m3fn [N, K]")
    (m, k), n = x.shape, weight.shape[0]
    if not (weight.shape[1] == k and out.shape == (m, n) and (x.stride(1) == 1 or m == 0)
            and (out.stride(1) == 1 or n <= 1 or m == 0) and weight.is_contiguous()):
        raise KernelError("linear_8bit: shapes or strides do not fit")
    if not (scales.dtype is torch.float32 and scales.is_contiguous() and scales.shape == (-(-n // BLOCK), -(-k // BLOCK))):
        raise KernelError(f"linear_8bit: scales are contiguous float32 [{-(-n // BLOCK)}, {-(-k // BLOCK)}]")
    if not (out.dtype in (torch.bfloat16, torch.float32) and (out.dtype is torch.float32 or not accumulate)):
        raise KernelError("linear_8bit: out is bfloat16 or float32, and only float32 accumulates")
    if not (bias is None or (bias.dtype == out.dtype and bias.numel() == n and bias.is_contiguous())):
        raise KernelError("linear_8bit: bias is [N] of out's dtype")
    if m == 0 or n == 0:
        return
    lib = library("eight_bit")
    size = lib.mir_linear_8bit_workspace(m, k)
    workspace = None
    if size:                    # (up to 16 rows are rounded where they are used)
        workspace = alloc((size,), torch.uint8) if alloc is not None else torch.empty((size,), dtype=torch.uint8, device=x.device)
        size = workspace.numel() * workspace.element_size()          # (what there is, which the launcher checks)
    _check(lib, lib.mir_linear_8bit(x.data_ptr(), x.stride(0), weight.data_ptr(), scales.data_ptr(), _ptr(bias), out.data_ptr(),
                                    out.stride(0), int(out.dtype is torch.float32), int(accumulate), m, n, k, _ptr(workspace),
                                    size, _stream()))
