"""Host layer of the operators that run on 8-bit values: argument checks, output allocation and the C ABI calls of the
block quantizer, the block-scaled product, and the append to / attention over a key / value cache held in 8 bits.

Inference only: results carry no gradient, so an argument that asks for one is refused while autograd records.
"""

from __future__ import annotations

import contextlib
import ctypes as C

import torch

from ._lib import DcqError, check, lib, ptr, storage_of, stream_of

__all__ = ["BLOCK", "E4M3", "quantize_blocks", "block_product", "kv_append", "kv_attention"]

BLOCK = 128  # elements along the last axis that share a scale
E4M3 = torch.float8_e4m3fn
_Strides = C.c_int64 * 3


def on_device_of(first: torch.Tensor, *others: torch.Tensor | None):
    """All tensors on one GPU, none asking for a gradient: the context in which kernels for that GPU are launched."""
    for t in (first, *others):
        if t is None:
            continue
        if not t.is_cuda:
            raise DcqError(f"deepcompressor_amd runs on MI355X GPUs only; got a tensor on '{t.device}' (there is no CPU path)")
        if t.device != first.device:
            raise DcqError(f"tensors on two devices: {first.device} and {t.device}")
        if t.requires_grad and torch.is_grad_enabled():
            raise DcqError("this operator has no gradient: call it under torch.no_grad(), or on detached tensors")
    if first.device.index == torch.cuda.current_device():
        return contextlib.nullcontext()
    return torch.cuda.device(first.device)


def _address(t: torch.Tensor | None):
    return None if t is None else C.c_void_p(t.data_ptr())


def _require(condition: bool, message: str) -> None:
    if not condition:
        raise ValueError(message)


# ---- block-scaled tensors ------------------------------------------------------------------------------------------


def quantize_blocks(x: torch.Tensor, block_rows: int) -> tuple[torch.Tensor, torch.Tensor]:
    """x [rows][cols] -> (codes [rows][cols] whose rows start at multiples of 16 bytes, scales [row blocks][col blocks])."""
    _require(x.ndim == 2, f"expected a matrix, got {x.ndim} dimensions")
    _require(block_rows in (1, BLOCK), f"blocks have 1 or {BLOCK} rows, not {block_rows}")
    storage = storage_of(x.dtype)
    with on_device_of(x):
        rows, cols = x.shape
        if x.stride(1) != 1 and cols > 1 or x.stride(0) < cols and rows > 1:
            x = x.contiguous()
        row_blocks, col_blocks = -(-rows // block_rows), -(-cols // BLOCK)
        codes = torch.empty((rows, -(-cols // 16) * 16), dtype=E4M3, device=x.device)
        # column-major for 1 x 128 blocks: the product wants the scales of consecutive rows side by side
        if block_rows == 1:
            scales = torch.empty((col_blocks, row_blocks), dtype=torch.float32, device=x.device).t()
        else:
            scales = torch.empty((row_blocks, col_blocks), dtype=torch.float32, device=x.device)
        check(lib().dcq_fp8_quantize_blocks(_address(x), storage, rows, cols, x.stride(0), block_rows, _address(codes),
                                            codes.stride(0), _address(scales), scales.stride(0), scales.stride(1),
                                            stream_of(x.device)), "dcq_fp8_quantize_blocks")
    return codes[:, :cols], scales


def _padded(codes: torch.Tensor) -> torch.Tensor:
    """The same codes, their rows at multiples of 16 bytes with readable memory up to the next one behind each row."""
    rows, cols = codes.shape
    pitch = -(-cols // 16) * 16
    base = codes.storage_offset()
    if (codes.stride(1) == 1 and codes.stride(0) % 16 == 0 and codes.stride(0) >= pitch and codes.data_ptr() % 16 == 0
            and base + max(rows - 1, 0) * codes.stride(0) + pitch <= codes.untyped_storage().nbytes()):
        return codes
    out = torch.empty((rows, pitch), dtype=torch.uint8, device=codes.device)
    out[:, :cols] = codes.view(torch.uint8)
    return out.view(E4M3)[:, :cols]


def checked_codes(codes: torch.Tensor, scales: torch.Tensor, block_rows: int) -> torch.Tensor:
    _require(codes.ndim == 2 and codes.dtype == E4M3, "codes are a float8_e4m3fn matrix")
    _require(block_rows in (1, BLOCK), f"blocks have 1 or {BLOCK} rows, not {block_rows}")
    want = (-(-codes.shape[0] // block_rows), -(-codes.shape[1] // BLOCK))
    _require(scales.dtype == torch.float32 and tuple(scales.shape) == want,
             f"scales are float32 of shape {want}, got {scales.dtype} of {tuple(scales.shape)}")
    return codes if codes.numel() == 0 else _padded(codes)


def block_product(x_codes: torch.Tensor, x_scales: torch.Tensor, w_codes: torch.Tensor, w_scales: torch.Tensor,
                  bias: torch.Tensor | None, dtype: torch.dtype) -> torch.Tensor:
    """[M][K] codes in 1 x 128 blocks times [N][K] codes in 128 x 128 blocks, transposed, -> [M][N] of `dtype`."""
    (M, K), N = x_codes.shape, w_codes.shape[0]
    _require(w_codes.shape[1] == K, f"inner sizes differ: {K} and {w_codes.shape[1]}")
    if bias is not None:
        _require(tuple(bias.shape) == (N,), f"bias has shape {tuple(bias.shape)}, expected ({N},)")
    storage, bias_storage = storage_of(dtype), 0 if bias is None else storage_of(bias.dtype)
    with on_device_of(x_codes, x_scales, w_codes, w_scales, bias):
        bias = None if bias is None else bias.contiguous()
        y = torch.empty((M, N), dtype=dtype, device=x_codes.device)
        if K == 0:
            return y.zero_() if bias is None else y.copy_(bias)
        check(lib().dcq_fp8_block_gemm(_address(x_codes), x_codes.stride(0), _address(x_scales), x_scales.stride(0), x_scales.stride(1),
                                       _address(w_codes), w_codes.stride(0), _address(w_scales), w_scales.stride(0), w_scales.stride(1),
                                       _address(bias), bias_storage, _address(y), storage, N, M, N, K,
                                       stream_of(y.device)), "dcq_fp8_block_gemm")
    return y


# ---- the cache -----------------------------------------------------------------------------------------------------------


def _tokens(t: torch.Tensor, starts: torch.Tensor | None, what: str, align: int) -> tuple[torch.Tensor, tuple[int, int, int]]:
    """A tensor of tokens, [sequence][token][head][channel] or packed [token][head][channel], that the kernels can address
    (copied if its strides or its address are not multiples of `align` elements), and its (sequence, token, head) strides."""
    _require(t.ndim == (4 if starts is None else 3),
             f"{what} has {t.ndim} dimensions: [sequence][token][head][channel], or packed [token][head][channel] with starts")
    if t.stride(-1) != 1 or any(s % align for s in t.stride()[:-1]) or t.data_ptr() % (align * t.element_size()):
        t = t.contiguous().clone() if t.is_contiguous() else t.contiguous()
    return t, (0, *t.stride()[:2]) if starts is not None else t.stride()[:3]


def _index(t: torch.Tensor, shape: tuple, what: str) -> torch.Tensor:
    _require(t.dtype == torch.int32, f"{what} is int32, got {t.dtype}")
    _require(len(t.shape) == len(shape) and all(w is None or w == n for n, w in zip(t.shape, shape)),
             f"{what} has shape {tuple(t.shape)}, expected {shape}")
    return t.contiguous()


def _sequences(t: torch.Tensor, table, lengths, starts):
    """(table, lengths, starts, sequences, tokens of all sequences together)"""
    table = _index(table, (None, None), "block_table")
    count = table.shape[0]
    _require(table.shape[1] >= 1, "block_table has no columns")
    lengths = _index(lengths, (count,), "lengths")
    if starts is not None:
        return table, lengths, _index(starts, (count + 1,), "starts"), count, t.shape[0]
    _require(t.shape[0] == count, f"{t.shape[0]} sequences of tokens, {count} in block_table")
    return table, lengths, None, count, t.shape[0] * t.shape[1]


def kv_append(key, value, k_codes, k_scales, v_codes, v_scales, table, lengths, starts) -> None:
    pool, heads, page, dim = k_codes.shape
    _require(key.shape == value.shape and key.dtype == value.dtype, "key and value differ in shape or type")
    _require(tuple(key.shape[-2:]) == (heads, dim), f"tokens have {tuple(key.shape[-2:])} heads and channels, the cache {(heads, dim)}")
    storage = storage_of(key.dtype)
    with on_device_of(k_codes, key, value, table, lengths, starts):
        align = 16 // key.element_size()
        key, key_strides = _tokens(key, starts, "key", align)
        value, value_strides = _tokens(value, starts, "value", align)
        table, lengths, starts, count, total = _sequences(key, table, lengths, starts)
        check(lib().dcq_kv8_append(_address(key), _address(value), storage, _Strides(*key_strides), _Strides(*value_strides),
                                   _address(k_codes), ptr(k_scales), _address(v_codes), ptr(v_scales), ptr(table), ptr(lengths),
                                   ptr(starts), count, total, pool, heads, page, dim, table.shape[1],
                                   stream_of(key.device)), "dcq_kv8_append")


def kv_attention(query, k_codes, k_scales, v_codes, v_scales, table, lengths, starts, scale, causal, out) -> torch.Tensor:
    pool, heads, page, dim = k_codes.shape
    _require(query.dtype in (torch.float16, torch.bfloat16), f"queries are float16 or bfloat16, got {query.dtype}")
    _require(query.ndim >= 2 and query.shape[-1] == dim and query.shape[-2] % heads == 0 and query.shape[-2] > 0,
             f"queries have {tuple(query.shape[-2:])} heads and channels, the cache {(heads, dim)}")
    group = query.shape[-2] // heads
    with on_device_of(k_codes, query, table, lengths, starts, out):
        query, query_strides = _tokens(query, starts, "query", 8)
        table, lengths, starts, count, total = _sequences(query, table, lengths, starts)
        given = out is not None
        if given:
            _require(out.shape == query.shape and out.dtype == query.dtype, "out differs from query in shape or type")
            _require(out.stride(-1) == 1 and all(s % 4 == 0 for s in out.stride()[:-1]) and out.data_ptr() % 8 == 0,
                     "out's channels must be contiguous and its strides multiples of 4")
        else:
            out = torch.empty(query.shape, dtype=query.dtype, device=query.device)
        out_strides = (0, *out.stride()[:2]) if starts is not None else out.stride()[:3]
        packed, capacity = int(starts is not None), table.shape[1] * page
        need = lib().dcq_kv8_attention_workspace_bytes(count, total, heads, group, dim, capacity, packed)
        workspace = torch.empty(need, dtype=torch.uint8, device=query.device) if need else None
        check(lib().dcq_kv8_attention(_address(query), storage_of(query.dtype), _Strides(*query_strides), _address(out),
                                      _Strides(*out_strides), _address(k_codes), ptr(k_scales), _address(v_codes), ptr(v_scales),
                                      ptr(table), ptr(lengths), ptr(starts), count, total, pool, heads, group, page, dim,
                                      table.shape[1], float(scale), int(causal), int(not given), ptr(workspace), need,
                                      stream_of(query.device)), "dcq_kv8_attention")
    return out
