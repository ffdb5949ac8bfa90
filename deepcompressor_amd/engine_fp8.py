"""Host layer of the operators that run on 8-bit values: argument checks, output allocation and the C ABI calls of the
block quantizer, the block-scaled product, and the append to / attention over a key / value cache held in 8 bits.

Inference only: results carry no gradient, so an argument that asks for one is refused while autograd records.
"""

from __future__ import annotations

import ctypes as C
import functools

import torch
from torch.autograd import forward_ad

from ._lib import DcqError, _raw_stream, check, lib, storage_of

__all__ = ["BLOCK", "E4M3", "quantize_blocks", "block_product", "kv_append", "kv_attention"]

BLOCK = 128  # elements along the last axis that share a scale
E4M3, F32, I32 = torch.float8_e4m3fn, torch.float32, torch.int32
_Strides = functools.lru_cache(maxsize=1024)(C.c_int64 * 3)  # (read by the call only: one array for all tensors alike)


def _device_of(*tensors: torch.Tensor | None) -> int:
    """The index of the one GPU that all tensors are on, none of them asking for a gradient or carrying a tangent."""
    device = -1
    if forward_ad._current_level >= 0 and any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise DcqError("this operator has no forward gradient: call it on tensors without tangents")
    for t in tensors:
        if t is None:
            continue
        at = t.get_device()
        if at != device or at < 0:
            if at < 0:
                raise DcqError(f"deepcompressor_amd runs on MI355X GPUs only; got a tensor on '{t.device}' (there is no CPU path)")
            if device >= 0:
                raise DcqError(f"tensors on two devices: cuda:{device} and cuda:{at}")
            device = at
        if t.requires_grad and torch.is_grad_enabled():
            raise DcqError("this operator has no gradient: call it under torch.no_grad(), or on detached tensors")
    return device


@functools.lru_cache(maxsize=None)
def _entry(name: str):
    return getattr(lib(), name)


def _launch(name: str, device: int, *args) -> None:
    """One C ABI call on the stream torch currently launches on for ``device``, whatever the current device is."""
    function = _entry(name)
    if torch._C._cuda_getDevice() == device:
        rc = function(*args, _raw_stream(device))
    else:
        with torch.cuda.device(device):
            rc = function(*args, _raw_stream(device))
    if rc != 0:
        check(rc, name)


# ---- block-scaled tensors ------------------------------------------------------------------------------------------


def quantize_blocks(x: torch.Tensor, block_rows: int) -> tuple[torch.Tensor, torch.Tensor]:
    """x [rows][cols] -> (codes [rows][cols] whose rows start at multiples of 16 bytes, scales [row blocks][col blocks])."""
    if block_rows not in (1, BLOCK):
        raise ValueError(f"blocks have 1 or {BLOCK} rows, not {block_rows}")
    storage, device = storage_of(x.dtype), _device_of(x)
    rows, cols = x.shape
    ld = x.stride(0)
    if x.stride(1) != 1 and cols > 1 or ld < cols and rows > 1:
        x, ld = x.contiguous(), cols
    pitch, row_blocks, col_blocks = -(-cols // 16) * 16, -(-rows // block_rows), -(-cols // BLOCK)
    codes = x.new_empty((rows, pitch), dtype=E4M3)
    # column-major for 1 x 128 blocks: the product wants the scales of consecutive rows side by side
    strides = (1, row_blocks) if block_rows == 1 else (col_blocks, 1)
    scales = x.new_empty_strided((row_blocks, col_blocks), strides, dtype=torch.float32)
    _launch("dcq_fp8_quantize_blocks", device, x.data_ptr(), storage, rows, cols, ld, block_rows, codes.data_ptr(), pitch,
            scales.data_ptr(), *strides)
    return codes if pitch == cols else codes[:, :cols], scales


def look_over(*matrices: torch.Tensor) -> None:
    """The product reads rows of codes up to the next multiple of 16 bytes: the last row's memory has to reach so far."""
    for codes in matrices:
        cols = codes.shape[-1]
        if codes.ndim == 2 and cols % 16 and len(codes) and (codes.storage_offset() + (len(codes) - 1) * codes.stride(0) + cols + -cols % 16
                                                             > codes.untyped_storage().nbytes()):
            raise ValueError("codes are read up to the next multiple of 16 bytes, and their memory ends before: BlockScaledTensor.from_codes copies such")


def checked_codes(codes: torch.Tensor, scales: torch.Tensor, block_rows: int) -> torch.Tensor:
    """The codes, their rows at multiples of 16 bytes with readable memory up to the next one behind each row: they
    themselves if that is so, else a copy."""
    if codes.dtype != E4M3 or codes.ndim != 2:
        raise ValueError("codes are a float8_e4m3fn matrix")
    if block_rows not in (1, BLOCK):
        raise ValueError(f"blocks have 1 or {BLOCK} rows, not {block_rows}")
    rows, cols = codes.shape
    if scales.dtype != F32 or scales.shape != (-(-rows // block_rows), -(-cols // BLOCK)):
        raise ValueError(f"scales are float32 of shape {(-(-rows // block_rows), -(-cols // BLOCK))}, got {scales.dtype} of "
                         f"{tuple(scales.shape)}")
    pitch, (ld, step) = -(-cols // 16) * 16, codes.stride()
    if rows == 0 or cols == 0:
        return codes
    if step == 1 and ld % 16 == 0 and ld >= pitch and codes.data_ptr() % 16 == 0 and (
            pitch == cols or codes.storage_offset() + (rows - 1) * ld + pitch <= codes.untyped_storage().nbytes()):
        return codes
    out = torch.empty((rows, pitch), dtype=torch.uint8, device=codes.device)
    out[:, :cols] = codes.view(torch.uint8)
    return out.view(E4M3)[:, :cols]


def block_product(x_codes: torch.Tensor, x_scales: torch.Tensor, w_codes: torch.Tensor, w_scales: torch.Tensor,
                  bias: torch.Tensor | None, dtype: torch.dtype) -> torch.Tensor:
    """[M][K] codes in 1 x 128 blocks times [N][K] codes in 128 x 128 blocks, transposed, -> [M][N] of `dtype`."""
    (M, K), (N, w_cols) = x_codes.shape, w_codes.shape
    if w_cols != K:
        raise ValueError(f"inner sizes differ: {K} and {w_cols}")
    blocks = -(-K // BLOCK)
    if x_scales.shape != (M, blocks) or w_scales.shape != (-(-N // BLOCK), blocks):
        raise ValueError(f"scales have shapes {tuple(x_scales.shape)} and {tuple(w_scales.shape)}, expected {(M, blocks)} and "
                         f"{(-(-N // BLOCK), blocks)}")
    if x_scales.dtype != F32 or w_scales.dtype != F32 or x_codes.dtype != E4M3 or w_codes.dtype != E4M3:
        raise ValueError("codes are float8_e4m3fn, scales float32")
    (x_ld, x_step), (w_ld, w_step) = x_codes.stride(), w_codes.stride()
    if (x_step != 1 or w_step != 1) and K > 1:
        raise ValueError("codes are contiguous along their rows")
    bias_at, bias_storage = None, 0
    if bias is not None:
        if bias.shape != (N,):
            raise ValueError(f"bias has shape {tuple(bias.shape)}, expected ({N},)")
        bias, bias_storage = bias.contiguous(), storage_of(bias.dtype)
        bias_at = bias.data_ptr()
    storage = storage_of(dtype)
    device = _device_of(x_codes, x_scales, w_codes, w_scales, bias)
    y = x_codes.new_empty((M, N), dtype=dtype)
    if K == 0:
        return y.zero_() if bias is None else y.copy_(bias)
    _launch("dcq_fp8_block_gemm", device, x_codes.data_ptr(), x_ld, x_scales.data_ptr(), *x_scales.stride(), w_codes.data_ptr(), w_ld,
            w_scales.data_ptr(), *w_scales.stride(), bias_at, bias_storage, y.data_ptr(), storage, N, M, N, K)
    return y


# ---- the cache -----------------------------------------------------------------------------------------------------------


def _used_strides(t: torch.Tensor) -> tuple[int, ...]:
    """The strides, 0 for axes of size 1: torch leaves any number there, also where it calls a tensor contiguous."""
    return tuple(s if n > 1 else 0 for n, s in zip(t.shape, t.stride()))


def _output_strides(out: torch.Tensor, query: torch.Tensor) -> tuple[int, ...]:
    """The strides of a caller's output that the kernels can write."""
    if out.shape != query.shape or out.dtype != query.dtype:
        raise ValueError("out differs from query in shape or type")
    strides = _used_strides(out)
    if strides[-1] != 1 or any(s % 4 for s in strides[:-1]) or out.data_ptr() % 8:
        raise ValueError("out's channels must be contiguous and its strides multiples of 4")
    end = 0  # how far the axes of smaller strides reach
    for s, n in sorted((s, n) for s, n in zip(strides, out.shape) if n > 1):
        if s <= end:
            raise ValueError("out has elements that share memory")
        end += (n - 1) * s
    return strides


def _tokens(t: torch.Tensor, packed: bool, what: str, align: int) -> tuple[torch.Tensor, C.Array]:
    """A tensor of tokens, [sequence][token][head][channel] or packed [token][head][channel], that the kernels can address
    (copied if its strides or its address are not multiples of `align` elements), and its (sequence, token, head) strides."""
    if t.ndim != (3 if packed else 4):
        raise ValueError(f"{what} has {t.ndim} dimensions: [sequence][token][head][channel], or packed [token][head][channel] with starts")
    strides = t.stride()
    if strides[-1] != 1 or strides[0] % align or strides[1] % align or strides[-2] % align or t.data_ptr() % 16:
        strides = _used_strides(t)
        if strides[-1] != 1 or any(s % align for s in strides[:-1]) or t.data_ptr() % 16:
            t = torch.empty(t.shape, dtype=t.dtype, device=t.device).copy_(t)
            strides = t.stride()
    return t, _Strides(0, strides[0], strides[1]) if packed else _Strides(strides[0], strides[1], strides[2])


def _sequences(t: torch.Tensor, table, lengths, starts):
    """(table, lengths, starts, sequences, columns, tokens of all sequences together)"""
    shape = table.shape
    if len(shape) != 2 or shape[1] < 1:
        raise ValueError("block_table is [sequence][column], with at least one column")
    count, columns = shape
    if table.dtype != I32 or lengths.dtype != I32 or lengths.shape != (count,) or starts is not None and (
            starts.dtype != I32 or starts.shape != (count + 1,)):
        raise ValueError(f"block_table, lengths and starts are int32, lengths of shape {(count,)}, starts of {(count + 1,)}; got {table.dtype}, "
                         f"{lengths.dtype} of {tuple(lengths.shape)}" + ("" if starts is None else f", {starts.dtype} of {tuple(starts.shape)}"))
    total = t.shape[0]
    if starts is None:
        if total != count:
            raise ValueError(f"{total} sequences of tokens, {count} in block_table")
        total *= t.shape[1]
    else:
        starts = starts.contiguous()
    return table.contiguous(), lengths.contiguous(), starts, count, columns, total


def kv_append(key, value, k_codes, k_scales, v_codes, v_scales, table, lengths, starts) -> None:
    pool, heads, page, dim = k_codes.shape
    shape = key.shape
    if shape != value.shape or key.dtype != value.dtype:
        raise ValueError("key and value differ in shape or type")
    if shape[-2:] != (heads, dim):
        raise ValueError(f"tokens have {tuple(shape[-2:])} heads and channels, the cache {(heads, dim)}")
    storage = storage_of(key.dtype)
    device = _device_of(k_codes, k_scales, v_scales, key, value, table, lengths, starts)
    align = 16 // key.element_size()
    key, key_strides = _tokens(key, starts is not None, "key", align)
    value, value_strides = _tokens(value, starts is not None, "value", align)
    table, lengths, starts, count, columns, total = _sequences(key, table, lengths, starts)
    _launch("dcq_kv8_append", device, key.data_ptr(), value.data_ptr(), storage, key_strides, value_strides,
            k_codes.data_ptr(), k_scales.data_ptr(), v_codes.data_ptr(), v_scales.data_ptr(), table.data_ptr(), lengths.data_ptr(),
            None if starts is None else starts.data_ptr(), count, total, pool, heads, page, dim, columns)


@functools.lru_cache(maxsize=256)
def _workspace_bytes(*sizes: int) -> int:
    return lib().dcq_kv8_attention_workspace_bytes(*sizes)


def kv_attention(query, k_codes, k_scales, v_codes, v_scales, table, lengths, starts, scale, causal, out) -> torch.Tensor:
    pool, heads, page, dim = k_codes.shape
    if query.dtype != torch.bfloat16 and query.dtype != torch.float16:
        raise ValueError(f"queries are float16 or bfloat16, got {query.dtype}")
    shape = query.shape
    if len(shape) < 2 or shape[-1] != dim or shape[-2] % heads or shape[-2] == 0:
        raise ValueError(f"queries have {tuple(shape[-2:])} heads and channels, the cache {(heads, dim)}")
    group = shape[-2] // heads
    given = out is not None
    if given:
        steps = _output_strides(out, query)
    device = _device_of(k_codes, k_scales, v_scales, query, table, lengths, starts, out)
    query, query_strides = _tokens(query, starts is not None, "query", 8)
    table, lengths, starts, count, columns, total = _sequences(query, table, lengths, starts)
    if not given:
        out = query.new_empty(shape)
        steps = out.stride()
    if count == 0:  # no sequence has any of the rows
        return out if given else out.zero_()
    out_strides = _Strides(0, steps[0], steps[1]) if starts is not None else _Strides(steps[0], steps[1], steps[2])
    need = _workspace_bytes(count, total, heads, group, dim, columns * page, int(starts is not None))
    workspace = query.new_empty(need, dtype=torch.uint8) if need else None
    _launch("dcq_kv8_attention", device, query.data_ptr(), storage_of(query.dtype), query_strides, out.data_ptr(), out_strides,
            k_codes.data_ptr(), k_scales.data_ptr(), v_codes.data_ptr(), v_scales.data_ptr(), table.data_ptr(),
            lengths.data_ptr(), None if starts is None else starts.data_ptr(), count, total, pool, heads, group, page, dim, columns,
            float(scale), int(causal), int(not given), None if workspace is None else workspace.data_ptr(), need)
    return out
