"""Plain numpy forms of the operators that run on 8-bit values: the definitions, one element or row after the other where
that is clearest, in float64 (quantization: in the float32 steps that define it)."""

from __future__ import annotations

import numpy as np

BLOCK, TOP = 128, 448.0
_MAGNITUDES = [m * 2.0**-9 for m in range(8)] + [(8 + m) * 2.0 ** (e - 10) for e in range(1, 16) for m in range(8)
                                                 if (e, m) != (15, 7)]
GRID = np.array(sorted({-m for m in _MAGNITUDES} | set(_MAGNITUDES)))


def nearest_e4m3(v: np.ndarray) -> np.ndarray:
    """Nearest value of the grid, a tie to the upper one; NaN stays NaN."""
    v = np.asarray(v, dtype=np.float64)
    out = GRID[np.searchsorted((GRID[1:] + GRID[:-1]) / 2, np.where(np.isnan(v), 0.0, v), side="right")]
    return np.where(np.isnan(v), np.nan, out)


def quantize_blocks(x: np.ndarray, block_rows: int):
    """float32 [rows][cols] -> (codes, scales), the scale float32(max / 448) (0 -> 1), the quotient float32(x / scale)."""
    x = np.asarray(x, dtype=np.float32)
    rows, cols = x.shape
    scales = np.zeros((-(-rows // block_rows), -(-cols // BLOCK)), dtype=np.float32)
    codes = np.zeros((rows, cols))
    with np.errstate(all="ignore"):
        for i in range(scales.shape[0]):
            for j in range(scales.shape[1]):
                at = np.s_[i * block_rows:(i + 1) * block_rows, j * BLOCK:(j + 1) * BLOCK]
                block = np.abs(x[at])
                s = np.float32(np.max(np.where(np.isnan(block), np.float32(0), block))) / np.float32(TOP)
                s = np.float32(1) if s == 0 else s
                scales[i, j] = s
                codes[at] = nearest_e4m3(x[at] / s)
    return codes, scales


def expand(scales: np.ndarray, block_rows: int, shape) -> np.ndarray:
    return np.repeat(np.repeat(scales.astype(np.float64), block_rows, 0), BLOCK, 1)[:shape[0], :shape[1]]


def product(x, xs, w, ws, bias=None):
    """(y, sum of the terms' magnitudes), float64"""
    x, w = x * expand(xs, 1, x.shape), w * expand(ws, BLOCK, w.shape)
    y, size = x @ w.T, np.abs(x) @ np.abs(w).T
    if bias is not None:
        y, size = y + bias, size + np.abs(bias)
    return y, size


def power_scale(largest: float) -> float:
    """Smallest power of two s >= 2^-126 with 448 s >= largest."""
    s = 2.0**-126
    while TOP * s < largest:
        s *= 2
    return s


def append(cache: dict, key, value, table, lengths, counts):
    """cache: k_codes [page][head][token][channel], v_codes [page][head][channel][token] as values, k_scales, v_scales;
    key, value: a list of [token][head][channel] per sequence.  Changes the cache in place."""
    pool, heads, page, _ = cache["k_codes"].shape
    for i, n in enumerate(counts):
        length = min(max(int(lengths[i]), 0), len(table[i]) * page)
        end = min(length + n, len(table[i]) * page)
        at = length
        while at < end:
            p, a = int(table[i][at // page]), at % page
            m = min(page - a, end - at)
            if 0 <= p < pool:
                for name, x in (("k", key[i]), ("v", value[i])):
                    codes = cache[name + "_codes"][p] if name == "k" else cache[name + "_codes"][p].transpose(0, 2, 1)
                    for h in range(heads):
                        new = np.asarray(x[at - length:at - length + m, h], dtype=np.float64)
                        finite = np.where(np.isfinite(new), new, np.nan)
                        size = np.abs(finite[np.isfinite(finite)])
                        s, old = power_scale(size.max() if size.size else 0.0), float(cache[name + "_scales"][p, h])
                        if a > 0:
                            s = max(s, old)
                            if s != old:
                                codes[h] = nearest_e4m3(codes[h] * (old / s))
                        codes[h, a:a + m] = nearest_e4m3(finite / s)
                        cache[name + "_scales"][p, h] = s
            at += m


def attend(cache: dict, queries, table, lengths, scale, causal=True):
    """queries: a list of [query][head][channel] per sequence -> a list of (outputs, sums p |v| / sums p, largest score
    magnitude sum) per sequence, float64."""
    pool, heads, page, dim = cache["k_codes"].shape
    results = []
    for i, q in enumerate(queries):
        q = np.asarray(q, dtype=np.float64)
        n, group = q.shape[0], q.shape[1] // heads
        length, capacity = max(int(lengths[i]), 0), len(table[i]) * page
        out, size, reach = np.zeros(q.shape), np.zeros(q.shape), np.zeros(q.shape[:2])
        for j in range(n):
            limit = min(max(length - n + j + 1, 0) if causal else length, capacity)
            tokens = [t for t in range(limit) if 0 <= int(table[i][t // page]) < pool]
            if not tokens:
                continue
            pages, slots = np.array([int(table[i][t // page]) for t in tokens]), np.array(tokens) % page
            for h in range(q.shape[1]):
                c = h // group
                k = cache["k_codes"][pages, c, slots] * cache["k_scales"][pages, c].astype(np.float64)[:, None]
                v = cache["v_codes"][pages, c, :, slots] * cache["v_scales"][pages, c].astype(np.float64)[:, None]
                with np.errstate(all="ignore"):
                    s = (k @ q[j, h]) * scale
                    p = np.exp(s - np.max(s))
                    out[j, h], size[j, h] = p @ v / p.sum(), p @ np.abs(v) / p.sum()
                    reach[j, h] = (np.abs(k) @ np.abs(q[j, h])).max() * abs(scale)
        results.append((out, size, reach))
    return results
