"""Caches, tables and tolerances shared by the tests of the 8-bit cache."""

import numpy as np
import torch

import fp8_oracle as fo
from deepcompressor_amd.nn.patch import Fp8KVCache

HALF_STEP = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11, torch.float32: 2.0**-24}


def values(codes: torch.Tensor) -> np.ndarray:
    return codes.float().cpu().numpy().astype(np.float64)


def as_dict(cache: Fp8KVCache) -> dict:
    return {"k_codes": values(cache.k_codes), "v_codes": values(cache.v_codes), "k_scales": cache.k_scales.cpu().numpy().copy(),
            "v_scales": cache.v_scales.cpu().numpy().copy()}


def make_cache(pool, heads, dim, page, seed, device="cuda", garbage=True) -> Fp8KVCache:
    """Pages of random codes; ``garbage``: NaN codes in every page and infinite scales, as in memory nobody has written."""
    cache = Fp8KVCache(pool, heads, dim, page, device=device)
    if garbage:
        for t in (cache.k_codes, cache.v_codes):
            t.view(torch.uint8).fill_(0x7F)
        cache.k_scales.fill_(float("inf"))
        cache.v_scales.fill_(float("nan"))
    return cache


def make_table(lengths, page, cols, pool, seed, hole=-1):
    """Each sequence's pages in random order, ``hole`` behind them; no page twice."""
    rng = np.random.RandomState(seed)
    free = list(rng.permutation(pool))
    table = np.full((len(lengths), cols), hole, dtype=np.int32)
    for i, n in enumerate(lengths):
        for c in range(min(-(-n // page), cols)):
            table[i, c] = free.pop()
    return table


def fill(cache, table, lengths, seed, dtype=torch.bfloat16, scale=1.0):
    """Append ``lengths`` tokens of each sequence to an empty cache (through the operator itself)."""
    g = torch.Generator().manual_seed(seed)
    _, heads, _, dim = cache.k_codes.shape
    starts = torch.tensor(np.concatenate([[0], np.cumsum(lengths)]), dtype=torch.int32)
    kv = [torch.randn((int(starts[-1]), heads, dim), generator=g).mul(scale).to(dtype) for _ in range(2)]
    dev = cache.k_codes.device
    cache.append(kv[0].to(dev), kv[1].to(dev), torch.from_numpy(table).to(dev), torch.zeros(len(lengths), dtype=torch.int32, device=dev),
                 starts=starts.to(dev))
    return kv, starts


def check_attention(got, queries, cache, table, lengths, scale, causal, dtype):
    """Against the definition in 64 bits.  Per row: the scores' float32 sums are off by at most (dim + 4) 2^-23 of their
    terms' magnitudes (`reach`), which changes a probability by the factor e^(2 d); a probability is rounded to bfloat16
    (2^-8) and its exponential to 2^-22; sums of n terms in float32 to n 2^-23; the output once to its type."""
    dim = cache["k_codes"].shape[-1]
    want = fo.attend(cache, queries, table, lengths, scale, causal)
    for i, (o, size, reach) in enumerate(want):
        d = (dim + 4) * 2.0**-23 * reach[..., None]
        n = min(max(int(lengths[i]), 1), len(table[i]) * cache["k_codes"].shape[2])
        tol = (2.0**-8 + 4 * d + (2 * n + 8) * 2.0**-23) * size + HALF_STEP[dtype] * np.abs(o) + 1e-38
        if dtype == torch.float16:
            tol = tol + 2.0**-25  # half the smallest subnormal
        x = got[i].float().cpu().numpy().astype(np.float64)
        np.testing.assert_array_equal(np.isnan(x), np.isnan(o), err_msg=f"sequence {i}")
        bad = np.abs(x - o) > tol
        assert not bad.any(), f"sequence {i}: {bad.sum()} of {bad.size} outside; worst {np.nanmax(np.abs(x - o) / tol)} of the tolerance"
