"""Attention over the 8-bit cache where small probabilities carry a row: one token far ahead whose value is 0 or small, as the
first token of a sequence often is.  Against the definition in 64 bits, each probability held to its own rounding."""

import numpy as np
import pytest
import torch

from _kv8 import HALF_STEP, as_dict, make_cache, make_table
from deepcompressor_amd.nn.patch import Fp8KVCache

pytestmark = pytest.mark.gpu

# float16 probabilities have steps of 2^-24 below 2^-14, and 1 is held as 2^14 for single tokens, as 2^8 against a running maximum that
# may lag by 2^6 for chunks: half a step relative to the row's largest
FLOOR = {"tokens": 2.0**-39, "chunks": 2.0**-33}
SIZES = {"tokens": (1, 2, 1), "chunks": (8, 8, 330)}  # cache heads, query heads on each, queries: what reaches each kernel


def tensor(a):
    return torch.tensor(np.asarray(a), dtype=torch.int32, device="cuda")


def dense(cache, pages, n, q, scale):
    """Probabilities relative to the row's largest [row][head][token], keys and values [head][token][channel], and the largest sum of
    a score's terms' magnitudes [row][head]; float64, every query seeing all of the n tokens."""
    c = as_dict(cache)
    heads, dim = c["k_codes"].shape[1], c["k_codes"].shape[3]
    k = (c["k_codes"] * c["k_scales"].astype(np.float64)[..., None, None])[pages].transpose(1, 0, 2, 3).reshape(heads, -1, dim)[:, :n]
    v = (c["v_codes"] * c["v_scales"].astype(np.float64)[..., None, None])[pages].transpose(1, 0, 3, 2).reshape(heads, -1, dim)[:, :n]
    group = q.shape[1] // heads
    p, reach = [], []
    for h in range(q.shape[1]):
        s = q[:, h] @ k[h // group].T * scale
        p.append(np.exp(s - s.max(-1, keepdims=True)))
        reach.append((np.abs(q[:, h]) @ np.abs(k[h // group]).T).max(-1) * abs(scale))
    return np.stack(p, 1), v, np.stack(reach, 1)


def check(got, cache, pages, n, q, scale, dtype, rounding):
    """rounding(p) -> by how much a probability may be off.  Beside it, as everywhere: scores' float32 sums, off by (dim + 4) 2^-23 of
    their terms' magnitudes, the exponential (2^-22), sums of n terms in float32, one rounding of the output."""
    p, v, reach = dense(cache, pages, n, q, scale)
    group = q.shape[1] // v.shape[0]
    for h in range(q.shape[1]):
        total, values = p[:, h].sum(-1)[:, None], v[h // group]
        o, size = p[:, h] @ values / total, p[:, h] @ np.abs(values) / total
        e = rounding(p[:, h])
        d = (q.shape[-1] + 4) * 2.0**-23 * reach[:, h, None]
        tol = (e @ np.abs(values) + np.abs(o) * e.sum(-1)[:, None]) / total + (4 * d + (2 * n + 8) * 2.0**-23) * size + HALF_STEP[dtype] * np.abs(o)
        tol = tol + (2.0**-25 if dtype == torch.float16 else 1e-38)
        x = got[:, h].double().cpu().numpy()
        bad = ~(np.abs(x - o) <= tol)
        assert not bad.any(), f"head {h}: {bad.sum()} of {bad.size} outside; worst {np.max(np.abs(x - o) / tol)} of the tolerance"


def ahead(kernel, dtype, lead, at, n, dim, page, size=1.0, sink=0.0, small=0):
    """A cache of n tokens, values around 1 (times ``size`` but for the first ``small``), token ``at`` ``lead`` ahead of the others,
    its value ``sink``; its table; queries."""
    heads, group, rows = SIZES[kernel]
    g = torch.Generator().manual_seed(int(lead * 10) + n + dim)
    key, value = torch.randn((n, heads, dim), generator=g) * 0.2, (torch.randn((n, heads, dim), generator=g) * 0.3 + 1) * size
    value[:small] /= size
    key[:, :, 0] = 0
    key[at, :, 0], value[at] = lead, sink
    q = torch.randn((rows, heads * group, dim), generator=g) * 0.5
    q[..., 0] = 1.0
    cache, table = make_cache(-(-n // page) + 2, heads, dim, page, 0), make_table([n], page, -(-n // page), -(-n // page) + 2, 1)
    cache.append(key.cuda(), value.cuda(), tensor(table), tensor([0]), starts=tensor([0, n]))
    return cache, table, q.to(dtype)


@pytest.mark.parametrize("kernel,n", [("tokens", 4096), ("tokens", 60), ("chunks", 1000)])
@pytest.mark.parametrize("lead", [0, 14, 16, 18, 20])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_one_token_far_ahead(kernel, n, lead, dtype):
    for at, page, dim in ((0, 64, 128), (n - 30, 16, 64)):
        cache, table, q = ahead(kernel, dtype, lead, at, n, dim, page)
        out = cache.attend(q.cuda()[None], tensor(table), tensor([n]), causal=False, scale=1.0)[0]
        rounding = (lambda p: np.maximum(2.0**-11 * p, np.minimum(p, FLOOR[kernel]))) if dtype == torch.float16 else (lambda p: 2.0**-8 * p)
        check(out, cache, table[0], n, q.double().numpy(), 1.0, dtype, rounding)


@pytest.mark.parametrize("kernel,n", [("tokens", 4096), ("chunks", 1000)])
@pytest.mark.parametrize("lead", [30, 60])
def test_one_token_beyond_the_reach_of_float16(kernel, n, lead):
    """Steps of 64 tokens that hold no larger probability go on in bfloat16; the far token's own step may lose its others, and of
    chunks so may the step behind it, where the loop without masks is left."""
    for at in (0, n - 30):
        cache, table, q = ahead(kernel, torch.float16, lead, at, n, 64, 64)
        out = cache.attend(q.cuda()[None], tensor(table), tensor([n]), causal=False, scale=1.0)[0]
        behind = np.arange(n) // 64 - at // 64
        half = np.where((behind == 0) | ((behind == 1) & (kernel == "chunks")), 1.0, 2.0**-8)
        check(out, cache, table[0], n, q.double().numpy(), 1.0, torch.float16, lambda p: half * p)


@pytest.mark.parametrize("kernel,n", [("tokens", 4096), ("chunks", 1000)])
@pytest.mark.parametrize("lead,size", [(10, 100.0), (16, 100.0), (14, 2.0**20), (18, 2.0**20)])
def test_large_values_at_small_probabilities(kernel, n, lead, size):
    """Behind a page of values around 1.  Its scale is within float16's reach of the others', or it is not: then the first 64
    tokens' probabilities are rounded to bfloat16."""
    cache, table, q = ahead(kernel, torch.float16, lead, 0, n, 64, 16, size, sink=1.0, small=16)
    out = cache.attend(q.cuda()[None], tensor(table), tensor([n]), causal=False, scale=1.0)[0]
    half = np.where((np.arange(n) < 64) & (size > 2**14), 2.0**-8, 2.0**-11)
    check(out, cache, table[0], n, q.double().numpy(), 1.0, torch.float16, lambda p: np.maximum(half * p, np.minimum(p, FLOOR[kernel])))


@pytest.mark.parametrize("size", [1.0, 2.0**-14])
@pytest.mark.parametrize("kernel", ["tokens", "chunks"])
def test_unseen_pages_do_not_change_the_answer(kernel, size):
    """Pages that the table lists behind the last token that a query sees hold anything: scales of any kind there, equal bits."""
    heads, group, page, cols = (2, 4, 16, 12) if kernel == "tokens" else (8, 8, 16, 12)
    lengths = [70, 5, 130] if kernel == "tokens" else [40] * 9
    pool = len(lengths) * cols
    made = make_cache(pool, heads, 64, page, 0)
    table = np.random.RandomState(0).permutation(pool).reshape(-1, cols).astype(np.int32)
    g = torch.Generator().manual_seed(1)
    starts = np.concatenate([[0], np.cumsum(lengths)])
    key, value = torch.randn((2, int(starts[-1]), heads, 64), generator=g)
    made.append(key.cuda(), (value * size).cuda(), tensor(table), tensor([0] * len(lengths)), starts=tensor(starts))
    counts = [1] * len(lengths) if kernel == "tokens" else lengths
    q = torch.randn((sum(counts), heads * group, 64), generator=g).half().cuda()
    at = tensor(np.concatenate([[0], np.cumsum(counts)]))
    unseen = torch.tensor(np.concatenate([t[-(-n // page):] for t, n in zip(table, lengths)]), device="cuda").long()
    want = None
    for scale in (1.0, float("nan"), float("inf"), 2.0**60, 2.0**-100, 3e-39):
        scales = [s.clone() for s in (made.k_scales, made.v_scales)]
        for s in scales:
            s[unseen] = scale
        cache = Fp8KVCache.from_buffers(made.k_codes, scales[0], made.v_codes, scales[1])
        out = cache.attend(q, tensor(table), tensor(lengths), starts=at)
        want = out if want is None else want
        assert torch.isfinite(out).all() and torch.equal(out, want), scale
