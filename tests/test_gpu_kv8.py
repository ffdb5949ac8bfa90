"""The 8-bit key / value cache: append and attention against their definitions in 64 bits."""

import numpy as np
import pytest
import torch

import fp8_oracle as fo
from _kv8 import as_dict, check_attention, fill, make_cache, make_table, values
from deepcompressor_amd.nn.patch import Fp8BlockLinear, Fp8KVCache

pytestmark = pytest.mark.gpu


def same_cache(cache, want):
    for name in ("k_codes", "v_codes"):
        np.testing.assert_array_equal(values(getattr(cache, name)), want[name], err_msg=name)
    for name in ("k_scales", "v_scales"):
        np.testing.assert_array_equal(getattr(cache, name).cpu().numpy(), want[name], err_msg=name)


def tensor(a):
    return torch.tensor(np.asarray(a), dtype=torch.int32, device="cuda")


def split(t, starts):
    return [t[int(a):int(b)] for a, b in zip(starts[:-1], starts[1:])]


def append_both(cache, table, lengths, counts, seed, dtype, scale=1.0, packed=True):
    """The operator and its definition on the same tokens; returns the definition's cache."""
    g = torch.Generator().manual_seed(seed)
    _, heads, _, dim = cache.k_codes.shape
    starts = np.concatenate([[0], np.cumsum(counts)])
    shape = (int(starts[-1]), heads, dim)
    size = torch.exp(2 * torch.randn((shape[0], 1, 1), generator=g)) * scale
    key, value = ((torch.randn(shape, generator=g) * size).to(dtype) for _ in range(2))
    want = as_dict(cache)
    as_list = lambda t: [x.float().numpy() for x in split(t, starts)]  # noqa: E731
    fo.append(want, as_list(key), as_list(value), table, lengths, counts)
    if packed:
        cache.append(key.cuda(), value.cuda(), tensor(table), tensor(lengths), starts=tensor(starts))
    else:
        to = lambda t: t.view(len(counts), -1, heads, dim).cuda()  # noqa: E731
        cache.append(to(key), to(value), tensor(table), tensor(lengths))
    return want


@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_append(page, dim, dtype):
    """Empty sequences, single tokens, starts inside a page, pages that end inside the new tokens; twice in a row."""
    lengths, counts = [0, 5, page - 1, page, 0, 3 * page + 7], [page + 3, 1, 2, 1, 0, 2 * page]
    total = [a + b + 4 for a, b in zip(lengths, counts)]
    table = make_table(total, page, 8, 40, 1)
    cache = make_cache(40, 2, dim, page, 0)
    want = append_both(cache, table, np.zeros(6, dtype=np.int32), lengths, 2, dtype)
    same_cache(cache, want)
    want = append_both(cache, table, lengths, counts, 3, dtype, scale=4.0)
    same_cache(cache, want)
    want = append_both(cache, table, [a + b for a, b in zip(lengths, counts)], [4] * 6, 4, dtype, scale=0.01, packed=False)
    same_cache(cache, want)


def test_append_token_by_token_grows_scales():
    cache, table = make_cache(3, 3, 64, 16, 0), make_table([40], 16, 3, 3, 0)
    for t in range(40):
        want = append_both(cache, table, [t], [1], t, torch.bfloat16, scale=2.0 ** (t % 7), packed=t % 2 == 0)
        same_cache(cache, want)


def test_append_values_that_are_not_finite_and_zero():
    cache, table = make_cache(4, 1, 64, 16, 0), make_table([20], 16, 2, 4, 0)
    key = torch.randn((20, 1, 64))
    key[3, 0, 5], key[4, 0, 6], key[18, 0, 7] = float("nan"), float("inf"), float("-inf")
    value = torch.zeros((20, 1, 64))
    value[17, 0, 1] = 1e-41
    want = as_dict(cache)
    fo.append(want, [key.numpy()], [value.numpy()], table, [0], [20])
    cache.append(key.cuda(), value.cuda(), tensor(table), tensor([0]), starts=tensor([0, 20]))
    same_cache(cache, want)


def test_append_bad_tables_stay_inside():
    """Pages outside the pool, tokens behind the table's end, lengths and starts that make no sense: what has no place is
    dropped, everything else is as the definition has it."""
    cache = make_cache(6, 2, 64, 16, 0)
    table = np.array([[0, 99, 1], [-5, 2, 3], [4, 5, -1]], dtype=np.int32)
    want = append_both(cache, table, [0, 10, 40], [60, 30, 30], 1, torch.bfloat16)
    same_cache(cache, want)
    key = torch.randn((10, 2, 64), device="cuda")
    before = as_dict(cache)
    cache.append(key, key, tensor(table), tensor([48, 1000, 2**31 - 1]), starts=tensor([0, 4, 8, 10]))
    cache.append(key, key, tensor(table), tensor([0, 0, 0]), starts=tensor([10, 10, 3, 3]))
    cache.append(key[:0], key[:0], tensor(table), tensor([0, 0, 0]), starts=tensor([0, 0, 0, 0]))
    same_cache(cache, before)


def test_append_leaves_other_memory_alone():
    cache = make_cache(5, 2, 128, 64, 0)
    table = make_table([10], 64, 2, 5, 3)
    before = as_dict(cache)
    fill(cache, table, [10], 0)
    page = int(table[0, 0])
    after = as_dict(cache)
    for name in before:
        rest = [p for p in range(5) if p != page]
        np.testing.assert_array_equal(after[name][rest], before[name][rest])
    np.testing.assert_array_equal(after["k_codes"][page][:, 10:], before["k_codes"][page][:, 10:])
    np.testing.assert_array_equal(after["v_codes"][page][:, :, 10:], before["v_codes"][page][:, :, 10:])


def test_append_strides():
    """Slices of a joint projection, and heads before tokens."""
    joint = torch.randn((3, 9, 4 * 64 * 3), device="cuda", dtype=torch.bfloat16)
    _, k, v = joint.view(3, 9, 3, 4, 64).unbind(2)
    table, lengths = tensor(make_table([20] * 3, 16, 2, 6, 0)), tensor([4, 0, 7])
    one, two, three = (make_cache(6, 4, 64, 16, 0) for _ in range(3))
    one.append(k, v, table, lengths)
    two.append(k.contiguous(), v.contiguous(), table, lengths)
    three.append(k.transpose(1, 2).contiguous().transpose(1, 2), v.transpose(1, 2).contiguous().transpose(1, 2), table, lengths)
    for other in (two, three):
        for name in ("k_codes", "v_codes"):
            assert torch.equal(getattr(one, name).view(torch.uint8), getattr(other, name).view(torch.uint8))
    odd = torch.randn((3, 9, 4 * 64 + 1), device="cuda", dtype=torch.bfloat16)[..., 1:].unflatten(-1, (4, 64))
    one.append(odd, odd, table, lengths)
    two.append(odd.contiguous(), odd.contiguous(), table, lengths)
    assert torch.equal(one.k_codes.view(torch.uint8), two.k_codes.view(torch.uint8))


# ---- attention -----------------------------------------------------------------------------------------------------------


def attend_both(page, dim, heads, group, totals, counts, dtype, seed, causal=True, packed=True, cols=None, scale=None, size=1.0):
    cols = cols or max(1, -(-max(totals) // page) + 2)
    pool = sum(-(-t // page) for t in totals) + 2
    table = make_table(totals, page, cols, pool, seed)
    cache = make_cache(pool, heads, dim, page, seed)
    fill(cache, table, totals, seed, scale=size)
    g = torch.Generator().manual_seed(seed + 1)
    starts = np.concatenate([[0], np.cumsum(counts)])
    q = torch.randn((int(starts[-1]), heads * group, dim), generator=g).mul(2).to(dtype)
    kwargs = dict(scale=scale, causal=causal)
    if packed:
        out = cache.attend(q.cuda(), tensor(table), tensor(totals), starts=tensor(starts), **kwargs)
        got = split(out, starts)
    else:
        out = cache.attend(q.view(len(counts), -1, heads * group, dim).cuda(), tensor(table), tensor(totals), **kwargs)
        got = list(out)
    check_attention(got, [x.double().numpy() for x in split(q, starts)], as_dict(cache), table, totals, dim**-0.5 if scale is None else scale,
                    causal, dtype)


@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_single_tokens(page, dim, dtype):
    attend_both(page, dim, 2, 4, [1, 2, 15, 16, 17, 63, 64, 65, 200, 0], [1] * 10, dtype, page + dim, packed=False)


@pytest.mark.parametrize("group", [1, 2, 3, 7, 8, 16, 17, 32])
def test_groups(group):
    attend_both(32, 64, 2, group, [70, 1, 130], [1, 1, 1], torch.bfloat16, group, packed=False)
    attend_both(32, 64, 2, group, [70, 9, 130], [20, 9, 1], torch.bfloat16, group)


@pytest.mark.parametrize("page", [16, 64, 128])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("causal", [True, False])
def test_chunks(page, dim, causal):
    """Whole prompts, chunks behind older tokens, no queries at all, fewer tokens than queries (rows that see nothing)."""
    attend_both(page, dim, 2, 2, [90, 150, 40, 5, 130], [90, 37, 0, 12, 1], torch.float16, page + dim, causal)


def test_long_sequence_is_split():
    attend_both(64, 64, 1, 1, [5000], [1], torch.bfloat16, 0, packed=False)
    attend_both(16, 128, 1, 4, [3001, 9], [1, 1], torch.float16, 1)


def test_many_queries_of_one_sequence():
    attend_both(64, 64, 1, 2, [400], [400], torch.bfloat16, 0)
    attend_both(64, 128, 1, 1, [300], [300], torch.float16, 0, packed=False)


def test_many_sequences():
    rng = np.random.RandomState(0)
    attend_both(16, 64, 1, 2, list(rng.randint(0, 40, 150)), [1] * 150, torch.bfloat16, 0)


def test_sharp_scores_and_large_values():
    attend_both(16, 64, 1, 2, [100, 33], [3, 1], torch.bfloat16, 3, scale=1.5)
    attend_both(16, 64, 1, 2, [100, 33], [3, 1], torch.bfloat16, 3, scale=-0.2, size=300.0)
    attend_both(16, 64, 1, 2, [100, 33], [3, 1], torch.bfloat16, 3, scale=0.0)


def test_lengths_behind_the_table_and_missing_pages():
    page, totals = 16, [40, 64, 30]
    table = make_table(totals, page, 3, 12, 0)
    cache = make_cache(12, 1, 64, page, 0)
    fill(cache, table, [min(t, 48) for t in totals], 0)
    table[0, 1], table[2, :] = 77, -3  # a page outside the pool in the middle; no page at all
    q = torch.randn((3, 2, 3, 64)).to(torch.bfloat16)
    out = cache.attend(q.cuda(), tensor(table), tensor(totals))
    check_attention(list(out), list(q.double().numpy()), as_dict(cache), table, totals, 0.125, True, torch.bfloat16)
    assert (out[2] == 0).all()


def test_nan_of_a_later_token_stays_with_those_that_see_it():
    cache, table = make_cache(4, 1, 64, 32, 0), make_table([50], 32, 2, 4, 0)
    k, v = torch.randn((2, 50, 1, 64))
    v[45, 0, 7] = float("nan")
    k[47, 0, 0] = float("nan")
    cache.append(k.cuda(), v.cuda(), tensor(table), tensor([0]), starts=tensor([0, 50]))
    q = torch.randn((50, 2, 64)).to(torch.bfloat16)
    out = cache.attend(q.cuda(), tensor(table), tensor([50]), starts=tensor([0, 50]))
    assert torch.isfinite(out[:45]).all()
    assert torch.isnan(out[45:47, :, 7]).all() and torch.isfinite(out[45:47, :, :7]).all() and torch.isfinite(out[45:47, :, 8:]).all()
    assert torch.isnan(out[47:]).all()


def test_queries_that_are_not_finite():
    cache, table = make_cache(4, 1, 64, 32, 0, garbage=False), make_table([50], 32, 2, 4, 0)
    fill(cache, table, [50], 1)
    q = torch.randn((4, 2, 64)).to(torch.bfloat16)
    q[1, 0, 3], q[2, 1, 4] = float("nan"), float("inf")
    out = cache.attend(q.cuda(), tensor(table), tensor([50]), starts=tensor([0, 4]))
    assert torch.isnan(out[1, 0]).all() and torch.isnan(out[2, 1]).all()
    assert torch.isfinite(out[[0, 3]]).all() and torch.isfinite(out[1, 1]).all() and torch.isfinite(out[2, 0]).all()


def test_rows_without_a_sequence():
    """Packed rows before the first and behind the last sequence: as they were in `out`, 0 without it."""
    for counts in ([5, 1], [200, 1]):
        totals = [250, 60]
        cache, table = make_cache(24, 2, 64, 16, 0), make_table(totals, 16, 16, 24, 0)
        fill(cache, table, totals, 2)
        starts = tensor(np.concatenate([[3], 3 + np.cumsum(counts)]))
        q = torch.randn((sum(counts) + 50, 4, 64), device="cuda").to(torch.float16)
        out = torch.full_like(q, 7.0)
        made = cache.attend(q, tensor(table), tensor(totals), starts=starts)
        cache.attend(q, tensor(table), tensor(totals), starts=starts, out=out)
        end = int(starts[-1])
        assert (out[:3] == 7).all() and (out[end:] == 7).all() and (made[:3] == 0).all() and (made[end:] == 0).all()
        assert torch.equal(out[3:end], made[3:end])


def test_attend_strides_and_out():
    cache, table = make_cache(8, 2, 64, 16, 0), make_table([40, 30], 16, 3, 8, 0)
    fill(cache, table, [40, 30], 2)
    joint = torch.randn((2, 5, 3, 4, 64), device="cuda").to(torch.bfloat16)
    table, lengths = tensor(table), tensor([40, 30])
    want = cache.attend(joint[:, :, 1].contiguous(), table, lengths)
    assert torch.equal(cache.attend(joint[:, :, 1], table, lengths), want)
    out = torch.zeros((2, 4, 5, 64), device="cuda", dtype=torch.bfloat16).transpose(1, 2)
    assert cache.attend(joint[:, :, 1], table, lengths, out=out).data_ptr() == out.data_ptr()
    assert torch.equal(out, want)


def test_offsets_beyond_32_bits():
    """A pool whose keys take more than 2^32 bytes: the pages at its end hold the same answers as those at its start."""
    pool = 2**32 // (8 * 128 * 128) + 8
    cache = Fp8KVCache.from_buffers(*(torch.empty(s, dtype=d, device="cuda") if d == torch.float32 else
                                      torch.empty(s, dtype=torch.uint8, device="cuda").view(d) for s, d in
                                      (((pool, 8, 128, 128), torch.float8_e4m3fn), ((pool, 8), torch.float32),
                                       ((pool, 8, 128, 128), torch.float8_e4m3fn), ((pool, 8), torch.float32))))
    kv = torch.randn((2, 1, 200, 8, 128), device="cuda", generator=torch.Generator("cuda").manual_seed(0)).to(torch.bfloat16)
    q = torch.randn((1, 3, 16, 128), device="cuda", generator=torch.Generator("cuda").manual_seed(1)).to(torch.bfloat16)
    outs = []
    for pages in ([0, 1], [pool - 1, pool - 2]):
        cache.append(kv[0], kv[1], tensor([pages]), tensor([0]))
        outs.append(cache.attend(q, tensor([pages]), tensor([200])))
    assert torch.isfinite(outs[0]).all() and torch.equal(outs[0], outs[1])


def test_streams_and_graphs():
    """Decode steps captured once and replayed with new tokens and lengths, against the same steps run one by one; two graphs
    whose workspaces are their own; another stream."""
    def step(cache, q, k, v, table, lengths):
        cache.append(k, v, table, lengths)
        return cache.attend(q, table, lengths + 1)

    table = tensor(make_table([600] * 2, 64, 10, 20, 0))
    fresh = lambda: make_cache(20, 2, 128, 64, 0)  # noqa: E731
    one, two = fresh(), fresh()
    g = torch.Generator("cuda").manual_seed(0)
    rand = lambda *s: torch.randn(s, device="cuda", generator=g).to(torch.bfloat16)  # noqa: E731
    prompt = rand(2, 2, 500, 2, 128)
    for c in (one, two):
        c.append(prompt[0], prompt[1], table, tensor([0, 0]))
    q, k, v, lengths = rand(2, 1, 8, 128), rand(2, 1, 2, 128), rand(2, 1, 2, 128), tensor([500, 500])
    step(one, q, k, v, table, lengths)
    graphs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()]
    outs = []
    for graph in graphs:
        with torch.cuda.graph(graph):
            outs.append(step(one, q, k, v, table, lengths))
    for t in range(4):
        for x, y in ((q, rand(2, 1, 8, 128)), (k, rand(2, 1, 2, 128)), (v, rand(2, 1, 2, 128)), (lengths, tensor([500 + t, 500 + t]))):
            x.copy_(y)
        graphs[t % 2].replay()
        want = step(two, q, k, v, table, lengths)
        torch.cuda.synchronize()
        assert torch.equal(outs[t % 2], want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = two.attend(q, table, lengths + 1)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)


def test_a_layer_end_to_end():
    """Projections, append and attention together as a decoder layer runs them: a prompt at once, and the same tokens in
    two chunks and then singly, give the same cache and (to the rounding of one probability) the same outputs."""
    torch.manual_seed(0)
    hidden, heads, group, dim, n = 256, 2, 2, 64, 70
    make = lambda i, o: Fp8BlockLinear.from_linear(torch.nn.Linear(i, o, bias=False, device="cuda", dtype=torch.bfloat16))  # noqa: E731
    qp, kp, vp, op = make(hidden, heads * group * dim), make(hidden, heads * dim), make(hidden, heads * dim), make(heads * group * dim, hidden)
    x = torch.randn((1, n, hidden), device="cuda", dtype=torch.bfloat16)
    table = tensor(make_table([n], 16, 5, 9, 0))

    def run(cache, x, at):
        m = x.shape[1]
        heads_of = lambda t, h: t.view(1, m, h, dim)  # noqa: E731
        cache.append(heads_of(kp(x), heads), heads_of(vp(x), heads), table, tensor([at]))
        return op(cache.attend(heads_of(qp(x), heads * group), table, tensor([at + m])).view(1, m, -1))

    with torch.no_grad():
        whole, parts = make_cache(9, heads, dim, 16, 0), make_cache(9, heads, dim, 16, 0)
        want = run(whole, x, 0)
        got, at = [], 0
        for m in (32, 32, 1, 1, 1, 1, 1, 1):
            got.append(run(parts, x[:, at:at + m], at))
            at += m
        got = torch.cat(got, dim=1)
    assert torch.isfinite(want).all()
    full = table[0, :4].long()
    assert torch.equal(whole.k_codes[full].float(), parts.k_codes[full].float())  # whole pages were written in one call
    assert (want.float() - got.float()).norm() <= 0.05 * want.float().norm()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("counts", [[1, 1], [100, 70]])
def test_values_of_far_apart_sizes(dtype, counts):
    """Pages whose values differ by up to 2^46 (float32 tokens), and scores that pick the small ones: each row's output is held to
    the sizes it attends to, so what is lost beside the large pages shows."""
    totals, page = [200, 130], 16
    table = make_table(totals, page, 16, 30, 5)
    cache = make_cache(30, 1, 64, page, 0)
    g = torch.Generator().manual_seed(3)
    starts = np.concatenate([[0], np.cumsum(totals)])
    key = torch.randn((int(starts[-1]), 1, 64), generator=g)
    value = torch.randn((int(starts[-1]), 1, 64), generator=g)
    for i, n in enumerate(totals):
        for t in range(n):
            value[starts[i] + t] *= 2.0 ** (-30 + 5 * (t // page % 10)) if i == 0 else 2.0 ** (12 - 7 * (t // page % 7))
            if t // page % 3 == 0:
                key[starts[i] + t, 0, 0] += 40.0  # rows look here, where the values are small for some
    cache.append(key.cuda(), value.cuda(), tensor(table), tensor([0, 0]), starts=tensor(starts))
    q = torch.randn((sum(counts), 2, 64), generator=g).to(dtype)
    q[:, 0, 0] = 8.0
    out = cache.attend(q.cuda(), tensor(table), tensor(totals), starts=tensor(np.concatenate([[0], np.cumsum(counts)])))
    at = np.concatenate([[0], np.cumsum(counts)])
    check_attention(split(out, at), [x.double().numpy() for x in split(q, at)], as_dict(cache), table, totals, 0.125, True, dtype)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("counts", [[1, 1], [130, 70]])
def test_scales_that_are_no_powers_of_two(dtype, counts):
    """A cache filled by other means: attention takes any positive scale."""
    totals = [200, 130]
    table = make_table(totals, 32, 8, 16, 5)
    made = make_cache(16, 2, 64, 32, 0, garbage=False)
    fill(made, table, totals, 1)
    g = torch.Generator("cuda").manual_seed(0)
    scales = [s * (0.3 + 3 * torch.rand(s.shape, generator=g, device="cuda")) for s in (made.k_scales, made.v_scales)]
    cache = Fp8KVCache.from_buffers(made.k_codes, scales[0], made.v_codes, scales[1])
    q = torch.randn((sum(counts), 4, 64), generator=torch.Generator().manual_seed(2)).to(dtype)
    at = np.concatenate([[0], np.cumsum(counts)])
    out = cache.attend(q.cuda(), tensor(table), tensor(totals), starts=tensor(at))
    check_attention(split(out, at), [x.double().numpy() for x in split(q, at)], as_dict(cache), table, totals, 0.125, True, dtype)


def test_no_sequences_at_all():
    cache = make_cache(2, 1, 64, 16, 0)
    q = torch.randn((3, 2, 64), device="cuda").half()
    none = torch.zeros((0, 2), dtype=torch.int32, device="cuda")
    assert (cache.attend(q, none, tensor([]), starts=tensor([0])) == 0).all()
    out = torch.full_like(q, 3.0)
    cache.attend(q, none, tensor([]), starts=tensor([0]), out=out)
    assert (out == 3).all()
    cache.append(q[:, :1], q[:, :1], none, tensor([]), starts=tensor([0]))
    assert cache.attend(q[:0].unsqueeze(0), tensor([[0]]), tensor([5])).shape == (1, 0, 2, 64)


def test_lengths_far_beyond_the_table():
    """The queries' places count from the given length, also where the table holds fewer tokens."""
    table = make_table([48, 48], 16, 3, 8, 0)
    cache = make_cache(8, 1, 64, 16, 0)
    fill(cache, table, [48, 48], 0)
    totals = [60, 2**31 - 1]
    q = torch.randn((2, 20, 2, 64), generator=torch.Generator().manual_seed(1)).to(torch.bfloat16)
    out = cache.attend(q.cuda(), tensor(table), tensor(totals))
    check_attention(list(out), list(q.double().numpy()), as_dict(cache), table, totals, 0.125, True, torch.bfloat16)


# ---- chunks of many rows: 160 workgroups of 128 rows and more have a kernel of their own -----------------------------------------

WIDE = (8, 8)  # cache heads, query heads on each: from 320 queries on


@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("causal", [True, False])
def test_wide_chunks(page, dim, dtype, causal):
    """Whole prompts, chunks behind older tokens, no queries at all, fewer tokens than queries, single tokens between them."""
    attend_both(page, dim, *WIDE, [190, 250, 40, 5, 130, 0], [190, 129, 0, 12, 1, 3], dtype, page + dim, causal)


@pytest.mark.parametrize("heads,group", [(1, 64), (7, 9), (40, 2), (33, 3)])
def test_wide_groups(heads, group):
    attend_both(64, 64, heads, group, [170, 190], [170, 180], torch.bfloat16, group)
    attend_both(16, 128, heads, group, [350], [350], torch.float16, group, packed=False)


def test_wide_chunks_behind_a_long_past():
    attend_both(128, 128, 2, 8, [2500, 1411], [700, 650], torch.float16, 0)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_wide_sharp_scores(dtype):
    """Maxima that grow all along the tokens, by less and by far more than the steps without a rescaling bear."""
    for scale, size in ((1.5, 1.0), (-0.2, 300.0), (0.0, 1.0), (0.02, 1.0)):
        attend_both(16, 64, *WIDE, [300, 133], [300, 33], dtype, 3, scale=scale, size=size)
    cache, table = make_cache(30, 8, 64, 16, 0), make_table([350], 16, 24, 30, 0)
    key, value = torch.randn((2, 350, 8, 64), generator=torch.Generator().manual_seed(0))
    key[..., 0] = torch.arange(350)[:, None] / 20
    cache.append(key.cuda(), value.cuda(), tensor(table), tensor([0]), starts=tensor([0, 350]))
    q = torch.randn((350, 64, 64), generator=torch.Generator().manual_seed(1)).to(dtype)
    for first in (4.0, -4.0, 40.0):
        q[..., 0] = first
        out = cache.attend(q.cuda()[None], tensor(table), tensor([350]), causal=False, scale=1.0)
        check_attention(list(out), [q.double().numpy()], as_dict(cache), table, [350], 1.0, False, dtype)


def test_wide_missing_pages_and_lengths_behind_the_table():
    page, totals = 16, [200, 400, 130]
    table = make_table(totals, page, 12, 60, 0)
    cache = make_cache(60, 8, 64, page, 0)
    fill(cache, table, [min(t, 192) for t in totals], 0)
    table[0, 3], table[1, 0], table[2, :] = 77, -1, -3  # pages outside the pool in the middle and first; no page at all
    q = torch.randn((3, 120, 64, 64), generator=torch.Generator().manual_seed(0)).to(torch.bfloat16)
    out = cache.attend(q.cuda(), tensor(table), tensor(totals))
    check_attention(list(out), list(q.double().numpy()), as_dict(cache), table, totals, 0.125, True, torch.bfloat16)
    assert (out[2] == 0).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_wide_values_that_are_not_finite(dtype):
    """A NaN is seen by the queries behind it only, in keys and in values; a query's own stays its own."""
    cache, table = make_cache(30, 8, 64, 16, 0), make_table([400], 16, 26, 30, 0)
    k, v = torch.randn((2, 400, 8, 64), generator=torch.Generator().manual_seed(0))
    v[333, :, 7] = float("nan")
    v[334, :, 9] = float("-inf")
    k[350, :, 0] = float("nan")
    cache.append(k.cuda(), v.cuda(), tensor(table), tensor([0]), starts=tensor([0, 400]))
    q = torch.randn((400, 64, 64), generator=torch.Generator().manual_seed(1)).to(dtype)
    q[10, 3, 3], q[20, 5, 4] = float("nan"), float("inf")
    out = cache.attend(q.cuda(), tensor(table), tensor([400]), starts=tensor([0, 400]))
    bad = torch.zeros(out.shape, dtype=torch.bool, device="cuda")
    bad[333:, :, 7] = bad[334:, :, 9] = bad[350:] = bad[10, 3] = bad[20, 5] = True
    assert torch.equal(torch.isnan(out), bad)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_wide_scales_of_all_kinds(dtype):
    """Scales that are no powers of two, on some pages or on all, and values whose sizes differ by up to 2^46."""
    totals = [300, 230]
    table = make_table(totals, 32, 10, 20, 5)
    made = make_cache(20, 8, 64, 32, 0, garbage=False)
    fill(made, table, totals, 1)
    g = torch.Generator("cuda").manual_seed(0)
    q = torch.randn((340, 64, 64), generator=torch.Generator().manual_seed(2)).to(dtype)
    at = np.array([0, 200, 340])
    for pages, far in ((20, 0), (4, 0), (0, 23), (20, 23)):
        scales = []
        for s in (made.k_scales, made.v_scales):
            s = s.clone()
            s[:pages] *= 0.3 + 3 * torch.rand((pages, 8), generator=g, device="cuda")
            scales.append(s)
        scales[1] *= torch.exp2(torch.randint(-far, far + 1, scales[1].shape, generator=g, device="cuda").float())
        if dtype == torch.float16:
            scales[1] *= 2.0 ** -(far // 2)  # (outputs within float16)
        cache = Fp8KVCache.from_buffers(made.k_codes, scales[0], made.v_codes, scales[1])
        out = cache.attend(q.cuda(), tensor(table), tensor(totals), starts=tensor(at))
        check_attention(split(out, at), [x.double().numpy() for x in split(q, at)], as_dict(cache), table, totals, 0.125, True, dtype)


def test_wide_rows_without_a_sequence_strides_and_out():
    totals = [250, 160]
    cache, table = make_cache(30, 8, 64, 16, 0), make_table(totals, 16, 16, 30, 0)
    fill(cache, table, totals, 2)
    starts = tensor([3, 203, 363])
    joint = torch.randn((400, 3, 64, 64), device="cuda", generator=torch.Generator("cuda").manual_seed(0)).to(torch.float16)
    q = joint[:, 1]
    made = cache.attend(q, tensor(table), tensor(totals), starts=starts)
    assert torch.equal(made, cache.attend(q.contiguous(), tensor(table), tensor(totals), starts=starts))
    assert (made[:3] == 0).all() and (made[363:] == 0).all() and made[3:363].ne(0).any(dim=-1).all()
    joint[:, 2] = 7.0
    cache.attend(q, tensor(table), tensor(totals), starts=starts, out=joint[:, 2])
    assert torch.equal(joint[3:363, 2], made[3:363]) and (joint[:3, 2] == 7).all() and (joint[363:, 2] == 7).all()
    cache.attend(q, tensor(table), tensor(totals), starts=starts, out=q)  # in place: each row is read before it is written
    assert torch.equal(joint[3:363, 1], made[3:363])


def test_wide_offsets_beyond_32_bits():
    pool = 2**32 // (8 * 128 * 128) + 8
    cache = Fp8KVCache(pool, 8, 128, 128)
    kv = torch.randn((2, 1, 400, 8, 128), device="cuda", generator=torch.Generator("cuda").manual_seed(0)).to(torch.bfloat16)
    q = torch.randn((1, 390, 64, 128), device="cuda", generator=torch.Generator("cuda").manual_seed(1)).to(torch.bfloat16)
    outs = []
    for pages in ([0, 1, 2, 3], [pool - 1, pool - 2, pool - 4, pool - 3]):
        cache.append(kv[0], kv[1], tensor([pages]), tensor([0]))
        outs.append(cache.attend(q, tensor([pages]), tensor([400])))
    assert torch.isfinite(outs[0]).all() and torch.equal(outs[0], outs[1])


def test_wide_chunks_in_a_graph_and_on_two_streams():
    """A chunk's append and attention captured and replayed with new tokens, between eager calls; two streams at once, each with a
    split sequence and a chunk of its own."""
    table = tensor(make_table([500, 500], 64, 8, 20, 0))
    g = torch.Generator("cuda").manual_seed(0)
    rand = lambda *s: torch.randn(s, device="cuda", generator=g).to(torch.bfloat16)  # noqa: E731
    one, two = (make_cache(20, 8, 128, 64, 0) for _ in range(2))
    q, k, v, lengths = rand(2, 180, 64, 128), rand(2, 180, 8, 128), rand(2, 180, 8, 128), tensor([0, 0])

    def step(cache):
        cache.append(k, v, table, lengths)
        return cache.attend(q, table, lengths + 180)

    step(one)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(one)
    for t in range(3):
        for x in (q, k, v):
            x.copy_(rand(*x.shape))
        lengths.copy_(tensor([100 * t, 90 * t]))
        graph.replay()
        want = step(two)
        torch.cuda.synchronize()
        assert torch.equal(out, want)
    single = rand(1, 1, 64, 128)
    calls = [lambda: two.attend(q, table, lengths + 180), lambda: two.attend(single, table[:1], lengths[:1] + 180)]
    want = [f() for f in calls]
    torch.cuda.synchronize()
    sides, got = [torch.cuda.Stream(), torch.cuda.Stream()], []
    for t in range(6):
        with torch.cuda.stream(sides[t % 2]):
            got.append([f() for f in calls])
    torch.cuda.synchronize()
    for pair in got:
        assert torch.equal(pair[0], want[0]) and torch.equal(pair[1], want[1])


def test_a_page_seen_by_several_sequences():
    """A common beginning in full pages, behind which each sequence goes on in pages of its own; a page listed twice is seen twice."""
    cache, beginning = make_cache(12, 2, 64, 16, 0), [4, 7]
    g = torch.Generator().manual_seed(0)
    rand = lambda n: torch.randn((1, n, 2, 64), generator=g).cuda()  # noqa: E731
    cache.append(rand(32), rand(32), tensor([beginning]), tensor([0]))
    table = np.array([beginning + [1, 2], beginning + [3, 0], [4, 4, 7, 4]], dtype=np.int32)
    new = [torch.cat([rand(20), rand(20)]) for _ in range(2)]
    cache.append(*new, tensor(table[:2]), tensor([32, 32]))
    q = torch.randn((3, 2, 4, 64), generator=g).to(torch.bfloat16)
    totals = [52, 52, 60]
    out = cache.attend(q.cuda(), tensor(table), tensor(totals))
    check_attention(list(out), list(q.double().numpy()), as_dict(cache), table, totals, 0.125, True, torch.bfloat16)


def test_outputs_that_cannot_be_written():
    cache = make_cache(2, 1, 64, 16, 0)
    q = torch.randn((2, 3, 2, 64), device="cuda").half()
    args = (tensor([[0], [1]]), tensor([3, 3]))
    wide = torch.empty((2, 3, 2, 65), device="cuda", dtype=torch.float16)
    for out in (torch.empty_like(q[:1]), q.bfloat16(), wide[..., 1:], q[:1].expand(2, 3, 2, 64), q.transpose(2, 3).contiguous().transpose(2, 3),
                torch.empty((2, 3, 2, 66), device="cuda", dtype=torch.float16)[..., :64]):
        with pytest.raises(ValueError, match="out"):
            cache.attend(q, *args, out=out)
    one = torch.empty((2, 3, 2, 64), device="cuda", dtype=torch.float16)[:1].as_strided((1, 3, 2, 64), (0, 128, 64, 1))
    cache.append(q[:1, :, :1], q[:1, :, :1], args[0][:1], tensor([0]))
    assert torch.equal(cache.attend(q[:1], args[0][:1], args[1][:1], out=one), cache.attend(q[:1], args[0][:1], args[1][:1]))


def test_axes_of_size_one_may_have_any_stride():
    """A sequence, a token or a head cut out of a matrix with an odd pitch, which torch counts as contiguous where the odd strides
    belong to axes of size 1; and an output of one token in such a place."""
    for cut in (np.s_[:1, :1], np.s_[1:2, 2:3], np.s_[1:2], np.s_[:, 2:3], np.s_[1:2, 3:4, :1]):
        odd = torch.randn((4, 9, 4 * 64 + 1), device="cuda", dtype=torch.bfloat16)[..., 1:].unflatten(-1, (4, 64))[cut]
        count, new, heads = odd.shape[:3]
        table, lengths = tensor(make_table([20] * count, 16, 2, 2 * count, 0)), tensor([4] * count)
        caches = [make_cache(2 * count, heads, 64, 16, 0, garbage=False) for _ in range(3)]
        plain = torch.empty(odd.shape, device="cuda", dtype=odd.dtype).copy_(odd)
        caches[0].append(odd, odd, table, lengths)
        caches[1].append(plain, plain, table, lengths)
        if count == 1:
            caches[2].append(odd[0], odd[0], table, lengths, starts=tensor([0, new]))
        for other in caches[1:2 + (count == 1)]:
            assert torch.equal(caches[0].k_codes.view(torch.uint8), other.k_codes.view(torch.uint8))
            assert torch.equal(caches[0].v_codes.view(torch.uint8), other.v_codes.view(torch.uint8))
        want = caches[1].attend(plain, table, lengths + new)
        assert torch.equal(caches[0].attend(odd, table, lengths + new), want)
        if count == 1:
            assert torch.equal(caches[0].attend(odd[0], table, lengths + new, starts=tensor([0, new]))[None], want)
        if count == new == 1:
            place = torch.zeros((4, 9, 4 * 64 + 2), device="cuda", dtype=torch.bfloat16)[..., :256].unflatten(-1, (4, 64))[:1, :1, :heads]
            assert torch.equal(caches[0].attend(odd, table, lengths + 1, out=place), want)
            assert torch.equal(caches[0].attend(odd[0], table, lengths + 1, starts=tensor([0, 1]), out=place[0])[None], want)


def test_gradients_are_refused_not_dropped():
    """Whatever asks for a gradient or carries a tangent, the cache's own scales included; without autograd the same calls run."""
    from torch.autograd import forward_ad

    from deepcompressor_amd._lib import DcqError

    made = make_cache(2, 1, 64, 16, 0, garbage=False)
    scales = made.k_scales.clone().requires_grad_()
    cache = Fp8KVCache.from_buffers(made.k_codes, scales, made.v_codes, made.v_scales)
    kv, table, lengths = torch.randn((1, 3, 1, 64), device="cuda").half(), tensor([[0, 1]]), tensor([0])
    for call in (lambda: cache.append(kv, kv, table, lengths), lambda: cache.attend(kv, table, lengths + 3),
                 lambda: made.attend(kv.clone().requires_grad_(), table, lengths + 3), lambda: made.append(kv, kv.clone().requires_grad_(), table, lengths),
                 lambda: made.attend(kv, table, lengths + 3, out=torch.empty_like(kv).requires_grad_())):
        with pytest.raises(DcqError, match="no gradient"):
            call()
        with torch.no_grad():
            call()
    with forward_ad.dual_level():
        made.attend(kv, table, lengths + 3)
        with pytest.raises(DcqError, match="forward gradient"):
            made.attend(forward_ad.make_dual(kv, kv), table, lengths + 3)


@pytest.mark.parametrize("tokens", [200, 5000])
def test_single_tokens_in_place(tokens):
    """The output may be the query itself, whole and where the tokens are split over workgroups."""
    table = make_table([tokens] * 2, 64, -(-tokens // 64), 2 * (-(-tokens // 64)), 0)
    cache = make_cache(table.size, 2, 64, 64, 0)
    fill(cache, table, [tokens] * 2, 0)
    q = torch.randn((2, 1, 8, 64), generator=torch.Generator().manual_seed(0)).half().cuda()
    want = cache.attend(q, tensor(table), tensor([tokens, 3]))
    assert torch.equal(cache.attend(q, tensor(table), tensor([tokens, 3]), out=q), want) and torch.equal(q, want)
