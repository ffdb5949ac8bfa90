"""The block quantizer and the block-scaled product against their definitions in 64 bits, and against the fake quantizer."""

import numpy as np
import pytest
import torch

import fp8_oracle as fo
from _kv8 import HALF_STEP, values
from deepcompressor_amd.data import BlockScaledTensor, QDType
from deepcompressor_amd.nn.patch import Fp8BlockLinear, block_scaled_linear
from deepcompressor_amd.quantizer import Quantizer, QuantizerConfig

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def sample(rows, cols, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((rows, cols), generator=g) * torch.exp(2 * torch.randn((1, cols), generator=g))
    return x.to(dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 128), (3, 127), (9, 129), (33, 1000), (130, 512), (257, 384)])
@pytest.mark.parametrize("block_rows", [1, 128])
def test_quantize_matches_definition(rows, cols, dtype, block_rows):
    x = sample(rows, cols, dtype, rows * 1000 + cols)
    got = BlockScaledTensor.quantize(x.cuda(), block_rows)
    codes, scales = fo.quantize_blocks(x.float().numpy(), block_rows)
    np.testing.assert_array_equal(got.scales.cpu().numpy(), scales)
    np.testing.assert_array_equal(values(got.codes), codes)


@pytest.mark.parametrize("block_rows", [1, 128])
def test_quantize_ties_and_signs(block_rows):
    """Every value of the grid and every midpoint, scale 1: ties go to the upper neighbour."""
    mid = (fo.GRID[1:] + fo.GRID[:-1]) / 2
    around = np.concatenate([fo.GRID, mid, np.nextafter(mid.astype(np.float32), np.float32(np.inf)).astype(np.float64),
                             np.nextafter(mid.astype(np.float32), np.float32(-np.inf)).astype(np.float64), [-0.0, 1e-30, -1e-30]])
    x = np.zeros((-(-len(around) // 127), 128), dtype=np.float32)
    x[:, 127] = 448
    flat = np.zeros(x.shape[0] * 127, dtype=np.float32)
    flat[:len(around)] = around
    x[:, :127] = flat.reshape(-1, 127)
    got = BlockScaledTensor.quantize(torch.from_numpy(x).cuda(), block_rows)
    assert (got.scales == 1).all()
    np.testing.assert_array_equal(values(got.codes), fo.nearest_e4m3(x))


@pytest.mark.parametrize("block_rows", [1, 128])
def test_quantize_extremes(block_rows):
    """Zero blocks, blocks near both ends of float32, subnormal scales, NaN and infinities."""
    x = torch.zeros((4, 896))
    x[:, 128:256] = torch.linspace(-1, 1, 128) * 3e38
    x[:, 256:384] = torch.linspace(-1, 1, 128) * 1e-36
    x[:, 384:512] = torch.linspace(-1, 1, 128) * 3e-43
    x[:, 512:640] = torch.linspace(-1, 1, 128)
    x[1, 515] = float("nan")
    x[:, 640:768] = torch.linspace(-1, 1, 128)
    x[2, 700] = float("inf")
    x[2, 701] = float("-inf")
    x[:, 768:] = torch.linspace(-1, 1, 128) * 1e-44
    got = BlockScaledTensor.quantize(x.cuda(), block_rows)
    codes, scales = fo.quantize_blocks(x.numpy(), block_rows)
    np.testing.assert_array_equal(got.scales.cpu().numpy(), scales)
    np.testing.assert_array_equal(values(got.codes), codes)


@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("dtype", DTYPES)
def test_quantize_equals_the_fake_quantizer(block_rows, dtype):
    x = sample(256, 640, dtype, 5).cuda()
    q = Quantizer(QuantizerConfig(dtype=QDType.sfp8_e4m3_nan, group_shapes=((block_rows, 128),), scale_dtypes=(torch.float32,)))
    fake = q.quantize(x, return_with_dequant=False, return_with_quant=True)
    got = BlockScaledTensor.quantize(x, block_rows)
    made = BlockScaledTensor.from_quantized(fake, block_rows)
    assert torch.equal(got.scales, made.scales)
    assert torch.equal(got.codes.float(), made.codes.float())


def test_quantize_strides_and_leading_axes():
    x = sample(64, 1000, torch.bfloat16, 1).cuda()
    whole = BlockScaledTensor.quantize(x[:, :520].contiguous())
    for part in (x[:, :520], x[:, 1:521], x.t()[:520].t()):
        want = BlockScaledTensor.quantize(part.contiguous())
        got = BlockScaledTensor.quantize(part)
        assert torch.equal(got.codes.float(), want.codes.float()) and torch.equal(got.scales, want.scales)
    assert torch.equal(BlockScaledTensor.quantize(x[:, :520]).scales, whole.scales)
    cube = BlockScaledTensor.quantize(x.view(4, 16, 1000))
    assert cube.shape == (4, 16, 1000) and cube.codes.shape == (64, 1000)
    assert BlockScaledTensor.quantize(x[:0]).codes.shape == (0, 1000)


def operands(M, N, K, seed):
    """Codes with memory behind each row that holds NaN, as a slice of a wider matrix has."""
    g = torch.Generator().manual_seed(seed)
    pitch = -(-K // 16) * 16

    def codes(rows):
        c = torch.full((rows, pitch), 0x7F, dtype=torch.uint8)
        c[:, :K] = (torch.randn((rows, K), generator=g) * 100).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
        return c.cuda().view(torch.float8_e4m3fn)[:, :K]

    kb = -(-K // 128)
    xs = torch.rand((kb, M), generator=g).add(0.01).cuda().t()
    ws = torch.rand((-(-N // 128), kb), generator=g).add(0.01).cuda()
    return codes(M), xs, codes(N), ws


def check_product(M, N, K, dtype, bias, seed):
    x, xs, w, ws = operands(M, N, K, seed)
    b = torch.randn(N, generator=torch.Generator().manual_seed(seed)).mul(100).to(dtype) if bias else None
    y = block_scaled_linear(BlockScaledTensor.from_codes(x, xs, 1), BlockScaledTensor.from_codes(w, ws, 128), None if b is None else b.cuda(),
                            dtype=dtype)
    assert y.shape == (M, N) and y.dtype == dtype
    want, size = fo.product(values(x), xs.cpu().numpy(), values(w), ws.cpu().numpy(), None if b is None else b.double().numpy())
    # a block's 128 products are exact, each addition is off by at most a step (2^-23) of the magnitudes so far; then two
    # scalings and an addition per block, the bias, and one rounding
    blocks = -(-K // 128)
    tol = (128 + 3 * blocks + 2) * 2.0**-23 * size + HALF_STEP[dtype] * np.abs(want)
    if dtype != torch.float32:
        # 16-bit outputs are summed by the 8-bit instruction, which takes products eight at a time and cuts them off below
        # 2^-13 of the power of two of the eight's largest (measured: 2^-13 beside 1 counts, 2^-14 does not, and only within
        # k = 8 i .. 8 i + 7).  Each of the other seven loses less than 2^-13 of the largest, hence the eight together less
        # than 7 * 2^-13 of their magnitudes' sum, and so all of them of `size`.
        tol = tol + 7 * 2.0**-13 * size
    got = y.double().cpu().numpy()
    if dtype == torch.float16:
        over = np.abs(want) > 65504
        got, want, tol = got[~over], want[~over], tol[~over]
    bad = ~(np.abs(got - want) <= tol)
    assert not bad.any(), f"{bad.sum()} of {bad.size} outside, worst {np.max(np.abs(got - want) / tol)} of the tolerance"


SIZES = [(1, 1, 1), (1, 128, 128), (1, 129, 100), (2, 4096, 512), (5, 100, 1000), (16, 64, 127), (17, 200, 129), (33, 1000, 384),
         (48, 300, 2000), (64, 128, 4096), (65, 70, 144), (100, 257, 1000), (128, 128, 128), (129, 513, 272), (300, 300, 300),
         (520, 640, 640)]


@pytest.mark.parametrize("M,N,K", SIZES)
@pytest.mark.parametrize("dtype,bias", [(torch.bfloat16, False), (torch.float16, True), (torch.float32, True)])
def test_product(M, N, K, dtype, bias):
    check_product(M, N, K, dtype, bias, M * 7 + N * 3 + K)


def test_product_propagates_nan_and_inf():
    x, xs, w, ws = operands(20, 200, 300, 1)
    x, xs = x.clone(), xs.clone()
    x.view(torch.uint8)[3, 299] = 0x7F
    xs[5, 1] = float("inf")
    y = block_scaled_linear(BlockScaledTensor.from_codes(x, xs, 1), BlockScaledTensor.from_codes(w, ws, 128), dtype=torch.float32)
    assert torch.isnan(y[3]).all() and not torch.isfinite(y[5]).any()
    rest = [i for i in range(20) if i not in (3, 5)]
    assert torch.isfinite(y[rest]).all()


def test_from_codes_copies_only_when_it_must():
    x, xs, _, _ = operands(8, 8, 256, 3)
    assert BlockScaledTensor.from_codes(x, xs).codes.data_ptr() == x.data_ptr()
    odd = torch.zeros((8, 250), dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
    assert BlockScaledTensor.from_codes(odd, xs).codes.stride(0) == 256
    last = torch.zeros(8 * 256 - 6, dtype=torch.uint8, device="cuda").as_strided((8, 250), (256, 1)).view(torch.float8_e4m3fn)
    assert BlockScaledTensor.from_codes(last, xs).codes.data_ptr() != last.data_ptr()


@pytest.mark.parametrize("dtype", DTYPES)
def test_module_stands_in_for_a_linear(dtype):
    g = torch.Generator().manual_seed(0)
    linear = torch.nn.Linear(300, 200).to(dtype)
    linear.weight.data.copy_(torch.randn((200, 300), generator=g) * 0.05)
    module = Fp8BlockLinear.from_linear(linear.cuda())
    x = torch.randn((2, 7, 300), generator=g).to(dtype).cuda()
    with torch.no_grad():
        y = module(x)
        again = Fp8BlockLinear(BlockScaledTensor.quantize(torch.zeros((200, 300), device="cuda"), 128), linear.bias)
        again.load_state_dict(module.state_dict())
        moved = module.to(torch.float16)  # codes and scales stay what they are
        assert moved.scales.dtype == torch.float32 and moved.codes.dtype == torch.uint8
        assert torch.equal(again(x), y)
        want = x.float() @ linear.weight.float().t() + linear.bias.float()
    assert y.shape == (2, 7, 200) and y.dtype == dtype
    # each operand's rounding is at most half a step of e4m3, 2^-4 of the value, or 2^-10 of the block's 448: relative to
    # the magnitudes' product (1 + 2^-4)^2 - 1, plus the smallest values' share
    size = x.float().abs() @ linear.weight.float().abs().t()
    top = x.float().abs().amax(-1, keepdim=True) * linear.weight.float().abs().amax() * 300
    tol = ((1 + 2.0**-4)**2 - 1) * size + 3 * 2.0**-10 / 448 * top + HALF_STEP[dtype] * 2 * (want.abs() + 1)
    assert ((y.float() - want).abs() <= tol).all()


def test_streams_and_graphs():
    """Another stream than the current one's, and a captured pair of calls replayed with new inputs."""
    x = torch.randn((40, 512), device="cuda", dtype=torch.bfloat16)
    linear = Fp8BlockLinear.from_linear(torch.nn.Linear(512, 384, device="cuda", dtype=torch.bfloat16))
    with torch.no_grad():
        want = linear(x)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = linear(x)
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(got, want)
        graph, held = torch.cuda.CUDAGraph(), x.clone()
        with torch.cuda.graph(graph):
            out = linear(held)
        for seed in range(3):
            held.copy_(torch.randn(held.shape, generator=torch.Generator().manual_seed(seed)))
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, linear(held))


# sizes that reach each kernel: whole tiles and ragged ones of 256, 128 and 64, K with and without a part of a block
LARGE = [(2049, 6200, 130), (1800, 6144, 512), (300, 8200, 257), (200, 12288, 384), (65, 17000, 1000), (130, 4000, 1040), (64, 12000, 640),
         (16, 9000, 300), (40, 1000, 1536)]


@pytest.mark.parametrize("M,N,K", LARGE)
@pytest.mark.parametrize("dtype,bias", [(torch.bfloat16, True), (torch.float16, False), (torch.float32, True)])
def test_product_large(M, N, K, dtype, bias):
    check_product(M, N, K, dtype, bias, M + N + K)


def test_product_strided_scales_and_outputs_at_odd_places():
    """Scales of any strides, codes that are a slice of a wider matrix, N that keeps outputs from being stored in whole pieces."""
    for M, N in ((40, 333), (700, 9003)):
        x, xs, w, ws = operands(M, N, 512, 5)
        want = block_scaled_linear(BlockScaledTensor.from_codes(x, xs, 1), BlockScaledTensor.from_codes(w, ws, 128))
        wide = torch.full((M, 1024), 0x7F, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
        wide[:, 256:768] = x
        rows = torch.zeros((M, 9), device="cuda")
        rows[:, 3:7] = xs
        cols = torch.zeros((ws.shape[1], 2 * ws.shape[0]), device="cuda").t()
        cols[::2] = ws
        a = BlockScaledTensor.from_codes(wide[:, 256:768], rows[:, 3:7], 1)
        assert a.codes.data_ptr() == wide[:, 256:].data_ptr()
        assert torch.equal(block_scaled_linear(a, BlockScaledTensor.from_codes(w, cols[::2], 128)), want)


@pytest.mark.parametrize("M,N,K", [(2049, 6200, 130), (333, 1001, 1000), (200, 12288, 384), (520, 4096, 512)])
def test_large_products_in_a_graph_and_on_two_streams(M, N, K):
    x, xs, w, ws = operands(M, N, K, 3)
    a, b = BlockScaledTensor.from_codes(x, xs, 1), BlockScaledTensor.from_codes(w, ws, 128)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = block_scaled_linear(a, b)
    for seed in range(3):
        xs.copy_(torch.rand(xs.shape, generator=torch.Generator().manual_seed(seed)))
        graph.replay()
        want = block_scaled_linear(a, b)
        torch.cuda.synchronize()
        assert torch.equal(out, want)
    sides, got = [torch.cuda.Stream(), torch.cuda.Stream()], []
    for t in range(4):
        with torch.cuda.stream(sides[t % 2]):
            got.append(block_scaled_linear(a, b))
    torch.cuda.synchronize()
    assert all(torch.equal(y, want) for y in got)


def test_offsets_beyond_32_bits():
    """Rows behind 2^32 bytes of inputs, codes or outputs: the same answers as at the beginning."""
    x = torch.empty((2**17 + 40, 2**15), device="cuda", dtype=torch.bfloat16)
    x[:40] = torch.randn((40, 2**15), device="cuda", generator=torch.Generator("cuda").manual_seed(0)).to(torch.bfloat16)
    x[40:-40] = 1.0
    x[-40:] = x[:40]
    a = BlockScaledTensor.quantize(x)
    assert torch.equal(a.codes[-40:].view(torch.uint8), a.codes[:40].view(torch.uint8)) and torch.equal(a.scales[-40:], a.scales[:40])
    t = BlockScaledTensor.quantize(x[:, :2**14], 128)
    assert (t.scales[1:1024] == t.scales[2]).all() and (t.codes[128:2**17].view(torch.uint8) == 0x7E).all()
    del x, t
    w = BlockScaledTensor.quantize(torch.randn((2**15, 128), device="cuda", generator=torch.Generator("cuda").manual_seed(1)), 128)
    part = BlockScaledTensor.from_codes(a.codes[:, :128], a.scales[:, :1])  # rows 2^15 bytes apart
    assert part.codes.data_ptr() == a.codes.data_ptr()
    y = block_scaled_linear(part, w, dtype=torch.float16)
    assert torch.equal(y[-40:], y[:40]) and torch.isfinite(y[-40:]).all()
    few = BlockScaledTensor.from_codes(a.codes[:20], a.scales[:20])
    rows = BlockScaledTensor.from_codes(a.codes, torch.ones((2**10 + 1, 2**8), device="cuda"), 128)  # weights behind 2^32 bytes
    y = block_scaled_linear(few, rows)
    assert torch.equal(y[:, -40:], y[:, :40]) and torch.isfinite(y[:, -40:]).all()


@pytest.mark.parametrize("M,N,K", [(256, 1024, 4096), (512, 768, 768), (640, 2112, 1200)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_equal_rows_have_equal_results(M, N, K, dtype):
    """What a token gives does not depend on its place in the batch (sizes with 64 x 64 tiles, split along K)."""
    x, xs, w, ws = operands(64, N, K, 9)
    x, xs = x.view(torch.uint8).repeat(M // 64, 1).view(x.dtype), xs.repeat(M // 64, 1)
    y = block_scaled_linear(BlockScaledTensor.from_codes(x, xs, 1), BlockScaledTensor.from_codes(w, ws, 128), dtype=dtype)
    for at in range(64, M, 64):
        assert torch.equal(y[at:at + 64], y[:64]), at


@pytest.mark.parametrize("dtype", DTYPES)
def test_no_columns_and_leading_axes(dtype):
    """K = 0 leaves the bias, whatever axes there are before it; no rows leave nothing."""
    bias = torch.randn(200, device="cuda").to(dtype)
    w = BlockScaledTensor.quantize(torch.zeros((200, 0), device="cuda"), 128)
    for shape in ((3, 0), (2, 3, 0), (0,), (2, 0, 0)):
        y = block_scaled_linear(torch.zeros(shape, device="cuda", dtype=dtype), w, bias)
        assert y.shape == (*shape[:-1], 200) and torch.equal(y, bias.expand(y.shape))
        assert (block_scaled_linear(torch.zeros(shape, device="cuda", dtype=dtype), w) == 0).all()
    w = BlockScaledTensor.quantize(torch.zeros((200, 130), device="cuda"), 128)
    assert block_scaled_linear(torch.zeros((2, 0, 130), device="cuda", dtype=dtype), w).shape == (2, 0, 200)


# sizes that reach each kernel: 256-tiles, 128-tiles, 64-tiles split along K, rows
KERNELS = [(2049, 6200, 512), (300, 8200, 384), (130, 4000, 1152), (16, 4096, 512)]


@pytest.mark.parametrize("M,N,K", KERNELS)
@pytest.mark.parametrize("dtype", DTYPES)
def test_product_of_small_whole_numbers_is_exact(M, N, K, dtype):
    """Codes from -3 to 3 and scales that are powers of two: no product is cut off, every sum is exact in float32, so the outputs
    are the exact sums rounded once."""
    g = torch.Generator().manual_seed(M)
    whole = lambda rows: torch.randint(-3, 4, (rows, K), generator=g).double()  # noqa: E731
    power = lambda rows: torch.exp2(torch.randint(-1, 2, (rows, K // 128), generator=g).float())  # noqa: E731
    x, w, xs, ws = whole(M), whole(N), power(M), power(-(-N // 128))
    y = block_scaled_linear(BlockScaledTensor.from_codes(x.to(torch.float8_e4m3fn).cuda(), xs.cuda(), 1),
                            BlockScaledTensor.from_codes(w.to(torch.float8_e4m3fn).cuda(), ws.cuda(), 128), dtype=dtype)
    want = (x * xs.double().repeat_interleave(128, 1)) @ (w * ws.double().repeat_interleave(128, 0)[:N].repeat_interleave(128, 1)).t()
    assert torch.equal(y.cpu(), want.to(dtype))


@pytest.mark.parametrize("M,N,K", KERNELS)
@pytest.mark.parametrize("dtype", DTYPES)
def test_what_the_sums_lose(M, N, K, dtype):
    """The sums before their rounding: the bias takes the exact ones away again.  Normally distributed codes; 16-bit outputs may lose
    what is below 2^-13 of the power of two of each eight products' largest (cut off here as whole steps, about 2e-5 of the sums in
    the 2-norm), and all what float32 sums of 128 products and of the blocks do."""
    g = torch.Generator().manual_seed(N)
    codes = lambda rows: (torch.randn((rows, K), generator=g) * 100).clamp(-448, 448).to(torch.float8_e4m3fn)  # noqa: E731
    x, w = codes(1), codes(N)
    terms = (w.double() * x.double()).view(N, K // 8, 8)
    step = torch.exp2(torch.floor(torch.log2(terms.abs().amax(-1, keepdim=True).clamp_min(2.0**-18))) - 13)
    lost = (terms - torch.trunc(terms / step) * step).sum((1, 2)) if dtype != torch.float32 else torch.zeros(N, dtype=torch.float64)
    exact = terms.sum((1, 2))
    ones = lambda rows: torch.ones((rows, K // 128), device="cuda")  # noqa: E731
    y = block_scaled_linear(BlockScaledTensor.from_codes(x.cuda().view(torch.uint8).repeat(M, 1).view(x.dtype), ones(M), 1),
                            BlockScaledTensor.from_codes(w.cuda(), ones(-(-N // 128)), 128), -exact.float().cuda(), dtype=dtype)
    assert torch.equal(y, y[:1].expand(M, N))
    norm = exact.pow(2).mean().sqrt()
    # (the bias is the exact sum to 2^-24, float32 sums are off by at most a step of 2^-23 of the magnitudes for each addition)
    sums = (K + 3 * (K // 128) + 2) * 2.0**-23 * terms.abs().sum((1, 2)).pow(2).mean().sqrt() if dtype == torch.float32 else 2.0**-20 * norm
    allowed = 1.1 * lost.pow(2).mean().sqrt() + sums
    assert y[0].double().cpu().pow(2).mean().sqrt() <= allowed
    if dtype != torch.float32:  # (of the data alone: 1.1 times 1.95e-5 on average, 2^-20, and a token's own spread of some tenths)
        assert allowed <= 3e-5 * norm
