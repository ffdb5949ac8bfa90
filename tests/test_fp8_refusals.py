"""What the operators on 8-bit values refuse, without a GPU: Python's checks on CPU tensors, the C ABI's on bad arguments
(they return before anything is launched)."""

import ctypes as C

import pytest
import torch

from deepcompressor_amd._lib import DcqError, lib
from deepcompressor_amd.data import BlockScaledTensor
from deepcompressor_amd.nn.patch import Fp8BlockLinear, Fp8KVCache, block_scaled_linear

E4M3 = torch.float8_e4m3fn


def codes(*shape):
    return torch.zeros(shape, dtype=torch.uint8).view(E4M3)


def test_no_cpu_path():
    with pytest.raises(DcqError, match="GPUs only"):
        BlockScaledTensor.quantize(torch.zeros(2, 128))
    x = BlockScaledTensor.from_codes(codes(2, 128), torch.ones(2, 1))
    w = BlockScaledTensor.from_codes(codes(4, 128), torch.ones(1, 1), 128)
    with pytest.raises(DcqError, match="GPUs only"):
        block_scaled_linear(x, w)
    cache = Fp8KVCache(2, 1, 64, 16, device="cpu")
    kv, table, lengths = torch.zeros(1, 1, 1, 64), torch.zeros((1, 1), dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    with pytest.raises(DcqError, match="GPUs only"):
        cache.append(kv, kv, table, lengths)
    with pytest.raises(DcqError, match="GPUs only"):
        cache.attend(kv.half(), table, lengths)


def test_quantize_refusals():
    for x, rows, error in ((torch.zeros(()), 1, ValueError), (torch.zeros(2, 128), 64, ValueError), (torch.zeros(2, 128, dtype=torch.float64), 1, TypeError),
                           (torch.zeros(2, 128, dtype=torch.int8), 1, TypeError)):
        with pytest.raises(error):
            BlockScaledTensor.quantize(x, rows)


def test_from_codes_refusals():
    good = torch.ones(2, 2)
    for c, s, rows in ((codes(2, 200).view(torch.uint8), good, 1), (codes(200), good, 1), (codes(2, 200), good.double(), 1),
                       (codes(2, 200), torch.ones(2, 1), 1), (codes(2, 200), torch.ones(1, 2), 1), (codes(2, 200), good, 128), (codes(2, 200), good, 2)):
        with pytest.raises(ValueError):
            BlockScaledTensor.from_codes(c, s, rows)


def test_product_refusals():
    x = BlockScaledTensor.from_codes(codes(2, 128), torch.ones(2, 1))
    w = BlockScaledTensor.from_codes(codes(4, 128), torch.ones(1, 1), 128)
    with pytest.raises(ValueError, match="inner sizes"):
        block_scaled_linear(x, BlockScaledTensor.from_codes(codes(4, 64), torch.ones(1, 1), 128))
    with pytest.raises(ValueError, match="128 x 128"):
        block_scaled_linear(x, x)
    with pytest.raises(ValueError, match="128 x 128"):
        block_scaled_linear(w, w)
    with pytest.raises(ValueError, match="bias"):
        block_scaled_linear(x, w, torch.zeros(3))
    with pytest.raises(TypeError):
        block_scaled_linear(x, w, dtype=torch.float64)
    with pytest.raises(ValueError, match="128 x 128"):
        Fp8BlockLinear(x)


def test_cache_refusals():
    for pages, heads, dim, page in ((0, 1, 64, 16), (1, 0, 64, 16), (1, 1, 96, 16), (1, 1, 64, 24), (1, 1, 64, 256)):
        with pytest.raises(ValueError):
            Fp8KVCache(pages, heads, dim, page, device="cpu")
    k, v, s = codes(2, 1, 16, 64), codes(2, 1, 64, 16), torch.ones(2, 1)
    for bad in ((k, s, k, s), (k, s, v, s.double()), (k, torch.ones(1, 2), v, s), (k.view(torch.uint8), s, v, s), (k, s, codes(2, 1, 16, 64).transpose(2, 3), s)):
        with pytest.raises(ValueError):
            Fp8KVCache.from_buffers(*bad)


def test_call_refusals():
    cache = Fp8KVCache(2, 2, 64, 16, device="cpu")
    kv = torch.zeros(1, 1, 2, 64)
    with pytest.raises(ValueError, match="differ"):
        cache.append(kv, kv.half(), None, None)
    with pytest.raises(ValueError, match="heads and channels"):
        cache.append(kv[:, :, :1], kv[:, :, :1], None, None)
    with pytest.raises(TypeError):
        cache.append(kv.double(), kv.double(), None, None)
    with pytest.raises(ValueError, match="float16 or bfloat16"):
        cache.attend(kv, None, None)
    with pytest.raises(ValueError, match="heads and channels"):
        cache.attend(torch.zeros((1, 1, 3, 64), dtype=torch.float16), None, None)


def test_product_refuses_tensors_put_together_by_hand():
    """A tensor made of its parts has not been looked over: the product does, before anything is read."""
    good = dict(codes=codes(2, 128), scales=torch.ones(2, 1))
    w = BlockScaledTensor.from_codes(codes(4, 128), torch.ones(1, 1), 128)
    for part in (dict(scales=torch.ones(1, 1)), dict(scales=torch.ones(2, 2)), dict(scales=torch.ones(2, 1).double()), dict(codes=codes(2, 128).view(torch.uint8)),
                 dict(codes=codes(128, 2).t())):
        p = {**good, **part}
        with pytest.raises(ValueError):
            block_scaled_linear(BlockScaledTensor(p["codes"], p["scales"], 1, p["codes"].shape), w)
    x = BlockScaledTensor.from_codes(**good)
    for scales in (torch.ones(2, 1), torch.ones(1, 1).half()):
        with pytest.raises(ValueError):
            block_scaled_linear(x, BlockScaledTensor(w.codes, scales, 128, w.shape))


FAKE = C.c_void_p(1 << 20)  # an aligned address that nothing may touch


def strides(*s):
    return (C.c_int64 * 3)(*s)


@pytest.mark.parametrize("change", [dict(storage=3), dict(rows=-1), dict(x=None), dict(block=2), dict(ldx=100), dict(ldc=120),
                                    dict(ldc=136), dict(codes=C.c_void_p((1 << 20) + 8)), dict(x=C.c_void_p((1 << 20) + 1)), dict(cols=1 << 40)])
def test_c_quantize_refusals(change):
    a = dict(x=FAKE, storage=1, rows=4, cols=128, ldx=128, block=1, codes=FAKE, ldc=128, scales=FAKE)
    a.update(change)
    if change.get("cols"):
        a["ldx"] = a["ldc"] = a["cols"]
    rc = lib().dcq_fp8_quantize_blocks(a["x"], a["storage"], a["rows"], a["cols"], a["ldx"], a["block"], a["codes"], a["ldc"], a["scales"], 1, 4, None)
    assert rc < 0 and lib().dcq_last_error()


@pytest.mark.parametrize("change", [dict(K=0), dict(M=-1), dict(y=None), dict(ys=3), dict(ldx=100), dict(ldx=136), dict(ldy=3), dict(w=C.c_void_p((1 << 20) + 4)),
                                    dict(N=1 << 40, ldy=1 << 40), dict(bias=FAKE, bs=7)])
def test_c_product_refusals(change):
    a = dict(x=FAKE, ldx=128, w=FAKE, bias=None, bs=0, y=FAKE, ys=0, ldy=8, M=2, N=8, K=128)
    a.update(change)
    rc = lib().dcq_fp8_block_gemm(a["x"], a["ldx"], FAKE, 1, 2, a["w"], 128, FAKE, 1, 1, a["bias"], a["bs"], a["y"], a["ys"], a["ldy"], a["M"], a["N"],
                                  a["K"], None)
    assert rc < 0 and lib().dcq_last_error()


@pytest.mark.parametrize("change", [dict(pool=0), dict(heads=0), dict(page=24), dict(dim=96), dict(cols=0), dict(cols=1 << 30), dict(total=5), dict(key=None),
                                    dict(ks=(64, 63, 64)), dict(key=C.c_void_p((1 << 20) + 8)), dict(storage=3)])
def test_c_append_refusals(change):
    a = dict(key=FAKE, ks=(128, 64, 64), storage=2, sequences=2, total=4, pool=4, heads=1, page=16, dim=64, cols=2)
    a.update(change)
    rc = lib().dcq_kv8_append(a["key"], FAKE, a["storage"], strides(*a["ks"]), strides(128, 64, 64), FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, None, a["sequences"],
                              a["total"], a["pool"], a["heads"], a["page"], a["dim"], a["cols"], None)
    assert rc < 0 and lib().dcq_last_error()


@pytest.mark.parametrize("change", [dict(storage=0), dict(group=0), dict(group=1 << 30), dict(page=8), dict(dim=256), dict(os=(128, 64, 62)), dict(total=5), dict(ws=16),
                                    dict(q=C.c_void_p((1 << 20) + 2))])
def test_c_attention_refusals(change):
    a = dict(q=FAKE, storage=2, os=(128, 64, 64), sequences=2, total=2, group=1, page=16, dim=64, ws=1 << 30)
    a.update(change)
    rc = lib().dcq_kv8_attention(a["q"], a["storage"], strides(128, 64, 64), FAKE, strides(*a["os"]), FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, None, a["sequences"],
                                 a["total"], 4, 1, a["group"], a["page"], a["dim"], 1 << 12, 1.0, 1, 0, FAKE, a["ws"], None)
    assert rc < 0 and lib().dcq_last_error()
    assert lib().dcq_kv8_attention_workspace_bytes(2, 2, 1, 1, 64, 1 << 16, 0) > 16


def test_strides_of_axes_of_size_one_do_not_count():
    """The host layer's view of tokens: strides that the kernels can address, without a copy where only an axis of size 1 is in the way."""
    from deepcompressor_amd.engine_fp8 import _tokens

    wide = torch.arange(4.0 * 9 * 264).view(4, 9, 264)
    for t, copied in ((wide[..., :256].unflatten(-1, (4, 64))[1:2], False), (torch.zeros(4, 9, 258)[..., :256].unflatten(-1, (4, 64))[:1, :1], False),
                      (torch.zeros(4, 9, 257)[..., 1:].unflatten(-1, (4, 64))[:1, :1], True), (torch.zeros(4, 9, 257)[..., 1:].unflatten(-1, (4, 64))[:, :1], True),
                      (torch.zeros(2, 385)[:, :384].unflatten(1, (3, 2, 64))[1:2], True)):
        got, strides = _tokens(t, False, "key", 8)
        assert torch.equal(got, t) and (got.data_ptr() != t.data_ptr()) == copied
        assert got.data_ptr() % 16 == 0 and all(s % 8 == 0 for s in strides)
        got, strides = _tokens(t[0], True, "key", 8)
        assert torch.equal(got, t[0]) and got.data_ptr() % 16 == 0 and all(s % 8 == 0 for s in strides)


def test_product_refuses_memory_that_ends_within_16_bytes():
    """Rows at multiples of 16 bytes whose last one ends with its buffer: from_codes copies them, by hand they are refused."""
    def ends(rows, cols):
        return torch.zeros((rows - 1) * 128 + cols, dtype=torch.uint8).as_strided((rows, cols), (128, 1)).view(E4M3)

    x = BlockScaledTensor.from_codes(ends(2, 100), torch.ones(2, 1))
    w = BlockScaledTensor.from_codes(ends(4, 100), torch.ones(1, 1), 128)
    for t, rows in ((x, 2), (w, 4)):
        bare = BlockScaledTensor(ends(rows, 100), t.scales, t.block_rows, t.shape)
        with pytest.raises(ValueError, match="from_codes"):
            block_scaled_linear(bare if t is x else x, bare if t is w else w)
    with pytest.raises(DcqError, match="GPUs only"):  # (looked over, and all right)
        block_scaled_linear(x, w)
    room = BlockScaledTensor(torch.zeros(128 + 112, dtype=torch.uint8).as_strided((2, 100), (128, 1)).view(E4M3), x.scales, 1, x.shape)
    with pytest.raises(DcqError, match="GPUs only"):
        block_scaled_linear(room, w)


def test_forward_gradients_are_refused():
    """A tangent would be dropped without a word: every tensor that may carry one is looked at."""
    from torch.autograd import forward_ad

    x = BlockScaledTensor.from_codes(codes(2, 128), torch.ones(2, 1))
    w = BlockScaledTensor.from_codes(codes(4, 128), torch.ones(1, 1), 128)
    cache, kv = Fp8KVCache(2, 1, 64, 16, device="cpu"), torch.zeros(1, 1, 1, 64)
    table, lengths = torch.zeros((1, 1), dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    with forward_ad.dual_level():
        dual = lambda t: forward_ad.make_dual(t, torch.ones_like(t))  # noqa: E731
        for call in (lambda: BlockScaledTensor.quantize(dual(torch.zeros(2, 128))), lambda: block_scaled_linear(x, w, dual(torch.zeros(4))),
                     lambda: block_scaled_linear(BlockScaledTensor(x.codes, dual(x.scales), 1, x.shape), w),
                     lambda: block_scaled_linear(dual(torch.zeros(2, 128)), w), lambda: cache.append(dual(kv), kv, table, lengths),
                     lambda: cache.append(kv, dual(kv), table, lengths), lambda: cache.attend(dual(kv.half()), table, lengths),
                     lambda: cache.attend(kv.half(), table, lengths, out=dual(kv.half())),
                     lambda: Fp8KVCache.from_buffers(cache.k_codes, dual(cache.k_scales), cache.v_codes, cache.v_scales).attend(kv.half(), table, lengths)):
            with pytest.raises(DcqError, match="forward gradient"):
                call()
        with pytest.raises(DcqError, match="GPUs only"):  # (no tangent: no objection)
            cache.append(kv, kv, table, lengths)


def test_module_conversions_leave_codes_and_scales_alone():
    """.to(), .half() and .double() convert the bias only; .type(), which asks for every buffer's type, is refused."""
    def module():
        held = torch.arange(4 * 256, dtype=torch.uint8).view(4, 256).view(E4M3)
        return Fp8BlockLinear(BlockScaledTensor.from_codes(held, torch.rand(1, 2), 128), torch.ones(4))

    made = module()
    codes_before, scales_before = made.codes.clone(), made.scales.clone()
    for convert in (lambda m: m.half(), lambda m: m.double(), lambda m: m.to(torch.bfloat16), lambda m: m.to(device="cpu", dtype=torch.float16)):
        m = convert(made)
        assert torch.equal(m.codes, codes_before) and torch.equal(m.scales, scales_before) and m.scales.dtype == torch.float32
        assert m.bias.dtype != torch.float32
    for dtype in (torch.bfloat16, torch.float64, torch.int32):
        m = module()
        with pytest.raises((TypeError, RuntimeError)):
            m.type(dtype)
        assert m.codes.dtype == torch.uint8 and m.scales.dtype == torch.float32 and m.scales.shape == (1, 2)
    assert made.to_empty(device="meta").scales.dtype == torch.float32


def test_from_quantized_refuses_other_groups_and_zero_points():
    """As many scales as blocks are not enough: they have to belong to the blocks."""
    from deepcompressor_amd.data import QuantScale, QuantTensor

    def quantized(rows, cols, scale_shape, zero=None):
        return QuantTensor(quantized=torch.zeros(rows, cols), scale=QuantScale().append(torch.rand(scale_shape)), zero=zero)

    for good in (quantized(256, 300, (2, 1, 3, 1)), quantized(256, 300, (2, 3)), quantized(256, 300, (2, 1, 3, 1), torch.tensor(0.0))):
        assert BlockScaledTensor.from_quantized(good).scales.shape == (2, 3)
    assert BlockScaledTensor.from_quantized(quantized(3, 300, (3, 1, 3, 1)), 1).scales.shape == (3, 3)
    assert BlockScaledTensor.from_quantized(quantized(60, 100, ())).scales.shape == (1, 1)
    for bad in (quantized(128, 16384, (128, 1, 1, 1)), quantized(256, 128, (1, 1, 2, 1)), quantized(256, 300, (2, 1, 1, 1)), quantized(256, 300, (3, 2))):
        with pytest.raises(ValueError, match="blocks"):
            BlockScaledTensor.from_quantized(bad)
    for zero in (torch.tensor([[[[0.0]], [[1.0]]]]), 2.0):
        with pytest.raises(ValueError, match="zero points"):
            BlockScaledTensor.from_quantized(quantized(128, 256, (1, 1, 2, 1), zero))


def test_outputs_whose_elements_share_memory_are_refused():
    cache, q = Fp8KVCache(2, 1, 64, 16, device="cpu"), torch.zeros((2, 3, 2, 64), dtype=torch.float16)
    table, lengths = torch.zeros((2, 1), dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    room = torch.zeros(4096, dtype=torch.float16)
    for strides in ((64, 64, 128, 1), (384, 64, 64, 1), (128, 128, 64, 1), (256, 128, 64, 1), (384, 128, 60, 1), (0, 128, 64, 1)):
        with pytest.raises(ValueError, match="share memory"):
            cache.attend(q, table, lengths, out=room.as_strided(q.shape, strides))
    for strides in ((384, 128, 64, 1), (64, 256, 128, 1), (400, 132, 64, 1), (1000, 64, 192, 1)):
        with pytest.raises(DcqError, match="GPUs only"):
            cache.attend(q, table, lengths, out=room.as_strided(q.shape, strides))
    for out in (room.as_strided(q.shape, (384, 128, 64, 2)), room.as_strided(q.shape, (386, 128, 64, 1)), q[:1], q.bfloat16()):
        with pytest.raises(ValueError, match="out"):
            cache.attend(q, table, lengths, out=out)


UNSUPPORTED = -2


def test_c_launches_beyond_a_grid_are_refused_before_the_launch():
    """A launch holds less than 2^32 threads, and sizes whose products leave 64 bits are no small ones."""
    L = lib()
    rows = 2**31 - 1
    assert L.dcq_fp8_quantize_blocks(FAKE, 2, rows, 128, 128, 1, FAKE, 128, FAKE, 1, rows, None) == UNSUPPORTED
    assert L.dcq_fp8_quantize_blocks(FAKE, 2, rows, 2**20, 2**20, 128, FAKE, 2**20, FAKE, 2**13, 1, None) == UNSUPPORTED
    for M, N in ((1, 2**30), (64, 2**30), (65535 * 64, 2**18), (65535 * 64, 2**22)):
        assert L.dcq_fp8_block_gemm(FAKE, 2**24, FAKE, 1, 1, FAKE, 2**24, FAKE, 1, 1, None, 0, FAKE, 2, N, M, N, 2048, None) == UNSUPPORTED
    s = strides(128, 64, 64)
    assert L.dcq_kv8_append(FAKE, FAKE, 2, s, s, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, None, 1, 2**29, 4, 4000, 16, 64, 2, None) == UNSUPPORTED
    for total, group in ((4, 2**62), (2**29, 2), (4, 2**40)):
        assert L.dcq_kv8_attention(FAKE, 2, s, FAKE, s, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, None, 1, total, 4, 1, group, 16, 64, 1 << 12, 1.0, 1, 0, FAKE,
                                   1 << 40, None) == UNSUPPORTED
    assert L.dcq_kv8_attention(FAKE, 2, s, FAKE, s, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, None, 1, 2**28, 4, 60000, 1, 16, 64, 1 << 12, 1.0, 1, 0, FAKE, 1 << 40,
                               None) == UNSUPPORTED
