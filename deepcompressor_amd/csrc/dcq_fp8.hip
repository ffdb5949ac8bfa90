// 8-bit floating-point (e4m3) tensors with a float32 scale for each block of 128, and their matrix product (gfx950).
#include "dcq_fp8.cuh"

namespace dcq {

constexpr int kBlock = 128;  // columns that share a scale

// =============================================================================================
// Quantizer.  Per block: s = max|x| / 448 (0 -> 1), code = nearest e4m3 value to x / s, both IEEE float32, a tie to the
// upper neighbour: what the fake quantizer computes for sfp8_e4m3_nan with float32 scales.  One read of x, one write of
// the codes: bound by HBM.
// =============================================================================================
struct QuantizeParams {
  const void* x;
  int64_t rows, cols, ld_x;
  uint8_t* codes;
  int64_t ld_codes;
  float* scales;
  int64_t scale_row, scale_col;
  int32_t col_blocks;
};

// 16 consecutive elements of a row from column `col` on; beyond the row's end 0
template <int ST, bool VECTOR>
__device__ __forceinline__ void load_16(const typename Storage<ST>::elem_t* row, int64_t col, int64_t cols, float (&v)[16]) {
  using S = Storage<ST>;
  if (VECTOR && col + 16 <= cols) {
    Chunk<typename S::elem_t, S::kVec> c[16 / S::kVec];
#pragma unroll
    for (int i = 0; i < 16 / S::kVec; ++i) c[i] = load_chunk<typename S::elem_t, S::kVec>(row + col + i * S::kVec);
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = S::load(c[i / S::kVec].v[i % S::kVec]);
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = col + i < cols ? S::load(row[col + i]) : 0.0f;
  }
}

__device__ __forceinline__ float largest_of(const float (&v)[16]) {
  float m = 0.0f;
#pragma unroll
  for (int i = 0; i < 16; ++i) m = fmaxf(m, fabsf(v[i]));
  return m;
}

__device__ __forceinline__ float scale_of(float largest) {
  const float s = largest / kE4m3Max;
  return s == 0.0f ? 1.0f : s;
}

// x / s lies within +-448 after rounding (s is the rounded max / 448: the quotient exceeds 448 by less than the half
// step to the next value), unless s has lost bits below the normal range: that case is clamped.
__device__ __forceinline__ uint4 codes_of(const float (&v)[16], float s, float largest) {
  float q[16];
  const Divisor d = make_divisor(s, largest);
  if (d.fast) {
#pragma unroll
    for (int i = 0; i < 16; ++i) q[i] = div_fast(v[i], d);
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i) q[i] = clamp_e4m3(v[i] / s);
  }
  return {to_e4m3x4(q[0], q[1], q[2], q[3]), to_e4m3x4(q[4], q[5], q[6], q[7]), to_e4m3x4(q[8], q[9], q[10], q[11]),
          to_e4m3x4(q[12], q[13], q[14], q[15])};
}

// A scale for each row and 128 columns.  Eight lanes take a block, 16 elements each; a workgroup takes 4 blocks side by
// side in 8 rows, REPEAT times below each other.
template <int ST, bool VECTOR, int REPEAT>
__global__ __launch_bounds__(256) void quantize_rows_kernel(const QuantizeParams p) {
  const int team = threadIdx.x / 8;
  const int64_t kb = static_cast<int64_t>(blockIdx.y) * 4 + (team & 3);
  const int64_t row0 = static_cast<int64_t>(blockIdx.x) * (8 * REPEAT) + (team >> 2);
  if (kb >= p.col_blocks) return;
  const int64_t col = kb * kBlock + (threadIdx.x & 7) * 16;
  using elem_t = typename Storage<ST>::elem_t;
#pragma unroll
  for (int i = 0; i < REPEAT; ++i) {
    const int64_t row = row0 + i * 8;
    if (row >= p.rows) return;  // (a team's lanes have one row)
    float v[16];
    load_16<ST, VECTOR>(static_cast<const elem_t*>(p.x) + row * p.ld_x, col, p.cols, v);
    const float largest = team_max(largest_of(v), 8);
    const float s = scale_of(largest);
    if (col < p.cols) *reinterpret_cast<uint4*>(p.codes + row * p.ld_codes + col) = codes_of(v, s, largest);
    if ((threadIdx.x & 7) == 0) p.scales[row * p.scale_row + kb * p.scale_col] = s;
  }
}

// A scale for each 128 x 128 tile: a workgroup holds the tile in registers between the maximum and the codes.
template <int ST, bool VECTOR>
__global__ __launch_bounds__(256) void quantize_tiles_kernel(const QuantizeParams p) {
  const int64_t kb = blockIdx.y, rb = blockIdx.x;
  const int64_t col = kb * kBlock + (threadIdx.x & 7) * 16;
  using elem_t = typename Storage<ST>::elem_t;
  float v[4][16];
  float largest = 0.0f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t row = rb * kBlock + i * 32 + threadIdx.x / 8;
    load_16<ST, VECTOR>(static_cast<const elem_t*>(p.x) + min(row, p.rows - 1) * p.ld_x, col, p.cols, v[i]);
    largest = fmaxf(largest, largest_of(v[i]));  // (a row read twice does not change the maximum)
  }
  __shared__ float part[4];
  largest = team_max(largest, kWave);
  if (threadIdx.x % kWave == 0) part[threadIdx.x / kWave] = largest;
  __syncthreads();
  largest = fmaxf(fmaxf(part[0], part[1]), fmaxf(part[2], part[3]));
  const float s = scale_of(largest);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t row = rb * kBlock + i * 32 + threadIdx.x / 8;
    if (row < p.rows && col < p.cols) *reinterpret_cast<uint4*>(p.codes + row * p.ld_codes + col) = codes_of(v[i], s, largest);
  }
  if (threadIdx.x == 0) p.scales[rb * p.scale_row + kb * p.scale_col] = s;
}

template <int ST, bool VECTOR>
int launch_quantize(const QuantizeParams& p, int block_rows, hipStream_t stream) {
  if (block_rows == kBlock) {
    const dim3 grid(static_cast<unsigned>((p.rows + kBlock - 1) / kBlock), p.col_blocks);
    quantize_tiles_kernel<ST, VECTOR><<<grid, 256, 0, stream>>>(p);
  } else {
    const dim3 grid(static_cast<unsigned>((p.rows + 7) / 8), (p.col_blocks + 3) / 4);
    quantize_rows_kernel<ST, VECTOR, 1><<<grid, 256, 0, stream>>>(p);
  }
  DCQ_LAUNCH_CHECK("dcq_fp8_quantize_blocks");
  return DCQ_OK;
}

// =============================================================================================
// Product  y[m][n] = bias[n] + sum_kb sx[m][kb] sw[n / 128][kb] sum_{k in block kb} x[m][k] w[n][k]
//
// The inner sum is one v_mfma_f32_16x16x128_f8f6f4 per 16 x 16 outputs: a scale block is exactly the instruction's depth,
// so each result is multiplied by its two scales and added in float32.  The weights' rows are the instruction's rows: a
// lane ends with 4 consecutive outputs of one token.
//
// The 8-bit instructions do not hold their sums in full float32: against float64 their error over 128 products was up
// to 2^-12.5 of the sum of magnitudes for codes drawn evenly from all bit patterns, 2^-15.7 (1.5e-5 of the result in the
// 2-norm) for normally distributed values.  That is well below what the rounding to float16 or bfloat16 costs.  Float32 outputs take the bfloat16
// instruction instead, whose sums were off by 1e-8 (the codes convert exactly), at half the rate.
// =============================================================================================
struct ProductParams {
  const uint8_t* x;
  const uint8_t* w;
  const float* xs;
  const float* ws;
  int64_t ld_x, ld_w, xs_row, xs_col, ws_row, ws_col;
  const void* bias;
  void* y;
  int64_t ld_y, M, N, K;
  int32_t bias_storage, y_storage, y_vector;
};

// A lane's 32 codes of a fragment as the matrix instruction takes them.
template <bool EXACT>
struct Operand {
  i32x8 codes;
  __device__ __forceinline__ explicit Operand(const i32x8& c) : codes(c) {}
  static __device__ __forceinline__ f32x4 product(const Operand& a, const Operand& b) {
    const f32x4 zero = {0.0f, 0.0f, 0.0f, 0.0f};
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a.codes, b.codes, zero, 0, 0, 0, 0, 0, 0);
  }
};
template <>
struct Operand<true> {
  uint4 part[4];
  __device__ __forceinline__ explicit Operand(const i32x8& c) {
#pragma unroll
    for (int i = 0; i < 4; ++i) part[i] = codes8<DCQ_BF16>(c[2 * i], c[2 * i + 1]);
  }
  static __device__ __forceinline__ f32x4 product(const Operand& a, const Operand& b) {
    f32x4 t = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < 4; ++i) t = Half<DCQ_BF16>::mfma(a.part[i], b.part[i], t);
    return t;
  }
};

__device__ __forceinline__ void store_outputs(const ProductParams& p, int64_t m, int64_t n, f32x4 v) {
  if (m >= p.M || n >= p.N) return;
  const int count = static_cast<int>(min<int64_t>(4, p.N - n));
  if (p.bias != nullptr) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i < count) v[i] += load_as_f32(p.bias, p.bias_storage, n + i);
  }
  const int64_t at = m * p.ld_y + n;
  if (p.y_storage == DCQ_F32) {
    float* y = static_cast<float*>(p.y) + at;
    if (p.y_vector && count == 4) {
      *reinterpret_cast<f32x4*>(y) = v;
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (i < count) y[i] = v[i];
    }
  } else {
    Chunk<uint16_t, 4> c;
#pragma unroll
    for (int i = 0; i < 4; ++i) c.v[i] = p.y_storage == DCQ_F16 ? f32_to_f16(v[i]) : f32_to_bf16(v[i]);
    uint16_t* y = static_cast<uint16_t*>(p.y) + at;
    if (p.y_vector && count == 4) {
      store_chunk<uint16_t, 4>(y, c);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (i < count) y[i] = c.v[i];
    }
  }
}

// a lane's 32 bytes of a 16-row fragment from memory; bytes from column K on are 0
template <bool TAIL>
__device__ __forceinline__ i32x8 load_fragment(const uint8_t* row, int64_t col, int64_t K) {
  i32x4 lo = {0, 0, 0, 0}, hi = {0, 0, 0, 0};
  if (!TAIL || col < K) lo = *reinterpret_cast<const i32x4*>(row + col);
  if (!TAIL || col + 16 < K) hi = *reinterpret_cast<const i32x4*>(row + col + 16);
  if (TAIL) {
    const int left = static_cast<int>(max<int64_t>(0, min<int64_t>(32, K - col)));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      lo[i] &= bytes_before(left, i);
      hi[i] &= bytes_before(left, i + 4);
    }
  }
  return {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
}

// Few tokens: bound by the weights' bytes.  A workgroup takes 16 NT weight rows and 16 MT tokens; its waves share out the
// blocks along K and read their fragments straight from memory (no weight byte is wanted twice, so LDS would only add a
// stop on the way), and their sums are added in the waves' order.
template <int MT, int NT, int WAVES, bool EXACT>
__global__ __launch_bounds__(WAVES* kWave) void product_rows_kernel(const ProductParams p) {
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  const int64_t n0 = static_cast<int64_t>(blockIdx.x) * (16 * NT), m0 = static_cast<int64_t>(blockIdx.y) * (16 * MT);
  const int r = lane % 16, g = lane / 16;
  const uint8_t* wr[NT];
  const float* ws[NT];
  const uint8_t* xr[MT];
  const float* xs[MT];
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    wr[j] = p.w + min(n0 + j * 16 + r, p.N - 1) * p.ld_w;
    ws[j] = p.ws + min(n0 + j * 16, p.N - 1) / kBlock * p.ws_row;
  }
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    const int64_t m = min(m0 + i * 16 + r, p.M - 1);
    xr[i] = p.x + m * p.ld_x;
    xs[i] = p.xs + m * p.xs_row;
  }
  f32x4 acc[MT][NT];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};

  const int64_t whole = p.K / kBlock, blocks = (p.K + kBlock - 1) / kBlock;
  auto step = [&](int64_t kb, auto tail) {
    constexpr bool kTail = decltype(tail)::value;
    const int64_t col = kb * kBlock + g * 32;
    i32x8 ac[NT], bc[MT];
    float sx[MT];
#pragma unroll
    for (int j = 0; j < NT; ++j) ac[j] = load_fragment<kTail>(wr[j], col, p.K);
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      bc[i] = load_fragment<kTail>(xr[i], col, p.K);
      sx[i] = xs[i][kb * p.xs_col];
    }
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      const float sw = ws[j][kb * p.ws_col];
      const Operand<EXACT> a(ac[j]);
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        const f32x4 t = Operand<EXACT>::product(a, Operand<EXACT>(bc[i]));
        const float s = sx[i] * sw;
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[i][j][e] = __builtin_fmaf(t[e], s, acc[i][j][e]);
      }
    }
  };
  const int64_t share = (blocks + WAVES - 1) / WAVES;
  const int64_t first = wave * share, last = min(first + share, blocks);
  const int64_t last_whole = min(last, whole);
#pragma unroll 4
  for (int64_t kb = first; kb < last_whole; ++kb) step(kb, std::false_type{});
  if (last > whole && first < last) step(whole, std::true_type{});

  __shared__ f32x4 sums[WAVES - 1][MT * NT][kWave];
  if (wave > 0) {
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int j = 0; j < NT; ++j) sums[wave - 1][i * NT + j][lane] = acc[i][j];
  }
  __syncthreads();
  if (wave == 0) {
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        f32x4 v = acc[i][j];
#pragma unroll
        for (int w = 0; w < WAVES - 1; ++w) v += sums[w][i * NT + j][lane];
        store_outputs(p, m0 + i * 16 + r, n0 + j * 16 + g * 4, v);
      }
  }
}

}  // namespace dcq

using namespace dcq;

extern "C" int dcq_fp8_quantize_blocks(const void* x, int32_t storage, int64_t rows, int64_t cols, int64_t ld_x,
                                       int32_t block_rows, uint8_t* codes, int64_t ld_codes, float* scales,
                                       int64_t scale_row_stride, int64_t scale_col_stride, dcq_stream_t stream) {
  DCQ_REQUIRE(storage == DCQ_F32 || storage == DCQ_F16 || storage == DCQ_BF16, DCQ_ERR_ARGUMENT, "bad storage %d", storage);
  DCQ_REQUIRE(rows >= 0 && cols >= 0, DCQ_ERR_ARGUMENT, "bad sizes");
  if (rows == 0 || cols == 0) return DCQ_OK;
  DCQ_REQUIRE(x != nullptr && codes != nullptr && scales != nullptr, DCQ_ERR_ARGUMENT, "null pointer");
  DCQ_REQUIRE(block_rows == 1 || block_rows == kBlock, DCQ_ERR_UNSUPPORTED, "blocks have 1 or 128 rows, not %d", block_rows);
  DCQ_REQUIRE(rows == 1 || ld_x >= cols, DCQ_ERR_ARGUMENT, "rows of x overlap");
  DCQ_REQUIRE(ld_codes >= cols && ld_codes % 16 == 0 && reinterpret_cast<uintptr_t>(codes) % 16 == 0, DCQ_ERR_ARGUMENT,
              "rows of codes must start at multiples of 16 bytes");
  DCQ_REQUIRE(cols <= int64_t{65535} * kBlock && rows <= int64_t{0x7fffffff}, DCQ_ERR_UNSUPPORTED, "too many rows or columns");
  const int64_t size = storage == DCQ_F32 ? 4 : 2;
  DCQ_REQUIRE(reinterpret_cast<uintptr_t>(x) % size == 0, DCQ_ERR_ARGUMENT, "x is not aligned to its elements");
  const QuantizeParams p{x, rows, cols, ld_x, codes, ld_codes, scales, scale_row_stride, scale_col_stride,
                         static_cast<int32_t>((cols + kBlock - 1) / kBlock)};
  const bool vector = reinterpret_cast<uintptr_t>(x) % 16 == 0 && (rows == 1 || ld_x * size % 16 == 0);
  hipStream_t s = static_cast<hipStream_t>(stream);
  switch (storage) {
    case DCQ_F32:
      return vector ? launch_quantize<DCQ_F32, true>(p, block_rows, s) : launch_quantize<DCQ_F32, false>(p, block_rows, s);
    case DCQ_F16:
      return vector ? launch_quantize<DCQ_F16, true>(p, block_rows, s) : launch_quantize<DCQ_F16, false>(p, block_rows, s);
    default:
      return vector ? launch_quantize<DCQ_BF16, true>(p, block_rows, s) : launch_quantize<DCQ_BF16, false>(p, block_rows, s);
  }
}

extern "C" int dcq_fp8_block_gemm(const uint8_t* x, int64_t ld_x, const float* x_scales, int64_t xs_row_stride,
                                  int64_t xs_col_stride, const uint8_t* w, int64_t ld_w, const float* w_scales,
                                  int64_t ws_row_stride, int64_t ws_col_stride, const void* bias, int32_t bias_storage,
                                  void* y, int32_t y_storage, int64_t ld_y, int64_t M, int64_t N, int64_t K,
                                  dcq_stream_t stream) {
  auto known = [](int32_t st) { return st == DCQ_F32 || st == DCQ_F16 || st == DCQ_BF16; };
  DCQ_REQUIRE(known(y_storage) && (bias == nullptr || known(bias_storage)), DCQ_ERR_ARGUMENT, "bad storage");
  DCQ_REQUIRE(M >= 0 && N >= 0 && K >= 1, DCQ_ERR_ARGUMENT, "bad sizes");
  if (M == 0 || N == 0) return DCQ_OK;
  DCQ_REQUIRE(x && x_scales && w && w_scales && y, DCQ_ERR_ARGUMENT, "null pointer");
  DCQ_REQUIRE(M <= int64_t{65535} * 16 && N <= int64_t{0x7fffffff} && K <= int64_t{0x7fffffff}, DCQ_ERR_UNSUPPORTED,
              "too many rows or columns");
  auto aligned = [](const void* q, int64_t ld) { return reinterpret_cast<uintptr_t>(q) % 16 == 0 && ld % 16 == 0; };
  DCQ_REQUIRE(aligned(x, ld_x) && aligned(w, ld_w) && ld_x >= K && ld_w >= K, DCQ_ERR_ARGUMENT,
              "rows of codes must start at multiples of 16 bytes");
  DCQ_REQUIRE(ld_y >= N, DCQ_ERR_ARGUMENT, "rows of y overlap");
  const int64_t y_vec = y_storage == DCQ_F32 ? 16 : 8;
  const int32_t y_vector = reinterpret_cast<uintptr_t>(y) % y_vec == 0 && ld_y % 4 == 0;
  const ProductParams p{x, w, x_scales, w_scales, ld_x, ld_w, xs_row_stride, xs_col_stride, ws_row_stride, ws_col_stride,
                        bias, y, ld_y, M, N, K, bias_storage, y_storage, y_vector};
  hipStream_t s = static_cast<hipStream_t>(stream);
  const dim3 grid(static_cast<unsigned>((N + 15) / 16), static_cast<unsigned>((M + 15) / 16));
  if (y_storage == DCQ_F32)
    product_rows_kernel<1, 1, 4, true><<<grid, 4 * kWave, 0, s>>>(p);
  else
    product_rows_kernel<1, 1, 4, false><<<grid, 4 * kWave, 0, s>>>(p);
  DCQ_LAUNCH_CHECK("dcq_fp8_block_gemm");
  return DCQ_OK;
}
