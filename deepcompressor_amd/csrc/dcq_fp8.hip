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

// Workgroups follow each other along the rows: 8191 x 14336 bfloat16 takes 62 us (5.7 TB/s; a copy of its bytes 87 us), 79 us
// with workgroups below each other, 14336 x 4096 float32 in 128 x 128 tiles 51 us instead of 63.

// A scale for each row and 128 columns.  Eight lanes take a block, 16 elements each; a workgroup takes WIDE blocks side by
// side in 32 / WIDE rows: 4, or 1 where a row has fewer (300000 x 128: 21 us, 57 us with 4).
template <int ST, bool VECTOR, int WIDE>
__global__ __launch_bounds__(256) void quantize_rows_kernel(const QuantizeParams p) {
  const int team = threadIdx.x / 8;
  const int64_t strips = (p.col_blocks + WIDE - 1) / WIDE;
  const int64_t kb = blockIdx.x % strips * WIDE + team % WIDE, row = blockIdx.x / strips * (32 / WIDE) + team / WIDE;
  if (kb >= p.col_blocks || row >= p.rows) return;  // (a team's lanes have one row and block)
  const int64_t col = kb * kBlock + (threadIdx.x & 7) * 16;
  using elem_t = typename Storage<ST>::elem_t;
  float v[16];
  load_16<ST, VECTOR>(static_cast<const elem_t*>(p.x) + row * p.ld_x, col, p.cols, v);
  const float largest = team_max(largest_of(v), 8);
  const float s = scale_of(largest);
  if (col < p.cols) *reinterpret_cast<uint4*>(p.codes + row * p.ld_codes + col) = codes_of(v, s, largest);
  if ((threadIdx.x & 7) == 0) p.scales[row * p.scale_row + kb * p.scale_col] = s;
}

// A scale for each 128 x 128 tile: a workgroup holds the tile in registers between the maximum and the codes.
template <int ST, bool VECTOR>
__global__ __launch_bounds__(256) void quantize_tiles_kernel(const QuantizeParams p) {
  const int64_t kb = blockIdx.x % p.col_blocks, rb = blockIdx.x / p.col_blocks;
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
  const int wide = p.col_blocks >= 4 ? 4 : 1;
  const int64_t bands = block_rows == kBlock ? (p.rows + kBlock - 1) / kBlock : (p.rows + 32 / wide - 1) / (32 / wide);
  const int64_t workgroups = bands * (block_rows == kBlock ? p.col_blocks : (p.col_blocks + wide - 1) / wide);
  DCQ_REQUIRE(launch_fits(workgroups, 256), DCQ_ERR_UNSUPPORTED, "too many rows and columns");
  const dim3 grid(static_cast<unsigned>(workgroups));
  if (block_rows == kBlock)
    quantize_tiles_kernel<ST, VECTOR><<<grid, 256, 0, stream>>>(p);
  else if (wide == 4)
    quantize_rows_kernel<ST, VECTOR, 4><<<grid, 256, 0, stream>>>(p);
  else
    quantize_rows_kernel<ST, VECTOR, 1><<<grid, 256, 0, stream>>>(p);
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
// The 8-bit instructions do not hold their sums in full float32: they take products eight at a time and cut them off below
// 2^-13 of the power of two of the eight's largest (the eights are then added in float32).  Against float64 the error over
// 128 products was up to 2^-12.5 of the sum of magnitudes for codes drawn evenly from all bit patterns, 2^-15.7 (1.5e-5 of the
// result in the 2-norm) for normally distributed values: below what the rounding to float16 or bfloat16 costs, unless terms
// cancel (whole steps cut off would cost 2e-5 there: a part of it is rounded or kept).  Float32
// outputs take the bfloat16 instruction instead, whose sums were off by 1e-8 (the codes convert exactly), at half the rate.
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
  int32_t bias_storage, y_storage;
  int32_t y_vector;  // outputs at multiples of 4 (columns) can be stored 4 at a time; 2: 8 at multiples of 8
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
    for (int i = 0; i < 4; ++i) part[i] = codes8<DCQ_BF16>(c[2 * i], c[2 * i + 1], 1.0f);
  }
  static __device__ __forceinline__ f32x4 product(const Operand& a, const Operand& b) {
    f32x4 t = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < 4; ++i) t = Half<DCQ_BF16>::mfma(a.part[i], b.part[i], t);
    return t;
  }
};

__device__ __forceinline__ uint16_t round_to_16(float v, int storage) {
  return storage == DCQ_F16 ? f32_to_f16(v) : __builtin_bit_cast(uint16_t, static_cast<__bf16>(v));
}

__device__ __forceinline__ f32x4 bias_of(const ProductParams& p, int64_t n) {
  f32x4 b = {0.0f, 0.0f, 0.0f, 0.0f};
  if (p.bias != nullptr) {
#pragma unroll
    for (int i = 0; i < 4; ++i) b[i] = load_as_f32(p.bias, p.bias_storage, min(n + i, p.N - 1));
  }
  return b;
}

__device__ __forceinline__ void store_outputs(const ProductParams& p, int64_t m, int64_t n, f32x4 v) {
  if (m >= p.M || n >= p.N) return;
  const int count = static_cast<int>(min<int64_t>(4, p.N - n));
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
    for (int i = 0; i < 4; ++i) c.v[i] = round_to_16(v[i], p.y_storage);
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

// columns of the last block from K on count as 0: `left` bytes of the lane's 32 stay
__device__ __forceinline__ i32x8 masked(i32x8 v, int left) {
#pragma unroll
  for (int k = 0; k < 8; ++k) v[k] &= bytes_before(left, k);
  return v;
}

// Few tokens: bound by the weights' bytes.  A workgroup takes 16 NT weight rows and 16 MT tokens; its waves share out the
// blocks along K and read their fragments straight from memory (no weight byte is wanted twice, so LDS would only add a
// stop on the way), DEPTH blocks at a time: a wave has that many 2 KiB fragments of each 16 rows under way.  The waves' sums
// are added in the waves' order.
template <int MT, int NT, int WAVES, int DEPTH, bool EXACT>
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

  const int64_t blocks = (p.K + kBlock - 1) / kBlock, last_piece = (p.K + 15) / 16 * 16 - 16;
  const int64_t share = (blocks + WAVES - 1) / WAVES;
  const int64_t first = wave * share, last = min(first + share, blocks);
  for (int64_t kb0 = first; kb0 < last; kb0 += DEPTH) {
    i32x8 ac[DEPTH][NT], bc[DEPTH][MT];
    float sx[DEPTH][MT], sw[DEPTH][NT];
#pragma unroll
    for (int d = 0; d < DEPTH; ++d) {
      // (blocks behind this wave's share and pieces behind the row's end: the last ones again, and not used)
      const int64_t kb = min(kb0 + d, last - 1);
      const int64_t c0 = min(kb * kBlock + g * 32, last_piece), c1 = min(kb * kBlock + g * 32 + 16, last_piece);
      auto fragment = [&](const uint8_t* row) {
        const i32x4 lo = *reinterpret_cast<const i32x4*>(row + c0), hi = *reinterpret_cast<const i32x4*>(row + c1);
        return i32x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
      };
#pragma unroll
      for (int j = 0; j < NT; ++j) ac[d][j] = fragment(wr[j]);
#pragma unroll
      for (int i = 0; i < MT; ++i) bc[d][i] = fragment(xr[i]);
#pragma unroll
      for (int j = 0; j < NT; ++j) sw[d][j] = ws[j][kb * p.ws_col];
#pragma unroll
      for (int i = 0; i < MT; ++i) sx[d][i] = xs[i][kb * p.xs_col];
    }
#pragma unroll
    for (int d = 0; d < DEPTH; ++d) {
      if (kb0 + d >= last) break;
      if ((kb0 + d + 1) * kBlock > p.K) {
        const int left = static_cast<int>(p.K - (kb0 + d) * kBlock) - g * 32;
#pragma unroll
        for (int j = 0; j < NT; ++j) ac[d][j] = masked(ac[d][j], left);
#pragma unroll
        for (int i = 0; i < MT; ++i) bc[d][i] = masked(bc[d][i], left);
      }
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        const Operand<EXACT> a(ac[d][j]);
#pragma unroll
        for (int i = 0; i < MT; ++i) {
          const f32x4 t = Operand<EXACT>::product(a, Operand<EXACT>(bc[d][i]));
          const float s = sx[d][i] * sw[d][j];
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[i][j][e] = __builtin_fmaf(t[e], s, acc[i][j][e]);
        }
      }
    }
  }

  __shared__ f32x4 sums[WAVES - 1][MT * NT][kWave];
  if (wave > 0) {
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int j = 0; j < NT; ++j) sums[wave - 1][i * NT + j][lane] = acc[i][j];
  }
  f32x4 bias[NT];
  if (wave == 0) {
#pragma unroll
    for (int j = 0; j < NT; ++j) bias[j] = bias_of(p, n0 + j * 16 + g * 4);
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
        store_outputs(p, m0 + i * 16 + r, n0 + j * 16 + g * 4, v + bias[j]);
      }
  }
}

// Tiles in order: 8 tiles of tokens side by side, then the next weights; each XCD (workgroups go round the 8 of them) takes
// a contiguous run of that order, so that the workgroups that share an L2 share rows and columns.
struct Tile {
  int64_t m0, n0;
};
template <int BM, int BN>
__device__ __forceinline__ Tile tile_of_workgroup(const ProductParams& p) {
  // (32 bits: a division of 64 takes a few hundred instructions, and the first load waits for three of them)
  const uint32_t tiles_m = static_cast<uint32_t>((p.M + BM - 1) / BM), tiles_n = static_cast<uint32_t>((p.N + BN - 1) / BN);
  const uint32_t tiles = tiles_m * tiles_n, xcd = blockIdx.x % 8, per = tiles / 8, rest = tiles % 8;
  const uint32_t t = xcd * per + min(xcd, rest) + blockIdx.x / 8;
  const uint32_t band = t / (8 * tiles_n), in_band = t % (8 * tiles_n), band_m = min(8u, tiles_m - band * 8);
  return {static_cast<int64_t>(band * 8 + in_band % band_m) * BM, static_cast<int64_t>(in_band / band_m) * BN};
}

// In between: tiles of 64 x 64, too few of them to fill the chip, so each is also split along K inside the workgroup.  Groups
// of four waves (2 x 2, 32 x 32 each) take SPLIT consecutive blocks of 128 columns at a time, whose codes go to LDS directly, one
// such stage ahead of the arithmetic; at the end the groups' sums are added in order.  LDS rows and pieces as in the tile
// kernel below.
constexpr int kRowBytes = kBlock;

template <int SPLIT, bool EXACT>
__global__ __launch_bounds__(SPLIT * 256) void product_split_kernel(const ProductParams p) {
  constexpr int kTile = 64;
  constexpr int kPart = 2 * kTile * kRowBytes, kStage = SPLIT * kPart;  // a block's weights, then its tokens
  extern __shared__ __align__(1024) unsigned char lds[];                // [2][SPLIT][kPart]
  const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int r = lane % 16, g = lane / 16, group = wave / 4, wm = wave % 2, wn = wave / 2 % 2;
  const Tile at = tile_of_workgroup<kTile, kTile>(p);
  const int64_t m0 = at.m0, n0 = at.n0;
  const int64_t blocks = (p.K + kBlock - 1) / kBlock, stages = (blocks + SPLIT - 1) / SPLIT;
  const int64_t last_piece = (p.K + 15) / 16 * 16 - 16;

  // a group's waves fetch its own block: 64 weight rows and 64 token rows, 4 pieces a lane
  const int piece = (lane % 8) ^ ((wave & 1) * 4 + lane / 16);
  const uint8_t* source[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int row = (i % 2) * 32 + (wave % 4) * 8 + lane / 8;
    source[i] = i < 2 ? p.w + min(n0 + row, p.N - 1) * p.ld_w : p.x + min(m0 + row, p.M - 1) * p.ld_x;
  }
  const float* xs[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) xs[i] = p.xs + min(m0 + wm * 32 + i * 16 + r, p.M - 1) * p.xs_row;
  const float* ws = p.ws + min(n0, p.N - 1) / kBlock * p.ws_row;
  float sx[2], sw;
  auto fetch = [&](int64_t stage, int buffer) {
    const int64_t kb = min(stage * SPLIT + group, blocks - 1);  // (blocks that are none: the last one again, and not used)
#pragma unroll
    for (int i = 0; i < 2; ++i) sx[i] = xs[i][kb * p.xs_col];
    sw = ws[kb * p.ws_col];
    const int64_t col = min(kb * kBlock + piece * 16, last_piece);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      load_to_lds_16(source[i] + col, lds + buffer * kStage + group * kPart + (i * 256 + wave % 4 * kWave) * 16);
  };
  const int a_base = group * kPart + (wn * 32 + r) * kRowBytes, b_base = group * kPart + (kTile + wm * 32 + r) * kRowBytes;
  const int lo = ((2 * g) ^ (r / 2)) * 16, hi = ((2 * g + 1) ^ (r / 2)) * 16;

  f32x4 acc[2][2], bias[2];
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    bias[j] = bias_of(p, n0 + wn * 32 + j * 16 + g * 4);  // (early: at the end nothing would hide the wait)
#pragma unroll
    for (int i = 0; i < 2; ++i) acc[j][i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  }
  // Tiles of different weights begin at different stages and go round: in step, all of them would read the same columns of rows that
  // lie a power of two apart, out of few of the memory's channels (48 x 28672 x 4096: 28 us in step, 26 so).  Not so tiles of
  // different tokens: what a token gives must not depend on its place in the batch, and sums in another order would.  (They were
  // no faster: 256 x 4096 x 4096 13.3 us, 12.6 now.)
  int64_t stage = static_cast<uint32_t>(at.n0 / kTile) % static_cast<uint32_t>(stages);
  fetch(stage, 0);
  for (int64_t turn = 0; turn < stages; ++turn) {
    const int buffer = static_cast<int>(turn & 1);
    const int64_t now = stage;
    stage = stage + 1 == stages ? 0 : stage + 1;
    wait_direct_loads();
    float s[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) s[i] = sx[i] * sw;
#pragma unroll
    for (int i = 0; i < 2; ++i) asm volatile("" : "+v"(s[i]));
    __syncthreads();  // the stage has landed, and everyone is done with the other one
    if (turn + 1 < stages) fetch(stage, buffer ^ 1);
    const int64_t kb = now * SPLIT + group;
    if (kb < blocks) {
      const unsigned char* part = lds + buffer * kStage;
      auto fragment = [&](int from) {
        const i32x4 x = *reinterpret_cast<const i32x4*>(part + from + lo), y = *reinterpret_cast<const i32x4*>(part + from + hi);
        return i32x8{x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]};
      };
      i32x8 ac[2], bc[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        ac[i] = fragment(a_base + i * 16 * kRowBytes);
        bc[i] = fragment(b_base + i * 16 * kRowBytes);
      }
      if ((kb + 1) * kBlock > p.K) {
        const int left = static_cast<int>(p.K - kb * kBlock) - g * 32;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          ac[i] = masked(ac[i], left);
          bc[i] = masked(bc[i], left);
        }
      }
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const Operand<EXACT> a(ac[j]);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const f32x4 t = Operand<EXACT>::product(a, Operand<EXACT>(bc[i]));
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[j][i][e] = __builtin_fmaf(t[e], s[i], acc[j][i][e]);
        }
      }
    }
  }
  __syncthreads();  // (every load has been waited for: LDS is free)
  f32x4* sums = reinterpret_cast<f32x4*>(lds);  // [SPLIT - 1][4 waves][4][64]
  if (group > 0) {
#pragma unroll
    for (int t = 0; t < 4; ++t) sums[(((group - 1) * 4 + wave % 4) * 4 + t) * kWave + lane] = acc[t / 2][t % 2];
  }
  __syncthreads();
  if (group > 0) return;
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int64_t n = n0 + wn * 32 + j * 16 + g * 4;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      f32x4 v = acc[j][i];
#pragma unroll
      for (int k = 0; k < SPLIT - 1; ++k) v += sums[((k * 4 + wave) * 4 + j * 2 + i) * kWave + lane];
      store_outputs(p, m0 + wm * 32 + i * 16 + r, n, v + bias[j]);
    }
  }
}

// Many tokens: bound by the matrix pipe.  A workgroup computes BM tokens x BN weight rows; its WM x WN waves take
// equal parts.  Per block of 128 columns both operands' tiles go from memory to LDS directly, one block ahead of the
// arithmetic (two buffers, one barrier per block).  A tile's row is the block's 128 bytes, 8 pieces of 16; piece c of row
// r lies at position c ^ (r / 2 & 7): the same piece of 16 rows takes all 64 banks once (with r & 7 in its place, half of
// the LDS cycles were conflicts); since direct
// loads fill LDS in lane order, the lanes choose their source pieces accordingly.
//
// The instructions' results are scaled into the sums a few instructions later, so that vector and matrix pipe run side by
// side (the scaling costs nothing: without it the time is the same).  The barrier between two blocks stands before the last
// two weight fragments' instructions, whose operands are in registers by then: behind it the next block's first fragments are
// read while those instructions run (5 % against a barrier between the blocks).  8192 x 14336 x 4096: 450 us, 2.14 PFLOP/s,
// 8192 x 4096 x 14336: 397 - 414 us, 2.32 - 2.4 PFLOP/s; a library's 8-bit product without block scales takes 393 and 287 us.  The same
// loop without its loads takes 340 us for the latter: what bounds it now is the operands' way into LDS beside the fragments'
// way out of it.
template <int BM, int BN, int WM, int WN, bool EXACT>
__global__ __launch_bounds__(WM* WN* kWave) __attribute__((amdgpu_waves_per_eu(2))) void product_tile_kernel(const ProductParams p) {
  constexpr int kThreads = WM * WN * kWave;
  constexpr int MT = BM / WM / 16, NT = BN / WN / 16;
  constexpr int kStage = (BM + BN) * kRowBytes;
  constexpr int kLoads = (BM + BN) * 8 / kThreads;  // 16-byte pieces per thread and block
  static_assert(BN * 8 % kThreads == 0 && BM * 8 % kThreads == 0, "whole loads");
  extern __shared__ __align__(1024) unsigned char lds[];  // [2][weights, tokens]
  const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int r = lane % 16, g = lane / 16;

  const Tile at = tile_of_workgroup<BM, BN>(p);
  const int64_t m0 = at.m0, n0 = at.n0;

  // where this thread's pieces come from: rows of W first, then of X, as offsets from the tiles' first rows (rows behind the
  // last repeat it)
  constexpr int kLoadsW = BN * 8 / kThreads;
  const int piece = (lane % 8) ^ ((wave & 1) * 4 + lane / 16);
  uint32_t offset[kLoads];
#pragma unroll
  for (int i = 0; i < kLoads; ++i) {
    const int row = (i * kThreads + static_cast<int>(threadIdx.x)) / 8;
    offset[i] = static_cast<uint32_t>(i < kLoadsW ? min<int64_t>(row, p.N - 1 - n0) * p.ld_w : min<int64_t>(row - BN, p.M - 1 - m0) * p.ld_x);
    offset[i] += piece * 16;
  }
  const uint8_t* w0 = p.w + n0 * p.ld_w;
  const uint8_t* x0 = p.x + m0 * p.ld_x;
  const int64_t blocks = (p.K + kBlock - 1) / kBlock;
  // the last block's pieces that lie behind column K are not read (the last one before it is, again); what they leave in
  // LDS is masked below
  const int last_piece = static_cast<int>((p.K - (blocks - 1) * kBlock + 15) / 16) - 1;
  const uint32_t short_of = static_cast<uint32_t>(max(piece - last_piece, 0)) * 16;
  auto fetch = [&](int64_t kb, int buffer, int i) {
    const uint32_t back = kb + 1 == blocks ? short_of : 0;
    load_to_lds_16((i < kLoadsW ? w0 : x0) + kb * kBlock, offset[i] - back, lds + buffer * kStage + (i * kThreads + wave * kWave) * 16);
  };
  auto fetch_all = [&](int64_t kb, int buffer) {
#pragma unroll
    for (int i = 0; i < kLoads; ++i) fetch(kb, buffer, i);
  };

  const int wm = wave % WM, wn = wave / WM;
  uint32_t xs_at[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) xs_at[i] = static_cast<uint32_t>(min<int64_t>(wm * (MT * 16) + i * 16 + r, p.M - 1 - m0) * p.xs_row);
  const float* xs = p.xs + m0 * p.xs_row;
  static_assert(kBlock % (NT * 16) == 0, "a wave's weight rows have one scale");
  // (a vector load, through the lane's own index: a scalar one would share its counter with the LDS reads, out of order)
  const float* ws = p.ws + min<int64_t>(n0 + static_cast<int>(threadIdx.x) / (WM * kWave) * (NT * 16), p.N - 1) / kBlock * p.ws_row;
  const int a_base = (wn * (NT * 16) + r) * kRowBytes, b_base = (BN + wm * (MT * 16) + r) * kRowBytes;
  const int lo = ((2 * g) ^ (r / 2)) * 16, hi = ((2 * g + 1) ^ (r / 2)) * 16;

  f32x4 acc[NT][MT];
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int i = 0; i < MT; ++i) acc[j][i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};

  float sx[MT], sw;
  auto fetch_scales = [&](int64_t kb) {
#pragma unroll
    for (int i = 0; i < MT; ++i) sx[i] = xs[kb * p.xs_col + xs_at[i]];
    sw = ws[kb * p.ws_col];
  };
  auto fragment = [&](const unsigned char* tile, int at) {
    const i32x4 x = *reinterpret_cast<const i32x4*>(tile + at + lo), y = *reinterpret_cast<const i32x4*>(tile + at + hi);
    return i32x8{x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]};
  };
  const int left = static_cast<int>(p.K - (blocks - 1) * kBlock) - g * 32;

  // Token fragments (all of a block's) and weight fragments (four places, taken in turns: the next block's first has one
  // that the last two do not use) live across blocks.
  i32x8 bc[MT], ac[NT == 8 ? 3 : 4];
  float s[MT];
  auto place = [](int j) {
    if (NT == 8) return j == 5 ? 0 : j == 4 || j == 7 ? 2 : j == 6 ? 1 : j % 2;
    return j == NT - 1 ? 2 : j == NT - 2 ? 1 : j % 2 ? 3 : 0;
  };
  auto scales = [&](float(&to)[MT]) {
#pragma unroll
    for (int i = 0; i < MT; ++i) to[i] = sx[i] * sw;
  };
  auto block = [&](int64_t kb, auto tail) {
    constexpr bool kTail = decltype(tail)::value;  // the last block, and not a whole one
    constexpr int kLag = 3, kCount = NT * MT, kEarly = (NT - 2) * MT;
    const unsigned char* tile = lds + (kb & 1) * kStage;
    const unsigned char* next_tile = lds + ((kb + 1) & 1) * kStage;
    const int64_t ahead = min(kb + 2, blocks - 1);  // (at the end the last block again: a branch would cut the schedule in two)
    f32x4 sums[kLag + 1];
    float next_s[MT];
    if (kTail) {
#pragma unroll
      for (int i = 0; i < MT; ++i) bc[i] = masked(bc[i], left);
    }
    static_for<kCount + kLag>([&](auto step) {
      constexpr int q = decltype(step)::value;
      // the last two weight fragments are multiplied token fragment by token fragment, so that these become free one by one
      auto row_of = [](int n) { return n < kEarly ? n / MT : NT - 2 + (n - kEarly) % 2; };
      auto col_of = [](int n) { return n < kEarly ? n % MT : (n - kEarly) / 2; };
      if constexpr (q < kEarly && q % MT == 0) {
        constexpr int j = q / MT + 1;
        ac[place(j)] = fragment(tile, a_base + j * 16 * kRowBytes);
        if constexpr (j == NT - 2) ac[place(j + 1)] = fragment(tile, a_base + (j + 1) * 16 * kRowBytes);
      }
      if constexpr (q == kEarly && !kTail) {
        wait_direct_loads();  // the next block's codes and scales have landed: this wave's ...
        scales(next_s);
#pragma unroll
        for (int i = 0; i < MT; ++i) asm volatile("" : "+v"(next_s[i]));
        __syncthreads();  // ... and everyone's, and everyone has read this block
        fetch_scales(ahead);
        ac[0] = fragment(next_tile, a_base);
      }
      if constexpr (q >= kEarly && q < kCount && !kTail) {
        // one or two loads per instruction: issued all at once they stall the wave until the others' have been taken too
        constexpr int kEach = (kLoads + 2 * MT - 1) / (2 * MT), first = (q - kEarly) * kEach;
#pragma unroll
        for (int i = first; i < first + kEach && i < kLoads; ++i) fetch(ahead, static_cast<int>(kb) & 1, i);
      }
      if constexpr (q < kCount) {
        constexpr int j = row_of(q), i = col_of(q);
        if constexpr (kTail && (q < kEarly ? i == 0 : q < kEarly + 2)) ac[place(j)] = masked(ac[place(j)], left);
        sums[q % (kLag + 1)] = Operand<EXACT>::product(Operand<EXACT>(ac[place(j)]), Operand<EXACT>(bc[i]));
        if constexpr (!kTail && q >= kEarly && j == NT - 1) bc[i] = fragment(next_tile, b_base + i * 16 * kRowBytes);
      }
      if constexpr (q >= kLag) {
        constexpr int d = q - kLag, j = row_of(d), i = col_of(d);
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[j][i][e] = __builtin_fmaf(sums[d % (kLag + 1)][e], s[i], acc[j][i][e]);
      }
      __builtin_amdgcn_sched_barrier(0);  // the order as written: left alone, the scheduler gathers reads and results
    });
    if (!kTail) {
#pragma unroll
      for (int i = 0; i < MT; ++i) s[i] = next_s[i];
    }
  };

  fetch_scales(0);
  fetch_all(0, 0);
  wait_direct_loads();
  scales(s);
#pragma unroll
  for (int i = 0; i < MT; ++i) asm volatile("" : "+v"(s[i]));
  __syncthreads();
  if (blocks > 1) {
    fetch_scales(1);
    fetch_all(1, 1);
  }
  ac[0] = fragment(lds, a_base);
#pragma unroll
  for (int i = 0; i < MT; ++i) bc[i] = fragment(lds, b_base + i * 16 * kRowBytes);
  // (the last block looks ahead like the others, at codes that are there and not used: one copy of the loop)
  const int64_t whole = p.K / kBlock;
  for (int64_t kb = 0; kb < whole; ++kb) block(kb, std::false_type{});
  if (whole < blocks) block(whole, std::true_type{});
  wait_direct_loads();  // (no load may be under way into LDS that is used again, here or by the next workgroup)
  __syncthreads();
  const int64_t wave_m = m0 + wm * (MT * 16), wave_n = n0 + wn * (NT * 16);
  if (!EXACT && p.y_vector == 2 && wave_n + NT * 16 <= p.N) {
    // Each wave turns its outputs round in LDS, so that a row's 16-byte pieces are stored side by side: MT * 16 rows of NT * 32
    // bytes, a row's pieces exchanged by its number.
    constexpr int kPieces = NT * 2, kBytes = NT * 32;
    unsigned char* out = lds + wave * (MT * 16 * kBytes);
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      const f32x4 b = bias_of(p, wave_n + j * 16 + g * 4);
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        const f32x4 v = acc[j][i] + b;
        Chunk<uint16_t, 4> c;
#pragma unroll
        for (int e = 0; e < 4; ++e) c.v[e] = round_to_16(v[e], p.y_storage);
        store_chunk<uint16_t, 4>(reinterpret_cast<uint16_t*>(out + (i * 16 + r) * kBytes + ((2 * j + g / 2) ^ (r % kPieces)) * 16 + (g & 1) * 8), c);
      }
    }
    // (one wave's own writes and reads: in order)
    constexpr int kRowsAtOnce = kWave / kPieces;
#pragma unroll
    for (int t = 0; t < MT * 16 / kRowsAtOnce; ++t) {
      const int row = t * kRowsAtOnce + lane / kPieces, c = lane % kPieces;
      const uint4 v = *reinterpret_cast<const uint4*>(out + row * kBytes + (c ^ (row % 16 % kPieces)) * 16);
      if (wave_m + row < p.M) *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.y) + (wave_m + row) * p.ld_y + wave_n + c * 8) = v;
    }
    return;
  }
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    const f32x4 b = bias_of(p, wave_n + j * 16 + g * 4);
#pragma unroll
    for (int i = 0; i < MT; ++i) store_outputs(p, wave_m + i * 16 + r, wave_n + j * 16 + g * 4, acc[j][i] + b);
  }
}

template <int BM, int BN, int WM, int WN, bool EXACT>
int launch_tiles(const ProductParams& p, hipStream_t stream) {
  const int bytes = 2 * (BM + BN) * kRowBytes;
  auto kernel = product_tile_kernel<BM, BN, WM, WN, EXACT>;
  if (bytes > 64 * 1024) {
    const int rc = hip_check(hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, bytes),
                             "hipFuncSetAttribute(product LDS)");
    if (rc != DCQ_OK) return rc;
  }
  const int64_t tiles = (p.M + BM - 1) / BM * ((p.N + BN - 1) / BN);
  DCQ_REQUIRE(launch_fits(tiles, WM * WN * kWave), DCQ_ERR_UNSUPPORTED, "too many rows or columns");
  kernel<<<static_cast<unsigned>(tiles), WM * WN * kWave, bytes, stream>>>(p);
  DCQ_LAUNCH_CHECK("dcq_fp8_block_gemm");
  return DCQ_OK;
}

template <int SPLIT, bool EXACT>
int launch_split(const ProductParams& p, hipStream_t stream) {
  const int bytes = 2 * SPLIT * 2 * 64 * kRowBytes;
  auto kernel = product_split_kernel<SPLIT, EXACT>;
  if (bytes > 64 * 1024) {
    const int rc = hip_check(hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, bytes),
                             "hipFuncSetAttribute(product LDS)");
    if (rc != DCQ_OK) return rc;
  }
  const int64_t tiles = (p.M + 63) / 64 * ((p.N + 63) / 64);
  DCQ_REQUIRE(launch_fits(tiles, SPLIT * 256), DCQ_ERR_UNSUPPORTED, "too many rows or columns");
  kernel<<<static_cast<unsigned>(tiles), SPLIT * 256, bytes, stream>>>(p);
  DCQ_LAUNCH_CHECK("dcq_fp8_block_gemm");
  return DCQ_OK;
}

template <int MT, int NT, int WAVES, int DEPTH, bool EXACT>
int launch_rows(const ProductParams& p, hipStream_t stream) {
  const dim3 grid(static_cast<unsigned>((p.N + 16 * NT - 1) / (16 * NT)), static_cast<unsigned>((p.M + 16 * MT - 1) / (16 * MT)));
  DCQ_REQUIRE(launch_fits(grid.x, WAVES * kWave), DCQ_ERR_UNSUPPORTED, "too many rows or columns");
  product_rows_kernel<MT, NT, WAVES, DEPTH, EXACT><<<grid, WAVES * kWave, 0, stream>>>(p);
  DCQ_LAUNCH_CHECK("dcq_fp8_block_gemm");
  return DCQ_OK;
}

// Which kernel: the largest tiles that still give most compute units one (a larger tile moves fewer bytes per product), the
// weights' bytes streamed once where there are few tokens.  Kernel times in us, bfloat16 / float32 outputs, M x N x K, with the
// neighbours':
//   256-tile   1024 x 14336 x 4096 (224 tiles)  58 (128-tile 71);  2048 x 4096 x 4096 (128)  53 (40).  16 bits only
//   128-tile   1024 x 4096 x 4096 (256 tiles)  28 / 44 (split 2: 36 / 52);  128 x 28672 x 4096 (224)  47 / 54 (46 / 54);
//              512 x 4096 x 4096 (128)  26 / 41 (20 / 28)
//   split 2    512 x 4096 x 4096 (512 tiles of 64)  20 / 28 (split 4: 24 / 32);  48 x 28672 x 4096 (448)  26 / 30 (35 / 36)
//   split 4    256 x 4096 x 4096 (256)  13 / 17.5 (split 2: 15 / 19);  64 x 14336 x 4096 (224)  15 / 17 (rows: 33 / 33);
//              64 x 4096 x 4096 (64)  13 / 15.6 (11.5 / 11.8)
//   rows       1 x 4096 x 4096  6.3;  16 x 14336 x 4096  15.6;  32 x 4096 x 14336  24 / 23 (split 4: 32 / 42);
//              64 x 4096 x 14336  29 / 29 (35 / 42)
// Short K leaves nothing to split: up to 1024, split 2  512 x 1024 x 1024 (128 tiles)  6.4 / 7.4 (split 4: 7.3 / 7.6);
// 333 x 1001 x 512  5.8 / 6.4 (6.4 / 6.9);  and where weights and tokens are few besides, rows  128 x 2048 x 1024 (64 tiles)
// 5.5 / 5.7 (split 2: 6.2 / 7.2);  256 x 512 x 2048 (32)  7.5 / 7.5 (split 4: 8.4 / 9.9);  but 512 x 768 x 768 (96)  6.8 / 6.6
// (split 2: 5.8 / 6.6).  Left for it: 128 x 1024 x 4096 (32)  11.9 / 15.4, by rows of 16 weights 9.5 / 9.0.
template <bool EXACT>
int launch_product(const ProductParams& p, hipStream_t stream) {
  auto tiles = [&](int64_t size) { return (p.M + size - 1) / size * ((p.N + size - 1) / size); };
  constexpr int64_t kMost = 192;  // three quarters of the 256 compute units
  // (the tile kernels address a tile's rows by 32-bit offsets from its first)
  const bool near = p.ld_x < (1 << 23) && p.ld_w < (1 << 23) && p.xs_row < (1 << 22);
  if constexpr (!EXACT) {
    if (near && tiles(256) >= kMost) return launch_tiles<256, 256, 4, 2, EXACT>(p, stream);
  }
  if (near && tiles(128) >= kMost && p.M > 64) return launch_tiles<128, 128, 2, 2, EXACT>(p, stream);
  if (p.M <= 16) return p.N > 8192 ? launch_rows<1, 2, 8, 2, EXACT>(p, stream) : launch_rows<1, 1, 8, 2, EXACT>(p, stream);
  if (p.M <= 64 && tiles(64) < 160) return p.M <= 32 ? launch_rows<2, 1, 8, 2, EXACT>(p, stream) : launch_rows<2, 2, 4, 2, EXACT>(p, stream);
  if (tiles(64) <= 64 && p.K <= 2048) return launch_rows<2, 2, 4, 2, EXACT>(p, stream);
  return tiles(64) > 256 || p.K <= 1024 ? launch_split<2, EXACT>(p, stream) : launch_split<4, EXACT>(p, stream);
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
  DCQ_REQUIRE(cols <= int64_t{0x7fffffff} && rows <= int64_t{0x7fffffff}, DCQ_ERR_UNSUPPORTED, "too many rows or columns");
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
  DCQ_REQUIRE(xs_row_stride >= 0 && xs_col_stride >= 0 && ws_row_stride >= 0 && ws_col_stride >= 0, DCQ_ERR_ARGUMENT, "negative stride");
  DCQ_REQUIRE(x && x_scales && w && w_scales && y, DCQ_ERR_ARGUMENT, "null pointer");
  DCQ_REQUIRE(M <= int64_t{65535} * 64 && N <= int64_t{1} << 30 && K <= int64_t{1} << 30 && (M + 63) / 64 * ((N + 63) / 64) <= int64_t{0x7fffffff}, DCQ_ERR_UNSUPPORTED,
              "too many rows or columns");
  auto aligned = [](const void* q, int64_t ld) { return reinterpret_cast<uintptr_t>(q) % 16 == 0 && ld % 16 == 0; };
  DCQ_REQUIRE(aligned(x, ld_x) && aligned(w, ld_w) && ld_x >= K && ld_w >= K, DCQ_ERR_ARGUMENT,
              "rows of codes must start at multiples of 16 bytes");
  DCQ_REQUIRE(ld_y >= N, DCQ_ERR_ARGUMENT, "rows of y overlap");
  const uintptr_t y_at = reinterpret_cast<uintptr_t>(y);
  const int32_t y_vector = y_at % 16 == 0 && ld_y % 8 == 0 ? 2 : y_at % (y_storage == DCQ_F32 ? 16 : 8) == 0 && ld_y % 4 == 0 ? 1 : 0;
  const ProductParams p{x, w, x_scales, w_scales, ld_x, ld_w, xs_row_stride, xs_col_stride, ws_row_stride, ws_col_stride,
                        bias, y, ld_y, M, N, K, bias_storage, y_storage, y_vector};
  hipStream_t s = static_cast<hipStream_t>(stream);
  return y_storage == DCQ_F32 ? launch_product<true>(p, s) : launch_product<false>(p, s);
}
