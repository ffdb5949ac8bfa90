// Keys and values of past tokens held as e4m3 codes, a power-of-two scale for each page (block of tokens) and head: the
// append that writes them and the attention that reads them (gfx950).
//
// A page holds P tokens (a multiple of 16) of every key / value head: keys [P][D], values transposed, [D][P], so that
// attention reads both as matrix-instruction operands straight from memory, without a transposition.  A table lists
// each sequence's pages; an entry outside the pool stands for no page: appends skip it, attention does not see its
// tokens.
#include "dcq_fp8.cuh"

#include <algorithm>
#include <cmath>

namespace dcq {

// One sequence's share of a launch whose tiles run over the sequences one after the other.
struct Place {
  int seq;      // -1: the tile lies behind the last sequence's
  int tile;     // the tile's number within the sequence
  int row0;     // the sequence's first row of a packed tensor
  int rows;     // its rows (new tokens, or queries)
  int length;   // its tokens in the cache, as the caller gave them, at most `capacity`
  int first, end;  // seq == -1: the rows that some sequence has lie in [first, end); `tile` counts from the last used one
};

// what lane `lane` holds, as a scalar (the same lane for the whole wave)
template <class T>
__device__ __forceinline__ T from_lane(T x, int lane) {
  return static_cast<T>(__builtin_amdgcn_readlane(static_cast<int>(x), lane));
}

// The sums over the lanes up to each, by shifts within rows of 16 lanes and broadcasts of the rows' last; sums beyond 32 bits
// stay at the largest number.
__device__ __forceinline__ uint32_t running_sums(uint32_t x) {
  auto add = [&](uint32_t y) { x = __builtin_elementwise_add_sat(x, y); };
  add(__builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false));  // from 1 lane before
  add(__builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false));  // 2
  add(__builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false));  // 4
  add(__builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false));  // 8
  add(__builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false));  // rows 1 and 3: the last lane of the row before
  add(__builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false));  // rows 2 and 3: lane 31
  return x;
}

// The sequence that tile `tile` belongs to, found by a wave: 64 sequences at a time, a lane each, with a running sum of
// their tile counts.  starts == nullptr: every sequence has `uniform` rows.  What the tables hold is not trusted: starts
// are cut to [0, total] and to ascending order, lengths to [0, capacity].
template <class Tiles>
__device__ __forceinline__ Place find_place(int tile, const int32_t* starts, int uniform, const int32_t* lengths, int count,
                                            int total, int capacity, Tiles tiles_of) {
  const int lane = threadIdx.x % kWave;
  uint32_t before = 0;  // never more than `tile`
  for (int base = 0; base < count; base += kWave) {
    const int s = base + lane;
    int row0 = 0, rows = 0, length = 0, tiles = 0;
    if (s < count) {
      if (starts != nullptr) {
        row0 = min(max(starts[s], 0), total);
        rows = max(min(starts[s + 1], total) - row0, 0);
      } else {
        row0 = s * uniform;
        rows = uniform;
      }
      length = min(max(lengths[s], 0), capacity);
      tiles = tiles_of(rows, length);
    }
    const uint32_t upto = __builtin_elementwise_add_sat(before, running_sums(tiles));
    const uint64_t hit = __ballot(static_cast<uint32_t>(tile) < upto);
    if (hit != 0) {
      const int at = __builtin_ctzll(hit);
      Place f;
      f.seq = base + at;
      f.tile = tile - static_cast<int>(at > 0 ? from_lane(upto, at - 1) : before);
      f.row0 = from_lane(row0, at);
      f.rows = from_lane(rows, at);
      f.length = from_lane(length, at);
      f.first = f.end = 0;
      return f;
    }
    before = from_lane(upto, kWave - 1);
  }
  const int first = starts != nullptr ? min(max(starts[0], 0), total) : 0;
  const int end = starts != nullptr ? min(max(starts[count], first), total) : total;
  return {-1, tile - static_cast<int>(before), 0, 0, 0, first, end};
}

// =============================================================================================
// Append.  A workgroup takes one page's new tokens of one head (of up to 4, if pages are small), keys and values: they are
// read once, into registers; then the largest finite magnitude, the scale, the older codes' move to it if it grew, the new
// codes.  The values are turned round in LDS.  Few tokens are bound by the chain of waits (tables, tokens, one exchange): 6.5 us
// for one token of each of 64 sequences, many by HBM behind that chain: 27 us for 16,300 tokens of 8 heads
// of 128, 3.7 TB/s.
//
// The scale is the smallest power of two that takes the magnitudes to 448 or less.  A floating-point code loses nothing
// by a power of two against max / 448 (its relative step is the same all over its normal range), and a page whose scale
// grows with a later token is rescaled by a power of two: exactly, but for values that sink below the normal range.
// A page only ever grows its scale while it fills; its first token sets it anew.
// =============================================================================================
struct AppendParams {
  const void* x[2];  // keys, values
  int64_t x_seq[2], x_token[2], x_head[2];
  uint8_t* codes[2];
  float* scales[2];
  const int32_t* table;
  const int32_t* lengths;
  const int32_t* starts;
  int32_t sequences, total, uniform, pool, heads, table_cols;
};

__device__ __forceinline__ int pages_touched(int rows, int length, int page, int capacity) {
  rows = min(rows, capacity - length);
  return rows <= 0 ? 0 : (length + rows - 1) / page - length / page + 1;
}

constexpr int heads_per_workgroup(int page) { return page == 16 ? 4 : page == 32 ? 2 : 1; }

// Waves per SIMD asked of the compiler: 8 where that spills nothing (16,300 float16 tokens 27.7 -> 26.9 us; bfloat16, with 2 spilled
// registers at 7 waves, 26.9 -> 29).
constexpr int append_waves(int storage, int page_elements) {
  return storage == DCQ_F16 && page_elements <= 64 * 128 ? 8 : 1;
}

// smallest power of two s >= 2^-126 with 448 s >= largest
__device__ __forceinline__ float power_scale(float largest) {
  const uint32_t u = __float_as_uint(largest);
  // 448 = 1.75 * 2^8: the exponent that takes the leading bit to 2^8, one more if the significand exceeds 1.75
  const int e = static_cast<int>(u >> 23) - 127 - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
  return __uint_as_float(static_cast<uint32_t>(max(e, -126) + 127) << 23);
}

__device__ __forceinline__ uint32_t rescale_codes(uint32_t w, float ratio) {
  typedef float pair __attribute__((ext_vector_type(2)));
  const pair a = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(w), false);
  const pair b = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(w), true);
  return to_e4m3x4(a[0] * ratio, a[1] * ratio, b[0] * ratio, b[1] * ratio);
}

template <int ST, int D, int P>
__global__ __launch_bounds__(256, append_waves(ST, D * P)) void append_kernel(const AppendParams p) {
  constexpr int kTeam = D / 8;                               // lanes of a token, 8 channels each
  constexpr int kTokens = 256 / kTeam;                       // tokens per pass
  constexpr int kPasses = (P + kTokens - 1) / kTokens;
  constexpr int kHeads = heads_per_workgroup(P);
  constexpr int kPitch = P + 4;                              // of the transposed tiles in LDS
  using S = Storage<ST>;
  using elem_t = typename S::elem_t;
  constexpr int kChunks = 8 / S::kVec;
  __shared__ float part[kHeads][2][4];
  __shared__ uint32_t tiles[kHeads][D * kPitch / 4];
  const int capacity = p.table_cols * P;
  const int groups = (p.heads + kHeads - 1) / kHeads, head0 = blockIdx.x % groups * kHeads, heads = min(kHeads, p.heads - head0);
  const Place f = find_place(blockIdx.x / groups, p.starts, p.uniform, p.lengths, p.sequences, p.total, capacity,
                             [&](int rows, int length) { return pages_touched(rows, length, P, capacity); });
  if (f.seq < 0) return;
  const int col = f.length / P + f.tile;
  const int page = p.table[static_cast<int64_t>(f.seq) * p.table_cols + col];
  if (page < 0 || page >= p.pool) return;
  const int begin = f.tile == 0 ? f.length - col * P : 0;            // first new slot of the page
  const int skip = col * P + begin - f.length;                       // new tokens on earlier pages
  const int n = min(P - begin, f.rows - skip);
  const int64_t unit0 = static_cast<int64_t>(page) * p.heads + head0;
  const int sub = threadIdx.x % kTeam, first = threadIdx.x / kTeam;

  float old[kHeads][2];
  Chunk<elem_t, S::kVec> x[kHeads][2][kPasses][kChunks];
#pragma unroll
  for (int h = 0; h < kHeads; ++h)  // (heads behind the last, tokens behind the last: that one again)
#pragma unroll
    for (int kind = 0; kind < 2; ++kind) {
      const int64_t row0 = p.starts != nullptr ? f.row0 * p.x_token[kind] : f.seq * p.x_seq[kind];
      const elem_t* from = static_cast<const elem_t*>(p.x[kind]) + row0 + skip * p.x_token[kind] + (head0 + min(h, heads - 1)) * p.x_head[kind] + sub * 8;
      old[h][kind] = p.scales[kind][unit0 + min(h, heads - 1)];
#pragma unroll
      for (int t = 0; t < kPasses; ++t)
#pragma unroll
        for (int c = 0; c < kChunks; ++c)
          x[h][kind][t][c] = load_chunk<elem_t, S::kVec>(from + min(first + t * kTokens, n - 1) * p.x_token[kind] + c * S::kVec);
    }
  auto value = [&](int h, int kind, int t, int i) { return S::load(x[h][kind][t][i / S::kVec].v[i % S::kVec]); };
#pragma unroll
  for (int h = 0; h < kHeads; ++h)
#pragma unroll
    for (int kind = 0; kind < 2; ++kind) {
      float m = 0.0f;
#pragma unroll
      for (int t = 0; t < kPasses; ++t)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float a = fabsf(value(h, kind, t, i));
          m = fmaxf(m, a < __builtin_inff() ? a : 0.0f);
        }
      m = team_max(m, kWave);
      if (threadIdx.x % kWave == 0) part[h][kind][threadIdx.x / kWave] = m;
    }
  __syncthreads();  // (also: every thread has read the old scales before one writes the new)
  if constexpr (ST == DCQ_BF16) {
    // (kept as they came: the compiler would convert them once and hold float32, twice the registers; 16,300 tokens 29.2 -> 27 us)
#pragma unroll
    for (int h = 0; h < kHeads; ++h)
#pragma unroll
      for (int kind = 0; kind < 2; ++kind)
#pragma unroll
        for (int t = 0; t < kPasses; ++t) {
          uint4 w = __builtin_bit_cast(uint4, x[h][kind][t][0]);
          asm volatile("" : "+v"(w.x), "+v"(w.y), "+v"(w.z), "+v"(w.w));
          x[h][kind][t][0] = __builtin_bit_cast(Chunk<elem_t, S::kVec>, w);
        }
  }
#pragma unroll
  for (int h = 0; h < kHeads; ++h) {
    if (h >= heads) break;
#pragma unroll
    for (int kind = 0; kind < 2; ++kind) {
      const int64_t unit = unit0 + h;
      uint8_t* codes = p.codes[kind] + unit * P * D;
      const float* m = part[h][kind];
      float scale = power_scale(fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3])));
      if (begin > 0) scale = fmaxf(scale, old[h][kind]);
      if (threadIdx.x == 0) p.scales[kind][unit] = scale;
      if (begin > 0 && scale != old[h][kind]) {
        const float ratio = old[h][kind] / scale;
        for (int i = threadIdx.x; i < P * D / 16; i += 256) {  // (slots behind the tokens too: nobody reads them)
          uint4* at = reinterpret_cast<uint4*>(codes) + i;
          const uint4 w = *at;
          *at = uint4{rescale_codes(w.x, ratio), rescale_codes(w.y, ratio), rescale_codes(w.z, ratio), rescale_codes(w.w, ratio)};
        }
        __syncthreads();  // the new codes overwrite some of these
      }
      const float inverse = 1.0f / scale;  // a power of two: exact
#pragma unroll
      for (int t = 0; t < kPasses; ++t) {
        const int token = first + t * kTokens;
        if (token >= n) break;
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = value(h, kind, t, i) * inverse;  // within +-448, or not finite: the NaN code
        const uint2 w = {to_e4m3x4(v[0], v[1], v[2], v[3]), to_e4m3x4(v[4], v[5], v[6], v[7])};
        if (kind == 0) {
          *reinterpret_cast<uint2*>(codes + (begin + token) * D + sub * 8) = w;
        } else {
          uint8_t* to = reinterpret_cast<uint8_t*>(tiles[h]) + sub * 8 * kPitch + begin + token;
#pragma unroll
          for (int i = 0; i < 8; ++i) to[i * kPitch] = static_cast<uint8_t>((i < 4 ? w.x : w.y) >> (8 * (i & 3)));
        }
      }
    }
  }
  __syncthreads();
  const int end = begin + n, c0 = begin / 16, per = (end + 15) / 16 - c0;
  for (int i = threadIdx.x; i < heads * D * per; i += 256) {
    const int row = i / per, c = c0 + i % per, h = row / D, d = row % D;
    const uint32_t* from = tiles[h] + (d * kPitch + c * 16) / 4;
    uint8_t* to = p.codes[1] + ((unit0 + h) * D + d) * P + c * 16;
    if (c * 16 >= begin && c * 16 + 16 <= end) {
      *reinterpret_cast<uint4*>(to) = uint4{from[0], from[1], from[2], from[3]};
    } else {
      const uint8_t* b = reinterpret_cast<const uint8_t*>(from);
      for (int k = max(begin - c * 16, 0); k < min(16, end - c * 16); ++k) to[k] = b[k];
    }
  }
}

// =============================================================================================
// Attention over the cache:  o = sum_t softmax_t(scale q . k_t) v_t over the tokens t that a query sees: those before
// `length`, and if causal before length - queries + i + 1 for query i.  A query that sees none gives 0.
//
// A wave keeps RT x 16 rows (queries x the heads that share a key / value head) and passes over the tokens 64 at a time
// with a running maximum and sum.  It computes transposed scores S' = K Q' and outputs O' = V' P', so that one lane
// holds tokens of one row throughout: the maximum and the sum take two lane exchanges, and P' leaves the exponentials
// in the very registers where the second product wants it.  What makes that fit is the choice of which token a lane
// loads: of a tile of 64, lane group g's tokens are 16 g .. 16 g + 15, tile t's instruction row 4 g + i being token
// 16 g + 4 t + i.  A lane's values are then 16 consecutive bytes of a row of the transposed page, and pages of 16
// tokens need no other path; a lane's 16 scores share one page, hence one scale.
//
// Codes become 16-bit operands exactly (4 significant bits).  The keys' scale goes into the exponent's multiply-add in
// float32.  The values' scale goes into their conversion, as far as it is a power of two; what is left of it, a factor from 1 to
// 2 (1 for the scales that appends make), goes into the probabilities as its logarithm, and out of their sum again.
// Probabilities are rounded to the type of the query: bfloat16 (2^-8 of each at most, uncorrelated; the outputs' rounding is
// as large), or float16 (2^-11), whose range holds neither every value * scale nor every probability.  Values are taken relative to
// the wave's first scale, and a step whose scales lie too far from it falls back to bfloat16.  Probabilities are held 2^LIFT times as
// large, as are the sums they are divided by, so that they lose bits from 2^-(14 + LIFT) of the row's largest on and not from
// 2^-14: one token far ahead whose value is small leaves the row to the others.  Steps whose probabilities all lie below
// 2^-(17 + LIFT), where float16 keeps fewer bits than bfloat16, fall back as well (of chunks the steps behind the first such one, by
// leaving the loop without masks: both types in that loop took 371 us instead of 353 for the chunks below).  Sums are float32.
// Where SLACK is not 0 the running maximum follows a row's largest score only when that is more than 2^SLACK ahead: float32 sums
// have room for it, and most steps spare the rescaling (float16 chunks with SLACK 8: 351 us, 6: 353, 4: 357; 6 leaves LIFT 8).
// Where it is 0 the largest probability is exactly 2^LIFT, which helps rows that attend to few tokens.
// =============================================================================================
struct AttendParams {
  const void* q;
  void* out;
  int64_t q_seq, q_token, q_head, o_seq, o_token, o_head;
  const uint8_t* k;
  const uint8_t* v;
  const float* ks;
  const float* vs;
  const int32_t* table;
  const int32_t* lengths;
  const int32_t* starts;
  float* partial;  // splits > 1: per (tile, split, head) the rows' sums [16][D], then maxima and sums [2][16]
  int32_t sequences, total, uniform, pool, heads, group, page, page_shift, table_cols, causal, zero_rest, splits, tiles;
  float scale_log2;  // >= 0
  uint32_t q_flip;   // sign bits to flip in a pair of query values: a negative scale
};

// how many tokens query `i` of a sequence sees
__device__ __forceinline__ int tokens_seen(const AttendParams& p, const Place& f, int i) {
  const int before = p.causal ? max(f.length - f.rows + i + 1, 0) : f.length;
  return min(before, p.table_cols * p.page);
}

__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
  const bf16x2 t = {static_cast<__bf16>(a), static_cast<__bf16>(b)};
  return __builtin_bit_cast(uint32_t, t);
}
__device__ __forceinline__ uint32_t pack_f16(float a, float b) {
  const f16x2 t = {static_cast<_Float16>(a), static_cast<_Float16>(b)};
  return __builtin_bit_cast(uint32_t, t);
}
template <int ST>
__device__ __forceinline__ uint32_t pack_16(float a, float b) {
  return ST == DCQ_F16 ? pack_f16(a, b) : pack_bf16(a, b);
}

// 0x80 in every byte of w that is an e4m3 NaN (0x7f or 0xff)
__device__ __forceinline__ uint32_t nan_codes(uint32_t w) { return ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; }

// the largest of the four lanes r, r + 16, r + 32 and r + 48, by exchanges of registers
__device__ __forceinline__ float groups_max(float x) {
  typedef uint32_t pair __attribute__((ext_vector_type(2)));
  uint32_t w = __float_as_uint(x);
  pair p = __builtin_bit_cast(pair, __builtin_amdgcn_permlane16_swap(w, w, false, false));
  w = __float_as_uint(fmaxf(__uint_as_float(p[0]), __uint_as_float(p[1])));
  p = __builtin_bit_cast(pair, __builtin_amdgcn_permlane32_swap(w, w, false, false));
  return fmaxf(__uint_as_float(p[0]), __uint_as_float(p[1]));
}

// A wave's rows and what it has summed up for them.
template <int ST, int D, int RT, int SLACK>
struct Rows {
  static constexpr int kKeyLoads = D / 64, kDims = D / 16;
  // 2^(LIFT + SLACK) times a factor below 2 is the largest that a probability is held as; float16 ends at 65504
  static constexpr int kLift = ST == DCQ_F16 ? 14 - SLACK : 0;
  static __device__ __forceinline__ float power_of(float scale) { return __uint_as_float(__float_as_uint(scale) & 0x7f800000u); }
  uint4 q[RT][2 * kKeyLoads];
  f32x4 acc[RT][kDims];  // in units of `unit`
  float m[RT], l[RT];    // l: this lane's tokens only
  f32x4 sums[RT];        // what steps without masks add to l (SLACK > 0): all four the row's whole sum
  int limit[RT];         // tokens that the row sees
  bool seen[RT];
  int most, least;       // over the wave's rows
  float per_unit;        // 1 / unit, a power of two
  bool behind;           // SLACK > 0: the last step without masks should have fallen back to bfloat16

  // rows row_base .. row_base + 16 RT - 1 of the place's (query, head in group) pairs
  __device__ __forceinline__ void load(const AttendParams& p, const Place& f, int head, int row_base) {
    const int r = threadIdx.x % 16, g = threadIdx.x % kWave / 16;
    const int64_t base = p.starts != nullptr ? f.row0 * p.q_token : f.seq * p.q_seq;
    most = 0;
    least = 0x7fffffff;
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      const int last = f.rows * p.group - 1, row = min(row_base + t * 16 + r, last);  // (rows that are none: the last one again)
      const bool in = row_base + t * 16 + r <= last;
      const int qi = row / p.group, h = row % p.group;
      limit[t] = in ? tokens_seen(p, f, qi) : -1;
      if (in) {
        most = max(most, limit[t]);
        least = min(least, limit[t]);
      }
      const uint16_t* at = static_cast<const uint16_t*>(p.q) + base + qi * p.q_token + static_cast<int64_t>(head * p.group + h) * p.q_head;
#pragma unroll
      for (int j = 0; j < 2 * kKeyLoads; ++j) {
        const uint4 w = *reinterpret_cast<const uint4*>(at + j / 2 * 64 + g * 16 + j % 2 * 8);
        q[t][j] = uint4{w.x ^ p.q_flip, w.y ^ p.q_flip, w.z ^ p.q_flip, w.w ^ p.q_flip};
      }
      m[t] = -__builtin_inff();
      l[t] = 0.0f;
      sums[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
      seen[t] = false;
#pragma unroll
      for (int d = 0; d < kDims; ++d) acc[t][d] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }
#pragma unroll
    for (int off = 1; off < 16; off <<= 1) {
      most = max(most, __shfl_xor(most, off, kWave));
      least = min(least, __shfl_xor(least, off, kWave));
    }
    most = __builtin_amdgcn_readfirstlane(most);
    least = __builtin_amdgcn_readfirstlane(least);
#pragma unroll
    for (int t = 0; t < RT; ++t)
      if (limit[t] < 0) limit[t] = most;  // rows that are none: whatever spares the mask
    per_unit = 1.0f;
    behind = false;
  }

  // Values are taken relative to the largest scale of the first step's lane groups (float16 only), of those whose first token `own`
  // some row sees: the scale of a page listed ahead may be anything.
  __device__ __forceinline__ void set_unit(float value_scale, bool own_ok, int own) {
    if (ST != DCQ_F16) return;
    float u = own_ok && own < most ? power_of(value_scale) : 0.0f;
    u = fmaxf(u, __shfl_xor(u, 16, kWave));
    u = fmaxf(u, __shfl_xor(u, 32, kWave));
    per_unit = u >= 0x1p-120f && u <= 0x1p120f ? 1.0f / u : 1.0f;
  }
  // whether float16 holds the codes times this scale exactly
  __device__ __forceinline__ bool fits(float value_scale) const {
    return ST != DCQ_F16 || (value_scale * per_unit >= 0x1p-15f && value_scale * per_unit < 0x1p8f);
  }

  // Memory behind the last visible token may hold anything, NaN codes too, which a probability of 0 does not silence:
  // those bytes become 0 (`count` of the lane's 16 tokens are visible to some row).  A token whose value is NaN may be
  // seen by some rows and not by others: a product of "is NaN" and "is seen" tells which outputs become NaN, and the code
  // becomes 0 too.
  __device__ __forceinline__ uint4 visible_values(uint4 v, int d, int own, int count) {
    uint32_t* w = reinterpret_cast<uint32_t*>(&v);
    uint32_t flag[4], bad = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      w[k] &= bytes_before(count, k);
      flag[k] = nan_codes(w[k]) >> 7;  // 1 per NaN byte
      bad |= flag[k];
    }
    if (__any(bad != 0)) {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        w[k] &= ~(flag[k] * 0xffu);
        flag[k] *= 0x38u;  // the code of 1
      }
#pragma unroll
      for (int i = 0; i < RT; ++i) {
        f32x4 hits = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          float see[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) see[e] = own + 8 * u + e < limit[i] ? 1.0f : 0.0f;
          const uint4 b = {pack_bf16(see[0], see[1]), pack_bf16(see[2], see[3]), pack_bf16(see[4], see[5]), pack_bf16(see[6], see[7])};
          hits = Half<DCQ_BF16>::mfma(codes8<DCQ_BF16>(flag[2 * u], flag[2 * u + 1], 1.0f), b, hits);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (hits[e] > 0.0f) acc[i][d][e] = __builtin_nanf("");
      }
    }
    return v;
  }

  // 64 tokens.  MASKED = false: every row sees all of them, and their scales fit (SLACK > 0: and are powers of two).  own: the lane
  // group's first token, own_ok: whether it has a page, key_scale (with the softmax scale and log2 e) and value_scale that page's;
  // query(i, j), key(t, j) and value(d): the lane's 16 bytes of row tile i, of key tile t and of value rows d; keys_read() is
  // called when no key is wanted any more.
  template <bool MASKED, class Query, class Key, class Value, class Then>
  __device__ __forceinline__ void step(int own, bool own_ok, float key_scale, float value_scale, Query query, Key key, Value value,
                                       Then keys_read) {
    f32x4 s[RT][4];
    uint4 ahead = key(0, 0);  // (each read one piece ahead of its use)
#pragma unroll
    for (int j = 0; j < kKeyLoads; ++j) {
      uint4 ql[RT], qh[RT];
#pragma unroll
      for (int i = 0; i < RT; ++i) {
        ql[i] = query(i, 2 * j);
        qh[i] = query(i, 2 * j + 1);
      }
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const uint4 c = ahead;
        if (4 * j + t + 1 < 4 * kKeyLoads) ahead = key((t + 1) % 4, j + (t + 1) / 4);
        const uint4 lo = codes8<ST>(c.x, c.y, 1.0f), hi = codes8<ST>(c.z, c.w, 1.0f);
#pragma unroll
        for (int i = 0; i < RT; ++i) {
          if (j == 0) s[i][t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
          s[i][t] = Half<ST>::mfma(lo, ql[i], s[i][t]);
        }
#pragma unroll
        for (int i = 0; i < RT; ++i) s[i][t] = Half<ST>::mfma(hi, qh[i], s[i][t]);
        __builtin_amdgcn_sched_barrier(0);  // (left alone, the scheduler converts everything first, and runs out of registers)
      }
    }
    keys_read();
    const float factor = __uint_as_float((__float_as_uint(value_scale) & 0x7fffffu) | 0x3f800000u);
    const float log_factor = __builtin_amdgcn_logf(factor), inverse_factor = __builtin_amdgcn_rcpf(factor);  // (of 1: exactly 0 and 1)
    constexpr bool kByProduct = !MASKED && SLACK > 0;
    float x[RT][16], top[RT];
    bool grows = false;
#pragma unroll
    for (int i = 0; i < RT; ++i) {
      top[i] = -__builtin_inff();
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        x[i][e] = s[i][e / 4][e % 4];
        if (MASKED) x[i][e] = own + e < limit[i] && own_ok ? x[i][e] * key_scale : -__builtin_inff();
        top[i] = fmaxf(top[i], x[i][e]);
      }
      if (!MASKED) top[i] *= key_scale;
      seen[i] = seen[i] || !MASKED || (own < limit[i] && own_ok);
      top[i] = groups_max(top[i]);
      grows = grows || top[i] > m[i] + SLACK;
    }
    if (__any(grows)) {
#pragma unroll
      for (int i = 0; i < RT; ++i) {
        const float now = fmaxf(m[i], top[i]), base = now == -__builtin_inff() ? 0.0f : now;
        const float fade = __builtin_amdgcn_exp2f(m[i] - base);
        m[i] = now;
        l[i] *= fade;
        if (SLACK > 0) sums[i] *= fade;
#pragma unroll
        for (int d = 0; d < kDims; ++d)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[i][d][e] *= fade;
      }
    }
    bool near = false;  // (a row that sees none of these tokens has no say)
#pragma unroll
    for (int i = 0; i < RT; ++i) {
      near = near || top[i] >= fmaxf(m[i] - (17 + kLift), -3.4e38f);
      const float base = (m[i] == -__builtin_inff() ? 0.0f : m[i]) - (kByProduct ? 0.0f : log_factor) - kLift;
      float sum = 0.0f;
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        x[i][e] = __builtin_amdgcn_exp2f(MASKED ? x[i][e] - base : __builtin_fmaf(x[i][e], key_scale, -base));
        sum += x[i][e];
      }
      if (!kByProduct) l[i] = __builtin_fmaf(sum, inverse_factor, l[i]);
    }
    const float relative = ST == DCQ_F16 ? power_of(value_scale) * per_unit : power_of(value_scale);
    if constexpr (!MASKED) {
      if constexpr (ST == DCQ_F16 && SLACK == 0) {
        if (__any(near))
          add_values<DCQ_F16, false>(x, own, 16, relative, value);
        else
          add_values<DCQ_BF16, false>(x, own, 16, relative, value);
      } else {
        add_values<ST, false>(x, own, 16, relative, value);
        if (ST == DCQ_F16) behind = !__any(near);
      }
    } else {
      const int count = own_ok ? min(max(most - own, 0), 16) : 0;
      if (ST == DCQ_F16 && __any(near) && __all(fits(value_scale) || count == 0))
        add_values<DCQ_F16, true>(x, own, count, relative, value);
      else
        add_values<DCQ_BF16, true>(x, own, count, relative, value);
    }
  }

  template <int VT, bool MASKED, class Value>
  __device__ __forceinline__ void add_values(const float (&x)[RT][16], int own, int count, float relative, Value value) {
    uint4 pr[RT][2];
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
      for (int u = 0; u < 2; ++u)
        pr[i][u] = {pack_16<VT>(x[i][8 * u], x[i][8 * u + 1]), pack_16<VT>(x[i][8 * u + 2], x[i][8 * u + 3]), pack_16<VT>(x[i][8 * u + 4], x[i][8 * u + 5]),
                    pack_16<VT>(x[i][8 * u + 6], x[i][8 * u + 7])};
    if (!MASKED && SLACK > 0) {  // (scales are powers of two here: there is no factor to take out again)
      const uint32_t one = VT == DCQ_F16 ? 0x3c003c00u : 0x3f803f80u;
#pragma unroll
      for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int u = 0; u < 2; ++u) sums[i] = Half<VT>::mfma(uint4{one, one, one, one}, pr[i][u], sums[i]);
    }
    if (MASKED && count == 0) relative = 1.0f;  // (nothing of this page is seen, and its scale may be anything)
    uint4 ahead = value(0);
#pragma unroll
    for (int d = 0; d < kDims; ++d) {
      uint4 c = ahead;
      if (d + 1 < kDims) ahead = value(d + 1);
      if (MASKED) c = visible_values(c, d, own, count);
      const uint4 lo = codes8<VT>(c.x, c.y, relative), hi = codes8<VT>(c.z, c.w, relative);
#pragma unroll
      for (int i = 0; i < RT; ++i) {
        acc[i][d] = Half<VT>::mfma(lo, pr[i][0], acc[i][d]);
        acc[i][d] = Half<VT>::mfma(hi, pr[i][1], acc[i][d]);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  }

  // the rows' sums over the lane groups; a row that saw only scores of -inf is NaN (0 / 0), one that saw nothing is 0
  __device__ __forceinline__ void finish() {
#pragma unroll
    for (int i = 0; i < RT; ++i) {
      if (seen[i] && m[i] == -__builtin_inff()) l[i] = __builtin_nanf("");
      l[i] += __shfl_xor(l[i], 16, kWave);
      l[i] += __shfl_xor(l[i], 32, kWave);
      if (SLACK > 0) l[i] += sums[i][0];
      if (ST == DCQ_F16) {
#pragma unroll
        for (int d = 0; d < kDims; ++d) acc[i][d] *= 1.0f / per_unit;
      }
    }
  }

  __device__ __forceinline__ void store(const AttendParams& p, const Place& f, int head, int row, int i) const {
    const int g = threadIdx.x % kWave / 16;
    const int qi = row / p.group, h = row % p.group;
    const int64_t base = p.starts != nullptr ? f.row0 * p.o_token : f.seq * p.o_seq;
    uint16_t* at = static_cast<uint16_t*>(p.out) + base + qi * p.o_token + static_cast<int64_t>(head * p.group + h) * p.o_head;
    const float inverse = l[i] == 0.0f ? 0.0f : 1.0f / l[i];
#pragma unroll
    for (int d = 0; d < kDims; ++d) {
      const uint2 w = {pack_16<ST>(acc[i][d][0] * inverse, acc[i][d][1] * inverse), pack_16<ST>(acc[i][d][2] * inverse, acc[i][d][3] * inverse)};
      *reinterpret_cast<uint2*>(at + d * 16 + g * 4) = w;
    }
  }
};

// A sequence's pages as the kernels walk them.
struct Pages {
  const int32_t* table;
  int cols, shift, mask, pool;
  __device__ __forceinline__ Pages(const AttendParams& p, const Place& f)
      : table(p.table + static_cast<int64_t>(f.seq) * p.table_cols), cols(p.table_cols), shift(p.page_shift), mask(p.page - 1), pool(p.pool) {}
  // the page of a token, -1 if it has none
  __device__ __forceinline__ int of(int token) const {
    const int c = token >> shift;
    const int id = c < cols ? table[c] : -1;
    return id < pool ? id : -1;
  }
};

// The rows of a packed output that no sequence has, set to 0 by the tiles behind the last sequence's (at least one).
template <int D>
__device__ __forceinline__ void zero_rows(const AttendParams& p, const Place& f, int tile, int head) {
  const int used = tile - f.tile;
  const int stride = p.tiles - used, rest = f.first + p.total - f.end;
  for (int u = f.tile; u < rest; u += stride) {
    const int64_t row = u < f.first ? u : u - f.first + f.end;
    for (int i = threadIdx.x; i < p.group * (D / 4); i += 256) {
      uint16_t* at = static_cast<uint16_t*>(p.out) + row * p.o_token + static_cast<int64_t>(head * p.group + i / (D / 4)) * p.o_head;
      store_chunk<uint16_t, 4>(at + i % (D / 4) * 4, Chunk<uint16_t, 4>{});
    }
  }
}

template <int TILE_ROWS>
__device__ __forceinline__ Place place_of(const AttendParams& p, int tile) {
  return find_place(tile, p.starts, p.uniform, p.lengths, p.sequences, p.total, 0x7fffffff,
                    [&](int rows, int) { return static_cast<int>((static_cast<int64_t>(rows) * p.group + TILE_ROWS - 1) / TILE_ROWS); });
}

// Single tokens: bound by the cache's bytes.  The four waves of a workgroup share out the tokens of 16 rows, each with its own
// running sums, and with loads under way at all times; their results are joined at the end, and those of several
// workgroups (splits) by join_kernel.
template <int ST, int D>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2))) void attend_tokens_kernel(const AttendParams p) {
  constexpr int kWaves = 4, kKeyLoads = D / 64, kDims = D / 16;
  const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int r = lane % 16, g = lane / 16;
  // heads side by side, so that with 8 of them each XCD keeps to one
  const int head = blockIdx.x % p.heads, split = blockIdx.x / p.heads % p.splits, tile = blockIdx.x / p.heads / p.splits;
  const Place f = place_of<16>(p, tile);
  if (f.seq < 0) {
    if (p.zero_rest && split == 0) zero_rows<D>(p, f, tile, head);
    return;
  }
  const int row_base = f.tile * 16;
  Rows<ST, D, 1, 0> rows;
  rows.load(p, f, head, row_base);
  const int steps = (rows.most + 63) / 64, share = (steps + p.splits - 1) / p.splits;
  const int first = split * share + wave, end = min((split + 1) * share, steps);

  const Pages pages(p, f);
  // keys (and both scales) of the next step are loaded when the present ones have been read, values at the beginning of their own step
  uint4 keys[4][kKeyLoads], values[kDims];
  struct Ids {
    int own, key;
  };
  auto ids_of = [&](int step) { return Ids{pages.of(step * 64 + 16 * g), pages.of(step * 64 + 16 * (r / 4) + (r & 3))}; };
  float ks = 0.0f, vs = 0.0f;
  auto load_keys = [&](int step, Ids id) {
    const int token = step * 64 + 16 * (r / 4) + (r & 3);
    const int64_t unit = static_cast<int64_t>(max(id.key, 0)) * p.heads + head, own_unit = static_cast<int64_t>(max(id.own, 0)) * p.heads + head;
    ks = p.ks[own_unit];
    vs = p.vs[own_unit];
    const uint8_t* at = p.k + (unit * p.page + (token & pages.mask)) * D + g * 16;
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int j = 0; j < kKeyLoads; ++j) keys[t][j] = *reinterpret_cast<const uint4*>(at + t * 4 * D + j * 64);
  };
  if (first < end) {
    Ids now = ids_of(first), next = ids_of(first + kWaves);
    load_keys(first, now);
    rows.set_unit(vs, now.own >= 0, first * 64 + 16 * g);
    int step = first;
    auto work = [&](auto masked) {
      const int own = step * 64 + 16 * g;
      const bool ok = now.own >= 0;
      const int64_t unit = static_cast<int64_t>(max(now.own, 0)) * p.heads + head;
      const float key_scale = ks * p.scale_log2, value_scale = vs;
      const uint8_t* at = p.v + (unit * D + r) * p.page + (own & pages.mask);
#pragma unroll
      for (int d = 0; d < kDims; ++d) values[d] = *reinterpret_cast<const uint4*>(at + d * 16 * p.page);
      now = next;
      rows.template step<decltype(masked)::value>(
          own, ok, key_scale, value_scale, [&](int, int j) { return rows.q[0][j]; }, [&](int t, int j) { return keys[t][j]; },
          [&](int d) { return values[d]; },
          [&] {
            load_keys(min(step + kWaves, end - 1), next);  // (at the end a step again that is not worked on)
            next = ids_of(step + 2 * kWaves);
          });
      step += kWaves;
    };
    // first the steps that every row sees whole, then, with masks, whatever is left: a loop of its own keeps the registers that
    // the masks take out of the other
    while (step < end && step * 64 + 64 <= rows.least && __all(now.own >= 0 && rows.fits(vs))) work(std::false_type{});
    while (step < end) work(std::true_type{});
  }
  rows.finish();

  __shared__ float part_m[kWaves][16], part_l[kWaves][16];
  __shared__ f32x4 part_o[kWaves - 1][kDims][kWave];
  if (g == 0) {
    part_m[wave][r] = rows.m[0];
    part_l[wave][r] = rows.l[0];
  }
  __syncthreads();
  float top = part_m[0][r];
#pragma unroll
  for (int w = 1; w < kWaves; ++w) top = fmaxf(top, part_m[w][r]);
  const float base = top == -__builtin_inff() ? 0.0f : top;
  const float fade = __builtin_amdgcn_exp2f(rows.m[0] - base);
#pragma unroll
  for (int d = 0; d < kDims; ++d) rows.acc[0][d] *= fade;
  if (wave > 0) {
#pragma unroll
    for (int d = 0; d < kDims; ++d) part_o[wave - 1][d][lane] = rows.acc[0][d];
  }
  __syncthreads();
  if (wave > 0) return;
  rows.l[0] = 0.0f;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) rows.l[0] += part_l[w][r] * __builtin_amdgcn_exp2f(part_m[w][r] - base);
#pragma unroll
  for (int w = 0; w < kWaves - 1; ++w)
#pragma unroll
    for (int d = 0; d < kDims; ++d) rows.acc[0][d] += part_o[w][d][lane];
  const int row = row_base + r;
  if (row >= f.rows * p.group) return;
  if (p.splits == 1) {
    rows.store(p, f, head, row, 0);
    return;
  }
  float* at = p.partial + static_cast<int64_t>(blockIdx.x) * (16 * (D + 2));
#pragma unroll
  for (int d = 0; d < kDims; ++d) *reinterpret_cast<f32x4*>(at + r * D + d * 16 + g * 4) = rows.acc[0][d];
  if (g == 0) {
    at[16 * D + r] = top;
    at[16 * (D + 1) + r] = rows.l[0];
  }
}

// Joins the splits of a row: one wave per row and head.
template <int ST, int D>
__global__ __launch_bounds__(256) void join_kernel(const AttendParams p) {
  const int lane = threadIdx.x % kWave;
  const int head = blockIdx.x % p.heads, tile = blockIdx.x / p.heads;
  const Place f = place_of<16>(p, tile);
  if (f.seq < 0) return;
  const int64_t unit = int64_t{16} * (D + 2), stride = unit * p.heads;
  const float* at = p.partial + (static_cast<int64_t>(tile) * p.splits * p.heads + head) * unit;
  for (int local = threadIdx.x / kWave; local < 16; local += 4) {
    const int row = f.tile * 16 + local;
    if (row >= f.rows * p.group) return;
    // (at most 64 splits: a lane each)
    float m = -__builtin_inff(), l = 0.0f;
    if (lane < p.splits) {
      m = at[lane * stride + 16 * D + local];
      l = at[lane * stride + 16 * (D + 1) + local];
    }
    const float top = team_max(m, kWave), base = top == -__builtin_inff() ? 0.0f : top;
    const float weight = __builtin_amdgcn_exp2f(m - base);
    l *= weight;
#pragma unroll
    for (int off = 1; off < kWave; off <<= 1) l += __shfl_xor(l, off, kWave);
    float o[D / kWave];
#pragma unroll
    for (int d = 0; d < D / kWave; ++d) o[d] = 0.0f;
    for (int s = 0; s < p.splits; ++s) {
      const float w = __shfl(weight, s, kWave);
      const float* from = at + s * stride + local * D + lane * (D / kWave);
#pragma unroll
      for (int d = 0; d < D / kWave; ++d) o[d] += w * from[d];
    }
    const int qi = row / p.group, h = row % p.group;
    const int64_t out_base = p.starts != nullptr ? f.row0 * p.o_token : f.seq * p.o_seq;
    uint16_t* to = static_cast<uint16_t*>(p.out) + out_base + qi * p.o_token + static_cast<int64_t>(head * p.group + h) * p.o_head;
    const float inverse = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
    for (int d = 0; d < D / kWave; ++d) to[lane * (D / kWave) + d] = Storage<ST>::store(o[d] * inverse);
  }
}

// Chunks of many queries.  Four waves take 32 rows each; the 64 tokens that all of them work on go from the pages to LDS directly,
// one step ahead, the keys' rows as 8 pieces of 16 bytes and the values' rows as 4, each at a position exchanged by bits of
// the row, so that the 16 rows of an operand take all 64 banks.  The tiles begin from the batch's last one on, each
// sequence's last and longest first.  (Sorted by their tokens, found by each workgroup anew: 8 sequences with 0 to 7000 older tokens,
// the longest listed first, 415 -> 364 us, but 350 -> 360 for the case below and 56 -> 59 us for a small one: the caller's order stays.)
// 4 chunks of up to 2048 queries on up to 4096 tokens, 32 heads on 8 of 128: 353 us in float16, 346 in bfloat16, 0.74 PFLOP/s.
// A wave's step has 64 matrix instructions (1024 cycles), and beside them 128 conversions, 32 exponentials and 120 others (about
// 1500).  Counters show the vector pipe busy 56 % of the time and the matrix pipe 31 %: neither binds, but they hardly overlap.  A
// workgroup's four waves convert, multiply and exponentiate in step (one barrier per 64 tokens, two buffers), a wave's two products
// and the softmax between them wait for each other, and only 1.7 waves per SIMD fill the gaps (2 fit, the last tiles leave some
// alone).  64 rows per wave share a conversion among twice the rows, but leave one wave per SIMD: 546 us.  Codes
// converted once per workgroup would be read from LDS at twice the bytes, which then bounds it.  Sums by the matrix pipe (a
// row of ones against the rounded probabilities) instead of 32 additions, with addresses and the loop's counts in scalar
// registers: 365 us before, 350 with.  A higher wave priority for the products: 348.
template <int ST, int D>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2))) void attend_chunks_kernel(const AttendParams p) {
  constexpr int RT = 2, kRows = 16 * RT, kTileRows = 4 * kRows, kHalf = 64 * D;
  constexpr int kLoads = kHalf / (256 * 16);  // pieces per thread, of keys and of values
  constexpr int kKeyPieces = D / 16;
  __shared__ __align__(1024) unsigned char lds[2][2][kHalf];  // [buffer][keys, values]
  __shared__ uint4 queries[4][RT][D / 32][kWave];             // operands that every step wants again, out of the registers' way
  const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int r = lane % 16, g = lane / 16;
  const int head = blockIdx.x % p.heads, tile = p.tiles - 1 - static_cast<int>(blockIdx.x) / p.heads;
  const Place f = place_of<kTileRows>(p, tile);
  if (f.seq < 0) {
    if (p.zero_rest) zero_rows<D>(p, f, tile, head);
    return;
  }
  const int row_base = f.tile * kTileRows + wave * kRows;
  Rows<ST, D, RT, ST == DCQ_F16 ? 6 : 8> rows;
  rows.load(p, f, head, row_base);
#pragma unroll
  for (int i = 0; i < RT; ++i)
#pragma unroll
    for (int j = 0; j < D / 32; ++j) queries[wave][i][j][lane] = rows.q[i][j];  // (a lane reads what it wrote)
  // the workgroup's tokens: those of its last row
  const int row_last = min((f.tile + 1) * kTileRows, f.rows * p.group) - 1;
  const int most = tokens_seen(p, f, row_last / p.group);
  const int steps = (most + 63) / 64;
  const int least = tokens_seen(p, f, f.tile * kTileRows / p.group);  // and of its first

  const Pages pages(p, f);
  auto key_swizzle = [](int row) { return (row >> 1 & 1) | (row >> 4 & 3) << 1; };  // the 16 rows of a tile: 4 from each 16
  // this thread's pieces: row and piece of the keys, row and piece of the values; their places in a page, to which a step adds
  // half a page if pages hold two steps
  constexpr int kKeyRows = 256 / kKeyPieces;  // rows per load of the workgroup
  const int key_row = threadIdx.x / kKeyPieces, key_piece = threadIdx.x % kKeyPieces;
  const int value_row = threadIdx.x / 4, value_piece = (threadIdx.x % 4) ^ (value_row >> 2 & 3);
  uint32_t key_at[kLoads];
#pragma unroll
  for (int i = 0; i < kLoads; ++i) {
    const int row = key_row + i * kKeyRows;
    key_at[i] = (row & pages.mask) * D + (key_piece ^ (key_swizzle(row) & (kKeyPieces - 1))) * 16;
  }
  const uint32_t value_at = value_row * p.page + (value_piece * 16 & pages.mask);
  // (a page of all heads has less than 2^31 bytes, the pool any number: one product of 32 bits with 32 per address)
  const uint32_t page_bytes = static_cast<uint32_t>(p.heads) * p.page * D;
  const uint8_t* const head_k = p.k + static_cast<int64_t>(head) * p.page * D;
  const uint8_t* const head_v = p.v + static_cast<int64_t>(head) * p.page * D;
  auto start_of = [](int id, uint32_t stride) { return static_cast<uint64_t>(static_cast<uint32_t>(max(id, 0))) * stride; };
  struct Ids {
    int key[kLoads], value, own;
  };
  auto ids_of = [&](int step) {
    Ids id;
#pragma unroll
    for (int i = 0; i < kLoads; ++i) id.key[i] = pages.of(step * 64 + key_row + i * kKeyRows);
    id.value = pages.of(step * 64 + value_piece * 16);
    id.own = pages.of(step * 64 + 16 * g);
    return id;
  };
  float ks, vs;
  bool ok;
  auto fetch = [&](int step, const Ids& id) {
    const uint64_t own_at = start_of(id.own, p.heads) + head;
    ks = p.ks[own_at];
    vs = p.vs[own_at];
    ok = id.own >= 0;
    const int half = step * 64 & pages.mask;
    unsigned char* to = &lds[step & 1][0][0];
#pragma unroll
    for (int i = 0; i < kLoads; ++i)
      load_to_lds_16(head_k + half * D + start_of(id.key[i], page_bytes) + key_at[i], to + (i * 256 + wave * kWave) * 16);
    const uint8_t* vp = head_v + half + start_of(id.value, page_bytes) + value_at;
#pragma unroll
    for (int i = 0; i < kLoads; ++i) load_to_lds_16(vp + i * 64 * p.page, to + kHalf + (i * 256 + wave * kWave) * 16);
  };
  if (steps > 0) {
    fetch(0, ids_of(0));
    Ids next = ids_of(1);
    int step = 0;
    auto work = [&](auto masked) {
      wait_direct_loads();
      const float key_scale = ks * p.scale_log2;
      float value_scale = vs;
      const bool own_ok = ok;
      asm volatile("" : "+v"(value_scale));
      __syncthreads();  // the step's tokens have landed, and everyone is done with the other buffer
      if (step + 1 < steps) {
        fetch(step + 1, next);
        next = ids_of(step + 2);
      }
      const int t0 = step * 64;
      const unsigned char* keys = lds[step & 1][0];
      const unsigned char* values = lds[step & 1][1];
      ++step;
      if (decltype(masked)::value && t0 >= rows.most) return;
      rows.template step<decltype(masked)::value>(
          t0 + 16 * g, own_ok, key_scale, value_scale, [&](int i, int j) { return queries[wave][i][j][lane]; },
          [&](int t, int j) {
            const int row = 16 * (r / 4) + 4 * t + (r & 3), at = (4 * j + g) ^ (key_swizzle(row) & (kKeyPieces - 1));
            return *reinterpret_cast<const uint4*>(keys + row * D + at * 16);
          },
          [&](int d) { return *reinterpret_cast<const uint4*>(values + (d * 16 + r) * 64 + (g ^ (r >> 2)) * 16); }, [] {});
    };
    // first the steps that every row of the workgroup sees whole, then, with masks, whatever is left: a loop of its own keeps
    // the registers that the masks take out of the other (a spilled one costs twice here: its reload waits for the loads
    // under way)
    rows.set_unit(vs, ok, 16 * g);
    while (step < steps && step * 64 + 64 <= least && !rows.behind && __all(ok && rows.fits(vs) && (__float_as_uint(vs) & 0x7fffff) == 0)) work(std::false_type{});
    while (step < steps) work(std::true_type{});
  }
  rows.finish();
#pragma unroll
  for (int i = 0; i < RT; ++i) {
    const int row = row_base + i * 16 + r;
    if (row < f.rows * p.group) rows.store(p, f, head, row, i);
  }
}

// How a launch covers its rows.  Few rows per sequence (single tokens): a workgroup's waves share out the tokens of 16 rows, and
// where that leaves compute units idle the tokens are split over workgroups too, 512 at least to each, and joined by a
// second launch.  In us, 32 query and 8 cache heads of 128: 1 sequence of 1000 tokens 11.7 whole and 11.5 in 2 splits, 2000 tokens
// 11.8 in 4 splits and 14.6 in 2, 8192 tokens 13.9 in 16 splits and 16.1 in 8; 64 of 8192 156 whole (5.2 TB/s), 161 in 2 splits.
// Workgroups of 8 waves: 18.6 for the 2000 tokens whole, 30 instead of 23 for 64 sequences of 1000.
// Many rows per sequence: workgroups of 128 rows, where there are enough of them (each step of 64 tokens takes 1.9 us, however few
// there are).  Whole tokens, then chunks: 1 sequence of 4000 tokens and 256 queries (64 workgroups of chunks) 50, 124;
// 4 of them with 693 queries in all (173) 134, 131; 32 with 529 (132) 122, 151, with 1059 (265) 191, 178, with 4233 (1058) 650, 398.
struct AttendPlan {
  bool share;
  int32_t tile_rows, splits;
  int64_t tiles;
};

AttendPlan plan_attend(int64_t sequences, int64_t total, int64_t heads, int64_t group, int64_t capacity, bool packed) {
  AttendPlan a;
  a.share = total * group < sequences * 128 || total * group * heads < 160 * 128;
  a.tile_rows = a.share ? 16 : 128;
  // (packed: tiles per sequence are rounded up, and one more zeroes the rows that no sequence has)
  a.tiles = packed ? (total * group + a.tile_rows - 1) / a.tile_rows + sequences + 1
                   : sequences * ((total / sequences * group + a.tile_rows - 1) / a.tile_rows);
  a.splits = 1;
  if (a.share) {
    const int64_t busy = std::max(sequences, total * group / 16) * heads;
    if (capacity > 1024) a.splits = static_cast<int32_t>(std::max<int64_t>(1, std::min<int64_t>({512 / busy, (capacity + 511) / 512, 64})));
  }
  return a;
}

template <int ST, int D>
int launch_attend(const AttendParams& p, const AttendPlan& a, hipStream_t stream) {
  const unsigned units = static_cast<unsigned>(a.tiles * p.heads);
  if (a.share) {
    attend_tokens_kernel<ST, D><<<units * a.splits, 256, 0, stream>>>(p);
    DCQ_LAUNCH_CHECK("dcq_kv8_attention");
    if (a.splits > 1) join_kernel<ST, D><<<units, 256, 0, stream>>>(p);
  } else {
    attend_chunks_kernel<ST, D><<<units, 256, 0, stream>>>(p);
  }
  DCQ_LAUNCH_CHECK("dcq_kv8_attention");
  return DCQ_OK;
}

int check_cache(int64_t pool, int64_t heads, int64_t page, int64_t dim, int64_t sequences, int64_t table_cols, int64_t total) {
  DCQ_REQUIRE(pool >= 1 && heads >= 1 && heads <= 65535 && table_cols >= 1 && sequences >= 0 && total >= 0, DCQ_ERR_ARGUMENT, "bad sizes");
  DCQ_REQUIRE(page == 16 || page == 32 || page == 64 || page == 128, DCQ_ERR_UNSUPPORTED, "pages hold 16, 32, 64 or 128 tokens, not %lld",
              static_cast<long long>(page));
  DCQ_REQUIRE(dim == 64 || dim == 128, DCQ_ERR_UNSUPPORTED, "heads have 64 or 128 channels, not %lld", static_cast<long long>(dim));
  DCQ_REQUIRE(pool <= 0x7fffffff && table_cols <= (int64_t{1} << 30) / page && sequences < (1 << 24) && total < (int64_t{1} << 30),
              DCQ_ERR_UNSUPPORTED, "too many tokens");
  return DCQ_OK;
}

bool aligned(const void* p, int64_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

}  // namespace dcq

using namespace dcq;

extern "C" int dcq_kv8_append(const void* key, const void* value, int32_t storage, const int64_t* key_strides,
                              const int64_t* value_strides, uint8_t* k_codes, float* k_scales, uint8_t* v_codes,
                              float* v_scales, const int32_t* table, const int32_t* lengths, const int32_t* starts,
                              int64_t sequences, int64_t total, int64_t pool, int64_t heads, int64_t page, int64_t dim,
                              int64_t table_cols, dcq_stream_t stream) {
  if (int rc = check_cache(pool, heads, page, dim, sequences, table_cols, total)) return rc;
  DCQ_REQUIRE(storage == DCQ_F32 || storage == DCQ_F16 || storage == DCQ_BF16, DCQ_ERR_ARGUMENT, "bad storage %d", storage);
  if (sequences == 0 || total == 0) return DCQ_OK;
  DCQ_REQUIRE(key && value && key_strides && value_strides && k_codes && k_scales && v_codes && v_scales && table && lengths, DCQ_ERR_ARGUMENT,
              "null pointer");
  DCQ_REQUIRE(starts != nullptr || total % sequences == 0, DCQ_ERR_ARGUMENT, "tokens do not divide into the sequences");
  const int64_t per = 16 / (storage == DCQ_F32 ? 4 : 2);
  for (const int64_t* st : {key_strides, value_strides})
    DCQ_REQUIRE(st[0] % per == 0 && st[1] % per == 0 && st[2] % per == 0, DCQ_ERR_ARGUMENT, "strides must be multiples of 16 bytes");
  DCQ_REQUIRE(aligned(key, 16) && aligned(value, 16) && aligned(k_codes, 16) && aligned(v_codes, 16), DCQ_ERR_ARGUMENT,
              "tensors must be aligned to 16 bytes");
  AppendParams p{};
  p.x[0] = key;
  p.x[1] = value;
  const int64_t* strides[2] = {key_strides, value_strides};
  for (int i = 0; i < 2; ++i) {
    p.x_seq[i] = strides[i][0];
    p.x_token[i] = strides[i][1];
    p.x_head[i] = strides[i][2];
  }
  p.codes[0] = k_codes;
  p.codes[1] = v_codes;
  p.scales[0] = k_scales;
  p.scales[1] = v_scales;
  p.table = table;
  p.lengths = lengths;
  p.starts = starts;
  p.sequences = static_cast<int32_t>(sequences);
  p.total = static_cast<int32_t>(total);
  p.uniform = starts != nullptr ? 0 : static_cast<int32_t>(total / sequences);
  p.pool = static_cast<int32_t>(pool);
  p.heads = static_cast<int32_t>(heads);
  p.table_cols = static_cast<int32_t>(table_cols);
  // n tokens touch at most (n - 1 + page - 1) / page + 1 pages
  const int64_t tiles = starts != nullptr ? total / page + 2 * sequences : sequences * ((p.uniform + page - 2) / page + 1);
  const int64_t groups = (heads + heads_per_workgroup(static_cast<int>(page)) - 1) / heads_per_workgroup(static_cast<int>(page));
  DCQ_REQUIRE(launch_fits(tiles * groups, 256), DCQ_ERR_UNSUPPORTED, "too many tokens");
  const unsigned grid = static_cast<unsigned>(tiles * groups);
  hipStream_t s = static_cast<hipStream_t>(stream);
  auto launch_page = [&](auto st, auto pages) {
    constexpr int ST = decltype(st)::value, P = decltype(pages)::value;
    if (dim == 64)
      append_kernel<ST, 64, P><<<grid, 256, 0, s>>>(p);
    else
      append_kernel<ST, 128, P><<<grid, 256, 0, s>>>(p);
  };
  auto launch = [&](auto st) {
    if (page == 16)
      launch_page(st, std::integral_constant<int, 16>{});
    else if (page == 32)
      launch_page(st, std::integral_constant<int, 32>{});
    else if (page == 64)
      launch_page(st, std::integral_constant<int, 64>{});
    else
      launch_page(st, std::integral_constant<int, 128>{});
  };
  if (storage == DCQ_F32)
    launch(std::integral_constant<int, DCQ_F32>{});
  else if (storage == DCQ_F16)
    launch(std::integral_constant<int, DCQ_F16>{});
  else
    launch(std::integral_constant<int, DCQ_BF16>{});
  DCQ_LAUNCH_CHECK("dcq_kv8_append");
  return DCQ_OK;
}

extern "C" int64_t dcq_kv8_attention_workspace_bytes(int64_t sequences, int64_t total, int64_t heads, int64_t group, int64_t dim,
                                                     int64_t capacity, int32_t packed) {
  if (sequences < 1 || total < 1 || heads < 1 || group < 1 || dim < 1 || capacity < 1) return 0;
  const AttendPlan a = plan_attend(sequences, total, heads, group, capacity, packed != 0);
  return a.splits > 1 ? a.tiles * heads * a.splits * a.tile_rows * (dim + 2) * 4 : 0;
}

extern "C" int dcq_kv8_attention(const void* query, int32_t storage, const int64_t* query_strides, void* out, const int64_t* out_strides,
                                 const uint8_t* k_codes, const float* k_scales, const uint8_t* v_codes, const float* v_scales,
                                 const int32_t* table, const int32_t* lengths, const int32_t* starts, int64_t sequences,
                                 int64_t total, int64_t pool, int64_t heads, int64_t group, int64_t page, int64_t dim,
                                 int64_t table_cols, float scale, int32_t causal, int32_t zero_rest, void* workspace,
                                 int64_t workspace_bytes, dcq_stream_t stream) {
  if (int rc = check_cache(pool, heads, page, dim, sequences, table_cols, total)) return rc;
  DCQ_REQUIRE(storage == DCQ_F16 || storage == DCQ_BF16, DCQ_ERR_UNSUPPORTED, "queries are float16 or bfloat16");
  DCQ_REQUIRE(group >= 1 && group < (int64_t{1} << 30) && total * group < (int64_t{1} << 30), DCQ_ERR_UNSUPPORTED, "too many query heads");
  if (sequences == 0 || total == 0) return DCQ_OK;
  DCQ_REQUIRE(query && query_strides && out && out_strides && k_codes && k_scales && v_codes && v_scales && table && lengths,
              DCQ_ERR_ARGUMENT, "null pointer");
  DCQ_REQUIRE(starts != nullptr || total % sequences == 0, DCQ_ERR_ARGUMENT, "queries do not divide into the sequences");
  for (int i = 0; i < 3; ++i)
    DCQ_REQUIRE(query_strides[i] % 8 == 0 && out_strides[i] % 4 == 0, DCQ_ERR_ARGUMENT,
                "strides must be multiples of 16 bytes (out: 8)");
  DCQ_REQUIRE(aligned(query, 16) && aligned(out, 8) && aligned(k_codes, 16) && aligned(v_codes, 16) && aligned(workspace, 16),
              DCQ_ERR_ARGUMENT, "tensors must be aligned to 16 bytes (out: 8)");
  const AttendPlan a = plan_attend(sequences, total, heads, group, table_cols * page, starts != nullptr);
  DCQ_REQUIRE(launch_fits(a.tiles * heads * a.splits, 256), DCQ_ERR_UNSUPPORTED, "too many queries");
  const int64_t need = dcq_kv8_attention_workspace_bytes(sequences, total, heads, group, dim, table_cols * page, starts != nullptr);
  DCQ_REQUIRE(need == 0 || (workspace != nullptr && workspace_bytes >= need), DCQ_ERR_ARGUMENT, "workspace of %lld bytes, %lld are needed",
              static_cast<long long>(workspace_bytes), static_cast<long long>(need));
  AttendParams p{};
  p.q = query;
  p.out = out;
  p.q_seq = query_strides[0];
  p.q_token = query_strides[1];
  p.q_head = query_strides[2];
  p.o_seq = out_strides[0];
  p.o_token = out_strides[1];
  p.o_head = out_strides[2];
  p.k = k_codes;
  p.v = v_codes;
  p.ks = k_scales;
  p.vs = v_scales;
  p.table = table;
  p.lengths = lengths;
  p.starts = starts;
  p.partial = static_cast<float*>(workspace);
  p.sequences = static_cast<int32_t>(sequences);
  p.total = static_cast<int32_t>(total);
  p.uniform = starts != nullptr ? 0 : static_cast<int32_t>(total / sequences);
  p.pool = static_cast<int32_t>(pool);
  p.heads = static_cast<int32_t>(heads);
  p.group = static_cast<int32_t>(group);
  p.page = static_cast<int32_t>(page);
  p.page_shift = page == 16 ? 4 : page == 32 ? 5 : page == 64 ? 6 : 7;
  p.table_cols = static_cast<int32_t>(table_cols);
  p.causal = causal;
  p.zero_rest = zero_rest != 0 && starts != nullptr;
  p.splits = a.splits;
  p.tiles = static_cast<int32_t>(a.tiles);
  p.scale_log2 = std::fabs(scale) * 1.4426950408889634f;
  p.q_flip = std::signbit(scale) ? 0x80008000u : 0u;
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (storage == DCQ_F16) return dim == 64 ? launch_attend<DCQ_F16, 64>(p, a, s) : launch_attend<DCQ_F16, 128>(p, a, s);
  return dim == 64 ? launch_attend<DCQ_BF16, 64>(p, a, s) : launch_attend<DCQ_BF16, 128>(p, a, s);
}
