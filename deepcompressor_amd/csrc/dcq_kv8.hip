// Keys and values of past tokens held as e4m3 codes, a power-of-two scale for each page (block of tokens) and head: the
// append that writes them and the attention that reads them (gfx950).
//
// A page holds P tokens (a multiple of 16) of every key / value head: keys [P][D], values transposed, [D][P], so that
// attention reads both as matrix-instruction operands straight from memory, without a transposition.  A table lists
// each sequence's pages; an entry outside the pool stands for no page: appends skip it, attention does not see its
// tokens.
#include "dcq_fp8.cuh"

#include <algorithm>

namespace dcq {

// One sequence's share of a launch whose tiles run over the sequences one after the other.
struct Place {
  int seq;      // -1: the tile lies behind the last sequence's
  int tile;     // the tile's number within the sequence
  int row0;     // the sequence's first row of a packed tensor
  int rows;     // its rows (new tokens, or queries)
  int length;   // its tokens in the cache, as the caller gave them, within the table's capacity
  int first, end;  // seq == -1: the rows that some sequence has lie in [first, end); `tile` counts from the last used one
};

// The sequence that tile `tile` belongs to, found by a wave: 64 sequences at a time, a lane each, with a running sum of
// their tile counts.  starts == nullptr: every sequence has `uniform` rows.  What the tables hold is not trusted: starts
// are cut to [0, total] and to ascending order, lengths to [0, capacity].
template <class Tiles>
__device__ __forceinline__ Place find_place(int64_t tile, const int32_t* starts, int uniform, const int32_t* lengths, int count,
                                            int total, int capacity, Tiles tiles_of) {
  const int lane = threadIdx.x % kWave;
  int64_t before = 0;
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
    int64_t upto = tiles;
#pragma unroll
    for (int off = 1; off < kWave; off <<= 1) {
      const int64_t other = __shfl_up(upto, off, kWave);
      if (lane >= off) upto += other;
    }
    const uint64_t hit = __ballot(tile < before + upto);
    if (hit != 0) {
      const int at = __builtin_ctzll(hit);
      Place f;
      f.seq = base + at;
      f.tile = static_cast<int>(tile - before - __shfl(upto, at, kWave)) + __shfl(tiles, at, kWave);
      f.row0 = __shfl(row0, at, kWave);
      f.rows = __shfl(rows, at, kWave);
      f.length = __shfl(length, at, kWave);
      f.first = f.end = 0;
      return f;
    }
    before += __shfl(upto, kWave - 1, kWave);
  }
  const int first = starts != nullptr ? min(max(starts[0], 0), total) : 0;
  const int end = starts != nullptr ? min(max(starts[count], first), total) : total;
  return {-1, static_cast<int>(tile - before), 0, 0, 0, first, end};
}

// =============================================================================================
// Append.  A workgroup takes one page's new tokens of one head, of the keys or of the values: the largest finite
// magnitude, the scale, the older codes' move to it if it grew, the new codes.
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
  int32_t sequences, total, uniform, pool, heads, page, table_cols;
};

constexpr int kMaxPage = 128;

__device__ __forceinline__ int pages_touched(int rows, int length, int page, int capacity) {
  rows = min(rows, capacity - length);
  return rows <= 0 ? 0 : (length + rows - 1) / page - length / page + 1;
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

template <int ST, int D>
__global__ __launch_bounds__(256) void append_kernel(const AppendParams p) {
  constexpr int kTeam = D / 8;             // lanes of a token, 8 channels each
  constexpr int kTokens = 256 / kTeam;     // tokens per pass
  constexpr int kPitch = kMaxPage + 4;     // of the transposed tile in LDS
  using S = Storage<ST>;
  using elem_t = typename S::elem_t;
  __shared__ float part[4];
  __shared__ uint32_t tile[D * kPitch / 4];
  const int capacity = p.table_cols * p.page;
  const int P = p.page;
  const Place f = find_place(blockIdx.x, p.starts, p.uniform, p.lengths, p.sequences, p.total, capacity,
                             [&](int rows, int length) { return pages_touched(rows, length, P, capacity); });
  if (f.seq < 0) return;
  const int head = blockIdx.y, kind = blockIdx.z;
  const int col = f.length / P + f.tile;
  const int page = p.table[static_cast<int64_t>(f.seq) * p.table_cols + col];
  if (page < 0 || page >= p.pool) return;
  const int begin = f.tile == 0 ? f.length - col * P : 0;            // first new slot of the page
  const int skip = col * P + begin - f.length;                       // new tokens on earlier pages
  const int n = min(P - begin, f.rows - skip);
  const int64_t row0 = p.starts != nullptr ? f.row0 * p.x_token[kind] : f.seq * p.x_seq[kind];
  const elem_t* x = static_cast<const elem_t*>(p.x[kind]) + row0 + skip * p.x_token[kind] + head * p.x_head[kind];
  const int64_t unit = static_cast<int64_t>(page) * p.heads + head;
  uint8_t* codes = p.codes[kind] + unit * P * D;
  const int sub = threadIdx.x % kTeam, first = threadIdx.x / kTeam;

  auto load_8 = [&](int token, float(&v)[8]) {
    const elem_t* at = x + token * p.x_token[kind] + sub * 8;
#pragma unroll
    for (int i = 0; i < 8 / S::kVec; ++i) {
      const auto c = load_chunk<elem_t, S::kVec>(at + i * S::kVec);
#pragma unroll
      for (int j = 0; j < S::kVec; ++j) v[i * S::kVec + j] = S::load(c.v[j]);
    }
  };
  float largest = 0.0f;
  for (int t = first; t < n; t += kTokens) {
    float v[8];
    load_8(t, v);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float a = fabsf(v[i]);
      largest = fmaxf(largest, a < __builtin_inff() ? a : 0.0f);
    }
  }
  largest = team_max(largest, kWave);
  if (threadIdx.x % kWave == 0) part[threadIdx.x / kWave] = largest;
  const float old = p.scales[kind][unit];
  __syncthreads();  // (also: every thread has read the old scale before one writes the new)
  largest = fmaxf(fmaxf(part[0], part[1]), fmaxf(part[2], part[3]));
  float scale = power_scale(largest);
  if (begin > 0) scale = fmaxf(scale, old);
  if (threadIdx.x == 0) p.scales[kind][unit] = scale;
  if (begin > 0 && scale != old) {
    const float ratio = old / scale;
    for (int i = threadIdx.x; i < P * D / 16; i += 256) {  // (slots behind the tokens too: nobody reads them)
      uint4* at = reinterpret_cast<uint4*>(codes) + i;
      const uint4 w = *at;
      *at = uint4{rescale_codes(w.x, ratio), rescale_codes(w.y, ratio), rescale_codes(w.z, ratio), rescale_codes(w.w, ratio)};
    }
    __syncthreads();  // the new codes overwrite some of these
  }
  const float inverse = 1.0f / scale;  // a power of two: exact
  for (int t = first; t < n; t += kTokens) {
    float v[8];
    load_8(t, v);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] *= inverse;  // within +-448, or not finite: those become the NaN code
    const uint2 w = {to_e4m3x4(v[0], v[1], v[2], v[3]), to_e4m3x4(v[4], v[5], v[6], v[7])};
    if (kind == 0) {
      *reinterpret_cast<uint2*>(codes + (begin + t) * D + sub * 8) = w;
    } else {
      uint8_t* to = reinterpret_cast<uint8_t*>(tile) + sub * 8 * kPitch + begin + t;
#pragma unroll
      for (int i = 0; i < 8; ++i) to[i * kPitch] = static_cast<uint8_t>((i < 4 ? w.x : w.y) >> (8 * (i & 3)));
    }
  }
  if (kind == 0) return;
  __syncthreads();
  const int end = begin + n, c0 = begin / 16, per = (end + 15) / 16 - c0;
  for (int i = threadIdx.x; i < D * per; i += 256) {
    const int d = i / per, c = c0 + i % per;
    const uint32_t* from = tile + (d * kPitch + c * 16) / 4;
    uint8_t* to = codes + d * P + c * 16;
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
// tokens need no other path.  Codes become bfloat16 or float16 exactly (4 significant bits), their scales are applied
// to scores and probabilities in float32.  The probabilities are rounded to bfloat16 for either type of query: the
// value's scale is multiplied into them, and float16 would lose small ones (2^-9 relative per probability, uncorrelated;
// the outputs' own rounding is as large for bfloat16).
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
  float* partial;  // splits > 1: per (tile, head, split) the rows' sums [16 RT][D], then maxima and sums [2][16 RT]
  int32_t sequences, total, uniform, pool, heads, group, page, page_shift, table_cols, causal, zero_rest, splits;
  float scale_log2;
};

__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
  const bf16x2 t = {static_cast<__bf16>(a), static_cast<__bf16>(b)};
  return __builtin_bit_cast(uint32_t, t);
}

// 0x80 in every byte of w that is an e4m3 NaN (0x7f or 0xff)
__device__ __forceinline__ uint32_t nan_codes(uint32_t w) { return ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; }

// The rows of a packed output that no sequence has, set to 0 by the tiles behind the last sequence's (at least one).
template <int D>
__device__ __forceinline__ void zero_rows(const AttendParams& p, const Place& f, int head) {
  const int used = static_cast<int>(blockIdx.x) - f.tile;
  const int stride = static_cast<int>(gridDim.x) - used, rest = f.first + p.total - f.end;
  for (int u = f.tile; u < rest; u += stride) {
    const int64_t row = u < f.first ? u : u - f.first + f.end;
    for (int i = threadIdx.x; i < p.group * (D / 4); i += 256) {
      uint16_t* at = static_cast<uint16_t*>(p.out) + row * p.o_token + static_cast<int64_t>(head * p.group + i / (D / 4)) * p.o_head;
      store_chunk<uint16_t, 4>(at + i % (D / 4) * 4, Chunk<uint16_t, 4>{});
    }
  }
}

// The four waves of a workgroup take four row tiles (SHARE = false), or share out the tokens of one (SHARE = true).
template <int ST, int D, int RT, bool SHARE>
__global__ __launch_bounds__(256) void attend_kernel(const AttendParams p) {
  constexpr int kWaves = 4, kRows = 16 * RT, kKeyLoads = D / 64, kDims = D / 16;
  constexpr int kTileRows = SHARE ? kRows : kRows * kWaves;
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  const int r = lane % 16, g = lane / 16;
  const int capacity = p.table_cols * p.page;
  const Place f = find_place(blockIdx.x, p.starts, p.uniform, p.lengths, p.sequences, p.total, capacity,
                             [&](int rows, int) { return static_cast<int>((static_cast<int64_t>(rows) * p.group + kTileRows - 1) / kTileRows); });
  const int head = blockIdx.y, split = blockIdx.z;
  if (f.seq < 0) {
    if (p.zero_rest && split == 0) zero_rows<D>(p, f, head);
    return;
  }
  const int row_count = f.rows * p.group;
  const int row_base = f.tile * kTileRows + (SHARE ? 0 : wave * kRows);

  // the rows' queries as operands, and how many tokens each row sees
  uint4 q[RT][2 * kKeyLoads];
  int limit[RT];
  int most = 0, least = 0x7fffffff;
  const int64_t q_base = p.starts != nullptr ? f.row0 * p.q_token : f.seq * p.q_seq;
#pragma unroll
  for (int t = 0; t < RT; ++t) {
    const int row = row_base + t * 16 + r;
    const bool in = row < row_count;
    const int qi = in ? row / p.group : 0, h = in ? row % p.group : 0;
    limit[t] = in ? (p.causal ? max(f.length - f.rows + qi + 1, 0) : f.length) : -1;
    if (in) {
      most = max(most, limit[t]);
      least = min(least, limit[t]);
    }
    const uint16_t* at = static_cast<const uint16_t*>(p.q) + q_base + qi * p.q_token + static_cast<int64_t>(head * p.group + h) * p.q_head;
#pragma unroll
    for (int j = 0; j < kKeyLoads; ++j)
#pragma unroll
      for (int e = 0; e < 2; ++e)
        q[t][2 * j + e] = in ? *reinterpret_cast<const uint4*>(at + j * 64 + g * 16 + e * 8) : uint4{0, 0, 0, 0};
  }
#pragma unroll
  for (int off = 1; off < 16; off <<= 1) {
    most = max(most, __shfl_xor(most, off, kWave));
    least = min(least, __shfl_xor(least, off, kWave));
  }
#pragma unroll
  for (int t = 0; t < RT; ++t)
    if (limit[t] < 0) limit[t] = most;  // rows that are none: whatever spares the mask

  // this workgroup's (and, if shared out, this wave's) steps of 64 tokens
  const int steps = (most + 63) / 64;
  const int share = (steps + p.splits - 1) / p.splits;
  const int step_end = min((split + 1) * share, steps);
  const int step_first = split * share + (SHARE ? wave : 0);
  constexpr int kStride = SHARE ? kWaves : 1;

  f32x4 acc[RT][kDims];
  float m[RT], l[RT];
  bool seen[RT];
#pragma unroll
  for (int t = 0; t < RT; ++t) {
    m[t] = -__builtin_inff();
    l[t] = 0.0f;
    seen[t] = false;
#pragma unroll
    for (int d = 0; d < kDims; ++d) acc[t][d] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  }
  const int32_t* table = p.table + static_cast<int64_t>(f.seq) * p.table_cols;
  const int page_mask = p.page - 1;
  auto page_of = [&](int token) {
    const int c = token >> p.page_shift;
    const int id = c < p.table_cols ? table[c] : -1;
    return id < p.pool ? id : -1;
  };

  for (int step = step_first; step < step_end; step += kStride) {
    const int t0 = step * 64;
    const int own = t0 + 16 * g;                                  // the lane's first token of the values
    const int key = t0 + 16 * (r / 4) + (r & 3);                  // the lane's token of key tile 0
    const int own_page = page_of(own), key_page = page_of(key);
    const int64_t own_unit = static_cast<int64_t>(max(own_page, 0)) * p.heads + head;
    const int64_t key_unit = static_cast<int64_t>(max(key_page, 0)) * p.heads + head;
    const uint8_t* kp = p.k + (key_unit * p.page + (key & page_mask)) * D + g * 16;
    const uint8_t* vp = p.v + (own_unit * D + r) * p.page + (own & page_mask);
    uint4 kc[4][kKeyLoads], vc[kDims];
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int j = 0; j < kKeyLoads; ++j) kc[t][j] = *reinterpret_cast<const uint4*>(kp + t * 4 * D + j * 64);
#pragma unroll
    for (int d = 0; d < kDims; ++d) vc[d] = *reinterpret_cast<const uint4*>(vp + d * 16 * p.page);
    const float key_scale = p.ks[own_unit] * p.scale_log2, value_scale = p.vs[own_unit];

    f32x4 s[RT][4];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
#pragma unroll
      for (int i = 0; i < RT; ++i) s[i][t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int j = 0; j < kKeyLoads; ++j) {
        const uint4 lo = codes8<ST>(kc[t][j].x, kc[t][j].y), hi = codes8<ST>(kc[t][j].z, kc[t][j].w);
#pragma unroll
        for (int i = 0; i < RT; ++i) {
          s[i][t] = Half<ST>::mfma(lo, q[i][2 * j], s[i][t]);
          s[i][t] = Half<ST>::mfma(hi, q[i][2 * j + 1], s[i][t]);
        }
      }
    }
    const bool masked = t0 + 64 > least || __any(own_page < 0);
    uint4 pr[RT][2];
#pragma unroll
    for (int i = 0; i < RT; ++i) {
      float top = -__builtin_inff();
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float v = s[i][t][e] * key_scale;
          if (masked) v = own + 4 * t + e < limit[i] && own_page >= 0 ? v : -__builtin_inff();
          s[i][t][e] = v;
          top = fmaxf(top, v);
        }
      seen[i] = seen[i] || !masked || (own < limit[i] && own_page >= 0);
      top = fmaxf(top, __shfl_xor(top, 16, kWave));
      top = fmaxf(top, __shfl_xor(top, 32, kWave));
      const float now = fmaxf(m[i], top);
      const float base = now == -__builtin_inff() ? 0.0f : now;
      const float fade = __builtin_amdgcn_exp2f(m[i] - base);
      m[i] = now;
      l[i] *= fade;
#pragma unroll
      for (int d = 0; d < kDims; ++d)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[i][d][e] *= fade;
      float w[16];
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float x = __builtin_amdgcn_exp2f(s[i][t][e] - base);
          l[i] += x;
          w[4 * t + e] = x * value_scale;
          if (masked && !(own + 4 * t + e < limit[i] && own_page >= 0)) w[4 * t + e] = 0.0f;  // (the scale may be anything)
        }
#pragma unroll
      for (int u = 0; u < 2; ++u)
        pr[i][u] = {pack_bf16(w[8 * u], w[8 * u + 1]), pack_bf16(w[8 * u + 2], w[8 * u + 3]), pack_bf16(w[8 * u + 4], w[8 * u + 5]),
                    pack_bf16(w[8 * u + 6], w[8 * u + 7])};
    }
    if (masked) {
      // Memory behind the last visible token may hold anything, NaN codes too, which a probability of 0 does not
      // silence: those bytes become 0.
      const int count = own_page < 0 ? 0 : min(max(most - own, 0), 16);
      const uint32_t keep[4] = {bytes_before(count, 0), bytes_before(count, 1), bytes_before(count, 2), bytes_before(count, 3)};
      uint32_t bad = 0;
#pragma unroll
      for (int d = 0; d < kDims; ++d) {
        vc[d].x &= keep[0];
        vc[d].y &= keep[1];
        vc[d].z &= keep[2];
        vc[d].w &= keep[3];
        bad |= nan_codes(vc[d].x) | nan_codes(vc[d].y) | nan_codes(vc[d].z) | nan_codes(vc[d].w);
      }
      if (__any(bad != 0)) {
        // A token whose value is NaN, seen by some rows and not by others: a product of "is NaN" and "is seen" tells
        // which outputs become NaN, and the codes are made 0 for the others.
#pragma unroll
        for (int d = 0; d < kDims; ++d) {
          uint32_t* w = reinterpret_cast<uint32_t*>(&vc[d]);
          uint32_t flag[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            flag[k] = nan_codes(w[k]) >> 7;  // 1 per NaN byte
            w[k] &= ~(flag[k] * 0xffu);
            flag[k] *= 0x38u;                // the code of 1
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
              hits = Half<DCQ_BF16>::mfma(codes8<DCQ_BF16>(flag[2 * u], flag[2 * u + 1]), b, hits);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (hits[e] > 0.0f) acc[i][d][e] = __builtin_nanf("");
          }
        }
      }
    }
#pragma unroll
    for (int d = 0; d < kDims; ++d) {
      const uint4 lo = codes8<DCQ_BF16>(vc[d].x, vc[d].y), hi = codes8<DCQ_BF16>(vc[d].z, vc[d].w);
#pragma unroll
      for (int i = 0; i < RT; ++i) {
        acc[i][d] = Half<DCQ_BF16>::mfma(lo, pr[i][0], acc[i][d]);
        acc[i][d] = Half<DCQ_BF16>::mfma(hi, pr[i][1], acc[i][d]);
      }
    }
  }

  // the rows' sums over the lane groups; a row that saw only scores of -inf is NaN (0 / 0), one that saw nothing is 0
#pragma unroll
  for (int i = 0; i < RT; ++i) {
    if (seen[i] && m[i] == -__builtin_inff()) l[i] = __builtin_nanf("");
    l[i] += __shfl_xor(l[i], 16, kWave);
    l[i] += __shfl_xor(l[i], 32, kWave);
  }
  if constexpr (SHARE) {
    static_assert(RT == 1, "waves share out the tokens of 16 rows");
    __shared__ float part_m[kWaves][16], part_l[kWaves][16];
    __shared__ f32x4 part_o[kWaves - 1][kDims][kWave];
    if (g == 0) {
      part_m[wave][r] = m[0];
      part_l[wave][r] = l[0];
    }
    __syncthreads();
    float top = fmaxf(fmaxf(part_m[0][r], part_m[1][r]), fmaxf(part_m[2][r], part_m[3][r]));
    const float base = top == -__builtin_inff() ? 0.0f : top;
    const float fade = __builtin_amdgcn_exp2f(m[0] - base);
#pragma unroll
    for (int d = 0; d < kDims; ++d)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[0][d][e] *= fade;
    if (wave > 0) {
#pragma unroll
      for (int d = 0; d < kDims; ++d) part_o[wave - 1][d][lane] = acc[0][d];
    }
    __syncthreads();
    if (wave > 0) return;
    l[0] = 0.0f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) l[0] += part_l[w][r] * __builtin_amdgcn_exp2f(part_m[w][r] - base);
    m[0] = top;
#pragma unroll
    for (int w = 0; w < kWaves - 1; ++w)
#pragma unroll
      for (int d = 0; d < kDims; ++d) acc[0][d] += part_o[w][d][lane];
  }
#pragma unroll
  for (int i = 0; i < RT; ++i) {
    const int row = row_base + i * 16 + r;
    if (row >= row_count) continue;
    if (SHARE && p.splits > 1) {
      const int64_t unit = (static_cast<int64_t>(blockIdx.x) * p.heads + head) * p.splits + split;
      float* at = p.partial + unit * (kTileRows * (D + 2));
      const int local = row - f.tile * kTileRows;
#pragma unroll
      for (int d = 0; d < kDims; ++d) *reinterpret_cast<f32x4*>(at + local * D + d * 16 + g * 4) = acc[i][d];
      if (g == 0) {
        at[kTileRows * D + local] = m[i];
        at[kTileRows * (D + 1) + local] = l[i];
      }
    } else {
      const int qi = row / p.group, h = row % p.group;
      const int64_t base = p.starts != nullptr ? f.row0 * p.o_token : f.seq * p.o_seq;
      uint16_t* at = static_cast<uint16_t*>(p.out) + base + qi * p.o_token + static_cast<int64_t>(head * p.group + h) * p.o_head;
      const float inverse = l[i] == 0.0f ? 0.0f : 1.0f / l[i];
#pragma unroll
      for (int d = 0; d < kDims; ++d) {
        Chunk<uint16_t, 4> c;
#pragma unroll
        for (int e = 0; e < 4; ++e) c.v[e] = Storage<ST>::store(acc[i][d][e] * inverse);
        store_chunk<uint16_t, 4>(at + d * 16 + g * 4, c);
      }
    }
  }
}

// Joins the splits of a row: one wave per row and head.
template <int ST, int D, int TILE_ROWS>
__global__ __launch_bounds__(256) void join_kernel(const AttendParams p) {
  const int lane = threadIdx.x % kWave;
  const int capacity = p.table_cols * p.page;
  const Place f = find_place(blockIdx.x, p.starts, p.uniform, p.lengths, p.sequences, p.total, capacity,
                             [&](int rows, int) { return static_cast<int>((static_cast<int64_t>(rows) * p.group + TILE_ROWS - 1) / TILE_ROWS); });
  const int head = blockIdx.y;
  if (f.seq < 0) return;
  const int row_count = f.rows * p.group;
  for (int local = threadIdx.x / kWave; local < TILE_ROWS; local += 4) {
    const int row = f.tile * TILE_ROWS + local;
    if (row >= row_count) return;
    const float* at = p.partial + (static_cast<int64_t>(blockIdx.x) * p.heads + head) * p.splits * (TILE_ROWS * (D + 2));
    float top = -__builtin_inff();
    for (int s = 0; s < p.splits; ++s) top = fmaxf(top, at[s * (TILE_ROWS * (D + 2)) + TILE_ROWS * D + local]);
    const float base = top == -__builtin_inff() ? 0.0f : top;
    float l = 0.0f, o[D / kWave];
#pragma unroll
    for (int d = 0; d < D / kWave; ++d) o[d] = 0.0f;
    for (int s = 0; s < p.splits; ++s) {
      const float* from = at + s * (TILE_ROWS * (D + 2));
      const float w = __builtin_amdgcn_exp2f(from[TILE_ROWS * D + local] - base);
      l += w * from[TILE_ROWS * (D + 1) + local];
#pragma unroll
      for (int d = 0; d < D / kWave; ++d) o[d] += w * from[local * D + lane * (D / kWave) + d];
    }
    const int qi = row / p.group, h = row % p.group;
    const int64_t out_base = p.starts != nullptr ? f.row0 * p.o_token : f.seq * p.o_seq;
    uint16_t* to = static_cast<uint16_t*>(p.out) + out_base + qi * p.o_token + static_cast<int64_t>(head * p.group + h) * p.o_head;
    const float inverse = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
    for (int d = 0; d < D / kWave; ++d) to[lane * (D / kWave) + d] = Storage<ST>::store(o[d] * inverse);
  }
}

// How a launch covers its rows.  Single tokens (few rows per sequence): a workgroup's waves share out the tokens of 16
// rows, and where that leaves compute units idle the tokens are split over workgroups too and joined by a second launch.
struct AttendPlan {
  bool share;
  int32_t tile_rows, splits;
  int64_t tiles;
};

AttendPlan plan_attend(int64_t sequences, int64_t total, int64_t heads, int64_t group, int64_t capacity, bool packed) {
  AttendPlan a;
  a.share = total * group < sequences * 64;
  a.tile_rows = a.share ? 16 : 128;
  // (packed: tiles per sequence are rounded up, and one more zeroes the rows that no sequence has)
  a.tiles = packed ? (total * group + a.tile_rows - 1) / a.tile_rows + sequences + 1
                   : sequences * ((total / sequences * group + a.tile_rows - 1) / a.tile_rows);
  a.splits = 1;
  if (a.share) {
    const int64_t busy = (packed ? sequences : a.tiles) * heads;
    a.splits = static_cast<int32_t>(std::max<int64_t>(1, std::min<int64_t>({(1024 + busy - 1) / busy, (capacity + 255) / 256, 64})));
  }
  return a;
}

template <int ST, int D>
int launch_attend(const AttendParams& p, const AttendPlan& a, hipStream_t stream) {
  const dim3 grid(static_cast<unsigned>(a.tiles), p.heads, a.splits);
  if (a.share) {
    attend_kernel<ST, D, 1, true><<<grid, 256, 0, stream>>>(p);
    DCQ_LAUNCH_CHECK("dcq_kv8_attention");
    if (a.splits > 1) join_kernel<ST, D, 16><<<dim3(grid.x, grid.y), 256, 0, stream>>>(p);
  } else {
    attend_kernel<ST, D, 2, false><<<grid, 256, 0, stream>>>(p);
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
  p.page = static_cast<int32_t>(page);
  p.table_cols = static_cast<int32_t>(table_cols);
  // n tokens touch at most (n - 1 + page - 1) / page + 1 pages
  const int64_t tiles = starts != nullptr ? total / page + 2 * sequences : sequences * ((p.uniform + page - 2) / page + 1);
  const dim3 grid(static_cast<unsigned>(tiles), static_cast<unsigned>(heads), 2);
  hipStream_t s = static_cast<hipStream_t>(stream);
  auto launch = [&](auto st) {
    constexpr int ST = decltype(st)::value;
    if (dim == 64)
      append_kernel<ST, 64><<<grid, 256, 0, s>>>(p);
    else
      append_kernel<ST, 128><<<grid, 256, 0, s>>>(p);
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
  DCQ_REQUIRE(group >= 1 && total * group < (int64_t{1} << 30), DCQ_ERR_UNSUPPORTED, "too many query heads");
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
  p.scale_log2 = scale * 1.4426950408889634f;
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (storage == DCQ_F16) return dim == 64 ? launch_attend<DCQ_F16, 64>(p, a, s) : launch_attend<DCQ_F16, 128>(p, a, s);
  return dim == 64 ? launch_attend<DCQ_BF16, 64>(p, a, s) : launch_attend<DCQ_BF16, 128>(p, a, s);
}
