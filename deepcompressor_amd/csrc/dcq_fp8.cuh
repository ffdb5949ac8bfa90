// Device helpers of the kernels that read and write e4m3 codes (gfx950 only).
#pragma once

#include "dcq_common.cuh"

namespace dcq {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

constexpr float kE4m3Max = 448.0f;

// The float32 whose round-to-nearest-even on any coarser grid is v's rounding with ties to the upper neighbour (the tie
// rule of this library's codebooks).  Every tie and every grid value of the coarser grid is an even float32 pattern:
// setting the last bit moves an even positive v up by one step, off the tie and towards the upper neighbour, and leaves
// an odd one, which is no tie, alone; for a negative v the pattern of the next smaller magnitude does the same.  The
// addition turns -0 into +0, whose pattern the subtraction must not see.
__device__ __forceinline__ float ties_up(float v) {
  const int32_t u = __float_as_int(v + 0.0f);
  return __int_as_float((u + (u >> 31)) | 1);
}

// four values (finite ones within +-448) -> four e4m3 codes in one word; NaN -> the NaN code
__device__ __forceinline__ uint32_t to_e4m3x4(float a, float b, float c, float d) {
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(ties_up(a), ties_up(b), 0, false);
  w = __builtin_amdgcn_cvt_pk_fp8_f32(ties_up(c), ties_up(d), w, true);
  return static_cast<uint32_t>(w);
}

__device__ __forceinline__ float clamp_e4m3(float v) {  // (NaN passes)
  v = v > kE4m3Max ? kE4m3Max : v;
  return v < -kE4m3Max ? -kE4m3Max : v;
}

// all ones in the bytes of the `word`-th 4 bytes of a run that lie before `count`
__device__ __forceinline__ uint32_t bytes_before(int count, int word) {
  const int n = count - 4 * word;
  return n >= 4 ? 0xffffffffu : (n <= 0 ? 0u : (1u << (8 * n)) - 1u);
}

__device__ __forceinline__ float load_as_f32(const void* p, int storage, int64_t i) {
  if (storage == DCQ_F32) return static_cast<const float*>(p)[i];
  const uint16_t b = static_cast<const uint16_t*>(p)[i];
  return storage == DCQ_F16 ? f16_to_f32(b) : bf16_to_f32(b);
}

// The matrix instruction over 16-bit operands, and codes as such operands (exact: e4m3 has 4 significant bits).
template <int ST>
struct Half;
template <>
struct Half<DCQ_BF16> {
  static __device__ __forceinline__ f32x4 mfma(const uint4& a, const uint4& b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ uint32_t codes2(uint32_t w, float scale, bool high) {
    return high ? __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, true))
                : __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, false));
  }
};
template <>
struct Half<DCQ_F16> {
  static __device__ __forceinline__ f32x4 mfma(const uint4& a, const uint4& b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ uint32_t codes2(uint32_t w, float scale, bool high) {
    return high ? __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, scale, true))
                : __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, scale, false));
  }
};

// eight codes, times a power of two -> eight 16-bit values
template <int ST>
__device__ __forceinline__ uint4 codes8(uint32_t lo, uint32_t hi, float scale) {
  return {Half<ST>::codes2(lo, scale, false), Half<ST>::codes2(lo, scale, true), Half<ST>::codes2(hi, scale, false),
          Half<ST>::codes2(hi, scale, true)};
}

}  // namespace dcq
