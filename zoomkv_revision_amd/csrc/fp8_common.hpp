// Shared pieces of the 8-bit linear kernels (fp8_rows.hip, fp8_linear.hip):
// values held as e4m3 codes with one fp32 scale per 128 channels (of a row, or
// of 128 rows of a weight).
#pragma once

#include "paged_common.hpp"

namespace zkv {

constexpr int kFp8Block = 128;
constexpr float kFp8Max = 448.0f;             // the largest e4m3 value
constexpr float kFp8LeastScale = 0x1p-100f;   // blocks of zeros; 1 / scale stays finite

enum RowType : int { kRowBf16 = 0, kRowF16 = 1, kRowF32 = 2 };

// The scale of a block whose largest magnitude has the bits amax: amax / 448,
// NaN where the block holds an infinity or a NaN (whose bits are the largest).
__device__ __forceinline__ float fp8_scale(uint32_t amax) {
  const float s = fmaxf(__uint_as_float(amax) / kFp8Max, kFp8LeastScale);
  return amax < 0x7F800000u ? s : __uint_as_float(0x7FC00000u);
}

// x / s, r the rounded reciprocal of s: x r corrected by its remainder, which is
// the IEEE quotient (Markstein).  At most 448 (1 + 2^-23), which the conversion
// rounds to 448.  A zero comes out positive.
__device__ __forceinline__ float fp8_quotient(float x, float s, float r) {
  const float q = x * r;
  return __builtin_fmaf(__builtin_fmaf(-q, s, x), r, q);
}

// Four codes of a block, first in the lowest byte.
__device__ __forceinline__ uint32_t fp8_codes4(const float* x, float s, float r) {
  int c = __builtin_amdgcn_cvt_pk_fp8_f32(fp8_quotient(x[0], s, r), fp8_quotient(x[1], s, r), 0, false);
  c = __builtin_amdgcn_cvt_pk_fp8_f32(fp8_quotient(x[2], s, r), fp8_quotient(x[3], s, r), c, true);
  return static_cast<uint32_t>(c);
}

__device__ __forceinline__ uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7FFFFFFFu; }

// The largest of 16 neighbouring lanes' values (a DPP row), in each of them.
__device__ __forceinline__ uint32_t row_max(uint32_t v) {
  v = max(v, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), 0x128, 0xF, 0xF, true)));
  v = max(v, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), 0x124, 0xF, 0xF, true)));
  v = max(v, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), 0x122, 0xF, 0xF, true)));
  v = max(v, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), 0x121, 0xF, 0xF, true)));
  return v;
}

template <int kType>
__device__ __forceinline__ float row_elem(const void* p, int64_t i) {
  if constexpr (kType == kRowF32)
    return static_cast<const float*>(p)[i];
  else
    return elem_to_f32<kType>(static_cast<const uint16_t*>(p)[i]);
}

// Rows start at any element: wide accesses at any of them (scalar ones took a row of
// 7405 fp32 elements 14 us).
typedef uint32_t u32x2_any __attribute__((ext_vector_type(2), aligned(2)));
typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(2)));

// Elements [k, k + 8) of a row of K; those past its end are 0.
template <int kType>
__device__ __forceinline__ void load_row8(const void* row, int k, int K, float (&v)[8]) {
  if (k + 8 <= K) {
    if constexpr (kType == kRowF32) {
      const u32x4_t a = *reinterpret_cast<const u32x4_any*>(static_cast<const float*>(row) + k);
      const u32x4_t b = *reinterpret_cast<const u32x4_any*>(static_cast<const float*>(row) + k + 4);
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = __uint_as_float(a[i]), v[4 + i] = __uint_as_float(b[i]);
    } else {
      const u32x4_t a = *reinterpret_cast<const u32x4_any*>(static_cast<const uint16_t*>(row) + k);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v[2 * i] = elem_to_f32<kType>(a[i] & 0xFFFFu);
        v[2 * i + 1] = elem_to_f32<kType>(a[i] >> 16);
      }
    }
  } else {  // (loads that no lane skips go out together)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float e = row_elem<kType>(row, min(k + i, K - 1));
      v[i] = k + i < K ? e : 0.0f;
    }
  }
}

template <int kType>
__device__ __forceinline__ void store_row8(void* row, int k, int K, const float (&v)[8]) {
  if (k + 8 <= K) {
    if constexpr (kType == kRowF32) {
      u32x4_t a, b;
#pragma unroll
      for (int i = 0; i < 4; ++i) a[i] = __float_as_uint(v[i]), b[i] = __float_as_uint(v[4 + i]);
      *reinterpret_cast<u32x4_any*>(static_cast<float*>(row) + k) = a;
      *reinterpret_cast<u32x4_any*>(static_cast<float*>(row) + k + 4) = b;
    } else {
      u32x4_t o;
#pragma unroll
      for (int i = 0; i < 4; ++i) o[i] = f32_to_elem<kType>(v[2 * i]) | (f32_to_elem<kType>(v[2 * i + 1]) << 16);
      *reinterpret_cast<u32x4_any*>(static_cast<uint16_t*>(row) + k) = o;
    }
  } else {
    for (int i = 0; i < 8 && k + i < K; ++i) {
      if constexpr (kType == kRowF32)
        static_cast<float*>(row)[k + i] = v[i];
      else
        static_cast<uint16_t*>(row)[k + i] = static_cast<uint16_t>(f32_to_elem<kType>(v[i]));
    }
  }
}

// Host side: whether rows of elements of `bytes` bytes at p, ld apart, start on 16 bytes.
inline bool rows_on_16(const void* p, int64_t ld, int bytes) {
  return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && (ld * bytes) % 16 == 0;
}

}  // namespace zkv
