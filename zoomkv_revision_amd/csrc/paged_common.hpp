// Shared pieces of the paged-cache kernels (paged.hip, paged_attention.hip).
#pragma once

#include "zkv_common.hpp"

namespace zkv {

// The page pool of one layer: page id and token-in-page -> element offset of
// K (and V, whose pool has the same strides) for a KV head.  Strides count
// elements; the head dim is contiguous.
struct PageLayout {
  int64_t page_stride, head_stride, token_stride;
  int num_pages, page_size;
};

// n / d of 31-bit n by a multiplication (round-up method: l = ceil(log2 d),
// mul = floor(2^32 (2^l - d) / d) + 1, n / d = (hi(n * mul) + n) >> l; the sum
// stays below 2^32 because n < 2^31).
struct FastDiv {
  uint32_t mul, shift, d;
};

inline FastDiv fast_div(uint32_t d) {
  uint32_t l = 0;
  while ((1ull << l) < d) ++l;
  return FastDiv{static_cast<uint32_t>(((1ull << 32) * ((1ull << l) - d)) / d + 1), l, d};
}

__device__ __forceinline__ uint32_t div_by(uint32_t n, const FastDiv& f) {
  return (__umulhi(n, f.mul) + n) >> f.shift;
}

enum ElemType : int { kBf16 = 0, kF16 = 1 };

template <int kType>
__device__ __forceinline__ float elem_to_f32(uint32_t bits16) {
  if constexpr (kType == kBf16)
    return __uint_as_float(bits16 << 16);
  else
    return static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(bits16)));
}

template <int kType>
__device__ __forceinline__ uint32_t f32_to_elem(float x) {
  if constexpr (kType == kBf16)
    return f32_to_bf16_bits(x);
  else
    return f32_to_f16_bits(x);
}

// The e4m3 code of x, values beyond the type's largest (448) clamped to it
// (the conversion alone would make them NaN), NaN kept.
__device__ __forceinline__ float clamp_e4m3(float x) {
  const float y = fminf(fmaxf(x, -448.0f), 448.0f);
  return x != x ? x : y;
}

// Four e4m3 codes, first in the lowest byte.
__device__ __forceinline__ uint32_t e4m3x4(float a, float b, float c, float d) {
  int r = __builtin_amdgcn_cvt_pk_fp8_f32(clamp_e4m3(a), clamp_e4m3(b), 0, false);
  r = __builtin_amdgcn_cvt_pk_fp8_f32(clamp_e4m3(c), clamp_e4m3(d), r, true);
  return static_cast<uint32_t>(r);
}

// Host side: why a page pool cannot be taken, or null.
inline const char* check_pages(const PageLayout& l, int kv, int d, int cell_bytes) {
  if (l.num_pages < 1 || l.page_size < 1) return "a pool has at least one page of at least one token";
  if (static_cast<int64_t>(l.num_pages) * l.page_size >= (1ll << 31)) return "a pool holds fewer than 2^31 tokens";
  if (kv < 1) return "no KV heads";
  if (d != 64 && d != 128 && d != 256) return "the head dim is 64, 128 or 256";
  if (l.page_stride < 0 || l.head_stride < 0 || l.token_stride < 0) return "negative strides";
  if ((l.page_stride * cell_bytes) % 16 || (l.head_stride * cell_bytes) % 16 || (l.token_stride * cell_bytes) % 16)
    return "every row of a pool starts on 16 bytes";
  return nullptr;
}

}  // namespace zkv
