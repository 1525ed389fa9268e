// Products of rows and weights held as e4m3 codes with a scale per block of 128:
//
//   y[m, n] = sum_b xs[m, b] ws[n / 128, b] sum_{k in block b} x[m, k] w[n, k]
//
// The codes go into the bf16 matrix instructions, which they enter exactly (one
// v_cvt_scalef32_pk_bf16_fp8 per two): their sums are those of fp32 (1e-8 to 4e-8 of
// the sum of magnitudes over a block, measured).  The 8-bit instructions run at
// twice the rate but add each 8 products with 14 bits below the largest (1.5e-5 to
// 2.3e-5): a small term next to two large ones that cancel would be gone.  A
// block's sum times its two scales is added to the running sums in fp32, one
// multiply-add per value.  An element sits in the same place of A (weight rows) and
// B (x rows), so which k a lane holds does not matter: a lane takes whole runs of 16
// bytes.
//
//  * linear: y [+ residual], rounded once to the output's type.
//  * gated: the weight's first half of rows is gate, the second up; y =
//    silu(gate) * up, never rounded to 16 bits, comes out as codes and scales.
#include "fp8_common.hpp"

#include <algorithm>

namespace zkv {
namespace {

struct LinearArgs {
  const uint8_t* x;  // [M, 128 nkb]
  int64_t x_ld;
  const float* xs;  // element (m, b) at m * xs_m + b * xs_b
  int64_t xs_m, xs_b;
  const uint8_t* w;  // [N, 128 nkb], or [2 N, ...] where gated
  int64_t w_ld;
  const float* ws;  // [blocks of N (twice where gated), nkb]
  int M, N, nkb;    // N: rows of the weight, of its gate half where gated
  // linear
  const void* res;
  int64_t res_ld;
  void* out;
  int64_t out_ld;
  int type;
  // gated
  uint8_t* codes;
  int64_t codes_ld;
  float* scales;
  int64_t s_m, s_b;
  float* act;                 // [blocks of N][M][128]
  unsigned long long* slots;  // arrivals per (block of N, group of x rows)
  unsigned long long epoch;
};

// 16 codes as two operands of 8 bf16 values.
__device__ __forceinline__ void codes_to_bf16(const u32x4_t c, bf16x8_t& lo, bf16x8_t& hi) {
  u32x4_t a, b;
#define ZKV_PAIR(w, half) __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, half))
  a[0] = ZKV_PAIR(c[0], false), a[1] = ZKV_PAIR(c[0], true);
  a[2] = ZKV_PAIR(c[1], false), a[3] = ZKV_PAIR(c[1], true);
  b[0] = ZKV_PAIR(c[2], false), b[1] = ZKV_PAIR(c[2], true);
  b[2] = ZKV_PAIR(c[3], false), b[3] = ZKV_PAIR(c[3], true);
#undef ZKV_PAIR
  lo = __builtin_bit_cast(bf16x8_t, a), hi = __builtin_bit_cast(bf16x8_t, b);
}

// A lane's 32 codes of a row's block, for the 16 x 16 products.
struct Operand16 {
  bf16x8_t v[4];
  __device__ __forceinline__ void set(const u32x4_t a, const u32x4_t b) {
    codes_to_bf16(a, v[0], v[1]);
    codes_to_bf16(b, v[2], v[3]);
  }
};

__device__ __forceinline__ float4_t block_sum(const Operand16& a, const Operand16& b) {
  float4_t s = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
  for (int q = 0; q < 4; ++q) s = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.v[q], b.v[q], s, 0, 0, 0);
  return s;
}

__device__ __forceinline__ void add_scaled(float4_t& acc, float4_t v, float s) {
#pragma unroll
  for (int i = 0; i < 4; ++i) acc[i] = __builtin_fmaf(v[i], s, acc[i]);
}

__device__ __forceinline__ float silu_mul(float g, float u) { return g / (1.0f + expf(-g)) * u; }

__device__ __forceinline__ void store_out(const LinearArgs& p, int m, int n, float y) {
  const int64_t o = m * p.out_ld + n, r = m * p.res_ld + n;
  if (p.type == kRowBf16) {
    if (p.res) y += elem_to_f32<kBf16>(static_cast<const uint16_t*>(p.res)[r]);
    static_cast<uint16_t*>(p.out)[o] = static_cast<uint16_t>(f32_to_elem<kBf16>(y));
  } else if (p.type == kRowF16) {
    if (p.res) y += elem_to_f32<kF16>(static_cast<const uint16_t*>(p.res)[r]);
    static_cast<uint16_t*>(p.out)[o] = static_cast<uint16_t>(f32_to_elem<kF16>(y));
  } else {
    if (p.res) y += static_cast<const float*>(p.res)[r];
    static_cast<float*>(p.out)[o] = y;
  }
}

// ---------------------------------------------------------------------------
// Few rows of x: the weights stream from memory into registers.  A unit is R
// (16, 8 or 4) weight rows (gated: R gate rows and the matching up rows) of 16 kMT rows
// of x; the waves of a workgroup split its blocks of k (wave w takes blocks w, w +
// nw, ...), so nothing is staged and every wave reads its own part of x.  Lanes
// whose A row is past R, or whose B column is past M, repeat the last: no more
// memory moves.  The waves' sums meet in LDS and are added in wave order.
// ---------------------------------------------------------------------------
template <int kTiles, int kMT>
struct StreamWave {
  float4_t acc[kTiles][kMT];

  // kCnt blocks, three in flight
  template <int kCnt>
  __device__ __forceinline__ void run(const uint8_t* const (&wr)[kTiles], const float* const (&wsr)[kTiles],
                                      const uint8_t* const (&xr)[kMT], const float* const (&xsr)[kMT], int64_t xs_b,
                                      int wave, int nw) {
#pragma unroll
    for (int t = 0; t < kTiles; ++t)
#pragma unroll
      for (int j = 0; j < kMT; ++j) acc[t][j] = float4_t{0.0f, 0.0f, 0.0f, 0.0f};
    if constexpr (kCnt > 0) {
      constexpr int kDepth = kCnt < 3 ? kCnt : 3;
      u32x4_t a[kDepth][kTiles][2], b[kDepth][kMT][2];
      float xs[kDepth][kMT], ws[kDepth][kTiles];
      auto load = [&](int i) {
        const int kb = wave + i * nw, d = i % kDepth;
#pragma unroll
        for (int t = 0; t < kTiles; ++t) {
          a[d][t][0] = *reinterpret_cast<const u32x4_t*>(wr[t] + kb * kFp8Block);
          a[d][t][1] = *reinterpret_cast<const u32x4_t*>(wr[t] + kb * kFp8Block + 64);
          ws[d][t] = wsr[t][kb];
        }
#pragma unroll
        for (int j = 0; j < kMT; ++j) {
          b[d][j][0] = *reinterpret_cast<const u32x4_t*>(xr[j] + kb * kFp8Block);
          b[d][j][1] = *reinterpret_cast<const u32x4_t*>(xr[j] + kb * kFp8Block + 64);
          xs[d][j] = xsr[j][kb * xs_b];
        }
      };
#pragma unroll
      for (int i = 0; i < kDepth; ++i) load(i);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int i = 0; i < kCnt; ++i) {
        const int d = i % kDepth;
        Operand16 A[kTiles];
#pragma unroll
        for (int t = 0; t < kTiles; ++t) A[t].set(a[d][t][0], a[d][t][1]);
#pragma unroll
        for (int j = 0; j < kMT; ++j) {
          Operand16 B;
          B.set(b[d][j][0], b[d][j][1]);
#pragma unroll
          for (int t = 0; t < kTiles; ++t) add_scaled(acc[t][j], block_sum(A[t], B), xs[d][j] * ws[d][t]);
        }
        if (i + kDepth < kCnt) load(i + kDepth);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  }
};

// The quantised output of one block of 128 gated values for rows [m0, m1): by the
// workgroup that arrives last there.
__device__ __forceinline__ void quantise_act(const LinearArgs& p, int jb, int m0, int m1) {
  const int q = threadIdx.x & 15;
  for (int m = m0 + (threadIdx.x >> 4); m < m1; m += blockDim.x >> 4) {
    const unsigned long long* src =
        reinterpret_cast<const unsigned long long*>(p.act + (static_cast<int64_t>(jb) * p.M + m) * kFp8Block + 8 * q);
    float y[8];
    uint32_t amax = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const unsigned long long v = __hip_atomic_load(src + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      y[2 * i] = __uint_as_float(static_cast<uint32_t>(v));
      y[2 * i + 1] = __uint_as_float(static_cast<uint32_t>(v >> 32));
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (jb * kFp8Block + 8 * q + i >= p.N) y[i] = 0.0f;
      amax = max(amax, abs_bits(y[i]));
    }
    const float s = fp8_scale(row_max(amax)), r = 1.0f / s;
    *reinterpret_cast<u32x2_t*>(p.codes + m * p.codes_ld + jb * kFp8Block + 8 * q) =
        u32x2_t{fp8_codes4(y, s, r), fp8_codes4(y + 4, s, r)};
    if (q == 0) p.scales[m * p.s_m + jb * p.s_b] = s;
  }
}

template <bool kGated, int kMT, int kCnt>
__global__ __launch_bounds__(1024) void fp8_stream_kernel(const LinearArgs p, int R) {
  constexpr int kTiles = kGated ? 2 : 1;
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  float4_t* red = reinterpret_cast<float4_t*>(lds);  // [wave][tile][x rows][lane]
  const int nw = blockDim.x >> 6;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int c = lane & 15, g = lane >> 4;
  const int n0 = blockIdx.x * R, m0 = blockIdx.y * 16 * kMT;
  const int row = min(n0 + min(c, R - 1), p.N - 1);
  const uint8_t *wr[kTiles], *xr[kMT];
  const float *wsr[kTiles], *xsr[kMT];
#pragma unroll
  for (int t = 0; t < kTiles; ++t) {
    wr[t] = p.w + (static_cast<int64_t>(t) * p.N + row) * p.w_ld + 16 * g;
    // (R divides 128: a unit lies in one block of rows)
    wsr[t] = p.ws + static_cast<int64_t>(t * ((p.N + kFp8Block - 1) / kFp8Block) + n0 / kFp8Block) * p.nkb;
  }
#pragma unroll
  for (int j = 0; j < kMT; ++j) {
    const int m = min(m0 + 16 * j + c, p.M - 1);
    xr[j] = p.x + m * p.x_ld + 16 * g;
    xsr[j] = p.xs + m * p.xs_m;
  }
  // a wave's blocks are all there but for the last: one without it takes a
  // straight line of its own
  const bool full = wave + (kCnt - 1) * nw < p.nkb;
  StreamWave<kTiles, kMT> s;
  if (full) {
    asm volatile("; all blocks");
    s.template run<kCnt>(wr, wsr, xr, xsr, p.xs_b, wave, nw);
  } else {
    asm volatile("; one fewer");
    s.template run<kCnt - 1>(wr, wsr, xr, xsr, p.xs_b, wave, nw);
  }
#pragma unroll
  for (int t = 0; t < kTiles; ++t)
#pragma unroll
    for (int j = 0; j < kMT; ++j) red[((wave * kTiles + t) * kMT + j) * 64 + lane] = s.acc[t][j];
  __syncthreads();
  // lane (c, g) holds rows 4 g + i of the unit for row c of x
  for (int j = wave; j < kMT; j += nw) {
    float4_t v[kTiles];
#pragma unroll
    for (int t = 0; t < kTiles; ++t) {
      v[t] = red[(t * kMT + j) * 64 + lane];
      for (int w = 1; w < nw; ++w) v[t] += red[((w * kTiles + t) * kMT + j) * 64 + lane];
    }
    const int m = m0 + 16 * j + c;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = 4 * g + i, n = n0 + r;
      if (m >= p.M || r >= R || n >= p.N) continue;
      if constexpr (kGated)
        __hip_atomic_store(p.act + (static_cast<int64_t>(n / kFp8Block) * p.M + m) * kFp8Block + n % kFp8Block,
                           silu_mul(v[0][i], v[kTiles - 1][i]), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      else
        store_out(p, m, n, v[0][i]);
    }
  }
  if constexpr (kGated) {
    // the units of a block of 128 outputs: the last one quantises it.  Values go
    // out and come back past the L2s, which the XCDs do not share; each lane's
    // stores have been acknowledged before the workgroup counts itself in
    __shared__ bool last;
    const int jb = n0 / kFp8Block;
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (threadIdx.x == 0)
      last = arrive_last(p.slots + static_cast<int64_t>(jb) * gridDim.y + blockIdx.y, p.epoch,
                         (min(kFp8Block, p.N - jb * kFp8Block) + R - 1) / R);
    __syncthreads();
    if (last) quantise_act(p, jb, m0, min(p.M, m0 + 16 * kMT));
  }
}

template <bool kGated>
int launch_stream(const LinearArgs& p, hipStream_t s) {
  constexpr int kMT = 1;
  const int R = 8;
  const int cnt = std::max(std::min(8, (p.nkb + 7) / 8), (p.nkb + 15) / 16);
  const int nw = (p.nkb + cnt - 1) / cnt;
  const dim3 grid((p.N + R - 1) / R, (p.M + 16 * kMT - 1) / (16 * kMT));
  const size_t lds = static_cast<size_t>(nw) * (kGated ? 2 : 1) * kMT * 1024;
#define ZKV_CNT(C)                                                         \
  case C:                                                                  \
    fp8_stream_kernel<kGated, kMT, C><<<grid, 64 * nw, lds, s>>>(p, R);    \
    break;
  switch (cnt) {
    ZKV_CNT(1) ZKV_CNT(2) ZKV_CNT(3) ZKV_CNT(4) ZKV_CNT(5) ZKV_CNT(6) ZKV_CNT(7) ZKV_CNT(8)
    default:
      return fail(ZKV_EINVAL, "fp8 linear: %d blocks per wave", cnt);
  }
#undef ZKV_CNT
  return check_launch("fp8_stream_kernel");
}

// ---------------------------------------------------------------------------
// Many rows of x: a workgroup of kWN x kWM waves computes 64 kWN weight rows (gated: 32
// kWN gate rows and the matching up rows) for 64 kWM rows of x, a wave 64 x 64 of
// it as 2 x 2 products of 32 x 32.  A block of 128 k of the tile's rows goes from
// memory straight into one of two LDS stages while the other is computed on.
//
// LDS: a row is 8 chunks of 16 bytes, chunk c in slot c ^ ((row >> 1) & 7): the 16
// lanes of a read phase, each with the same chunk of its own row, hit every bank
// once.  A lane converts its codes after reading them (64 conversions per wave, block
// and 32 rows): the LDS moves bytes, not bf16.
// ---------------------------------------------------------------------------
typedef float float16_t __attribute__((ext_vector_type(16)));

__device__ __forceinline__ uint32_t lds_offset(const void* p) {
  return static_cast<uint32_t>(reinterpret_cast<uintptr_t>((const lds_void_t*)(p)));
}

// 64 lanes x 16 bytes, each at its offset from a base (wave-uniform, as dst), into LDS at dst + 16 lane, not seen by the
// compiler's wait counts: with the builtin every LDS read waits for all of them.
__device__ __forceinline__ void dma16_tile(const void* base, uint32_t off, uint32_t dst) {
  asm volatile("global_load_lds_dwordx4 %0, %1" : : "v"(off), "s"(base), "{m0}"(dst) : "memory");
}

__device__ __forceinline__ void dma4_tile(const void* src, uint32_t dst) {
  asm volatile("global_load_lds_dword %0, off" : : "v"(src), "{m0}"(dst) : "memory");
}

// 8 codes as an operand.
__device__ __forceinline__ bf16x8_t codes8_to_bf16(uint32_t c0, uint32_t c1) {
  u32x4_t a;
#define ZKV_PAIR(w, half) __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, half))
  a[0] = ZKV_PAIR(c0, false), a[1] = ZKV_PAIR(c0, true);
  a[2] = ZKV_PAIR(c1, false), a[3] = ZKV_PAIR(c1, true);
#undef ZKV_PAIR
  return __builtin_bit_cast(bf16x8_t, a);
}

__device__ __forceinline__ void add_scaled(float16_t& acc, const float16_t& v, float s) {
#pragma unroll
  for (int i = 0; i < 16; ++i) acc[i] = __builtin_fmaf(v[i], s, acc[i]);
}

// Four neighbouring columns of a row of the output.
__device__ __forceinline__ void store_out4(const LinearArgs& p, int m, int n, const float (&y)[4], bool vec) {
  if (!vec || n + 4 > p.N) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (n + i < p.N) store_out(p, m, n + i, y[i]);
    return;
  }
  const int64_t o = m * p.out_ld + n, r = m * p.res_ld + n;
  if (p.type == kRowF32) {
    float4_t v = {y[0], y[1], y[2], y[3]};
    if (p.res) v += *reinterpret_cast<const float4_t*>(static_cast<const float*>(p.res) + r);
    *reinterpret_cast<float4_t*>(static_cast<float*>(p.out) + o) = v;
  } else {
    float v[4] = {y[0], y[1], y[2], y[3]};
    const bool bf = p.type == kRowBf16;
    if (p.res) {
      const u32x2_t h = *reinterpret_cast<const u32x2_t*>(static_cast<const uint16_t*>(p.res) + r);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t e = i & 1 ? h[i >> 1] >> 16 : h[i >> 1] & 0xFFFFu;
        v[i] += bf ? elem_to_f32<kBf16>(e) : elem_to_f32<kF16>(e);
      }
    }
    u32x2_t q;
#pragma unroll
    for (int i = 0; i < 2; ++i)
      q[i] = bf ? f32_to_elem<kBf16>(v[2 * i]) | (f32_to_elem<kBf16>(v[2 * i + 1]) << 16)
                : f32_to_elem<kF16>(v[2 * i]) | (f32_to_elem<kF16>(v[2 * i + 1]) << 16);
    *reinterpret_cast<u32x2_t*>(static_cast<uint16_t*>(p.out) + o) = q;
  }
}

constexpr int kStages = 3;

template <bool kGated, int kWN, int kWM>
struct TileShape {
  static constexpr int kRowsN = 64 * kWN, kRowsM = 64 * kWM;
  static constexpr int kCols = kGated ? kRowsN / 2 : kRowsN;  // output columns
  static constexpr int kStage = (kRowsN + kRowsM) * kFp8Block;
};

template <bool kGated, int kWN, int kWM>
__global__ __launch_bounds__(64 * kWN * kWM, 2) void fp8_tile_kernel(const LinearArgs p, int tiles_n, int tiles_m,
                                                                    int vec) {
  using Shape = TileShape<kGated, kWN, kWM>;
  constexpr int kWaves = kWN * kWM;
  constexpr int kDmas = Shape::kStage / 1024 / kWaves;  // per wave and block
  static_assert(Shape::kStage % (1024 * kWaves) == 0, "whole DMAs");
  __shared__ __attribute__((aligned(1024))) uint8_t lds[kStages * (Shape::kStage + 256 * (kWM + 1))];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int r = lane & 31, h = lane >> 5;
  const int wn = wave % kWN, wm = wave / kWN;

  // Workgroups go to the eight XCDs in turn: each takes a run of tiles, in bands of
  // four tiles of weight rows, so that those at work at one time share rows in its L2
  const int T = tiles_n * tiles_m, per = (T + 7) / 8;
  const int t = static_cast<int>(blockIdx.x & 7) * per + static_cast<int>(blockIdx.x >> 3);
  if (t >= T || static_cast<int>(blockIdx.x >> 3) >= per) return;
  const int band = t / (4 * tiles_m), in_band = t - band * 4 * tiles_m, width = min(4, tiles_n - 4 * band);
  const int tn = 4 * band + in_band % width, tm = in_band / width;
  const int n0 = tn * Shape::kCols, m0 = tm * Shape::kRowsM;

  // where the DMAs read: eight rows of 128 bytes each, slots permuted, at a lane's
  // offset from a row of the wave's (host side: rows at most 8 MiB apart)
  const uint8_t* src[kDmas];
  uint32_t off[kDmas];
#pragma unroll
  for (int i = 0; i < kDmas; ++i) {
    const int top = 8 * (wave * kDmas + i), row = top + (lane >> 3);
    const uint32_t chunk = (lane & 7) ^ ((row >> 1) & 7);
    if (top >= Shape::kRowsN) {
      src[i] = p.x + m0 * p.x_ld;
      off[i] = min(row - Shape::kRowsN, p.M - 1 - m0) * static_cast<uint32_t>(p.x_ld) + 16 * chunk;
    } else if (kGated) {  // 32 gate rows and the 32 matching up rows in turn
      src[i] = p.w + (static_cast<int64_t>(n0) + (top & 32 ? p.N : 0)) * p.w_ld;
      off[i] = min((row >> 6) * 32 + (row & 31), p.N - 1 - n0) * static_cast<uint32_t>(p.w_ld) + 16 * chunk;
    } else {
      src[i] = p.w + n0 * p.w_ld;
      off[i] = min(row, p.N - 1 - n0) * static_cast<uint32_t>(p.w_ld) + 16 * chunk;
    }
  }
  const uint32_t dst = lds_offset(lds) + wave * kDmas * 1024;
  // scales of a block: of the tile's x rows, then of each wave row's weight rows (gated:
  // gate and up), 64 to a wave's DMA
  constexpr int kScaleWaves = kWM + 1;
  const float* scale_src;
  int64_t scale_step;
  {
    const int w = wave % kScaleWaves;
    if (w < kWM) {
      scale_src = p.xs + min(m0 + 64 * w + lane, p.M - 1) * p.xs_m;
      scale_step = p.xs_b;
    } else {
      const int nb = (p.N + kFp8Block - 1) / kFp8Block, part = lane & 1, group = (lane >> 1) % kWN;
      const int n = min(n0 + (kGated ? 32 : 64) * group, p.N - 1);
      scale_src = p.ws + static_cast<int64_t>((kGated ? part * nb : 0) + n / kFp8Block) * p.nkb;
      scale_step = 1;
    }
  }
  const uint32_t scale_dst = lds_offset(lds) + kStages * Shape::kStage + (wave % kScaleWaves) * 256;
  // the i-th DMA of the block that is requested next, into its stage; past the last
  // block they repeat it, which keeps the counts of what is in flight
  int req = 0, req_stage = 0;
  auto request = [&](int i) {
    const int step = req + 1 < p.nkb ? 1 : 0;
    if (i < kDmas) {
      dma16_tile(src[i], off[i], __builtin_amdgcn_readfirstlane(dst + req_stage * Shape::kStage + i * 1024));
      src[i] += step * kFp8Block;
    } else {
      dma4_tile(scale_src, __builtin_amdgcn_readfirstlane(scale_dst + req_stage * 256 * kScaleWaves));
      scale_src += step * scale_step;
      req += step;
      req_stage = req_stage + 1 == kStages ? 0 : req_stage + 1;
    }
  };

  // lane (r, h) reads chunks 4 h + t of its rows; pair t of a block is two slices of 16 k
  const uint32_t first = 16 * ((4 * h) ^ ((r >> 1) & 7));
  const uint8_t* rows_n = lds + (64 * wn + r) * kFp8Block;
  const uint8_t* rows_m = lds + (Shape::kRowsN + 64 * wm + r) * kFp8Block;
  u32x4_t raw[2][4];  // of two pairs: the rows of the weight's two products, then of x's
  auto read_codes = [&](int i, uint32_t at, int t) {
    raw[t & 1][i] =
        *reinterpret_cast<const u32x4_t*>((i < 2 ? rows_n : rows_m) + 32 * (i & 1) * kFp8Block + at + (first ^ (16 * t)));
  };
  bf16x8_t op[2][4];  // operands of two slices
  float16_t acc[2][2] = {}, part[2][2] = {};
  float xs[2] = {0.0f, 0.0f}, ws[2] = {0.0f, 0.0f};  // of the block whose sums are in `part`

  // a block's DMAs are spread over eight slices: those of block b from the fifth of
  // block b - 3, where its stage is free, to the fourth of b - 2
  constexpr int kPerSlice = (kDmas + 8) / 8, kHead = 4 * kPerSlice < kDmas + 1 ? 4 * kPerSlice : kDmas + 1;
#pragma unroll
  for (int k = 0; k < 3; ++k)
#pragma unroll
    for (int i = 0; i < (k < 2 ? kDmas + 1 : kHead); ++i) request(i);
  wait_vmcnt<kDmas + 1 + kHead>();
  __builtin_amdgcn_s_barrier();
#pragma unroll
  for (int t = 0; t < 2; ++t)
#pragma unroll
    for (int i = 0; i < 4; ++i) read_codes(i, 0, t);
#pragma unroll
  for (int i = 0; i < 4; ++i) op[0][i] = codes8_to_bf16(raw[0][i][0], raw[0][i][1]);
  int stage = 0;
  for (int kb = 0; kb < p.nkb; ++kb) {
    const int next = stage + 1 == kStages ? 0 : stage + 1;
#pragma unroll
    for (int q = 0; q < 8; ++q) {
      if (q == 4) {
        // the block's codes are in registers, the next one's have landed
        wait_vmcnt<kDmas + 1>();
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
      }
      // a wave behind the other of its SIMD goes first: alone, neither fills it
      if (q == 4) __builtin_amdgcn_s_setprio(3);
      if (q == 6) __builtin_amdgcn_s_setprio(2);
      if (q == 0) __builtin_amdgcn_s_setprio(1);
      if (q == 2) __builtin_amdgcn_s_setprio(0);
      __builtin_amdgcn_sched_barrier(0);
      // four products, and in their shadow the next slice's conversions, reads two
      // pairs ahead and a DMA
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const int i = t >> 1, j = t & 1;
        if (q == 0) {
          add_scaled(acc[i][j], part[i][j], xs[j] * ws[kGated ? i : 0]);
          asm volatile("" : "+v"(acc[i][j]));  // (here: left to itself the compiler moves the sums behind the loop's branches and copies `part`)
          part[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(op[0][i], op[0][2 + j], float16_t{}, 0, 0, 0);
        } else {
          part[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(op[q & 1][i], op[q & 1][2 + j], part[i][j], 0, 0, 0);
        }
        const u32x4_t c = raw[((q + 1) / 2) & 1][t];
        op[(q + 1) & 1][t] = q & 1 ? codes8_to_bf16(c[0], c[1]) : codes8_to_bf16(c[2], c[3]);
        if (q % 2 == 0) read_codes(t, (q < 4 ? stage : next) * Shape::kStage, (q / 2 + 2) & 3);
        if (t == 1) {
          const int n = (q + 4) % 8 * kPerSlice;  // of block kb + 3 from q = 4 on, else of kb + 2
#pragma unroll
          for (int k = n; k < n + kPerSlice && k <= kDmas; ++k) request(k);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
      if (q == 0) {
        const float* sc =
            reinterpret_cast<const float*>(lds + kStages * Shape::kStage + stage * 256 * kScaleWaves);
#pragma unroll
        for (int j = 0; j < 2; ++j) xs[j] = sc[64 * wm + 32 * j + r];
#pragma unroll
        for (int i = 0; i < (kGated ? 2 : 1); ++i) ws[i] = sc[64 * kWM + 2 * wn + i];
      }
    }
    stage = next;
  }
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j) add_scaled(acc[i][j], part[i][j], xs[j] * ws[kGated ? i : 0]);
  wait_vmcnt<0>();

  // lane (r, h) holds columns 8 q + 4 h + 0..3 of row r of each product
  if constexpr (!kGated) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int m = m0 + 64 * wm + 32 * j + r;
      if (m >= p.M) continue;
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const float y[4] = {acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
          store_out4(p, m, n0 + 64 * wn + 32 * i + 8 * q + 4 * h, y, vec);
        }
    }
  } else {
    // 128 columns, one block: its largest magnitudes meet in LDS, [wn][row]
    static_assert(Shape::kCols == kFp8Block, "one block of outputs");
    __syncthreads();
    uint32_t* amax = reinterpret_cast<uint32_t*>(lds);
    float y[2][16];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      uint32_t a = 0;
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int n = n0 + 32 * wn + 8 * (e >> 2) + 4 * h + (e & 3);
        y[j][e] = n < p.N ? silu_mul(acc[0][j][e], acc[1][j][e]) : 0.0f;
        a = max(a, abs_bits(y[j][e]));
      }
      a = max(a, static_cast<uint32_t>(__shfl_xor(static_cast<int>(a), 32)));
      if (h == 0) amax[wn * Shape::kRowsM + 64 * wm + 32 * j + r] = a;
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int row = 64 * wm + 32 * j + r, m = m0 + row;
      uint32_t a = amax[row];
#pragma unroll
      for (int w = 1; w < kWN; ++w) a = max(a, amax[w * Shape::kRowsM + row]);
      const float sc = fp8_scale(a), rc = 1.0f / sc;
      if (m >= p.M) continue;
#pragma unroll
      for (int q = 0; q < 4; ++q)
        *reinterpret_cast<uint32_t*>(p.codes + m * p.codes_ld + n0 + 32 * wn + 8 * q + 4 * h) =
            fp8_codes4(y[j] + 4 * q, sc, rc);
      if (wn == 0 && h == 0) p.scales[m * p.s_m + tn * p.s_b] = sc;
    }
  }
}

template <bool kGated, int kWN, int kWM>
int launch_tile(const LinearArgs& p, hipStream_t s) {
  using Shape = TileShape<kGated, kWN, kWM>;
  const int tiles_n = (p.N + Shape::kCols - 1) / Shape::kCols, tiles_m = (p.M + Shape::kRowsM - 1) / Shape::kRowsM;
  const int item = p.type == kRowF32 ? 4 : 2;
  const int vec = !kGated && reinterpret_cast<uintptr_t>(p.out) % (4 * item) == 0 && p.out_ld % 4 == 0 &&
                  (!p.res || (reinterpret_cast<uintptr_t>(p.res) % (4 * item) == 0 && p.res_ld % 4 == 0));
  const unsigned grid = (static_cast<unsigned>(tiles_n) * tiles_m + 7) / 8 * 8;
  fp8_tile_kernel<kGated, kWN, kWM><<<grid, 64 * kWN * kWM, 0, s>>>(p, tiles_n, tiles_m, vec);
  return check_launch("fp8_tile_kernel");
}

int blocks_of(int n) { return (n + kFp8Block - 1) / kFp8Block; }

// Checks what both entry points take; null or what is wrong.
const char* check_operands(const uint8_t* x, int64_t x_ld, const float* xs, const uint8_t* w, int64_t w_ld,
                           const float* ws, int M, int N, int K) {
  if (!x || !xs || !w || !ws) return "null pointer";
  if (M < 1 || N < 1 || K < 1) return "empty product";
  if (K % kFp8Block || K > 128 * kFp8Block) return "K is a multiple of 128, at most 16384";
  if (x_ld < K || w_ld < K || !rows_on_16(x, x_ld, 1) || !rows_on_16(w, w_ld, 1))
    return "rows of codes hold K bytes and start on 16";
  return nullptr;
}

}  // namespace
}  // namespace zkv

using namespace zkv;

extern "C" int zkv_fp8_linear(const uint8_t* x, int64_t x_ld, const float* xs, int64_t xs_m, int64_t xs_b,
                              const uint8_t* w, int64_t w_ld, const float* ws, int M, int N, int K,
                              const void* residual, int64_t res_ld, void* out, int64_t out_ld, int type,
                              zkv_stream_t stream) {
  const char* bad = check_operands(x, x_ld, xs, w, w_ld, ws, M, N, K);
  ZKV_REQUIRE(!bad, "zkv_fp8_linear: %s (M=%d N=%d K=%d)", bad, M, N, K);
  ZKV_REQUIRE(out && type >= kRowBf16 && type <= kRowF32, "zkv_fp8_linear: bad output");
  LinearArgs p{};
  p.x = x, p.x_ld = x_ld, p.xs = xs, p.xs_m = xs_m, p.xs_b = xs_b, p.w = w, p.w_ld = w_ld, p.ws = ws;
  p.M = M, p.N = N, p.nkb = K / kFp8Block;
  p.res = residual, p.res_ld = res_ld, p.out = out, p.out_ld = out_ld, p.type = type;
  auto s = reinterpret_cast<hipStream_t>(stream);
  if (M <= 64) return launch_stream<false>(p, s);
  return launch_tile<false, 4, 2>(p, s);
}

extern "C" size_t zkv_fp8_gated_workspace_size(int M, int F) {
  if (M < 1 || F < 1) return 0;
  const size_t nb = blocks_of(F);
  return (nb * ((M + 15) / 16) * 8 + 255) / 256 * 256 + nb * M * kFp8Block * 4;
}

extern "C" int zkv_fp8_gated_linear(const uint8_t* x, int64_t x_ld, const float* xs, int64_t xs_m, int64_t xs_b,
                                    const uint8_t* w, int64_t w_ld, const float* ws, int M, int F, int K,
                                    uint8_t* codes, int64_t codes_ld, float* scales, int64_t s_m, int64_t s_b,
                                    void* workspace, size_t workspace_bytes, zkv_stream_t stream) {
  const char* bad = check_operands(x, x_ld, xs, w, w_ld, ws, M, F, K);
  ZKV_REQUIRE(!bad, "zkv_fp8_gated_linear: %s (M=%d F=%d K=%d)", bad, M, F, K);
  ZKV_REQUIRE(codes && scales && codes_ld >= static_cast<int64_t>(blocks_of(F)) * kFp8Block && codes_ld % 8 == 0 &&
                  (reinterpret_cast<uintptr_t>(codes) & 7) == 0,
              "zkv_fp8_gated_linear: rows of codes hold whole blocks of 128 and start on 8 bytes");
  const size_t need = zkv_fp8_gated_workspace_size(M, F);
  if (workspace_bytes < need || (need && !workspace) || (reinterpret_cast<uintptr_t>(workspace) & 15))
    return fail(ZKV_ESPACE, "zkv_fp8_gated_linear: %zu bytes of workspace on 16 bytes, %zu needed", workspace_bytes,
                need);
  LinearArgs p{};
  p.x = x, p.x_ld = x_ld, p.xs = xs, p.xs_m = xs_m, p.xs_b = xs_b, p.w = w, p.w_ld = w_ld, p.ws = ws;
  p.M = M, p.N = F, p.nkb = K / kFp8Block;
  p.codes = codes, p.codes_ld = codes_ld, p.scales = scales, p.s_m = s_m, p.s_b = s_b;
  p.slots = static_cast<unsigned long long*>(workspace);
  p.act = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) +
                                   (static_cast<size_t>(blocks_of(F)) * ((M + 15) / 16) * 8 + 255) / 256 * 256);
  p.epoch = next_epoch();
  auto s = reinterpret_cast<hipStream_t>(stream);
  if (M <= 64) return launch_stream<true>(p, s);
  return launch_tile<true, 4, 2>(p, s);
}
