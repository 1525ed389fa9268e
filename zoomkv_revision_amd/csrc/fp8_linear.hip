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
  // sums that a second launch goes on with: [part, split][M][sums_ld], the blocks of k
  // in `splits` runs (null: the output is final)
  float* sums;
  int64_t sums_ld;
  int splits;
};

// The part of the weight and the run of blocks [first, last) of a workgroup.
struct Piece {
  int part, first, last;
};
__device__ __forceinline__ Piece piece_of(const LinearArgs& p, int z) {
  const int part = z / p.splits, split = z - part * p.splits;
  return Piece{part, split * p.nkb / p.splits, (split + 1) * p.nkb / p.splits};
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

// Outputs 8 l + 0..7 of block jb of row m, from each of 16 neighbouring lanes.
__device__ __forceinline__ void put_gated(const LinearArgs& p, int m, int jb, int l, const float (&y)[8]) {
  uint32_t a = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) a = max(a, abs_bits(y[i]));
  const float s = fp8_scale(row_max(a)), r = 1.0f / s;
  *reinterpret_cast<u32x2_t*>(p.codes + m * p.codes_ld + jb * kFp8Block + 8 * l) =
      u32x2_t{fp8_codes4(y, s, r), fp8_codes4(y + 4, s, r)};
  if (l == 0) p.scales[m * p.s_m + jb * p.s_b] = s;
}

// Four neighbouring columns of a row of the residual, as they are stored.
__device__ __forceinline__ u32x4_t load_res4(const LinearArgs& p, int m, int n) {
  const int64_t r = m * p.res_ld + n;
  if (p.type == kRowF32) return *reinterpret_cast<const u32x4_any*>(static_cast<const float*>(p.res) + r);
  const u32x2_any h = *reinterpret_cast<const u32x2_any*>(static_cast<const uint16_t*>(p.res) + r);
  return u32x4_t{h[0], h[1], 0, 0};
}

// Four columns of the output, all of them in it; res where there is a residual.
__device__ __forceinline__ void store_whole4(const LinearArgs& p, int m, int n, const float (&y)[4], u32x4_t res) {
  const int64_t o = m * p.out_ld + n;
  if (p.type == kRowF32) {
    u32x4_t v;
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = __float_as_uint(p.res ? y[i] + __uint_as_float(res[i]) : y[i]);
    *reinterpret_cast<u32x4_any*>(static_cast<float*>(p.out) + o) = v;
  } else {
    float v[4] = {y[0], y[1], y[2], y[3]};
    const bool bf = p.type == kRowBf16;
    if (p.res) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t e = i & 1 ? res[i >> 1] >> 16 : res[i >> 1] & 0xFFFFu;
        v[i] += bf ? elem_to_f32<kBf16>(e) : elem_to_f32<kF16>(e);
      }
    }
    u32x2_t q;
#pragma unroll
    for (int i = 0; i < 2; ++i)
      q[i] = bf ? f32_to_elem<kBf16>(v[2 * i]) | (f32_to_elem<kBf16>(v[2 * i + 1]) << 16)
                : f32_to_elem<kF16>(v[2 * i]) | (f32_to_elem<kF16>(v[2 * i + 1]) << 16);
    *reinterpret_cast<u32x2_any*>(static_cast<uint16_t*>(p.out) + o) = q;
  }
}

// Four columns of the output, or of the sums that a second launch goes on with.
__device__ __forceinline__ void store_out4(const LinearArgs& p, int z, int m, int n, const float (&y)[4]) {
  if (p.sums) {  // (rows of whole groups of four)
    if (n < p.N)
      *reinterpret_cast<float4_t*>(p.sums + (static_cast<int64_t>(z) * p.M + m) * p.sums_ld + n) =
          float4_t{y[0], y[1], y[2], y[3]};
  } else if (n + 4 > p.N) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (n + i < p.N) store_out(p, m, n + i, y[i]);
  } else {
    store_whole4(p, m, n, y, p.res ? load_res4(p, m, n) : u32x4_t{});
  }
}

// ---------------------------------------------------------------------------
// What the LDS kernels share.  A row of a block of k is 128 bytes there, 8 chunks of 16,
// chunk c in slot c ^ ((row >> 1) & 7): the 16 lanes of a read phase, each with the
// same chunk of its own row, hit every bank once.
// ---------------------------------------------------------------------------
__device__ __forceinline__ uint32_t lds_offset(const void* p) {
  return static_cast<uint32_t>(reinterpret_cast<uintptr_t>((const lds_void_t*)(p)));
}

// 64 lanes x 16 bytes, each at its offset from a base (wave-uniform, as dst), into LDS at
// dst + 16 lane, not seen by the compiler's wait counts: with the builtin every LDS read
// waits for all of them.
__device__ __forceinline__ void dma16_tile(const void* base, uint32_t off, uint32_t dst) {
  asm volatile("global_load_lds_dwordx4 %0, %1" : : "v"(off), "s"(base), "{m0}"(dst) : "memory");
}

__device__ __forceinline__ void dma4_tile(const void* src, uint32_t dst) {
  asm volatile("global_load_lds_dword %0, off" : : "v"(src), "{m0}"(dst) : "memory");
}

// ---------------------------------------------------------------------------
// Few rows of x, or few tiles: a unit computes 16 kNT weight rows for kXR rows of x (8,
// or 16 kMT); its waves split the blocks of k (wave w takes blocks w, w + nw, ...), so
// no wave waits for another, and their sums meet at the end, added in wave order.  Each
// wave has kD blocks on their way into its own part of the LDS, eight whole lines to
// a load: straight into the registers of a product's operands, a load's neighbouring
// lanes are in different rows, which the address unit takes one by one, and at 64
// cycles a load it was what bounded the kernel (16 x 2560 x 9728 12.7 -> 10.4 us, 100 x
// 1000 x 2600 8.4 -> 6.1, gated 4 x 9728 x 2560 16.0 -> 14.5 with its second launch).
// A unit may have R < 16 weight rows per tile, to fill the CUs: lanes past R, N or M
// repeat the last row, which moves no more memory.
// ---------------------------------------------------------------------------
template <int kNT, int kXR, int kWaves, int kD>
__global__ __launch_bounds__(64 * kWaves) void fp8_stream_kernel(const LinearArgs p, int R) {
  constexpr int kMT = (kXR + 15) / 16, kDmas = (16 * kNT + kXR) / 8;
  constexpr int kRegion = kDmas * 1024 + 256;  // a block: rows of the weight, rows of x, scales
  static_assert(kXR + 4 * kNT <= 64 && kD >= 2 && kD <= 3 && kNT * kMT * 1024 <= kD * kRegion, "");
  __shared__ __attribute__((aligned(1024))) uint8_t lds[kWaves * kD * kRegion];
  const int nw = blockDim.x >> 6;
  // (turned from unit to unit, so that those at work at one time do not all ask for the
  // same part of x first: 1 x 6144 x 2560 6.37 -> 6.20 us, 16 x 6144 x 2560 8.59 -> 8.35)
  const int wave = __builtin_amdgcn_readfirstlane(((threadIdx.x >> 6) + blockIdx.x) % nw), lane = threadIdx.x & 63;
  const int c = lane & 15, g = lane >> 4;
  const int n0 = blockIdx.x * R * kNT, m0 = blockIdx.y * 16 * kMT;
  const Piece piece = piece_of(p, blockIdx.z);

  // where the loads read (host side: rows at most 8 MiB apart)
  const int first = piece.first + wave;
  const uint8_t* wb = p.w + (static_cast<int64_t>(piece.part) * p.N + n0) * p.w_ld + first * kFp8Block;
  const uint8_t* xb = p.x + m0 * p.x_ld + first * kFp8Block;
  uint32_t off[kDmas];
#pragma unroll
  for (int i = 0; i < kDmas; ++i) {
    const int row = 8 * i + (lane >> 3);
    const uint32_t chunk = 16 * ((lane & 7) ^ ((row >> 1) & 7));
    if (i < 2 * kNT)
      off[i] = min(row / 16 * R + min(row % 16, R - 1), p.N - 1 - n0) * static_cast<uint32_t>(p.w_ld) + chunk;
    else
      off[i] = min(row - 16 * kNT, p.M - 1 - m0) * static_cast<uint32_t>(p.x_ld) + chunk;
  }
  // scales: of the rows of x, then of each four columns of the weight's tiles (in one block
  // each: R is a multiple of 4)
  const float* sb;
  int64_t s_step;
  if (lane < kXR) {
    sb = p.xs + min(m0 + lane, p.M - 1) * p.xs_m + first * p.xs_b;
    s_step = nw * p.xs_b;
  } else {
    const int j = min(lane - kXR, 4 * kNT - 1);
    const int n = min(n0 + (j >> 2) * R + min(4 * (j & 3), R - 4), p.N - 1);
    const int nb = (p.N + kFp8Block - 1) / kFp8Block;
    sb = p.ws + static_cast<int64_t>(piece.part * nb + n / kFp8Block) * p.nkb + first;
    s_step = nw;
  }
  uint8_t* const mine = lds + wave * kD * kRegion;
  const uint32_t dst = __builtin_amdgcn_readfirstlane(lds_offset(mine));
  auto request = [&](int stage) {
#pragma unroll
    for (int i = 0; i < kDmas; ++i) dma16_tile(i < 2 * kNT ? wb : xb, off[i], dst + stage * kRegion + i * 1024);
    dma4_tile(sb, dst + stage * kRegion + kDmas * 1024);
    wb += nw * kFp8Block, xb += nw * kFp8Block, sb += s_step;
  };

  const int cnt = (piece.last - first + nw - 1) / nw;  // (0 for the last wave of a shorter run of k)
#pragma unroll
  for (int d = 0; d < kD; ++d)
    if (d < cnt) request(d);
  const uint32_t at = c * kFp8Block + 16 * (g ^ ((c >> 1) & 7));
  float4_t acc[kNT][kMT] = {};
  int stage = 0;
  for (int i = 0; i < cnt; ++i) {
    const int left = cnt - 1 - i;  // behind this block, min(left, kD - 1) of them requested
    if (left >= kD - 1)
      wait_vmcnt<(kD - 1) * (kDmas + 1)>();
    else if (kD > 2 && left == 1)
      wait_vmcnt<kDmas + 1>();
    else
      wait_vmcnt<0>();
    // (to the compiler neither the wait nor the DMAs' arrival touches memory: the reads stay
    // behind it)
    asm volatile("" ::: "memory");
    const uint8_t* src = mine + stage * kRegion;
    u32x4_t a[kNT][2], b[kMT][2];
    float ws[kNT], xs[kMT];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int t = 0; t < kNT; ++t) a[t][h] = *reinterpret_cast<const u32x4_t*>(src + t * 2048 + (at ^ (64 * h)));
#pragma unroll
      for (int t = 0; t < kMT; ++t)
        b[t][h] = *reinterpret_cast<const u32x4_t*>(src + (kNT + t) * 2048 + ((kXR < 16 ? at & ~1024u : at) ^ (64 * h)));
    }
    const float* sc = reinterpret_cast<const float*>(src + kDmas * 1024);
#pragma unroll
    for (int t = 0; t < kNT; ++t) ws[t] = sc[kXR + 4 * t + g];
#pragma unroll
    for (int t = 0; t < kMT; ++t) xs[t] = sc[16 * t + (kXR < 16 ? c & 7 : c)];
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    if (left >= kD) request(stage);
    stage = stage + 1 == kD ? 0 : stage + 1;
    float4_t part[kNT][kMT];
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        bf16x8_t A[kNT], B[kMT];
#pragma unroll
        for (int t = 0; t < kNT; ++t) A[t] = codes8_to_bf16(a[t][h][2 * q], a[t][h][2 * q + 1]);
#pragma unroll
        for (int t = 0; t < kMT; ++t) B[t] = codes8_to_bf16(b[t][h][2 * q], b[t][h][2 * q + 1]);
#pragma unroll
        for (int t = 0; t < kNT; ++t)
#pragma unroll
          for (int j = 0; j < kMT; ++j)
            part[t][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                A[t], B[j], h + q ? part[t][j] : float4_t{0.0f, 0.0f, 0.0f, 0.0f}, 0, 0, 0);
      }
#pragma unroll
    for (int t = 0; t < kNT; ++t)
#pragma unroll
      for (int j = 0; j < kMT; ++j) add_scaled(acc[t][j], part[t][j], xs[j] * ws[t]);
  }
  // nothing is on its way into this wave's part any more: [weight tile][x tile][lane]
  float4_t* red = reinterpret_cast<float4_t*>(lds);
  constexpr int kStep = kD * kRegion / 16;
#pragma unroll
  for (int t = 0; t < kNT; ++t)
#pragma unroll
    for (int j = 0; j < kMT; ++j) red[wave * kStep + (t * kMT + j) * 64 + lane] = acc[t][j];
  __syncthreads();
  // lane (c, g) holds columns 4 g + 0..3 of a tile for row c of x
  for (int t = wave; t < kNT * kMT; t += nw) {
    const float4_t* src = red + t * 64 + lane;
    float4_t v = src[0];
    for (int k = 1; k < nw; ++k) v += src[k * kStep];
    const int m = m0 + 16 * (t % kMT) + c, n = n0 + t / kMT * R + 4 * g;
    if (m >= p.M || 4 * g >= R) continue;
    const float y[4] = {v[0], v[1], v[2], v[3]};
    store_out4(p, blockIdx.z, m, n, y);
  }
}

// Units of up to 16 weight rows: eight waves where k is long (4 x 2560 x 4096 5.9 us with
// four, 5.3 with eight; 4 x 6144 x 2560 6.2 and 6.6), and so many weight rows that the
// number of units is rounded up to whole rounds of 256 CUs (4 x 2560 x 9728, 12 rows each
// 8.15 us, 16 rows 8.6, 8 rows 10.8).
int stream_waves(int nkb) { return nkb > 26 ? 8 : std::min(nkb, 4); }

int stream_rows(int N, int parts) {
  const int units = ((N + 15) / 16 * parts + 255) / 256 * 256 / parts;
  return std::min(16, ((N + units - 1) / units + 3) / 4 * 4);
}

template <int kXR>
int launch_stream(const LinearArgs& p, int parts, hipStream_t s) {
  const int nw = stream_waves((p.nkb + p.splits - 1) / p.splits), R = stream_rows(p.N, parts);
  const dim3 grid((p.N + R - 1) / R, (p.M + kXR - 1) / kXR, parts * p.splits);
  if (nw > 4)
    fp8_stream_kernel<1, kXR, 8, kXR == 8 ? 3 : 2><<<grid, 64 * nw, 0, s>>>(p, R);
  else
    fp8_stream_kernel<1, kXR, 4, 2><<<grid, 64 * nw, 0, s>>>(p, R);
  return check_launch("fp8_stream_kernel");
}

// 32 weight rows and 32 rows of x per workgroup.
int launch_split(const LinearArgs& p, int parts, hipStream_t s) {
  const int nw = std::min((p.nkb + p.splits - 1) / p.splits, 4);
  const dim3 grid((p.N + 31) / 32, (p.M + 31) / 32, parts * p.splits);
  fp8_stream_kernel<2, 32, 4, 2><<<grid, 64 * nw, 0, s>>>(p, 16);
  return check_launch("fp8_stream_kernel");
}

// ---------------------------------------------------------------------------
// The second launch where the first left sums: the splits added in order, then the
// output's residual and rounding, or silu(gate) * up as codes.
// ---------------------------------------------------------------------------
template <int kSplits>
__device__ __forceinline__ float4_t sum_of(const LinearArgs& p, int part, int m, int n) {
  const float* src = p.sums + (static_cast<int64_t>(part) * kSplits * p.M + m) * p.sums_ld + n;
  float4_t v[kSplits];  // (requested together)
#pragma unroll
  for (int k = 0; k < kSplits; ++k) v[k] = *reinterpret_cast<const float4_t*>(src + k * p.M * p.sums_ld);
#pragma unroll
  for (int k = 1; k < kSplits; ++k) v[0] += v[k];
  return v[0];
}

template <int kSplits>
__global__ __launch_bounds__(256) void fp8_join_kernel(const LinearArgs p) {
  const int n = 4 * (blockIdx.y * 256 + threadIdx.x), m = blockIdx.x;
  if (n >= p.N) return;
  const float4_t v = sum_of<kSplits>(p, 0, m, n);
  LinearArgs q = p;
  q.sums = nullptr;
  const float y[4] = {v[0], v[1], v[2], v[3]};
  store_out4(q, 0, m, n, y);
}

// 16 lanes per row and block of 128 outputs, 8 outputs each.
template <int kSplits>
__global__ __launch_bounds__(256) void fp8_gated_join_kernel(const LinearArgs p) {
  const int jb = blockIdx.y, m = blockIdx.x * 16 + (threadIdx.x >> 4), n = jb * kFp8Block + 8 * (threadIdx.x & 15);
  if (m >= p.M) return;  // (whole groups of 16 lanes)
  float y[8];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    float4_t g = {0.0f, 0.0f, 0.0f, 0.0f}, u = g;
    if (n + 4 * i < p.N) g = sum_of<kSplits>(p, 0, m, n + 4 * i), u = sum_of<kSplits>(p, 1, m, n + 4 * i);
#pragma unroll
    for (int e = 0; e < 4; ++e) y[4 * i + e] = n + 4 * i + e < p.N ? silu_mul(g[e], u[e]) : 0.0f;
  }
  put_gated(p, m, jb, threadIdx.x & 15, y);
}

constexpr int kMaxSplits = 8;

template <int kSplits>
void launch_join_of(const LinearArgs& p, bool gated, dim3 grid, hipStream_t s) {
  if (gated)
    fp8_gated_join_kernel<kSplits><<<grid, 256, 0, s>>>(p);
  else if constexpr (kSplits > 1)  // (a linear product leaves sums in two runs or more)
    fp8_join_kernel<kSplits><<<grid, 256, 0, s>>>(p);
}

int launch_join(const LinearArgs& p, bool gated, hipStream_t s) {
  const dim3 grid = gated ? dim3((p.M + 15) / 16, (p.N + kFp8Block - 1) / kFp8Block) : dim3(p.M, (p.N + 1023) / 1024);
  switch (p.splits) {
    case 1: launch_join_of<1>(p, gated, grid, s); break;
    case 2: launch_join_of<2>(p, gated, grid, s); break;
    case 3: launch_join_of<3>(p, gated, grid, s); break;
    case 4: launch_join_of<4>(p, gated, grid, s); break;
    case 5: launch_join_of<5>(p, gated, grid, s); break;
    case 6: launch_join_of<6>(p, gated, grid, s); break;
    case 7: launch_join_of<7>(p, gated, grid, s); break;
    case 8: launch_join_of<8>(p, gated, grid, s); break;
    default: return fail(ZKV_EINVAL, "fp8 linear: %d runs of k", p.splits);
  }
  return check_launch("fp8_join_kernel");
}

// ---------------------------------------------------------------------------
// Many rows of x: a workgroup of kWN x kWM waves, each with kI x kJ products of 32 x
// 32, computes 32 kI kWN weight rows (gated: half of them gate rows, half the matching up
// rows) for 32 kJ kWM rows of x.  A block of 128 k of the tile's rows goes from memory
// straight into one of three LDS stages, two blocks ahead of the one that is computed on.
// A lane converts its codes after reading them (8 instructions per 16 of them): the
// LDS moves bytes, not bf16.
//
//   tile of w x x  waves  products  workgroups on a CU
//     256 x 128      8     2 x 2           1   the fewest bytes and conversions per product
//     128 x 128      8     2 x 1           1
//     128 x 64       8     1 x 1           2   more of them run
//      64 x 64       4     1 x 1           3   at a time where there are few
//
// 8192^3 takes 860 us with the first (1278 TF, 857 at the rate of a bf16 product of the
// library), 512 x 6144 x 2560 33.6, 22.5, 24.8 and 23.6 with the four, 300 x 4096 x 4096
// 44.8, 29.2, 21.8 and 23.4.
// ---------------------------------------------------------------------------
typedef float float16_t __attribute__((ext_vector_type(16)));

__device__ __forceinline__ void add_scaled(float16_t& acc, const float16_t& v, float s) {
#pragma unroll
  for (int i = 0; i < 16; ++i) acc[i] = __builtin_fmaf(v[i], s, acc[i]);
}

// kWN x kWM waves of kI x kJ products of 32 x 32.
template <bool kGated, int kWN, int kWM, int kI, int kJ>
struct TileShape {
  static constexpr int kWaves = kWN * kWM;
  static constexpr int kRowsN = 32 * kI * kWN, kRowsM = 32 * kJ * kWM;
  static constexpr int kCols = kGated ? kRowsN / 2 : kRowsN;  // output columns
  static constexpr int kStage = (kRowsN + kRowsM) * kFp8Block;
  static constexpr int kDmas = kStage / 1024 / kWaves;  // per wave and block
  static constexpr int kScaleWaves = kRowsM / 64 + 1;
  static_assert(kStage % (1024 * kWaves) == 0 && kRowsM % 64 == 0 && kScaleWaves <= kWaves, "whole DMAs");
  static_assert(!kGated || (kI == 2 && kCols == kFp8Block), "gate and up, and one block of outputs");
};

// What every wave has requested by DMA, but for the last kLeft, is in the LDS for all
// of the workgroup, and what they read before has been read.
template <int kLeft>
__device__ __forceinline__ void tile_barrier() {
  wait_vmcnt<kLeft>();
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");  // (to the compiler the barrier touches no memory)
}

template <bool kGated, int kWN, int kWM, int kI, int kJ>
__global__ __launch_bounds__(64 * kWN * kWM, kI * kJ > 1 ? 2 : kWN * kWM > 4 ? 4 : 3) void fp8_tile_kernel(
    const LinearArgs p, int tiles_n, int tiles_m, int parts) {
  using Shape = TileShape<kGated, kWN, kWM, kI, kJ>;
  constexpr int kStages = 3, kDmas = Shape::kDmas, kScaleWaves = Shape::kScaleWaves;
  __shared__ __attribute__((aligned(1024))) uint8_t lds[kStages * (Shape::kStage + 256 * kScaleWaves)];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int r = lane & 31, h = lane >> 5;
  const int wn = wave % kWN, wm = wave / kWN;

  // Workgroups go to the eight XCDs in turn: each takes a run of the tiles of the first
  // run of k, then of the next, in bands of four tiles of weight rows, so that those
  // at work at one time share rows in its L2
  const int T = tiles_n * tiles_m, all = T * p.splits * parts, per = (all + 7) / 8;
  const int item = static_cast<int>(blockIdx.x & 7) * per + static_cast<int>(blockIdx.x >> 3);
  if (item >= all || static_cast<int>(blockIdx.x >> 3) >= per) return;
  const int z = item / T, t = item - z * T;
  const int band = t / (4 * tiles_m), in_band = t - band * 4 * tiles_m, width = min(4, tiles_n - 4 * band);
  const int tn = 4 * band + in_band % width, tm = in_band / width;
  const int n0 = tn * Shape::kCols, m0 = tm * Shape::kRowsM;
  const Piece piece = piece_of(p, z);

  // where the DMAs read: eight rows of 128 bytes each, slots permuted, at a lane's
  // offset from a row of the wave's (host side: rows at most 8 MiB apart)
  const uint8_t* src[kDmas];
  uint32_t off[kDmas];
#pragma unroll
  for (int i = 0; i < kDmas; ++i) {
    const int top = 8 * (wave * kDmas + i), row = top + (lane >> 3);
    const uint32_t chunk = (lane & 7) ^ ((row >> 1) & 7);
    if (top >= Shape::kRowsN) {
      src[i] = p.x + m0 * p.x_ld + piece.first * kFp8Block;
      off[i] = min(row - Shape::kRowsN, p.M - 1 - m0) * static_cast<uint32_t>(p.x_ld) + 16 * chunk;
    } else if (kGated) {  // 32 gate rows and the 32 matching up rows in turn
      src[i] = p.w + (static_cast<int64_t>(n0) + (top & 32 ? p.N : 0)) * p.w_ld + piece.first * kFp8Block;
      off[i] = min((row >> 6) * 32 + (row & 31), p.N - 1 - n0) * static_cast<uint32_t>(p.w_ld) + 16 * chunk;
    } else {
      src[i] = p.w + (static_cast<int64_t>(piece.part) * p.N + n0) * p.w_ld + piece.first * kFp8Block;
      off[i] = min(row, p.N - 1 - n0) * static_cast<uint32_t>(p.w_ld) + 16 * chunk;
    }
  }
  const uint32_t dst = lds_offset(lds) + wave * kDmas * 1024;
  // scales of a block: of the tile's x rows, then of each wave row's weight rows (gated:
  // gate and up), 64 to a wave's DMA
  const float* scale_src;
  int64_t scale_step;
  {
    const int w = wave % kScaleWaves;
    if (w < kScaleWaves - 1) {
      scale_src = p.xs + min(m0 + 64 * w + lane, p.M - 1) * p.xs_m + piece.first * p.xs_b;
      scale_step = p.xs_b;
    } else {
      const int nb = (p.N + kFp8Block - 1) / kFp8Block, part = kGated ? lane & 1 : piece.part;
      const int n = min(n0 + (kGated ? 32 : 32 * kI) * ((lane >> 1) % kWN), p.N - 1);
      scale_src = p.ws + static_cast<int64_t>(part * nb + n / kFp8Block) * p.nkb + piece.first;
      scale_step = 1;
    }
  }
  const uint32_t scale_dst = lds_offset(lds) + kStages * Shape::kStage + (wave % kScaleWaves) * 256;
  // the i-th DMA of the block that is requested next, into its stage; past the last
  // block they repeat it, which keeps the counts of what is in flight
  int req = piece.first, req_stage = 0;
  auto request = [&](int i) {
    const int step = req + 1 < piece.last ? 1 : 0;
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
  const uint8_t* rows_n = lds + (32 * kI * wn + r) * kFp8Block;
  const uint8_t* rows_m = lds + (Shape::kRowsN + 32 * kJ * wm + r) * kFp8Block;
  constexpr int kOps = kI + kJ;
  u32x4_t raw[2][kOps];  // of two pairs: the weight rows of the products, then x's
  auto read_codes = [&](int i, uint32_t at, int t) {
    raw[t & 1][i] = *reinterpret_cast<const u32x4_t*>((i < kI ? rows_n + 32 * i * kFp8Block
                                                              : rows_m + 32 * (i - kI) * kFp8Block) +
                                                      at + (first ^ (16 * t)));
  };
  bf16x8_t op[2][kOps];  // operands of two slices
  float16_t acc[kI][kJ] = {}, part[kI][kJ] = {};
  float xs[kJ] = {}, ws[2] = {0.0f, 0.0f};  // of the block whose sums are in `part`

  // A block's DMAs are spread over eight slices, those of block b from the fifth of
  // block b - kStages, where its stage is free, and have landed by the fifth of b - 1
  constexpr int kPerSlice = (kDmas + 8) / 8, kHead = 4 * kPerSlice < kDmas + 1 ? 4 * kPerSlice : kDmas + 1;
  constexpr int kLater = (kStages - 2) * (kDmas + 1);  // requested behind a block that has to be there
#pragma unroll
  for (int k = 0; k < kStages; ++k)
#pragma unroll
    for (int i = 0; i < (k < kStages - 1 ? kDmas + 1 : kHead); ++i) request(i);
  tile_barrier<kLater + kHead>();
#pragma unroll
  for (int t = 0; t < 2; ++t)
#pragma unroll
    for (int i = 0; i < kOps; ++i) read_codes(i, 0, t);
#pragma unroll
  for (int i = 0; i < kOps; ++i) op[0][i] = codes8_to_bf16(raw[0][i][0], raw[0][i][1]);
  int stage = 0;
  for (int kb = piece.first; kb < piece.last; ++kb) {
    const int next = stage + 1 == kStages ? 0 : stage + 1;
#pragma unroll
    for (int q = 0; q < 8; ++q) {
      // the block's codes are in registers, the next one's have landed
      if (q == 4) tile_barrier<kLater>();
      // a wave behind the other of its SIMD goes first: alone, neither fills it
      if (q == 4) __builtin_amdgcn_s_setprio(3);
      if (q == 6) __builtin_amdgcn_s_setprio(2);
      if (q == 0) __builtin_amdgcn_s_setprio(1);
      if (q == 2) __builtin_amdgcn_s_setprio(0);
      __builtin_amdgcn_sched_barrier(0);
      // the products, and in their shadow the next slice's conversions, reads two
      // pairs ahead and a DMA
#pragma unroll
      for (int t = 0; t < (kI * kJ > kOps ? kI * kJ : kOps); ++t) {
        if (t < kI * kJ) {
          const int i = t / kJ, j = t % kJ;
          if (q == 0) {
            add_scaled(acc[i][j], part[i][j], xs[j] * ws[kGated ? i : 0]);
            // (here: left to itself the compiler moves the sums behind the loop's branches
            // and copies `part`)
            asm volatile("" : "+v"(acc[i][j]));
            part[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(op[0][i], op[0][kI + j], float16_t{}, 0, 0, 0);
          } else {
            part[i][j] =
                __builtin_amdgcn_mfma_f32_32x32x16_bf16(op[q & 1][i], op[q & 1][kI + j], part[i][j], 0, 0, 0);
          }
        }
        if (t < kOps) {
          const u32x4_t c = raw[((q + 1) / 2) & 1][t];
          op[(q + 1) & 1][t] = q & 1 ? codes8_to_bf16(c[0], c[1]) : codes8_to_bf16(c[2], c[3]);
          if (q % 2 == 0) read_codes(t, (q < 4 ? stage : next) * Shape::kStage, (q / 2 + 2) & 3);
        }
        if (t == kOps / 2 - 1) {
          const int n = (q + 4) % 8 * kPerSlice;  // of the block kStages on from q = 4, else one nearer
#pragma unroll
          for (int k = n; k < n + kPerSlice && k <= kDmas; ++k) request(k);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
      if (q == 0) {
        const float* sc =
            reinterpret_cast<const float*>(lds + kStages * Shape::kStage + stage * 256 * kScaleWaves);
#pragma unroll
        for (int j = 0; j < kJ; ++j) xs[j] = sc[32 * kJ * wm + 32 * j + r];
#pragma unroll
        for (int i = 0; i < (kGated ? 2 : 1); ++i) ws[i] = sc[Shape::kRowsM + 2 * wn + i];
      }
    }
    stage = next;
  }
#pragma unroll
  for (int i = 0; i < kI; ++i)
#pragma unroll
    for (int j = 0; j < kJ; ++j) add_scaled(acc[i][j], part[i][j], xs[j] * ws[kGated ? i : 0]);

  // The sums go through the LDS, [row of x][weight row], 16-byte chunks of a row
  // permuted: what follows is a loop over whole rows, written out once (unrolled over the
  // registers it was 80 KB of code, which no tile finds in the instruction cache) and
  // with whole lines stored
  tile_barrier<0>();
  float4_t* tile = reinterpret_cast<float4_t*>(lds);
  constexpr int kChunks = Shape::kRowsN / 4, kThreads = 64 * Shape::kWaves;
  static_assert(Shape::kRowsM * kChunks * 16 <= sizeof(lds), "");
#pragma unroll
  for (int i = 0; i < kI; ++i)
#pragma unroll
    for (int j = 0; j < kJ; ++j)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        // lane (r, h) holds weight rows 8 q + 4 h + 0..3 of row r of each product
        const int row = 32 * (kJ * wm + j) + r;
        const float16_t& v = acc[i][j];
        tile[row * kChunks + ((8 * (kI * wn + i) + 2 * q + h) ^ (row & 15))] =
            float4_t{v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]};
      }
  __syncthreads();
  if constexpr (!kGated) {
    constexpr int kSteps = Shape::kRowsM * kChunks / kThreads, kGroup = kSteps < 8 ? kSteps : 8;
    static_assert(Shape::kRowsM * kChunks % kThreads == 0 && kSteps % kGroup == 0, "");
    if (p.res && !p.sums && p.N >= 4) {
      // (eight rows of the residual on their way at a time: with one or two, what comes
      // after the products took longer than they did at short k.  Past the edges a load
      // repeats the last whole group, which is not used)
#pragma unroll 1
      for (int first = threadIdx.x; first < kSteps * kThreads; first += kGroup * kThreads) {
        u32x4_t res[kGroup];
#pragma unroll
        for (int i = 0; i < kGroup; ++i) {
          const int t = first + i * kThreads;
          res[i] = load_res4(p, min(m0 + t / kChunks, p.M - 1), min(n0 + 4 * (t % kChunks), p.N - 4));
        }
#pragma unroll
        for (int i = 0; i < kGroup; ++i) {
          const int t = first + i * kThreads, row = t / kChunks, c = t % kChunks, n = n0 + 4 * c;
          const float4_t v = tile[row * kChunks + (c ^ (row & 15))];
          const float y[4] = {v[0], v[1], v[2], v[3]};
          if (m0 + row >= p.M) continue;
          if (n + 4 <= p.N)
            store_whole4(p, m0 + row, n, y, res[i]);
          else
            store_out4(p, z, m0 + row, n, y);
        }
      }
    } else {
#pragma unroll 2
      for (int t = threadIdx.x; t < kSteps * kThreads; t += kThreads) {
        const int row = t / kChunks, c = t % kChunks;
        if (m0 + row >= p.M) break;
        const float4_t v = tile[row * kChunks + (c ^ (row & 15))];
        const float y[4] = {v[0], v[1], v[2], v[3]};
        store_out4(p, z, m0 + row, n0 + 4 * c, y);
      }
    }
  } else {
    // 128 columns, one block: 16 lanes per row, 8 outputs each (weight rows 64 w + 0..31
    // of the tile are gate, 64 w + 32..63 the matching up)
#pragma unroll 1
    for (int t = threadIdx.x; t < Shape::kRowsM * 16; t += kThreads) {
      const int row = t >> 4, l = t & 15, m = m0 + row;
      if (m >= p.M) break;  // (whole groups of 16 lanes)
      float y[8];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int c = 16 * (l >> 2) + 2 * (l & 3) + i;
        const float4_t g = tile[row * kChunks + (c ^ (row & 15))], u = tile[row * kChunks + ((c + 8) ^ (row & 15))];
#pragma unroll
        for (int e = 0; e < 4; ++e)
          y[4 * i + e] = n0 + 8 * l + 4 * i + e < p.N ? silu_mul(g[e], u[e]) : 0.0f;
      }
      put_gated(p, m, tn, l, y);
    }
  }
}

template <bool kGated, int kWN, int kWM, int kI, int kJ>
int launch_tile(const LinearArgs& p, int parts, hipStream_t s) {
  using Shape = TileShape<kGated, kWN, kWM, kI, kJ>;
  const int tiles_n = (p.N + Shape::kCols - 1) / Shape::kCols, tiles_m = (p.M + Shape::kRowsM - 1) / Shape::kRowsM;
  const unsigned grid = (static_cast<unsigned>(tiles_n) * tiles_m * p.splits * parts + 7) / 8 * 8;
  // A launch holds fewer than 2^32 threads.  (Of all products within the limits on sizes only
  // gated ones of nearly 2^37 outputs reach that: rows in two halves)
  if constexpr (kGated) {
    if (grid >= (int64_t{1} << 32) / (64 * Shape::kWaves)) {
      LinearArgs a = p, b = p;
      a.M = tiles_m / 2 * Shape::kRowsM, b.M = p.M - a.M;
      b.x += a.M * p.x_ld, b.xs += a.M * p.xs_m, b.codes += a.M * p.codes_ld, b.scales += a.M * p.s_m;
      const int rc = launch_tile<kGated, kWN, kWM, kI, kJ>(a, parts, s);
      return rc != ZKV_OK ? rc : launch_tile<kGated, kWN, kWM, kI, kJ>(b, parts, s);
    }
  }
  fp8_tile_kernel<kGated, kWN, kWM, kI, kJ>
      <<<grid, 64 * Shape::kWaves, 0, s>>>(p, tiles_n, tiles_m, parts);
  return check_launch("fp8_tile_kernel");
}

// ---------------------------------------------------------------------------
// Which kernel, and in how many runs of k: the shortest by a model of their times, in
// us: a start, and a time per block of k (per wave, where waves share k) that grows as the
// CUs fill, which lowers the clock; and where the runs are joined by a second launch,
// that and the sums' way out and back.  Against all kernels that it considers its choice took
// 1.016 times the best over the 162 sizes that its constants were fitted to (geometric mean;
// at worst 1.27), 1.023 over 80 others (at worst 1.38).  It has no term for the output's
// bytes: wide outputs over one or two blocks of k take up to 3.6 times what it says
// (profiles/fp8_linear_choice.md has the sizes).  With as many runs as it takes 64 x 1024 x 9728 went from 15.0 to 9.3 us, 64 x 256 x 16384 from 16.7 to 7.9,
// gated 16 x 256 x 16384 from 11.3 to 9.4.  Up to 16 rows a tile of the matrix instruction
// holds them all, and units of 16 weight rows are the smallest.
// ---------------------------------------------------------------------------
enum Variant : int { kStream8, kStream16, kStream32, kSplit, kTile256, kTile128, kTileFlat, kTile64, kTileGated };

struct Plan {
  int variant, splits;
  bool sums;
};

struct Pace {
  double start;    // until the first block and behind the last
  int most;        // steps of the list
  double step[4];  // a block's time with 256, 512, ... workgroups at work
  double low;      // of the first of them where nearly all CUs are idle
};

double rounds_us(int64_t groups, int steps, const Pace& pace) {
  const int64_t per_round = 256 * pace.most, full = groups / per_round, rest = groups % per_round;
  double us = pace.start + full * steps * pace.step[pace.most - 1];
  if (rest) {
    const int c = static_cast<int>((rest + 255) / 256);
    const double low = c > 1 ? pace.step[c - 2] : pace.low * pace.step[0], fill = (rest - (c - 1) * 256) / 256.0;
    us += steps * (low + fill * (pace.step[c - 1] - low));
  }
  return us + 0.074 * pace.start * (full + (rest > 0) - 1);
}

int64_t tiles_of(int a, int b) { return (a + b - 1) / b; }

// M rows of x, N weight rows in each of `parts`.  Two parts, gate and up, leave sums
// for a second launch, but for the kernel that computes whole blocks of outputs.
Plan plan_product(int M, int N, int nkb, int parts) {
  const bool gated = parts == 2;
  constexpr Pace kFewPace{3.49, 1, {0.25}, 1.29}, kStreamPace{3.49, 2, {0.44, 0.88}, 0.5},
      kStreamLongPace{3.49, 1, {0.79}, 0.5}, kSplitPace{4.43, 2, {0.57, 1.54}, 0.5}, k256Pace{7.27, 1, {2.01}, 0.5},
      k128Pace{7.27, 2, {1.02, 3.51}, 0.5}, kFlatPace{7.27, 2, {0.72, 1.47}, 0.5},
      k64Pace{7.27, 4, {0.37, 0.89, 1.07, 1.74}, 0.5}, kGatedPace{11.5, 1, {1.78}, 0.5};
  Plan best{kTile256, 1, gated};
  double best_us = 1e30;
  auto consider = [&](int variant, int splits, int64_t tiles, int steps, const Pace& pace, bool own) {
    const bool sums = !own && (gated || splits > 1);
    double us = rounds_us(tiles * splits * (own ? 1 : parts), steps, pace);
    if (sums) us += (gated ? 2.72 : 1.61) + 8.0 * parts * splits * M * static_cast<double>(N) / 5.51e6;
    if (us < best_us) best_us = us, best = Plan{variant, splits, sums};
  };
  const int64_t units = tiles_of(N, stream_rows(N, parts));
  for (int k = 1; k <= kMaxSplits && (k == 1 || 2 * k <= nkb + 1); ++k) {
    const int steps = (nkb + k - 1) / k, waves = stream_waves(steps), stream_steps = (steps + waves - 1) / waves;
    if (M <= 16) {
      if (k == 1 || units * k * parts <= 256)
        consider(M <= 8 ? kStream8 : kStream16, k, units, stream_steps, kFewPace, false);
      continue;
    }
    consider(kStream32, k, units * tiles_of(M, 32), stream_steps, waves > 4 ? kStreamLongPace : kStreamPace, false);
    consider(kSplit, k, tiles_of(N, 32) * tiles_of(M, 32), (steps + 3) / 4, kSplitPace, false);
    consider(kTile256, k, tiles_of(N, 256) * tiles_of(M, 128), steps, k256Pace, false);
    consider(kTile128, k, tiles_of(N, 128) * tiles_of(M, 128), steps, k128Pace, false);
    consider(kTileFlat, k, tiles_of(N, 128) * tiles_of(M, 64), steps, kFlatPace, false);
    consider(kTile64, k, tiles_of(N, 64) * tiles_of(M, 64), steps, k64Pace, false);
  }
  if (gated && M > 16) consider(kTileGated, 1, tiles_of(N, 128) * tiles_of(M, 128), nkb, kGatedPace, true);
  return best;
}

int launch_variant(const LinearArgs& p, int variant, int parts, hipStream_t s) {
  switch (variant) {
    case kStream8: return launch_stream<8>(p, parts, s);
    case kStream16: return launch_stream<16>(p, parts, s);
    case kStream32: return launch_stream<32>(p, parts, s);
    case kSplit: return launch_split(p, parts, s);
    case kTile256: return launch_tile<false, 4, 2, 2, 2>(p, parts, s);
    case kTile128: return launch_tile<false, 2, 4, 2, 1>(p, parts, s);
    case kTileFlat: return launch_tile<false, 4, 2, 1, 1>(p, parts, s);
    case kTile64: return launch_tile<false, 2, 2, 1, 1>(p, parts, s);
    default: return launch_tile<true, 4, 2, 2, 2>(p, 1, s);
  }
}

size_t sums_bytes(const Plan& plan, int parts, int M, int N) {
  return plan.sums ? static_cast<size_t>(parts) * plan.splits * M * ((N + 3) / 4 * 4) * 4 : 0;
}

int blocks_of(int n) { return (n + kFp8Block - 1) / kFp8Block; }

// The sizes that both entry points take; null or what is wrong.  (K: the kernels and the
// workspace have no limit of their own there; the choice is measured, and the bounds on
// errors tested, up to 128 blocks.)
const char* check_sizes(int M, int N, int K) {
  if (M < 1 || N < 1 || K < 1) return "empty product";
  if (M >= 1 << 20 || N >= 1 << 22 || static_cast<int64_t>(M) * N > int64_t{1} << 37)
    return "below 2^20 rows of x, 2^22 rows of the weight, and at most 2^37 outputs";
  if (K % kFp8Block || K > 128 * kFp8Block) return "K is a multiple of 128, at most 16384";
  return nullptr;
}

// Whether they take the sizes with K rounded up to whole blocks.
bool takes_sizes(int M, int N, int K) {
  return K >= 1 && K <= 128 * kFp8Block && !check_sizes(M, N, blocks_of(K) * kFp8Block);
}

// And their operands.
const char* check_operands(const uint8_t* x, int64_t x_ld, const float* xs, const uint8_t* w, int64_t w_ld,
                           const float* ws, int M, int N, int K) {
  if (!x || !xs || !w || !ws) return "null pointer";
  if (const char* bad = check_sizes(M, N, K)) return bad;
  if (x_ld < K || w_ld < K || !rows_on_16(x, x_ld, 1) || !rows_on_16(w, w_ld, 1))
    return "rows of codes hold K bytes and start on 16";
  if (x_ld >= 1 << 23 || w_ld >= 1 << 23) return "rows of codes lie less than 8 MiB apart";
  return nullptr;
}

}  // namespace
}  // namespace zkv

using namespace zkv;

extern "C" int zkv_fp8_plan(int M, int N, int K, int parts) {
  if (check_sizes(M, N, K) || parts < 1 || parts > 2) return -1;
  const Plan plan = plan_product(M, N, K / kFp8Block, parts);
  return 16 * plan.variant + plan.splits;
}

extern "C" size_t zkv_fp8_linear_workspace_size(int M, int N, int K) {
  if (!takes_sizes(M, N, K)) return 0;
  return sums_bytes(plan_product(M, N, blocks_of(K), 1), 1, M, N);
}

extern "C" int zkv_fp8_linear(const uint8_t* x, int64_t x_ld, const float* xs, int64_t xs_m, int64_t xs_b,
                              const uint8_t* w, int64_t w_ld, const float* ws, int M, int N, int K,
                              const void* residual, int64_t res_ld, void* out, int64_t out_ld, int type,
                              void* workspace, size_t workspace_bytes, zkv_stream_t stream) {
  const char* bad = check_operands(x, x_ld, xs, w, w_ld, ws, M, N, K);
  ZKV_REQUIRE(!bad, "zkv_fp8_linear: %s (M=%d N=%d K=%d)", bad, M, N, K);
  ZKV_REQUIRE(out && type >= kRowBf16 && type <= kRowF32, "zkv_fp8_linear: bad output");
  const Plan plan = plan_product(M, N, K / kFp8Block, 1);
  const size_t need = sums_bytes(plan, 1, M, N);
  if (need && (workspace_bytes < need || !workspace || (reinterpret_cast<uintptr_t>(workspace) & 15)))
    return fail(ZKV_ESPACE, "zkv_fp8_linear: %zu bytes of workspace on 16 bytes, %zu needed", workspace_bytes, need);
  LinearArgs p{};
  p.x = x, p.x_ld = x_ld, p.xs = xs, p.xs_m = xs_m, p.xs_b = xs_b, p.w = w, p.w_ld = w_ld, p.ws = ws;
  p.M = M, p.N = N, p.nkb = K / kFp8Block;
  p.res = residual, p.res_ld = res_ld, p.out = out, p.out_ld = out_ld, p.type = type;
  p.sums = plan.sums ? static_cast<float*>(workspace) : nullptr, p.sums_ld = (N + 3) / 4 * 4, p.splits = plan.splits;
  auto s = reinterpret_cast<hipStream_t>(stream);
  const int rc = launch_variant(p, plan.variant, 1, s);
  return rc != ZKV_OK || !plan.sums ? rc : launch_join(p, false, s);
}

extern "C" int zkv_fp8_linear_call(const zkv_fp8_linear_args* a, zkv_stream_t stream) {
  ZKV_REQUIRE(a, "zkv_fp8_linear: null pointer");
  return zkv_fp8_linear(a->x, a->x_ld, a->xs, a->xs_m, a->xs_b, a->w, a->w_ld, a->ws, a->M, a->N, a->K, a->residual,
                        a->res_ld, a->out, a->out_ld, a->type, a->workspace, a->workspace_bytes, stream);
}

extern "C" size_t zkv_fp8_gated_workspace_size(int M, int F, int K) {
  if (!takes_sizes(M, F, K)) return 0;
  return sums_bytes(plan_product(M, F, blocks_of(K), 2), 2, M, F);
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
  const Plan plan = plan_product(M, F, K / kFp8Block, 2);
  const size_t need = sums_bytes(plan, 2, M, F);
  if (need && (workspace_bytes < need || !workspace || (reinterpret_cast<uintptr_t>(workspace) & 15)))
    return fail(ZKV_ESPACE, "zkv_fp8_gated_linear: %zu bytes of workspace on 16 bytes, %zu needed", workspace_bytes,
                need);
  LinearArgs p{};
  p.x = x, p.x_ld = x_ld, p.xs = xs, p.xs_m = xs_m, p.xs_b = xs_b, p.w = w, p.w_ld = w_ld, p.ws = ws;
  p.M = M, p.N = F, p.nkb = K / kFp8Block;
  p.codes = codes, p.codes_ld = codes_ld, p.scales = scales, p.s_m = s_m, p.s_b = s_b;
  p.sums = plan.sums ? static_cast<float*>(workspace) : nullptr, p.sums_ld = (F + 3) / 4 * 4, p.splits = plan.splits;
  auto s = reinterpret_cast<hipStream_t>(stream);
  const int rc = launch_variant(p, plan.variant, 2, s);
  return rc != ZKV_OK || !plan.sums ? rc : launch_join(p, true, s);
}

extern "C" int zkv_fp8_gated_linear_call(const zkv_fp8_gated_linear_args* a, zkv_stream_t stream) {
  ZKV_REQUIRE(a, "zkv_fp8_gated_linear: null pointer");
  return zkv_fp8_gated_linear(a->x, a->x_ld, a->xs, a->xs_m, a->xs_b, a->w, a->w_ld, a->ws, a->M, a->F, a->K, a->codes,
                              a->codes_ld, a->scales, a->s_m, a->s_b, a->workspace, a->workspace_bytes, stream);
}
