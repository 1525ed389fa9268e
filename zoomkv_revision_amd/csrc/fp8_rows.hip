// Rows of a hidden state, and weights, as e4m3 codes with a scale per block:
//
//  * fp8_norm_rows_kernel: [h = x + residual;] y = h * rsqrt(mean(h^2) + eps) * w,
//    quantised per row and 128 channels: s = max |y| / 448, code = e4m3(y / s).
//  * fp8_rows_kernel: the same for y = x.
//  * fp8_weight_kernel: a weight in blocks of 128 x 128.
//
// fp32 from the input to the code; the sum h is rounded once, where it is
// stored, and the norm goes by the unrounded one.  Codes are written up to whole
// blocks (zeros behind K), so that what multiplies them needs no tails.
//
// Bound: HBM (x, residual and sum once, a byte per code), launch and one round
// trip for a few rows.
#include "fp8_common.hpp"

#include <algorithm>

namespace zkv {
namespace {

struct RowsParams {
  const void* x;
  int64_t x_ld;
  const void* w;  // norm weight [K]
  const void* res;
  int64_t res_ld;
  void* sum;
  int64_t sum_ld;
  uint8_t* codes;  // [M, whole blocks]
  int64_t codes_ld;
  float* scales;  // element (m, b) at m * s_m + b * s_b
  int64_t s_m, s_b;
  float eps;
  int M, K;
  int rows_per_xcd;
};

// Workgroups go to the eight XCDs in turn: workgroup b takes a row (or group of rows) of
// the b % 8-th eighth of them, so that neighbouring rows' scales (4 bytes each, columns of
// M) meet in one L2.
__device__ __forceinline__ int xcd_row(const RowsParams& p) {
  return static_cast<int>(blockIdx.x & 7) * p.rows_per_xcd + static_cast<int>(blockIdx.x >> 3);
}

// 8 values of a row as codes: 16 neighbouring lanes hold a block.
__device__ __forceinline__ void put_codes(const RowsParams& p, int row, int chunk, const float (&y)[8]) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, abs_bits(y[i]));
  const float s = fp8_scale(row_max(m)), r = 1.0f / s;
  if (8 * chunk >= (p.K + kFp8Block - 1) / kFp8Block * kFp8Block) return;
  *reinterpret_cast<u32x2_t*>(p.codes + row * p.codes_ld + 8 * chunk) =
      u32x2_t{fp8_codes4(y, s, r), fp8_codes4(y + 4, s, r)};
  if ((chunk & 15) == 0) p.scales[row * p.s_m + (chunk >> 4) * p.s_b] = s;
}

// One workgroup per row, kC chunks of 8 channels per thread, held in registers.
template <int kType, int kC>
__global__ __launch_bounds__(1024) void fp8_norm_rows_kernel(const RowsParams p) {
  __shared__ float red[16];
  const int row = xcd_row(p);
  if (row >= p.M) return;
  constexpr int kItem = kType == kRowF32 ? 4 : 2;
  const int nw = blockDim.x >> 6, wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const void* x = static_cast<const uint8_t*>(p.x) + row * p.x_ld * kItem;
  float h[kC][8];
#pragma unroll
  for (int c = 0; c < kC; ++c) load_row8<kType>(x, 8 * (threadIdx.x + c * blockDim.x), p.K, h[c]);
  if (p.res) {
    const void* res = static_cast<const uint8_t*>(p.res) + row * p.res_ld * kItem;
    float a[kC][8];
#pragma unroll
    for (int c = 0; c < kC; ++c) load_row8<kType>(res, 8 * (threadIdx.x + c * blockDim.x), p.K, a[c]);
#pragma unroll
    for (int c = 0; c < kC; ++c)
#pragma unroll
      for (int i = 0; i < 8; ++i) h[c][i] += a[c][i];
  }
  // (the norm's weight with them, a round trip less: 1 x 2560 2.60 -> 2.53 us; with two
  // chunks per thread its registers cost more, 2000 x 12288 38 -> 41)
  constexpr bool kEarly = kC == 1;
  float w[kC][8];
  if (kEarly) {
#pragma unroll
    for (int c = 0; c < kC; ++c) load_row8<kType>(p.w, 8 * (threadIdx.x + c * blockDim.x), p.K, w[c]);
  }
  float ss = 0.0f;
#pragma unroll
  for (int c = 0; c < kC; ++c)
#pragma unroll
    for (int i = 0; i < 8; ++i) ss = __builtin_fmaf(h[c][i], h[c][i], ss);
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) ss += __shfl_xor(ss, d);
  if (lane == 0) red[wave] = ss;
  if (p.sum) {
    void* sum = static_cast<uint8_t*>(p.sum) + row * p.sum_ld * kItem;
#pragma unroll
    for (int c = 0; c < kC; ++c) store_row8<kType>(sum, 8 * (threadIdx.x + c * blockDim.x), p.K, h[c]);
  }
  __syncthreads();
  float total = red[0];
  for (int i = 1; i < nw; ++i) total += red[i];
  const float r = rsqrtf(total / static_cast<float>(p.K) + p.eps);
#pragma unroll
  for (int c = 0; c < kC; ++c) {
    const int chunk = threadIdx.x + c * blockDim.x;
    float y[8];
    if (!kEarly) load_row8<kType>(p.w, 8 * chunk, p.K, w[c]);
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = h[c][i] * r * w[c][i];
    put_codes(p, row, chunk, y);
  }
}

// Rows of up to 8 kLanes channels: 256 / kLanes rows per workgroup, a chunk per lane, and
// no barrier.  (A workgroup of one wave per row was bound by the rate at which they
// start: 49150 rows of 68 26 us.)
template <int kType, int kLanes, bool kNorm>
__global__ __launch_bounds__(256) void fp8_short_rows_kernel(const RowsParams p) {
  const int row = xcd_row(p) * (256 / kLanes) + static_cast<int>(threadIdx.x) / kLanes, chunk = threadIdx.x % kLanes;
  if (row >= p.M) return;  // (whole groups of lanes)
  constexpr int kItem = kType == kRowF32 ? 4 : 2;
  float h[8];
  load_row8<kType>(static_cast<const uint8_t*>(p.x) + row * p.x_ld * kItem, 8 * chunk, p.K, h);
  if constexpr (kNorm) {
    float w[8], ss = 0.0f;
    load_row8<kType>(p.w, 8 * chunk, p.K, w);
    if (p.res) {
      float a[8];
      load_row8<kType>(static_cast<const uint8_t*>(p.res) + row * p.res_ld * kItem, 8 * chunk, p.K, a);
#pragma unroll
      for (int i = 0; i < 8; ++i) h[i] += a[i];
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) ss = __builtin_fmaf(h[i], h[i], ss);
#pragma unroll
    for (int d = kLanes / 2; d > 0; d >>= 1) ss += __shfl_xor(ss, d);
    if (p.sum) store_row8<kType>(static_cast<uint8_t*>(p.sum) + row * p.sum_ld * kItem, 8 * chunk, p.K, h);
    const float r = rsqrtf(ss / static_cast<float>(p.K) + p.eps);
#pragma unroll
    for (int i = 0; i < 8; ++i) h[i] = h[i] * r * w[i];
  }
  put_codes(p, row, chunk, h);
}

// Blocks are independent: a row's chunks in strides of the workgroup.
template <int kType>
__global__ __launch_bounds__(1024) void fp8_rows_kernel(const RowsParams p) {
  const int row = xcd_row(p);
  if (row >= p.M) return;
  const void* x = static_cast<const uint8_t*>(p.x) + row * p.x_ld * (kType == kRowF32 ? 4 : 2);
  const int chunks = (p.K + kFp8Block - 1) / kFp8Block * (kFp8Block / 8);
  for (int first = 0; first < chunks; first += blockDim.x) {
    float v[8];
    load_row8<kType>(x, 8 * (first + threadIdx.x), p.K, v);
    put_codes(p, row, first + threadIdx.x, v);
  }
}

struct WeightParams {
  const void* w;
  int64_t w_ld;
  int N, K, parts;
  uint8_t* codes;
  int64_t codes_ld;
  float* scales;  // [parts * blocks of a part's rows, blocks of K]
};

// One workgroup per block of 128 x 128: thread t holds chunk t % 16 of rows t / 16 + 16 i.
template <int kType>
__global__ __launch_bounds__(256) void fp8_weight_kernel(const WeightParams p) {
  __shared__ uint32_t red[4];
  const int kb = blockIdx.x, rows = p.N / p.parts, nb = (rows + kFp8Block - 1) / kFp8Block;
  const int part = blockIdx.y / nb, b = blockIdx.y % nb;
  const int k = kb * kFp8Block + 8 * (threadIdx.x & 15);
  float v[8][8];
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int r = b * kFp8Block + (threadIdx.x >> 4) + 16 * i;
    const void* src = static_cast<const uint8_t*>(p.w) +
                      (static_cast<int64_t>(part) * rows + min(r, rows - 1)) * p.w_ld * (kType == kRowF32 ? 4 : 2);
    load_row8<kType>(src, k, p.K, v[i]);
#pragma unroll
    for (int j = 0; j < 8; ++j) m = max(m, abs_bits(v[i][j]));
  }
  m = row_max(m);
  m = max(m, static_cast<uint32_t>(__shfl_xor(static_cast<int>(m), 16)));
  m = max(m, static_cast<uint32_t>(__shfl_xor(static_cast<int>(m), 32)));
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = m;
  __syncthreads();
  const float s = fp8_scale(max(max(red[0], red[1]), max(red[2], red[3]))), r1 = 1.0f / s;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int r = b * kFp8Block + (threadIdx.x >> 4) + 16 * i;
    if (r < rows)
      *reinterpret_cast<u32x2_t*>(p.codes + (static_cast<int64_t>(part) * rows + r) * p.codes_ld + k) =
          u32x2_t{fp8_codes4(v[i], s, r1), fp8_codes4(v[i] + 4, s, r1)};
  }
  if (threadIdx.x == 0) p.scales[static_cast<int64_t>(blockIdx.y) * gridDim.x + kb] = s;
}

constexpr int kNormMaxK = 65536;  // 1024 threads of 8 chunks
constexpr int kLaunchRows = 1 << 21;

int blocks_of(int n) { return (n + kFp8Block - 1) / kFp8Block; }

}  // namespace
}  // namespace zkv

using namespace zkv;

extern "C" int zkv_fp8_rows(const void* x, int64_t x_ld, int M, int K, int type, const void* norm_w, float eps,
                            const void* residual, int64_t res_ld, void* sum_out, int64_t sum_ld, uint8_t* codes,
                            int64_t codes_ld, float* scales, int64_t s_m, int64_t s_b, zkv_stream_t stream) {
  ZKV_REQUIRE(x && codes && scales, "zkv_fp8_rows: null pointer");
  ZKV_REQUIRE(M >= 1 && M < (1 << 27) && K >= 1 && K <= (1 << 30), "zkv_fp8_rows: M=%d K=%d", M, K);
  ZKV_REQUIRE(type >= kRowBf16 && type <= kRowF32, "zkv_fp8_rows: type %d", type);
  ZKV_REQUIRE(norm_w || (!residual && !sum_out), "zkv_fp8_rows: a residual goes with a norm");
  ZKV_REQUIRE(!norm_w || K <= kNormMaxK, "zkv_fp8_rows: rows of %d, at most %d with a norm", K, kNormMaxK);
  ZKV_REQUIRE(codes_ld >= static_cast<int64_t>(blocks_of(K)) * kFp8Block && codes_ld % 8 == 0 &&
                  (reinterpret_cast<uintptr_t>(codes) & 7) == 0,
              "zkv_fp8_rows: rows of codes hold whole blocks of 128 and start on 8 bytes");
  // (a launch holds fewer than 2^32 threads, a row takes up to 1024 of them: more rows go in
  // several launches)
  const int64_t item = type == kRowF32 ? 4 : 2;
  for (; M > kLaunchRows; M -= kLaunchRows) {
    const int rc = zkv_fp8_rows(x, x_ld, kLaunchRows, K, type, norm_w, eps, residual, res_ld, sum_out, sum_ld, codes,
                                codes_ld, scales, s_m, s_b, stream);
    if (rc != ZKV_OK) return rc;
    x = static_cast<const uint8_t*>(x) + kLaunchRows * x_ld * item;
    if (residual) residual = static_cast<const uint8_t*>(residual) + kLaunchRows * res_ld * item;
    if (sum_out) sum_out = static_cast<uint8_t*>(sum_out) + kLaunchRows * sum_ld * item;
    codes += kLaunchRows * codes_ld, scales += kLaunchRows * s_m;
  }
  const int per = (M + 7) / 8;
  const RowsParams p{x, x_ld, norm_w, residual, res_ld, sum_out, sum_ld, codes, codes_ld, scales,
                     s_m, s_b, eps, M, K, per};
  auto s = reinterpret_cast<hipStream_t>(stream);
  const int chunks = blocks_of(K) * (kFp8Block / 8);
  if (chunks <= 64) {
    const int lanes = chunks <= 16 ? 16 : chunks <= 32 ? 32 : 64, groups = ((M + 256 / lanes - 1) / (256 / lanes) + 7) / 8;
    RowsParams q = p;
    q.rows_per_xcd = groups;
#define ZKV_SHORT(T, L)                                                        \
  do {                                                                         \
    if (norm_w) fp8_short_rows_kernel<T, L, true><<<groups * 8, 256, 0, s>>>(q); \
    else fp8_short_rows_kernel<T, L, false><<<groups * 8, 256, 0, s>>>(q);     \
  } while (0)
#define ZKV_SHORT_TYPE(T)                                                      \
  do {                                                                         \
    if (lanes == 16) ZKV_SHORT(T, 16);                                         \
    else if (lanes == 32) ZKV_SHORT(T, 32);                                    \
    else ZKV_SHORT(T, 64);                                                     \
  } while (0)
    if (type == kRowBf16) ZKV_SHORT_TYPE(kRowBf16);
    else if (type == kRowF16) ZKV_SHORT_TYPE(kRowF16);
    else ZKV_SHORT_TYPE(kRowF32);
#undef ZKV_SHORT_TYPE
#undef ZKV_SHORT
    return check_launch("fp8_short_rows_kernel");
  }
  if (!norm_w) {
    const int threads = std::min((chunks + 63) / 64, 16) * 64;
    if (type == kRowBf16) fp8_rows_kernel<kRowBf16><<<per * 8, threads, 0, s>>>(p);
    else if (type == kRowF16) fp8_rows_kernel<kRowF16><<<per * 8, threads, 0, s>>>(p);
    else fp8_rows_kernel<kRowF32><<<per * 8, threads, 0, s>>>(p);
    return check_launch("fp8_rows_kernel");
  }
  const int c = chunks <= 1024 ? 1 : chunks <= 2048 ? 2 : chunks <= 4096 ? 4 : 8;
  const int threads = (chunks + 64 * c - 1) / (64 * c) * 64;
#define ZKV_ROWS(T)                                                             \
  do {                                                                          \
    if (c == 1) fp8_norm_rows_kernel<T, 1><<<per * 8, threads, 0, s>>>(p);      \
    else if (c == 2) fp8_norm_rows_kernel<T, 2><<<per * 8, threads, 0, s>>>(p); \
    else if (c == 4) fp8_norm_rows_kernel<T, 4><<<per * 8, threads, 0, s>>>(p); \
    else fp8_norm_rows_kernel<T, 8><<<per * 8, threads, 0, s>>>(p);             \
  } while (0)
  if (type == kRowBf16) ZKV_ROWS(kRowBf16);
  else if (type == kRowF16) ZKV_ROWS(kRowF16);
  else ZKV_ROWS(kRowF32);
#undef ZKV_ROWS
  return check_launch("fp8_norm_rows_kernel");
}

extern "C" int zkv_fp8_rows_call(const zkv_fp8_rows_args* a, zkv_stream_t stream) {
  ZKV_REQUIRE(a, "zkv_fp8_rows: null pointer");
  return zkv_fp8_rows(a->x, a->x_ld, a->M, a->K, a->type, a->norm_w, a->eps, a->residual, a->res_ld, a->sum_out,
                      a->sum_ld, a->codes, a->codes_ld, a->scales, a->s_m, a->s_b, stream);
}

extern "C" int zkv_fp8_weight(const void* w, int64_t w_ld, int N, int K, int type, int parts, uint8_t* codes,
                              int64_t codes_ld, float* scales, zkv_stream_t stream) {
  ZKV_REQUIRE(w && codes && scales, "zkv_fp8_weight: null pointer");
  ZKV_REQUIRE(N >= 1 && K >= 1 && K <= (1 << 30), "zkv_fp8_weight: N=%d K=%d", N, K);
  ZKV_REQUIRE(type >= kRowBf16 && type <= kRowF32, "zkv_fp8_weight: type %d", type);
  ZKV_REQUIRE(parts >= 1 && N % parts == 0, "zkv_fp8_weight: %d rows in %d parts", N, parts);
  ZKV_REQUIRE(codes_ld >= static_cast<int64_t>(blocks_of(K)) * kFp8Block && codes_ld % 8 == 0 &&
                  (reinterpret_cast<uintptr_t>(codes) & 7) == 0,
              "zkv_fp8_weight: rows of codes hold whole blocks of 128 and start on 8 bytes");
  const int64_t nb = static_cast<int64_t>(parts) * blocks_of(N / parts);
  ZKV_REQUIRE(nb <= 65535, "zkv_fp8_weight: %lld blocks of rows, at most 65535", static_cast<long long>(nb));
  const WeightParams p{w, w_ld, N, K, parts, codes, codes_ld, scales};
  const dim3 grid(blocks_of(K), static_cast<unsigned>(nb));
  auto s = reinterpret_cast<hipStream_t>(stream);
  if (type == kRowBf16) fp8_weight_kernel<kRowBf16><<<grid, 256, 0, s>>>(p);
  else if (type == kRowF16) fp8_weight_kernel<kRowF16><<<grid, 256, 0, s>>>(p);
  else fp8_weight_kernel<kRowF32><<<grid, 256, 0, s>>>(p);
  return check_launch("fp8_weight_kernel");
}
