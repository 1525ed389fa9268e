// Attention of one new token per request over a paged K / V cache (gfx950).
//
// For request b, KV head h and each of its query heads, over the tokens t of
// [first_b, len_b) (first_b = max(0, len_b - window) with a window, else 0):
//
//   s_t = scale * q . K[t],  m = max s_t,  l = sum exp(s_t - m),
//   out = sum exp(s_t - m) V[t] / l,  lse = m + log l
//
// where token t lives in row t % page_size of page block_table[b, t / page_size].
// One pass over the cache with the running maximum and sum of the softmax.
//
// Work.  A unit is one (b, KV head, group of up to 16 query heads); its tokens
// are cut into tiles of 32.  On a line, each unit takes a place per tile and
// kUnitCost more for its start and end; workgroup w takes places [w C, (w + 1)
// C), and inside it each wave an equal run, whatever the lengths are (they are
// read on the device, so a captured launch follows them).  A wave finishes the
// units that lie wholly in its run by itself; the ends of its run go to LDS as
// partials (m, l, O) and are joined there; the ends of the workgroup's run go
// to the workspace and are joined by the last of the workgroups that share the
// unit (where these are many, by the last of each few first).  Each workgroup
// leaves at most two partials, whatever the batch is, and which tiles are joined
// in which order depends on the lengths alone, so the result is the same from
// run to run.
//
// Stream.  A wave walks its run as one stream of tiles across the units: a
// ring of kDepth tiles in registers, the request running kDepth - 1 tiles (and
// the rows' places one more) ahead of the use, so a unit's first tile does not
// wait for memory any more than its others.  Of two waves on a SIMD the older
// is served first; each publishes its tiles done and raises its priority while
// it is behind (32 requests in e4m3 71 -> 68 us; the 16-bit caches end with
// their memory either way).
//
// Bound by HBM: 16 requests of 32768 tokens, 32 / 8 heads of 128, bf16 (2.1 GB):
// 328 us, 6.5 TB/s; 64 requests of 1 to 8192 tokens 63 us (5.6 TB/s, behind
// about 9 us of launch, first round trips and joins); 1 x 700 tokens 12.9 us, a
// chain of round trips (lengths, page ids and q, a tile, the partials out and
// back).  1 x 131072 tokens: 91 us, 96 where the pool is laid out [page, token,
// head].
//
// Tile.  S^T = K q^T and O^T = V^T P^T on v_mfma_f32_16x16x32: K rows are the
// A operand (lane 16 g + c: token c, channels 32 s + 8 g ..), q the B operand
// (head c).  The scores come out with head c and tokens 4 g + i in lane
// 16 g + c, which is where P has to be as the B operand of the second product
// when its k-slice g is tokens 4 g .. 4 g + 3 and 16 + 4 g .. 16 + 4 g + 3: no
// value of S or P moves between lanes.  V rows are read whole by 16 lanes
// (lane c: channels c D / 16 ..) and turned in registers, two tokens to a word,
// by v_perm: row c of the j-th A operand is channel c D / 16 + j.  P enters as
// the sum of its leading 16-bit parts, one product each (the matrix cores wait
// for memory here anyway), cut towards zero: three of 8 bits for bf16; two of 11
// for fp16, the second times 2^11 into a product of its own, as fp16 ends at
// 2^-24.  So the weights keep 21 bits and more down to 2^-126 (bf16) or, less
// finely, 2^-47 (fp16) of the largest one.  An infinite V stays infinite
// whatever its weight is (0 * Inf or -part * Inf would make it NaN): bf16's parts
// behind the first are at least 2^-126, which no sum sees; fp16's second part is
// at least its last place, and where the first may be 0 such V are taken out and
// multiplied apart.  The second part's own product takes 0 to 1.5% of a call
// in fp16 against one sum for both parts, which held 2^-31 of the largest weight,
// 3% at head dim 256 (16 requests of 8192 tokens, 16 / 4 heads: 91.7 us, 88.9);
// with scores so far apart that V is looked through in every tile 0.3 to 3.5%, 9%
// at head dim 256.
#include "paged_common.hpp"

#include <algorithm>

namespace zkv {
namespace {

constexpr int kTile = 32;          // tokens of a tile: one k-step of the P V product
constexpr int kHeads = 16;         // query heads of a unit: the columns of an MFMA
constexpr int kMaxBatch = 4096;    // requests of a call: 4 bytes of LDS each
constexpr int kMaxGroups = 256;    // workgroups
constexpr int kUnitCost = 2;       // places of a unit beyond its tiles
// A batch of units of this many places on average, twice that and more in a
// workgroup's run: cuts are moved out of them (235 requests of 66 tokens, 64 / 8
// heads of 64, e4m3, 17.5 -> 11.2 us; 88 of up to 162, 192 / 8 of 256, 40 -> 30).
constexpr int kSmallUnit = 8;
constexpr float kInf = __builtin_inff();
constexpr float kLog2e = 1.4426950408889634f, kLn2v = 0.6931471805599453f;
// Rows of one head at a stride of 512 bytes or a multiple (pools [page, token,
// head]) share few of the first cache's sets, which holds the lines on their
// way: fewer loads of a CU are in flight.  There a unit is a set of KV heads
// (two to eight, up to 16 query heads) that neighbouring waves take, from
// kSetPlaces places per wave on: 16 requests of 32768 tokens, 32 / 8 heads of
// 128, bf16 372 -> 328 us (322 as [page, head, token]); 64 of 4096 in e4m3, heads
// of 64, 79 -> 66; 1 x 131072 103.3 -> 96.5, its join having four times the
// partials per unit; below, 64 requests of 1 to 8192 tokens, 7 tiles a wave,
// would take 54.2 for 52.6.  Head dim 256, whose rows are two and four sets wide,
// does not gain (64 x 4096: 174 us, 180 with sets).
constexpr int kSetPlaces = 12;
// Partials of the last join that a thread requests at once, and the batches of
// them one after the other that a second step costs (131072 tokens of one KV
// head with 8 query heads, 256 partials: 26 us, 50 in one step).
constexpr int kBatch = 8, kStepRounds = 2;

struct PagedAttnParams {
  const uint16_t* q;
  int64_t q_sb, q_sh;
  const void* k;
  const void* v;
  const float* k_scale;
  const float* v_scale;
  PageLayout layout;
  FastDiv page;
  const int32_t* table;
  int64_t table_stride;
  const int32_t* lens;
  void* out;
  float* lse;
  float* part_o;   // [workgroup][2][kHeads][D]
  float* part_ml;  // [workgroup][2][kHeads][2]
  unsigned int* arrivals;  // per workgroup: those of the unit that starts in it
  FastDiv units;   // units of one request: kv * groups
  FastDiv sets;    // where a unit is a set of KV heads: kv / set
  int set;         // KV heads of a set (a power of two)
  FastDiv groups;  // groups of up to 16 query heads of a KV head
  float scale;     // softmax scale * log2 e
  int bs, hq, kv, gqa, window, out_f32;
  int max_len;     // width of the table * page size
  int heads_lds;   // query heads kept per partial in LDS: min(gqa, 16)
};

template <int kType>
struct Elem;
template <>
struct Elem<kBf16> {
  typedef bf16x8_t x8;
  // The softmax's reference exponent m is the scores' running maximum less kUp,
  // and follows it only when that is more than kLazyBits powers of two above
  // it: O is rescaled a few times per run, not per tile, and P is at most 2^8.
  static constexpr float kUp = 0.0f, kLazyBits = 8.0f;
  static constexpr int kParts = 3, kTailBits = 0;
  // two values cut to the type, and what is left of them
  static __device__ __forceinline__ uint32_t cut(float& a, float& b) {
    const uint32_t ua = __float_as_uint(a), ub = __float_as_uint(b);
    a -= __uint_as_float(ua & 0xFFFF0000u);
    b -= __uint_as_float(ub & 0xFFFF0000u);
    return __builtin_amdgcn_perm(ub, ua, 0x07060302u);
  }
  static constexpr float kLeast = 0x1p-126f;  // the smallest normal number
  static __device__ __forceinline__ float4_t mfma(x8 a, x8 b, float4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
  template <bool kHigh>
  static __device__ __forceinline__ uint32_t pair_of_fp8(uint32_t w) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, kHigh));
  }
};
template <>
struct Elem<kF16> {
  typedef half8_t x8;
  // P is at most 2^15, its largest at least 2^12, and the second part, less than
  // 2^(15 - 11) times 2^11, ends at 2^-35: 2^-47 of the largest weight.
  static constexpr float kUp = 12.0f, kLazyBits = 3.0f;
  static constexpr int kParts = 2, kTailBits = 11;
  static constexpr float kLeast = 0x1p-24f;
  static constexpr float kLeadBits = -23.0f;  // the leading part of a weight of 2^-23 is not 0
  static __device__ __forceinline__ uint32_t cut(float& a, float& b) {
    const auto h = __builtin_amdgcn_cvt_pkrtz(a, b);
    a -= static_cast<float>(h[0]);
    b -= static_cast<float>(h[1]);
    return __builtin_bit_cast(uint32_t, h);
  }
  static __device__ __forceinline__ float4_t mfma(x8 a, x8 b, float4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
  template <bool kHigh>
  static __device__ __forceinline__ uint32_t pair_of_fp8(uint32_t w) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, kHigh));
  }
};

// One instruction where fmaxf first quiets both operands.  Not for the results
// of a matrix product: the wait states they need are not inserted before asm.
__device__ __forceinline__ float vmax(float a, float b) {
  float r;
  asm("v_max_f32 %0, %1, %2" : "=v"(r) : "v"(a), "v"(b));
  return r;
}

// Maximum and sum over the four lanes 16 g + c of one c.
__device__ __forceinline__ float across_max(float x) {
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  const float y = vmax(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(y), __float_as_uint(y), false, false);
  return vmax(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float across_sum(float x) {
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  const float y = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(y), __float_as_uint(y), false, false);
  return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// Running sum over the wave's lanes, this one's included.
__device__ __forceinline__ int scan64(int x) {
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xF, 0xF, true);   // from 1, 2, 4, 8 lanes before, in a row of 16
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xF, 0xF, true);
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xF, 0xF, true);
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xF, 0xF, true);
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xA, 0xF, false);  // the last of the row before, to rows 1 and 3
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xC, 0xF, false);  // the last of lane 31, to rows 2 and 3
  return x;
}

// Device-coherent accesses of the partials: the sharing workgroups run on
// different XCDs, whose L2s are not coherent.  16 bytes a lane go through a
// buffer descriptor, whose accesses take the same coherence bit as an atomic of
// up to 8 bytes (half the lines touched per byte: 8 KV heads of 256 with 16 query
// heads each, 1295 tokens, 31.1 us, 33.9 with pairs).
constexpr int kDevice = 16;  // sc1: past the caches that a device's XCDs do not share
__device__ __forceinline__ void store_dev(__amdgpu_buffer_rsrc_t r, uint32_t at, const float4_t& x) {
  __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4_t, x), r, static_cast<int>(4 * at), 0, kDevice);
}
__device__ __forceinline__ float4_t load_dev(__amdgpu_buffer_rsrc_t r, uint32_t at) {
  return __builtin_bit_cast(float4_t, __builtin_amdgcn_raw_buffer_load_b128(r, static_cast<int>(4 * at), 0, kDevice));
}
__device__ __forceinline__ void store_dev(float* p, float a, float b) {
  __hip_atomic_store(reinterpret_cast<unsigned long long*>(p), __builtin_bit_cast(unsigned long long, float2_t{a, b}),
                     __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float2_t load_dev(const float* p) {
  return __builtin_bit_cast(float2_t, __hip_atomic_load(reinterpret_cast<const unsigned long long*>(p),
                                                        __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
}

template <int kWords>
__device__ __forceinline__ void load_words(const uint8_t* p, uint32_t* w) {
  if constexpr (kWords == 1) {
    w[0] = __builtin_nontemporal_load(reinterpret_cast<const uint32_t*>(p));
  } else if constexpr (kWords == 2) {
    const u32x2_t x = __builtin_nontemporal_load(reinterpret_cast<const u32x2_t*>(p));
    w[0] = x[0], w[1] = x[1];
  } else {
    const u32x4_t x = __builtin_nontemporal_load(reinterpret_cast<const u32x4_t*>(p));
    w[0] = x[0], w[1] = x[1], w[2] = x[2], w[3] = x[3];
  }
}

// Compile-time shape of a kernel.
template <bool kFp8, int kD>
struct Shape {
  static constexpr int kCell = kFp8 ? 1 : 2;
  static constexpr int kSteps = kD / 32;                 // k-steps of q K^T
  static constexpr int kKLoads = kD * kCell / 64;        // 16-byte loads of a K row per lane
  static constexpr int kJ = kD / 16;                     // channels of V per lane, A operands of P V
  static constexpr int kChunk = std::min(kJ, 16 / kCell);  // of them in one load
  static constexpr int kChunks = kJ / kChunk;
  static constexpr int kChunkWords = kChunk * kCell / 4;
  static constexpr int kVWords = kChunks * kChunkWords;
  static constexpr int kLoads = 2 * kKLoads + 8 * kChunks;  // of a tile
  // 8 waves: 2 on a SIMD, 256 registers each.  Head dim 256 holds twice the
  // tile and twice the output per wave: 4 waves with up to 512.
  static constexpr int kWaves = kD == 256 ? 4 : 8;
  // Where there is no more than a place per wave, cuts are moved out of units of
  // at most kWholeTiles tiles: joining their parts across workgroups takes
  // longer than two or three tiles of a wave one after the other.  Us whole, cut
  // (one request, 32 / 8 heads): head dim 128, 8 tiles 9.1, 13.7; 16 12.6, 13.5;
  // 24 14.2, 13.5; 48 23.3, 13.7 (seven requests with 16 query heads of one KV
  // head: 24 15.2, 17.9; 32 19.2, 17.5); head dim 64, 24 10.7, 12.6; 32 12.4,
  // 12.5; 48 15.3, 12.6; head dim 256, 4 tiles 10.3 both, 8 14.0, 13.5 (16 query
  // heads 17.6, 21.4); 16 19.8, 13.7.
  static constexpr int kWholeTiles = kD == 64 ? 28 : 5 * kWaves / 2;
  // Tiles of the ring: two, one in use and one on its way, also where more
  // registers are left (32 requests of up to 32768 tokens in e4m3, head dim
  // 128: 69 us; with three 72, four 73, five 87: the longer unrolled loop costs
  // more than the loads in flight gain); three for e4m3 at head dim 256 (176
  // us for 16 requests of 32768 tokens, 189 with two).
  static constexpr int kDepth = kD == 256 && kFp8 ? 3 : 2;
  // first channel of chunk n of output row r (r = 0 .. 15)
  static __device__ __forceinline__ int channel(int r, int n) { return n * (16 * kChunk) + r * kChunk; }
};

template <bool kFp8, int kD>
struct TileRegs {
  u32x4_t k[2][Shape<kFp8, kD>::kKLoads];
  uint32_t v[8][Shape<kFp8, kD>::kVWords];
  uint32_t mask;  // bit t: token t is attended
  int unit;       // the unit's number, -1: no tile
  int flags;      // kFirst, kLast: of the wave's part of the unit; kWhole: the part is all of it
};
enum TileFlags : int { kFirst = 1, kLast = 2, kWhole = 4 };

// A place in a wave's stream of tiles.
struct Cursor {
  int b, rest;      // request, unit within it
  int base, tiles;  // the unit's first place on the line, its tiles
  int tile, left;   // the present tile of the request, the wave's tiles of the unit from it on (0: past the run)
  int len;          // the request's length
  int flags;        // kFirst, kWhole
  uint32_t mask;    // the present tile's tokens that are attended
};

template <int kType, bool kFp8, int kD>
struct PagedAttn {
  using S = Shape<kFp8, kD>;
  using E = Elem<kType>;
  using x8 = typename E::x8;
  using Tile = TileRegs<kFp8, kD>;
  static constexpr float kTail = 1 << E::kTailBits;
  // V's infinities are multiplied apart where a leading part may be 0 (e4m3 has none).
  static constexpr bool kApart = E::kTailBits > 0 && !kFp8;

  float4_t o[S::kJ];
  float m, l;
  x8 q[S::kSteps];

  // Requests the K and V of a cursor's tile, whose rows' places (in 16 bytes
  // from the pool's start) are in LDS.  A cursor past the run's end reads one
  // row over and over.
  static __device__ __forceinline__ void request(const PagedAttnParams& p, const Cursor& at, int units, int set,
                                                 int member, const uint32_t* rows, int lane, Tile& x) {
    x.mask = at.mask;
    x.unit = at.left > 0 ? at.b * units + at.rest : -1;
    x.flags = at.left > 0 ? at.flags | (at.left == 1 ? kLast : 0) : 0;
    const int c = lane & 15, g = lane >> 4;
    const uint32_t krow[2] = {rows[c], rows[16 + c]};
    const u32x4_t vrow[2] = {*reinterpret_cast<const u32x4_t*>(rows + 4 * g),
                             *reinterpret_cast<const u32x4_t*>(rows + 16 + 4 * g)};
    const int64_t head = (static_cast<int>(div_by(at.rest, p.groups)) * set + member) * p.layout.head_stride * S::kCell;
    const uint8_t* kp = static_cast<const uint8_t*>(p.k) + head + 16 * g;
    const uint8_t* vp = static_cast<const uint8_t*>(p.v) + head + c * (S::kChunk * S::kCell);
#pragma unroll
    for (int mt = 0; mt < 2; ++mt) {
      const uint8_t* r = kp + (static_cast<uint64_t>(krow[mt]) << 4);
#pragma unroll
      for (int i = 0; i < S::kKLoads; ++i)
        x.k[mt][i] = __builtin_nontemporal_load(reinterpret_cast<const u32x4_t*>(r + 64 * i));
    }
    __builtin_amdgcn_sched_barrier(0);  // K is used first: V behind it
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const uint8_t* r = vp + (static_cast<uint64_t>(vrow[e >> 2][e & 3]) << 4);
#pragma unroll
      for (int n = 0; n < S::kChunks; ++n)
        load_words<S::kChunkWords>(r + n * (16 * S::kChunk * S::kCell), x.v[e] + n * S::kChunkWords);
    }
    // the use of an earlier tile stays behind these loads
    __builtin_amdgcn_sched_barrier(0);
  }

  static __device__ __forceinline__ x8 words8(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    const u32x4_t r = {a, b, c, d};
    return __builtin_bit_cast(x8, r);
  }

  // K operand of k-step s: bf16 / fp16 as loaded; e4m3 two steps per load.
  static __device__ __forceinline__ x8 k_operand(const Tile& x, int mt, int s) {
    if constexpr (kFp8) {
      const uint32_t a = x.k[mt][s >> 1][2 * (s & 1)], b = x.k[mt][s >> 1][2 * (s & 1) + 1];
      return words8(E::template pair_of_fp8<false>(a), E::template pair_of_fp8<true>(a),
                    E::template pair_of_fp8<false>(b), E::template pair_of_fp8<true>(b));
    } else {
      return __builtin_bit_cast(x8, x.k[mt][s]);
    }
  }

  // Channels 2 w, 2 w + 1 of token e's part of V, as a pair of 16-bit values.
  static __device__ __forceinline__ uint32_t v_pair(const Tile& x, int e, int w) {
    if constexpr (kFp8) {
      const uint32_t word = x.v[e][w >> 1];
      return (w & 1) ? E::template pair_of_fp8<true>(word) : E::template pair_of_fp8<false>(word);
    } else {
      return x.v[e][w];
    }
  }

  __device__ __forceinline__ void accumulate(Tile& x, float sc, int lane) {
    const int g = lane >> 4;
    float4_t s[2];
#pragma unroll
    for (int mt = 0; mt < 2; ++mt) {
      s[mt] = float4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int i = 0; i < S::kSteps; ++i) s[mt] = E::mfma(k_operand(x, mt, i), q[i], s[mt]);
    }
    if (x.mask != 0xFFFFFFFFu) {
      // tokens that are not attended: score -inf (whatever their row holds),
      // V 0, so that 0 * Inf and 0 * NaN never form
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        if (!((x.mask >> ((e & 4) * 4 + 4 * g + (e & 3))) & 1)) {
          s[e >> 2][e & 3] = -kInf;
#pragma unroll
          for (int w = 0; w < S::kVWords; ++w) x.v[e][w] = 0;
        }
      }
    }
    // (sc is positive: the largest score is the largest product)
    float top = s[0][0], low = top;
#pragma unroll
    for (int e = 1; e < 8; ++e) {
      top = fmaxf(top, s[e >> 2][e & 3]);
      if constexpr (kApart) low = fminf(low, s[e >> 2][e & 3]);
    }
    top = across_max(top) * sc - E::kUp;
    const auto lost = [&]() {  // a weight whose leading part may be 0
      if constexpr (kApart) return fmaf(low, sc, m == -kInf ? 0.0f : -m) < E::kLeadBits;
      return false;
    };
    if (__any(top > m + E::kLazyBits || lost())) {
      const float now = vmax(m, top);
      // (m = -inf: nothing summed yet; a lane that stays at -inf keeps its zeros)
      const float a = now == -kInf ? 1.0f : __builtin_amdgcn_exp2f(m - now);
      m = now;
      l *= a;
#pragma unroll
      for (int j = 0; j < S::kJ; ++j) o[j] *= a;
      if constexpr (kApart)
        if (__any(lost()) && has_wild(x)) take_wild(x, s, sc);
    }
    const float base = m == -kInf ? 0.0f : m;
    uint32_t parts[E::kParts][4];
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
      float p0 = __builtin_amdgcn_exp2f(fmaf(s[e >> 2][e & 3], sc, -base));
      float p1 = __builtin_amdgcn_exp2f(fmaf(s[e >> 2][(e & 3) + 1], sc, -base));
      l += p0 + p1;
#pragma unroll
      for (int n = 0; n < E::kParts; ++n) {
        if (E::kTailBits > 0 && n > 0) p0 *= kTail, p1 *= kTail;
        if (!kFp8 && n > 0) p0 = fmaxf(p0, E::kLeast), p1 = fmaxf(p1, E::kLeast);  // (e4m3 has no infinities)
        parts[n][e >> 1] = E::cut(p0, p1);
      }
    }
#pragma unroll
    for (int w = 0; w < S::kJ / 2; ++w) {
      uint32_t r[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) r[e] = v_pair(x, e, w);
      const x8 even = even_of(r), odd = odd_of(r);
      if constexpr (E::kTailBits > 0) {
        const x8 tail = words8(parts[1][0], parts[1][1], parts[1][2], parts[1][3]);
        const float4_t a = E::mfma(even, tail, float4_t{}), b = E::mfma(odd, tail, float4_t{});
        const x8 lead = words8(parts[0][0], parts[0][1], parts[0][2], parts[0][3]);
        o[2 * w] = E::mfma(even, lead, o[2 * w]);
        o[2 * w + 1] = E::mfma(odd, lead, o[2 * w + 1]);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          o[2 * w][i] = fmaf(a[i], 1.0f / kTail, o[2 * w][i]);
          o[2 * w + 1][i] = fmaf(b[i], 1.0f / kTail, o[2 * w + 1][i]);
        }
      } else {
#pragma unroll
        for (int n = 0; n < E::kParts; ++n) {
          const x8 pn = words8(parts[n][0], parts[n][1], parts[n][2], parts[n][3]);
          o[2 * w] = E::mfma(even, pn, o[2 * w]);
          o[2 * w + 1] = E::mfma(odd, pn, o[2 * w + 1]);
        }
      }
    }
  }

  // Whether V holds an infinity or a NaN: those times 0 are NaN, everything else
  // is 0.
  static __device__ __forceinline__ bool has_wild(const Tile& x) {
    half2_t sum[4] = {};
#pragma unroll
    for (int e = 0; e < 8; ++e)
#pragma unroll
      for (int w = 0; w < S::kVWords; ++w)
        sum[w & 3] = __builtin_elementwise_fma(__builtin_bit_cast(half2_t, x.v[e][w]), half2_t{0, 0}, sum[w & 3]);
    sum[0] = (sum[0] + sum[1]) + (sum[2] + sum[3]);
    return __any(__builtin_bit_cast(uint32_t, sum[0]) & 0x7FFF7FFFu);
  }

  // V's infinities and NaN times 1 where a weight is not 0, and out of V.
  __device__ __forceinline__ void take_wild(Tile& x, const float4_t (&s)[2], float sc) {
    const float base = m == -kInf ? 0.0f : m;
    uint32_t one[4];
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
      const float p0 = __builtin_amdgcn_exp2f(fmaf(s[e >> 2][e & 3], sc, -base));
      const float p1 = __builtin_amdgcn_exp2f(fmaf(s[e >> 2][(e & 3) + 1], sc, -base));
      one[e >> 1] = (p0 > 0.0f ? 0x3C00u : 0u) | (p1 > 0.0f ? 0x3C000000u : 0u);
    }
    const x8 pn = words8(one[0], one[1], one[2], one[3]);
#pragma unroll
    for (int w = 0; w < S::kJ / 2; ++w) {
      uint32_t r[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const uint32_t v = x.v[e][w];
        const uint32_t which = ((v & 0x7C00u) == 0x7C00u ? 0xFFFFu : 0u) | ((v & 0x7C000000u) == 0x7C000000u ? 0xFFFF0000u : 0u);
        r[e] = v & which;
        x.v[e][w] = v & ~which;
      }
      o[2 * w] = E::mfma(even_of(r), pn, o[2 * w]);
      o[2 * w + 1] = E::mfma(odd_of(r), pn, o[2 * w + 1]);
    }
  }

  // One channel of eight tokens out of their words of two.
  static __device__ __forceinline__ x8 even_of(const uint32_t (&r)[8]) {
    return words8(__builtin_amdgcn_perm(r[1], r[0], 0x05040100u), __builtin_amdgcn_perm(r[3], r[2], 0x05040100u),
                  __builtin_amdgcn_perm(r[5], r[4], 0x05040100u), __builtin_amdgcn_perm(r[7], r[6], 0x05040100u));
  }
  static __device__ __forceinline__ x8 odd_of(const uint32_t (&r)[8]) {
    return words8(__builtin_amdgcn_perm(r[1], r[0], 0x07060302u), __builtin_amdgcn_perm(r[3], r[2], 0x07060302u),
                  __builtin_amdgcn_perm(r[5], r[4], 0x07060302u), __builtin_amdgcn_perm(r[7], r[6], 0x07060302u));
  }

  // q of a unit as the B operand, in the channel order of the K operand's k-steps.
  // A negative scale is taken as its magnitude and the negated q.
  __device__ __forceinline__ void load_q(const PagedAttnParams& p, int b, int head0, int heads, bool negate, int lane) {
    const int c = lane & 15, g = lane >> 4;
    const uint16_t* qr = p.q + b * p.q_sb + (head0 + min(c, heads - 1)) * p.q_sh;
#pragma unroll
    for (int i = 0; i < S::kSteps; ++i) {
      const int ch = kFp8 ? 64 * (i >> 1) + 16 * g + 8 * (i & 1) : 32 * i + 8 * g;
      q[i] = __builtin_bit_cast(x8, *reinterpret_cast<const u32x4_t*>(qr + ch));
    }
    if (negate) {
#pragma unroll
      for (int i = 0; i < S::kSteps; ++i)
        q[i] = __builtin_bit_cast(x8, __builtin_bit_cast(u32x4_t, q[i]) ^ 0x80008000u);
    }
  }
  // Uses, and so waits for, q: pending at every tile of the loop its loads
  // would make each wait for the newest requests.
  __device__ __forceinline__ void settle_q() {
#pragma unroll
    for (int i = 0; i < S::kSteps; ++i) asm volatile("" : "+v"(q[i]));
  }

  // output row r's (of this lane's four) channels j .. j + 3
  __device__ __forceinline__ float4_t four(int j, int r) const {
    return float4_t{o[j][r], o[j + 1][r], o[j + 2][r], o[j + 3][r]};
  }

  __device__ __forceinline__ void start() {
    m = -kInf;
    l = 0.0f;
#pragma unroll
    for (int j = 0; j < S::kJ; ++j) o[j] = float4_t{0.0f, 0.0f, 0.0f, 0.0f};
  }
};

// Four results (of one head, on 4 channels).
template <int kType>
__device__ __forceinline__ void store_result(const PagedAttnParams& p, int64_t at, const float4_t& v) {
  if (p.out_f32)
    *reinterpret_cast<float4_t*>(static_cast<float*>(p.out) + at) = v;
  else
    *reinterpret_cast<u32x2_t*>(static_cast<uint16_t*>(p.out) + at) =
        u32x2_t{f32_to_elem<kType>(v[0]) | (f32_to_elem<kType>(v[1]) << 16),
                f32_to_elem<kType>(v[2]) | (f32_to_elem<kType>(v[3]) << 16)};
}

__device__ __forceinline__ float natural_lse(float m, float l) {
  return l == 0.0f ? -kInf : (m + __log2f(l)) * kLn2v;
}

// LDS before the partials: the counters of a workgroup, the rows of each wave's
// next tile, and a place per request.
__host__ __device__ constexpr size_t counter_bytes(int waves, int bs) {
  return static_cast<size_t>((4 * waves + 2 + 3) / 4 + kTile * waves / 4 + (bs + 1 + 3) / 4) * 16;
}

// One unit of the line.
struct Unit {
  int b, head0, heads;       // request, first query head, query heads (of a set: of all of its KV heads)
  int base, tiles;           // first place on the line (its tiles start kUnitCost further), tiles
};

template <int kType, bool kFp8, int kD, bool kSets>
__global__ __launch_bounds__((64 * Shape<kFp8, kD>::kWaves)) void paged_attention_kernel(const PagedAttnParams p) {
  using S = Shape<kFp8, kD>;
  constexpr int kWaves = S::kWaves, kThreads = 64 * kWaves, kSlots = 2 * kWaves;
  constexpr int kFan = 2 * kWaves;  // partials of a first step of the last join, where it has two
  constexpr int kItems = std::max(1, kHeads * (kD / 4) / kThreads);  // of the last join, of a thread
  constexpr int kRow = kD + 4;  // row stride of a partial in LDS: 4 banks of skew between heads
  extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
  int* s_unit = reinterpret_cast<int*>(smem);  // [kSlots]: unit of a partial or -1
  int* s_part = s_unit + kSlots;               // [kWaves + 2]: scan, last-arrival flags
  int* s_done = s_part + kWaves + 2;           // [kWaves]: tiles done
  uint32_t* s_rows = reinterpret_cast<uint32_t*>(smem + 16 * ((4 * kWaves + 2 + 3) / 4));  // [kWaves][kTile]
  int* s_cum = reinterpret_cast<int*>(s_rows + kTile * kWaves);  // [bs + 1]: places of the requests before, per unit
  // (the last join uses the partials' space anew, beyond s_ml if it must: it comes last)
  float* s_o = reinterpret_cast<float*>(smem + counter_bytes(kWaves, p.bs));  // [kSlots][heads][kRow]
  float* s_ml = s_o + kSlots * p.heads_lds * kRow;                            // [kSlots][heads][2]
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);

  // --- places of every request, and their running sum -----------------------
  const auto len_of = [&](int b) { return min(max(p.lens[b], 0), p.max_len); };
  const auto tile0_of = [&](int len) { return p.window > 0 ? max(0, len - p.window) / kTile : 0; };
  const auto tiles_of = [&](int len) { return (len + kTile - 1) / kTile - tile0_of(len); };
  const bool few = p.bs <= 64;
  int ends = 0, total = 0;  // few requests: the places up to the lane's one's end
  if (few) {
    // every wave for itself, without a barrier (all write the same; 16 requests
    // of 700 tokens 16.2 -> 15.7 us)
    const int n = lane < p.bs ? tiles_of(len_of(lane)) : 0;
    ends = scan64(n ? n + kUnitCost : 0);
    if (lane < p.bs) s_cum[lane + 1] = ends;
    if (lane == 0) s_cum[0] = 0, s_done[wave] = 0;
    if (lane < kSlots / kWaves) s_unit[kSlots / kWaves * wave + lane] = -1;
    total = __builtin_amdgcn_readlane(ends, 63);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  } else {
    const int per = (p.bs + kThreads - 1) / kThreads;
    const int b0 = min(tid * per, p.bs), b1 = min(b0 + per, p.bs);
    int mine = 0;
    for (int b = b0; b < b1; ++b) {
      const int n = tiles_of(len_of(b));
      s_cum[b] = n ? n + kUnitCost : 0;
      mine += s_cum[b];
    }
    const int scan = scan64(mine);
    if (lane == 63) s_part[wave] = scan;
    if (tid < kSlots) s_unit[tid] = -1;
    if (tid < kWaves) s_done[tid] = 0;
    __syncthreads();
    int sum = scan - mine;
    for (int w = 0; w < kWaves; ++w) {
      if (w < wave) sum += s_part[w];
      total += s_part[w];
    }
    for (int b = b0; b < b1; ++b) {
      const int n = s_cum[b];
      s_cum[b] = sum;
      sum += n;
    }
    if (tid == 0) s_cum[p.bs] = total;
    __syncthreads();
  }
  total = __builtin_amdgcn_readfirstlane(total);
  const int grid = static_cast<int>(gridDim.x);
  const bool sets = kSets && total * static_cast<int>(p.units.d) >= kSetPlaces * kWaves * grid;
  const FastDiv units_div = sets ? p.sets : p.units;
  const int units = static_cast<int>(units_div.d), set = sets ? p.set : 1, member = wave & (set - 1);
  const int runs = kWaves / set;  // the workgroup's run is cut into
  total *= units;

  // --- requests without a token: zeros -------------------------------------
  for (int b = blockIdx.x; b < p.bs; b += gridDim.x) {
    if (s_cum[b + 1] != s_cum[b]) continue;
    const int64_t row = static_cast<int64_t>(b) * p.hq;
    for (int i = tid; i < p.hq * (kD / 4); i += kThreads)
      store_result<kType>(p, row * kD + 4 * i, float4_t{0.0f, 0.0f, 0.0f, 0.0f});
    if (p.lse)
      for (int i = tid; i < p.hq; i += kThreads) p.lse[row + i] = -kInf;
  }

  // --- this workgroup's run of places --------------------------------------
  const auto cum = [&](int b) { return __builtin_amdgcn_readfirstlane(s_cum[b]); };
  // the request that place x belongs to (`cum` for a place of the whole wave,
  // plain reads where each lane has its own)
  const auto request_at = [&](int x, auto cum) {
    const int at = static_cast<int>(div_by(x, units_div));
    int lo = 0, hi = p.bs - 1;
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (cum(mid + 1) > at)
        hi = mid;
      else
        lo = mid + 1;
    }
    return lo;
  };
  const int chunk = max(runs, (total + grid - 1) / grid);
  // both ends of the run, one a lane
  const int64_t y64 = (static_cast<int64_t>(blockIdx.x) + (lane & 1)) * chunk;
  int end = static_cast<int>(min(y64, static_cast<int64_t>(total)));
  const bool small = 2 * kSmallUnit <= chunk && total / kSmallUnit < p.bs * units;
  if (!sets && (chunk == kWaves || small) && y64 < total) {
    const int b = request_at(end, [&](int i) { return s_cum[i]; });
    const int size = s_cum[b + 1] - s_cum[b], in = (end - s_cum[b] * units) % size;
    if (size <= (chunk == kWaves ? S::kWholeTiles + kUnitCost : kSmallUnit)) end += 2 * in < size ? -in : size - in;
  }
  const int wg0 = __builtin_amdgcn_readlane(end, 0), wg1 = __builtin_amdgcn_readlane(end, 1);
  if (wg0 >= wg1) return;
  const auto unit_at = [&](int id) {
    Unit u;
    u.b = static_cast<int>(div_by(id, units_div));
    const int rest = id - u.b * units;
    const int kvh = static_cast<int>(div_by(rest, p.groups)), group = rest - kvh * static_cast<int>(p.groups.d);
    u.heads = min(kHeads, set * p.gqa - kHeads * group);
    u.head0 = kvh * set * p.gqa + kHeads * group;
    const int size = cum(u.b + 1) - cum(u.b);
    u.tiles = size - kUnitCost;
    u.base = cum(u.b) * units + rest * size;
    return u;
  };
  const auto v_scale_of = [&](int head) { return kFp8 && p.v_scale ? p.v_scale[head / p.gqa] : 1.0f; };

  // --- the wave's stream of tiles -------------------------------------------
  const int share = (wg1 - wg0 + runs - 1) / runs;
  const int x0 = wg0 + wave / set * share, x1 = min(x0 + share, wg1);
  if (x0 < x1) {
    Cursor at;
    uint32_t* rows = s_rows + kTile * wave;
    int tile0, first;  // the request's first tile and first token
    const uint32_t page16 = static_cast<uint32_t>(p.layout.page_stride * S::kCell / 16);
    const uint32_t token16 = static_cast<uint32_t>(p.layout.token_stride * S::kCell / 16);
    const auto enter = [&](int b) {  // a request's numbers
      at.b = b;
      at.len = len_of(b);
      tile0 = tile0_of(at.len);
      first = p.window > 0 ? at.len - p.window : 0;
      at.tiles = cum(b + 1) - cum(b) - kUnitCost;
    };
    const auto part = [&](int from) {  // the wave's part of the unit: its tiles from `from` on
      const int end = min(at.tiles, x1 - at.base - kUnitCost);
      at.tile = tile0 + from;
      at.left = max(0, end - from);
      at.flags = kFirst | (at.left == at.tiles ? kWhole : 0);
    };
    const auto next_unit = [&]() {
      at.base += at.tiles + kUnitCost;
      at.left = 0;
      if (at.base + kUnitCost >= x1) return;  // (x1 is at most the line's end: there is a next unit)
      if (++at.rest == units) {
        at.rest = 0;
        int b = at.b + 1;
        while (cum(b + 1) == cum(b)) ++b;
        enter(b);
      }
      part(0);
    };
    // Page ids: 64 consecutive entries of the request's table row at a time,
    // one a lane, handed out by ds_bpermute.  The load is waited for where it
    // is made (the asm uses its value): a load that might be pending at every
    // tile would make every tile wait for all but the newest request.
    int window = 0, window0 = 0, window_of = -1;
    // places of the present tile's tokens (past the end: of the last), and
    // which of them are attended
    const auto look_up = [&]() {
      const int t0 = at.tile * kTile, t1 = min(t0 + kTile, at.len) - 1;
      const int e0 = static_cast<int>(div_by(t0, p.page)), e1 = static_cast<int>(div_by(t1, p.page));
      if (at.b != window_of || e0 < window0 || e1 >= window0 + 64) {
        window_of = at.b;
        window0 = e0;
        window = p.table[at.b * p.table_stride + min(e0 + lane, static_cast<int>(div_by(at.len - 1, p.page)))];
        asm volatile("" : "+v"(window));
      }
      const int t = t0 + (lane & 31), tc = min(t, t1);
      const uint32_t entry = div_by(tc, p.page), in_page = tc - entry * p.page.d;
      const uint32_t page = __builtin_amdgcn_ds_bpermute(4 * (static_cast<int>(entry) - window0), window);
      const bool there = at.left > 0 && page < static_cast<uint32_t>(p.layout.num_pages);
      rows[lane & 31] = (there ? page : 0) * page16 + (there ? in_page : 0) * token16;
      at.mask = static_cast<uint32_t>(__ballot(there && t <= t1 && t >= first));
    };
    const auto advance = [&]() {
      if (at.left > 1) {
        --at.left;
        ++at.tile;
        at.flags &= ~kFirst;
      } else if (at.left == 1) {
        next_unit();
      }
      look_up();
    };
    enter(few ? __builtin_popcountll(__ballot(ends <= static_cast<int>(div_by(x0, units_div)))) : request_at(x0, cum));
    {
      const int size = at.tiles + kUnitCost, from = x0 - cum(at.b) * units;
      at.rest = from / size;
      at.base = x0 - from + at.rest * size;
      part(max(0, x0 - at.base - kUnitCost));
      if (at.left == 0) next_unit();
    }
    PagedAttn<kType, kFp8, kD> attn;
    float sc = 0.0f;
    const auto mine_of = [&](Unit u) {  // the wave's KV head of a set
      if (sets) u.heads = p.gqa, u.head0 += member * p.gqa;
      return u;
    };
    const auto begin_unit = [&](int id) {
      const Unit u = mine_of(unit_at(id));
      sc = p.scale * (kFp8 && p.k_scale ? p.k_scale[u.head0 / p.gqa] : 1.0f);
      attn.load_q(p, u.b, u.head0, u.heads, sc < 0.0f, lane);
      // (positive also for a scale of 0, whose product with -Inf would be NaN)
      sc = sc != sc ? sc : fmaxf(fabsf(sc), 0x1p-120f);
      attn.start();
    };
    begin_unit(at.b * units + at.rest);  // (its q and the first page ids in one round trip)
    look_up();
    attn.settle_q();
    TileRegs<kFp8, kD> ring[S::kDepth];
    int slot = kSlots / kWaves * wave, done = 0;
#pragma unroll
    for (int i = 0; i < S::kDepth - 1; ++i) {
      attn.request(p, at, units, set, member, rows, lane, ring[i]);
      advance();
    }
    ring[0].flags &= ~kFirst;
    do {
#pragma unroll
      for (int i = 0; i < S::kDepth; ++i) {
        TileRegs<kFp8, kD>& x = ring[i];
        if (x.flags & kFirst) {
          begin_unit(x.unit);
          attn.settle_q();
        }
        attn.request(p, at, units, set, member, rows, lane, ring[(i + S::kDepth - 1) % S::kDepth]);
        advance();
        // The tile's loads are older than those of the kDepth - 1 requests
        // behind it: waited for here by count, on every path, or a path that
        // seems to pass them by would make the compiler wait for the newest.
        wait_vmcnt<(S::kDepth - 1) * S::kLoads>();
        if (x.unit < 0) continue;
        attn.accumulate(x, sc, lane);
        if constexpr (kWaves == 8) {
          ++done;
          __hip_atomic_store(&s_done[wave], done, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
          const int other = __hip_atomic_load(&s_done[wave ^ 4], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
          if (__builtin_amdgcn_readfirstlane(other) > done)
            __builtin_amdgcn_s_setprio(1);
          else
            __builtin_amdgcn_s_setprio(0);
        }
        if (x.flags & kLast) {
          const Unit u = mine_of(unit_at(x.unit));
          const int c = lane & 15, g = lane >> 4;
          const float l = across_sum(attn.l);
          if (x.flags & kWhole) {
            if (c < u.heads) {
              const float inv = (l == 0.0f ? 0.0f : 1.0f / l) * v_scale_of(u.head0);
              const int64_t row = static_cast<int64_t>(u.b) * p.hq + u.head0 + c;
#pragma unroll
              for (int r = 0; r < 4; ++r)
#pragma unroll
                for (int n = 0; n < S::kChunks; ++n) {
                  const int64_t at0 = row * kD + S::channel(4 * g + r, n);
#pragma unroll
                  for (int j = 0; j < S::kChunk; j += 4)
                    store_result<kType>(p, at0 + j, attn.four(n * S::kChunk + j, r) * inv);
                }
              if (p.lse && g == 0) p.lse[row] = natural_lse(attn.m, l);
            }
          } else {
            // at most the run's first and last unit are cut
            if (c < u.heads) {
              float* dst = s_o + (slot * p.heads_lds + c) * kRow;
#pragma unroll
              for (int r = 0; r < 4; ++r)
#pragma unroll
                for (int n = 0; n < S::kChunks; ++n)
#pragma unroll
                  for (int j = 0; j < S::kChunk; j += 4)
                    *reinterpret_cast<float4_t*>(dst + S::channel(4 * g + r, n) + j) = attn.four(n * S::kChunk + j, r);
              if (g == 0) {
                s_ml[(slot * p.heads_lds + c) * 2] = attn.m;
                s_ml[(slot * p.heads_lds + c) * 2 + 1] = l;
              }
            }
            if (lane == 0) s_unit[slot] = x.unit;
            ++slot;
          }
        }
      }
    } while (ring[0].unit >= 0);
    __builtin_amdgcn_s_setprio(0);
  }
  __syncthreads();

  // --- join the waves' partials --------------------------------------------
  // 64 items (four channels of a head) of a unit a wave at a time
  int ids[kSlots];
#pragma unroll
  for (int i = 0; i < kSlots; ++i) ids[i] = __builtin_amdgcn_readfirstlane(s_unit[i]);
  const int slot_unit = lane < kSlots ? s_unit[lane] : -1;
  // the first slot of each unit: they ascend (through one wave of each run)
  const bool taken = slot_unit >= 0 && (lane / (kSlots / kWaves) & (set - 1)) == 0;
  const uint32_t below = static_cast<uint32_t>(__ballot(taken)) & ((1u << (lane & 31)) - 1);
  const int before = __builtin_amdgcn_ds_bpermute(4 * (31 - __builtin_clz(below | 1)), slot_unit);
  const uint32_t firsts = static_cast<uint32_t>(__ballot(taken && (below == 0 || before != slot_unit)));
  if (!firsts) return;
  const auto starts = [&](const Unit& u) { return u.base + kUnitCost >= wg0; };
  const auto whole = [&](const Unit& u) { return starts(u) && u.base + kUnitCost + u.tiles <= wg1; };
  const auto unit_of_slot = [&](int i) { return __builtin_amdgcn_readlane(slot_unit, i); };
  const __amdgpu_buffer_rsrc_t part_o =
      __builtin_amdgcn_make_buffer_rsrc(p.part_o, 0, kMaxGroups * 2 * kHeads * kD * 4, 0x00020000);
  const int per_unit = (set * p.heads_lds * (kD / 4) + 63) / 64;
  uint32_t rest = firsts;
#pragma unroll 1
  for (int at64 = wave;; at64 += kWaves) {
    for (; rest && at64 >= per_unit; at64 -= per_unit) rest &= rest - 1;
    if (!rest) break;
    const int id = unit_of_slot(__builtin_ctz(rest));
    const Unit u = unit_at(id);
    const int e = 64 * at64 + lane;
    if (e < u.heads * (kD / 4)) {
      const int c = e / (kD / 4), d = 4 * (e % (kD / 4));
      // (a set's KV heads are the neighbouring waves')
      const int of = sets ? c / p.gqa : 0, at = c - of * p.gqa;
      const auto has = [&](int i) { return ids[i] == id && (i / (kSlots / kWaves) & (set - 1)) == of; };
      float mv[kSlots], lv[kSlots], top = -kInf;
#pragma unroll
      for (int i = 0; i < kSlots; ++i) {
        const float2_t ml = *reinterpret_cast<const float2_t*>(s_ml + (i * p.heads_lds + at) * 2);
        mv[i] = has(i) ? ml[0] : -kInf;
        lv[i] = has(i) ? ml[1] : 0.0f;
        top = fmaxf(top, mv[i]);
      }
      const float base = top == -kInf ? 0.0f : top;
      float den = 0.0f;
      float4_t num = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int i = 0; i < kSlots; ++i) {
        if (!has(i)) continue;
        const float w = __builtin_amdgcn_exp2f(mv[i] - base);
        den += w * lv[i];
        num += w * *reinterpret_cast<const float4_t*>(s_o + (i * p.heads_lds + at) * kRow + d);
      }
      if (whole(u)) {
        const float inv = (den == 0.0f ? 0.0f : 1.0f / den) * v_scale_of(u.head0 + c);
        const int64_t row = static_cast<int64_t>(u.b) * p.hq + u.head0 + c;
        store_result<kType>(p, row * kD + d, num * inv);
        if (p.lse && d == 0) p.lse[row] = natural_lse(top, den);
      } else {
        const uint32_t row = (blockIdx.x * 2 + (starts(u) ? 1 : 0)) * kHeads + c;
        store_dev(part_o, row * kD + d, num);
        if (d == 0) store_dev(p.part_ml + row * 2, top, den);
      }
    }
  }

  // --- the last workgroup of a shared unit joins the workgroups' partials ---
  // This lane's partial stores have reached the device's coherence point
  // before the workgroup counts in (write-through stores, waited for), and the
  // joining loads read there: no cache is written back or invalidated.
  // A unit of many workgroups is joined in two steps: the last of each kFan
  // neighbours joins theirs, in the place of the first one's, and the last of
  // those joins what they left.  The counts of a unit's fans are those of the
  // workgroups behind its first one: no unit starts in these.
  int cut[2] = {-1, -1};  // units shared with earlier / later workgroups: at most the first and the last of them
  int w0[2] = {0, 0}, n[2] = {0, 0}, fans[2] = {0, 0};  // first of the workgroups that share it, how many, fans
  const int lo = unit_of_slot(__builtin_ctz(firsts)), hi = unit_of_slot(31 - __builtin_clz(firsts));
#pragma unroll
  for (int side = 0; side < 2; ++side) {
    const int id = side ? hi : lo;
    const Unit u = unit_at(id);
    if (side ? id == cut[0] || whole(u) || !starts(u) : starts(u)) continue;
    cut[side] = id;
    w0[side] = (u.base + kUnitCost) / chunk;
    n[side] = (u.base + kUnitCost + u.tiles - 1) / chunk - w0[side] + 1;
    const auto rounds = [&](int count) {  // of loads, one after the other
      const int at_once = kBatch * max(1, min(kThreads / 2 / (u.heads * (kD / 4)), count));
      return (count + at_once - 1) / at_once;
    };
    const int of = (n[side] + kFan - 1) / kFan;
    if (n[side] > kFan && rounds(n[side]) > rounds(kFan) + rounds(of) + kStepRounds) fans[side] = of;
  }
  if (cut[0] < 0 && cut[1] < 0) return;
  // Four channels of a head per item; an item's partials in as many parts as
  // half of the workgroup has threads for, eight partials requested at once;
  // the parts meet in LDS.  Where two units end here, each has half of the
  // threads, where one does, more items at a time, but not more parts: which
  // of the two end here is a matter of time, and the order of the sums must
  // not follow it.
  bool in0 = cut[0] >= 0, in1 = cut[1] >= 0;  // the sides still to be joined
#pragma unroll 1
  for (int step = 0; step < 2; ++step) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (tid < 2) {  // (both arrivals in one round trip)
      const int first = tid ? w0[1] : w0[0], count = tid ? n[1] : n[0], fans_of = tid ? fans[1] : fans[0];
      const int mine = (static_cast<int>(blockIdx.x) - first) / kFan;
      const bool by_fan = fans_of && step == 0;
      s_part[tid] = (tid ? in1 : in0) &&
                    arrive_last_count(p.arrivals + first + (by_fan ? 1 + mine : 0),
                                      by_fan ? min(kFan, count - kFan * mine) : fans_of ? fans_of : count);
    }
    __syncthreads();
    const bool last0 = __builtin_amdgcn_readfirstlane(s_part[0]), last1 = __builtin_amdgcn_readfirstlane(s_part[1]);
    if (!last0 && !last1) return;
    const bool both = last0 && last1;
    const int side = both ? (wave >= kWaves / 2 ? 1 : 0) : (last1 ? 1 : 0);
    const int width = both ? kThreads / 2 : kThreads, me = both ? tid % (kThreads / 2) : tid;
    const int from = side ? w0[1] : w0[0], all = side ? n[1] : n[0], fanned = side ? fans[1] : fans[0];
    const int fan = fanned ? (static_cast<int>(blockIdx.x) - from) / kFan : 0;
    float* s_mine = s_o + (both ? side * (kThreads / 2 * 8) : 0);  // [part][item][8]
    // (as many passes for both sides: the barriers are the workgroup's)
    const int passes = (set * p.heads_lds * (kD / 4) + kItems * width - 1) / (kItems * width);
    const bool ends = !fanned || step == 1;  // this step gives the unit's result
    const Unit u = unit_at(side ? cut[1] : cut[0]);
    const int count = !fanned ? all : step ? fanned : min(kFan, all - kFan * fan);
    // partial i of the step: the unit's first workgroup kept it as its later
    // cut, the others as their earlier one
    const int begin = fanned && step == 0 ? kFan * fan : 0, stride = fanned && step ? kFan : 1;
    const auto row_of = [&](int i, int c) {
      const int at = begin + i * stride;
      return static_cast<uint32_t>(((from + at) * 2 + (at == 0 ? 1 : 0)) * kHeads + c);
    };
    const int items = u.heads * (kD / 4), parts = max(1, min(kThreads / 2 / items, count));
#pragma unroll 1
    for (int pass = 0; pass < passes; ++pass) {  // (of whole heads)
      const int e0 = pass * kItems * width, here = max(1, min(width, items - e0));
      const int part = me / here, item = me - part * here;
      float top[kItems], den[kItems];
      float4_t num[kItems];
      int head[kItems], d[kItems];
      bool mine[kItems];
#pragma unroll
      for (int j = 0; j < kItems; ++j) {
        const int e = e0 + j * width + item;
        mine[j] = e < items && part < parts;
        head[j] = mine[j] ? e / (kD / 4) : 0;
        d[j] = 4 * (e % (kD / 4));
        top[j] = -kInf;
        den[j] = 0.0f;
        num[j] = float4_t{0.0f, 0.0f, 0.0f, 0.0f};
      }
      for (int i0 = part; i0 < count && mine[0]; i0 += kBatch * parts) {
        float2_t ml[kItems][kBatch];
        float4_t o[kItems][kBatch];
#pragma unroll
        for (int j = 0; j < kItems; ++j) {
          if (e0 + j * width >= items) continue;
#pragma unroll
          for (int i = 0; i < kBatch; ++i) {
            const uint32_t row = row_of(min(i0 + i * parts, count - 1), head[j]);
            ml[j][i] = load_dev(p.part_ml + row * 2);
            o[j][i] = load_dev(part_o, row * kD + d[j]);
          }
        }
#pragma unroll
        for (int j = 0; j < kItems; ++j) {
          if (e0 + j * width >= items) continue;
          float now = top[j];
#pragma unroll
          for (int i = 0; i < kBatch; ++i) now = i0 + i * parts < count ? fmaxf(now, ml[j][i][0]) : now;
          const float base = now == -kInf ? 0.0f : now, a = __builtin_amdgcn_exp2f(top[j] - base);
          top[j] = now;
          den[j] *= a;
          num[j] *= a;
#pragma unroll
          for (int i = 0; i < kBatch; ++i) {
            if (i0 + i * parts >= count) continue;
            const float w = __builtin_amdgcn_exp2f(ml[j][i][0] - base);
            den[j] += w * ml[j][i][1];
            num[j] += w * o[j][i];
          }
        }
      }
      __syncthreads();  // (s_o of the join before is read)
      if (parts > 1 && mine[0]) {  // (one item a thread then)
        float* dst = s_mine + me * 8;
        *reinterpret_cast<float4_t*>(dst) = num[0];
        dst[4] = top[0];
        dst[5] = den[0];
      }
      __syncthreads();
      if (parts > 1 && mine[0] && part == 0) {
#pragma unroll 4
        for (int i = 0; i < parts; ++i) top[0] = fmaxf(top[0], s_mine[(i * here + me) * 8 + 4]);
        const float base = top[0] == -kInf ? 0.0f : top[0];
        den[0] = 0.0f;
        num[0] = float4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
        for (int i = 0; i < parts; ++i) {
          const float* src = s_mine + (i * here + me) * 8;
          const float w = __builtin_amdgcn_exp2f(src[4] - base);
          den[0] += w * src[5];
          num[0] += w * *reinterpret_cast<const float4_t*>(src);
        }
      }
#pragma unroll
      for (int j = 0; j < kItems; ++j) {
        if (!mine[j] || part != 0) continue;
        const int c = head[j];
        if (ends) {
          const float inv = (den[j] == 0.0f ? 0.0f : 1.0f / den[j]) * v_scale_of(u.head0 + c);
          const int64_t row = static_cast<int64_t>(u.b) * p.hq + u.head0 + c;
          store_result<kType>(p, row * kD + d[j], num[j] * inv);
          if (p.lse && d[j] == 0) p.lse[row] = natural_lse(top[j], den[j]);
        } else {
          const uint32_t row = row_of(0, c);
          store_dev(part_o, row * kD + d[j], num[j]);
          if (d[j] == 0) store_dev(p.part_ml + row * 2, top[j], den[j]);
        }
      }
    }
    in0 = last0 && fans[0] && step == 0;
    in1 = last1 && fans[1] && step == 0;
    if (!in0 && !in1) return;
  }
}

size_t workspace_bytes_for(int d) {
  static_assert(kMaxGroups * 4 == ZKV_PAGED_ARRIVAL_BYTES, "arrival counts");
  return static_cast<size_t>(kMaxGroups) * 4 + static_cast<size_t>(kMaxGroups) * 2 * kHeads * (d + 2) * 4;
}

template <int kType, bool kFp8, int kD>
int launch_paged_attention(PagedAttnParams& p, int64_t most_tiles, hipStream_t s) {
  using S = Shape<kFp8, kD>;
  auto kernel = paged_attention_kernel<kType, kFp8, kD, false>;
  p.set = 1;
  if constexpr (kD < 256) {
    if (p.layout.head_stride < p.layout.token_stride && p.layout.token_stride * S::kCell % 512 == 0)
      while (2 * p.set <= S::kWaves && 2 * p.set * p.gqa <= kHeads && p.kv % (2 * p.set) == 0) p.set *= 2;
    if (p.set > 1) kernel = paged_attention_kernel<kType, kFp8, kD, true>;
  }
  p.sets = fast_div(static_cast<uint32_t>(p.kv / p.set));
  // the counters, then the partials (in the last join, 32 bytes a thread)
  const size_t lds = std::max(static_cast<size_t>(2 * S::kWaves) * p.heads_lds * (kD + 6) * 4,
                              static_cast<size_t>(64 * S::kWaves) * 32) +
                     counter_bytes(S::kWaves, p.bs);
  if (lds > 60 * 1024 &&
      hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize,
                          160 * 1024) != hipSuccess)
    return fail(ZKV_ELAUNCH, "zkv_paged_attention: cannot raise the LDS limit to 160 KiB");
  // one workgroup per CU, or as many as the longest lengths the table can
  // hold give a tile for every wave
  const int64_t want = (most_tiles + S::kWaves - 1) / S::kWaves;
  const int grid = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(kMaxGroups, want)));
  kernel<<<grid, 64 * S::kWaves, lds, s>>>(p);
  return check_launch("paged_attention_kernel");
}

template <int kType, bool kFp8>
int launch_by_dim(PagedAttnParams& p, int d, int64_t most_tiles, hipStream_t s) {
  if (d == 64) return launch_paged_attention<kType, kFp8, 64>(p, most_tiles, s);
  if (d == 128) return launch_paged_attention<kType, kFp8, 128>(p, most_tiles, s);
  return launch_paged_attention<kType, kFp8, 256>(p, most_tiles, s);
}

}  // namespace
}  // namespace zkv

using namespace zkv;

extern "C" size_t zkv_paged_attention_workspace_size(int d) {
  return d == 64 || d == 128 || d == 256 ? workspace_bytes_for(d) : 0;
}

extern "C" int zkv_paged_attention(const void* q, int64_t q_sb, int64_t q_sh, int is_f16, const void* k_pages,
                                   const void* v_pages, int is_fp8, const float* k_scale, const float* v_scale,
                                   int num_pages, int page_size, int64_t page_stride, int64_t head_stride,
                                   int64_t token_stride, const int32_t* block_table, int64_t table_stride, int width,
                                   const int32_t* seq_lens, int bs, int hq, int kv, int d, float sm_scale, int window,
                                   void* out, int out_f32, float* lse, void* workspace, size_t workspace_bytes,
                                   zkv_stream_t stream) {
  ZKV_REQUIRE(q && k_pages && v_pages && block_table && seq_lens && out && workspace,
              "zkv_paged_attention: null pointer");
  const PageLayout layout{page_stride, head_stride, token_stride, num_pages, page_size};
  const char* why = check_pages(layout, kv, d, is_fp8 ? 1 : 2);
  ZKV_REQUIRE(why == nullptr, "zkv_paged_attention: %s", why);
  ZKV_REQUIRE(bs >= 1 && bs <= kMaxBatch, "zkv_paged_attention: %d requests outside [1, %d]", bs, kMaxBatch);
  ZKV_REQUIRE(hq >= 1 && hq % kv == 0, "zkv_paged_attention: %d query heads over %d KV heads", hq, kv);
  ZKV_REQUIRE(width >= 1 && table_stride >= 0 && window >= 0, "zkv_paged_attention: width %d, row stride %lld, window %d",
              width, static_cast<long long>(table_stride), window);
  ZKV_REQUIRE(static_cast<int64_t>(width) * page_size < (1ll << 31) - kTile,
              "zkv_paged_attention: a request holds fewer than 2^31 - 32 tokens");
  ZKV_REQUIRE(q_sb % 8 == 0 && q_sh % 8 == 0 &&
                  ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k_pages) |
                    reinterpret_cast<uintptr_t>(v_pages) | reinterpret_cast<uintptr_t>(out)) & 15) == 0,
              "zkv_paged_attention: rows start on 16 bytes");
  ZKV_REQUIRE((reinterpret_cast<uintptr_t>(workspace) & 15) == 0, "zkv_paged_attention: the workspace starts on 16 bytes");
  const int gqa = hq / kv, groups = (gqa + kHeads - 1) / kHeads;
  const int64_t most_tiles = static_cast<int64_t>(bs) * kv * groups *
                             ((static_cast<int64_t>(width) * page_size + kTile - 1) / kTile + 1 + kUnitCost);
  // (places on the line are 31-bit numbers)
  ZKV_REQUIRE(most_tiles < (1ll << 31) - (1 << 20),
              "zkv_paged_attention: %d requests of %d KV heads over %lld tokens are too many tiles for one call", bs, kv,
              static_cast<long long>(width) * page_size);
  // (rows are found by 32-bit numbers of 16 bytes)
  ZKV_REQUIRE(((num_pages - 1) * page_stride + (page_size - 1) * token_stride) * (is_fp8 ? 1 : 2) < (1ll << 36),
              "zkv_paged_attention: the rows of a pool start within 64 GiB");
  if (workspace_bytes < workspace_bytes_for(d))
    return fail(ZKV_ESPACE, "zkv_paged_attention: workspace of %zu bytes, %zu needed", workspace_bytes,
                workspace_bytes_for(d));
  PagedAttnParams p{};
  p.q = static_cast<const uint16_t*>(q);
  p.q_sb = q_sb;
  p.q_sh = q_sh;
  p.k = k_pages;
  p.v = v_pages;
  p.k_scale = k_scale;
  p.v_scale = v_scale;
  p.layout = layout;
  p.page = fast_div(static_cast<uint32_t>(page_size));
  p.table = block_table;
  p.table_stride = table_stride;
  p.lens = seq_lens;
  p.out = out;
  p.lse = lse;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  p.arrivals = reinterpret_cast<unsigned int*>(ws);
  ws += kMaxGroups * 4;
  p.part_ml = reinterpret_cast<float*>(ws);
  p.part_o = p.part_ml + static_cast<size_t>(kMaxGroups) * 2 * kHeads * 2;
  p.units = fast_div(static_cast<uint32_t>(kv * groups));
  p.groups = fast_div(static_cast<uint32_t>(groups));
  p.scale = sm_scale * kLog2e;
  p.bs = bs;
  p.hq = hq;
  p.kv = kv;
  p.gqa = gqa;
  p.window = window;
  p.out_f32 = out_f32;
  p.max_len = width * page_size;
  p.heads_lds = std::min(gqa, kHeads);
  auto s = reinterpret_cast<hipStream_t>(stream);
  if (is_f16) return is_fp8 ? launch_by_dim<kF16, true>(p, d, most_tiles, s) : launch_by_dim<kF16, false>(p, d, most_tiles, s);
  return is_fp8 ? launch_by_dim<kBf16, true>(p, d, most_tiles, s) : launch_by_dim<kBf16, false>(p, d, most_tiles, s);
}
