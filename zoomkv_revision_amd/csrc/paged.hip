// The paged cache's bookkeeping and writes (gfx950):
//
//  * page_advance_kernel: one step of a batch's page tables.  Request i goes
//    from len_i to len_i + new_i tokens; pages are taken from the head of a
//    ring of free page ids and given back behind its last, the block table
//    grows in place, and every new token gets its slot (page * page_size +
//    offset) and position.
//  * paged_write_kernel: rows of K and V into their slots, as they are or as
//    e4m3 codes of row / scale.
//  * paged_rope_kernel: RMSNorm and rotary embedding of the q and k heads of a
//    decode batch, each row at its own position, and the K / V rows into their
//    slots.
#include "paged_common.hpp"

#include <algorithm>

namespace zkv {
namespace {

// ---------------------------------------------------------------------------
// page tables
// ---------------------------------------------------------------------------
constexpr int kMaxRequests = 8192;      // the scans' LDS: 16 bytes a request
// Beyond either: 1024 threads, so that one scans at most 8 requests and fewer
// workgroups scan (decode steps of 100 requests 4.4 us, 4.9 with 1024 threads;
// of 300 6.0, 5.1; 128 requests with 65536 slots 8.0, 5.9).
constexpr int kFewRequests = 256, kFewSlots = 8192;
constexpr uint32_t kGranted = 0x80000000u;

struct AdvanceParams {
  const int32_t* lens;
  int32_t* lens_out;
  const int32_t* new_tokens;
  int32_t* table;
  int64_t table_stride;
  int32_t* ring;
  int32_t* state;      // [head, free pages, status bits, arrivals]
  int32_t* state_out;
  int64_t* slots;
  int32_t* positions;  // or null
  int32_t* starts;     // or null
  int requests, num_pages, cap;
  FastDiv page;
  FastDiv row;         // d > 0: request i's tokens end row i of d places; else packed in request order
  int64_t max_len;     // width * page size
};

// Sum of two non-negative numbers up to a limit (associative, so a scan of
// such sums is one of the true sums, limited).
__device__ __forceinline__ int limited(int a, int b, int top) {  // (two limits may pass 31 bits)
  return static_cast<int>(min(static_cast<unsigned>(a) + static_cast<unsigned>(b), static_cast<unsigned>(top)));
}

// Running limited sum over the wave's lanes, this one's included (over rows of
// 16 lanes only if !kAll).
template <bool kAll>
__device__ __forceinline__ int scan_lanes(int v, int top) {
  v = limited(v, __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, false), top);  // from 1, 2, 4, 8 lanes before
  v = limited(v, __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, false), top);
  v = limited(v, __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, false), top);
  v = limited(v, __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, false), top);
  if constexpr (kAll) {
    v = limited(v, __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false), top);  // the last of the row before
    v = limited(v, __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false), top);  // the last of lane 31
  }
  return v;
}

// The limited sums of kN values over the threads before this one, in one pass
// (part: kN x 16, no two calls the same).
template <int kN>
__device__ __forceinline__ void scan_before(int (&v)[kN], int top, int (*part)[16]) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int up[kN];
#pragma unroll
  for (int i = 0; i < kN; ++i) {
    const int sum = scan_lanes<true>(v[i], top);
    up[i] = __builtin_amdgcn_update_dpp(0, sum, 0x138, 0xF, 0xF, false);  // of the lane before
    if (lane == 63) part[i][wave] = sum;
  }
  __syncthreads();
  const int waves = blockDim.x >> 6;
#pragma unroll
  for (int i = 0; i < kN; ++i) {
    const int sums = scan_lanes<false>((lane & 15) < waves ? part[i][lane & 15] : 0, top);
    v[i] = limited(up[i], wave ? __builtin_amdgcn_readlane(sums, wave - 1) : 0, top);
  }
}

__device__ __forceinline__ int pages_of(uint32_t n, const FastDiv& page) {
  const uint32_t q = div_by(n, page);
  return static_cast<int>(q + (q * page.d != n));
}

// First i of ends[0 .. n) with ends[i] > x (n - 1 at most).
__device__ __forceinline__ int owner_of(const int* ends, int n, int x) {
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (ends[mid] > x)
      hi = mid;
    else
      lo = mid + 1;
  }
  return lo;
}

// Every workgroup scans the whole batch (16 bytes a request, from the caches)
// and then serves its share of the tokens and of the pages given back: no
// second launch, no order between workgroups.  The lengths and the state are
// written by the workgroup that counts in last, when every workgroup has read
// them, so they may be updated in place; a captured step replays on the
// lengths that the step before it left.  The pages taken and those given back
// are different places of the ring (together they are at most all of it), and
// a request either grows or shrinks, so no workgroup reads what another
// writes.
//
// Bound by latency: one read of the batch, one LDS search and one dependent
// read of a page id per token.  4.9 us for 64 requests of one token; 1024 mixed
// requests with 65536 slots 7.1 us, 8192 requests 20 us.
template <int kThreads>
__global__ __launch_bounds__(kThreads) void page_advance_kernel(const AdvanceParams p) {
  extern __shared__ int smem[];
  const int R = p.requests, tid = threadIdx.x;
  uint32_t* s_len = reinterpret_cast<uint32_t*>(smem);  // length; kGranted: grows in this step
  int* s_tok = smem + R;                                // ends of the requests' tokens (rows: how many)
  int* s_need = s_tok + R;                              // ends of the pages they take
  int* s_give = s_need + R;                             // ends of the pages they give back
  __shared__ int part[3][16];
  __shared__ int s_status, s_taken, s_last;
  const int head = static_cast<int>(static_cast<uint32_t>(p.state[0]) % static_cast<uint32_t>(p.num_pages));
  const int count = min(max(p.state[1], 0), p.num_pages);
  const int old_status = p.state[2];
  if (tid == 0) {
    s_status = 0;
    s_taken = 0;
  }
  // the batch in one coalesced read (its lengths and new tokens as they are)
#pragma unroll 4
  for (int i = tid; i < R; i += kThreads) {
    s_len[i] = static_cast<uint32_t>(p.lens[i]);
    s_tok[i] = p.new_tokens[i];
  }
  __syncthreads();
  const int per = (R + kThreads - 1) / kThreads;
  const int i0 = min(tid * per, R), i1 = min(i0 + per, R);
  const int tok_top = p.cap + 1, page_top = p.num_pages + 1;
  // tokens: every request's new ones count, whether or not it is served, so
  // that the rows of a packed batch keep their places
  const int row = static_cast<int>(p.row.d);
  int sum = 0;
  for (int i = i0; i < i1; ++i) sum = limited(sum, min(max(s_tok[i], 0), tok_top), tok_top);
  {
    int v[1] = {sum};
    scan_before<1>(v, tok_top, part);
    sum = v[0];
  }
  int status = 0, need_sum = 0, give_sum = 0;
  for (int i = i0; i < i1; ++i) {
    const int len = static_cast<int>(s_len[i]), n = s_tok[i];
    const int64_t after = static_cast<int64_t>(len) + n;
    sum = limited(sum, min(max(n, 0), tok_top), tok_top);
    int need = -1, give = 0;  // need < 0: not to be served
    if (len < 0 || len > p.max_len) {
      status |= ZKV_PAGES_BAD_LENGTH;
    } else if (n > 0) {
      if (after > p.max_len)
        status |= ZKV_PAGES_TABLE_FULL;
      else if (row ? n > row : sum > p.cap)
        status |= ZKV_PAGES_SLOTS_FULL;
      else
        need = pages_of(static_cast<uint32_t>(after), p.page) - pages_of(len, p.page);
    } else if (n < 0) {
      give = pages_of(len, p.page) - pages_of(static_cast<uint32_t>(max(after, int64_t{0})), p.page);
    }
    s_len[i] = static_cast<uint32_t>(max(len, 0));
    s_tok[i] = row ? n : sum;
    s_need[i] = need;
    s_give[i] = give;
    need_sum = limited(need_sum, max(need, 0), page_top);
    give_sum = limited(give_sum, give, page_top);
  }
  {
    int v[2] = {need_sum, give_sum};
    scan_before<2>(v, page_top, part + 1);
    need_sum = v[0], give_sum = v[1];
  }
  int taken = 0;
  for (int i = i0; i < i1; ++i) {
    const int need = s_need[i];
    need_sum = limited(need_sum, max(need, 0), page_top);
    give_sum = limited(give_sum, s_give[i], page_top);
    if (need >= 0) {
      if (need == 0 || need_sum <= count) {
        s_len[i] |= kGranted;
        if (need > 0) taken = need_sum;
      } else {
        status |= ZKV_PAGES_POOL_EMPTY;
      }
    }
    s_need[i] = need_sum;
    s_give[i] = give_sum;
  }
  if (status) atomicOr(&s_status, status);
  if (taken) atomicMax(&s_taken, taken);
  __syncthreads();
  // this workgroup has read the lengths and the state
  if (tid == 0)
    s_last = gridDim.x == 1 || arrive_last_count(reinterpret_cast<unsigned*>(p.state + 3), static_cast<int>(gridDim.x));
  const int total = s_tok[R - 1], freed = s_give[R - 1];
  const int page_size = static_cast<int>(p.page.d), stride = static_cast<int>(gridDim.x) * kThreads;
  const auto ring_at = [&](uint32_t rank) {  // (head + rank < 2 num_pages)
    const uint32_t w = static_cast<uint32_t>(head) + rank;
    return w >= static_cast<uint32_t>(p.num_pages) ? w - p.num_pages : w;
  };
  // slots and positions; the token that opens a new page writes its table entry
  for (int t = blockIdx.x * kThreads + tid; t < p.cap; t += stride) {
    int64_t slot = -1;
    int pos = -1;
    const int r = row ? static_cast<int>(div_by(t, p.row)) : owner_of(s_tok, R, t);
    // the token's number among its request's
    const int j = row ? t - (r + 1) * row + s_tok[r] : t - (r ? s_tok[r - 1] : 0);
    if (row ? j >= 0 : t < total) {
      const uint32_t lg = s_len[r];
      if (lg & kGranted) {
        const int len = static_cast<int>(lg & ~kGranted);
        pos = len + j;
        const int at = static_cast<int>(div_by(pos, p.page)), off = pos - at * page_size;
        const int held = pages_of(len, p.page);
        int32_t* entry = p.table + r * p.table_stride + at;
        int page;
        if (at >= held) {
          page = p.ring[ring_at((r ? s_need[r - 1] : 0) + at - held)];
          if (off == 0) *entry = page;
        } else {
          page = *entry;
        }
        slot = static_cast<int64_t>(page) * page_size + off;
      }
    }
    p.slots[t] = slot;
    if (p.positions) p.positions[t] = pos;
  }
  // pages given back, in request order and table order, behind the ring's
  // last; never beyond the ring (an inconsistent state would overrun it)
  const int room = min(freed, p.num_pages - count);
  for (int j = blockIdx.x * kThreads + tid; j < room; j += stride) {
    const int r = owner_of(s_give, R, j);
    const int held = pages_of(s_len[r], p.page);
    p.ring[ring_at(count + j)] = p.table[r * p.table_stride + held - (s_give[r] - j)];
  }
  __syncthreads();  // s_last
  if (!s_last) return;
  for (int i = tid; i < R; i += kThreads) {
    const int len = p.lens[i], n = p.new_tokens[i];
    int now = len;
    if (s_len[i] & kGranted)
      now = len + n;
    else if (n < 0 && len >= 0 && len <= p.max_len)
      now = max(len + n, 0);  // (len >= 0 > n: no overflow)
    p.lens_out[i] = now;
    if (p.starts) p.starts[i + 1] = s_tok[i];
  }
  if (tid == 0) {
    if (p.starts) p.starts[0] = 0;
    const int64_t held = static_cast<int64_t>(count) + freed;
    p.state_out[0] = static_cast<int>(ring_at(s_taken));
    p.state_out[1] = static_cast<int>(min(held, static_cast<int64_t>(p.num_pages))) - s_taken;
    p.state_out[2] = old_status | s_status | (held > p.num_pages ? ZKV_PAGES_RING_FULL : 0);
    if (p.state_out != p.state) p.state_out[3] = 0;
  }
}

// ---------------------------------------------------------------------------
// rows into their slots
// ---------------------------------------------------------------------------
// Eight channels of a row: 16 bytes of 16-bit values.
template <int kType>
__device__ __forceinline__ void unpack8(const u32x4_t& x, float (&y)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    y[2 * i] = elem_to_f32<kType>(x[i] & 0xFFFFu);
    y[2 * i + 1] = elem_to_f32<kType>(x[i] >> 16);
  }
}

template <int kType>
__device__ __forceinline__ u32x4_t pack8(const float (&y)[8]) {
  u32x4_t r;
#pragma unroll
  for (int i = 0; i < 4; ++i) r[i] = f32_to_elem<kType>(y[2 * i]) | (f32_to_elem<kType>(y[2 * i + 1]) << 16);
  return r;
}

// y / scale as e4m3: the quotient as an IEEE division rounds it, clamped, and
// rounded once to the code.  The quotient is x r (r the rounded reciprocal),
// corrected by its remainder: q + (x - q s) r, which is the rounded quotient
// for a rounded reciprocal (Markstein); beyond 512 the code is the largest
// whatever the last bits are, and the product alone is kept (its remainder
// could be Inf - Inf).  6 instructions a value, an IEEE division 11: it is the
// write's bound (32768 tokens of 8 heads of 128: 44.5 us with it).  Scales near
// the ends of fp32, whose products would leave it, are divided by.
struct Quotient {
  float s, r;
  bool plain;
  __device__ __forceinline__ explicit Quotient(float scale)
      : s(scale), r(1.0f / scale), plain(!(scale >= 0x1p-100f && scale <= 0x1p100f)) {}
  __device__ __forceinline__ float of(float x) const {
    const float q = x * r;
    const float c = fmaf(fmaf(-q, s, x), r, q);
    return fabsf(q) < 512.0f ? copysignf(c, q) : q;  // (the sum of -0 and 0 is 0)
  }
};

__device__ __forceinline__ u32x2_t quant8(const float (&y)[8], const Quotient& by) {
  float z[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) z[i] = by.of(y[i]);
  if (by.plain) {
#pragma unroll
    for (int i = 0; i < 8; ++i) z[i] = y[i] / by.s;
  }
  return u32x2_t{e4m3x4(z[0], z[1], z[2], z[3]), e4m3x4(z[4], z[5], z[6], z[7])};
}

// Element offset of a slot's row of head h, or -1 when the slot is none.
__device__ __forceinline__ int64_t slot_row(int64_t slot, const PageLayout& l, const FastDiv& page, int h) {
  if (slot < 0 || slot >= static_cast<int64_t>(l.num_pages) * l.page_size) return -1;
  const uint32_t s = static_cast<uint32_t>(slot), at = div_by(s, page);
  return at * l.page_stride + (s - at * page.d) * l.token_stride + h * l.head_stride;
}

struct WriteParams {
  const uint16_t* src[2];  // K, V rows
  int64_t src_token[2], src_head[2];
  const int64_t* slots;
  void* dst[2];
  const float* scale[2];   // one per head, or null for 1
  PageLayout layout;
  FastDiv page, row_chunks;  // row_chunks: chunks (16-byte stores) of a token's kv heads
  int tokens, chunk_shift;   // 1 << chunk_shift chunks of one head's row
};

// A chunk of a row per thread and trip, the 8 or, as e4m3, 16 channels of a
// 16-byte store; kWriteUnroll trips with their loads requested together;
// consecutive threads take consecutive chunks of a token's heads, so a wave
// writes 1 KiB of whole rows (256 bytes at head dim 128).  Bound by HBM: each
// row is read and written once, the stores streamed.  32768 tokens of 8 heads
// of 128: 39 us (6.9 TB/s read and written) in 16 bits (42 with stores that stay
// in the cache, 40 with one trip or four), 34.6 us (5.7 TB/s; 38.7 where the
// inputs change from call to call) as e4m3 (36.0 with plain stores, 36.6 with
// one trip, 36.8 with four, 35.9 with 8 channels and 8-byte stores).
constexpr int kWriteThreads = 256, kWriteUnroll = 2;

template <int kType, bool kFp8>
__global__ __launch_bounds__(kWriteThreads) void paged_write_kernel(const WriteParams p) {
  const int which = blockIdx.y;
  const uint32_t n = static_cast<uint32_t>(p.tokens) * p.row_chunks.d;  // (< 2^31)
  const uint32_t first = blockIdx.x * (kWriteThreads * kWriteUnroll) + threadIdx.x;
  constexpr int kLoads = kFp8 ? 2 : 1;  // 16-byte loads of a chunk
  u32x4_t x[kWriteUnroll][kLoads];
  int64_t row[kWriteUnroll];
  float scale[kWriteUnroll];
  uint32_t ch[kWriteUnroll];
#pragma unroll
  for (int u = 0; u < kWriteUnroll; ++u) {
    const uint32_t i = min(first + u * kWriteThreads, n - 1);
    const uint32_t t = div_by(i, p.row_chunks), c = i - t * p.row_chunks.d;
    const uint32_t h = c >> p.chunk_shift;
    ch[u] = 8 * kLoads * (c & ((1u << p.chunk_shift) - 1));
    const uint16_t* src = p.src[which] + t * p.src_token[which] + h * p.src_head[which] + ch[u];
#pragma unroll
    for (int k = 0; k < kLoads; ++k) x[u][k] = reinterpret_cast<const u32x4_t*>(src)[k];
    row[u] = first + u * kWriteThreads < n ? slot_row(p.slots[t], p.layout, p.page, h) : -1;
    if constexpr (kFp8) scale[u] = p.scale[which] ? p.scale[which][h] : 1.0f;
  }
#pragma unroll
  for (int u = 0; u < kWriteUnroll; ++u) {
    if (row[u] < 0) continue;
    if constexpr (kFp8) {
      const Quotient by(scale[u]);
      u32x2_t r[2];
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        float y[8];
        unpack8<kType>(x[u][k], y);
        r[k] = quant8(y, by);
      }
      __builtin_nontemporal_store(u32x4_t{r[0][0], r[0][1], r[1][0], r[1][1]},
                                  reinterpret_cast<u32x4_t*>(static_cast<uint8_t*>(p.dst[which]) + row[u] + ch[u]));
    } else {
      __builtin_nontemporal_store(x[u][0], reinterpret_cast<u32x4_t*>(static_cast<uint16_t*>(p.dst[which]) + row[u] + ch[u]));
    }
  }
}

struct RopeParams {
  const uint16_t* qkv;
  int64_t qkv_stride;
  const uint16_t* q_norm;
  const uint16_t* k_norm;
  float eps;
  const float* cos;   // [max_positions, d / 2]
  const float* sin;
  const int32_t* positions;
  const int64_t* slots;
  uint16_t* q_out;    // [rows, hq, d]
  void* dst[2];
  const float* scale[2];
  PageLayout layout;
  FastDiv page, heads;  // heads: hq + 2 kv
  int rows, hq, kv, max_positions;
};

// A head is d / 8 lanes of 8 channels (16-byte loads and stores): the sum of
// squares is a butterfly over those lanes, and the rotation's partner channel
// i +- d / 2 is the same place of the lane d / 16 further.  Everything between
// the 16-bit input and the one rounding of the result is fp32.  Bound by
// latency at decode sizes, three trips to memory one after the other: x and the
// position, cos and sin, and for K and V rows the slot (in e4m3 the head's scale
// behind it) before the store.  32 / 8 heads of 128, kernel: 8 rows 3.1 us, 512 4.8; 4096
// rows 19.6 (a call; e4m3 pages 19.4).
template <int kType, bool kFp8, int kD>
__global__ __launch_bounds__(256) void paged_rope_kernel(const RopeParams p) {
  constexpr int kLanes = kD / 8;
  const uint32_t gid = (blockIdx.x * 256 + threadIdx.x) / kLanes;
  const int l = threadIdx.x & (kLanes - 1);
  const uint32_t item = min(gid, static_cast<uint32_t>(p.rows) * p.heads.d - 1);
  const uint32_t row = div_by(item, p.heads);
  const int h = static_cast<int>(item - row * p.heads.d);
  const int pos = p.positions[row];
  const bool live = gid == item && pos >= 0 && pos < p.max_positions;
  const u32x4_t x = *reinterpret_cast<const u32x4_t*>(p.qkv + row * p.qkv_stride + h * kD + 8 * l);
  const bool is_v = h >= p.hq + p.kv;
  const bool is_q = h < p.hq;
  float y[8];
  unpack8<kType>(x, y);
  // (the heads of one wave need not be of one kind: v heads take the same
  // steps, so that the butterflies have every lane, and keep their values)
  const uint16_t* nw = is_q ? p.q_norm : p.k_norm;
  float w[8];
  unpack8<kType>(*reinterpret_cast<const u32x4_t*>(nw + 8 * l), w);
  const int at = (8 * l) & (kD / 2 - 1);
  const int64_t cs = static_cast<int64_t>(live ? pos : 0) * (kD / 2) + at;
  const float4_t c0 = *reinterpret_cast<const float4_t*>(p.cos + cs);
  const float4_t c1 = *reinterpret_cast<const float4_t*>(p.cos + cs + 4);
  const float4_t s0 = *reinterpret_cast<const float4_t*>(p.sin + cs);
  const float4_t s1 = *reinterpret_cast<const float4_t*>(p.sin + cs + 4);
  float ss = 0.0f;
#pragma unroll
  for (int i = 0; i < 8; ++i) ss = fmaf(y[i], y[i], ss);
#pragma unroll
  for (int o = 1; o < kLanes; o <<= 1) ss += __shfl_xor(ss, o);
  const float r = rsqrtf(ss * (1.0f / kD) + p.eps);
  float z[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float n = y[i] * r * w[i];
    const float o = __shfl_xor(n, kLanes / 2);
    const float c = i < 4 ? c0[i & 3] : c1[i & 3], s = i < 4 ? s0[i & 3] : s1[i & 3];
    z[i] = 8 * l < kD / 2 ? n * c - o * s : n * c + o * s;
    if (is_v) z[i] = y[i];
  }
  if (!live) return;
  if (is_q) {
    *reinterpret_cast<u32x4_t*>(p.q_out + (static_cast<int64_t>(row) * p.hq + h) * kD + 8 * l) = pack8<kType>(z);
    return;
  }
  const int kh = h - p.hq - (is_v ? p.kv : 0);
  const int64_t dst = slot_row(p.slots[row], p.layout, p.page, kh);
  if (dst < 0) return;
  void* base = is_v ? p.dst[1] : p.dst[0];
  if constexpr (kFp8) {
    const float* sp = is_v ? p.scale[1] : p.scale[0];
    *reinterpret_cast<u32x2_t*>(static_cast<uint8_t*>(base) + dst + 8 * l) = quant8(z, Quotient(sp ? sp[kh] : 1.0f));
  } else {
    *reinterpret_cast<u32x4_t*>(static_cast<uint16_t*>(base) + dst + 8 * l) = is_v ? x : pack8<kType>(z);
  }
}

}  // namespace
}  // namespace zkv

using namespace zkv;

extern "C" int zkv_page_advance(const int32_t* seq_lens, const int32_t* new_tokens, int requests, int32_t* block_table,
                                int64_t table_stride, int width, int32_t* free_pages, int num_pages, int page_size,
                                int32_t* state, int64_t* slots, int32_t* positions, int capacity, int row,
                                int32_t* starts, int32_t* seq_lens_out, int32_t* state_out, zkv_stream_t stream) {
  ZKV_REQUIRE(seq_lens && new_tokens && block_table && free_pages && state && seq_lens_out && state_out,
              "zkv_page_advance: null pointer");
  ZKV_REQUIRE(requests >= 1 && requests <= kMaxRequests, "zkv_page_advance: %d requests outside [1, %d]", requests,
              kMaxRequests);
  ZKV_REQUIRE(width >= 1 && table_stride >= width && page_size >= 1 && num_pages >= 1,
              "zkv_page_advance: width %d, row stride %lld, page size %d, %d pages", width,
              static_cast<long long>(table_stride), page_size, num_pages);
  ZKV_REQUIRE(static_cast<int64_t>(width) * page_size < (1ll << 31) &&
                  static_cast<int64_t>(num_pages) * page_size < (1ll << 31) && num_pages <= (1 << 30),
              "zkv_page_advance: a request and the pool hold fewer than 2^31 tokens");
  ZKV_REQUIRE(capacity >= 0 && capacity <= (1 << 30) && (capacity == 0 || slots),
              "zkv_page_advance: a slot map of %d", capacity);
  ZKV_REQUIRE(row >= 0 && (row == 0 || (static_cast<int64_t>(row) * requests == capacity && starts == nullptr)),
              "zkv_page_advance: %d requests in rows of %d make a slot map of that many, without starts (%d)", requests,
              row, capacity);
  const AdvanceParams p{seq_lens,  seq_lens_out, new_tokens, block_table, table_stride, free_pages, state,
                        state_out, slots,        positions,  starts,      requests,     num_pages,  capacity,
                        fast_div(static_cast<uint32_t>(page_size)),
                        row ? fast_div(static_cast<uint32_t>(row)) : FastDiv{0, 0, 0},
                        static_cast<int64_t>(width) * page_size};
  const bool few = requests <= kFewRequests && capacity <= kFewSlots;
  const size_t lds = static_cast<size_t>(requests) * 16;
  // dynamic LDS above 64 KiB has to be allowed (per device: the call is cheap)
  if (lds > 60 * 1024 &&
      hipFuncSetAttribute(reinterpret_cast<const void*>(&page_advance_kernel<1024>),
                          hipFuncAttributeMaxDynamicSharedMemorySize, kMaxRequests * 16) != hipSuccess)
    return fail(ZKV_ELAUNCH, "zkv_page_advance: cannot raise the LDS limit to 128 KiB");
  // a token a thread, or a page to give back for every request; every
  // workgroup scans the whole batch, so no more than one per CU
  const int threads = few ? 256 : 1024;
  const int64_t want = (std::max<int64_t>(capacity, requests) + threads - 1) / threads;
  const int grid = static_cast<int>(std::min<int64_t>(256, want));
  auto s = reinterpret_cast<hipStream_t>(stream);
  if (few)
    page_advance_kernel<256><<<grid, 256, lds, s>>>(p);
  else
    page_advance_kernel<1024><<<grid, 1024, lds, s>>>(p);
  return check_launch("page_advance_kernel");
}

extern "C" int zkv_paged_write(const void* k, int64_t k_token, int64_t k_head, const void* v, int64_t v_token,
                               int64_t v_head, const int64_t* slots, int tokens, int kv, int d, int is_f16,
                               void* k_pages, void* v_pages, int is_fp8, const float* k_scale, const float* v_scale,
                               int num_pages, int page_size, int64_t page_stride, int64_t head_stride,
                               int64_t token_stride, zkv_stream_t stream) {
  ZKV_REQUIRE(k && v && slots && k_pages && v_pages, "zkv_paged_write: null pointer");
  const PageLayout layout{page_stride, head_stride, token_stride, num_pages, page_size};
  const char* why = check_pages(layout, kv, d, is_fp8 ? 1 : 2);
  ZKV_REQUIRE(why == nullptr, "zkv_paged_write: %s", why);
  ZKV_REQUIRE(tokens >= 0 && k_token % 8 == 0 && k_head % 8 == 0 && v_token % 8 == 0 && v_head % 8 == 0,
              "zkv_paged_write: %d tokens; rows start on 16 bytes", tokens);
  ZKV_REQUIRE(((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v) | reinterpret_cast<uintptr_t>(k_pages) |
                reinterpret_cast<uintptr_t>(v_pages)) & 15) == 0,
              "zkv_paged_write: rows start on 16 bytes");
  ZKV_REQUIRE(static_cast<int64_t>(tokens) * kv * (d / 8) < (1ll << 31) - kWriteThreads * kWriteUnroll,
              "zkv_paged_write: %d tokens of %d heads in one call", tokens, kv);
  if (tokens == 0) return ZKV_OK;
  const int chunk = is_fp8 ? 16 : 8;  // channels that a thread takes
  const uint32_t chunks = static_cast<uint32_t>(kv) * (d / chunk);
  const WriteParams p{{static_cast<const uint16_t*>(k), static_cast<const uint16_t*>(v)},
                      {k_token, v_token},
                      {k_head, v_head},
                      slots,
                      {k_pages, v_pages},
                      {k_scale, v_scale},
                      layout,
                      fast_div(static_cast<uint32_t>(page_size)),
                      fast_div(chunks),
                      tokens,
                      (d == 64 ? 3 : (d == 128 ? 4 : 5)) - (is_fp8 ? 1 : 0)};
  const uint32_t n = static_cast<uint32_t>(tokens) * chunks;
  const dim3 grid((n + kWriteThreads * kWriteUnroll - 1) / (kWriteThreads * kWriteUnroll), 2);
  auto s = reinterpret_cast<hipStream_t>(stream);
  if (is_fp8) {
    if (is_f16)
      paged_write_kernel<kF16, true><<<grid, kWriteThreads, 0, s>>>(p);
    else
      paged_write_kernel<kBf16, true><<<grid, kWriteThreads, 0, s>>>(p);
  } else {
    // the bits are copied: one kernel for both 16-bit types
    paged_write_kernel<kBf16, false><<<grid, kWriteThreads, 0, s>>>(p);
  }
  return check_launch("paged_write_kernel");
}

extern "C" int zkv_paged_qk_norm_rope(const void* qkv, int64_t qkv_stride, int rows, int hq, int kv, int d, int is_f16,
                                      const void* q_norm, const void* k_norm, float eps, const float* cos,
                                      const float* sin, int max_positions, const int32_t* positions,
                                      const int64_t* slots, void* q_out, void* k_pages, void* v_pages, int is_fp8,
                                      const float* k_scale, const float* v_scale, int num_pages, int page_size,
                                      int64_t page_stride, int64_t head_stride, int64_t token_stride,
                                      zkv_stream_t stream) {
  ZKV_REQUIRE(qkv && q_norm && k_norm && cos && sin && positions && slots && q_out && k_pages && v_pages,
              "zkv_paged_qk_norm_rope: null pointer");
  const PageLayout layout{page_stride, head_stride, token_stride, num_pages, page_size};
  const char* why = check_pages(layout, kv, d, is_fp8 ? 1 : 2);
  ZKV_REQUIRE(why == nullptr, "zkv_paged_qk_norm_rope: %s", why);
  ZKV_REQUIRE(rows >= 0 && hq >= 1 && max_positions >= 1 && qkv_stride % 8 == 0,
              "zkv_paged_qk_norm_rope: rows=%d hq=%d max_positions=%d row stride %lld", rows, hq, max_positions,
              static_cast<long long>(qkv_stride));
  ZKV_REQUIRE(((reinterpret_cast<uintptr_t>(qkv) | reinterpret_cast<uintptr_t>(q_norm) |
                reinterpret_cast<uintptr_t>(k_norm) | reinterpret_cast<uintptr_t>(cos) |
                reinterpret_cast<uintptr_t>(sin) | reinterpret_cast<uintptr_t>(q_out) |
                reinterpret_cast<uintptr_t>(k_pages) | reinterpret_cast<uintptr_t>(v_pages)) & 15) == 0,
              "zkv_paged_qk_norm_rope: rows start on 16 bytes");
  const int64_t threads = static_cast<int64_t>(rows) * (hq + 2 * static_cast<int64_t>(kv)) * (d / 8);
  ZKV_REQUIRE(threads < (1ll << 31) - 256, "zkv_paged_qk_norm_rope: %d rows in one call", rows);
  if (rows == 0) return ZKV_OK;
  const RopeParams p{static_cast<const uint16_t*>(qkv),
                     qkv_stride,
                     static_cast<const uint16_t*>(q_norm),
                     static_cast<const uint16_t*>(k_norm),
                     eps,
                     cos,
                     sin,
                     positions,
                     slots,
                     static_cast<uint16_t*>(q_out),
                     {k_pages, v_pages},
                     {k_scale, v_scale},
                     layout,
                     fast_div(static_cast<uint32_t>(page_size)),
                     fast_div(static_cast<uint32_t>(hq + 2 * kv)),
                     rows,
                     hq,
                     kv,
                     max_positions};
  const int grid = static_cast<int>((threads + 255) / 256);
  auto s = reinterpret_cast<hipStream_t>(stream);
#define ZKV_ROPE(T, F, D) paged_rope_kernel<T, F, D><<<grid, 256, 0, s>>>(p)
#define ZKV_ROPE_D(T, F)   \
  do {                     \
    if (d == 64)           \
      ZKV_ROPE(T, F, 64);  \
    else if (d == 128)     \
      ZKV_ROPE(T, F, 128); \
    else                   \
      ZKV_ROPE(T, F, 256); \
  } while (0)
  if (is_f16) {
    if (is_fp8)
      ZKV_ROPE_D(kF16, true);
    else
      ZKV_ROPE_D(kF16, false);
  } else {
    if (is_fp8)
      ZKV_ROPE_D(kBf16, true);
    else
      ZKV_ROPE_D(kBf16, false);
  }
#undef ZKV_ROPE_D
#undef ZKV_ROPE
  return check_launch("paged_rope_kernel");
}
