// Rotary positions, the new tokens of ragged sequences filed into cache pages, and the pages' own maintenance.
#include <algorithm>
#include <climits>

#include "ttb_paged.cuh"

using namespace ttb;
using namespace ttb::paged;

namespace {

// ---- rotary positions -------------------------------------------------------------------------------------------------
// A pair (a, b) of a head becomes scale * (a cos r - b sin r, b cos r + a sin r) with r = position * frequency: pairs (i, i + n/2) of the first n elements, or
// neighbours. Bound by reading and writing the rows once. A block takes a few tokens: their sines and cosines are made once for all heads and kept in shared
// memory. The angle is a product of doubles in turns, of which the whole ones are dropped before it is rounded to fp32: a position of a
// million times a frequency in fp32 would be off by a tenth of a radian. With a pool of pages, k is turned on its way into its page and v copied beside it: a pass
// of its own over both, and a launch, saved. The rows are on their way while the block looks up its positions and pages.
// 8000 tokens of 40 heads of 128, fp32, all of each turned: 59 us, 5.5 TB/s; 64 and 200 tokens of 40 heads of 128, 16 bits: 5 and 7 us, a chain of dependent reads.
// Units of a thread, threads of an SM and units of a block were measured together, at sizes that the kernel by heads below has taken over since: two, 1536 and 1024 (15000 tokens of 32 heads
// of 64, fp16, and 7900 of 48 of 128, with the launch: 31 and 47 us; four units and 1024 threads 31 and 51; one unit and 512 to a block 31 to 43 and 49 to 63).
constexpr int kRotaryThreads = 256;
constexpr int kRotaryTokens = 8;  // of a block, at most
constexpr int kRotaryUnits = 2;   // that a thread has on their way

struct RotaryParams {
  const void *q, *k, *v;
  void *q_out, *k_out;
  long long ldq, ldk, ldv, ldq_out, ldk_out;
  int tokens, heads, kv_heads, d, half, interleaved, block_tokens;
  int rows;                 // heads of a token, all together
  unsigned per;             // units of a head
  unsigned per_magic, rows_magic;  // their reciprocals, times 2^32 and rounded up; rows_magic is 0 for blocks of one token
  float scale;
  const int64_t* positions;
  const double* freqs;
  Sequences s;              // PAGED
  const int32_t* room;      // may be null
  void *keys, *values;
  long long page_stride;
};

// Which sequence row t belongs to, by the whole warp: the entries of cu that are at most t, counted in two looks of a lane each.
__device__ __forceinline__ int sequence_at(const Sequences& s, int t, int lane) {
  const int step = (s.B + 32) / 32;  // at most 33 for kMaxSequences
  const int at = lane * step;
  const int before = __popc(__ballot_sync(0xffffffffu, at <= s.B && s.cu[min(at, s.B)] <= t));
  if (before == 0) return -1;
  const int lo = (before - 1) * step, i = lo + 1 + lane;
  return lo + __popc(__ballot_sync(0xffffffffu, i < lo + step && i <= s.B && s.cu[min(i, s.B)] <= t));
}

// What a thread turns at a time: WIDE, eight pairs (halves) or four (neighbours), or eight elements that are not turned; else a pair or an element.
template <typename T, bool WIDE> struct Piece;
template <typename T> struct Piece<T, true> {
  static constexpr int kWords = sizeof(T) / 2;  // of 16 bytes
  uint4 w[kWords];
  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (int i = 0; i < kWords; ++i) w[i] = reinterpret_cast<const uint4*>(p)[i];
  }
  __device__ __forceinline__ void store(T* p) const {
#pragma unroll
    for (int i = 0; i < kWords; ++i) reinterpret_cast<uint4*>(p)[i] = w[i];
  }
};
template <typename T> struct Piece<T, false> {
  T w;
  __device__ __forceinline__ void load(const T* p) { w = *p; }
  __device__ __forceinline__ void store(T* p) const { *p = w; }
};

// Where unit `idx` of a block lies: its token, its head among the token's query, key and (PAGED) value heads, its elements `first` and (a pair of halves)
// `second`, else -1, and its first pair, -1 where nothing is turned. Every head has the same units, those of the values too.
struct UnitPlace {
  int token, head, first, second, pair;
};
template <bool WIDE>
__device__ __forceinline__ UnitPlace unit_place(const RotaryParams& p, unsigned idx) {
  UnitPlace w;
  // WIDE: at most 64 units of 196605 heads, so that the rounded-up reciprocals are exact (their error times idx stays below 2^32); blocks of more than one
  // token are small. Plain divisions of both took half of the kernel's instructions.
  const unsigned row = !WIDE ? idx / p.per : p.per == 1 ? idx : __umulhi(idx, p.per_magic);
  w.token = p.rows == 1 ? (int)row : (int)__umulhi(row, p.rows_magic);
  w.head = (int)(row - w.token * (unsigned)p.rows);
  const int u = (int)(idx - row * p.per), wide = WIDE ? 8 : 1;
  w.second = -1;
  if (WIDE && p.interleaved) {
    w.first = u * 8;
    w.pair = u * 4 < p.half ? u * 4 : -1;
  } else if (u * wide < p.half) {
    w.first = p.interleaved ? 2 * u : u * wide;
    w.second = p.interleaved ? 2 * u + 1 : p.half + u * wide;
    w.pair = u * wide;
  } else {
    w.first = p.half + u * wide;
    w.pair = -1;
  }
  return w;
}

template <typename T>
__device__ __forceinline__ void turn(Piece<T, true>& x, Piece<T, true>& y, bool halves, const float2* cs) {
  Vec8<T> a, b;
  a.load(reinterpret_cast<const T*>(x.w));
  if (halves) {
    b.load(reinterpret_cast<const T*>(y.w));
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
      const float4 c = *reinterpret_cast<const float4*>(cs + e);
      const float f = a.v[e], g = b.v[e], h = a.v[e + 1], i = b.v[e + 1];
      a.v[e] = f * c.x - g * c.y;
      b.v[e] = g * c.x + f * c.y;
      a.v[e + 1] = h * c.z - i * c.w;
      b.v[e + 1] = i * c.z + h * c.w;
    }
    b.store(reinterpret_cast<T*>(y.w));
  } else {
#pragma unroll
    for (int e = 0; e < 4; e += 2) {
      const float4 c = *reinterpret_cast<const float4*>(cs + e);
      const float f = a.v[2 * e], g = a.v[2 * e + 1], h = a.v[2 * e + 2], i = a.v[2 * e + 3];
      a.v[2 * e] = f * c.x - g * c.y;
      a.v[2 * e + 1] = g * c.x + f * c.y;
      a.v[2 * e + 2] = h * c.z - i * c.w;
      a.v[2 * e + 3] = i * c.z + h * c.w;
    }
  }
  a.store(reinterpret_cast<T*>(x.w));
}
template <typename T>
__device__ __forceinline__ void turn(Piece<T, false>& x, Piece<T, false>& y, bool, const float2* cs) {
  const float f = to_f(x.w), g = to_f(y.w);
  x.w = from_f<T>(f * cs->x - g * cs->y);
  y.w = from_f<T>(g * cs->x + f * cs->y);
}

// The block's positions, and (PAGED) the places of its tokens; then cosines and sines of all their pairs, times the scale. All threads.
template <bool PAGED>
__device__ __forceinline__ void block_angles(const RotaryParams& p, int t0, int n, double* s_pos, long long* s_page, float2* cs) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  for (int i = PAGED ? warp : tid; i < n; i += PAGED ? kRotaryThreads / 32 : kRotaryThreads) {
    const int t = t0 + i;
    if (!PAGED) {
      s_pos[i] = (double)p.positions[t];
      continue;
    }
    const int b = sequence_at(p.s, t, lane);
    bool bad = false, mine = false;
    long long place = -1;
    int at = 0;
    if (b >= 0 && b < p.s.B && !(p.room && p.room[b] == 0)) {
      const Sequence q = sequence_of(p.s, b, &bad);
      mine = t >= q.tok0 && t < q.tok0 + q.n;
      at = q.past + t - q.tok0;
      if (mine && at < p.s.cap) {
        bool bad_page;
        const int page = page_of(p.s, b, at, &bad_page);
        bad |= bad_page;
        if (!bad_page) place = (long long)page * p.page_stride + (long long)(at & ((1 << p.s.page_shift) - 1)) * p.d;
      }
    }
    if (lane == 0) {
      if (bad) bad_index(p.s.status);
      s_pos[i] = mine ? (double)at : -1.0;
      s_page[i] = place;
    }
  }
  __syncthreads();
  for (int i = tid; i < n * p.half; i += kRotaryThreads) {
    const double turns = s_pos[i / p.half] * p.freqs[i % p.half] * 0.15915494309189533577;  // 1 / (2 pi)
    float s, c;
    sincospif(2.0f * (float)(turns - rint(turns)), &s, &c);
    cs[i] = make_float2(c * p.scale, s * p.scale);
  }
  __syncthreads();
}

template <typename T, bool WIDE, bool PAGED>
__global__ void __launch_bounds__(kRotaryThreads, sizeof(T) == 2 ? 6 : 4)
rotary_kernel(const RotaryParams p) {
  extern __shared__ __align__(16) float2 cs[];  // [block_tokens][half]
  __shared__ double s_pos[kRotaryTokens];
  __shared__ long long s_page[kRotaryTokens];  // PAGED: the token's first element of the pools, -1: it has no place
  pdl_trigger();
  pdl_wait();
  const int tid = threadIdx.x;
  const int t0 = blockIdx.x * p.block_tokens, n = min(p.block_tokens, p.tokens - t0);
  const int units = n * p.rows * (int)p.per;
  Piece<T, WIDE> x[kRotaryUnits], y[kRotaryUnits];
  auto load = [&](int idx0) {
#pragma unroll
    for (int b = 0; b < kRotaryUnits; ++b) {
      const int idx = idx0 + b * kRotaryThreads;
      if (idx >= units) break;
      const UnitPlace w = unit_place<WIDE>(p, idx);
      const long long t = t0 + w.token;
      const T* src;
      if (w.head < p.heads) src = static_cast<const T*>(p.q) + t * p.ldq + w.head * p.d;
      else if (!PAGED || w.head < p.heads + p.kv_heads) src = static_cast<const T*>(p.k) + t * p.ldk + (w.head - p.heads) * p.d;
      else src = static_cast<const T*>(p.v) + t * p.ldv + (w.head - p.heads - p.kv_heads) * p.d;
      x[b].load(src + w.first);
      if (w.second >= 0) y[b].load(src + w.second);
    }
  };
  load(tid);  // on their way while the block works out its positions
  block_angles<PAGED>(p, t0, n, s_pos, s_page, cs);
  for (int idx0 = tid; idx0 < units;) {
#pragma unroll
    for (int b = 0; b < kRotaryUnits; ++b) {
      const int idx = idx0 + b * kRotaryThreads;
      if (idx >= units) break;
      const UnitPlace w = unit_place<WIDE>(p, idx);
      const bool query = w.head < p.heads, key = w.head < p.heads + p.kv_heads;
      if (PAGED && (query ? s_pos[w.token] < 0 : s_page[w.token] < 0)) continue;
      if (w.pair >= 0 && (!PAGED || key)) turn(x[b], y[b], w.second >= 0, cs + w.token * p.half + w.pair);
      const long long t = t0 + w.token;
      T* dst;
      if (query) dst = static_cast<T*>(p.q_out) + t * p.ldq_out + w.head * p.d;
      else if (!PAGED) dst = static_cast<T*>(p.k_out) + t * p.ldk_out + (w.head - p.heads) * p.d;
      else dst = static_cast<T*>(key ? p.keys : p.values) + s_page[w.token] + (((long long)w.head - p.heads - (key ? 0 : p.kv_heads)) << p.s.page_shift) * p.d;
      x[b].store(dst + w.first);
      if (w.second >= 0) y[b].store(dst + w.second);
    }
    idx0 += kRotaryUnits * kRotaryThreads;
    load(idx0);
  }
}

// The same for prompts of many heads whose units are a power of two (at most a warp): a warp takes a token, and a lane the same unit of every head, so that its cosines
// and sines stay in registers and a head costs its loads, products and stores, where the places of units in the kernel above take a third of its instructions.
// 15000 tokens of 32 heads of 64, half of each turned, fp16: 21.5 us, 5.7 TB/s (26.7 there); 7900 tokens, 32 heads of 128 turned and 8 filed with their values: 34.5 us, 5.6 TB/s (42.3).
// With fewer units of a token, or fewer tokens, a warp has too little on its way: 15000 tokens of 24 heads of 64 (96 units) 27 us and 25 there, 1300 tokens of 40 heads
// of 128 (320 units) 14 and 12, 5000 of them 29 and 27, 8000 33 and 37 (with the launch). fp32 is bound by memory there already (8000 tokens: 68 and 63).
template <typename T, bool HALVES, bool PAGED>
__global__ void __launch_bounds__(kRotaryThreads, 4)
rotary_heads_kernel(const RotaryParams p) {
  static_assert(kRotaryThreads / 32 == kRotaryTokens, "a warp a token");
  constexpr int U = HALVES ? 2 : 4;                     // heads of a lane on their way
  extern __shared__ __align__(16) float2 cs[];          // [kRotaryTokens][half]
  __shared__ double s_pos[kRotaryTokens];
  __shared__ long long s_page[kRotaryTokens];
  pdl_trigger();
  pdl_wait();
  const int lane = threadIdx.x & 31, i = threadIdx.x >> 5, shift = 31 - __clz(p.per), step = 32 >> shift;
  const int t0 = blockIdx.x * kRotaryTokens, n = min(kRotaryTokens, p.tokens - t0);
  const long long t = t0 + i;
  const int u = lane & (int)(p.per - 1), mine = lane >> shift;
  const bool turned = u * (HALVES ? 8 : 4) < p.half, two = HALVES && turned;
  const int first = HALVES && !turned ? p.half + u * 8 : u * 8;
  // kinds of heads: queries, keys, (PAGED) values
  const T* src = nullptr;
  T* dst = nullptr;
  long long out = 0;  // elements between heads
  int kind = -1, heads = 0, h = 0;
  Piece<T, true> x[U], y[U];
  auto more = [&]() {  // heads h and following of a kind; false: none is left
    while (h >= heads) {
      if (++kind == (PAGED ? 3 : 2)) return false;
      heads = kind ? p.kv_heads : p.heads;
      h = 0;
      src = (kind == 0 ? static_cast<const T*>(p.q) + t * p.ldq : kind == 1 ? static_cast<const T*>(p.k) + t * p.ldk : static_cast<const T*>(p.v) + t * p.ldv) + first;
    }
    return true;
  };
  auto load = [&]() {
#pragma unroll
    for (int e = 0; e < U; ++e) {
      const int head = h + e * step + mine;
      if (head >= heads) break;
      x[e].load(src + head * p.d);
      if (two) y[e].load(src + head * p.d + p.half);
    }
  };
  const bool any = i < n && more();
  if (any) load();  // on their way while the block works out its positions
  block_angles<PAGED>(p, t0, n, s_pos, s_page, cs);
  if (!any) return;
  constexpr int P = HALVES ? 8 : 4;
  float4 c[P / 2];
  if (turned) {
#pragma unroll
    for (int e = 0; e < P / 2; ++e) c[e] = *reinterpret_cast<const float4*>(cs + i * p.half + u * P + 2 * e);
  }
  const bool placed = !PAGED || s_page[i] >= 0, known = !PAGED || s_pos[i] >= 0;
  do {
    if (kind == 0) dst = static_cast<T*>(p.q_out) + t * p.ldq_out + first, out = p.d;
    else if (!PAGED) dst = static_cast<T*>(p.k_out) + t * p.ldk_out + first, out = p.d;
    else dst = static_cast<T*>(kind == 1 ? p.keys : p.values) + s_page[i] + first, out = (long long)p.d << p.s.page_shift;
    if (kind ? placed : known) {
#pragma unroll
      for (int e = 0; e < U; ++e) {
        const int head = h + e * step + mine;
        if (head >= heads) break;
        if (turned && (!PAGED || kind < 2)) turn(x[e], y[e], HALVES, reinterpret_cast<const float2*>(c));
        x[e].store(dst + head * out);
        if (two) y[e].store(dst + head * out + p.half);
      }
    }
    h += U * step;
    if (!more()) break;
    load();
  } while (true);
}

template <typename T, bool PAGED>
int launch_rotary(ttb_ctx* ctx, RotaryParams& p, const char* what) {
  const uintptr_t at = reinterpret_cast<uintptr_t>(p.q) | reinterpret_cast<uintptr_t>(p.k) | reinterpret_cast<uintptr_t>(p.v) |
                       reinterpret_cast<uintptr_t>(p.q_out) | reinterpret_cast<uintptr_t>(p.k_out);
  const bool wide = (at & 15) == 0 && ((p.ldq | p.ldk | p.ldv | p.ldq_out | p.ldk_out) * (int)sizeof(T)) % 16 == 0 && p.half % (p.interleaved ? 4 : 8) == 0;
  // tokens of a block: enough for every thread to have some units, few enough for the tokens to reach all SMs
  p.rows = p.heads + (PAGED ? 2 : 1) * p.kv_heads;
  p.per = !wide ? p.d - p.half : p.interleaved ? p.d / 8 : (p.d - p.half) / 8;
  const int units = p.rows * p.d / 16;
  p.block_tokens = std::max(1, std::min(std::min(kRotaryTokens, 2 * kRotaryUnits * kRotaryThreads / std::max(1, units)), p.tokens / (4 * ctx->sm_count)));
  p.per_magic = (unsigned)(((1ull << 32) + p.per - 1) / p.per);
  p.rows_magic = p.block_tokens == 1 ? 0 : (unsigned)(((1ull << 32) + p.rows - 1) / p.rows);
  const bool by_heads = sizeof(T) == 2 && wide && p.per <= 32 && (p.per & (p.per - 1)) == 0 && (int64_t)p.rows * p.per >= 256 && p.tokens >= 48 * ctx->sm_count;
  if (by_heads) p.block_tokens = kRotaryTokens;
  const dim3 grid((unsigned)((p.tokens + p.block_tokens - 1) / p.block_tokens));
  const size_t smem = (size_t)p.block_tokens * p.half * sizeof(float2);
  if constexpr (sizeof(T) == 2) {
    if (by_heads) {
      if (p.interleaved) launch_pdl(rotary_heads_kernel<T, false, PAGED>, grid, dim3(kRotaryThreads), smem, ctx->stream, p);
      else launch_pdl(rotary_heads_kernel<T, true, PAGED>, grid, dim3(kRotaryThreads), smem, ctx->stream, p);
      return launched(ctx, what);
    }
  }
  if (wide) launch_pdl(rotary_kernel<T, true, PAGED>, grid, dim3(kRotaryThreads), smem, ctx->stream, p);
  else launch_pdl(rotary_kernel<T, false, PAGED>, grid, dim3(kRotaryThreads), smem, ctx->stream, p);
  return launched(ctx, what);
}

// ---- page maintenance ---------------------------------------------------------------------------------------------------
// The page table, the lengths and the reference counts stay on the device, and so do the decisions: a step of a captured graph forks beams and takes pages
// without the host. Every choice goes by rows' and pages' order, so that it is the same on every run. All are bound by latency but the copies
// (301 pages of 32 KB in 24 planes: 78 us, 6.1 TB/s).
constexpr int kManageThreads = 1024;
// reference counts a thread looks at in one round (one of them: three rounds for 3000 pages; sixteen one after the other: 1 to 2 us more in a compaction, 0.8 in a reservation)
constexpr int kScanRefs = 4;

// Exclusive prefix sum over the block; *total receives the sum. `scratch` holds 33 ints.
__device__ __forceinline__ int block_scan(int v, int* scratch, int* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  int incl = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int x = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += x;
  }
  __syncthreads();  // the scratch's last readers are through
  if (lane == 31) scratch[warp] = incl;
  __syncthreads();
  if (warp == 0) {
    int w = lane < warps ? scratch[lane] : 0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, w, o);
      if (lane >= o) w += x;
    }
    scratch[lane] = w;
    if (lane == 31) scratch[32] = w;
  }
  __syncthreads();
  *total = scratch[32];
  return incl - v + (warp ? scratch[warp - 1] : 0);
}

struct Tables {
  int32_t* table;
  long long stride;
  int B, width, pages;
  int32_t *lens, *refs;
  int* status;
};

// Pages for new[b] more tokens of every row (see ttb.h for the rules). One block; thread b decides for row b.
// A row writes to the columns from the page that it has begun, or else the next one, to the last that its new tokens reach. What it lists there (it may have kept fewer tokens
// than it once had room for) stays its own; a page in any of them is left for a fresh one only where other rows list it too, unless the row is the last of holders that all
// write. A row's thread looks at its first columns. What is beyond them (a prompt's) warps fill in; only a row that lists a page in each of its first columns can list more there
// (nothing is listed behind a row's first -1), and those go by keeper[page], made before the first count changes: 64 prompts of 4096 tokens 17 us, and 23 with all columns looked at.
// 64 rows over 1300 pages, most of them sharing the page that they go on in: 8 us with cold caches.
// free_list [pages], sharers [pages], keeper [pages]: scratch, not initialised.
constexpr int kOwnColumns = 2;
constexpr int kNobody = -1, kUncounted = -2, kWhoever = INT_MAX;  // keeper: all holders leave it; its count is zero, so that it is free; one row alone lists it
__global__ void __launch_bounds__(kManageThreads, 1)
paged_reserve_kernel(const Tables t, const int32_t* __restrict__ fresh, int page_tokens, int32_t* granted, int32_t* copies, int32_t* room, int* free_list,
                     int* sharers, int* keeper) {
  __shared__ int scratch[33];
  __shared__ int s_first[kMaxSequences], s_want[kMaxSequences], s_at[kMaxSequences];
  __shared__ bool s_more[kMaxSequences];  // whether a row may list pages beyond its first columns
  pdl_trigger();
  pdl_wait();
  const int b = threadIdx.x, lane = threadIdx.x & 31;
  auto listed = [&](int row, int col) {  // -1: nothing that is in the pool
    const int page = t.table[row * t.stride + col];
    return page >= 0 && page < t.pages ? page : -1;
  };
  int len = 0, add = 0, first = 0, want = 0;
  bool fits = false, begun = false, bad = false;  // bad: the row's length or what is asked for is no number of tokens, or its last page is none
  if (b < t.B) {
    len = t.lens[b];
    add = fresh[b];
    const long long cap = (long long)t.width * page_tokens;
    fits = len >= 0 && add >= 0 && (long long)len + add <= cap;
    bad = len < 0 || add < 0 || len > cap;
    if (fits && add > 0) {
      begun = len % page_tokens != 0;
      first = len / page_tokens;
      bad = len > 0 && listed(b, first - (begun ? 0 : 1)) < 0;
      if (!bad) want = (len + add + page_tokens - 1) / page_tokens;
    }
    if (bad) bad_index(t.status);
    s_first[b] = first;
    s_want[b] = want;
    s_at[b] = 0;
  }
  int page[kOwnColumns], refs[kOwnColumns];
#pragma unroll
  for (int i = 0; i < kOwnColumns; ++i) page[i] = first + i < want ? listed(b, first + i) : -1;
#pragma unroll
  for (int i = 0; i < kOwnColumns; ++i) refs[i] = page[i] >= 0 ? t.refs[page[i]] : 0;
  auto begin = [&](int page, int refs) {
    if (page < 0) return;
    sharers[page] = 0;
    keeper[page] = refs > 1 ? kNobody : refs == 1 ? kWhoever : kUncounted;
  };
#pragma unroll
  for (int i = 0; i < kOwnColumns; ++i) begin(page[i], refs[i]);
  __threadfence_block();
  const bool far = want - first > kOwnColumns, more = far && page[kOwnColumns - 1] >= 0;
  if (b < t.B) s_more[b] = more;
  const bool some = __syncthreads_or(more);
  auto beyond = [&](auto&& f) {
    for (int row = threadIdx.x >> 5; row < t.B; row += kManageThreads / 32)
      if (s_more[row])
        for (int col = s_first[row] + kOwnColumns + lane; col < s_want[row]; col += 32) f(row, listed(row, col));
  };
  if (some) {
    beyond([&](int, int page) { begin(page, page >= 0 ? t.refs[page] : 0); });
    __threadfence_block();
    __syncthreads();
  }
  auto share = [&](int row, int page, int refs) {
    if (page < 0 || refs <= 1) return;
    atomicAdd(sharers + page, 1);
    atomicMax(keeper + page, row);
  };
#pragma unroll
  for (int i = 0; i < kOwnColumns; ++i) share(b, page[i], refs[i]);
  if (some) beyond([&](int row, int page) { share(row, page, page >= 0 ? t.refs[page] : 0); });
  __threadfence_block();
  __syncthreads();
  // Which columns take a page. (A page that is begun holds the row's tokens, whatever its count says.)
  bool takes[kOwnColumns];
  int own = 0, need;
#pragma unroll
  for (int i = 0; i < kOwnColumns; ++i) {
    const bool holds = begun && i == 0;
    if (refs[i] > 1) takes[i] = !(__ldcg(sharers + page[i]) == refs[i] && __ldcg(keeper + page[i]) == b);
    else takes[i] = first + i < want && refs[i] != 1 && !holds;
    own += takes[i];
  }
  need = own + (far && !more ? want - first - kOwnColumns : 0);
  auto passed = [&](int row, int page) {  // of a column beyond, when the keepers are settled
    if (page < 0) return true;
    const int k = __ldcg(keeper + page);
    return k != kWhoever && k != row;
  };
  if (some) {
    beyond([&](int, int page) {
      if (page < 0) return;
      const int refs = t.refs[page];
      if (refs > 1 && __ldcg(sharers + page) != refs) keeper[page] = kNobody;
    });
    __threadfence_block();
    __syncthreads();
    beyond([&](int row, int page) {
      if (passed(row, page)) atomicAdd(s_at + row, 1);
    });
    __syncthreads();
    if (b < t.B) need += s_at[b];
  }
  const bool writes = add > 0;
  int total, found = 0;
  const int before = block_scan(need, scratch, &total);
  // the lowest free pages, as many as are needed
  for (int p0 = 0; p0 < t.pages && found < total; p0 += kManageThreads * kScanRefs) {
    uint32_t free = 0;
    const int mine = p0 + (int)threadIdx.x * kScanRefs;
#pragma unroll
    for (int i = 0; i < kScanRefs; ++i)
      if (mine + i < t.pages && t.refs[mine + i] <= 0) free |= 1u << i;
    int round;
    int at = found + block_scan(__popc(free), scratch, &round);
    for (; free && at < total; free &= free - 1) free_list[at++] = mine + __ffs(free) - 1;
    found += round;
  }
  __threadfence_block();
  __syncthreads();
  const bool ok = !bad && (!writes || (fits && (long long)before + need <= found));
  const bool copy = ok && begun && takes[0];
  int n_copies;
  const int c = block_scan(copy ? 1 : 0, scratch, &n_copies);
  if (b < t.B) {
    granted[b] = ok;
    if (room) room[b] = ok;
    if (!ok) s_want[b] = first;  // nothing to fill in
    s_at[b] = before + own;
    if (copy) {
      copies[2 * c] = page[0];
      copies[2 * c + 1] = free_list[before];
    }
    if (b >= n_copies) copies[2 * b] = copies[2 * b + 1] = -1;
    int at = before;
#pragma unroll
    for (int i = 0; i < kOwnColumns; ++i)
      if (ok && takes[i]) {
        const int taken = free_list[at++];
        t.table[b * t.stride + first + i] = taken;
        t.refs[taken] = 1;
        if (refs[i] > 0) atomicSub(t.refs + page[i], 1);
      }
  }
  if (!__syncthreads_or(ok && far)) return;
  for (int row = threadIdx.x >> 5; row < t.B; row += kManageThreads / 32) {
    if (!s_more[row]) {
      for (int col = s_first[row] + kOwnColumns + lane, at = s_at[row] + lane; col < s_want[row]; col += 32, at += 32) {
        const int taken = free_list[at];
        t.table[row * t.stride + col] = taken;
        t.refs[taken] = 1;
      }
      continue;
    }
    for (int c0 = s_first[row] + kOwnColumns, at = s_at[row]; c0 < s_want[row]; c0 += 32) {
      const int col = c0 + lane, had = col < s_want[row] ? listed(row, col) : -1;
      const bool take = col < s_want[row] && passed(row, had);
      const unsigned mask = __ballot_sync(0xffffffffu, take);
      if (take) {
        const int taken = free_list[at + __popc(mask & ((1u << lane) - 1))];
        t.table[row * t.stride + col] = taken;
        t.refs[taken] = 1;
        if (had >= 0 && __ldcg(keeper + had) != kUncounted) atomicSub(t.refs + had, 1);
      }
      at += __popc(mask);
    }
  }
}

// Row b becomes what row parents[b] was. A block takes some columns of all rows: it has read them all before it writes the first, and no other block touches
// them. Reference counts are sums, which no order changes.
constexpr int kForkColumns = 16;
__global__ void __launch_bounds__(256)
paged_fork_kernel(const Tables t, const int32_t* __restrict__ parents) {
  extern __shared__ int32_t old[];  // [B][kForkColumns], then the lengths
  pdl_trigger();
  pdl_wait();
  const int c0 = blockIdx.x * kForkColumns, n = min(kForkColumns, t.width - c0);
  int32_t* s_lens = old + t.B * kForkColumns;
  for (int i = threadIdx.x; i < t.B * kForkColumns; i += blockDim.x)
    if (i % kForkColumns < n) old[i] = t.table[i / kForkColumns * t.stride + c0 + i % kForkColumns];
  if (blockIdx.x == 0)
    for (int b = threadIdx.x; b < t.B; b += blockDim.x) s_lens[b] = t.lens[b];
  __syncthreads();
  auto parent_of = [&](int b) {
    const int p = parents[b];
    if (p < -1 || p >= t.B) {
      bad_index(t.status);
      return b;
    }
    return p;
  };
  for (int i = threadIdx.x; i < t.B * kForkColumns; i += blockDim.x) {
    const int b = i / kForkColumns, c = i % kForkColumns;
    if (c >= n) continue;
    const int parent = parent_of(b);
    const int before = old[i], after = parent < 0 ? -1 : old[parent * kForkColumns + c];
    if (after == before) continue;
    if (after >= t.pages || before >= t.pages) bad_index(t.status);
    if (after >= 0 && after < t.pages) atomicAdd(t.refs + after, 1);
    if (before >= 0 && before < t.pages) atomicSub(t.refs + before, 1);
    t.table[b * t.stride + c0 + c] = after;
  }
  if (blockIdx.x == 0)
    for (int b = threadIdx.x; b < t.B; b += blockDim.x) {
      const int parent = parent_of(b);
      t.lens[b] = parent < 0 ? 0 : s_lens[parent];
    }
}

// Page pairs[i][1] of every plane becomes a copy of page pairs[i][0]. A block copies a page of one plane at a time; pairs with a negative entry are left out.
constexpr int kCopyThreads = 256;
constexpr int kCopyDepth = 8;  // 16-byte loads a thread has in flight
// Of a compaction (`to` not null) the grid's threads also bring the page table in line; `count` is then how many pairs there are.
__global__ void __launch_bounds__(kCopyThreads)
paged_copy_kernel(uint4* pool, int planes, long long plane_stride, int page_chunks, long long page_stride, int pages, const int32_t* pairs, int n_pairs, const int* count,
                  const Tables t, const int32_t* to, int* status) {
  pdl_trigger();
  pdl_wait();
  if (to) {
    for (long long i = (long long)blockIdx.x * kCopyThreads + threadIdx.x; i < (long long)t.B * t.width; i += (long long)gridDim.x * kCopyThreads) {
      int32_t* e = t.table + i / t.width * t.stride + i % t.width;
      const int page = *e;
      if (page >= t.pages) bad_index(t.status);
      else if (page >= 0) *e = to[page];
    }
  }
  const long long n = (long long)(count ? min(*count, n_pairs) : n_pairs) * planes;
  for (long long w = blockIdx.x; w < n; w += gridDim.x) {
    const int pair = (int)(w / planes), plane = (int)(w - (long long)pair * planes);
    const int from = pairs[2 * pair], to = pairs[2 * pair + 1];
    if (from < 0 || to < 0) continue;
    if (from >= pages || to >= pages) {
      bad_index(status);
      continue;
    }
    const uint4* src = pool + plane * plane_stride + from * page_stride;
    uint4* dst = pool + plane * plane_stride + to * page_stride;
    for (int i0 = threadIdx.x; i0 < page_chunks; i0 += kCopyThreads * kCopyDepth) {
      uint4 v[kCopyDepth];
#pragma unroll
      for (int k = 0; k < kCopyDepth; ++k)
        if (i0 + k * kCopyThreads < page_chunks) v[k] = src[i0 + k * kCopyThreads];
#pragma unroll
      for (int k = 0; k < kCopyDepth; ++k)
        if (i0 + k * kCopyThreads < page_chunks) dst[i0 + k * kCopyThreads] = v[k];
    }
  }
}

// Which pages move where: the used ones behind the front (as many as are used), in order, into the free ones within it, in order. One block.
// to [pages]: where each page is afterwards; pairs [pages / 2][2]; n_moves.
__global__ void __launch_bounds__(kManageThreads, 1)
paged_compact_kernel(int32_t* refs, int pages, int32_t* used, int32_t* to, int32_t* pairs, int* n_moves) {
  __shared__ int scratch[33];
  pdl_trigger();
  pdl_wait();
  int live = 0, front;
  for (int p = threadIdx.x; p < pages; p += kManageThreads) live += refs[p] > 0;
  block_scan(live, scratch, &front);
  int outs = 0, holes = 0;
  for (int p0 = 0; p0 < pages; p0 += kManageThreads * kScanRefs) {
    const int mine = p0 + (int)threadIdx.x * kScanRefs;
    uint32_t out = 0, hole = 0;
#pragma unroll
    for (int i = 0; i < kScanRefs; ++i) {
      const int p = mine + i;
      if (p >= pages) continue;
      const bool in_use = refs[p] > 0;
      if (in_use && p >= front) out |= 1u << i;
      if (!in_use && p < front) hole |= 1u << i;
      to[p] = p;
    }
    int total;
    const int at = block_scan(__popc(out) << 16 | __popc(hole), scratch, &total);  // both at once: at most 2^12 of each in a round
    for (int k = outs + (at >> 16); out; out &= out - 1) pairs[2 * k++] = mine + __ffs(out) - 1;
    for (int k = holes + (at & 0xffff); hole; hole &= hole - 1) pairs[2 * k++ + 1] = mine + __ffs(hole) - 1;
    outs += total >> 16;
    holes += total & 0xffff;
  }
  __threadfence_block();
  __syncthreads();
  for (int i = threadIdx.x; i < outs; i += kManageThreads) {
    const int from = pairs[2 * i], hole = pairs[2 * i + 1];
    to[from] = hole;
    refs[hole] = refs[from];
    refs[from] = 0;
  }
  if (threadIdx.x == 0) {
    *used = front;
    *n_moves = outs;
  }
}

int check_tables(ttb_ctx* ctx, const char* what, const ttb_paged_tables* a, Tables* t) {
  TTB_REQUIRE(ctx, a, "%s: null arguments", what);
  TTB_REQUIRE(ctx, a->refs && (a->table || a->B == 0), "%s: null pointer", what);
  TTB_REQUIRE(ctx, a->B >= 0 && a->B <= kMaxSequences, "%s: at most %d rows", what, kMaxSequences);
  TTB_REQUIRE(ctx, a->width > 0 && a->width < (1ll << 30) && a->stride >= a->width, "%s: bad table width", what);
  TTB_REQUIRE(ctx, a->pages > 0 && a->pages < (1ll << 30), "%s: bad number of pages", what);
  *t = Tables{a->table, a->stride, (int)a->B, (int)a->width, (int)a->pages, a->lens, a->refs, ctx->d_status};
  return TTB_OK;
}

int check_pool(ttb_ctx* ctx, const char* what, const ttb_paged_pool* a) {
  TTB_REQUIRE(ctx, a && a->base, "%s: null pool", what);
  TTB_REQUIRE(ctx, a->planes > 0 && a->planes < (1ll << 20) && a->pages > 0 && a->pages < (1ll << 30) && a->page_bytes > 0 && a->page_bytes < (1ll << 31),
              "%s: bad pool shape", what);
  TTB_REQUIRE(ctx, a->page_stride >= a->page_bytes && (a->planes == 1 || a->plane_stride >= (a->pages - 1) * a->page_stride + a->page_bytes),
              "%s: the pool's pages overlap", what);
  TTB_REQUIRE(ctx, ((reinterpret_cast<uintptr_t>(a->base) | (uintptr_t)a->page_bytes | (uintptr_t)a->page_stride | (uintptr_t)a->plane_stride) & 15) == 0,
              "%s: the pool, its pages and its planes must be multiples of 16 bytes", what);
  return TTB_OK;
}

int launch_copy(ttb_ctx* ctx, const ttb_paged_pool* a, const int32_t* pairs, int64_t n, const int* count, const Tables& t, const int32_t* to) {
  const int64_t entries = to ? ((int64_t)t.B * t.width + kCopyThreads - 1) / kCopyThreads : 0;
  const unsigned grid = (unsigned)std::min<int64_t>(std::max(n * a->planes, entries), (int64_t)ctx->sm_count * 8);
  launch_pdl(paged_copy_kernel, dim3(grid), dim3(kCopyThreads), 0, ctx->stream, static_cast<uint4*>(a->base), (int)a->planes, (long long)(a->plane_stride / 16),
             (int)(a->page_bytes / 16), (long long)(a->page_stride / 16), (int)a->pages, pairs, (int)n, count, t, to, ctx->d_status);
  return launched(ctx, "paged_copy");
}

}  // namespace

extern "C" int ttb_rotary(ttb_ctx* ctx, const ttb_rotary_args* a) {
  if (!ctx) return TTB_ERR_INVALID;
  TTB_REQUIRE(ctx, a, "rotary: null arguments");
  TTB_REQUIRE(ctx, a->dtype == TTB_F32 || a->dtype == TTB_F16 || a->dtype == TTB_BF16, "rotary: dtype must be F32, F16 or BF16");
  TTB_REQUIRE(ctx, a->tokens >= 0 && a->tokens < (1ll << 29) && a->heads > 0 && a->heads <= 65535 && a->kv_heads >= 0 && a->kv_heads <= 65535, "rotary: bad shape");
  TTB_REQUIRE(ctx, a->d > 0 && a->d % 8 == 0 && a->d <= 512, "rotary: the head size must be a multiple of 8, at most 512");
  TTB_REQUIRE(ctx, a->rotary_dim > 0 && a->rotary_dim % 2 == 0 && a->rotary_dim <= a->d, "rotary: an even number of a head's elements is turned");
  if (a->tokens == 0) return TTB_OK;
  TTB_REQUIRE(ctx, (a->kv_heads == 0) == (a->k == nullptr), "rotary: keys without key heads, or key heads without keys");
  TTB_REQUIRE(ctx, a->q && a->q_out && (a->kv_heads == 0 || a->k_out) && a->positions && a->freqs, "rotary: null pointer");
  const int64_t nq = a->heads * a->d, nk = a->kv_heads * a->d;
  TTB_REQUIRE(ctx, a->ldq >= nq && a->ldq_out >= nq && (nk == 0 || (a->ldk >= nk && a->ldk_out >= nk)), "rotary: rows overlap");
  DeviceGuard g(ctx->device);
  RotaryParams p = {};
  p.q = a->q; p.q_out = a->q_out; p.ldq = a->ldq; p.ldq_out = a->ldq_out;
  if (nk) { p.k = a->k; p.k_out = a->k_out; p.ldk = a->ldk; p.ldk_out = a->ldk_out; }
  p.tokens = (int)a->tokens; p.heads = (int)a->heads; p.kv_heads = (int)a->kv_heads; p.d = (int)a->d;
  p.half = (int)(a->rotary_dim / 2);
  p.interleaved = a->interleaved != 0;
  p.scale = a->scale;
  p.positions = a->positions;
  p.freqs = a->freqs;
  if (a->dtype == TTB_F32) return launch_rotary<float, false>(ctx, p, "rotary");
  if (a->dtype == TTB_F16) return launch_rotary<__half, false>(ctx, p, "rotary");
  return launch_rotary<__nv_bfloat16, false>(ctx, p, "rotary");
}

extern "C" int ttb_paged_append(ttb_ctx* ctx, int dtype, const ttb_paged_kv* kv, int64_t tokens, const void* k, int64_t ldk, const void* v, int64_t ldv,
                                const ttb_paged_rotary* r) {
  return ttb_paged_append_room(ctx, dtype, kv, tokens, k, ldk, v, ldv, r, nullptr);
}

extern "C" int ttb_paged_append_room(ttb_ctx* ctx, int dtype, const ttb_paged_kv* kv, int64_t tokens, const void* k, int64_t ldk, const void* v, int64_t ldv,
                                     const ttb_paged_rotary* r, const int32_t* room) {
  if (!ctx) return TTB_ERR_INVALID;
  RotaryParams p = {};
  const int bad = check_kv(ctx, "paged_append", dtype, kv, tokens, &p.s);
  if (bad) return bad;
  const int64_t n = kv->kv_heads * kv->d;
  p.d = (int)kv->d;
  p.kv_heads = (int)kv->kv_heads;
  if (r) {
    TTB_REQUIRE(ctx, r->freqs && r->rotary_dim > 0 && r->rotary_dim % 2 == 0 && r->rotary_dim <= kv->d,
                "paged_append: an even number of a head's elements is turned");
    TTB_REQUIRE(ctx, r->heads >= 0 && r->heads <= 65535, "paged_append: bad number of query heads");
    TTB_REQUIRE(ctx, tokens == 0 || ((r->heads == 0) == (r->q == nullptr) && (r->heads == 0) == (r->q_out == nullptr)),
                "paged_append: queries without heads, or heads without queries");
    TTB_REQUIRE(ctx, r->heads == 0 || (r->ldq >= r->heads * kv->d && r->ldq_out >= r->heads * kv->d), "paged_append: rows overlap");
    p.half = (int)(r->rotary_dim / 2);
    p.interleaved = r->interleaved != 0;
    p.scale = r->scale;
    p.freqs = r->freqs;
    p.heads = (int)r->heads;
    if (p.heads) { p.q = r->q; p.q_out = r->q_out; p.ldq = r->ldq; p.ldq_out = r->ldq_out; }
  }
  if (tokens == 0 || kv->B == 0) return TTB_OK;
  TTB_REQUIRE(ctx, k && v, "paged_append: null pointer");
  TTB_REQUIRE(ctx, ldk >= n && ldv >= n, "paged_append: rows overlap");
  DeviceGuard g(ctx->device);
  p.k = k; p.v = v; p.ldk = ldk; p.ldv = ldv;
  p.keys = kv->keys; p.values = kv->values; p.page_stride = kv->page_stride;
  p.room = room;
  p.tokens = (int)tokens;
  return dtype == TTB_F16 ? launch_rotary<__half, true>(ctx, p, "paged_append") : launch_rotary<__nv_bfloat16, true>(ctx, p, "paged_append");
}

extern "C" int ttb_paged_reserve(ttb_ctx* ctx, const ttb_paged_tables* a, const int32_t* new_tokens, int64_t page_tokens, int32_t* granted, int32_t* copies) {
  return ttb_paged_reserve_room(ctx, a, new_tokens, page_tokens, granted, copies, nullptr);
}

extern "C" int ttb_paged_reserve_room(ttb_ctx* ctx, const ttb_paged_tables* a, const int32_t* new_tokens, int64_t page_tokens, int32_t* granted, int32_t* copies,
                                      int32_t* room) {
  if (!ctx) return TTB_ERR_INVALID;
  Tables t;
  const int bad = check_tables(ctx, "paged_reserve", a, &t);
  if (bad) return bad;
  TTB_REQUIRE(ctx, page_tokens > 0 && page_tokens <= (1ll << 20) && page_tokens * a->width <= (1ll << 30), "paged_reserve: bad page size");
  // the pages that all rows want together are summed in 32 bits
  TTB_REQUIRE(ctx, a->B * a->width < (1ll << 31), "paged_reserve: a table has fewer than 2^31 entries");
  if (a->B == 0) return TTB_OK;
  TTB_REQUIRE(ctx, a->lens && new_tokens && granted && copies, "paged_reserve: null pointer");
  DeviceGuard g(ctx->device);
  void* ws = nullptr;
  int s = ttb_alloc(ctx, (size_t)a->pages * 3 * sizeof(int), "paged_reserve/scratch", &ws);
  if (s) return s;
  int* w = static_cast<int*>(ws);
  launch_pdl(paged_reserve_kernel, dim3(1), dim3(kManageThreads), 0, ctx->stream, t, new_tokens, (int)page_tokens, granted, copies, room, w, w + a->pages,
             w + 2 * a->pages);
  s = launched(ctx, "paged_reserve");
  const int f = ttb_free(ctx, ws, "paged_reserve/scratch");
  return s ? s : f;
}

extern "C" int ttb_paged_fork(ttb_ctx* ctx, const ttb_paged_tables* a, const int32_t* parents) {
  if (!ctx) return TTB_ERR_INVALID;
  Tables t;
  const int bad = check_tables(ctx, "paged_fork", a, &t);
  if (bad) return bad;
  if (a->B == 0) return TTB_OK;
  TTB_REQUIRE(ctx, a->lens && parents, "paged_fork: null pointer");
  DeviceGuard g(ctx->device);
  const size_t smem = (size_t)a->B * (kForkColumns + 1) * sizeof(int32_t);
  static bool configured[64] = {};
  const int dev = ctx->device < 64 ? ctx->device : 63;
  if (!configured[dev]) {
    TTB_CUDA(ctx, cudaFuncSetAttribute(paged_fork_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxSequences * (kForkColumns + 1) * 4));
    configured[dev] = true;
  }
  launch_pdl(paged_fork_kernel, dim3((unsigned)((a->width + kForkColumns - 1) / kForkColumns)), dim3(256), smem, ctx->stream, t, parents);
  return launched(ctx, "paged_fork");
}

extern "C" int ttb_paged_copy(ttb_ctx* ctx, const ttb_paged_pool* pool, const int32_t* pairs, int64_t n) {
  if (!ctx) return TTB_ERR_INVALID;
  const int bad = check_pool(ctx, "paged_copy", pool);
  if (bad) return bad;
  TTB_REQUIRE(ctx, n >= 0 && n < (1ll << 30), "paged_copy: bad number of pairs");
  if (n == 0) return TTB_OK;
  TTB_REQUIRE(ctx, pairs, "paged_copy: null pointer");
  DeviceGuard g(ctx->device);
  return launch_copy(ctx, pool, pairs, n, nullptr, Tables{}, nullptr);
}

extern "C" int ttb_paged_compact(ttb_ctx* ctx, const ttb_paged_tables* a, const ttb_paged_pool* pool, int32_t* used) {
  if (!ctx) return TTB_ERR_INVALID;
  Tables t;
  int s = check_tables(ctx, "paged_compact", a, &t);
  if (s) return s;
  s = check_pool(ctx, "paged_compact", pool);
  if (s) return s;
  TTB_REQUIRE(ctx, pool->pages == a->pages, "paged_compact: the pool and the reference counts differ in pages");
  TTB_REQUIRE(ctx, used, "paged_compact: null pointer");
  DeviceGuard g(ctx->device);
  void* ws = nullptr;
  s = ttb_alloc(ctx, ((size_t)a->pages * 2 + 3) * sizeof(int32_t), "paged_compact/scratch", &ws);
  if (s) return s;
  int32_t *to = static_cast<int32_t*>(ws), *pairs = to + a->pages, *moves = pairs + a->pages + 2;
  launch_pdl(paged_compact_kernel, dim3(1), dim3(kManageThreads), 0, ctx->stream, a->refs, (int)a->pages, used, to, pairs, moves);
  s = launched(ctx, "paged_compact");
  if (!s && (a->pages > 1 || a->B > 0)) s = launch_copy(ctx, pool, pairs, a->pages / 2, moves, t, to);
  const int f = ttb_free(ctx, ws, "paged_compact/scratch");
  return s ? s : f;
}
