// Attention over cache pages for many rows: chunks of prompts, and tokens of many heads to a key head. Bound by the tensor cores and the special-function units
// where the rows fill the tiles, by reading keys and values where they do not.
//
// One CTA an SM walks its stretch of the line (ttb_paged_rules.cuh). A tile is two sets of 128 query rows (tokens x heads of a key head) that share every key and value
// tile of 128 tokens, so that 64 KB of them (heads of 128) feed 2 x 128 rows: with a set alone the tensor cores would want them twice as fast. A tile whose rows all
// fit one set (a few tokens) puts them into both: the sets take the key tiles in turn and are joined at the tile's end, so that one's products still run beside the other's softmax.
//   warps 0, 2  : loads - warp 0 queries and keys, warp 2 values, each as soon as its ring (of two or four tiles) has room; a lane for each box (a page, or 128 tokens)
//                 and half of a head
//   warps 1, 3  : matrix products of a set each - S = Q K^T (128 x 128, fp32 in TMEM), O += P V with P in TMEM over the scores it came from, V as it lies, in
//                 the order QK(0), PV(0), QK(1), PV(1), ...; everything a product waits for but the softmax is a barrier poll
//   warps 4..11 : softmax, a warpgroup a set, a row a thread: scores from TMEM, exp2 with the scale folded in, P back to TMEM in 16 bits. The row's reference is the maximum of
//                 its first 32 keys (fp16: 2^6 below it); it is raised (and O rescaled) only where the sum of 32 probabilities passes 2^15: the division by the sum makes the result
//                 independent of it. References are whole numbers (of log2), so that probabilities that are brought to a new one are not rounded a second time (unless, in fp16,
//                 they fall below 2^-14 there, 2^-20 of the largest).
// A tile's output is written while the next one's first scores are made. Every wait is bounded. The probabilities are rounded to the values' 16 bits, as in the kernel for few
// rows; their sums are not.
// 4000 tokens over 12000, 32 heads of 128 on 8 key heads, bf16: 890 us, 1.03 PFLOP/s of products that the mask leaves; a pair of units takes 4400 cycles, of which the products
// are 2050 and a set's exponentials alone 1024 on their own unit, with the conversions, sums and tensor memory traffic of 256 rows beside them. 16 requests of 3 to 6
// tokens over up to 16000, 64 heads of 128 on 8: 144 to 151 us, 4.2 to 4.4 TB/s: two tiles of values are the most that fit beside the queries, and their way from memory shows
// (a third place for keys changed nothing).
#include <algorithm>
#include <type_traits>

#include "ttb_paged_attention.cuh"
#include "ttb_sm100.cuh"

using namespace ttb;
using namespace ttb::paged;
using namespace ttb::sm100;

namespace {

constexpr int kThreads = 384;
constexpr int kSet = kManyRows / 2;      // rows of a set
constexpr int kHalf = kUnit * 128;       // bytes of 128 rows of 64 elements
constexpr uint32_t kTmemCols = 512;
constexpr float kSumLimit = 32768.0f;  // a sum of probabilities below this keeps each of them inside fp16's and bf16's range
static_assert(kUnit == 128 && kSet == 128, "the products are 128 x 128");

template <int D> struct Shape {
  static constexpr int kHalves = D / 64;
  static constexpr int kTile = kHalves * kHalf;
  static constexpr int kStages = D == 128 ? 4 : 8;
  static constexpr int kRing = 2 * kTile;                           // after the two sets' queries
  static constexpr int kStaging = kRing + kStages * kTile;          // 2 KB for each softmax warp: 32 rows of 32 outputs
  static constexpr int kExchange = kStaging + 8 * 2048;             // float [4 warps][16 columns][32 rows]
  static constexpr int kStats = kExchange + 4 * 16 * 32 * 4;        // float2 [4 warps][32 rows]
  static constexpr int kPrefix = kStats + 4 * 32 * 8;
  static constexpr int kScratch = kPrefix + (kMaxSequences + 1) * 8;
  static constexpr int kWorks = kScratch + kThreads / 32 * 8;
  static constexpr int kBars = kWorks + kRingWorks * (int)sizeof(Work);
  static constexpr int kFirstSlotBar = 20 + 2 * kRingWorks;
  static constexpr int kNumBars = kFirstSlotBar + 5 * kStages;
  static constexpr int kBytes = kBars + kNumBars * 8 + 16;
};

// mbar_wait in few instructions, for the same reason as Work: a round lasts up to kSuspendHintNs, some 40 ns at least.
__device__ __forceinline__ bool wait_on(uint32_t bar, uint32_t parity, volatile int* abort_flag) {
#pragma unroll 1
  for (int i = 0; i < 1 << 18; ++i) {
    if (mbar_try_wait(bar, parity)) return true;
    if (*abort_flag) return false;
  }
  *abort_flag = 1;
  return false;
}

// Two fp32 operations an instruction.
__device__ __forceinline__ void fma2(uint32_t a0, uint32_t a1, float b, float c, float* d0, float* d1) {
  asm("{\n"
      ".reg .b64 a, b, c, d;\n"
      "mov.b64 a, {%2, %3};\n"
      "mov.b64 b, {%4, %4};\n"
      "mov.b64 c, {%5, %5};\n"
      "fma.rn.f32x2 d, a, b, c;\n"
      "mov.b64 {%0, %1}, d;\n"
      "}\n"
      : "=f"(*d0), "=f"(*d1)
      : "r"(a0), "r"(a1), "f"(b), "f"(c));
}
__device__ __forceinline__ unsigned long long add2(unsigned long long s, float a0, float a1) {
  unsigned long long d;
  asm("{\n"
      ".reg .b64 a;\n"
      "mov.b64 a, {%2, %3};\n"
      "add.rn.f32x2 %0, %1, a;\n"
      "}\n"
      : "=l"(d)
      : "l"(s), "f"(a0), "f"(a1));
  return d;
}
__device__ __forceinline__ float lo2(unsigned long long s) { return __uint_as_float((uint32_t)s); }
__device__ __forceinline__ float hi2(unsigned long long s) { return __uint_as_float((uint32_t)(s >> 32)); }

// 2^n for a whole n of at most 0.
__device__ __forceinline__ float power_of_2(float n) { return n < -126.f ? 0.f : __int_as_float(((int)n + 127) << 23); }

// How a part's units fall to the two sets.
__device__ __forceinline__ void share_out(const Params& p, Work* w) {
  const int tokens = p.split.half;  // of a set
  if (w->turns) {
    w->count[0] = (w->units + 1) / 2;
    w->count[1] = w->units / 2;
  } else {
    const int keys = p.split.causal ? min(w->pos0 + tokens, w->keys) : w->keys;
    w->count[0] = max(0, min(w->units, (keys + kUnit - 1) / kUnit - w->first));
    w->count[1] = w->units;
  }
}

template <typename T, int D>
__global__ void __launch_bounds__(kThreads, 1)
paged_tc_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v, const Params p) {
  using S = Shape<D>;
  constexpr int FMT = std::is_same<T, __nv_bfloat16>::value ? 1 : 0;
  constexpr uint32_t IDESC_S = idesc_f16(FMT, 128, kUnit, 0), IDESC_O = idesc_f16(FMT, 128, D, 1);
  extern __shared__ __align__(1024) uint8_t smem[];
  const uint32_t base = smem_u32(smem);
  long long* prefix = reinterpret_cast<long long*>(smem + S::kPrefix);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + S::kBars);
  const uint32_t bar0 = smem_u32(bars);
  auto bar = [&](int k) { return bar0 + 8u * k; };
  auto q_full = [&](int s) { return bar(s); };
  auto q_empty = [&](int s) { return bar(2 + s); };
  auto s_full = [&](int s) { return bar(4 + s); };
  auto p_ready = [&](int s) { return bar(6 + s); };
  auto o_done = [&](int s) { return bar(8 + s); };
  auto ex_full = [&](int quad) { return bar(10 + quad); };
  auto ex_empty = [&](int quad) { return bar(14 + quad); };
  auto q_empty_b = [&]() { return bar(18); };  // the first queries' buffer, by the second set where both read it
  // A tile has landed for the first set, the second, or both (2). A wait tells a phase from the next and not from the one after: a barrier's waiters have to
  // wait for its every phase, so that a tile that one set passes over is not told to it.
  const uint32_t v_tail = bar(19);  // values that end inside their tile, for the warp that loads them
  auto part_full = [&](uint32_t n) { return bar(20 + (int)(n % kRingWorks)); };
  auto part_empty = [&](uint32_t n) { return bar(20 + kRingWorks + (int)(n % kRingWorks)); };
  auto kv_full = [&](int f, uint32_t g) { return bar(S::kFirstSlotBar + f * S::kStages + (int)(g % S::kStages)); };
  auto kv_empty = [&](int s, uint32_t g) { return bar(S::kFirstSlotBar + (3 + s) * S::kStages + (int)(g % S::kStages)); };  // by the sets that read the tile
  auto kv_tile = [&](uint32_t g) { return base + S::kRing + (g % S::kStages) * S::kTile; };
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + S::kNumBars);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  volatile int* passed = reinterpret_cast<volatile int*>(tmem_slot + 2);  // [2]: units whose products a set has sent out, or passed over
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  pdl_trigger();
  if (threadIdx.x == 0) {
    for (int k = 0; k < S::kNumBars; ++k) {
      int count = 1;
      if (k == 6 || k == 7) count = 4;                                                            // p_ready: the set's four warps
      if (k >= 20 + kRingWorks && k < 20 + 2 * kRingWorks) count = kThreads / 32 - 1;             // part_empty: all warps but the one that fills it
      mbar_init(bar(k), count);
    }
    *abort_flag = 0;
    passed[0] = passed[1] = 0;
    mbar_init_fence();
  }
  if (warp == 1) tmem_alloc(smem_u32(tmem_slot), kTmemCols);
  if (threadIdx.x == 64) {
    prefetch_tensormap(&tm_q);
    prefetch_tensormap(&tm_k);
    prefetch_tensormap(&tm_v);
  }
  pdl_wait();
  const long long total = line_up(p, prefix, reinterpret_cast<long long*>(smem + S::kScratch), kThreads);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const int ctas = ctas_of(total, (int)gridDim.x, 1), cta = blockIdx.x;
  const long long lo = cta < ctas ? first_unit(total, ctas, cta) : 0, hi = cta < ctas ? first_unit(total, ctas, cta + 1) : 0;
  if (cta >= ctas && threadIdx.x == 0) p.parts.cuts[cta].pieces = 0;
  const int set_tokens = p.split.half;
  Work* works = reinterpret_cast<Work*>(smem + S::kWorks);
  // The n-th part, for every warp but the one that works them out. False: no part, there are no more or something gave up.
  auto take_part = [&](uint32_t n, Work* w) {
    const bool ok = __all_sync(0xffffffffu, wait_on(part_full(n), (n / kRingWorks) & 1u, abort_flag));
    if (!ok) return false;
    *w = works[n % kRingWorks];
    __syncwarp();
    if (lane == 0) mbar_arrive(part_empty(n));
    return w->units >= 0;
  };

  if (cta < ctas && warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
    if ((warp & 1) == 0) {
      // ------------------------------------------------------------------ loads
      const int loader = warp >> 1;
      const int page_tokens = 1 << p.s.page_shift, box_rows = min(page_tokens, kUnit);
      const int box = lane / S::kHalves, half = lane % S::kHalves;
      uint32_t g = loader, n_q[2] = {0, 0}, n_b = 0, n_tail = 0, n = 0;  // g: tile, keys even and values odd
      uint32_t used[2] = {0, 0}, parity[2] = {0, 0};  // a bit for each slot: whether the set reads what is there, and the phase of its kv_empty
      bool ok = true, both = false;                   // both: the second set reads the first queries' buffer too
      // The first loader works the parts out, one ahead of its own loads.
      Part t = {};
      long long u = lo;
      bool cut_here = false;
      auto publish = [&](Work* w) {
        w->units = -1;
        if (n > 0) u += t.take;
        if (u < hi) {
          if (n > 0) next_part(p, t, hi - u);
          else t = part_at(p, prefix, lo, hi - lo);
          *w = work_of(p, t, 2 * cta + (u == lo ? 0 : 1));
          share_out(p, w);
          if (w->slot >= 0 && t.first == 0) {
            cut_here = true;
            if (lane == 0) p.parts.cuts[cta] = cut_of(p, t, u, total, cta, ctas, w->slot);
          }
        }
        ok = __all_sync(0xffffffffu, ok && wait_on(part_empty(n), ((n / kRingWorks) & 1u) ^ 1u, abort_flag));
        if (ok && lane == 0) works[n % kRingWorks] = *w;
        __syncwarp();
        if (ok && lane == 0) mbar_arrive(part_full(n));
        return ok && w->units >= 0;
      };
      // A lane's page is looked up a unit ahead (and looked at when it is needed), and serves its keys and values.
      auto page_at = [&](const Work& w, int i) {
        const int key = (w.first + i) * kUnit + box * box_rows;
        return key < w.keys && box * box_rows < kUnit ? p.s.table[w.b * p.s.table_stride + (key >> p.s.page_shift)] : 0;
      };
      Work w = {}, w2;
      int page = 0;
      for (;; ++n) {  // w2 is the n-th part; the loads are those of w, the one before
        const bool more = loader == 0 ? publish(&w2) : take_part(n, &w2);
        if (w.units == 0 && more) page = page_at(w2, 0);  // at the beginning, and behind a part without keys (more tokens than the table lists)
        for (int i = 0; i < w.units && ok; ++i) {
          const int key = (w.first + i) * kUnit + box * box_rows, y = w.key_row + (key & (page_tokens - 1));
          int mine = -1;
          if (key < w.keys && box * box_rows < kUnit) {
            mine = page;
            if (mine < 0 || mine >= p.s.pages) {
              bad_index(p.s.status);
              mine = 0;
            }
          }
          page = i + 1 < w.units ? page_at(w, i + 1) : more ? page_at(w2, 0) : 0;
          const uint32_t bytes = (uint32_t)(__popc(__ballot_sync(0xffffffffu, mine >= 0)) * box_rows * 128);
          const bool reads[2] = {w.turns ? (i & 1) == 0 : i < w.count[0], w.turns ? (i & 1) == 1 : true};
          const uint32_t slot = 1u << (g % S::kStages);
#pragma unroll
          for (int s = 0; s < 2; ++s) {
            if (used[s] & slot) {
              ok = ok && wait_on(kv_empty(s, g), (parity[s] & slot) != 0, abort_flag);
              parity[s] ^= slot;
            }
            used[s] = reads[s] ? used[s] | slot : used[s] & ~slot;
          }
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          // Values behind the last key become zero, whatever the page happens to hold there: a probability of zero would not undo what is not finite.
          const int there = w.keys - (w.first + i) * kUnit;
          const bool tail = loader && there < kUnit;
          const uint32_t full = kv_full(reads[0] ? (reads[1] ? 2 : 0) : 1, g), landed = tail ? v_tail : full;
          if (lane == 0) mbar_expect_tx(landed, bytes);
          __syncwarp();
          if (mine >= 0) tma_load_3d(kv_tile(g) + half * kHalf + box * box_rows * 128, loader ? &tm_v : &tm_k, landed, half * 64, y, mine);
          if (tail) {
            ok = __all_sync(0xffffffffu, wait_on(v_tail, n_tail++ & 1u, abort_flag));
            if (!ok) break;
#pragma unroll 1
            for (int c = lane; c < (kUnit - there) * S::kHalves * 8; c += 32) {
              const int r = there + c / (S::kHalves * 8), col = c % (S::kHalves * 8);
              asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(kv_tile(g) + (col >> 3) * kHalf + r * 128 + (col & 7) * 16), "r"(0) : "memory");
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(full);
          }
          g += 2;
          // the queries go behind the first keys, which need no other tile to end
#pragma unroll
          for (int s = 0; s < 2; ++s) {
            if (!ok || loader || i > 0 || w.count[s] == 0 || (s == 1 && w.turns)) continue;
            ok = wait_on(q_empty(s), (n_q[s] & 1u) ^ 1u, abort_flag);
            if (s == 0) {
              if (both) ok = ok && wait_on(q_empty_b(), n_b++ & 1u, abort_flag);
              both = w.turns && w.count[1] > 0;
            }
            ok = __all_sync(0xffffffffu, ok);
            if (ok && lane == 0) {
              mbar_expect_tx(q_full(s), (uint32_t)(set_tokens * p.split.block_heads * D * 2));
              for (int h = 0; h < S::kHalves; ++h)
                tma_load_3d(base + s * S::kTile + h * kHalf, &tm_q, q_full(s), h * 64, w.head0, w.tok0 + s * set_tokens);
            }
            ++n_q[s];
          }
        }
        if (!more || !ok) break;
        w = w2;
      }
      if (loader == 0 && !cut_here && lane == 0) p.parts.cuts[cta].pieces = 0;
      if (*abort_flag) {  // copies in flight land before shared memory is given back
        const long long t0 = clock64();
        while (clock64() - t0 < 4000000LL) {
        }
      }
    } else {
      // ------------------------------------------------------------------ matrix products of set s
      // One lane, and few instructions between the arrival of the probabilities and the products: beside the softmax they come from the second-level instruction
      // cache every time.
      const int s = warp >> 1;
      if (lane == 0) {
        const uint32_t tm_s = tmem + (uint32_t)(s * 128), tm_o = tmem + 256u + (uint32_t)(s * D);
        uint32_t g = 0, n_q[2] = {0, 0}, n_p = 0, w_g = 0;  // w_g: the tile of values that waits for its probabilities
        uint32_t full_parity[2] = {0, 0};                   // a bit for each slot: the phase of the set's kv_full, and of both sets'
        int n_units = 0;
        bool ok = true, any = false, w_first = false, w_last = false, w_shared = false;
        auto landed = [&](bool shared, uint32_t g) {
          const uint32_t slot = 1u << (g % S::kStages), parity = shared ? full_parity[1] : full_parity[0];
          if (shared) full_parity[1] ^= slot;
          else full_parity[0] ^= slot;
          return wait_on(kv_full(shared ? 2 : s, g), (parity & slot) != 0, abort_flag);
        };
        for (uint32_t n = 0;; ++n) {
          if (!wait_on(part_full(n), (n / kRingWorks) & 1u, abort_flag)) break;
          const Work& part = works[n % kRingWorks];
          const bool more = part.units >= 0, turns = part.turns;
          const int units = more ? part.units : 1, count0 = part.count[0], count1 = part.count[1], count = s ? count1 : count0, buf = turns ? 0 : s;
          mbar_arrive(part_empty(n));
          int j = 0;
          for (int i = 0; i < units; ++i, g += 2) {  // (behind the last part: its last output product)
            const bool mine = more && (turns ? (i & 1) == s : i < count), shared = !turns && i < count0;
            // an output product never stays behind a tile's end: the sets' softmax warps wait for one another there
            const bool output = any && (mine || i == 0 || !turns);
            if (mine) ok = landed(shared, g) && (j > 0 || wait_on(q_full(buf), (buf ? n_q[1] : n_q[0]) & 1u, abort_flag));
            if (ok && output) ok = landed(w_shared, w_g) && wait_on(p_ready(s), n_p++ & 1u, abort_flag);  // the probabilities come last
            if (!ok) break;
            if (mine) {
              // The sets' steps (an output product with the next scores) go out in turn, unit by unit. Both at once they would mix in the pipe and end side by side,
              // and both softmax at once would leave the tensor cores idle after; and a set a unit ahead would wait for keys whose place the other still holds. Only
              // an order: a set that does not get its turn in time goes on without.
              const int unit = n_units + i;
#pragma unroll 1
              for (int tries = 0; passed[1 - s] < unit + s && tries < 500; ++tries) {
              }
            }
            tc_fence_after();
            if (output) {
              // the values' 64-column halves are kHalf bytes apart: the descriptor's leading offset
              const uint32_t v_lo = ((kv_tile(w_g) & 0x3FFFFu) >> 4) | ((uint32_t)(kHalf >> 4) << 16);
#pragma unroll
              for (int k = 0; k < kUnit / 16; ++k)  // 16 keys: 8 TMEM columns of P, 16 rows of 128 bytes of V
                umma_f16_ts(tm_o, tm_s + (uint32_t)(k * 8), v_lo + (uint32_t)(k * (16 * 128 >> 4)), IDESC_O, !w_first || k != 0);
            }
            if (mine) {
              const uint32_t q_lo = desc_lo(base + buf * S::kTile), k_lo = desc_lo(kv_tile(g));
#pragma unroll
              for (int k = 0; k < D / 16; ++k) {
                const uint32_t off = (uint32_t)((k >> 2) * (kHalf >> 4) + (k & 3) * 2);
                umma_f16(tm_s, q_lo + off, k_lo + off, IDESC_S, k != 0);
              }
              tc_commit(s_full(s));
            }
            passed[s] = n_units + i + 1;
            if (output) {
              if (w_last) tc_commit(o_done(s));
              tc_commit(kv_empty(s, w_g));
              any = false;
            }
            if (mine) {
              tc_commit(kv_empty(s, g));
              if (j == count - 1) tc_commit(buf == s ? q_empty(s) : q_empty_b());
              any = true;
              w_g = g + 1;
              w_first = j == 0;
              w_last = j == count - 1;
              w_shared = shared;
              ++j;
            }
          }
          if (!more || !ok) break;
          n_units += units;
          n_q[0] += count0 > 0;
          n_q[1] += !turns && count1 > 0;
        }
      }
      __syncwarp();
    }
  } else if (cta < ctas) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
    // ------------------------------------------------------------------ softmax and output
    const int s = (warp - 4) >> 2, quad = warp & 3;  // TMEM lanes [32 * quad, 32 * quad + 32) are the ones this warp may touch
    const int row = quad * 32 + lane;
    const uint32_t lane_addr = (uint32_t)(quad * 32) << 16;
    const uint32_t ts = tmem + (uint32_t)(s * 128) + lane_addr, to = tmem + 256u + (uint32_t)(s * D) + lane_addr;
    uint8_t* stage = smem + S::kStaging + (warp - 4) * 2048;
    float* exchange = reinterpret_cast<float*>(smem + S::kExchange) + quad * 16 * 32;
    float2* stats = reinterpret_cast<float2*>(smem + S::kStats) + quad * 32;
    uint32_t n_s = 0, n_o = 0, n_x = 0;
    bool ok = true;
    // what is left to do of the tile before
    struct {
      bool any, has, join, skip;
      int tok0, head0, heads, row0, rows, slot;
      float m, l;
    } w = {};
    auto all_ok = [&](bool mine) { return __all_sync(0xffffffffu, mine); };

    auto flush = [&]() {  // whole warp
      w.any = false;
      if (w.has) {
        if (!all_ok(wait_on(o_done(s), n_o & 1u, abort_flag))) return false;
        ++n_o;
        tc_fence_after();
      }
      if (w.skip) return true;  // the warp has no rows (its sibling of the other set neither, where they are joined)
      float scale = w.has ? 1.f : 0.f, other = 0.f;
      if (w.join) {  // both sets hold sums of the same rows: the second's go to the first
        if (s == 1) {
          if (!all_ok(wait_on(ex_empty(quad), (n_x & 1u) ^ 1u, abort_flag))) return false;
          stats[lane] = make_float2(w.m, w.l);
          __syncwarp();
          if (lane == 0) mbar_arrive(ex_full(quad));
          ++n_x;
#pragma unroll 1
          for (int c = 0; c < D / 16; ++c, ++n_x) {
            uint32_t r[16];
            tmem_ld16_issue(to + (uint32_t)(c * 16), r);
            tmem_ld_wait();
            if (!all_ok(wait_on(ex_empty(quad), (n_x & 1u) ^ 1u, abort_flag))) return false;
#pragma unroll
            for (int e = 0; e < 16; ++e) exchange[e * 32 + lane] = __uint_as_float(r[e]);
            __syncwarp();
            if (lane == 0) mbar_arrive(ex_full(quad));
          }
          return true;
        }
        if (!all_ok(wait_on(ex_full(quad), n_x & 1u, abort_flag))) return false;
        const float2 o = stats[lane];
        __syncwarp();
        if (lane == 0) mbar_arrive(ex_empty(quad));
        ++n_x;
        const float m = fmaxf(w.m, o.x), sub = m == -INFINITY ? 0.f : m;
        scale = ex2(w.m - sub);
        other = ex2(o.x - sub);
        w.l = w.l * scale + o.y * other;
        w.m = m;
      }
      const float inv = (w.slot < 0) ? (w.l == 0.f ? 0.f : 1.f / w.l) : 1.f;
      scale *= inv;
      other *= inv;
      // rows of this warp: their number, and where lane / 4 + 8 k lies
      const int rows = w.rows - quad * 32;
      T* dst[4];
      if ((w.slot < 0)) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int r = quad * 32 + k * 8 + (lane >> 2), i = r / p.split.block_heads, h = r % p.split.block_heads;
          dst[k] = r < w.rows && h < w.heads ? static_cast<T*>(p.out) + (long long)(w.tok0 + i) * p.ldo + (long long)(w.head0 + h) * D + (lane & 3) * 8 : nullptr;
        }
      }
      const long long at = (long long)w.slot * kManyRows + w.row0 + row;
      float* part = p.parts.o + at * D;
      if (w.slot >= 0 && row < w.rows) p.parts.ml[at] = make_float2(w.m, w.l);
#pragma unroll 1
      for (int c = 0; c < D / 32; ++c) {
        uint32_t r[32];
        if (w.has) {
          tmem_ld32_issue(to + (uint32_t)(c * 32), r);
          tmem_ld_wait();
        } else {
#pragma unroll
          for (int e = 0; e < 32; ++e) r[e] = 0u;
        }
#pragma unroll
        for (int e = 0; e < 32; ++e) r[e] = __float_as_uint(scale == 0.f ? 0.f : __uint_as_float(r[e]) * scale);
        if (w.join) {
#pragma unroll
          for (int h = 0; h < 2; ++h, ++n_x) {
            if (!all_ok(wait_on(ex_full(quad), n_x & 1u, abort_flag))) return false;
#pragma unroll
            for (int e = 0; e < 16; ++e) r[h * 16 + e] = __float_as_uint(__uint_as_float(r[h * 16 + e]) + (other == 0.f ? 0.f : exchange[e * 32 + lane] * other));
            __syncwarp();
            if (lane == 0) mbar_arrive(ex_empty(quad));
          }
        }
        if ((w.slot < 0)) {  // through shared memory: stores of 64 bytes a row
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            uint4 v;
            v.x = pack2<T>(__uint_as_float(r[e * 8]), __uint_as_float(r[e * 8 + 1]));
            v.y = pack2<T>(__uint_as_float(r[e * 8 + 2]), __uint_as_float(r[e * 8 + 3]));
            v.z = pack2<T>(__uint_as_float(r[e * 8 + 4]), __uint_as_float(r[e * 8 + 5]));
            v.w = pack2<T>(__uint_as_float(r[e * 8 + 6]), __uint_as_float(r[e * 8 + 7]));
            *reinterpret_cast<uint4*>(stage + lane * 64 + ((e ^ (lane >> 1 & 3)) << 4)) = v;  // swizzled: no bank conflicts either way
          }
          __syncwarp();
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const int q = k * 8 + (lane >> 2);
            const uint4 v = *reinterpret_cast<const uint4*>(stage + q * 64 + (((lane & 3) ^ (q >> 1 & 3)) << 4));
            if (dst[k]) *reinterpret_cast<uint4*>(dst[k] + c * 32) = v;
          }
          __syncwarp();
        } else if (lane < rows) {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            *reinterpret_cast<float4*>(part + c * 32 + e * 4) =
                make_float4(__uint_as_float(r[e * 4]), __uint_as_float(r[e * 4 + 1]), __uint_as_float(r[e * 4 + 2]), __uint_as_float(r[e * 4 + 3]));
        }
      }
      return true;
    };

    Work t;
    for (uint32_t n = 0;; ++n) {
      const bool more = take_part(n, &t);
      if (w.any && !flush()) break;
      if (!more) break;
      const int set = t.turns ? 0 : s, count = s ? t.count[1] : t.count[0];
      const int set_row0 = set * set_tokens * p.split.block_heads;
      const int rows = min(set_tokens * p.split.block_heads, t.rows - set_row0);  // of the set
      const bool alive = quad * 32 < rows;                                        // whether the warp has any
      const int tok = set * set_tokens + row / p.split.block_heads;               // the row's token in the tile
      const int limit = p.split.causal && row < rows ? min(t.pos0 + tok + 1, t.keys) : t.keys;
      const int all_see = p.split.causal ? min(t.pos0 + set * set_tokens + quad * 32 / p.split.block_heads + 1, t.keys) : t.keys;
      const int any_sees = p.split.causal ? min(t.pos0 + set * set_tokens + min(quad * 32 + 31, rows - 1) / p.split.block_heads + 1, t.keys) : t.keys;
      float m_used = -INFINITY, l_run = 0.f;
      for (int j = 0; j < count; ++j, ++n_s) {
        const int k0 = (t.first + (t.turns ? 2 * j + s : j)) * kUnit;
        if (!all_ok(wait_on(s_full(s), n_s & 1u, abort_flag))) { ok = false; break; }
        if (alive) {
          tc_fence_after();
          const int live = max(0, min(any_sees - k0, kUnit) + 31) >> 5;  // chunks that some row of the warp sees
          const bool edge = k0 + kUnit > all_see;
          uint32_t r[32];
          auto mask = [&](int c) {
            if (k0 + (c + 1) * 32 > all_see) {
              const int n = limit - k0 - c * 32;
#pragma unroll
              for (int e = 0; e < 32; ++e)
                if (e >= n) r[e] = 0xff800000u;
            }
          };
          // The reference: any score near the largest does, and another pass over the tile would cost a third of its softmax (six prompts of 200 to 2000 tokens, heads of
          // 64: 130 us with the maximum of all 128, 125). A row that sees none of these 32 keys sees none of the others.
          if (j == 0) {
            tmem_ld32_issue(ts, r);
            tmem_ld_wait();
            mask(0);
            float top = -INFINITY;
#pragma unroll
            for (int e = 0; e < 32; e += 2) top = fmaxf(fmaxf(top, __uint_as_float(r[e])), __uint_as_float(r[e + 1]));
            m_used = floorf(top * p.scale) - kBelow<T>;
          }
          // A tile that every row sees the whole of: straight through, P kept until its sum says that the reference still holds. Short code, since the instruction cache is the other warps' too (with masks and rescaling in it 16 products took 3500 cycles in place of 1250).
          float l0 = 0.f, l1 = 0.f;
          bool done = false;
          if (!edge) {
            uint32_t pk[2][32];
            unsigned long long sum = 0, sum2 = 0;
            const float m_sub = m_used == -INFINITY ? 0.f : m_used;
            tmem_ld32_issue(ts, r);
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              float x[32];
              tmem_ld_wait();
#pragma unroll
              for (int e = 0; e < 32; e += 2) fma2(r[e], r[e + 1], p.scale, -m_sub, &x[e], &x[e + 1]);
              if (c < 3) tmem_ld32_issue(ts + (uint32_t)((c + 1) * 32), r);
#pragma unroll
              for (int e = 0; e < 32; e += 4) {
                const float a0 = ex2(x[e]), a1 = ex2(x[e + 1]), a2 = ex2(x[e + 2]), a3 = ex2(x[e + 3]);
                sum = add2(sum, a0, a1);
                sum2 = add2(sum2, a2, a3);
                pk[c >> 1][(c & 1) * 16 + (e >> 1)] = pack2<T>(a0, a1);
                pk[c >> 1][(c & 1) * 16 + (e >> 1) + 1] = pack2<T>(a2, a3);
              }
            }
            l0 = lo2(sum) + lo2(sum2);
            l1 = hi2(sum) + hi2(sum2);
            done = __all_sync(0xffffffffu, row >= rows || l0 + l1 < kSumLimit);
            if (done) {
              tmem_st32(ts, pk[0]);
              tmem_st32(ts + 32u, pk[1]);
            }
          }
          if (!done) {
            // 32 scores at a time; their probabilities replace scores that have been read
            l0 = l1 = 0.f;
            tmem_ld32_issue(ts, r);
#pragma unroll 1
            for (int c = 0; c < 4; ++c) {
              uint32_t pk[16];
              tmem_ld_wait();
              if (c < live) {  // warp-uniform
                mask(c);
                const float m_sub = m_used == -INFINITY ? 0.f : m_used;
                float x[32];
#pragma unroll
                for (int e = 0; e < 32; e += 2) fma2(r[e], r[e + 1], p.scale, -m_sub, &x[e], &x[e + 1]);
                if (c < 3) tmem_ld32_issue(ts + (uint32_t)((c + 1) * 32), r);
                unsigned long long sum = 0;
#pragma unroll
                for (int e = 0; e < 32; e += 2) {
                  const float a0 = ex2(x[e]), a1 = ex2(x[e + 1]);
                  sum = add2(sum, a0, a1);
                  pk[e >> 1] = pack2<T>(a0, a1);
                }
                float s0 = lo2(sum), s1 = hi2(sum);
                if (__builtin_expect(__any_sync(0xffffffffu, row < rows && !(s0 + s1 < kSumLimit)), 0)) {
                  // A score far above the reference (or no number): everything so far is brought to a new one, and these are made again. (O holds the tiles before:
                  // their products were complete before these scores were.)
                  float top = -INFINITY;
#pragma unroll
                  for (int e = 0; e < 32; ++e) top = fmaxf(top, x[e]);
                  const float m_new = fmaxf(m_used, floorf(m_sub + top) - kBelow<T>), corr = m_new == -INFINITY ? 1.f : power_of_2(m_used - m_new);
                  const float down = m_sub - (m_new == -INFINITY ? 0.f : m_new);
                  m_used = m_new;
                  l_run *= corr;
                  l0 *= corr;
                  l1 *= corr;
                  tmem_st_wait();
                  tmem_ld_wait();
#pragma unroll 1
                  for (int i = j > 0 ? 0 : D / 16; i < D / 16 + c; ++i) {
                    const uint32_t at = i < D / 16 ? to + (uint32_t)(i * 16) : ts + (uint32_t)((i - D / 16) * 16);
                    tmem_ld16_issue(at, pk);
                    tmem_ld_wait();
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                      const float2 f = unpack2<T>(pk[e]);
                      pk[e] = i < D / 16 ? __float_as_uint(__uint_as_float(pk[e]) * corr) : pack2<T>(f.x * corr, f.y * corr);
                    }
                    tmem_st16(at, pk);
                  }
                  tmem_st_wait();
                  s0 = s1 = 0.f;
#pragma unroll
                  for (int e = 0; e < 16; ++e) {
                    const float a0 = ex2(x[2 * e] + down), a1 = ex2(x[2 * e + 1] + down);
                    s0 += a0;
                    s1 += a1;
                    pk[e] = pack2<T>(a0, a1);
                  }
                }
                l0 += s0;
                l1 += s1;
              } else {
#pragma unroll
                for (int e = 0; e < 16; ++e) pk[e] = 0u;
              }
              tmem_st16(ts + (uint32_t)(c * 16), pk);
            }
          }
          l_run += l0 + l1;
          tmem_st_wait();
          tc_fence_before();
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(p_ready(s));
      }
      if (!ok) break;
      // what becomes of the tile. A set whose rows all lie before the part's keys has no sums, but says so to whoever joins the parts.
      w.any = count > 0 || !t.turns || s == 0;
      w.has = count > 0;
      w.join = t.turns && t.count[1] > 0;
      w.skip = !alive;
      w.tok0 = t.tok0 + set * set_tokens;
      w.head0 = t.head0;
      w.heads = t.heads;
      w.row0 = set_row0;
      w.rows = rows;
      w.slot = t.slot;
      w.m = m_used;
      w.l = l_run;
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, kTmemCols);
  }
  if (threadIdx.x == 0 && *abort_flag) atomicExch(p.s.status, (int)TTB_ERR_DEVICE_WAIT);
}

template <typename T, int D>
int launch(ttb_ctx* ctx, const ttb_paged_kv* kv, int64_t heads, const Params& p) {
  using S = Shape<D>;
  CUtensorMap tm_q, tm_k, tm_v;
  if (!encode_maps(kv, std::is_same<T, __nv_bfloat16>::value, heads, p, p.split.tile_tokens / 2, &tm_q, &tm_k, &tm_v))
    return fail(ctx, TTB_ERR_CUDA, "paged_attention: a tensor map was refused");
  static bool configured[64] = {};
  const int dev = ctx->device < 64 ? ctx->device : 63;
  if (!configured[dev]) {
    TTB_CUDA(ctx, cudaFuncSetAttribute(paged_tc_kernel<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kBytes));
    configured[dev] = true;
  }
  launch_pdl(paged_tc_kernel<T, D>, dim3((unsigned)ctx->sm_count), dim3(kThreads), S::kBytes, ctx->stream, tm_q, tm_k, tm_v, p);
  return launched(ctx, "paged_attention_tc");
}

}  // namespace

namespace ttb {
namespace paged {

int paged_tc_launch(ttb_ctx* ctx, int dtype, const ttb_paged_kv* kv, int64_t heads, const Params& p) {
  if (kv->d == 64) return dtype == TTB_F16 ? launch<__half, 64>(ctx, kv, heads, p) : launch<__nv_bfloat16, 64>(ctx, kv, heads, p);
  return dtype == TTB_F16 ? launch<__half, 128>(ctx, kv, heads, p) : launch<__nv_bfloat16, 128>(ctx, kv, heads, p);
}

}  // namespace paged
}  // namespace ttb
