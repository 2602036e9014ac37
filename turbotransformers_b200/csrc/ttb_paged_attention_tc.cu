// Attention over cache pages for many rows: chunks of prompts, and tokens of many heads to a key head. Bound by the tensor cores and the special-function units
// where the rows fill the tiles, by reading keys and values where they do not.
//
// One CTA an SM walks its stretch of the line (ttb_paged_rules.cuh). A tile is two sets of 128 query rows (tokens x heads of a key head) that share every key and value
// tile of 128 tokens, so that 64 KB of them (heads of 128) feed 2 x 128 rows: with a set alone the tensor cores would want them twice as fast. A tile whose rows all
// fit one set (a few tokens) puts them into both: the sets take the key tiles in turn and are joined at the tile's end, so that one's products still run beside the other's softmax.
//   warp 0      : loads - a lane for each box (a page, or 128 keys) and half of a head: queries, then keys and values in turn through one ring
//   warp 1      : matrix products - S = Q K^T (128 x 128, fp32 in TMEM), O += P V with P in TMEM over the scores it came from, V as it lies. Of a set the
//                 order is QK(0), PV(0), QK(1), PV(1), ..., the other set's products between; everything a product waits for but the softmax is a barrier poll.
//                 Rows of V behind the last key are set to zero here: a probability of zero would not undo what the page happens to hold.
//   warps 4..11 : softmax, a warpgroup a set, a row a thread: scores from TMEM, exp2 with the scale folded in, P back to TMEM in 16 bits. The row's maximum is that of its
//                 first tile; it is raised (and O rescaled) only where a tile's sum passes 2^15: the division by the sum makes the result independent of it.
// A tile's output is written while the next one's first scores are made. Every wait is bounded.
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
constexpr float kRowSumLimit = 32768.0f;  // a tile row sum below this keeps every probability inside fp16 / bf16 range
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
  static constexpr int kBars = kScratch + kThreads / 32 * 8;
  static constexpr int kNumBars = 10 + 2 * kStages + 8;
  static constexpr int kBytes = kBars + kNumBars * 8 + 16;
};

// How a part's units fall to the two sets.
struct Sets {
  bool turns;      // both hold the same rows and take the units in turn
  int units;       // of the part that have keys
  int count[2];    // each set's
};
__device__ __forceinline__ Sets sets_of(const Params& p, const Part& t) {
  const int tokens = p.split.tile_tokens / 2;  // of a set
  Sets s;
  s.turns = t.rows <= tokens * p.split.block_heads;
  s.units = max(0, min(t.take, (t.keys + kUnit - 1) / kUnit - (int)t.first));
  if (s.turns) {
    s.count[0] = (s.units + 1) / 2;
    s.count[1] = s.units / 2;
  } else {
    const int keys = p.split.causal ? min(t.pos0 + tokens, t.keys) : t.keys;
    s.count[0] = max(0, min(s.units, (keys + kUnit - 1) / kUnit - (int)t.first));
    s.count[1] = s.units;
  }
  return s;
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
  auto kv_full = [&](uint32_t g) { return bar(18 + (int)(g % S::kStages)); };
  auto kv_empty = [&](uint32_t g) { return bar(18 + S::kStages + (int)(g % S::kStages)); };
  auto kv_tile = [&](uint32_t g) { return base + S::kRing + (g % S::kStages) * S::kTile; };
  auto kv_phase = [&](uint32_t g) { return (g / S::kStages) & 1u; };
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + S::kNumBars);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  pdl_trigger();
  if (threadIdx.x == 0) {
    for (int k = 0; k < S::kNumBars; ++k) mbar_init(bar(k), k == 6 || k == 7 ? 4 : 1);  // p_ready: the set's four warps
    *abort_flag = 0;
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
  const int set_tokens = p.split.tile_tokens / 2;

  if (cta < ctas && warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
    if (warp == 0) {
      // ------------------------------------------------------------------ loads
      const int page_tokens = 1 << p.s.page_shift, box_rows = min(page_tokens, kUnit);
      uint32_t g = 0, nq[2] = {0, 0};
      bool ok = true;
      Part t = part_at(p, prefix, lo, hi - lo);
      for (long long u = lo; u < hi && ok;) {
        const Sets sets = sets_of(p, t);
        for (int i = 0; i < 2 * sets.units && ok; ++i) {
          const int key0 = ((int)t.first + (i >> 1)) * kUnit;
          const int boxes = (min(kUnit, t.keys - key0) + box_rows - 1) / box_rows;
          const int box = lane / S::kHalves, half = lane % S::kHalves;
          // a lane's page does not wait for the slot
          int page = 0;
          if (box < boxes) {
            bool bad;
            page = page_of(p.s, t.b, key0 + box * box_rows, &bad);
            if (bad) {
              bad_index(p.s.status);
              page = 0;
            }
          }
          ok = mbar_wait(kv_empty(g), kv_phase(g) ^ 1u, abort_flag);
          if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
          if (lane == 0) mbar_expect_tx(kv_full(g), (uint32_t)(boxes * box_rows * D * 2));
          __syncwarp();
          if (box < boxes) {
            const int y = (t.block / p.split.head_blocks << p.s.page_shift) + ((key0 + box * box_rows) & (page_tokens - 1));
            tma_load_3d(kv_tile(g) + half * kHalf + box * box_rows * 128, (i & 1) ? &tm_v : &tm_k, kv_full(g), half * 64, y, page);
          }
          ++g;
          if (i == 0) {  // behind the first keys, which need no other tile to end
#pragma unroll
            for (int s = 0; s < 2; ++s) {
              if (!ok || sets.count[s] == 0 || (s == 1 && sets.turns)) continue;
              ok = mbar_wait(q_empty(s), (nq[s] & 1u) ^ 1u, abort_flag);
              ok = __all_sync(0xffffffffu, ok);
              if (!ok) continue;
              if (lane == 0) {
                mbar_expect_tx(q_full(s), (uint32_t)(set_tokens * p.split.block_heads * D * 2));
                for (int h = 0; h < S::kHalves; ++h)
                  tma_load_3d(base + s * S::kTile + h * kHalf, &tm_q, q_full(s), h * 64, first_head(p, t.block), t.tok0 + s * set_tokens);
              }
              ++nq[s];
            }
          }
        }
        u += t.take;
        if (u < hi) next_part(p, t, hi - u);
      }
      if (*abort_flag) {  // copies in flight land before shared memory is given back
        const long long t0 = clock64();
        while (clock64() - t0 < 4000000LL) {
        }
      }
    } else if (warp == 1) {
      // ------------------------------------------------------------------ matrix products
      struct Pending {  // a set's output product that waits for its probabilities
        bool any, first, last, release;
        uint32_t g;  // its values
        int keys;    // of them that there are
      } pend[2] = {};
      uint32_t g0 = 0, nq[2] = {0, 0}, np[2] = {0, 0}, zeroed = 0xffffffffu;
      bool ok = true;
      auto pv = [&](int s) {
        Pending& w = pend[s];
        w.any = false;
        ok = mbar_wait(p_ready(s), np[s]++ & 1u, abort_flag) && mbar_wait(kv_full(w.g), kv_phase(w.g), abort_flag);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) return;
        const uint32_t tile = kv_tile(w.g);
        if (w.keys < kUnit && zeroed != w.g) {
          zeroed = w.g;
          for (int i = lane; i < (kUnit - w.keys) * S::kHalves * 8; i += 32) {
            const int r = w.keys + i / (S::kHalves * 8), c = i % (S::kHalves * 8);
            asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(tile + (c >> 3) * kHalf + r * 128 + (c & 7) * 16), "r"(0) : "memory");
          }
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          __syncwarp();
        }
        if (lane == 0) {
          tc_fence_after();
          // the values' 64-column halves are kHalf bytes apart: the descriptor's leading offset
          const uint32_t v_lo = ((tile & 0x3FFFFu) >> 4) | ((uint32_t)(kHalf >> 4) << 16);
#pragma unroll
          for (int k = 0; k < kUnit / 16; ++k)  // 16 keys: 8 TMEM columns of P, 16 rows of 128 bytes of V
            umma_f16_ts(tmem + 256u + (uint32_t)(s * D), tmem + (uint32_t)(s * 128 + k * 8), v_lo + (uint32_t)(k * (16 * 128 >> 4)), IDESC_O, !w.first || k != 0);
          if (w.last) tc_commit(o_done(s));
          if (w.release) tc_commit(kv_empty(w.g));
        }
        __syncwarp();
      };
      Part t = part_at(p, prefix, lo, hi - lo);
      for (long long u = lo; u < hi && ok;) {
        const Sets sets = sets_of(p, t);
        for (int i = 0; i < sets.units && ok; ++i) {
          const uint32_t gk = g0 + 2 * i;
#pragma unroll
          for (int s = 0; s < 2; ++s) {
            if (!ok) break;
            const bool mine = sets.turns ? (i & 1) == s : i < sets.count[s];
            // an output product never stays behind a tile's end: the sets' softmax warps wait for one another there
            if (pend[s].any && (mine || i == 0 || !sets.turns)) pv(s);
            if (!mine || !ok) continue;
            const int j = sets.turns ? i >> 1 : i, buf = sets.turns ? 0 : s;
            ok = mbar_wait(kv_full(gk), kv_phase(gk), abort_flag) && (j > 0 || mbar_wait(q_full(buf), (buf ? nq[1] : nq[0]) & 1u, abort_flag));
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            if (lane == 0) {
              tc_fence_after();
              const uint32_t q_lo = desc_lo(base + buf * S::kTile), k_lo = desc_lo(kv_tile(gk));
#pragma unroll
              for (int k = 0; k < D / 16; ++k) {
                const uint32_t off = (uint32_t)((k >> 2) * (kHalf >> 4) + (k & 3) * 2);
                umma_f16(tmem + (uint32_t)(s * 128), q_lo + off, k_lo + off, IDESC_S, k != 0);
              }
              tc_commit(s_full(s));
              if (sets.turns || s == 1) tc_commit(kv_empty(gk));
              if (sets.turns ? i == sets.units - 1 : j == sets.count[s] - 1) tc_commit(q_empty(buf));
            }
            __syncwarp();
            pend[s] = Pending{true, j == 0, j == sets.count[s] - 1, sets.turns || s == 1, gk + 1, min(kUnit, t.keys - ((int)t.first + i) * kUnit)};
          }
        }
        if (sets.units > 0) {
          if (sets.turns) ++nq[0];
          else {
            nq[0] += sets.count[0] > 0;
            nq[1] += sets.count[1] > 0;
          }
        }
        g0 += 2 * sets.units;
        u += t.take;
        if (u < hi) next_part(p, t, hi - u);
      }
#pragma unroll
      for (int s = 0; s < 2; ++s)
        if (ok && pend[s].any) pv(s);
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
    bool ok = true, cut_here = false;
    // what is left to do of the tile before
    struct {
      bool any, has, whole, join, skip;
      int tok0, head0, heads, row0, rows, slot;
      float m, l;
    } w = {};
    auto all_ok = [&](bool mine) { return __all_sync(0xffffffffu, mine); };

    auto flush = [&]() {  // whole warp
      w.any = false;
      if (w.has) {
        if (!all_ok(mbar_wait(o_done(s), n_o & 1u, abort_flag))) return false;
        ++n_o;
        tc_fence_after();
      }
      if (w.skip) return true;  // the warp has no rows (its sibling of the other set neither, where they are joined)
      float scale = w.has ? 1.f : 0.f, other = 0.f;
      if (w.join) {  // both sets hold sums of the same rows: the second's go to the first
        if (s == 1) {
          if (!all_ok(mbar_wait(ex_empty(quad), (n_x & 1u) ^ 1u, abort_flag))) return false;
          stats[lane] = make_float2(w.m, w.l);
          __syncwarp();
          if (lane == 0) mbar_arrive(ex_full(quad));
          ++n_x;
          for (int c = 0; c < D / 16; ++c, ++n_x) {
            uint32_t r[16];
            tmem_ld16_issue(to + (uint32_t)(c * 16), r);
            tmem_ld_wait();
            if (!all_ok(mbar_wait(ex_empty(quad), (n_x & 1u) ^ 1u, abort_flag))) return false;
#pragma unroll
            for (int e = 0; e < 16; ++e) exchange[e * 32 + lane] = __uint_as_float(r[e]);
            __syncwarp();
            if (lane == 0) mbar_arrive(ex_full(quad));
          }
          return true;
        }
        if (!all_ok(mbar_wait(ex_full(quad), n_x & 1u, abort_flag))) return false;
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
      const float inv = w.whole ? (w.l == 0.f ? 0.f : 1.f / w.l) : 1.f;
      scale *= inv;
      other *= inv;
      // rows of this warp: their number, and where lane / 4 + 8 k lies
      const int rows = w.rows - quad * 32;
      T* dst[4];
      if (w.whole) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int r = quad * 32 + k * 8 + (lane >> 2), i = r / p.split.block_heads, h = r % p.split.block_heads;
          dst[k] = r < w.rows && h < w.heads ? static_cast<T*>(p.out) + (long long)(w.tok0 + i) * p.ldo + (long long)(w.head0 + h) * D + (lane & 3) * 8 : nullptr;
        }
      }
      const long long at = (long long)w.slot * kManyRows + w.row0 + row;
      float* part = p.parts.o + at * D;
      if (!w.whole && row < w.rows) p.parts.ml[at] = make_float2(w.m, w.l);
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
            if (!all_ok(mbar_wait(ex_full(quad), n_x & 1u, abort_flag))) return false;
#pragma unroll
            for (int e = 0; e < 16; ++e) r[h * 16 + e] = __float_as_uint(__uint_as_float(r[h * 16 + e]) + (other == 0.f ? 0.f : exchange[e * 32 + lane] * other));
            __syncwarp();
            if (lane == 0) mbar_arrive(ex_empty(quad));
          }
        }
        if (w.whole) {  // through shared memory: stores of 64 bytes a row
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

    Part t = part_at(p, prefix, lo, hi - lo);
    for (long long u = lo; u < hi && ok;) {
      const Sets sets = sets_of(p, t);
      const int set = sets.turns ? 0 : s, count = sets.count[s];
      const int set_row0 = set * set_tokens * p.split.block_heads;
      const int rows = min(set_tokens * p.split.block_heads, t.rows - set_row0);  // of the set
      const bool alive = quad * 32 < rows;                                        // whether the warp has any
      const int tok = set * set_tokens + row / p.split.block_heads;               // the row's token in the tile
      const int limit = p.split.causal && row < rows ? min(t.pos0 + tok + 1, t.keys) : t.keys;
      const int all_see = p.split.causal ? min(t.pos0 + set * set_tokens + quad * 32 / p.split.block_heads + 1, t.keys) : t.keys;
      const int any_sees = p.split.causal ? min(t.pos0 + set * set_tokens + min(quad * 32 + 31, rows - 1) / p.split.block_heads + 1, t.keys) : t.keys;
      float m_used = -INFINITY, l_run = 0.f;
      for (int j = 0; j < count; ++j, ++n_s) {
        const int k0 = ((int)t.first + (sets.turns ? 2 * j + s : j)) * kUnit;
        if (w.any && !flush()) { ok = false; break; }
        if (!all_ok(mbar_wait(s_full(s), n_s & 1u, abort_flag))) { ok = false; break; }
        if (alive) {
          tc_fence_after();
          // The scores stay in TMEM until P replaces them, and are taken 32 at a time, the next ones on their way meanwhile (all 128 at once, with P, would not
          // leave registers for the rest).
          const int live = max(0, min(any_sees - k0, kUnit) + 31) >> 5;  // chunks of 32 keys that some row of the warp sees
          const bool edge = k0 + kUnit > all_see;
          bool need_max = j == 0;
          float rs0, rs1;
          uint32_t pk[2][32];
          while (true) {
            if (need_max) {
              float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
              for (int c = 0; c < 4; ++c) {
                if (c >= live) break;
                uint32_t r[32];
                tmem_ld32_issue(ts + (uint32_t)(c * 32), r);
                tmem_ld_wait();
#pragma unroll
                for (int e = 0; e < 32; ++e)
                  if (!edge || k0 + c * 32 + e < limit) mx[e & 3] = fmaxf(mx[e & 3], __uint_as_float(r[e]));
              }
              const float m_new = fmaxf(m_used, fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * p.scale);
              if (j > 0) {  // O holds the tiles before: their products were complete before these scores were
                const float corr = m_new == -INFINITY ? 1.f : ex2(m_used - m_new);
                l_run *= corr;
#pragma unroll 1
                for (int c = 0; c < D / 32; ++c) {
                  uint32_t r[32];
                  tmem_ld32_issue(to + (uint32_t)(c * 32), r);
                  tmem_ld_wait();
#pragma unroll
                  for (int e = 0; e < 32; ++e) r[e] = __float_as_uint(__uint_as_float(r[e]) * corr);
                  tmem_st32(to + (uint32_t)(c * 32), r);
                }
              }
              m_used = m_new;
            }
            const float m_sub = m_used == -INFINITY ? 0.f : m_used;
            rs0 = rs1 = 0.f;
            uint32_t sr[2][32];
            tmem_ld32_issue(ts, sr[0]);
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              uint32_t* dst = &pk[c >> 1][(c & 1) * 16];
              uint32_t* r = sr[c & 1];
              tmem_ld_wait();
              if (c < 3) tmem_ld32_issue(ts + (uint32_t)((c + 1) * 32), sr[(c + 1) & 1]);
              if (c < live) {  // warp-uniform
                if (edge) {
#pragma unroll
                  for (int e = 0; e < 32; ++e)
                    if (k0 + c * 32 + e >= limit) r[e] = 0xff800000u;
                }
#pragma unroll
                for (int e = 0; e < 32; e += 4) {
                  const float a0 = ex2(fmaf(__uint_as_float(r[e]), p.scale, -m_sub)), a1 = ex2(fmaf(__uint_as_float(r[e + 1]), p.scale, -m_sub));
                  const float a2 = ex2(fmaf(__uint_as_float(r[e + 2]), p.scale, -m_sub)), a3 = ex2(fmaf(__uint_as_float(r[e + 3]), p.scale, -m_sub));
                  rs0 += a0 + a1;
                  rs1 += a2 + a3;
                  dst[e >> 1] = pack2<T>(a0, a1);
                  dst[(e >> 1) + 1] = pack2<T>(a2, a3);
                }
              } else {
#pragma unroll
                for (int e = 0; e < 16; ++e) dst[e] = 0u;
              }
            }
            if (need_max || !__any_sync(0xffffffffu, row < rows && !(rs0 + rs1 < kRowSumLimit))) break;
            need_max = true;  // a score far above the reference: once more, against its true maximum
          }
          l_run += rs0 + rs1;
          tmem_st32(ts, pk[0]);
          tmem_st32(ts + 32u, pk[1]);
          tmem_st_wait();
          tc_fence_before();
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(p_ready(s));
      }
      if (!ok) break;
      // what becomes of the tile. A set whose rows all lie before the stretch's keys has no sums, but says so to whoever joins the parts.
      const bool whole = t.take == t.units;
      if (w.any && !flush()) { ok = false; break; }  // (it had no tile of its own to do that in)
      w.any = count > 0 || !sets.turns || s == 0;
      w.has = count > 0;
      w.join = sets.turns && sets.count[1] > 0;
      w.whole = whole;
      w.skip = !alive;
      w.tok0 = t.tok0 + set * set_tokens;
      w.head0 = first_head(p, t.block);
      w.heads = heads_of(p, t.block);
      w.row0 = set_row0;
      w.rows = rows;
      w.slot = 2 * cta + (u == lo ? 0 : 1);
      w.m = m_used;
      w.l = l_run;
      if (!whole && t.first == 0) {
        cut_here = true;
        if (threadIdx.x == 128) p.parts.cuts[cta] = cut_of(p, t, u, total, cta, ctas, w.slot);
      }
      u += t.take;
      if (u < hi) next_part(p, t, hi - u);
    }
    if (ok && w.any) flush();
    if (!cut_here && threadIdx.x == 128) p.parts.cuts[cta].pieces = 0;
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
  constexpr bool bf16 = std::is_same<T, __nv_bfloat16>::value;
  const uint32_t box_rows = (uint32_t)std::min<int64_t>(kv->page_tokens, kUnit);
  const uint64_t pages = (uint64_t)kv->pages, rows = (uint64_t)(kv->kv_heads * kv->page_tokens), stride = (uint64_t)kv->page_stride;
  if (!encode_tile_map_3d(&tm_q, p.q, bf16, (uint64_t)p.s.tokens, (uint64_t)heads, D, (uint64_t)p.ldq, D, (uint32_t)(p.split.tile_tokens / 2),
                          (uint32_t)p.split.block_heads) ||
      !encode_tile_map_3d(&tm_k, kv->keys, bf16, pages, rows, D, stride, D, 1, box_rows) ||
      !encode_tile_map_3d(&tm_v, kv->values, bf16, pages, rows, D, stride, D, 1, box_rows))
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
