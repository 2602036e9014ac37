// Attention of the new tokens of ragged sequences over a pool of cache pages: out = softmax(scale * q . K^T) . V, token i of a sequence over the cached
// tokens 0 .. past + i (causal), or over all of them. `group` query heads share a key head.
//
// For few rows the call is bound by reading the keys and values once. All query rows of a tile (tokens x heads of one key head, 8, 16 or 32) go through the keys
// together; the line of all tiles' keys is dealt out to one CTA an SM in equal stretches (ttb_paged_rules.cuh), so that one long sequence and a ragged batch
// keep every SM's loads busy alike. In a CTA four warps load (units of 128 tokens, TMA boxes of a page, 128-byte swizzled, 192 KB on their way) and run on
// into the next tile; four take 32 keys each of every unit, with a softmax state of their own, and join the four states at the tile's end. Their products are
// mma.sync m16n8k16 with the keys as rows: a tile of eight queries fills it, where the tensor memory's 128 rows would be empty but for eight. Parts of a tile that was cut
// go to a workspace in fp32 and a second kernel joins them, in the order of the keys.
// A row's reference is the maximum of its first keys (fp16: 2^6 below it), raised (and its sums rescaled) only where four probabilities, a lane's, sum to 2^15 and more; the division by
// the sum makes the result independent of it. Scores, references and sums are fp32; the probabilities are rounded to the values' 16 bits, the only form in which the
// tensor cores take both (half a step of each, of both signs, against a sum of them that is not rounded).
// 64 requests of 20 to 4000 tokens, 12 heads of 64, fp16: 89 us, 5.1 TB/s (110 with one loading warp and 16-row tiles throughout). One token over 8000, 32 heads of
// 128 on 8 key heads, bf16: 15 us, of which 3 go by before the first load (the sequences, the part, its pages) and some 5 are the join and its launch.
#include <algorithm>
#include <climits>
#include <cmath>
#include <type_traits>

#include "ttb_paged_attention.cuh"
#include "ttb_sm100.cuh"

using namespace ttb;
using namespace ttb::paged;
using namespace ttb::sm100;

namespace {

constexpr int kWarps = 4, kLoaders = 4, kThreads = (kWarps + kLoaders) * 32;
constexpr int kBlock = 32;             // a warp's keys of a unit
constexpr int kParts = 4;              // worked out ahead
constexpr float kSumLimit = 32768.0f;  // a sum of probabilities below this keeps each of them inside fp16's and bf16's range
static_assert(kBlock * kWarps == kUnit, "the four warps share a unit");

__device__ __forceinline__ void ldsm_x4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
__device__ __forceinline__ void ldsm_x4_trans(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
template <typename T> __device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <> __device__ __forceinline__ void mma16816<__half>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <> __device__ __forceinline__ void mma16816<__nv_bfloat16>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// A tile of NT groups of eight query rows.
template <int D, int NT> struct Shape {
  static constexpr int kRows = 8 * NT;
  static constexpr int kHalves = D / 64;
  static constexpr int kHalfBytes = kUnit * 128;
  static constexpr int kTile = kHalves * kHalfBytes;  // 128 keys, or 128 values
  static constexpr int kStages = D == 128 ? 3 : 6;
  static constexpr int kQHalf = kRows * 128;
  static constexpr int kQ = kStages * 2 * kTile;
  static constexpr int kPitch = D + 4;                       // floats between rows of the states that are joined (no bank conflicts)
  static constexpr int kJoin = kQ + 2 * kHalves * kQHalf;  // float [kWarps][8][kPitch]; before the first part, the sequences' places
  static constexpr int kStats = kJoin + kWarps * 8 * kPitch * 4;   // float2 [2][kWarps][kRows]
  static constexpr int kScratch = kStats + 2 * kWarps * kRows * 8;
  static constexpr int kWorks = kScratch + kThreads / 32 * 8;
  static constexpr int kBars = kWorks + kParts * (int)sizeof(Work);
  static constexpr int kNumBars = 2 * kStages + 5 + 2 * kParts;
  static constexpr int kBytes = kBars + kNumBars * 8 + 16;
  static_assert(kWarps * 8 * kPitch * 4 >= (kMaxSequences + 1) * 8, "the sequences' places");
};

// An 8 x 8 matrix of 16-bit pairs, transposed across the warp.
__device__ __forceinline__ uint32_t transposed(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ float column_max(float v) {  // over the lanes that hold the same column
#pragma unroll
  for (int o = 4; o < 32; o <<= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

template <typename T, int D, int NT>
__global__ void __launch_bounds__(kThreads, 1)
paged_rows_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v, const Params p) {
  using S = Shape<D, NT>;
  extern __shared__ __align__(1024) uint8_t smem[];
  const uint32_t base = smem_u32(smem);
  float* join = reinterpret_cast<float*>(smem + S::kJoin);
  float2* stats = reinterpret_cast<float2*>(smem + S::kStats);
  Work* works = reinterpret_cast<Work*>(smem + S::kWorks);
  const uint32_t bar0 = smem_u32(smem + S::kBars);
  auto bar = [&](int k) { return bar0 + 8u * k; };
  auto full = [&](uint32_t g) { return bar((int)(g % S::kStages)); };
  auto empty = [&](uint32_t g) { return bar(S::kStages + (int)(g % S::kStages)); };
  auto phase = [&](uint32_t g) { return (g / S::kStages) & 1u; };
  auto q_full = [&](uint32_t n) { return bar(2 * S::kStages + (int)(n & 1)); };
  auto q_empty = [&](uint32_t n) { return bar(2 * S::kStages + 2 + (int)(n & 1)); };
  auto q_phase = [&](uint32_t n) { return (n >> 1) & 1u; };
  auto q_at = [&](uint32_t n) { return base + S::kQ + (n & 1) * S::kHalves * S::kQHalf; };
  auto part_full = [&](uint32_t n) { return bar(2 * S::kStages + 5 + (int)(n % kParts)); };
  auto part_empty = [&](uint32_t n) { return bar(2 * S::kStages + 5 + kParts + (int)(n % kParts)); };
  auto part_phase = [&](uint32_t n) { return (n / kParts) & 1u; };
  const uint32_t meet = bar(2 * S::kStages + 4);  // the computing warps'
  auto keys_at = [&](uint32_t g) { return base + (g % S::kStages) * 2 * S::kTile; };
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + S::kBars + S::kNumBars * 8);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;

  pdl_trigger();
  if (tid == 0) {
    for (int i = 0; i < S::kStages; ++i) {
      mbar_init(full(i), kLoaders);
      mbar_init(empty(i), kWarps);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(bar(2 * S::kStages + i), 1);
      mbar_init(bar(2 * S::kStages + 2 + i), kWarps);
    }
    for (int i = 0; i < kParts; ++i) {
      mbar_init(part_full(i), 1);
      mbar_init(part_empty(i), kWarps + kLoaders - 1);
    }
    mbar_init(meet, kWarps);
    *abort_flag = 0;
    prefetch_tensormap(&tm_q);
    prefetch_tensormap(&tm_k);
    prefetch_tensormap(&tm_v);
    mbar_init_fence();
  }
  pdl_wait();
  long long* prefix = reinterpret_cast<long long*>(smem + S::kJoin);
  const long long total = line_up(p, prefix, reinterpret_cast<long long*>(smem + S::kScratch), kThreads);
  const int ctas = ctas_of(total, (int)gridDim.x, 1), cta = blockIdx.x;
  if (cta >= ctas) {
    if (tid == 0) p.parts.cuts[cta].pieces = 0;
    return;
  }
  // The n-th part, for every warp but the one that works them out. False: no part, there are no more or something gave up.
  auto take_part = [&](uint32_t n, Work* w) {
    if (!__all_sync(0xffffffffu, mbar_wait(part_full(n), part_phase(n), abort_flag))) return false;
    *w = works[n % kParts];
    __syncwarp();
    if (lane == 0) mbar_arrive(part_empty(n));
    return w->units >= 0;
  };

  if (warp >= kWarps) {
    // ---- loads: a lane for each box (a page, or 128 keys) of keys or values and half of a head, every fourth of them a warp's: a copy takes its thread some 60
    // cycles to issue, one lane after the other. A lane's pages are looked up two units ahead. The first of the warps works the parts out.
    const int loader = warp - kWarps;
    const int page_tokens = 1 << p.s.page_shift, box_rows = min(page_tokens, kUnit);
    const int at = lane * kLoaders + loader, box = at / (2 * S::kHalves), which = at / S::kHalves & 1, half = at % S::kHalves;
    const long long lo = first_unit(total, ctas, cta), hi = first_unit(total, ctas, cta + 1);
    uint32_t g = 0, n = 0;
    bool ok = true, cut_here = false;
    long long u = lo;
    Part t = {};
    auto publish = [&](Work* w) {
      w->units = -1;
      if (n > 0) u += t.take;
      if (u < hi) {
        if (n > 0) next_part(p, t, hi - u);
        else t = part_at(p, prefix, lo, hi - lo);
        *w = work_of(p, t, 2 * cta + (u == lo ? 0 : 1));
        if (w->slot >= 0 && t.first == 0) {
          cut_here = true;
          if (lane == 0) p.parts.cuts[cta] = cut_of(p, t, u, total, cta, ctas, w->slot);
        }
      }
      ok = __all_sync(0xffffffffu, ok && mbar_wait(part_empty(n), part_phase(n) ^ 1u, abort_flag));
      if (ok && lane == 0) works[n % kParts] = *w;
      __syncwarp();
      if (ok && lane == 0) mbar_arrive(part_full(n));
      return ok && w->units >= 0;
    };
    auto page_at = [&](const Work& w, int i) {  // (looked at when it is needed)
      const int key = (w.first + i) * kUnit + box * box_rows;
      return key < w.keys && box * box_rows < kUnit ? p.s.table[w.b * p.s.table_stride + (key >> p.s.page_shift)] : 0;
    };
    auto next = [&](Work* w) { return loader == 0 ? publish(w) : take_part(n, w); };  // the n-th part
    Work w, w2;
    bool more = next(&w);
    int page = more ? page_at(w, 0) : 0, page2 = more ? page_at(w, 1) : 0;  // the lane's, of this unit and the next
    while (more) {
      if (loader == 0) {
        ok = __all_sync(0xffffffffu, mbar_wait(q_empty(n), q_phase(n) ^ 1u, abort_flag));
        if (ok && lane == 0) {
          mbar_expect_tx(q_full(n), (uint32_t)(p.split.tile_tokens * p.split.block_heads * D * 2));
          for (int h = 0; h < S::kHalves; ++h) tma_load_3d(q_at(n) + h * S::kQHalf, &tm_q, q_full(n), h * 64, w.head0, w.tok0);
        }
      }
      ++n;
      for (int i = 0; i < w.units && ok; ++i, ++g) {
        const int key = (w.first + i) * kUnit + box * box_rows;
        int mine = -1;
        if (key < w.keys && box * box_rows < kUnit) {
          mine = page;
          if (mine < 0 || mine >= p.s.pages) {
            bad_index(p.s.status);
            mine = 0;
          }
        }
        ok = __all_sync(0xffffffffu, mbar_wait(empty(g), phase(g) ^ 1u, abort_flag));
        if (!ok) break;
        const int boxes = __popc(__ballot_sync(0xffffffffu, mine >= 0));
        if (lane == 0) mbar_expect_tx(full(g), (uint32_t)(boxes * box_rows * 128));
        __syncwarp();
        if (mine >= 0)
          tma_load_3d(keys_at(g) + which * S::kTile + half * S::kHalfBytes + box * box_rows * 128, which ? &tm_v : &tm_k, full(g), half * 64,
                      w.key_row + (key & (page_tokens - 1)), mine);
        if (i == 0) more = next(&w2);
        page = i + 1 < w.units ? page2 : more ? page_at(w2, 0) : 0;
        page2 = i + 2 < w.units ? page_at(w, i + 2) : more ? page_at(w2, i + 2 - w.units) : 0;
      }
      if (!ok) break;
      if (w.units == 0) {  // a part without keys (more tokens than the table lists)
        more = next(&w2);
        page = more ? page_at(w2, 0) : 0;
        page2 = more ? page_at(w2, 1) : 0;
      }
      w = w2;
    }
    if (loader == 0 && !cut_here && lane == 0) p.parts.cuts[cta].pieces = 0;
    if (*abort_flag) {  // copies in flight land before shared memory is given back
      const long long t0 = clock64();
      while (clock64() - t0 < 4000000LL) {
      }
    }
    return;
  }

  // ---- computation: warp w takes keys 32 w to 32 w + 31 of every unit. Keys are the rows of the products and queries their columns, so that a tile of eight query rows
  // leaves none of the product empty: S^T = K Q^T, O^T = V^T P^T, with the probabilities transposed in between.
  bool ok = true;
  uint32_t g = 0, n_meet = 0;
  // A barrier of the four warps that gives up like every wait.
  auto together = [&]() {
    __syncwarp();
    if (lane == 0) mbar_arrive(meet);
    ok = __all_sync(0xffffffffu, mbar_wait(meet, n_meet++ & 1u, abort_flag));
    return ok;
  };
  Work t;
  for (uint32_t n = 0; take_part(n, &t); ++n) {
    constexpr bool kQInRegisters = NT <= 2;
    uint32_t qf[kQInRegisters ? D / 32 : 1][NT][4];
    auto load_q = [&](int j, uint32_t (&q)[4], int nt) {  // columns 32 j to 32 j + 31 of eight queries: two products' operands
      const int row = nt * 8 + (lane & 7), c = (j & 1) * 4 + (lane >> 3);
      ldsm_x4(q, q_at(n) + (j >> 1) * S::kQHalf + row * 128 + ((c ^ (row & 7)) << 4));
    };
    ok = __all_sync(0xffffffffu, mbar_wait(q_full(n), q_phase(n), abort_flag));
    if (!ok) break;
    if constexpr (kQInRegisters) {
#pragma unroll
      for (int j = 0; j < D / 32; ++j)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) load_q(j, qf[j][nt], nt);
      __syncwarp();
      if (lane == 0) mbar_arrive(q_empty(n));
    }
    const int all_see = p.split.causal ? min(t.pos0 + 1, t.keys) : t.keys;
    // this lane's queries are columns 2 (lane % 4) and the next of every group: their reference, the sums of its keys, and of their outputs rows lane / 4 and + 8
    float m[NT][2], l[NT][2], o[D / 16][NT][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      m[nt][0] = m[nt][1] = -INFINITY;
      l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
      for (int d = 0; d < D / 16; ++d)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[d][nt][e] = 0.f;
    }
    bool fresh = true;
    for (int i = 0; i < t.units; ++i, ++g) {
      ok = __all_sync(0xffffffffu, mbar_wait(full(g), phase(g), abort_flag));
      if (!ok) break;
      const int k0 = (t.first + i) * kUnit + warp * kBlock;
      if (k0 < t.keys) {
        const uint32_t kt = keys_at(g) + warp * kBlock * 128, vt = kt + S::kTile;
        if (k0 + kBlock > t.keys) {
          // rows behind the last key: what the page or the ring happens to hold there, which a probability of zero does not undo where it is not finite
#pragma unroll 1
          for (int c = lane; c < (kBlock - (t.keys - k0)) * S::kHalves * 8; c += 32) {
            const int r = (t.keys - k0) + c / (S::kHalves * 8), col = c % (S::kHalves * 8);
            asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(vt + (col >> 3) * S::kHalfBytes + r * 128 + (col & 7) * 16), "r"(0) : "memory");
          }
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // before the next load into these rows
          __syncwarp();
        }
        float s[2][NT][4];
#pragma unroll
        for (int mt = 0; mt < 2; ++mt)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 4; ++e) s[mt][nt][e] = 0.f;
#pragma unroll
        for (int j = 0; j < D / 32; ++j) {
          if constexpr (!kQInRegisters) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) load_q(j, qf[0][nt], nt);
          }
#pragma unroll
          for (int k = 0; k < 2; ++k) {
#pragma unroll
            for (int mt = 0; mt < 2; ++mt) {  // 16 keys x 16 columns
              const int row = mt * 16 + (lane & 15), c = (j & 1) * 4 + k * 2 + (lane >> 4);
              uint32_t a[4];
              ldsm_x4(a, kt + (j >> 1) * S::kHalfBytes + row * 128 + ((c ^ (row & 7)) << 4));
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) {
                const uint32_t (&q)[4] = qf[kQInRegisters ? j : 0][nt];
                mma16816<T>(s[mt][nt], a, q[2 * k], q[2 * k + 1]);
              }
            }
          }
        }
        if (k0 + kBlock > all_see) {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int q = 0; q < 2; ++q) {
              const int row = nt * 8 + (lane & 3) * 2 + q;
              const int limit = (p.split.causal && row < t.rows ? min(t.pos0 + row / p.split.block_heads + 1, t.keys) : t.keys) - k0 - (lane >> 2);
#pragma unroll
              for (int x = 0; x < 4; ++x)
                if (x * 8 >= limit) s[x >> 1][nt][(x & 1) * 2 + q] = -INFINITY;
            }
        }
        // A row's reference is the maximum of its first keys (fp16: 2^6 below it); it is raised (and the sums rescaled) only where a lane's four probabilities sum up to 2^15 and
        // more: the division by the sum makes the result independent of it.
        uint32_t pf[2][NT][2];
        while (true) {
          if (fresh) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int q = 0; q < 2; ++q) {
                const float top = column_max(fmaxf(fmaxf(s[0][nt][q], s[0][nt][2 + q]), fmaxf(s[1][nt][q], s[1][nt][2 + q]))) * p.scale - kBelow<T>;
                const float m_new = fmaxf(m[nt][q], top), corr = m_new == -INFINITY ? 1.f : ex2(m[nt][q] - m_new);
                m[nt][q] = m_new;
                l[nt][q] *= corr;
#pragma unroll
                for (int d = 0; d < D / 16; ++d) {
                  o[d][nt][q] *= corr;
                  o[d][nt][2 + q] *= corr;
                }
              }
          }
          bool far = false;
          float sum[NT][2];
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            const float m0 = m[nt][0] == -INFINITY ? 0.f : m[nt][0], m1 = m[nt][1] == -INFINITY ? 0.f : m[nt][1];
            sum[nt][0] = sum[nt][1] = 0.f;
#pragma unroll
            for (int mt = 0; mt < 2; ++mt)
#pragma unroll
              for (int r = 0; r < 2; ++r) {
                const float a = ex2(fmaf(s[mt][nt][2 * r], p.scale, -m0)), b = ex2(fmaf(s[mt][nt][2 * r + 1], p.scale, -m1));
                sum[nt][0] += a;
                sum[nt][1] += b;
                pf[mt][nt][r] = pack2<T>(a, b);
              }
            const int row = nt * 8 + (lane & 3) * 2;
            far = far || (row < t.rows && !(sum[nt][0] < kSumLimit)) || (row + 1 < t.rows && !(sum[nt][1] < kSumLimit));
          }
          if (fresh || !__any_sync(0xffffffffu, far)) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              l[nt][0] += sum[nt][0];
              l[nt][1] += sum[nt][1];
            }
            break;
          }
          fresh = true;
        }
        fresh = false;
#pragma unroll
        for (int mt = 0; mt < 2; ++mt) {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int r = 0; r < 2; ++r) pf[mt][nt][r] = transposed(pf[mt][nt][r]);
#pragma unroll
          for (int d = 0; d < D / 16; ++d) {  // 16 columns of the values x 16 keys
            const int row = mt * 16 + (lane & 7) + ((lane >> 4) << 3), c = (d & 3) * 2 + ((lane >> 3) & 1);
            uint32_t a[4];
            ldsm_x4_trans(a, vt + (d >> 2) * S::kHalfBytes + row * 128 + ((c ^ (row & 7)) << 4));
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) mma16816<T>(o[d][nt], a, pf[mt][nt][0], pf[mt][nt][1]);
          }
        }
        __syncwarp();
      }
      if (lane == 0) mbar_arrive(empty(g));
    }
    if constexpr (!kQInRegisters) {
      __syncwarp();
      if (lane == 0) mbar_arrive(q_empty(n));
    }
    // ---- the four warps' states become one, eight rows at a time
    float2* mine = stats + (n & 1) * kWarps * S::kRows;  // (the part before's may still be read)
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int q = 0; q < 2; ++q) {
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) l[nt][q] += __shfl_xor_sync(0xffffffffu, l[nt][q], x);
        if (lane < 4) mine[warp * S::kRows + nt * 8 + lane * 2 + q] = make_float2(m[nt][q], l[nt][q]);
      }
    if (!ok) break;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      if (nt * 8 >= t.rows) break;
      if (!together()) break;  // the rows before have been read
#pragma unroll
      for (int d = 0; d < D / 16; ++d)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int q = (lane & 3) * 2 + (e & 1);
          if (nt * 8 + q < t.rows) join[(warp * 8 + q) * S::kPitch + d * 16 + (lane >> 2) + (e >> 1) * 8] = o[d][nt][e];
        }
      if (!together()) break;
      const int tasks = min(8, t.rows - nt * 8) * (D / 4);
      for (int x = tid; x < tasks; x += kWarps * 32) {
        const int q = x / (D / 4), d = x % (D / 4) * 4, row = nt * 8 + q, i = row / p.split.block_heads, h = row % p.split.block_heads;
        if (h >= t.heads) continue;
        float M = -INFINITY;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) M = fmaxf(M, mine[w * S::kRows + row].x);
        const float sub = M == -INFINITY ? 0.f : M;
        float L = 0.f, v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
          const float2 ml = mine[w * S::kRows + row];
          const float f = ex2(ml.x - sub);
          const float4 a = *reinterpret_cast<const float4*>(join + (w * 8 + q) * S::kPitch + d);
          L = fmaf(ml.y, f, L);
          v[0] = fmaf(a.x, f, v[0]);
          v[1] = fmaf(a.y, f, v[1]);
          v[2] = fmaf(a.z, f, v[2]);
          v[3] = fmaf(a.w, f, v[3]);
        }
        if (t.slot < 0) {
          const float inv = L == 0.f ? 0.f : 1.f / L;
          uint2 y;
          y.x = pack2<T>(v[0] * inv, v[1] * inv);
          y.y = pack2<T>(v[2] * inv, v[3] * inv);
          *reinterpret_cast<uint2*>(static_cast<T*>(p.out) + (long long)(t.tok0 + i) * p.ldo + (long long)(t.head0 + h) * D + d) = y;
        } else {
          const long long to = (long long)t.slot * S::kRows + row;
          *reinterpret_cast<float4*>(p.parts.o + to * D + d) = make_float4(v[0], v[1], v[2], v[3]);
          if (d == 0) p.parts.ml[to] = make_float2(M, L);
        }
      }
    }
    if (!ok) break;
  }
  if ((!ok || *abort_flag) && lane == 0) atomicExch(p.s.status, (int)TTB_ERR_DEVICE_WAIT);
}

// Joins the parts of the tiles that were cut, of both kernels: a block (and its neighbours along y) for each of their CTAs, R rows a warp, parts in the
// order of the keys.
struct JoinParams {
  Parts parts[2];
  int rows[2];
  void* out;
  long long ldo;
};
template <typename T, int D, int R>
__global__ void __launch_bounds__(128)
paged_join_kernel(const JoinParams p) {
  pdl_trigger();
  pdl_wait();
  const int which = blockIdx.z, lane = threadIdx.x & 31;
  const Parts parts = which ? p.parts[1] : p.parts[0];
  const int stride = which ? p.rows[1] : p.rows[0];
  const Cut c = parts.cuts[blockIdx.x];
  if (c.pieces == 0) return;
  constexpr int V = D / 32, E = 8 / R;  // sums of eight rows and parts are on their way
  auto slot = [&](int k) { return (long long)(k == 0 ? c.slot : 2 * ((int)blockIdx.x + k)) * stride; };
  for (int row0 = (blockIdx.y * 4 + (threadIdx.x >> 5)) * R; row0 < c.rows; row0 += gridDim.y * 4 * R) {
    float M[R], L[R], o[R][V];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      M[r] = -INFINITY;
      L[r] = 0.f;
#pragma unroll
      for (int v = 0; v < V; ++v) o[r][v] = 0.f;
    }
    for (int k = lane; k < c.pieces; k += 32) {
      const long long at = slot(k) + row0;
#pragma unroll
      for (int r = 0; r < R; ++r)
        if (row0 + r < c.rows) M[r] = fmaxf(M[r], parts.ml[at + r].x);
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      M[r] = warp_max(M[r]);
      M[r] = M[r] == -INFINITY ? 0.f : M[r];
    }
    for (int k0 = 0; k0 < c.pieces; k0 += 32) {  // a lane has a part's weights
      float mine[R];
#pragma unroll
      for (int r = 0; r < R; ++r) {
        mine[r] = 0.f;
        if (k0 + lane < c.pieces && row0 + r < c.rows) {
          const float2 ml = parts.ml[slot(k0 + lane) + row0 + r];
          mine[r] = ex2(ml.x - M[r]);
          L[r] = fmaf(ml.y, mine[r], L[r]);
        }
      }
      const int n = min(32, c.pieces - k0);
      for (int k1 = 0; k1 < n; k1 += E) {
        float x[E][R][V];
#pragma unroll
        for (int e = 0; e < E; ++e)
          if (k1 + e < n) {
            const float* src = parts.o + (slot(k0 + k1 + e) + row0) * D + lane;
#pragma unroll
            for (int r = 0; r < R; ++r)
              if (row0 + r < c.rows) {
#pragma unroll
                for (int v = 0; v < V; ++v) x[e][r][v] = src[r * D + v * 32];
              }
          }
#pragma unroll
        for (int e = 0; e < E; ++e) {
          if (k1 + e >= n) break;
#pragma unroll
          for (int r = 0; r < R; ++r) {
            const float w = __shfl_sync(0xffffffffu, mine[r], k1 + e);  // zero for a part without a key for this row, which has no sums
#pragma unroll
            for (int v = 0; v < V; ++v) o[r][v] = w == 0.f ? o[r][v] : fmaf(x[e][r][v], w, o[r][v]);
          }
        }
      }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int row = row0 + r, i = row / c.block_heads, g = row % c.block_heads;
      const float l = warp_sum(L[r]);
      if (row >= c.rows || g >= c.heads) continue;
      const float inv = l == 0.f ? 0.f : 1.f / l;
      T* dst = static_cast<T*>(p.out) + (long long)(c.tok0 + i) * p.ldo + (long long)(c.head0 + g) * D;
#pragma unroll
      for (int v = 0; v < V; ++v) dst[v * 32 + lane] = from_f<T>(o[r][v] * inv);
    }
  }
}

template <typename T, int D, int NT>
int launch_rows(ttb_ctx* ctx, const ttb_paged_kv* kv, int64_t heads, const Params& p) {
  using S = Shape<D, NT>;
  CUtensorMap tm_q, tm_k, tm_v;
  if (!encode_maps(kv, std::is_same<T, __nv_bfloat16>::value, heads, p, p.split.tile_tokens, &tm_q, &tm_k, &tm_v))
    return fail(ctx, TTB_ERR_CUDA, "paged_attention: a tensor map was refused");
  static bool configured[64] = {};
  const int dev = ctx->device < 64 ? ctx->device : 63;
  if (!configured[dev]) {
    TTB_CUDA(ctx, cudaFuncSetAttribute(paged_rows_kernel<T, D, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kBytes));
    configured[dev] = true;
  }
  launch_pdl(paged_rows_kernel<T, D, NT>, dim3((unsigned)ctx->sm_count), dim3(kThreads), S::kBytes, ctx->stream, tm_q, tm_k, tm_v, p);
  return launched(ctx, "paged_attention");
}

template <typename T, int D>
int launch_all(ttb_ctx* ctx, int dtype, const ttb_paged_kv* kv, int64_t heads, Params& p) {
  // Which kernels, and the rows of a tile of the one for few. The host knows the sum of the new tokens only. With no more tokens than sequences, tiles of a token's rows (up to 32)
  // take all of them, a sequence of several tokens several tiles. Otherwise tiles of an average sequence's rows, up to 32 (24 with heads of
  // 128), and the sequences that have more go to the kernel for many; where the average has more, tiles of 16. Sequences without new tokens count: a table of many idle rows looks
  // like one of single tokens, and a chunk among them is walked in small tiles (right, and slower). Rows of a sequence, us in tiles of 32 here and on the kernel for
  // many, with cold caches: 64 requests of 3 tokens over 500 to 4000, 24 rows, heads of 64 76 and 88, of 128 172 and 182; 100 of 8 over 100 to 1000, 32 rows, 68 and 70, 148 and
  // 130; 16 of 3 to 6 over up to 16000, 24 to 48 rows, 128: 171 and 144 to 151.
  const int64_t tokens = p.s.tokens, B = kv->B, each = (tokens + B - 1) / B * p.group;
  const int64_t need = std::max<int64_t>(p.group, each <= (D == 64 ? 32 : 24) ? each : std::min<int64_t>(each, 16));
  const int groups = need <= 8 ? 1 : need <= 16 ? 2 : 4, few = 8 * groups / p.group;
  const bool rows_only = few > 0 && tokens <= (B == 1 ? few : B), many_only = few == 0 || (B == 1 && !rows_only);
  const int ctas = ctx->sm_count;
  size_t at = 0, o[2], ml[2], cuts[2];
  const int rows[2] = {8 * groups, kManyRows};
  const bool used[2] = {!many_only, !rows_only};
  auto take = [&](size_t bytes) { const size_t x = at; at = (at + bytes + 255) & ~(size_t)255; return x; };
  for (int i = 0; i < 2; ++i) {
    if (!used[i]) continue;
    o[i] = take((size_t)2 * ctas * rows[i] * D * 4);
    ml[i] = take((size_t)2 * ctas * rows[i] * 8);
    cuts[i] = take((size_t)ctas * sizeof(Cut));
  }
  void* ws = nullptr;
  int st = ttb_alloc(ctx, at, "paged_attention/parts", &ws);
  if (st) return st;
  JoinParams j = {};
  j.out = p.out;
  j.ldo = p.ldo;
  int n = 0;
  for (int i = 0; i < 2 && !st; ++i) {
    if (!used[i]) continue;
    char* base = static_cast<char*>(ws);
    p.parts = Parts{reinterpret_cast<float*>(base + o[i]), reinterpret_cast<float2*>(base + ml[i]), reinterpret_cast<Cut*>(base + cuts[i])};
    p.low = i == 0 || many_only ? 0 : few + 1;
    p.high = i == 1 || rows_only ? INT_MAX : few;
    j.parts[n] = p.parts;
    j.rows[n++] = rows[i];
    if (i == 0) {
      p.split = split_of((int)heads, (int)kv->kv_heads, rows[0], 1, kUnit, p.split.causal, 0);
      st = groups == 1 ? launch_rows<T, D, 1>(ctx, kv, heads, p) : groups == 2 ? launch_rows<T, D, 2>(ctx, kv, heads, p) : launch_rows<T, D, 4>(ctx, kv, heads, p);
    } else {
      // A tile of one set's rows takes two units of keys in the time of one of both sets' with heads of 64 (six prompts of 200 to 2000 tokens: 130 us, and 135 with each
      // counted as one). With heads of 128 it waits for values, whose ring is two tiles long, and a unit takes more than half (a chunk of 4000 tokens over
      // 12000: 1040 us in pairs, 900 alone).
      p.split = split_of((int)heads, (int)kv->kv_heads, kManyRows / 2, 2, kUnit, p.split.causal, D == 64 ? 1 : 0);
      st = paged_tc_launch(ctx, dtype, kv, heads, p);
    }
  }
  if (!st) {
    if (used[1]) launch_pdl(paged_join_kernel<T, D, 4>, dim3((unsigned)ctas, kManyRows / 16, (unsigned)n), dim3(128), 0, ctx->stream, j);
    else launch_pdl(paged_join_kernel<T, D, 1>, dim3((unsigned)ctas, rows[0] / 4, (unsigned)n), dim3(128), 0, ctx->stream, j);
    st = launched(ctx, "paged_attention_join");
  }
  const int f = ttb_free(ctx, ws, "paged_attention/parts");
  return st ? st : f;
}

}  // namespace

extern "C" int ttb_paged_attention(ttb_ctx* ctx, int dtype, const ttb_paged_kv* kv, const void* q, int64_t ldq, int64_t tokens, int64_t heads, int causal,
                                   float scale, void* out, int64_t ldo) {
  return ttb_paged_attention_room(ctx, dtype, kv, q, ldq, tokens, heads, causal, scale, out, ldo, nullptr);
}

extern "C" int ttb_paged_attention_room(ttb_ctx* ctx, int dtype, const ttb_paged_kv* kv, const void* q, int64_t ldq, int64_t tokens, int64_t heads, int causal,
                                        float scale, void* out, int64_t ldo, const int32_t* room) {
  if (!ctx) return TTB_ERR_INVALID;
  Params p = {};
  const int bad = check_kv(ctx, "paged_attention", dtype, kv, tokens, &p.s);
  if (bad) return bad;
  TTB_REQUIRE(ctx, heads > 0 && heads % kv->kv_heads == 0 && heads <= 65535, "paged_attention: the query heads must be a multiple of the key heads");
  TTB_REQUIRE(ctx, scale > 0.f && scale < INFINITY, "paged_attention: the scale must be positive");
  if (tokens == 0 || kv->B == 0) return TTB_OK;
  TTB_REQUIRE(ctx, q && out, "paged_attention: null pointer");
  TTB_REQUIRE(ctx, ldq >= heads * kv->d && ldo >= heads * kv->d && ldq % 8 == 0 && ldo % 8 == 0 && ldq < (1ll << 31) && ldo < (1ll << 31),
              "paged_attention: rows of q and out are at least heads * d elements apart, a multiple of 8");
  TTB_REQUIRE(ctx, ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out)) & 15) == 0, "paged_attention: q and out must be 16-byte aligned");
  DeviceGuard g(ctx->device);
  p.q = q;
  p.out = out;
  p.ldq = ldq;
  p.ldo = ldo;
  p.group = (int)(heads / kv->kv_heads);
  p.scale = scale * kLog2e;
  p.room = room;
  p.split.causal = causal != 0;
  if (kv->d == 64) return dtype == TTB_F16 ? launch_all<__half, 64>(ctx, dtype, kv, heads, p) : launch_all<__nv_bfloat16, 64>(ctx, dtype, kv, heads, p);
  return dtype == TTB_F16 ? launch_all<__half, 128>(ctx, dtype, kv, heads, p) : launch_all<__nv_bfloat16, 128>(ctx, dtype, kv, heads, p);
}
