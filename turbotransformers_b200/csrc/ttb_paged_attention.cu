// Attention of the new tokens of ragged sequences over a pool of cache pages: out = softmax(scale * q . K^T) . V, token i of a sequence over the cached
// tokens 0 .. past + i (causal), or over all of them. `group` query heads share a key head.
//
// For few rows the call is bound by reading the keys and values once. All query rows of a tile (tokens x heads of one key head, up to 16) go through the keys
// together; the line of all tiles' keys is dealt out to one CTA an SM in equal stretches (ttb_paged_rules.cuh), so that one long sequence and a ragged batch
// keep every SM's loads busy alike. In a CTA one warp loads (units of 128 tokens, TMA boxes of a page, 128-byte swizzled, 192 KB on their way) and runs on
// into the next tile; four warps take 32 keys each of every unit, with a softmax state of their own (running maximum and sum in fp32, mma.sync m16n8k16), and join
// the four states at the tile's end. Parts of a tile that was cut go to a workspace in fp32 and a second kernel joins them, in the order of the keys.
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
constexpr int kRows = kFewRows;
constexpr int kBlock = 32;  // a warp's keys of a unit
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

template <int D> struct Shape {
  static constexpr int kHalves = D / 64;
  static constexpr int kHalfBytes = kUnit * 128;
  static constexpr int kTile = kHalves * kHalfBytes;  // 128 keys, or 128 values
  static constexpr int kStages = D == 128 ? 3 : 6;
  static constexpr int kQHalf = kRows * 128;
  static constexpr int kQ = kStages * 2 * kTile;       // two tiles' queries
  static constexpr int kJoin = kQ + 2 * kHalves * kQHalf;  // float [2][kRows][D]
  static constexpr int kPrefix = kJoin + 2 * kRows * D * 4;
  static constexpr int kScratch = kPrefix + (kMaxSequences + 1) * 8;
  static constexpr int kStats = kScratch + kThreads / 32 * 8;
  static constexpr int kBars = kStats + kWarps * kRows * 8;
  static constexpr int kNumBars = 2 * kStages + 4;
  static constexpr int kBytes = kBars + kNumBars * 8 + 16;
};

__device__ __forceinline__ void warps_sync() { asm volatile("bar.sync 1, 128;" ::: "memory"); }  // of the four computing warps
__device__ __forceinline__ bool warps_all(bool mine) {
  int all;
  asm volatile(
      "{\n"
      ".reg .pred p, q;\n"
      "setp.ne.b32 p, %1, 0;\n"
      "bar.red.and.pred q, 1, 128, p;\n"
      "selp.u32 %0, 1, 0, q;\n"
      "}\n"
      : "=r"(all)
      : "r"((int)mine)
      : "memory");
  return all != 0;
}

template <typename T, int D>
__global__ void __launch_bounds__(kThreads, 1)
paged_rows_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v, const Params p) {
  using S = Shape<D>;
  extern __shared__ __align__(1024) uint8_t smem[];
  const uint32_t base = smem_u32(smem);
  long long* prefix = reinterpret_cast<long long*>(smem + S::kPrefix);
  float* join = reinterpret_cast<float*>(smem + S::kJoin);
  float2* stats = reinterpret_cast<float2*>(smem + S::kStats);  // [kWarps][kRows]
  const uint32_t bar0 = smem_u32(smem + S::kBars);
  auto full = [&](uint32_t g) { return bar0 + 8 * (g % S::kStages); };
  auto empty = [&](uint32_t g) { return bar0 + 8 * (S::kStages + g % S::kStages); };
  auto phase = [&](uint32_t g) { return (g / S::kStages) & 1u; };
  auto q_full = [&](uint32_t n) { return bar0 + 8 * (2 * S::kStages + (n & 1)); };
  auto q_empty = [&](uint32_t n) { return bar0 + 8 * (2 * S::kStages + 2 + (n & 1)); };
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
      mbar_init(q_full(i), 1);
      mbar_init(q_empty(i), kWarps);
    }
    *abort_flag = 0;
    prefetch_tensormap(&tm_q);
    prefetch_tensormap(&tm_k);
    prefetch_tensormap(&tm_v);
    mbar_init_fence();
  }
  pdl_wait();
  const long long total = line_up(p, prefix, reinterpret_cast<long long*>(smem + S::kScratch), kThreads);
  const int ctas = ctas_of(total, (int)gridDim.x, 1), cta = blockIdx.x;
  if (cta >= ctas) {
    if (tid == 0) p.parts.cuts[cta].pieces = 0;
    return;
  }
  const long long lo = first_unit(total, ctas, cta), hi = first_unit(total, ctas, cta + 1);
  Part t = part_at(p, prefix, lo, hi - lo);

  if (warp >= kWarps) {
    // ---- loads: a lane for each box (a page, or 128 keys) of keys or values and half of a head, every fourth of them a warp's: a copy takes its thread some 60
    // cycles to issue, one lane after the other. The pages of a unit are looked up while the one before is loaded.
    const int loader = warp - kWarps;
    const int page_tokens = 1 << p.s.page_shift, box_rows = min(page_tokens, kUnit);
    const int at = lane * kLoaders + loader, box = at / (2 * S::kHalves), which = at / S::kHalves & 1, half = at % S::kHalves;
    uint32_t g = 0, n = 0;
    bool ok = true;
    auto page_at = [&](const Part& t, int key0) {
      const int key = key0 + box * box_rows;
      if (key >= t.keys || box * box_rows >= kUnit) return -1;
      bool bad;
      const int page = page_of(p.s, t.b, key, &bad);
      if (bad) bad_index(p.s.status);
      return bad ? 0 : page;
    };
    int page = page_at(t, (int)t.first * kUnit);
    for (long long u = lo; u < hi && ok;) {
      const int k_end = min((int)(t.first + t.take) * kUnit, t.keys), y0 = t.block / p.split.head_blocks << p.s.page_shift;
      if (loader == 0) {
        ok = __all_sync(0xffffffffu, mbar_wait(q_empty(n), (n >> 1 & 1u) ^ 1u, abort_flag));
        if (!ok) break;
      }
      if (loader == 0 && lane == 0) {
        mbar_expect_tx(q_full(n), (uint32_t)(p.split.tile_tokens * p.split.block_heads * D * 2));
        for (int h = 0; h < S::kHalves; ++h)
          tma_load_3d(base + S::kQ + (n & 1) * S::kHalves * S::kQHalf + h * S::kQHalf, &tm_q, q_full(n), h * 64, first_head(p, t.block), t.tok0);
      }
      ++n;
      const long long next = u + t.take;
      Part t2 = t;
      if (next < hi) next_part(p, t2, hi - next);
      if ((int)t.first * kUnit >= k_end && next < hi) page = page_at(t2, (int)t2.first * kUnit);  // a part without keys (more tokens than the table lists)
      for (int k0 = (int)t.first * kUnit; k0 < k_end; k0 += kUnit, ++g) {
        const int mine = page;
        page = k0 + kUnit < k_end ? page_at(t, k0 + kUnit) : next < hi ? page_at(t2, (int)t2.first * kUnit) : -1;
        ok = __all_sync(0xffffffffu, mbar_wait(empty(g), phase(g) ^ 1u, abort_flag));
        if (!ok) break;
        const int mine_boxes = __popc(__ballot_sync(0xffffffffu, mine >= 0));
        if (lane == 0) mbar_expect_tx(full(g), (uint32_t)(mine_boxes * box_rows * 128));
        __syncwarp();
        if (mine >= 0)
          tma_load_3d(keys_at(g) + which * S::kTile + half * S::kHalfBytes + box * box_rows * 128, which ? &tm_v : &tm_k, full(g), half * 64,
                      y0 + ((k0 + box * box_rows) & (page_tokens - 1)), mine);
      }
      t = t2;
      u = next;
    }
    if (*abort_flag) {  // copies in flight land before shared memory is given back
      const long long t0 = clock64();
      while (clock64() - t0 < 4000000LL) {
      }
    }
    return;
  }

  // ---- computation: warp w takes keys 32 w to 32 w + 31 of every unit
  bool cut_here = false, ok = true;
  uint32_t g = 0, n = 0;
  for (long long u = lo; u < hi; ++n) {
    const int head0 = first_head(p, t.block), heads = heads_of(p, t.block);
    int limit[2];  // keys that rows lane / 4 and lane / 4 + 8 see
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int row = (lane >> 2) + r * 8;
      limit[r] = p.split.causal && row < t.rows ? min(t.pos0 + row / p.split.block_heads + 1, t.keys) : t.keys;
    }
    uint32_t qf[D / 16][4];
    ok = ok && mbar_wait(q_full(n), n >> 1 & 1u, abort_flag);
    if (ok) {
      const uint32_t q = base + S::kQ + (n & 1) * S::kHalves * S::kQHalf;
#pragma unroll
      for (int k = 0; k < D / 16; ++k) {
        const int row = lane & 15, c = (k & 3) * 2 + (lane >> 4);
        ldsm_x4(qf[k], q + (k >> 2) * S::kQHalf + row * 128 + ((c ^ (row & 7)) << 4));
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(q_empty(n));
    }
    const int all_see = p.split.causal ? min(t.pos0 + 1, t.keys) : t.keys;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f}, o[D / 8][4];
#pragma unroll
    for (int i = 0; i < D / 8; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[i][e] = 0.f;

    const int k_end = min((int)(t.first + t.take) * kUnit, t.keys);
    for (int u0 = (int)t.first * kUnit; u0 < k_end && ok; u0 += kUnit, ++g) {
      ok = mbar_wait(full(g), phase(g), abort_flag);
      if (!ok) break;
      const int k0 = u0 + warp * kBlock;
      if (k0 < t.keys) {
        const uint32_t kt = keys_at(g) + warp * kBlock * 128, vt = kt + S::kTile;
        if (k0 + kBlock > t.keys) {
          // rows behind the last key: what the page or the ring happens to hold there, which a probability of zero does not undo where it is not finite
          for (int i = lane; i < (kBlock - (t.keys - k0)) * S::kHalves * 8; i += 32) {
            const int r = (t.keys - k0) + i / (S::kHalves * 8), c = i % (S::kHalves * 8);
            asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(vt + (c >> 3) * S::kHalfBytes + r * 128 + (c & 7) * 16), "r"(0) : "memory");
          }
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // before the next load into these rows
          __syncwarp();
        }
        float s[4][4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[i][e] = 0.f;
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
#pragma unroll
          for (int n2 = 0; n2 < 2; ++n2) {  // 16 keys: matrices (keys 0-7, columns 0-7), (0-7, 8-15), (8-15, 0-7), (8-15, 8-15)
            const int row = n2 * 16 + (lane & 7) + ((lane >> 4) << 3), c = (k & 3) * 2 + ((lane >> 3) & 1);
            uint32_t b[4];
            ldsm_x4(b, kt + (k >> 2) * S::kHalfBytes + row * 128 + ((c ^ (row & 7)) << 4));
            mma16816<T>(s[n2 * 2], qf[k], b[0], b[1]);
            mma16816<T>(s[n2 * 2 + 1], qf[k], b[2], b[3]);
          }
        }
        if (k0 + kBlock > all_see) {
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (k0 + i * 8 + (lane & 3) * 2 + (e & 1) >= limit[e >> 1]) s[i][e] = -INFINITY;
        }
        uint32_t pf[2][4];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          float mx = -INFINITY;
#pragma unroll
          for (int i = 0; i < 4; ++i) mx = fmaxf(mx, fmaxf(s[i][2 * r], s[i][2 * r + 1]));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
          const float m_new = fmaxf(m[r], mx * p.scale), sub = m_new == -INFINITY ? 0.f : m_new;
          const float corr = ex2(m[r] - sub);
          m[r] = m_new;
          float sum = 0.f;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float a = ex2(fmaf(s[i][2 * r], p.scale, -sub)), b = ex2(fmaf(s[i][2 * r + 1], p.scale, -sub));
            sum += a + b;
            pf[i >> 1][(i & 1) * 2 + r] = pack2<T>(a, b);
          }
          l[r] = l[r] * corr + sum;  // of this lane's columns
          if (__any_sync(0xffffffffu, corr != 1.f)) {
#pragma unroll
            for (int i = 0; i < D / 8; ++i) {
              o[i][2 * r] *= corr;
              o[i][2 * r + 1] *= corr;
            }
          }
        }
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
          for (int n2 = 0; n2 < D / 16; ++n2) {  // 16 keys x 16 columns of the values
            const int row = k * 16 + (lane & 15), c = (n2 & 3) * 2 + (lane >> 4);
            uint32_t b[4];
            ldsm_x4_trans(b, vt + (n2 >> 2) * S::kHalfBytes + row * 128 + ((c ^ (row & 7)) << 4));
            mma16816<T>(o[n2 * 2], pf[k], b[0], b[1]);
            mma16816<T>(o[n2 * 2 + 1], pf[k], b[2], b[3]);
          }
        __syncwarp();
      }
      if (lane == 0) mbar_arrive(empty(g));
    }
    // ---- the four warps' states become one
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
      l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
      if ((lane & 3) == 0) stats[warp * kRows + (lane >> 2) + r * 8] = make_float2(m[r], l[r]);
    }
    if (!warps_all(ok)) { ok = false; break; }
    float M[2], L[2], w[2];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int row = (lane >> 2) + r * 8;
      M[r] = -INFINITY;
      for (int i = 0; i < kWarps; ++i) M[r] = fmaxf(M[r], stats[i * kRows + row].x);
      const float sub = M[r] == -INFINITY ? 0.f : M[r];
      L[r] = 0.f;
      for (int i = 0; i < kWarps; ++i) L[r] += stats[i * kRows + row].y * ex2(stats[i * kRows + row].x - sub);
      w[r] = ex2(m[r] - sub);
    }
#pragma unroll
    for (int i = 0; i < D / 8; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[i][e] *= w[e >> 1];
#pragma unroll
    for (int half = 2; half > 0; half >>= 1) {  // warps 2, 3 to 0, 1; then 1 to 0
      float* mine = join + (warp & (half - 1)) * kRows * D;
      if (warp >= half && warp < 2 * half) {
#pragma unroll
        for (int i = 0; i < D / 8; ++i)
#pragma unroll
          for (int r = 0; r < 2; ++r)
            *reinterpret_cast<float2*>(mine + ((lane >> 2) + r * 8) * D + i * 8 + (lane & 3) * 2) = make_float2(o[i][2 * r], o[i][2 * r + 1]);
      }
      warps_sync();
      if (warp < half) {
#pragma unroll
        for (int i = 0; i < D / 8; ++i)
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const float2 v = *reinterpret_cast<const float2*>(mine + ((lane >> 2) + r * 8) * D + i * 8 + (lane & 3) * 2);
            o[i][2 * r] += v.x;
            o[i][2 * r + 1] += v.y;
          }
      }
      warps_sync();
    }
    const bool whole = t.take == t.units;
    const int slot = 2 * cta + (u == lo ? 0 : 1);
    if (warp == 0) {
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const int row = (lane >> 2) + r * 8, i = row / p.split.block_heads, h = row % p.split.block_heads;
        if (row >= t.rows || h >= heads) continue;
        if (whole) {
          const float inv = L[r] == 0.f ? 0.f : 1.f / L[r];
          T* dst = static_cast<T*>(p.out) + (long long)(t.tok0 + i) * p.ldo + (long long)(head0 + h) * D + (lane & 3) * 2;
#pragma unroll
          for (int c = 0; c < D / 8; ++c) *reinterpret_cast<uint32_t*>(dst + c * 8) = pack2<T>(o[c][2 * r] * inv, o[c][2 * r + 1] * inv);
        } else {
          float* dst = p.parts.o + ((long long)slot * kRows + row) * D + (lane & 3) * 2;
#pragma unroll
          for (int c = 0; c < D / 8; ++c) *reinterpret_cast<float2*>(dst + c * 8) = make_float2(o[c][2 * r], o[c][2 * r + 1]);
          if ((lane & 3) == 0) p.parts.ml[(long long)slot * kRows + row] = make_float2(M[r], L[r]);
        }
      }
    }
    if (!whole && t.first == 0) {  // the tile's beginning is here, its rest the next CTAs'
      cut_here = true;
      if (tid == 0) p.parts.cuts[cta] = cut_of(p, t, u, total, cta, ctas, slot);
    }
    u += t.take;
    if (u < hi) next_part(p, t, hi - u);
  }
  if (!cut_here && tid == 0) p.parts.cuts[cta].pieces = 0;
  if (!ok && lane == 0) atomicExch(p.s.status, (int)TTB_ERR_DEVICE_WAIT);
}

// Joins the parts of the tiles that were cut, of both kernels: a block (and its neighbours along y) for each of their CTAs, a warp for each row, parts in the
// order of the keys.
struct JoinParams {
  Parts parts[2];
  int rows[2];
  void* out;
  long long ldo;
};
template <typename T, int D>
__global__ void __launch_bounds__(128)
paged_join_kernel(const JoinParams p) {
  pdl_trigger();
  pdl_wait();
  const int which = blockIdx.z, lane = threadIdx.x & 31;
  const Parts parts = which ? p.parts[1] : p.parts[0];
  const int stride = which ? p.rows[1] : p.rows[0];
  const Cut c = parts.cuts[blockIdx.x];
  if (c.pieces == 0) return;
  constexpr int V = D / 32;
  for (int row = blockIdx.y * 4 + (threadIdx.x >> 5); row < c.rows; row += gridDim.y * 4) {
    const int i = row / c.block_heads, g = row % c.block_heads;
    if (g >= c.heads) continue;
    auto at = [&](int k) { return (long long)(k == 0 ? c.slot : 2 * ((int)blockIdx.x + k)) * stride + row; };
    float M = -INFINITY;
    for (int k = lane; k < c.pieces; k += 32) M = fmaxf(M, parts.ml[at(k)].x);
    M = warp_max(M);
    const float sub = M == -INFINITY ? 0.f : M;
    float L = 0.f, o[V];
#pragma unroll
    for (int v = 0; v < V; ++v) o[v] = 0.f;
    for (int k0 = 0; k0 < c.pieces; k0 += 32) {  // a lane has a part's weight; the parts' sums come eight at a time
      float mine = 0.f;
      if (k0 + lane < c.pieces) {
        const float2 ml = parts.ml[at(k0 + lane)];
        mine = ex2(ml.x - sub);
        L = fmaf(ml.y, mine, L);
      }
      const int n = min(32, c.pieces - k0);
      for (int k1 = 0; k1 < n; k1 += 8) {
        float x[8][V];
#pragma unroll
        for (int e = 0; e < 8; ++e)
#pragma unroll
          for (int v = 0; v < V; ++v) x[e][v] = parts.o[at(min(k0 + k1 + e, c.pieces - 1)) * D + v * 32 + lane];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float w = __shfl_sync(0xffffffffu, mine, k1 + e);  // zero behind the last, and for a part without a key for this row, which has no sums
#pragma unroll
          for (int v = 0; v < V; ++v) o[v] = w == 0.f ? o[v] : fmaf(x[e][v], w, o[v]);
        }
      }
    }
    L = warp_sum(L);
    const float inv = L == 0.f ? 0.f : 1.f / L;
    T* dst = static_cast<T*>(p.out) + (long long)(c.tok0 + i) * p.ldo + (long long)(c.head0 + g) * D;
#pragma unroll
    for (int v = 0; v < V; ++v) dst[v * 32 + lane] = from_f<T>(o[v] * inv);
  }
}

template <typename T, int D>
int launch_rows(ttb_ctx* ctx, const ttb_paged_kv* kv, int64_t heads, const Params& p) {
  using S = Shape<D>;
  CUtensorMap tm_q, tm_k, tm_v;
  if (!encode_maps(kv, std::is_same<T, __nv_bfloat16>::value, heads, p, p.split.tile_tokens, &tm_q, &tm_k, &tm_v))
    return fail(ctx, TTB_ERR_CUDA, "paged_attention: a tensor map was refused");
  static bool configured[64] = {};
  const int dev = ctx->device < 64 ? ctx->device : 63;
  if (!configured[dev]) {
    TTB_CUDA(ctx, cudaFuncSetAttribute(paged_rows_kernel<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kBytes));
    configured[dev] = true;
  }
  launch_pdl(paged_rows_kernel<T, D>, dim3((unsigned)ctx->sm_count), dim3(kThreads), S::kBytes, ctx->stream, tm_q, tm_k, tm_v, p);
  return launched(ctx, "paged_attention");
}

template <typename T, int D>
int launch_all(ttb_ctx* ctx, int dtype, const ttb_paged_kv* kv, int64_t heads, Params& p) {
  // Which kernel: sequences whose new tokens make kFewRows rows at most go to the one for few rows, the others to the other. The host knows the lengths'
  // sum only: with no more tokens than sequences one kernel takes all, whatever a single sequence has.
  const int few = p.group <= kFewRows ? kFewRows / p.group : 0;
  const bool one = kv->B == 1, rows_only = few > 0 && p.s.tokens <= (one ? few : (int)kv->B), many_only = few == 0 || (one && !rows_only);
  const int ctas = ctx->sm_count;
  size_t at = 0, o[2], ml[2], cuts[2];
  const int rows[2] = {kFewRows, kManyRows};
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
      p.split = split_of((int)heads, (int)kv->kv_heads, kFewRows, 1, kUnit, p.split.causal);
      st = launch_rows<T, D>(ctx, kv, heads, p);
    } else {
      p.split = split_of((int)heads, (int)kv->kv_heads, kManyRows / 2, 2, kUnit, p.split.causal);
      st = paged_tc_launch(ctx, dtype, kv, heads, p);
    }
  }
  if (!st) {
    launch_pdl(paged_join_kernel<T, D>, dim3((unsigned)ctas, used[1] ? 16 : kFewRows / 4, (unsigned)n), dim3(128), 0, ctx->stream, j);
    st = launched(ctx, "paged_attention_join");
  }
  const int f = ttb_free(ctx, ws, "paged_attention/parts");
  return st ? st : f;
}

}  // namespace

extern "C" int ttb_paged_attention(ttb_ctx* ctx, int dtype, const ttb_paged_kv* kv, const void* q, int64_t ldq, int64_t tokens, int64_t heads, int causal,
                                   float scale, void* out, int64_t ldo) {
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
  p.split.causal = causal != 0;
  if (kv->d == 64) return dtype == TTB_F16 ? launch_all<__half, 64>(ctx, dtype, kv, heads, p) : launch_all<__nv_bfloat16, 64>(ctx, dtype, kv, heads, p);
  return dtype == TTB_F16 ? launch_all<__half, 128>(ctx, dtype, kv, heads, p) : launch_all<__nv_bfloat16, 128>(ctx, dtype, kv, heads, p);
}
