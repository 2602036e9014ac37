// Attention of the new tokens of ragged sequences over a pool of cache pages: out = softmax(scale * q . K^T) . V, token i of a sequence over the cached
// tokens 0 .. past + i (causal), or over all of them. `group` query heads share a key head.
//
// For few rows the call is bound by reading the keys and values once. All query rows of a tile (tokens x heads of one key head, up to 16) go through the keys
// together; the line of all tiles' keys is dealt out to one CTA an SM in equal stretches (ttb_paged_rules.cuh), so that one long sequence and a ragged batch
// keep every SM's loads busy alike. In a CTA four warps take blocks of 32 keys in turn, each with a ring of its own (three blocks in flight, TMA boxes of a page
// or of 32 keys, 128-byte swizzled) and a softmax state of its own (running maximum and sum in fp32, mma.sync m16n8k16): nothing is waited for but
// the own loads until the tile's end, where the four states are joined, and the rings run on into the next tile meanwhile. Parts of a tile that
// was cut go to a workspace in fp32 and a second kernel joins them, in the order of the keys.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "ttb_paged.cuh"
#include "ttb_sm100.cuh"

using namespace ttb;
using namespace ttb::paged;
using namespace ttb::sm100;

namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kWarps = 4, kThreads = kWarps * 32;
constexpr int kRows = 16;    // of a tile
constexpr int kBlock = 32;   // keys of a warp's step
constexpr int kUnit = kBlock * kWarps;

struct Params {
  Sequences s;
  Split split;
  const void* q;
  void* out;
  long long ldq, ldo;
  int group;        // query heads of a key head
  float scale;      // times log2 e
  float* part_o;    // [2 * CTAs][rows][d]: a CTA's first and last part
  float2* part_ml;  // [2 * CTAs][rows]: maximum (log2 units) and sum
  struct Cut* cuts; // [CTAs]
};

// A tile that was cut, written by the CTA that has its beginning.
struct Cut {
  int pieces;             // 0: none; the first is in slot `slot`, the others are the next CTAs' first parts
  int slot, tok0, head0, rows, block_heads;
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
template <typename T> __device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <> __device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
  __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&h);
}
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
  __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&h);
}
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

// The places of the sequences in the line: prefix[b] units before sequence b; prefix[B] is returned. All threads of the block.
__device__ __forceinline__ long long line_up(const Params& p, long long* prefix, long long* scratch, int threads) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  bool any_bad = false;
  for (int b = tid; b < p.s.B; b += threads) {
    bool bad;
    const Sequence q = sequence_of(p.s, b, &bad);
    any_bad |= bad;
    prefix[b] = units_of_sequence(p.split, q.past, q.n);
  }
  if (any_bad && blockIdx.x == 0) bad_index(p.s.status);
  __syncthreads();
  long long carry = 0;
  for (int b0 = 0; b0 < p.s.B; b0 += threads) {
    const int b = b0 + tid;
    const long long mine = b < p.s.B ? prefix[b] : 0;
    long long incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long v = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += v;
    }
    if (lane == 31) scratch[warp] = incl;
    __syncthreads();
    long long before = carry;
    for (int w = 0; w < threads / 32; ++w) {
      if (w < warp) before += scratch[w];
      carry += scratch[w];
    }
    if (b < p.s.B) prefix[b] = before + incl - mine;
    __syncthreads();
  }
  if (tid == 0) prefix[p.s.B] = carry;
  __syncthreads();
  return carry;
}

// A stretch's next part: units [first, first + take) of one tile and head block.
struct Part {
  int b, block, take;
  int tok0, rows, keys;   // first token's row of q, rows of the tile, keys of the sequence that the tile's last token sees
  int pos0;               // the first token's place in the sequence
  long long tile, units, first;
  Sequence q;
};

__device__ __forceinline__ void fill_part(const Params& p, Part& t, long long left) {
  const int tile0 = (int)t.tile * p.split.tile_tokens, n = min(p.split.tile_tokens, t.q.n - tile0);
  t.tok0 = t.q.tok0 + tile0;
  t.rows = n * p.split.block_heads;
  t.pos0 = t.q.past + tile0;
  t.keys = (int)min((long long)t.q.past + (p.split.causal ? tile0 + n : t.q.n), (long long)p.s.cap);
  t.take = (int)min(left, t.units - t.first);
}

// The part at unit u, of which `left` are the stretch's.
__device__ __forceinline__ Part part_at(const Params& p, const long long* prefix, long long u, long long left) {
  int lo = 0, hi = p.s.B;  // the last sequence with prefix <= u (that of an empty sequence equals its successor's)
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (prefix[mid] <= u) lo = mid;
    else hi = mid;
  }
  bool bad;
  Part t;
  t.b = lo;
  t.q = sequence_of(p.s, lo, &bad);
  const Place at = place_of(p.split, t.q.past, t.q.n, u - prefix[lo]);
  t.tile = at.tile;
  t.block = at.block;
  t.units = at.units;
  t.first = at.first;
  fill_part(p, t, left);
  return t;
}

// The part behind t, `left` units being left of the stretch (more than none).
__device__ __forceinline__ void next_part(const Params& p, Part& t, long long left) {
  t.first = 0;
  if (++t.block == p.split.blocks) {
    t.block = 0;
    ++t.tile;
    while (t.tile * p.split.tile_tokens >= t.q.n) {  // the next sequence that has new tokens: there is one
      bool bad;
      t.q = sequence_of(p.s, ++t.b, &bad);
      t.tile = 0;
    }
    t.units = units_of_tile(p.split, t.q.past, t.q.n, t.tile);
  }
  fill_part(p, t, left);
}

// first query head of a head block, and how many of its rows per token exist (the last block of a key head may be short)
__device__ __forceinline__ int first_head(const Params& p, int block) {
  return block / p.split.head_blocks * p.group + block % p.split.head_blocks * p.split.block_heads;
}

template <int D> struct Shape {
  static constexpr int kHalves = D / 64;
  static constexpr int kHalfBytes = kBlock * 128;
  static constexpr int kTile = kHalves * kHalfBytes;  // 32 keys, or 32 values
  static constexpr int kStages = D == 128 ? 3 : 6;
  static constexpr int kRing = kWarps * kStages * 2 * kTile;
  static constexpr int kJoin = 2 * kRows * D * 4;
  static constexpr int kPrefix = kRing + kJoin;
  static constexpr int kScratch = kPrefix + (kMaxSequences + 1) * 8;
  static constexpr int kStats = kScratch + kWarps * 8;
  static constexpr int kBars = kStats + kWarps * kRows * 8;
  static constexpr int kBytes = kBars + kWarps * kStages * 8 + 16;
};

template <typename T, int D>
__global__ void __launch_bounds__(kThreads, 1)
paged_rows_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v, const Params p) {
  using S = Shape<D>;
  extern __shared__ __align__(1024) uint8_t smem[];
  long long* prefix = reinterpret_cast<long long*>(smem + S::kPrefix);
  float* join = reinterpret_cast<float*>(smem + S::kRing);           // [2][kRows][D]
  float2* stats = reinterpret_cast<float2*>(smem + S::kStats);             // [kWarps][kRows]
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + S::kBars + kWarps * S::kStages * 8);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t ring = smem_u32(smem) + warp * S::kStages * 2 * S::kTile;
  const uint32_t bar0 = smem_u32(smem + S::kBars) + warp * S::kStages * 8;

  pdl_trigger();
  if (lane == 0) {
    for (int i = 0; i < S::kStages; ++i) mbar_init(bar0 + 8 * i, 1);
    if (warp == 0) {
      *abort_flag = 0;
      prefetch_tensormap(&tm_k);
      prefetch_tensormap(&tm_v);
    }
    mbar_init_fence();
  }
  pdl_wait();
  const long long total = line_up(p, prefix, reinterpret_cast<long long*>(smem + S::kScratch), kThreads);
  const int ctas = ctas_of(total, (int)gridDim.x, 1), cta = blockIdx.x;
  if (cta >= ctas) {
    if (tid == 0) p.cuts[cta].pieces = 0;
    return;
  }
  const long long lo = first_unit(total, ctas, cta), hi = first_unit(total, ctas, cta + 1);
  bool cut_here = false;

  // ---- this warp's loads: blocks of 32 keys, every fourth of a part
  const int box_rows = min(1 << p.s.page_shift, kBlock), boxes = kBlock / box_rows;
  Part lp = part_at(p, prefix, lo, hi - lo);
  long long lu = lo;          // where the part begins in the line
  int lk = (int)lp.first * kUnit + warp * kBlock;  // next block's first key
  uint32_t issued = 0, used = 0;
  // moves the load cursor to a block that exists; false: the stretch is through
  auto find_block = [&]() {
    while (lk >= min((int)(lp.first + lp.take) * kUnit, lp.keys)) {
      lu += lp.take;
      if (lu >= hi) return false;
      next_part(p, lp, hi - lu);
      lk = (int)lp.first * kUnit + warp * kBlock;
    }
    return true;
  };
  bool more = find_block();
  auto issue = [&]() {  // whole warp
    const int stage = issued % S::kStages;
    const int n = min(boxes, (lp.keys - lk + box_rows - 1) / box_rows);
    const uint32_t bar = bar0 + 8 * stage, dst = ring + stage * 2 * S::kTile;
    if (lane == 0) mbar_expect_tx(bar, (uint32_t)(n * box_rows * D * 2 * 2));
    __syncwarp();
    // lane: box of the block, keys or values, half of the head
    const int box = lane / (2 * S::kHalves), which = lane / S::kHalves & 1, half = lane % S::kHalves;
    if (box < n) {
      const int key = lk + box * box_rows;
      bool bad;
      int page = page_of(p.s, lp.b, key, &bad);
      if (bad) {
        bad_index(p.s.status);
        page = 0;
      }
      const int y = (lp.block / p.split.head_blocks << p.s.page_shift) + (key & ((1 << p.s.page_shift) - 1));
      tma_load_3d(dst + which * S::kTile + half * S::kHalfBytes + box * box_rows * 128, which ? &tm_v : &tm_k, bar, half * 64, y, page);
    }
    ++issued;
    lk += kUnit;
    more = find_block();
  };
  for (int i = 0; i < S::kStages && more; ++i) issue();

  // ---- this warp's part of the computation
  Part t = part_at(p, prefix, lo, hi - lo);
  bool ok = true;
  for (long long u = lo; u < hi;) {
    const int head0 = first_head(p, t.block);
    const int heads = min(p.split.block_heads, p.group - t.block % p.split.head_blocks * p.split.block_heads);
    // queries: rows lane / 4 and lane / 4 + 8, columns of mma fragments
    uint32_t qf[D / 16][4];
    int limit[2];  // keys that the row sees
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int row = (lane >> 2) + r * 8, i = row / p.split.block_heads, g = row % p.split.block_heads;
      const bool there = row < t.rows && g < heads;
      limit[r] = p.split.causal && row < t.rows ? min(t.pos0 + i + 1, t.keys) : t.keys;
      const T* src = static_cast<const T*>(p.q) + (long long)(t.tok0 + i) * p.ldq + (long long)(head0 + g) * D + (lane & 3) * 2;
#pragma unroll
      for (int k = 0; k < D / 16; ++k) {
        qf[k][r] = there ? *reinterpret_cast<const uint32_t*>(src + k * 16) : 0u;
        qf[k][r + 2] = there ? *reinterpret_cast<const uint32_t*>(src + k * 16 + 8) : 0u;
      }
    }
    const int all_see = p.split.causal ? min(t.pos0 + 1, t.keys) : t.keys;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f}, o[D / 8][4];
#pragma unroll
    for (int n = 0; n < D / 8; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[n][e] = 0.f;

    const int end = min((int)(t.first + t.take) * kUnit, t.keys);
    for (int k0 = (int)t.first * kUnit + warp * kBlock; k0 < end; k0 += kUnit) {
      const int stage = used % S::kStages;
      const uint32_t kt = ring + stage * 2 * S::kTile, vt = kt + S::kTile;
      if (!mbar_wait(bar0 + 8 * stage, (used / S::kStages) & 1u, abort_flag)) { ok = false; break; }
      ++used;
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
      for (int n = 0; n < 4; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[n][e] = 0.f;
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
        for (int n = 0; n < 4; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (k0 + n * 8 + (lane & 3) * 2 + (e & 1) >= limit[e >> 1]) s[n][e] = -INFINITY;
      }
      uint32_t pf[2][4];
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        float mx = -INFINITY;
#pragma unroll
        for (int n = 0; n < 4; ++n) mx = fmaxf(mx, fmaxf(s[n][2 * r], s[n][2 * r + 1]));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        const float m_new = fmaxf(m[r], mx * p.scale), sub = m_new == -INFINITY ? 0.f : m_new;
        const float corr = ex2(m[r] - sub);
        m[r] = m_new;
        float sum = 0.f;
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          const float a = ex2(fmaf(s[n][2 * r], p.scale, -sub)), b = ex2(fmaf(s[n][2 * r + 1], p.scale, -sub));
          sum += a + b;
          pf[n >> 1][(n & 1) * 2 + r] = pack2<T>(a, b);
        }
        l[r] = l[r] * corr + sum;  // of this lane's columns
        if (__any_sync(0xffffffffu, corr != 1.f)) {
#pragma unroll
          for (int n = 0; n < D / 8; ++n) {
            o[n][2 * r] *= corr;
            o[n][2 * r + 1] *= corr;
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
      if (more) issue();
    }
    if (!__syncthreads_and(ok)) break;

    // ---- the four warps' states become one
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
      l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
      if ((lane & 3) == 0) stats[warp * kRows + (lane >> 2) + r * 8] = make_float2(m[r], l[r]);
    }
    __syncthreads();
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
    for (int n = 0; n < D / 8; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[n][e] *= w[e >> 1];
#pragma unroll
    for (int half = 2; half > 0; half >>= 1) {  // warps 2, 3 to 0, 1; then 1 to 0
      float* mine = join + (warp & (half - 1)) * kRows * D;
      if (warp >= half && warp < 2 * half) {
#pragma unroll
        for (int n = 0; n < D / 8; ++n)
#pragma unroll
          for (int r = 0; r < 2; ++r)
            *reinterpret_cast<float2*>(mine + ((lane >> 2) + r * 8) * D + n * 8 + (lane & 3) * 2) = make_float2(o[n][2 * r], o[n][2 * r + 1]);
      }
      __syncthreads();
      if (warp < half) {
#pragma unroll
        for (int n = 0; n < D / 8; ++n)
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const float2 v = *reinterpret_cast<const float2*>(mine + ((lane >> 2) + r * 8) * D + n * 8 + (lane & 3) * 2);
            o[n][2 * r] += v.x;
            o[n][2 * r + 1] += v.y;
          }
      }
      __syncthreads();
    }
    const bool whole = t.take == t.units;
    const int slot = 2 * cta + (u == lo ? 0 : 1);
    if (warp == 0) {
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const int row = (lane >> 2) + r * 8, i = row / p.split.block_heads, g = row % p.split.block_heads;
        if (row >= t.rows || g >= heads) continue;
        if (whole) {
          const float inv = L[r] > 0.f ? 1.f / L[r] : 0.f;
          T* dst = static_cast<T*>(p.out) + (long long)(t.tok0 + i) * p.ldo + (long long)(head0 + g) * D + (lane & 3) * 2;
#pragma unroll
          for (int n = 0; n < D / 8; ++n) *reinterpret_cast<uint32_t*>(dst + n * 8) = pack2<T>(o[n][2 * r] * inv, o[n][2 * r + 1] * inv);
        } else {
          float* dst = p.part_o + ((long long)slot * kRows + row) * D + (lane & 3) * 2;
#pragma unroll
          for (int n = 0; n < D / 8; ++n) *reinterpret_cast<float2*>(dst + n * 8) = make_float2(o[n][2 * r], o[n][2 * r + 1]);
          if ((lane & 3) == 0) p.part_ml[(long long)slot * kRows + row] = make_float2(M[r], L[r]);
        }
      }
    }
    if (!whole && t.first == 0) {  // the tile's beginning is here, its rest the next CTAs'
      cut_here = true;
      if (tid == 0) {
        int pieces = 1;
        while (cta + pieces < ctas && first_unit(total, ctas, cta + pieces) < u + t.units) ++pieces;
        p.cuts[cta] = Cut{pieces, slot, t.tok0, head0, t.rows, heads};
      }
    }
    u += t.take;
    if (u < hi) next_part(p, t, hi - u);
  }
  if (!cut_here && tid == 0) p.cuts[cta].pieces = 0;
  __syncthreads();
  if (*abort_flag) {
    if (tid == 0) atomicExch(p.s.status, (int)TTB_ERR_DEVICE_WAIT);
    const long long t0 = clock64();  // copies in flight land before shared memory is given back
    while (clock64() - t0 < 4000000LL) {
    }
  }
}

// Joins the parts of the tiles that were cut: a block for each CTA of the kernel before, a warp for each row, parts in the order of the keys.
template <typename T, int D>
__global__ void __launch_bounds__(128)
paged_join_kernel(const Params p, int rows) {
  pdl_trigger();
  pdl_wait();
  const Cut c = p.cuts[blockIdx.x];
  if (c.pieces == 0) return;
  const int lane = threadIdx.x & 31;
  constexpr int V = D / 32;
  for (int row = blockIdx.y * 4 + (threadIdx.x >> 5); row < c.rows; row += gridDim.y * 4) {
    const int i = row / p.split.block_heads, g = row % p.split.block_heads;
    if (g >= c.block_heads) continue;
    auto slot = [&](int k) { return (long long)(k == 0 ? c.slot : 2 * ((int)blockIdx.x + k)) * rows + row; };
    float M = -INFINITY;
    for (int k = lane; k < c.pieces; k += 32) M = fmaxf(M, p.part_ml[slot(k)].x);
    M = warp_max(M);
    const float sub = M == -INFINITY ? 0.f : M;
    float L = 0.f, o[V];
#pragma unroll
    for (int v = 0; v < V; ++v) o[v] = 0.f;
#pragma unroll 4
    for (int k = 0; k < c.pieces; ++k) {
      const float2 ml = p.part_ml[slot(k)];
      const float w = ex2(ml.x - sub);
      L = fmaf(ml.y, w, L);
#pragma unroll
      for (int v = 0; v < V; ++v) o[v] = fmaf(p.part_o[slot(k) * D + v * 32 + lane], w, o[v]);
    }
    const float inv = L > 0.f ? 1.f / L : 0.f;
    T* dst = static_cast<T*>(p.out) + (long long)(c.tok0 + i) * p.ldo + (long long)(c.head0 + g) * D;
#pragma unroll
    for (int v = 0; v < V; ++v) dst[v * 32 + lane] = from_f<T>(o[v] * inv);
  }
}

template <typename T, int D>
int launch_rows(ttb_ctx* ctx, const ttb_paged_kv* kv, Params& p) {
  using S = Shape<D>;
  CUtensorMap tm_k, tm_v;
  const bool bf16 = sizeof(T) == 2 && std::is_same<T, __nv_bfloat16>::value;
  const uint32_t box_rows = (uint32_t)std::min<int64_t>(kv->page_tokens, kBlock);
  for (int i = 0; i < 2; ++i)
    if (!encode_tile_map_3d(i ? &tm_v : &tm_k, i ? kv->values : kv->keys, bf16, (uint64_t)kv->pages, (uint64_t)(kv->kv_heads * kv->page_tokens), D,
                            (uint64_t)kv->page_stride, D, 1, box_rows))
      return fail(ctx, TTB_ERR_CUDA, "paged_attention: the pools' tensor map was refused");
  static bool configured[64] = {};
  const int dev = ctx->device < 64 ? ctx->device : 63;
  if (!configured[dev]) {
    TTB_CUDA(ctx, cudaFuncSetAttribute(paged_rows_kernel<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kBytes));
    configured[dev] = true;
  }
  const int ctas = ctx->sm_count;
  void* ws = nullptr;
  const size_t o_bytes = (size_t)2 * ctas * kRows * D * 4, ml_bytes = (size_t)2 * ctas * kRows * 8;
  int st = ttb_alloc(ctx, o_bytes + ml_bytes + (size_t)ctas * sizeof(Cut), "paged_attention/parts", &ws);
  if (st) return st;
  p.part_o = static_cast<float*>(ws);
  p.part_ml = reinterpret_cast<float2*>(static_cast<char*>(ws) + o_bytes);
  p.cuts = reinterpret_cast<Cut*>(static_cast<char*>(ws) + o_bytes + ml_bytes);
  launch_pdl(paged_rows_kernel<T, D>, dim3((unsigned)ctas), dim3(kThreads), S::kBytes, ctx->stream, tm_k, tm_v, p);
  st = launched(ctx, "paged_attention");
  if (!st) {
    launch_pdl(paged_join_kernel<T, D>, dim3((unsigned)ctas, kRows / 4), dim3(128), 0, ctx->stream, p, kRows);
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
  p.split = split_of((int)heads, (int)kv->kv_heads, kRows, 1, kUnit, causal != 0);
  if (kv->d == 64) return dtype == TTB_F16 ? launch_rows<__half, 64>(ctx, kv, p) : launch_rows<__nv_bfloat16, 64>(ctx, kv, p);
  return dtype == TTB_F16 ? launch_rows<__half, 128>(ctx, kv, p) : launch_rows<__nv_bfloat16, 128>(ctx, kv, p);
}
