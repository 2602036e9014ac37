// What the two kernels of the attention over cache pages share: a call's parameters, the places of its tiles in the line of units (ttb_paged_rules.cuh), and the
// parts of tiles that were cut.
#pragma once
#include <algorithm>

#include "ttb_paged.cuh"
#include "ttb_sm100.cuh"

namespace ttb {
namespace paged {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kUnit = 128;    // keys
constexpr int kManyRows = 256;  // of a tile of the kernel for many rows

// A tile that was cut, written by the CTA that has its beginning.
struct Cut {
  int pieces;  // 0: none; the first is in slot `slot`, the others are the next CTAs' first parts
  int slot, tok0, head0, rows, block_heads, heads;  // rows: token * block_heads + head, of which the first `heads` exist
};

struct Parts {
  float* o;    // [2 * CTAs][rows of a tile][d]: a CTA's first and last part, sums of values
  float2* ml;  // [2 * CTAs][rows of a tile]: maximum (log2 units) and sum
  Cut* cuts;   // [CTAs]
};

struct Params {
  Sequences s;
  Split split;
  const void* q;
  void* out;
  long long ldq, ldo;
  int group;      // query heads of a key head
  int low, high;  // the kernel takes the sequences of low to high new tokens
  float scale;    // times log2 e
  const int32_t* room;  // may be null
  Parts parts;
};

// How far below the maximum of its first keys a row's reference lies (log2). fp16 has no normal numbers under 2^-14: where one key outweighs each of thousands of others by that much, as
// the first of a text may, every one of theirs would be rounded to a multiple of 2^-24 (17 above them: to 1.4 times itself). So the largest probabilities are 2^6 and more,
// and the edge lies at 2^-20 of them, half a step below it being 2^-31. More would bring sums of 128 equal ones to the limit of 2^15 at which a reference is raised.
// bf16 has fp32's range.
template <typename T> constexpr float kBelow = 0.f;
template <> constexpr float kBelow<__half> = 6.f;

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
// Sequence b, without new tokens where it is the other kernel's, or passed over for want of room.
__device__ __forceinline__ Sequence taken(const Params& p, int b, bool* bad) {
  Sequence q = sequence_of(p.s, b, bad);
  if (p.room && p.room[b] == 0) {
    q.n = 0;
    *bad = false;
  }
  if (q.n < p.low || q.n > p.high) q.n = 0;
  return q;
}

template <typename T> __device__ __forceinline__ float2 unpack2(uint32_t v);
template <> __device__ __forceinline__ float2 unpack2<__half>(uint32_t v) { return __half22float2(*reinterpret_cast<const __half2*>(&v)); }
template <> __device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t v) { return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&v)); }

// The places of the sequences in the line: prefix[b] units before sequence b; prefix[B] is returned. All threads of the block.
__device__ __forceinline__ long long line_up(const Params& p, long long* prefix, long long* scratch, int threads) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  bool any_bad = false;
  long long carry = 0;
  for (int b0 = 0; b0 < p.s.B; b0 += threads) {
    const int b = b0 + tid;
    long long mine = 0;
    if (b < p.s.B) {
      bool bad;
      const Sequence q = taken(p, b, &bad);
      any_bad |= bad;
      mine = units_of_sequence(p.split, q.past, q.n);
    }
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
    if (b0 + threads < p.s.B) __syncthreads();  // the scratch's last readers are through
  }
  if (any_bad && blockIdx.x == 0) bad_index(p.s.status);
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
  t.q = taken(p, lo, &bad);
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
      t.q = taken(p, ++t.b, &bad);
      t.tile = 0;
    }
    t.units = units_of_tile(p.split, t.q.past, t.q.n, t.tile);
  }
  fill_part(p, t, left);
}

// The first query head of a head block.
__device__ __forceinline__ int first_head(const Params& p, int block) {
  return block / p.split.head_blocks * p.group + block % p.split.head_blocks * p.split.block_heads;
}

// The query heads of a head block that exist (the last block of a key head may be short).
__device__ __forceinline__ int heads_of(const Params& p, int block) {
  return min(p.split.block_heads, p.group - block % p.split.head_blocks * p.split.block_heads);
}

// Whoever has the beginning of a tile that ends in another CTA's stretch, at unit u of the line, says so.
__device__ __forceinline__ Cut cut_of(const Params& p, const Part& t, long long u, long long total, int cta, int ctas, int slot) {
  // CTA c begins before the tile's end if total * c / ctas, rounded down or not, is less than that
  const int last = (int)quotient((u + t.units) * ctas + total - 1, total);
  const int pieces = min(last, ctas) - cta;
  return Cut{pieces, slot, t.tok0, first_head(p, t.block), t.rows, p.split.block_heads, heads_of(p, t.block)};
}

// A part of the line as a CTA's warps read it: one of them works it out, the others would have its code in the instruction cache besides (with it in every role the kernel
// for many rows was 192 KB long, and the products stood still for instructions).
struct Work {
  int units;       // that have keys; -1: there is no more
  int turns;       // many rows: both sets hold the same rows and take the units in turn
  int count[2];    // and each set's units
  int first;       // the part's first unit in its tile
  int b, key_row;  // sequence, and the key head's first row in a page
  int keys, pos0, tok0, rows;  // as in Part
  int head0, heads;
  int slot;        // of its sums, -1: the tile is whole
  int pad[2];
};
constexpr int kRingWorks = 8;

__device__ __forceinline__ Work work_of(const Params& p, const Part& t, int slot) {
  Work w;
  w.turns = t.rows <= p.split.half * p.split.block_heads;
  const int shift = w.turns ? p.split.pair_shift : 0;
  w.first = (int)t.first << shift;
  w.units = max(0, min(t.take << shift, (t.keys + kUnit - 1) / kUnit - w.first));
  w.count[0] = w.count[1] = 0;
  w.b = t.b;
  w.key_row = t.block / p.split.head_blocks << p.s.page_shift;
  w.keys = t.keys;
  w.pos0 = t.pos0;
  w.tok0 = t.tok0;
  w.rows = t.rows;
  w.head0 = first_head(p, t.block);
  w.heads = heads_of(p, t.block);
  w.slot = t.take == t.units ? -1 : slot;
  w.pad[0] = w.pad[1] = 0;
  return w;
}

// The tensor maps: boxes of `tokens` tokens of a head block's queries, of a page (128 tokens at most) of one key head's keys and values; 64 elements wide each.
inline bool encode_maps(const ttb_paged_kv* kv, bool bf16, int64_t heads, const Params& p, int tokens, CUtensorMap* q, CUtensorMap* k, CUtensorMap* v) {
  const uint32_t box_rows = (uint32_t)std::min<int64_t>(kv->page_tokens, kUnit);
  const uint64_t pages = (uint64_t)kv->pages, rows = (uint64_t)(kv->kv_heads * kv->page_tokens), stride = (uint64_t)kv->page_stride, d = (uint64_t)kv->d;
  return sm100::encode_tile_map_3d(q, p.q, bf16, (uint64_t)p.s.tokens, (uint64_t)heads, d, (uint64_t)p.ldq, d, (uint32_t)tokens, (uint32_t)p.split.block_heads) &&
         sm100::encode_tile_map_3d(k, kv->keys, bf16, pages, rows, d, stride, d, 1, box_rows) &&
         sm100::encode_tile_map_3d(v, kv->values, bf16, pages, rows, d, stride, d, 1, box_rows);
}

// The kernel for many rows (ttb_paged_attention_tc.cu) on tiles of kManyRows: launches it, parts of cut tiles going to p.parts (39 MB with heads of 128 and 148 SMs, whatever the
// call: lengths are not known here).
int paged_tc_launch(ttb_ctx* ctx, int dtype, const ttb_paged_kv* kv, int64_t heads, const Params& p);

}  // namespace paged
}  // namespace ttb
