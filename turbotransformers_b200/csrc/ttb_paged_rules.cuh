// How the attention over cache pages (ttb_paged_attention.cu) deals out its work. Host code as well, so that it can be checked without a GPU.
//
// A tile is the query rows that go through the keys together: `tile_tokens` new tokens of one sequence for `block_heads` query heads of one key head (row
// token * block_heads + head). Its keys are walked in units of `unit` tokens of the cache. All units of a batch stand in one line, by sequence, tile, head
// block and key, and every CTA takes an equal stretch of it, wherever that begins and ends: lengths are known on the device only, and the share of a CTA is
// the same whether the batch is one long sequence or many short ones. A tile whose units fall to several CTAs is joined from their parts.
#pragma once
#include <stdint.h>

#ifdef __CUDACC__
#define TTB_PAGED_FN __host__ __device__ __forceinline__
#else
#define TTB_PAGED_FN inline
#endif

namespace ttb {
namespace paged {

constexpr int kMaxSequences = 1024;  // of a call: their places in the line are kept in shared memory

// sum of floor((a * i + b) / m) for i < n, all of them not negative, m > 0: the lattice points under a line. Whole multiples of m come out of a and b; of what is left rows and
// columns of the points change places, which changes a and m as a step of Euclid's algorithm does (Graham, Knuth and Patashnik, Concrete Mathematics, 3.5, floor sums)
TTB_PAGED_FN int64_t floor_sum(int64_t n, int64_t m, int64_t a, int64_t b) {
  int64_t sum = 0;
  while (n > 0) {
    sum += (n - 1) * n / 2 * (a / m) + n * (b / m);
    a %= m;
    b %= m;
    const int64_t top = a * n + b;
    if (top < m) break;
    n = top / m;
    b = top % m;
    const int64_t t = m;
    m = a;
    a = t;
  }
  return sum;
}

// ---- a call's sequences as the device sees them
struct Sequences {
  const int32_t* table;
  long long table_stride;
  const int32_t* cu;
  const int32_t* past;
  int B, tokens;              // rows of q / k / v
  int pages, page_shift;      // pages of the pool, log2 of a page's tokens
  int cap;                    // tokens that a row of the table can list
  int* status;
};

struct Sequence {
  int tok0, n;  // its new tokens are rows tok0 .. tok0 + n - 1
  int past;     // tokens before them in the cache
};

// Sequence b. What does not fit the call (offsets outside its rows, a negative past, more tokens than the table lists) is cut to what does.
TTB_PAGED_FN Sequence sequence_of(const Sequences& s, int b, bool* bad) {
  Sequence q;
  const int tok0 = s.cu[b], end = s.cu[b + 1], past = s.past[b];
  const bool fits = tok0 >= 0 && end >= tok0 && end <= s.tokens;
  q.tok0 = fits ? tok0 : 0;
  q.n = fits ? end - tok0 : 0;
  q.past = past < 0 ? 0 : past > s.cap ? s.cap : past;
  *bad = !fits || past != q.past || (long long)q.past + q.n > s.cap;
  return q;
}

// The page that holds token `at` of sequence b (at < cap).
TTB_PAGED_FN int page_of(const Sequences& s, int b, int at, bool* bad) {
  const int page = s.table[b * s.table_stride + (at >> s.page_shift)];
  *bad = page < 0 || page >= s.pages;
  return page;
}

// ---- how the line is dealt out
struct Split {
  int block_heads;  // query heads of a tile
  int blocks;       // head blocks of a sequence, over all key heads
  int head_blocks;  // of them a key head's
  int tile_tokens, unit_shift, causal;
  int half;         // of two sets: tokens of one. A tile of no more is both sets' together, which take its units of keys in turn:
  int pair_shift;   // so many of them (log2) are one unit of the line
};

// `rows` rows a tile of `parts` separate sets: a set's rows are whole tokens. `unit` is a power of two.
TTB_PAGED_FN Split split_of(int heads, int kv_heads, int rows, int parts, int unit, int causal, int pair_shift) {
  Split s;
  const int group = heads / kv_heads;
  s.head_blocks = (group + rows - 1) / rows;
  s.block_heads = (group + s.head_blocks - 1) / s.head_blocks;
  s.head_blocks = (group + s.block_heads - 1) / s.block_heads;  // (none of them empty)
  s.blocks = kv_heads * s.head_blocks;
  s.tile_tokens = rows / s.block_heads * parts;
  s.half = parts == 2 ? s.tile_tokens / 2 : 0;
  s.pair_shift = pair_shift;
  s.unit_shift = 0;
  while ((1 << s.unit_shift) < unit) ++s.unit_shift;
  s.causal = causal;
  return s;
}

// A quotient of numbers that are not negative: of 32 bits where they fit, which takes a tenth of the instructions.
TTB_PAGED_FN int64_t quotient(int64_t a, int64_t b) { return ((a | b) >> 32) == 0 ? (int64_t)((uint32_t)a / (uint32_t)b) : a / b; }

TTB_PAGED_FN int64_t tiles_of(const Split& s, int64_t n) { return quotient(n + s.tile_tokens - 1, s.tile_tokens); }

// units of `keys` keys
TTB_PAGED_FN int64_t units_of(const Split& s, int64_t keys) { return (keys + (1 << s.unit_shift) - 1) >> s.unit_shift; }

// of one head block of tile t: of the keys that its last token sees
TTB_PAGED_FN int64_t units_of_tile(const Split& s, int64_t past, int64_t n, int64_t t) {
  const int64_t end = (t + 1) * s.tile_tokens, units = units_of(s, past + (s.causal && end < n ? end : n));
  return n - t * s.tile_tokens <= s.half ? (units + (1 << s.pair_shift) - 1) >> s.pair_shift : units;
}

// of the tiles before t together (t at most tiles_of)
TTB_PAGED_FN int64_t units_before_tile(const Split& s, int64_t past, int64_t n, int64_t t) {
  if (t == 0) return 0;
  const int64_t tiles = tiles_of(s, n);
  int64_t last = 0;  // of the sequence's last tile, where it is among them
  if (t == tiles) {
    last = units_of_tile(s, past, n, --t);
    if (t == 0) return last;
  }
  if (!s.causal) return t * units_of(s, past + n) + last;
  return floor_sum(t, 1 << s.unit_shift, s.tile_tokens, past + s.tile_tokens + (1 << s.unit_shift) - 1) + last;
}

TTB_PAGED_FN int64_t units_of_sequence(const Split& s, int64_t past, int64_t n) { return n > 0 ? units_before_tile(s, past, n, tiles_of(s, n)) * s.blocks : 0; }

// A piece of a tile's units in the line.
struct Place {
  int64_t tile;
  int block;             // head block
  int64_t units, first;  // units of the tile, and which of them
};

// Where unit x of a sequence (x < units_of_sequence) is.
TTB_PAGED_FN Place place_of(const Split& s, int64_t past, int64_t n, int64_t x) {
  int64_t lo = 0, hi = tiles_of(s, n);  // the last tile with units_before_tile * blocks <= x
  while (hi - lo > 1) {
    const int64_t mid = (lo + hi) >> 1;
    if (units_before_tile(s, past, n, mid) * s.blocks <= x) lo = mid;
    else hi = mid;
  }
  Place p;
  p.tile = lo;
  x -= lo ? units_before_tile(s, past, n, lo) * s.blocks : 0;
  p.units = units_of_tile(s, past, n, lo);
  p.block = (int)quotient(x, p.units);
  p.first = x - p.block * p.units;
  return p;
}

// CTAs that share a line of `units`, at least `least` units each; and where the stretch of CTA c begins.
TTB_PAGED_FN int ctas_of(int64_t units, int ctas, int least) {
  const int64_t n = quotient(units + least - 1, least);
  return n < ctas ? (int)n : ctas;
}
TTB_PAGED_FN int64_t first_unit(int64_t units, int ctas, int c) { return quotient(units * c, ctas); }

}  // namespace paged
}  // namespace ttb
