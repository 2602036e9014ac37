// What the kernels over cache pages share: a call's sequences as the device sees them.
#pragma once
#include "ttb_common.cuh"
#include "ttb_paged_rules.cuh"

namespace ttb {
namespace paged {

// An index that the caller's tables hold and that is outside what it indexes: recorded, and never used.
__device__ __forceinline__ void bad_index(int* status) { atomicCAS(status, 0, (int)TTB_ERR_BAD_INDEX); }

// Checks of a ttb_paged_kv that its entry points have in common; TTB_OK and the device's view of it, or the status of the refusal.
inline int check_kv(ttb_ctx* ctx, const char* what, int dtype, const ttb_paged_kv* kv, int64_t tokens, Sequences* out) {
  TTB_REQUIRE(ctx, dtype == TTB_F16 || dtype == TTB_BF16, "%s: dtype must be F16 or BF16", what);
  TTB_REQUIRE(ctx, kv, "%s: null arguments", what);
  TTB_REQUIRE(ctx, kv->d == 64 || kv->d == 128, "%s: head size must be 64 or 128", what);
  TTB_REQUIRE(ctx, kv->kv_heads > 0 && kv->kv_heads <= 65535 && kv->pages > 0 && kv->pages < (1ll << 31), "%s: bad shape", what);
  int shift = 4;
  while (shift < 8 && (1 << shift) != kv->page_tokens) ++shift;
  TTB_REQUIRE(ctx, (1 << shift) == kv->page_tokens, "%s: a page holds 16, 32, 64, 128 or 256 tokens", what);
  TTB_REQUIRE(ctx, kv->B >= 0 && kv->B <= kMaxSequences, "%s: at most %d sequences", what, kMaxSequences);
  TTB_REQUIRE(ctx, kv->table_width > 0 && kv->table_width <= (1ll << 30) / kv->page_tokens && kv->table_stride >= kv->table_width,
              "%s: a row of the page table lists 1 to 2^30 tokens and is at most its stride wide", what);
  TTB_REQUIRE(ctx, tokens >= 0 && tokens < (1ll << 29), "%s: bad number of tokens", what);
  TTB_REQUIRE(ctx, kv->page_stride >= kv->kv_heads * kv->page_tokens * kv->d && kv->page_stride % 8 == 0 && kv->page_stride < (1ll << 37),
              "%s: pages are at least kv_heads * page_tokens * d elements apart, a multiple of 8", what);
  TTB_REQUIRE(ctx, ((reinterpret_cast<uintptr_t>(kv->keys) | reinterpret_cast<uintptr_t>(kv->values)) & 15) == 0,
              "%s: pools must be 16-byte aligned", what);
  const bool empty = kv->B == 0 || tokens == 0;  // nothing to do, and possibly nothing to point at
  TTB_REQUIRE(ctx, empty || (kv->keys && kv->values && kv->table && kv->cu_seqlens && kv->past_lens), "%s: null pointer", what);
  *out = Sequences{kv->table, kv->table_stride, kv->cu_seqlens, kv->past_lens, (int)kv->B, (int)tokens, (int)kv->pages, shift,
                   (int)(kv->table_width * kv->page_tokens), ctx->d_status};
  return TTB_OK;
}

}  // namespace paged
}  // namespace ttb
