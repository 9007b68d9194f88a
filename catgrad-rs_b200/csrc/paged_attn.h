// paged_attn.h — the arguments of attention over a paged cache, and the kernels it is run on.
#pragma once

#include "paged.h"

namespace cg {

struct PagedAttnArgs {
  PagedRows rows;
  const void *q, *k_pages, *v_pages;
  void* out;
  int64_t q_ld, q_hs;   // from one token and one head of q to the next
  int64_t most;         // new tokens of a row, at most
  int64_t window;       // 0 = none
  float scale, cap;     // cap 0 = none
  int nh, nkv, d;
};

// Prompts in bf16 on tcgen05 (paged_fa.cu)
bool paged_fa_supported(const PagedAttnArgs& a);
int paged_fa(cg_ctx* c, const PagedAttnArgs& a);
// A few tokens per row, bf16 (paged_dec.cu)
bool paged_dec_supported(const PagedAttnArgs& a);
int paged_dec(cg_ctx* c, const PagedAttnArgs& a);

}  // namespace cg
