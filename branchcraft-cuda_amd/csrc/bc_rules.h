// Which way the attention of new tokens goes, by a call's sizes: rules for the launch
// code and for the bindings, which take no workspace where none is used.
#pragma once

#include "branchcraft.h"

namespace bch {

constexpr int kFewRows = 32;  // rows of a request that take the narrow form

// Whether a window is as short as tables that are not cut, see cut_of (32 requests of
// 8 new tokens, window 1024, 24/8 heads, bias: 26 us, cut 40).  bc_chunk_attention
// does not ask: its results for such windows keep the bits that they had before this
// rule, those of sums joined from parts.
inline bool short_window(const bc_shape& s, const bc_chunk_inputs& in) {
  const bool few = (long long)in.tokens * (s.query_heads / s.kv_heads) <= (long long)kFewRows * s.batch;
  return in.causal && in.window > 0 && in.window <= (few ? 1024 : 512);
}

// Whether reading shared pages once can pay for the entries' own starts and the
// join, by what the host knows: the K and V that the requests may see, each its own,
// and their rows.  Measured, 32/8 heads, D = 128, single tokens, with and without:
//  - 69 MB (8 requests, 2048 shared tokens) 22.0 and 21.3 us, 136 MB (4096 tokens)
//    25.5 and 27.3, 277 MB (32 requests) 24 and 40, 8.9 GB (64, 32768) 82 and 774.
//  - Tables of up to 1024 tokens, which are not cut there: 64 requests, 512 tokens 31
//    and 16; past them, 1024 and up to 64 more, 22 and 35.
//  - Many requests of little each: every workgroup walks the batch, some 5 us per 64
//    requests.  Groups of 4: 504 requests of 0.5 MB 105 and 72, of 1 MB 110 and 107,
//    120 of 2.1 MB 34 and 47; of 8: 1024 of 2.1 MB 355 and 503.
//  - Under a window what is shared is less: 1024 tokens, 268 MB 50 and 47, 537 MB 38
//    and 51.
//  - Requests of many rows fill tiles by themselves: 8 of 64 rows over 8192 shared
//    tokens 46 and 51 us, of 96 rows 58 and 55.
inline bool sharing_pays(const bc_shape& s, int tokens, int window) {
  const long long table = (long long)s.max_pages * BC_PAGE_SIZE, rows = (long long)tokens * (s.query_heads / s.kv_heads);
  const long long seen = window > 0 && window < table ? window : table;
  const double mb = (double)s.batch * (double)seen * s.kv_heads * s.dim * 4 / 1e6;
  return s.batch > 1 && table > 1024 && rows <= 80ll * s.batch && mb >= (seen < table ? 400 : 100) &&
         mb >= 1.2 * s.batch;
}

}  // namespace bch
