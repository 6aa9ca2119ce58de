// Attention of a ragged batch of new tokens over a paged cache, for gfx950.
//
//   o[t,h,:] = sum_k p_k kv[k,:] / (sum_k p_k + e^{sink_h - m}),  p_k = e^{scale q[t,h] . kv[k] - m},
//   lse[t,h] = log(sum_k p_k + e^{sink_h - m}) + m,
//
// over the keys that token t at position p sees: entries k of its request's first cache with p - window < k <= p, and
// entries i of its second cache with ratio (i + 1) - 1 <= p.  Keys and values are the same rows, shared by the heads.
#pragma once

#include "attn_common.h"
#include "si_common.h"

namespace si {

// One paged cache.  Row offsets are kept in 16-byte units in 32 bits (a cache spans at most 64 GiB).
struct PagedCache {
  const uint16_t* base;
  const int32_t* table;  // [R, P]
  int64_t tstride;
  uint32_t pstride, rstride;  // page and row, 16-byte units
  int pages;                  // 0: no key has a page
  int keys;                   // that a block table row can name
  uint32_t ps, magic, shift, one;  // key / ps = (mulhi(key, magic) + (key & one)) >> shift for keys below 2^31
};

struct PagedAttnArgs {
  const uint16_t* q;
  int64_t qst, qsh;
  PagedCache c1, c2;
  int window;        // 0x7fffffff: every earlier entry
  int ratio;         // second cache; 0: none
  const int32_t *cu, *lens;
  const float* sink;
  uint16_t* o;       // [N,H,D] contiguous
  float* lse;        // [N,H] contiguous
  int N, H, R;
  float scale_log2;
  int want;          // workgroups that run at once
  float part_cost;   // of a partial output, in tiles
  int behind;        // tokens of a row block before its last one at most
  float* part_o;     // [items, kRows / 16, D / 16, 64, 4]: blocks of 16 rows x 16 dimensions as a wave holds them; null:
                     // rows are not split
  float2* part_ml;   // [items, kRows]
  int32_t* rec;      // [0]: split row blocks; then 4 each: first item, shares, first row, rows
};

constexpr int kPagedThreads = 256;
constexpr int kRows = 64;  // (token, head) rows of a workgroup

}  // namespace si
