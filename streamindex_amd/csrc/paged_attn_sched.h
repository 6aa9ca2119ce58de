// What the paged attentions over 16-bit and 8-bit caches share on the device: views of a cache, and the schedule of the
// requests' row blocks and shares over the workgroups.
#pragma once

#include <cstdint>
#include <type_traits>

#include "paged_attn.h"

namespace si {

// Keeps a wave-uniform value in scalar registers from here on: a kernel argument fetched again inside the tile loop would
// be a scalar load in flight among the LDS reads, whose lgkmcnt waits count on completion in order.
template <typename T>
__device__ __forceinline__ void scalar_tie(T& x) {
  static_assert(sizeof(T) == 4 || sizeof(T) == 8, "one or two registers");
  // (readfirstlane on both sides: the asm needs a scalar, and its result does not count as uniform by itself)
  auto tied = [](uint32_t w) {
    w = static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(w)));
    asm volatile("" : "+s"(w));
    return static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(w)));
  };
  if constexpr (sizeof(T) == 4) {
    x = __builtin_bit_cast(T, tied(__builtin_bit_cast(uint32_t, x)));
  } else {
    const uint64_t w = __builtin_bit_cast(uint64_t, x);
    x = __builtin_bit_cast(T, static_cast<uint64_t>(tied(static_cast<uint32_t>(w >> 32))) << 32 | tied(static_cast<uint32_t>(w)));
  }
}

// A cache as one workgroup reads it.
struct CacheView {
  const int32_t* table;  // the request's row
  uint32_t ps, rstride, magic, shift, one;
  __device__ __forceinline__ uint32_t page_of(uint32_t key) const { return (__umulhi(key, magic) + (key & one)) >> shift; }
};
struct CacheBase {
  const char* base;
  uint32_t pstride, pages;
};
// (by value: a choice between two caches stays one between values at hand, not between addresses in memory)
__device__ __forceinline__ void view_cache(PagedCache c, int req, CacheView& v, CacheBase& b) {
  v.table = c.table + req * c.tstride;
  v.ps = c.ps;
  v.rstride = c.rstride;
  v.magic = c.magic;
  v.shift = c.shift;
  v.one = c.one;
  b.base = reinterpret_cast<const char*>(c.base);
  b.pstride = c.pstride;
  b.pages = static_cast<uint32_t>(c.pages);
  scalar_tie(v.table);
  scalar_tie(v.ps);
  scalar_tie(v.rstride);
  scalar_tie(v.magic);
  scalar_tie(v.shift);
  scalar_tie(v.one);
  scalar_tie(b.base);
  scalar_tie(b.pstride);
  scalar_tie(b.pages);
}
template <typename T>
__device__ __forceinline__ T pick(bool second, T x, T y) {
  return second ? y : x;
}

// ---------------------------------------------------------------------------
// Schedule
//
// Request r has blocks(r) = ceil(n_r H / 64) row blocks of about tiles(r) key tiles each.  With U = sum blocks tiles and
// `want` workgroups at once, a row block is cut into ceil(tiles / c) shares.  c is the cheapest of: no cut, and four steps
// from U / want up, the last one with which all shares run at once.  The cost is the longest share, in tiles, and 1/24 of a
// tile for each partial output of 64 rows, its write and read (us: 64 row blocks of 12, 24 and 40 tiles, D = 576, cut in two 27, 35 and
// 44 and whole 25, 41 and 60; 128 of them 36, 44, 54 and 28, 42, 62; with D = 128, 256 of 24 and 40, 30, 36 and 26, 38).
// With more row blocks than `want`, c = 2 U / want cuts only requests far longer than the average, which would otherwise
// end last on their own.
// Every workgroup does these sums itself, with lane-shift scans in 32 bits, and where there are at most 64 requests every
// wave, without a barrier (7,149 row blocks: 576 us with the barriers, 555 without).  An ascending cu_q makes the
// requests' rows disjoint, on which every bound here and the sizes of the partial outputs rest; with one that descends
// somewhere no request has rows.
// ---------------------------------------------------------------------------
struct PagedReq {
  int first, n, len;  // first row of q, new tokens, entries of the first cache
  int blocks, tiles;
  bool down;          // cu_q descends here
};

// Tiles of TK keys, 32 or 64, that hold x keys.
template <int TK>
__device__ __forceinline__ int key_tiles(int x) {
  return static_cast<int>((static_cast<uint32_t>(x) + (TK - 1u)) / static_cast<uint32_t>(TK));
}

// Keys [lo, hi) of the first cache that a token at position p sees, and entries of the second.  Lengths are taken from 0 on,
// so positions run from -N to 2^31 - 2 and nothing here leaves 32 bits.
__device__ __forceinline__ int win_lo(const PagedAttnArgs& a, int p) { return max(max(p + 1, 0) - a.window, 0); }
__device__ __forceinline__ int win_hi(const PagedAttnArgs& a, int p) { return max(min(p + 1, a.c1.keys), 0); }
__device__ __forceinline__ int ent_hi(const PagedAttnArgs& a, int p) {
  if (a.ratio == 0 || p < 0) return 0;
  return min(static_cast<int>(static_cast<uint32_t>(p + 1) / static_cast<uint32_t>(a.ratio)), a.c2.keys);
}

template <int TK>
__device__ __forceinline__ PagedReq paged_req(const PagedAttnArgs& a, int r) {
  PagedReq q;
  const int c0 = a.cu[r], c1 = a.cu[r + 1];
  q.len = max(a.lens[r], 0);
  q.first = min(max(c0, 0), a.N);
  q.n = max(min(c1, a.N) - q.first, 0);
  q.down = c1 < c0;
  q.blocks = static_cast<int>((static_cast<uint32_t>(q.n) * static_cast<uint32_t>(a.H) + (kRows - 1)) / kRows);
  // tiles of the last row block, which sees the most
  const int p = q.len - 1;
  const int span = max(win_hi(a, p) - win_lo(a, p - a.behind), 0);
  q.tiles = max(key_tiles<TK>(span) + key_tiles<TK>(ent_hi(a, p)), 1);
  return q;
}

struct PagedItem {  // what a workgroup does
  int first, n, len;  // the request, as PagedReq
  int req, block, share, shares;
  int slot;           // its partial output, where shares > 1
  int rec;            // number of its row block among the split ones
};

// Inclusive prefix sum over the wave: shifts within rows of 16 lanes, then the rows' last lanes to the rows behind.
__device__ __forceinline__ int wave_scan(int x) {
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false);  // row_shr:1
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);  // row_bcast:15 to rows 1 and 3
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);  // row_bcast:31 to rows 2 and 3
  return x;
}

__device__ __forceinline__ int shares_of(int tiles, uint32_t c) {
  return tiles <= 1 ? 1 : static_cast<int>((static_cast<uint32_t>(tiles) + c - 1) / c);
}

constexpr uint32_t kWhole = 0x7fffffffu;  // no row block is cut

// Number of this workgroup's item among `total`; `total` and on where it has none.  Consecutive workgroups go to the eight
// XCDs in turn: each XCD takes runs of up to 32 items, one to a CU, whose keys its L2 then holds once, and all of them the
// same number, however many of the launched workgroups the lengths leave without an item.  (512 row blocks of 288 tiles, D =
// 256: runs of 32 319 us, of 64 332, of 16 321.)
__device__ __forceinline__ int paged_item_number(int total) {
  const int xcd = blockIdx.x & 7, k = blockIdx.x >> 3;
  const int whole = total >> 8;  // rounds of 8 x 32
  if (k < 32 * whole) return ((k >> 5) * 8 + xcd) * 32 + (k & 31);
  const int rest = total - 256 * whole, run = (rest + 7) >> 3, i = k - 32 * whole;
  return i < run ? 256 * whole + xcd * run + i : total;
}

// The sum over the wave, in lane 63.
__device__ __forceinline__ float wave_sum_last(float x) {
  auto shifted = [](float v, auto CTRL, auto MASK) {
    return __uint_as_float(static_cast<uint32_t>(__builtin_amdgcn_update_dpp(
        0, static_cast<int>(__float_as_uint(v)), decltype(CTRL)::value, decltype(MASK)::value, 0xf, false)));
  };
  using std::integral_constant;
  x += shifted(x, integral_constant<int, 0x111>{}, integral_constant<int, 0xf>{});
  x += shifted(x, integral_constant<int, 0x112>{}, integral_constant<int, 0xf>{});
  x += shifted(x, integral_constant<int, 0x114>{}, integral_constant<int, 0xf>{});
  x += shifted(x, integral_constant<int, 0x118>{}, integral_constant<int, 0xf>{});
  x += shifted(x, integral_constant<int, 0x142>{}, integral_constant<int, 0xa>{});
  x += shifted(x, integral_constant<int, 0x143>{}, integral_constant<int, 0xc>{});
  return x;
}

// The largest over the wave, in lane 63, of values from 0 on.
__device__ __forceinline__ int wave_max_last(int x) {
  x = max(x, __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false));
  x = max(x, __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false));
  x = max(x, __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false));
  x = max(x, __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false));
  x = max(x, __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false));
  return max(x, __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false));
}

constexpr int kSteps = 4;
constexpr int kLeastTiles = 4;  // of a share at least
// Tiles of a share: the steps to try, from the sum of blocks x tiles (rounded up: fp32 sums of whole numbers, at most 2^-20
// too small over the few thousand additions of a call) and the number of row blocks.
struct ShareSteps {
  uint32_t step[kSteps];
  static __device__ __forceinline__ uint32_t tiles_of(float x, int least) {
    return static_cast<uint32_t>(__builtin_fminf(__builtin_fmaxf(__builtin_ceilf(x), static_cast<float>(least)), 0x1p30f));
  }
  __device__ __forceinline__ ShareSteps(float sum, int all, int want) {
    const float units = sum * (1.0f + 0x1p-16f), each = units / static_cast<float>(want);
    step[0] = tiles_of(each, kLeastTiles);
    step[1] = tiles_of(1.25f * each, 6);
    step[2] = tiles_of(1.5f * each, 8);
    // (sum of ceil(tiles / c) <= units / c + all <= want)
    step[3] = tiles_of(__builtin_fmaxf(2.f * each, all < want ? units / static_cast<float>(want - all) : 0.f), 16);
  }
  // For all < want row blocks, the longest of `longest` tiles, and items[i] shares with step i: see above.
  __device__ __forceinline__ uint32_t pick(const int (&items)[kSteps], int all, int longest, const PagedAttnArgs& a) const {
    uint32_t c = kWhole;
    float cost = static_cast<float>(longest);
#pragma unroll
    for (int i = kSteps - 1; i >= 0; --i) {
      const int more = items[i] - all, parts = more + min(more, all);  // partial outputs, at most
      const float x = static_cast<float>(min(static_cast<int>(step[i]), longest)) + static_cast<float>(parts) * a.part_cost;
      if (items[i] <= a.want && x < cost) {
        c = step[i];
        cost = x;
      }
    }
    return c;
  }
};

// This workgroup's item, or false.  For up to 64 requests, one to a lane, every wave for itself: no LDS and no barrier.
template <int TK>
__device__ __forceinline__ bool paged_schedule_wave(const PagedAttnArgs& a, PagedItem& it, bool& down) {
  const int lane = threadIdx.x & 63;
  PagedReq q{};
  if (lane < a.R) q = paged_req<TK>(a, lane);
  down = __builtin_amdgcn_ballot_w64(q.down) != 0;
  if (down) q.blocks = 0;
  auto last = [](int x) { return __builtin_amdgcn_readlane(x, kWave - 1); };
  uint32_t c = kWhole;
  if (a.part_o) {
    const float sum = wave_sum_last(static_cast<float>(q.blocks) * static_cast<float>(q.tiles));
    const int all = last(wave_scan(q.blocks)), longest = last(wave_max_last(q.blocks > 0 ? q.tiles : 0));
    const ShareSteps steps(__uint_as_float(static_cast<uint32_t>(last(static_cast<int>(__float_as_uint(sum))))), all, a.want);
    c = steps.step[kSteps - 1];
    if (all < a.want) {
      int shares[kSteps];
#pragma unroll
      for (int i = 0; i < kSteps; ++i) shares[i] = last(wave_scan(q.blocks * shares_of(q.tiles, steps.step[i])));
      c = steps.pick(shares, all, longest, a);
    }
  }
  const int s = shares_of(q.tiles, c);
  const int items = q.blocks * s, parts = s > 1 ? items : 0, recs = s > 1 ? q.blocks : 0;
  const int end = wave_scan(items), end_parts = wave_scan(parts), end_recs = wave_scan(recs);
  if (a.part_o && blockIdx.x == 0 && threadIdx.x == kWave - 1) a.rec[0] = end_recs;
  const int total = last(end), id = paged_item_number(total);
  if (id >= total) return false;
  const int r = __builtin_ctzll(__builtin_amdgcn_ballot_w64(id < end));  // the first request that ends behind it
  auto at = [&](int x) { return __builtin_amdgcn_readlane(x, r); };
  const int shares = at(s), k = id - at(end - items), block = k / shares;
  // (the last row blocks see the most keys: they start first)
  it = PagedItem{at(q.first), at(q.n), at(q.len), r, at(q.blocks) - 1 - block, k - block * shares, shares,
                 at(end_parts - parts) + k, at(end_recs - recs) + block};
  return true;
}

// The same for any number.  All threads call it.
template <int TK>
__device__ __forceinline__ bool paged_schedule(const PagedAttnArgs& a, PagedItem& it, bool& down) {
  constexpr int W = kPagedThreads / kWave;
  __shared__ float units_lds[W];
  __shared__ int blocks_lds[W], longest_lds[W], items_lds[W][kSteps], sums_lds[3][W];
  __shared__ PagedItem found;
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  const int per = (a.R + kPagedThreads - 1) / kPagedThreads;
  const int r0 = min(t * per, a.R), r1 = min(r0 + per, a.R);
  PagedReq mine{};  // kept where a thread has one request
  float units = 0.f;
  int blocks = 0, longest = 0;
  bool descends = false;
  for (int r = r0; r < r1; ++r) {
    mine = paged_req<TK>(a, r);
    units = __builtin_fmaf(static_cast<float>(mine.blocks), static_cast<float>(mine.tiles), units);
    blocks += mine.blocks;
    longest = max(longest, mine.blocks > 0 ? mine.tiles : 0);
    descends = descends || mine.down;
  }
  down = __syncthreads_or(descends) != 0;
  if (down) {
    if (a.part_o && blockIdx.x == 0 && t == 0) a.rec[0] = 0;
    return false;
  }
  auto req = [&](int r) { return per == 1 ? mine : paged_req<TK>(a, r); };
  uint32_t c = kWhole;  // tiles of a share
  if (a.part_o) {
    units = wave_sum_last(units);
    blocks = wave_scan(blocks);
    longest = wave_max_last(longest);
    if (lane == kWave - 1) {
      units_lds[wave] = units;
      blocks_lds[wave] = blocks;
      longest_lds[wave] = longest;
    }
    __syncthreads();
    const int all = (blocks_lds[0] + blocks_lds[1]) + (blocks_lds[2] + blocks_lds[3]);
    longest = max(max(longest_lds[0], longest_lds[1]), max(longest_lds[2], longest_lds[3]));
    const ShareSteps steps((units_lds[0] + units_lds[1]) + (units_lds[2] + units_lds[3]), all, a.want);
    c = steps.step[kSteps - 1];
    if (all < a.want) {
      int n[kSteps] = {};
      for (int r = r0; r < r1; ++r) {
        const PagedReq q = req(r);
#pragma unroll
        for (int i = 0; i < kSteps; ++i) n[i] += q.blocks * shares_of(q.tiles, steps.step[i]);
      }
#pragma unroll
      for (int i = 0; i < kSteps; ++i) {
        n[i] = wave_scan(n[i]);
        if (lane == kWave - 1) items_lds[wave][i] = n[i];
      }
      __syncthreads();
#pragma unroll
      for (int i = 0; i < kSteps; ++i) n[i] = (items_lds[0][i] + items_lds[1][i]) + (items_lds[2][i] + items_lds[3][i]);
      c = steps.pick(n, all, longest, a);
    }
  }
  int items = 0, parts = 0, recs = 0;
  for (int r = r0; r < r1; ++r) {
    const PagedReq q = req(r);
    const int s = shares_of(q.tiles, c);
    items += q.blocks * s;
    if (s > 1) {
      parts += q.blocks * s;
      recs += q.blocks;
    }
  }
  int before[3];
  const int x3[3] = {items, parts, recs};
#pragma unroll
  for (int i = 0; i < 3; ++i) {
    const int v = wave_scan(x3[i]);
    if (lane == kWave - 1) sums_lds[i][wave] = v;
    before[i] = v - x3[i];
  }
  __syncthreads();
  int total[3];
#pragma unroll
  for (int i = 0; i < 3; ++i) {
    total[i] = 0;
#pragma unroll
    for (int w = 0; w < kPagedThreads / kWave; ++w) {
      if (w < wave) before[i] += sums_lds[i][w];
      total[i] += sums_lds[i][w];
    }
  }
  if (a.part_o && blockIdx.x == 0 && t == 0) a.rec[0] = total[2];
  const int id = paged_item_number(total[0]);
  if (id >= total[0]) return false;
  if (before[0] <= id && id < before[0] + items) {
    int at = before[0], part0 = before[1], rec0 = before[2];
    for (int r = r0; r < r1; ++r) {
      const PagedReq q = req(r);
      const int s = shares_of(q.tiles, c);
      const int n = q.blocks * s;
      if (id < at + n) {
        const int k = id - at;
        const int block = k / s;
        // (the last row blocks see the most keys: they start first)
        found = PagedItem{q.first, q.n, q.len, r, q.blocks - 1 - block, k - block * s, s, part0 + k, rec0 + block};
        break;
      }
      at += n;
      if (s > 1) {
        part0 += n;
        rec0 += q.blocks;
      }
    }
  }
  __syncthreads();
  it = found;
  return true;
}

constexpr float kNever = -__builtin_inff();
// A sink in log2 units: finite where it outweighs everything (inf - inf would follow).  Finite ones below the range become
// -inf, which weighs the same, nothing, beside a key, and a row whose keys weigh nothing takes its lse from the sink itself.
__device__ __forceinline__ float sink_log2(float sink) {
  constexpr float kMost = 3.4028234663852886e38f;
  const float x = sink * 1.4426950408889634f;
  return x > kMost ? kMost : x;  // (NaN stays)
}
__device__ __forceinline__ float lse_of_sink(float sink) { return sink == kNever ? -1.0e30f : sink; }
constexpr int kOdd = 1;    // a masked score that is not finite
constexpr int kMoved = 2;  // a reference maximum has moved: alpha is not one

}  // namespace si
