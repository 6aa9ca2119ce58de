// Kernels of the paged attention (formulas in paged_attn.h).
//
// A workgroup of four waves takes 64 rows, a row being one head of one token: with 64 heads one token, with 16 heads
// four neighbouring tokens, so every key row that is fetched serves 64 query rows whatever the head count.  It walks
// the keys that any of its rows sees, 32 at a time, the window's first:
//   * the tile's rows are copied from their pages straight into LDS (global_load_lds, 16 bytes a lane, no staging
//     registers), one tile ahead of use, two tiles resident; the page numbers are fetched one tile further ahead;
//   * S^T = K Q^T on 16x16x32 MFMAs, keys on M: wave w takes rows 16w .. 16w+15, Q^T stays in registers;
//   * the online softmax is in-lane (a lane holds eight keys of one row) plus two lane exchanges when a maximum moves,
//     which it does only once a score exceeds it by 2^64 (fp16: 2^8), so the accumulator is rarely rescaled;
//   * P^T goes through LDS, and O^T += V^T P^T with the output dimensions dealt to the waves.
// P is rounded to the element type for the matrix core, the denominator sums the unrounded values in fp32.
// At D >= 512 two workgroups fit a CU (79 KB of LDS each); they run out of step, so one's copies, softmax and barriers
// fall behind the other's MFMAs.
//
// A key that only some of the 64 rows see is masked for the others by a weight of zero; the matrix core would still
// turn 0 x inf into NaN.  Keys and values being the same rows, such a value makes the key's raw score non-finite as
// well, so on a masked non-finite score the tile's values that are not finite are zeroed in LDS before P V; a row that
// does see such a key gets a weight of NaN there, and with it its output.
//
// Few rows over many keys: each workgroup works out from the requests' lengths how many shares a row block's tiles are
// cut into (Schedule below) and which share is its own; shares leave fp32 partial outputs that a second kernel joins.
// Nothing of the lengths is read on the host.
#include <string>
#include <type_traits>

#include "paged_attn.h"
#include "si_status.h"

namespace si {

// Keeps a wave-uniform value in scalar registers from here on: a kernel argument fetched again inside the tile loop would
// be a scalar load in flight among the LDS reads, whose lgkmcnt waits count on completion in order.
template <typename T>
__device__ __forceinline__ void scalar_tie(T& x) {
  asm volatile("" : "+s"(x));
}

// A cache as one workgroup reads it.
struct CacheView {
  const uint16_t* base;
  const int32_t* table;  // the request's row
  uint32_t pstride, rstride, ps, magic, shift;
  int pages;
  __device__ __forceinline__ CacheView(const PagedCache& c, int req)
      : base(c.base), table(c.table + (c.pages > 0 ? req * c.tstride : 0)), pstride(c.pstride), rstride(c.rstride), ps(c.ps),
        magic(c.magic), shift(c.shift), pages(c.pages) {
    scalar_tie(base);
    scalar_tie(table);
    scalar_tie(pstride);
    scalar_tie(rstride);
    scalar_tie(ps);
    scalar_tie(magic);
    scalar_tie(shift);
    scalar_tie(pages);
  }
};
__device__ __forceinline__ uint32_t page_div(uint32_t key, uint32_t magic, uint32_t shift) {
  return magic ? __umulhi(key, magic) >> shift : key;
}

// ---------------------------------------------------------------------------
// Schedule
//
// Request r has blocks(r) = ceil(n_r H / 64) row blocks of about tiles(r) key tiles each.  With U = sum blocks tiles and
// `want` workgroups, a row block is cut into ceil(tiles / c) shares; c is the smallest of eight steps from U / want to
// 2.75 U / want with which all shares run at once.  With more row blocks than that, c = 2 U / want cuts only requests
// far longer than the average, which would otherwise end last on their own.
// ---------------------------------------------------------------------------
struct PagedReq {
  int first, n, len;  // first row of q, new tokens, entries of the first cache
  int blocks, tiles;
};

__device__ __forceinline__ int ceil_div32(int x) { return static_cast<int>((static_cast<uint32_t>(x) + 31u) >> 5); }

// Keys [lo, hi) of the first cache that a token at position p sees.
__device__ __forceinline__ int64_t win_lo(const PagedAttnArgs& a, int64_t p) {
  const int64_t lo = p + 1 - a.window;
  return lo > 0 ? lo : 0;
}
__device__ __forceinline__ int64_t key_cap(const PagedCache& c) {  // keys that a block table row can name
  const int64_t cap = c.pages > 0 ? static_cast<int64_t>(c.P) * c.ps : 0;
  return cap < 0x7fffffff ? cap : 0x7fffffff;
}
__device__ __forceinline__ int64_t win_hi(const PagedAttnArgs& a, int64_t p) {
  const int64_t cap = key_cap(a.c1);
  const int64_t hi = p + 1 < cap ? p + 1 : cap;
  return hi > 0 ? hi : 0;
}
__device__ __forceinline__ int64_t ent_hi(const PagedAttnArgs& a, int64_t p) {  // entries of the second cache
  if (a.ratio == 0 || p < 0) return 0;
  const int64_t cap = key_cap(a.c2);
  const int64_t n = static_cast<uint32_t>(p + 1) / static_cast<uint32_t>(a.ratio);
  return n < cap ? n : cap;
}

__device__ __forceinline__ PagedReq paged_req(const PagedAttnArgs& a, int r) {
  PagedReq q;
  const int c0 = a.cu[r], c1 = a.cu[r + 1];
  q.first = c0 < 0 ? 0 : (c0 < a.N ? c0 : a.N);
  const int end = c1 < q.first ? q.first : (c1 < a.N ? c1 : a.N);
  q.n = end - q.first;
  q.len = a.lens[r];
  q.blocks = static_cast<int>((static_cast<uint32_t>(q.n) * static_cast<uint32_t>(a.H) + (kPagedRows - 1)) / kPagedRows);
  // tiles of the last row block, which sees the most
  const int64_t p = static_cast<int64_t>(q.len) - 1;
  const int64_t span = win_hi(a, p) - win_lo(a, p - (kPagedRows - 1) / a.H);
  q.tiles = ceil_div32(static_cast<int>(span > 0 ? span : 0)) + ceil_div32(static_cast<int>(ent_hi(a, p)));
  if (q.tiles < 1) q.tiles = 1;
  return q;
}

struct PagedItem {  // what a workgroup does
  int first, n, len;  // the request, as PagedReq
  int req, block, share, shares;
  int slot;           // its partial output, where shares > 1
  int rec;            // number of its row block among the split ones
};

// Sum of x over the workgroup and, with PREFIX, the sum over lower threads in *before.
template <bool PREFIX>
__device__ __forceinline__ int64_t wg_sum(int64_t x, int64_t* lds, int64_t* before) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int64_t v = x;
#pragma unroll
  for (int d = 1; d < kWave; d *= 2) {
    const int64_t y = __shfl_up(v, d);
    if (lane >= d) v += y;
  }
  if (lane == kWave - 1) lds[wave] = v;
  __syncthreads();
  int64_t all = 0, low = 0;
#pragma unroll
  for (int w = 0; w < kPagedThreads / kWave; ++w) {
    if (w < wave) low += lds[w];
    all += lds[w];
  }
  __syncthreads();
  if (PREFIX) *before = low + v - x;
  return all;
}

// This workgroup's item, or false.  All threads call it.
__device__ __forceinline__ bool paged_schedule(const PagedAttnArgs& a, int64_t id, PagedItem& it) {
  __shared__ int64_t lds[kPagedThreads / kWave];
  __shared__ PagedItem found;
  const int t = threadIdx.x;
  const int per = (a.R + kPagedThreads - 1) / kPagedThreads;
  const int r0 = min(t * per, a.R), r1 = min(r0 + per, a.R);
  int64_t units = 0, blocks = 0, before;
  PagedReq mine{};  // kept where a thread has one request
  for (int r = r0; r < r1; ++r) {
    mine = paged_req(a, r);
    units += static_cast<int64_t>(mine.blocks) * mine.tiles;
    blocks += mine.blocks;
  }
  auto req = [&](int r) { return per == 1 ? mine : paged_req(a, r); };
  int64_t c = 0x7fffffff;  // tiles of a share
  if (a.part_o) {
    units = wg_sum<false>(units, lds, nullptr);
    const int64_t all = wg_sum<false>(blocks, lds, nullptr);
    auto step = [&](int i) {
      const int64_t x = (units * (4 + i) + 4 * a.want - 1) / (4 * static_cast<int64_t>(a.want));
      return x > a.least ? x : static_cast<int64_t>(a.least);
    };
    c = step(4);
    if (all < a.want) {
      // shares of this thread's requests under each step
      int64_t pick = -1;
      for (int i = 0; i < 8 && pick < 0; ++i) {
        const int64_t ci = step(i);
        int64_t n = 0;
        for (int r = r0; r < r1; ++r) {
          const PagedReq q = req(r);
          n += static_cast<int64_t>(q.blocks) * ((q.tiles + ci - 1) / ci);
        }
        if (wg_sum<false>(n, lds, nullptr) <= a.want) pick = ci;
      }
      if (pick < 0) {  // (sum of ceil(tiles / c) <= units / c + blocks <= want)
        pick = (units + (a.want - all) - 1) / (a.want - all);
        if (pick < a.least) pick = a.least;
      }
      c = pick;
    }
  }
  int64_t items = 0, parts = 0, recs = 0;
  auto shares_of = [&](const PagedReq& q) { return static_cast<int>((q.tiles + c - 1) / c); };
  for (int r = r0; r < r1; ++r) {
    const PagedReq q = req(r);
    const int s = shares_of(q);
    items += static_cast<int64_t>(q.blocks) * s;
    if (s > 1) {
      parts += static_cast<int64_t>(q.blocks) * s;
      recs += q.blocks;
    }
  }
  int64_t part0, rec0;
  const int64_t total = wg_sum<true>(items, lds, &before);
  wg_sum<true>(parts, lds, &part0);
  const int64_t all_recs = wg_sum<true>(recs, lds, &rec0);
  if (a.part_o && id == 0 && t == 0) a.rec[0] = static_cast<int>(all_recs);
  if (id >= total) return false;
  if (before <= id && id < before + items) {
    int64_t at = before;
    for (int r = r0; r < r1; ++r) {
      const PagedReq q = req(r);
      const int s = shares_of(q);
      const int64_t n = static_cast<int64_t>(q.blocks) * s;
      if (id < at + n) {
        const int64_t k = id - at;
        // (the last row blocks see the most keys: they start first)
        const int block = static_cast<int>(k / s);
        found = PagedItem{q.first, q.n, q.len, r, q.blocks - 1 - block, static_cast<int>(k - static_cast<int64_t>(block) * s), s,
                          static_cast<int>(part0 + k), static_cast<int>(rec0 + block)};
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

// Waves of a SIMD, which is resident workgroups of a CU: 216 registers of a wave are Q^T and O^T at D = 576, 96 at D = 256.
constexpr int per_cu(int D) { return D >= 512 ? 1 : D == 256 ? 2 : 4; }

constexpr float kNever = -__builtin_inff();

// x with infinities and NaN replaced by zero.
template <bool F16>
__device__ __forceinline__ bf16x8 finite_or_zero(bf16x8 x) {
  constexpr uint32_t lo = F16 ? 0x7c00u : 0x7f80u, hi = lo << 16;
  u32x4 w = __builtin_bit_cast(u32x4, x);
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    uint32_t keep = 0;
    keep |= (w[c] & lo) != lo ? 0x0000ffffu : 0u;
    keep |= (w[c] & hi) != hi ? 0xffff0000u : 0u;
    w[c] &= keep;
  }
  return __builtin_bit_cast(bf16x8, w);
}

template <int D, bool F16>
__global__ __launch_bounds__(kPagedThreads, per_cu(D)) void paged_attn_kernel(PagedAttnArgs a) {
  using SH = AttnShape<D>;
  constexpr int KS = SH::KS, MBW = SH::MBW, ROW = SH::ROW;
  constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
  __shared__ __attribute__((aligned(16))) char kv_lds[2 * SH::TILE];
  __shared__ __attribute__((aligned(16))) char p_lds[4 * 64 * 16];
  __shared__ float alpha_lds[64], scale_lds[64];
  __shared__ int odd_lds[4];  // a masked non-finite score in this tile, by wave

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  __builtin_assume(wave >= 0 && wave < 4);
  const int g = lane >> 4, i16 = lane & 15;

  // Rows of no request: as a row without a key.
  {
    const int last = a.R > 0 ? a.cu[a.R] : 0;
    const int end = last < 0 ? 0 : (last < a.N ? last : a.N);
    for (int64_t t = end + static_cast<int64_t>(blockIdx.x); t < a.N; t += gridDim.x) {
      u32x4* orow = reinterpret_cast<u32x4*>(a.o + t * a.H * D);
      for (int e = threadIdx.x; e < a.H * SH::CPR; e += kPagedThreads) orow[e] = u32x4{0, 0, 0, 0};
      for (int h = threadIdx.x; h < a.H; h += kPagedThreads) {
        const float s = a.sink[h];
        a.lse[t * a.H + h] = s == kNever ? -1.0e30f : s;
      }
    }
  }
  PagedItem item;
  if (!paged_schedule(a, xcd_block_order(), item)) return;

  const int row0 = __builtin_amdgcn_readfirstlane(item.block) * kPagedRows;  // within the request
  const int nrows = min(__builtin_amdgcn_readfirstlane(item.n) * a.H - row0, kPagedRows);
  const int64_t pos0 = static_cast<int64_t>(__builtin_amdgcn_readfirstlane(item.len)) - __builtin_amdgcn_readfirstlane(item.n);
  const int req = __builtin_amdgcn_readfirstlane(item.req);
  const int shares = __builtin_amdgcn_readfirstlane(item.shares);
  const int64_t pa = pos0 + row0 / a.H, pb = pos0 + (row0 + nrows - 1) / a.H;  // first and last token
  // tiles of this row block: the window's, then the second cache's; and this share of them
  const int k1lo = static_cast<int>(win_lo(a, pa)), k1hi = static_cast<int>(win_hi(a, pb));
  const int k2hi = static_cast<int>(ent_hi(a, pb));
  const int n1 = k1hi > k1lo ? ceil_div32(k1hi - k1lo) : 0;
  const int ntiles = n1 + ceil_div32(k2hi);
  const int share = __builtin_amdgcn_readfirstlane(item.share);
  const int tbeg = static_cast<int>(static_cast<int64_t>(ntiles) * share / shares);
  const int tend = static_cast<int>(static_cast<int64_t>(ntiles) * (share + 1) / shares);

  // this lane's row: its Q^T fragments and the keys it sees
  const int lrow = wave * 16 + i16;
  const bool live = lrow < nrows;
  const int tok = live ? (row0 + lrow) / a.H : 0;
  const int head = live ? row0 + lrow - tok * a.H : 0;
  const int64_t pos = pos0 + tok;
  const int lo1 = live ? static_cast<int>(win_lo(a, pos)) : 0;
  const int cnt1 = live ? static_cast<int>(max(win_hi(a, pos) - win_lo(a, pos), int64_t{0})) : 0;
  const int cnt2 = live ? static_cast<int>(ent_hi(a, pos)) : 0;
  bf16x8 qf[KS];
  {
    const uint16_t* qrow = a.q + (static_cast<int64_t>(item.first) + tok) * a.qst + head * a.qsh;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) qf[ks] = live ? *reinterpret_cast<const bf16x8*>(qrow + ks * 32 + g * 8) : bf16x8{};
  }

  // ---- copies ----------------------------------------------------------------
  // Lanes l and l + 32 resolve key l of a tile; a key past the tile's last one stands in for by that one (it is masked,
  // and a tile always has a first key).  A key without a page reads row 0 of the cache and is masked.
  const CacheView c1(a.c1, req), c2(a.c2, req);
  struct Tile {
    int k0, end;
    bool second;
  };
  auto tile_of = [&](int t) {
    const bool second = t >= n1;
    return second ? Tile{(t - n1) * 32, k2hi, true} : Tile{k1lo + t * 32, k1hi, false};
  };
  auto load_page = [&](int t) {  // page number of this lane's key
    const Tile x = tile_of(t);
    const uint32_t key = static_cast<uint32_t>(min(x.k0 + (lane & 31), x.end - 1));
    const uint32_t magic = x.second ? c2.magic : c1.magic, shift = x.second ? c2.shift : c1.shift;
    const int32_t* table = x.second ? c2.table : c1.table;
    return table[page_div(key, magic, shift)];
  };
  auto row_off = [&](int t, int page, bool& ok) {  // offset of this lane's key, 16-byte units
    const Tile x = tile_of(t);
    const uint32_t key = static_cast<uint32_t>(min(x.k0 + (lane & 31), x.end - 1));
    const uint32_t magic = x.second ? c2.magic : c1.magic, shift = x.second ? c2.shift : c1.shift;
    const uint32_t ps = x.second ? c2.ps : c1.ps;
    const uint32_t pstride = x.second ? c2.pstride : c1.pstride, rstride = x.second ? c2.rstride : c1.rstride;
    const int pages = x.second ? c2.pages : c1.pages;
    ok = page >= 0 && page < pages;
    const uint32_t off = static_cast<uint32_t>(page) * pstride + (key - page_div(key, magic, shift) * ps) * rstride;
    return ok ? off : 0u;
  };
  auto copy_tile = [&](int t, uint32_t off) {
    const char* base = reinterpret_cast<const char*>(tile_of(t).second ? c2.base : c1.base);
    char* dst0 = kv_lds + (t & 1) * SH::TILE;
    int ln = lane;
    reg_tie(ln);  // (the copies' keys and chunks are worked out anew for each tile: kept, they would take 2 LPT registers)
#pragma unroll
    for (int i = 0; i < SH::LPT; ++i) {
      const int e0 = i * SH::NT + wave * 64;
      if (SH::CH % SH::NT == 0 || i + 1 < SH::LPT || e0 < SH::CH) {
        const int e = e0 + ln;
        const int key = e / SH::CPR;
        const uint32_t chunk = static_cast<uint32_t>((e % SH::CPR) ^ kv_swz<D>(key));
        const uint32_t row = static_cast<uint32_t>(__builtin_amdgcn_ds_bpermute(key * 4, static_cast<int>(off)));
        const uint16_t* src = reinterpret_cast<const uint16_t*>(base + (static_cast<uint64_t>(row + chunk) << 4));
        __builtin_amdgcn_global_load_lds(src, (lds_void_t*)(dst0 + e0 * 16), 16, 0, 0);
      }
    }
  };

  // ---- S^T -------------------------------------------------------------------
  // A-fragment addresses: key 16mb + i16, chunk 4ks + g; with f = kv_swz(i16), (4ks + g) ^ f = 4 (ks ^ (f >> 2)) +
  // (g ^ (f & 3)), so the offset is a per-lane base (one per parity of ks) plus 64 ks + 16 ROW mb.
  const int qf_swz = kv_swz<D>(i16);
  const int qbase = i16 * ROW + 16 * (g ^ (qf_swz & 3));
  const int qadj = 64 * (qf_swz >> 2);
  constexpr int QPD = KS < 3 ? KS : 3;
  auto qk = [&](int t, f32x4 (&st)[2]) {
    const uint32_t tile = lds_addr(kv_lds + (t & 1) * SH::TILE);
    const uint32_t qa_e = tile + qbase + qadj, qa_o = tile + qbase - qadj;
    bf16x8 kq[QPD][2];
    auto issue = [&](auto KC) {
      constexpr int ks = decltype(KC)::value;
      const uint32_t base = (ks & 1) ? qa_o : qa_e;
      kq[ks % QPD][0] = ld128<64 * ks>(base);
      kq[ks % QPD][1] = ld128<64 * ks + 16 * ROW>(base);
    };
    attn_static_for<0, QPD>(issue);
    st[0] = f32x4{0.f, 0.f, 0.f, 0.f};
    st[1] = f32x4{0.f, 0.f, 0.f, 0.f};
    attn_static_for<0, KS>([&](auto KC) {
      constexpr int ks = decltype(KC)::value;
      constexpr int later = (KS - 1 - ks) < (QPD - 1) ? (KS - 1 - ks) : (QPD - 1);
      lds_wait<2 * later>(kq[ks % QPD][0], kq[ks % QPD][1]);
      st[0] = mfma16x16x32<F16>(kq[ks % QPD][0], qf[ks], st[0]);
      st[1] = mfma16x16x32<F16>(kq[ks % QPD][1], qf[ks], st[1]);
      if constexpr (ks + QPD < KS) issue(std::integral_constant<int, ks + QPD>{});
    });
    mfma_result_fence(st[0], st[1]);
  };

  // Keys that every row sees: [all1lo, all1hi) of the first cache, [0, all2hi) of the second; none where rows are missing.
  int all1lo = static_cast<int>(win_lo(a, pb)), all1hi = nrows == kPagedRows ? static_cast<int>(win_hi(a, pa)) : -1;
  int all2hi = nrows == kPagedRows ? static_cast<int>(ent_hi(a, pa)) : -1;
  float scale = a.scale_log2;
  scalar_tie(all1lo);
  scalar_tie(all1hi);
  scalar_tie(all2hi);
  scalar_tie(scale);

  // ---- softmax -----------------------------------------------------------------
  float m_ref = kNever, l_run = 0.f;  // reference maximum (log2 domain) and this lane's share of the denominator
  auto softmax = [&](int t, uint32_t okmask, f32x4 (&st)[2]) {
    const Tile x = tile_of(t);
    // every row sees every key of the tile (32-bit sums: k0 is below the end of a range that fits 31 bits)
    const bool full = okmask == 0xffffffffu && (x.second ? x.k0 <= all2hi - 32 : x.k0 >= all1lo && x.k0 <= all1hi - 32);
    uint32_t seen = 0xffu;
    bool odd = false;
    if (!full) {
      seen = 0;
      const int lo = x.second ? 0 : lo1, cnt = x.second ? cnt2 : cnt1;
#pragma unroll
      for (int mb = 0; mb < 2; ++mb)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int kk = 16 * mb + 4 * g + r;
          const bool ok = static_cast<uint32_t>(x.k0 + kk - lo) < static_cast<uint32_t>(cnt) && ((okmask >> kk) & 1);
          if (ok) seen |= 1u << (4 * mb + r);
          const bool fin = __builtin_fabsf(st[mb][r]) < __builtin_inff();
          odd = odd || (!ok && !fin);
          st[mb][r] = ok ? (fin ? st[mb][r] : __builtin_nanf("")) : kNever;
        }
    }
    float y[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = st[i >> 2][i & 3] * scale;
    if (!full) {
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] = (seen >> i) & 1 ? y[i] : kNever;  // (a negative scale)
    }
    const float lmax = __builtin_fmaxf(__builtin_fmaxf(__builtin_fmaxf(y[0], y[1]), __builtin_fmaxf(y[2], y[3])),
                                       __builtin_fmaxf(__builtin_fmaxf(y[4], y[5]), __builtin_fmaxf(y[6], y[7])));
    constexpr float kLazy = F16 ? 8.0f : 64.0f;  // 2^8 keeps P in fp16's range, 2^64 in bf16's
    const bool first = m_ref == kNever;
    float alpha = 1.0f;
    if (__builtin_amdgcn_ballot_w64(first ? lmax > kNever : lmax > m_ref + kLazy) != 0) {
      const auto r16 = __builtin_amdgcn_permlane16_swap(__float_as_uint(lmax), __float_as_uint(lmax), false, false);
      float tmax = __builtin_fmaxf(__uint_as_float(r16[0]), __uint_as_float(r16[1]));
      const SwapPair r32 = permlane32_swap(__float_as_uint(tmax), __float_as_uint(tmax));
      tmax = __builtin_fmaxf(__uint_as_float(r32.x), __uint_as_float(r32.y));
      if (first ? tmax > kNever : tmax > m_ref + kLazy) {
        alpha = first ? 1.0f : __builtin_amdgcn_exp2f(m_ref - tmax);
        m_ref = tmax;
      }
    }
    const float ref = m_ref == kNever ? 0.f : m_ref;
    float p[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) p[i] = __builtin_amdgcn_exp2f(y[i] - ref);
    l_run = l_run * alpha + (((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7])));
    // P^T B-fragment: k-slots 8g+0..3 <-> keys 4g+0..3, 8g+4..7 <-> keys 16+4g+0..3
    u32x4 w;
#pragma unroll
    for (int c = 0; c < 4; ++c) w[c] = pack2<F16>(p[2 * c], p[2 * c + 1]);
    const uint32_t pdst = lds_addr(&p_lds[(wave * 64 + lane) * 16]);
    asm volatile("ds_write_b128 %0, %1" ::"v"(pdst), "v"(w) : "memory");
    if (g == 0) {
      const uint32_t adst = lds_addr(reinterpret_cast<const char*>(&alpha_lds[lrow]));
      asm volatile("ds_write_b32 %0, %1" ::"v"(adst), "v"(alpha) : "memory");
    }
    const int any_odd = __builtin_amdgcn_ballot_w64(odd) != 0;
    if (lane == 0) {
      const uint32_t odst = lds_addr(reinterpret_cast<const char*>(&odd_lds[wave]));
      asm volatile("ds_write_b32 %0, %1" ::"v"(odst), "v"(any_odd) : "memory");
    }
  };

  // ---- O^T += V^T P^T -------------------------------------------------------------
  f32x4 oacc[MBW][4];
#pragma unroll
  for (int j = 0; j < MBW; ++j)
#pragma unroll
    for (int nb = 0; nb < 4; ++nb) oacc[j][nb] = f32x4{0.f, 0.f, 0.f, 0.f};
  // V^T transposing reads: source lane (g, i16) points at key 4g + (i16 >> 2) (+16 for k-slots 4..7), dims d0 + 4 (i16 & 3)
  // with d0 = 16 (4j + wave); chunk 8j + x, x = 2 wave + ((i16 & 3) >> 1) < 8, swizzles to 8j + (x ^ f): a fixed base + 128 j.
  const int tkey = 4 * g + (i16 >> 2);
  const int tx = 2 * wave + ((i16 & 3) >> 1);
  const int tbase = tkey * ROW + 16 * ((tx ^ kv_swz<D>(tkey)) & (SH::CPR - 1)) + 8 * (i16 & 1);
  auto pv = [&](int t) {
    const uint32_t pa_ = lds_addr(&p_lds[0]) + lane * 16;
    bf16x8 pb_[4];
    pb_[0] = ld128<0>(pa_);
    pb_[1] = ld128<1024>(pa_);
    pb_[2] = ld128<2048>(pa_);
    pb_[3] = ld128<3072>(pa_);
    const uint32_t ta = lds_addr(kv_lds + (t & 1) * SH::TILE) + tbase;
    v4i16 lo[2], hi[2];
    lo[0] = tr_read<0>(ta);
    hi[0] = tr_read<16 * ROW>(ta);
    if constexpr (MBW > 1) {
      lo[1] = tr_read<128>(ta);
      hi[1] = tr_read<16 * ROW + 128>(ta);
    }
    attn_static_for<0, MBW>([&](auto JC) {
      constexpr int j = decltype(JC)::value;
      if constexpr (j + 1 < MBW) lds_wait<2>(lo[j & 1], hi[j & 1]); else lds_wait<0>(lo[j & 1], hi[j & 1]);
      if constexpr (j == 0) {
#pragma unroll
        for (int nb = 0; nb < 4; ++nb) reg_tie(pb_[nb]);
      }
      const bf16x8 vf = __builtin_bit_cast(bf16x8, __builtin_shufflevector(lo[j & 1], hi[j & 1], 0, 1, 2, 3, 4, 5, 6, 7));
#pragma unroll
      for (int nb = 0; nb < 4; ++nb) oacc[j][nb] = mfma16x16x32<F16>(vf, pb_[nb], oacc[j][nb]);
      if constexpr (j + 2 < MBW) {
        lo[j & 1] = tr_read<128 * (j + 2)>(ta);
        hi[j & 1] = tr_read<16 * ROW + 128 * (j + 2)>(ta);
      }
    });
  };
  // Values of tile t that are not finite become zero, in its LDS (every wave has done with its scores).
  auto clean_tile = [&](int t) {
    const uint32_t tile = lds_addr(kv_lds + (t & 1) * SH::TILE);
    for (int e = threadIdx.x; e < SH::CH; e += kPagedThreads) {
      bf16x8 x;
      asm volatile("ds_read_b128 %0, %1\n\ts_waitcnt lgkmcnt(0)" : "=v"(x) : "v"(tile + e * 16));
      x = finite_or_zero<F16>(x);
      asm volatile("ds_write_b128 %0, %1" ::"v"(tile + e * 16), "v"(x) : "memory");
    }
  };

  // ---- the tiles -------------------------------------------------------------
  if (tbeg < tend) {
    int page = load_page(tbeg);
    bool ok;
    uint32_t off = row_off(tbeg, page, ok);
    uint32_t okmask = static_cast<uint32_t>(__builtin_amdgcn_ballot_w64(ok));
    copy_tile(tbeg, off);
    if (tbeg + 1 < tend) page = load_page(tbeg + 1);
    for (int t = tbeg; t < tend; ++t) {
      // this wave's copies of tile t (and the page numbers of t + 1) have landed; behind the barrier every wave's have, and
      // every wave has left tile t - 1 and its P
      __builtin_amdgcn_s_waitcnt(vm_lgkm0(0));
      attn_tile_barrier();
      uint32_t ok_next = 0;
      if (t + 1 < tend) {
        bool ok1;
        const uint32_t off1 = row_off(t + 1, page, ok1);
        ok_next = static_cast<uint32_t>(__builtin_amdgcn_ballot_w64(ok1));
        copy_tile(t + 1, off1);
        if (t + 2 < tend) page = load_page(t + 2);
      }
      f32x4 st[2];
      qk(t, st);
      softmax(t, okmask, st);
      attn_tile_barrier();  // P, alpha published
      float al[4];
      int odd[4];
      {
        const uint32_t asrc = lds_addr(reinterpret_cast<const char*>(&alpha_lds[i16]));
        asm volatile("ds_read_b32 %0, %4\n\tds_read_b32 %1, %4 offset:64\n\tds_read_b32 %2, %4 offset:128\n\t"
                     "ds_read_b32 %3, %4 offset:192\n\ts_waitcnt lgkmcnt(0)"
                     : "=&v"(al[0]), "=&v"(al[1]), "=&v"(al[2]), "=&v"(al[3])
                     : "v"(asrc));
        const uint32_t osrc = lds_addr(reinterpret_cast<const char*>(&odd_lds[0]));
        u32x4 o4;
        asm volatile("ds_read_b128 %0, %1\n\ts_waitcnt lgkmcnt(0)" : "=v"(o4) : "v"(osrc));
#pragma unroll
        for (int nb = 0; nb < 4; ++nb) odd[nb] = __builtin_amdgcn_readfirstlane(static_cast<int>(o4[nb]));
      }
      if (__builtin_expect(__builtin_amdgcn_ballot_w64(al[0] != 1.0f || al[1] != 1.0f || al[2] != 1.0f || al[3] != 1.0f) != 0, 0)) {
#pragma unroll
        for (int j = 0; j < MBW; ++j)
#pragma unroll
          for (int nb = 0; nb < 4; ++nb) oacc[j][nb] = oacc[j][nb] * al[nb];
      }
      if (__builtin_expect((odd[0] | odd[1] | odd[2] | odd[3]) != 0, 0)) {
        clean_tile(t);
        attn_tile_barrier();
      }
      pv(t);
      okmask = ok_next;
    }
  }

  asm volatile("s_nop 7\n\ts_nop 7\n\ts_nop 3" ::: "memory");  // (the last MFMAs' wait states, see mfma_result_fence)

  // ---- the result ----------------------------------------------------------------
  float l_tot = l_run;
  {
    const auto r16 = __builtin_amdgcn_permlane16_swap(__float_as_uint(l_tot), __float_as_uint(l_tot), false, false);
    l_tot = __uint_as_float(r16[0]) + __uint_as_float(r16[1]);
    const SwapPair r32 = permlane32_swap(__float_as_uint(l_tot), __float_as_uint(l_tot));
    l_tot = __uint_as_float(r32.x) + __uint_as_float(r32.y);
  }
  const int64_t flat0 = static_cast<int64_t>(__builtin_amdgcn_readfirstlane(item.first)) * a.H + row0;  // first row of o
  if (shares > 1) {
    const int64_t slot = __builtin_amdgcn_readfirstlane(item.slot);
    if (g == 0) a.part_ml[slot * kPagedRows + lrow] = float2{m_ref, l_tot};
    float* po = a.part_o + slot * kPagedRows * D;
#pragma unroll
    for (int j = 0; j < MBW; ++j) {
      const int mbi = j * kAttnWaves + wave;
      if (SH::MBT % kAttnWaves == 0 || mbi < SH::MBT) {
#pragma unroll
        for (int nb = 0; nb < 4; ++nb)
          if (nb * 16 < nrows) *reinterpret_cast<f32x4*>(po + (nb * 16 + i16) * D + mbi * 16 + 4 * g) = oacc[j][nb];
      }
    }
    if (share == 0 && threadIdx.x == 0) {
      int32_t* rec = a.rec + 4 + 4 * static_cast<int64_t>(item.rec);
      *reinterpret_cast<int4*>(rec) = int4{static_cast<int>(slot), shares, static_cast<int>(flat0), nrows};
    }
    return;
  }
  {
    const float sink = live ? a.sink[head] : kNever;
    const float sink2 = sink * kLog2e;
    const float m_fin = __builtin_fmaxf(m_ref, sink2);
    const float ref = m_fin == kNever ? 0.f : m_fin;
    const float resc = __builtin_amdgcn_exp2f(m_ref - ref);
    const float l_fin = l_tot * resc + __builtin_amdgcn_exp2f(sink2 - ref);
    if (g == 0) {
      scale_lds[lrow] = l_fin == 0.f ? 0.f : resc / l_fin;
      if (live)
        a.lse[flat0 + lrow] = l_fin == 0.f ? -1.0e30f : l_tot == 0.f ? sink : (__builtin_amdgcn_logf(l_fin) + ref) * kLn2;
    }
  }
  __syncthreads();  // scales published, every wave has left the last tile
  // staged row by row in the tiles' LDS, chunk c of row r at c ^ (r & 7), then written in one piece: the rows follow each
  // other in o
  float sc[4];
#pragma unroll
  for (int nb = 0; nb < 4; ++nb) sc[nb] = scale_lds[nb * 16 + i16];
#pragma unroll
  for (int j = 0; j < MBW; ++j) {
    const int mbi = j * kAttnWaves + wave;
    if (SH::MBT % kAttnWaves == 0 || mbi < SH::MBT) {
#pragma unroll
      for (int nb = 0; nb < 4; ++nb) {
        const int row = nb * 16 + i16;
        uint2 w;
        w.x = pack2<F16>(oacc[j][nb][0] * sc[nb], oacc[j][nb][1] * sc[nb]);
        w.y = pack2<F16>(oacc[j][nb][2] * sc[nb], oacc[j][nb][3] * sc[nb]);
        *reinterpret_cast<uint2*>(kv_lds + kv_off<D>(row, 2 * mbi + (g >> 1)) + 8 * (g & 1)) = w;
      }
    }
  }
  __syncthreads();
  char* obase = reinterpret_cast<char*>(a.o + flat0 * D);
  for (int e = threadIdx.x; e < nrows * SH::CPR; e += kPagedThreads)
    *reinterpret_cast<u32x4*>(obase + static_cast<int64_t>(e) * 16) =
        *reinterpret_cast<const u32x4*>(kv_lds + kv_off<D>(e / SH::CPR, e % SH::CPR));
}

// Joins the shares of the split row blocks: a wave for each row, lanes along the dimensions.  Bound: the partial outputs,
// read once (they fit the last-level cache).
template <bool F16>
__global__ __launch_bounds__(kPagedThreads) void paged_combine_kernel(PagedAttnArgs a, int D) {
  constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int count = a.rec[0];
  for (int b = blockIdx.y; b < count; b += gridDim.y) {
    const int4 rec = *reinterpret_cast<const int4*>(a.rec + 4 + 4 * static_cast<int64_t>(b));
    const int row = blockIdx.x * 4 + wave;
    if (row >= rec.w) continue;
    const int64_t flat = static_cast<int64_t>(rec.z) + row;
    const float sink = a.sink[flat % a.H];
    const float sink2 = sink * kLog2e;
    const float2* ml = a.part_ml + static_cast<int64_t>(rec.x) * kPagedRows + row;
    float m = sink2;
    for (int i = 0; i < rec.y; ++i) m = __builtin_fmaxf(m, ml[static_cast<int64_t>(i) * kPagedRows].x);
    const float ref = m == kNever ? 0.f : m;
    float keys = 0.f;
    for (int i = 0; i < rec.y; ++i) {
      const float2 v = ml[static_cast<int64_t>(i) * kPagedRows];
      keys = __builtin_fmaf(v.y, __builtin_amdgcn_exp2f(v.x - ref), keys);
    }
    const float l = keys + __builtin_amdgcn_exp2f(sink2 - ref);
    const float inv = l == 0.f ? 0.f : 1.f / l;
    for (int d = lane * 4; d < D; d += 256) {
      const float* po = a.part_o + (static_cast<int64_t>(rec.x) * kPagedRows + row) * D + d;
      f32x4 acc = f32x4{0.f, 0.f, 0.f, 0.f};
      for (int i0 = 0; i0 < rec.y; i0 += 8) {
        f32x4 x[8];
        float w[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) {
          const int i = i0 + u < rec.y ? i0 + u : rec.y - 1;
          x[u] = *reinterpret_cast<const f32x4*>(po + static_cast<int64_t>(i) * kPagedRows * D);
          w[u] = ml[static_cast<int64_t>(i) * kPagedRows].x;
        }
#pragma unroll
        for (int u = 0; u < 8; ++u) {
          if (i0 + u >= rec.y) continue;
          const float e = __builtin_amdgcn_exp2f(w[u] - ref);
#pragma unroll
          for (int c = 0; c < 4; ++c) acc[c] = __builtin_fmaf(x[u][c], e, acc[c]);
        }
      }
      uint2 o;
      o.x = pack2<F16>(acc[0] * inv, acc[1] * inv);
      o.y = pack2<F16>(acc[2] * inv, acc[3] * inv);
      *reinterpret_cast<uint2*>(a.o + flat * D + d) = o;
    }
    if (lane == 0)
      a.lse[flat] = l == 0.f ? -1.0e30f : keys == 0.f ? sink : (__builtin_amdgcn_logf(l) + ref) * kLn2;
  }
}

template <int D>
static int launch_paged_attn_d(bool f16, const PagedAttnArgs& a, int64_t blocks, int64_t split_blocks, hipStream_t st) {
  if (f16) hipLaunchKernelGGL((paged_attn_kernel<D, true>), dim3(static_cast<unsigned>(blocks)), dim3(kPagedThreads), 0, st, a);
  else hipLaunchKernelGGL((paged_attn_kernel<D, false>), dim3(static_cast<unsigned>(blocks)), dim3(kPagedThreads), 0, st, a);
  int rc = check_launch("paged_attn_kernel");
  if (rc || !a.part_o) return rc;
  const dim3 grid(kPagedRows / 4, static_cast<unsigned>(split_blocks));
  if (f16) hipLaunchKernelGGL(paged_combine_kernel<true>, grid, dim3(kPagedThreads), 0, st, a, D);
  else hipLaunchKernelGGL(paged_combine_kernel<false>, grid, dim3(kPagedThreads), 0, st, a, D);
  return check_launch("paged_combine_kernel");
}

static bool served(int64_t D) { return D == 32 || D == 64 || D == 128 || D == 256 || D == 512 || D == 576; }

// Sizes of a call, from what the host knows.
struct PagedPlan {
  int64_t blocks;        // row blocks at most
  int64_t want;          // workgroups that run at once
  int64_t grid;          // workgroups
  int64_t items;         // partial outputs at most, 0: no row block is split
  int64_t split_blocks;  // split row blocks at most
  int64_t bytes;         // scratch
};
constexpr int kLeastTiles = 4;  // tiles of a share at least

static PagedPlan paged_plan_of(int64_t N, int64_t H, int64_t D, int64_t R, int64_t window, int64_t keys1, int64_t keys2) {
  PagedPlan p{};
  // a request's last row block is part empty unless 64 divides n H
  int64_t g = kPagedRows;
  while (H % g) g /= 2;
  p.blocks = (N * H + (R < N ? R : N) * (kPagedRows - g)) / kPagedRows;
  p.want = 256 * per_cu(static_cast<int>(D));
  p.grid = 2 * p.blocks <= p.want ? p.want : p.blocks + p.want;
  // tiles of a row block at most
  const int64_t span = kPagedRows / H + 1 + window;
  const int64_t tiles = ((window < keys1 && span < keys1 ? span : keys1) + 31) / 32 + (keys2 + 31) / 32;
  if (tiles <= kLeastTiles) {
    p.grid = p.blocks;
    return p;
  }
  // shares of split row blocks: sum of ceil(tiles / c) <= 2 sum tiles / c <= 2 want, where tiles > c >= U / want
  p.items = 2 * p.want;
  const int64_t each = p.blocks * ((tiles + kLeastTiles - 1) / kLeastTiles);
  if (each < p.items) p.items = each;
  p.split_blocks = p.items / 2;
  if (p.blocks < p.split_blocks) p.split_blocks = p.blocks;
  if (2 * p.blocks <= p.want && each < p.grid) p.grid = each;
  p.bytes = p.items * kPagedRows * (D * 4 + 8) + 16 * (p.split_blocks + 1);
  return p;
}

}  // namespace si

using namespace si;

static int64_t cache_keys(int64_t pages, int64_t P, int64_t ps) {
  const int64_t k = pages > 0 ? P * ps : 0;
  return k < 0x7fffffff ? k : 0x7fffffff;
}

extern "C" int64_t si_paged_attn_fwd_scratch_bytes(int64_t N, int64_t H, int64_t D, int64_t R, int64_t window,
                                                   int64_t keys, int64_t keys2) {
  const int64_t lim = 0x7fffffff;
  if (N <= 0 || H <= 0 || R <= 0 || window < 0 || keys < 0 || keys2 < 0 || !served(D) || N > lim || H > lim ||
      N * H > lim || R > lim)
    return 0;
  return paged_plan_of(N, H, D, R, window == 0 || window > lim ? lim : window, keys < lim ? keys : lim,
                       keys2 < lim ? keys2 : lim).bytes;
}

static int set_cache(PagedCache& c, const void* base, const int64_t* strides, int64_t pages, int64_t ps, int64_t D,
                     const int32_t* table, int64_t tstride, int64_t P, int64_t R, const char* name) {
  const std::string n(name);
  if (!strides) return set_error(SI_ERR_INVALID, n + ": null stride argument");
  if (pages < 0 || ps <= 0 || P < 0) return set_error(SI_ERR_INVALID, n + ": bad dimension");
  if (pages > 0x7fffffff || ps > 0x7fffffff || P > 0x7fffffff) return set_error(SI_ERR_UNSUPPORTED, n + ": dimension exceeds int32");
  if (R == 0) P = 0;
  if (pages > 0 && P > 0 && (!base || !table)) return set_error(SI_ERR_INVALID, n + ": null pointer argument");
  if (R > 1 && tstride < 0) return set_error(SI_ERR_INVALID, n + ": negative block table stride");
  if (strides[2] != 1 || strides[0] < 0 || strides[1] < 0 || (strides[0] | strides[1]) % 8 ||
      (reinterpret_cast<uintptr_t>(base) & 15))
    return set_error(SI_ERR_INVALID, n + " needs a contiguous last dimension, 16-byte rows and alignment");
  // (each factor below 2^31: no product overflows 64 bits before it is compared)
  const int64_t lim = int64_t{1} << 35;  // 64 GiB in elements
  if (pages > 0 && (strides[0] >= lim || strides[1] >= lim || (pages - 1) > (lim - 1) / (strides[0] > 0 ? strides[0] : 1) ||
                    (ps - 1) > (lim - 1) / (strides[1] > 0 ? strides[1] : 1) ||
                    (pages - 1) * strides[0] + (ps - 1) * strides[1] + D > lim))
    return set_error(SI_ERR_UNSUPPORTED, n + " larger than 64 GiB");
  c.base = static_cast<const uint16_t*>(base);
  c.table = table;
  c.tstride = tstride;
  c.pstride = static_cast<uint32_t>(strides[0] / 8);
  c.rstride = static_cast<uint32_t>(strides[1] / 8);
  c.P = static_cast<int>(P);
  c.pages = P > 0 ? static_cast<int>(pages) : 0;
  c.ps = static_cast<uint32_t>(ps);
  c.magic = 0;
  c.shift = 0;
  if (ps > 1) {
    // l = ceil(log2 ps): magic = ceil(2^(31 + l) / ps) is below 2^32 and exceeds 2^(31 + l) / ps by less than one, so
    // for key < 2^31 the product is off by less than 2^31 <= 2^(31 + l) / ps and the quotient is exact
    int l = 1;
    while ((int64_t{1} << l) < ps) ++l;
    c.magic = static_cast<uint32_t>(((uint64_t{1} << (31 + l)) + static_cast<uint64_t>(ps) - 1) / static_cast<uint64_t>(ps));
    c.shift = static_cast<uint32_t>(l - 1);
  }
  return SI_OK;
}

extern "C" int si_paged_attn_fwd(const void* q, const int64_t* q_strides, const void* kv, const int64_t* kv_strides,
                                 int64_t pages, int64_t page_size, const int32_t* block_table, int64_t table_stride,
                                 int64_t P, const void* kv2, const int64_t* kv2_strides, int64_t pages2,
                                 int64_t page_size2, const int32_t* block_table2, int64_t table_stride2, int64_t P2,
                                 int64_t window, int64_t ratio, const int32_t* cu_q, const int32_t* seq_lens,
                                 const float* attn_sink, int64_t N, int64_t H, int64_t D, int64_t R,
                                 float softmax_scale, int qkv_dtype, void* o, float* lse, void* scratch,
                                 int64_t scratch_bytes, void* stream) {
  if (qkv_dtype != SI_DTYPE_BF16 && qkv_dtype != SI_DTYPE_F16)
    return set_error(SI_ERR_INVALID, "qkv_dtype must be SI_DTYPE_BF16 (0) or SI_DTYPE_F16 (1)");
  if (N < 0 || H <= 0 || D <= 0 || R < 0 || window < 0 || ratio < 0) return set_error(SI_ERR_INVALID, "bad dimension");
  if (!served(D))
    return set_error(SI_ERR_UNSUPPORTED,
                     "unsupported head dim D=" + std::to_string(D) + " (supported: 32, 64, 128, 256, 512, 576)");
  if (N > 0x7fffffff || H > 0x7fffffff || R > 0x7fffffff || N * H > 0x7fffffff || ratio > 0x7fffffff)
    return set_error(SI_ERR_UNSUPPORTED, "dimension exceeds int32");
  if (!q_strides) return set_error(SI_ERR_INVALID, "null stride argument");
  if (N > 0 && (!q || !attn_sink || !o || !lse || !cu_q || (R > 0 && !seq_lens)))
    return set_error(SI_ERR_INVALID, "null pointer argument");
  if (q_strides[2] != 1 || (q_strides[0] | q_strides[1]) % 8)
    return set_error(SI_ERR_INVALID, "q needs a contiguous last dimension and strides that are multiples of 8 elements");
  if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(o) | reinterpret_cast<uintptr_t>(scratch)) & 15)
    return set_error(SI_ERR_INVALID, "q, o and scratch must be 16-byte aligned");
  PagedAttnArgs a{};
  int rc = set_cache(a.c1, kv, kv_strides, pages, page_size, D, block_table, table_stride, P, R, "kv");
  if (rc) return rc;
  if (ratio > 0) {
    rc = set_cache(a.c2, kv2, kv2_strides, pages2, page_size2, D, block_table2, table_stride2, P2, R, "kv2");
    if (rc) return rc;
  }
  if (N == 0) return SI_OK;
  a.q = static_cast<const uint16_t*>(q);
  a.qst = q_strides[0];
  a.qsh = q_strides[1];
  a.window = window == 0 || window > 0x7fffffff ? 0x7fffffff : static_cast<int>(window);
  a.ratio = static_cast<int>(ratio);
  a.cu = cu_q;
  a.lens = seq_lens;
  a.sink = attn_sink;
  a.o = static_cast<uint16_t*>(o);
  a.lse = lse;
  a.N = static_cast<int>(N);
  a.H = static_cast<int>(H);
  a.R = static_cast<int>(R);
  a.scale_log2 = softmax_scale * 1.4426950408889634f;
  PagedPlan p = paged_plan_of(N, H, D, R > 0 ? R : 1, a.window, cache_keys(pages, P, page_size),
                              ratio > 0 ? cache_keys(pages2, P2, page_size2) : 0);
  a.want = static_cast<int>(p.want);
  a.least = kLeastTiles;
  if (p.bytes > 0 && scratch && scratch_bytes >= p.bytes) {
    a.part_o = static_cast<float*>(scratch);
    a.part_ml = reinterpret_cast<float2*>(a.part_o + p.items * kPagedRows * D);
    a.rec = reinterpret_cast<int32_t*>(a.part_ml + p.items * kPagedRows);
  } else {
    p.grid = p.blocks;
  }
  if (p.grid < 1) p.grid = 1;
  hipStream_t st = static_cast<hipStream_t>(stream);
  const bool f16 = qkv_dtype == SI_DTYPE_F16;
  switch (D) {
    case 32: return launch_paged_attn_d<32>(f16, a, p.grid, p.split_blocks, st);
    case 64: return launch_paged_attn_d<64>(f16, a, p.grid, p.split_blocks, st);
    case 128: return launch_paged_attn_d<128>(f16, a, p.grid, p.split_blocks, st);
    case 256: return launch_paged_attn_d<256>(f16, a, p.grid, p.split_blocks, st);
    case 512: return launch_paged_attn_d<512>(f16, a, p.grid, p.split_blocks, st);
    default: return launch_paged_attn_d<576>(f16, a, p.grid, p.split_blocks, st);
  }
}
