// Attention of a ragged batch of new tokens over paged caches held in 8 bits, for gfx950: the formulas of paged_attn.h with
// kv[k,:] = s_k c[k,:], e4m3 codes c and an fp32 scale s_k for each block of tokens.
//
// The work is laid out as over 16-bit caches (paged_attn_sched.h): a workgroup of four waves takes 64 rows, walks the keys
// that any of them sees, 64 at a time, copies each tile's codes straight into LDS, and few rows over many keys are
// split into shares.  What differs is the arithmetic:
//
//   * S^T = C Q^T on 16x16x32 MFMAs of q's type: a wave converts the codes, which it reads from LDS at half the bytes, as it
//     uses them, exactly, since every e4m3 value is one of bf16 and of fp16.  (The 8-bit matrix instructions would take the codes as
//     they are, with Q as a sum of e4m3 pieces, but sum eight products at a time to 2^-13 of the largest.  Measured: one of
//     900 beside one of 65,536 comes back as 896.)
//   * A score is (accumulator) x (s_k x the softmax scale), in fp32.
//   * O^T += V^T P^T with V's codes converted on their way from LDS, where each is read by one wave, and P s_k rounded to q's
//     type, so that the scales cost no pass over V.
//
// Bound, long keys: issue.  Two vector instructions beside a matrix instruction cost it a third of its time, and four waves convert
// each code for S^T.  (Converting each code once, into a second ring of tiles in LDS from which S^T and P V read elements,
// was slower all the same: 742 TFLOP/s at D = 512 and 688 at 256, against 888 and 940, one request of 8,192 earlier tokens,
// 64 heads, 1,024 and 2,048 new ones.)
//
// bf16, one request of 1,024 new tokens (2,048 at D = 256 and below) behind 8,192, 64 heads: 576 835 - 847 TFLOP/s, 512 888 - 901,
// 256 931 - 950, 128 785 - 792, 64 541, 32 297 (16-bit caches: 1,190, 1,117, 990, 735, 590, 305).  Decode, 64 heads, D = 576,
// 32 requests of 20,000 keys: 133 us, 2.8 TB/s of codes (16-bit caches 155).
//
// A masked key's code NaN is zeroed in LDS before P V (0 x NaN is NaN); every row that sees it has a score of NaN.
#include <cstdint>
#include <string>
#include <type_traits>

#include "paged_attn_sched.h"
#include "si_status.h"

namespace si {

// Scales of a cache: [pages, keys of a page / block].
struct QScales {
  const float* base;
  int64_t pstride;               // floats
  uint32_t magic, shift, one;    // key / block, as PagedCache's key / ps
  uint32_t per_page;
};
struct PagedAttnQArgs {
  PagedAttnArgs a;
  QScales s1, s2;
};

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x2 __attribute__((ext_vector_type(2)));

// PAIR: tiles of 32 keys, a tile's steps one after the other, and one workgroup more a CU, which fills the gaps.
template <int D, bool PAIR>
struct QShape {
  static constexpr int TK = PAIR ? 32 : 64;      // keys of a tile
  static constexpr int CPR = D / 16;             // 16-byte chunks of a key row
  static constexpr int ROW = D;                  // bytes
  static constexpr int TILE = TK * ROW;
  static constexpr int CH = TK * CPR;            // chunks of a tile
  static constexpr int LPT = (CH + kPagedThreads - 1) / kPagedThreads;  // copies of a thread
  static constexpr int LANDED = CH / kPagedThreads;                     // of every thread
  static constexpr int NG = D / 64;              // whole groups of 64 dimensions
  static constexpr int MBT = D / 16;             // 16-dim output blocks
  static constexpr int MBW = (MBT + 3) / 4;      // per wave
  static constexpr int NS = D == 512 && !PAIR ? 4 : 3;  // tiles in LDS
};
// Workgroups of a CU: LDS and registers set them.
constexpr int q_per_cu(int D, bool PAIR) { return PAIR ? 2 : D >= 512 ? 1 : D == 256 ? 2 : D == 128 ? 3 : 4; }

// Chunk c of key k is stored at c ^ q_swz(k), so that both reads of a tile spread over the banks: 16 keys 16 mb + 0 .. 15 at one
// chunk (S^T), and keys 4 g + 0 .. 3 and 16 + 4 g + 0 .. 3 at one chunk (V^T).
template <int D>
__device__ __forceinline__ int q_swz(int k) {
  const int h = ((k >> 2) ^ (k >> 4)) & 1;
  if constexpr (D == 32) return h;
  else if constexpr (D / 16 % 8 == 0) return (k & 3) | (h << 2);
  else return ((k >> 1) & 1) | (h << 1);
}

// ds_read_b64_tr_b8: lane i of 16 gets dimension i of eight keys, key j's 16 bytes behind lanes 2j and 2j + 1.
template <int OFF>
__device__ __forceinline__ i32x2 tr_read8(uint32_t addr) {
  i32x2 r;
  asm volatile("ds_read_b64_tr_b8 %0, %1 offset:%2" : "=v"(r) : "v"(addr), "n"(OFF));
  return r;
}
template <int OFF>
__device__ __forceinline__ i32x4 ldq(uint32_t addr) {
  i32x4 r;
  asm volatile("ds_read_b128 %0, %1 offset:%2" : "=v"(r) : "v"(addr), "n"(OFF));
  return r;
}
template <int OFF>
__device__ __forceinline__ i32x2 ldq64(uint32_t addr) {
  i32x2 r;
  asm volatile("ds_read_b64 %0, %1 offset:%2" : "=v"(r) : "v"(addr), "n"(OFF));
  return r;
}
// lds_wait for any registers.
template <int N, typename T>
__device__ __forceinline__ void lds_wait_for(T& x, T& y) {
  asm volatile("s_waitcnt lgkmcnt(%2)" : "+v"(x), "+v"(y) : "n"(N));
}
template <int N, typename T>
__device__ __forceinline__ void lds_wait_one(T& x) {
  asm volatile("s_waitcnt lgkmcnt(%1)" : "+v"(x) : "n"(N));
}
// Two of four codes as elements of the type (exact).
template <bool F16>
__device__ __forceinline__ uint32_t codes2(int codes, bool high) {
  const uint32_t x = static_cast<uint32_t>(codes);
  if constexpr (F16) {
    return __builtin_bit_cast(uint32_t, high ? __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(x, 1.0f, true)
                                             : __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(x, 1.0f, false));
  } else {
    return __builtin_bit_cast(uint32_t, high ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x, 1.0f, true)
                                             : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x, 1.0f, false));
  }
}
template <bool F16>
__device__ __forceinline__ bf16x8 codes8(int lo, int hi) {
  return __builtin_bit_cast(bf16x8, u32x4{codes2<F16>(lo, false), codes2<F16>(lo, true), codes2<F16>(hi, false), codes2<F16>(hi, true)});
}

struct QScaleView {
  const float* base;
  int64_t pstride;
  uint32_t magic, shift, one, per_page;
};

template <int D, bool F16, bool PAIR>
__global__ __launch_bounds__(kPagedThreads, q_per_cu(D, PAIR)) void paged_attn_q_kernel(PagedAttnQArgs args) {
  using SH = QShape<D, PAIR>;
  const PagedAttnArgs& a = args.a;
  constexpr int TK = SH::TK, MB = TK / 16, KSTEPS = TK / 32;
  constexpr int MBW = SH::MBW, ROW = SH::ROW, NG = SH::NG;
  constexpr int M = kRows, NB = M / 16;
  constexpr int NS = SH::NS, AHEAD = NS - 1, PAGES = 4, NP = PAIR ? 1 : 2;
  constexpr float kLn2 = 0.6931471805599453f;
  constexpr int PARTS = NS * SH::TILE >= M * D * 2 ? 1 : 2;  // of the output, staged in the tiles' LDS
  static_assert(NS * SH::TILE >= M * D * 2 / PARTS, "the output is staged in the tiles' LDS");
  __shared__ __attribute__((aligned(16))) char kv_lds[NS * SH::TILE];
  __shared__ __attribute__((aligned(16))) char p_lds[NP][KSTEPS][NB * 64 * 16];
  __shared__ __attribute__((aligned(16))) float alpha_lds[NP][M];
  __shared__ float sink_lds[M];
  __shared__ __attribute__((aligned(16))) int flag_lds[NP][4];
  __shared__ __attribute__((aligned(16))) int page_lds[kAttnWaves][PAGES][64];
  __shared__ __attribute__((aligned(16))) float scale_lds[kAttnWaves][NS][64];

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  __builtin_assume(wave >= 0 && wave < 4);
  const int g = lane >> 4, i16 = lane & 15;
  int begin = a.R > 0 ? min(max(a.cu[0], 0), a.N) : 0, end = a.R > 0 ? min(max(a.cu[a.R], 0), a.N) : 0;
  PagedItem item;
  bool down;
  const bool work = a.R <= kWave ? paged_schedule_wave<TK>(a, item, down) : paged_schedule<TK>(a, item, down);
  if (down) begin = end = 0;
  // Rows of no request: as a row without a key.
  for (int64_t i = blockIdx.x; i < begin + static_cast<int64_t>(a.N - end); i += gridDim.x) {
    const int64_t t = i < begin ? i : end + i - begin;
    u32x4* orow = reinterpret_cast<u32x4*>(a.o + t * a.H * D);
    for (int64_t e = threadIdx.x; e < static_cast<int64_t>(a.H) * (D / 8); e += kPagedThreads) orow[e] = u32x4{0, 0, 0, 0};
    for (int h = threadIdx.x; h < a.H; h += kPagedThreads) a.lse[t * a.H + h] = lse_of_sink(a.sink[h]);
  }
  if (!work) return;

  scalar_tie(item.first);
  scalar_tie(item.n);
  scalar_tie(item.len);
  scalar_tie(item.req);
  scalar_tie(item.block);
  scalar_tie(item.share);
  scalar_tie(item.shares);
  scalar_tie(item.slot);
  scalar_tie(item.rec);
  const int row0 = item.block * M;  // within the request
  const int nrows = min(item.n * a.H - row0, M);
  const int pos0 = item.len - item.n;
  const int req = item.req, shares = item.shares, share = item.share;
  const int pa = pos0 + row0 / a.H, pb = pos0 + (row0 + nrows - 1) / a.H;  // first and last token
  const int k1lo = win_lo(a, pa), k1hi = win_hi(a, pb);
  const int k2hi = ent_hi(a, pb);
  const int n1 = k1hi > k1lo ? key_tiles<TK>(k1hi - k1lo) : 0;
  const int ntiles = n1 + key_tiles<TK>(k2hi);
  const int tbeg = static_cast<int>(static_cast<int64_t>(ntiles) * share / shares);
  const int tend = static_cast<int>(static_cast<int64_t>(ntiles) * (share + 1) / shares);

  // (Lane addresses are worked out anew for each tile where registers are short: an opaque copy of the lane number keeps
  // the compiler from hoisting them.)
  auto lane_now = [&]() __attribute__((always_inline)) {
    int ln = lane;
    if constexpr (PAIR) reg_tie(ln);
    return ln;
  };

  // ---- copies ----------------------------------------------------------------
  // Lane l resolves key l of a tile, or l mod 32 (a key past the last one as that one, a key without a page as row 0; both are masked).
  // Every wave fetches all page numbers and scales for itself, a tile and no tile ahead of its copies, into LDS.
  CacheView view1, view2;
  CacheBase base1, base2;
  view_cache(a.c1, req, view1, base1);
  view_cache(a.c2, req, view2, base2);
  QScaleView sv1{args.s1.base, args.s1.pstride, args.s1.magic, args.s1.shift, args.s1.one, args.s1.per_page};
  QScaleView sv2{args.s2.base, args.s2.pstride, args.s2.magic, args.s2.shift, args.s2.one, args.s2.per_page};
  auto tie_scales = [](QScaleView& v) {
    scalar_tie(v.base);
    scalar_tie(v.pstride);
    scalar_tie(v.magic);
    scalar_tie(v.shift);
    scalar_tie(v.one);
    scalar_tie(v.per_page);
  };
  tie_scales(sv1);
  tie_scales(sv2);
  struct Source {  // of a tile to copy
    CacheBase cache;
    const float* scales;
    int64_t sstride;
  };
  CacheView view;       // of the next tile to fetch page numbers for
  QScaleView sview;
  Source from, from_next;
  uint32_t fkey = 0, fend = 0;
  int ftile = tbeg;
  auto enter = [&](int t) __attribute__((always_inline)) {
    const bool second = t >= n1;
    view = CacheView{pick(second, view1.table, view2.table), pick(second, view1.ps, view2.ps),
                     pick(second, view1.rstride, view2.rstride), pick(second, view1.magic, view2.magic),
                     pick(second, view1.shift, view2.shift), pick(second, view1.one, view2.one)};
    sview = QScaleView{pick(second, sv1.base, sv2.base), pick(second, sv1.pstride, sv2.pstride), pick(second, sv1.magic, sv2.magic),
                       pick(second, sv1.shift, sv2.shift), pick(second, sv1.one, sv2.one), pick(second, sv1.per_page, sv2.per_page)};
    from_next.cache = CacheBase{pick(second, base1.base, base2.base), pick(second, base1.pstride, base2.pstride),
                                pick(second, base1.pages, base2.pages)};
    fkey = second ? static_cast<uint32_t>(t - n1) * TK : static_cast<uint32_t>(k1lo) + static_cast<uint32_t>(t) * TK;
    fend = static_cast<uint32_t>(second ? k2hi : k1hi);
    scalar_tie(view.table);
    scalar_tie(view.ps);
    scalar_tie(view.rstride);
    scalar_tie(view.magic);
    scalar_tie(view.shift);
    scalar_tie(view.one);
    tie_scales(sview);
    scalar_tie(from_next.cache.base);
    scalar_tie(from_next.cache.pstride);
    scalar_tie(from_next.cache.pages);
    scalar_tie(fkey);
    scalar_tie(fend);
    from_next.scales = sview.base;
    from_next.sstride = sview.pstride;
  };
  struct Within {  // what a key's place in its page adds
    uint32_t row, block;
  };
  auto fetch_pages = [&]() __attribute__((always_inline)) {
    if (__builtin_expect(ftile == n1, 0) && ntiles > n1) enter(n1);
    const uint32_t key = min(fkey + static_cast<uint32_t>(lane_now() & (TK - 1)), fend - 1);
    const uint32_t col = view.page_of(key);
    __builtin_amdgcn_global_load_lds(reinterpret_cast<const uint32_t*>(view.table + col),
                                     (lds_void_t*)&page_lds[wave][ftile % PAGES][0], 4, 0, 0);
    ++ftile;
    fkey += TK;
    const uint32_t blk = (__umulhi(key, sview.magic) + (key & sview.one)) >> sview.shift;
    return Within{(key - col * view.ps) * view.rstride, blk - col * sview.per_page};
  };
  struct Rows {
    uint32_t row[SH::LPT];  // of this lane's copies, 16-byte units
  };
  // Sources of the tile whose page numbers are `page`, its scales on their way; returns which keys have a page.
  auto address_tile = [&](int page, const Within& in, Rows& y, int slot) __attribute__((always_inline)) {
    const bool ok = static_cast<uint32_t>(page) < from.cache.pages;
    const uint32_t p = ok ? static_cast<uint32_t>(page) : 0u;
    const uint32_t row = ok ? p * from.cache.pstride + in.row : 0u;
    const float* sc = from.scales + (ok ? static_cast<int64_t>(p) * from.sstride + in.block : 0);
    __builtin_amdgcn_global_load_lds(reinterpret_cast<const uint32_t*>(sc), (lds_void_t*)&scale_lds[wave][slot][0], 4, 0, 0);
#pragma unroll
    for (int i = 0; i < SH::LPT; ++i)  // the row of chunk 256 i + 64 wave + lane
      y.row[i] = static_cast<uint32_t>(__builtin_amdgcn_ds_bpermute(
          ((i * kPagedThreads + wave * 64 + lane_now()) / SH::CPR & (TK - 1)) * 4, static_cast<int>(row)));
    return __builtin_amdgcn_ballot_w64(ok);
  };
  auto copy = [&](const Rows& y, char* tile, auto IC) __attribute__((always_inline)) {
    constexpr int i = decltype(IC)::value;
    const int e = i * kPagedThreads + wave * 64 + lane_now(), k = e / SH::CPR;
    const uint32_t src = y.row[i] + static_cast<uint32_t>((e - k * SH::CPR) ^ q_swz<D>(k));
    char* dst = tile + i * (kPagedThreads * 16) + wave * 1024;
    if (SH::CH % kPagedThreads == 0 || i + 1 < SH::LPT || i * kPagedThreads + wave * 64 < SH::CH)
      __builtin_amdgcn_global_load_lds(reinterpret_cast<const uint32_t*>(from.cache.base + (static_cast<uint64_t>(src) << 4)),
                                       (lds_void_t*)dst, 16, 0, 0);
  };
  constexpr int LANDED = SH::LANDED;
  auto ring = [&](int slot) __attribute__((always_inline)) { return kv_lds + slot * SH::TILE; };
  auto page_addr = [&](int t) __attribute__((always_inline)) {
    return lds_addr(reinterpret_cast<const char*>(&page_lds[wave][t % PAGES][0])) + lane_now() * 4;
  };
  Within within[AHEAD + 1];
  Source froms[AHEAD + 1];
  enter(tbeg);
#pragma unroll
  for (int i = 0; i <= AHEAD; ++i) {
    within[i] = Within{0, 0};
    if (tbeg + i < tend) within[i] = fetch_pages();
    froms[i] = from_next;
  }
  __builtin_amdgcn_sched_barrier(0);

  // ---- this lane's row of Q -----------------------------------------------------
  // Of each group of 64 dimensions lane group g holds 16 g .. 16 g + 15 in two fragments, as it reads the codes; D = 32: 8 g ..
  // 8 g + 7 in one.
  constexpr int QG = D == 32 ? 1 : NG, QH = D == 32 ? 1 : 2;
  const int lrow = wave * 16 + i16;
  const bool live = lrow < nrows;
  const int tok = live ? (row0 + lrow) / a.H : 0;
  const int head = live ? row0 + lrow - tok * a.H : 0;
  const int rpos = live ? pos0 + tok : -1;
  const float* sink_at = a.sink + head;
  const uint16_t* qrow = a.q + (static_cast<int64_t>(item.first) + tok) * a.qst + head * a.qsh + 8 * QH * g;
  bf16x8 qf[QG][QH];
#pragma unroll
  for (int j = 0; j < QG; ++j)
#pragma unroll
    for (int h = 0; h < QH; ++h) qf[j][h] = *reinterpret_cast<const bf16x8*>(qrow + 64 * j + 8 * h);
  __builtin_amdgcn_sched_barrier(0);
  __builtin_amdgcn_s_waitcnt(vm_lgkm0(QH * QG));  // the page numbers, asked for before Q, have landed
  __builtin_amdgcn_sched_barrier(0);
  const float sink_v = *sink_at;

  uint64_t okq[AHEAD];
  Rows src;
#pragma unroll
  for (int i = 0; i < AHEAD; ++i) {
    okq[i] = 0;
    if (tbeg + i < tend) {
      int page;
      asm volatile("ds_read_b32 %0, %1\n\ts_waitcnt lgkmcnt(0)" : "=v"(page) : "v"(page_addr(tbeg + i)));
      from = froms[i];
      okq[i] = address_tile(page, within[i], src, i);
      attn_static_for<0, SH::LPT>([&](auto IC) { copy(src, ring(i), IC); });
    }
  }
  Within in_next = within[AHEAD];
  from = froms[AHEAD];

  const float rscale = a.scale_log2;  // of the scores, in log2 units
  auto sink_to_lds = [&]() __attribute__((always_inline)) {
    const uint32_t dst = lds_addr(reinterpret_cast<const char*>(&sink_lds[wave * 16 + i16]));
    asm volatile("ds_write_b32 %0, %1" ::"v"(dst), "v"(sink_v) : "memory");  // (the four lanes of a row write the same)
  };

  // ---- S^T -------------------------------------------------------------------
  // Pair n: 32 keys, 16 mb and 16 (mb + 1) on, of one group j of 64 dimensions, groups outermost.  A-fragments: key 16 mb + i16,
  // chunk 4 j + g (D = 32: half a chunk).  The codes of pair n + 1 are converted between the MFMAs of pair n, whose accumulators
  // alternate; with PAIR, where registers are short and the other workgroup fills the gaps, 16 keys' in front of their own.
  constexpr int PAIRS = QG * MB / 2, QP = PAIRS < 2 ? PAIRS : 2;
  auto qk = [&](int slot, f32x4 (&st)[MB], f32x4 (&sc)[MB], auto&& start, auto&& beside) __attribute__((always_inline)) {
    const uint32_t tile = lds_addr(ring(slot));
    const int ln = lane_now(), lg = ln >> 4, lk = ln & 15;
    uint32_t kbase[2][2];  // by mb's and j's parity
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      const int f = q_swz<D>(16 * b + lk);
      const uint32_t at = tile + lk * ROW + (D == 32 ? 16 * ((lg >> 1) ^ f) + 8 * (lg & 1) : 16 * (lg ^ (f & 3)));
      kbase[b][0] = at + 64 * (f >> 2);
      kbase[b][1] = at - 64 * (f >> 2);
    }
    const uint32_t sat = lds_addr(reinterpret_cast<const char*>(&scale_lds[wave][slot][0])) + 16 * lg;
    typedef typename std::conditional<D == 32, i32x2, i32x4>::type Codes;
    auto ask = [&](auto JC, auto BC) __attribute__((always_inline)) {  // 16 keys of a group
      constexpr int j = decltype(JC)::value, mb = decltype(BC)::value;
      if constexpr (D == 32) return ldq64<16 * ROW * mb>(kbase[mb & 1][0]);
      else return ldq<64 * j + 16 * ROW * mb>(kbase[mb & 1][j & 1]);
    };
    i32x4 s4[MB];
    auto ask_scales = [&]() __attribute__((always_inline)) {  // behind the last codes
      attn_static_for<0, MB>([&](auto BC) {
        constexpr int mb = decltype(BC)::value;
        s4[mb] = ldq<64 * mb>(sat);
      });
    };
    if constexpr (PAIR) {
      Codes k[2];
      k[0] = ask(std::integral_constant<int, 0>{}, std::integral_constant<int, 0>{});
      k[1] = ask(std::integral_constant<int, 0>{}, std::integral_constant<int, 1>{});
      start();
      static_assert(!PAIR || MB == 2, "tiles of 32 keys");
      st[0] = st[1] = f32x4{0.f, 0.f, 0.f, 0.f};
      attn_static_for<0, 2 * QG>([&](auto UC) {
        constexpr int u = decltype(UC)::value, j = u / 2, b = u % 2;
        constexpr int later = u + 1 < 2 * QG ? 1 : MB;
        lds_wait_one<later>(k[b]);
#pragma unroll
        for (int h = 0; h < QH; ++h) st[b] = mfma16x16x32<F16>(codes8<F16>(k[b][2 * h], k[b][2 * h + 1]), qf[j][h], st[b]);
        if constexpr (j + 1 < QG) k[b] = ask(std::integral_constant<int, j + 1>{}, std::integral_constant<int, b>{});
        else if constexpr (b == 0) ask_scales();
        beside(UC);
      });
    } else {
    Codes k[QP][2];
    auto issue = [&](auto NC) __attribute__((always_inline)) {  // pair n; behind the last one the scales
      constexpr int n = decltype(NC)::value, j = n / (MB / 2), b = 2 * (n % (MB / 2));
      if constexpr (n < PAIRS) {
        k[n % QP][0] = ask(std::integral_constant<int, j>{}, std::integral_constant<int, b>{});
        k[n % QP][1] = ask(std::integral_constant<int, j>{}, std::integral_constant<int, b + 1>{});
      } else if constexpr (n == PAIRS) {
        ask_scales();
      }
    };
    auto wait = [&](auto NC) __attribute__((always_inline)) {  // for pair n, where those up to n - 1 + QP have been asked for
      constexpr int n = decltype(NC)::value, last = n == 0 ? QP - 1 : n - 1 + QP;
      constexpr int later = 2 * ((last < PAIRS - 1 ? last : PAIRS - 1) - n) + (last >= PAIRS ? MB : 0);
      lds_wait_for<later>(k[n % QP][0], k[n % QP][1]);
    };
    attn_static_for<0, QP>(issue);
    start();
#pragma unroll
    for (int mb = 0; mb < MB; ++mb) st[mb] = f32x4{0.f, 0.f, 0.f, 0.f};
    bf16x8 f[QH][2];
    auto convert = [&](int slot) __attribute__((always_inline)) {
#pragma unroll
      for (int h = 0; h < QH; ++h)
#pragma unroll
        for (int b = 0; b < 2; ++b) f[h][b] = codes8<F16>(k[slot][b][2 * h], k[slot][b][2 * h + 1]);
    };
    wait(std::integral_constant<int, 0>{});
    convert(0);
    issue(std::integral_constant<int, QP>{});
    attn_static_for<0, PAIRS>([&](auto NC) {
      constexpr int n = decltype(NC)::value, j = n / (MB / 2), b0 = 2 * (n % (MB / 2));
      bf16x8 next[QH][2];
      if constexpr (n + 1 < PAIRS) wait(std::integral_constant<int, n + 1>{});
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int h = 0; h < QH; ++h)
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          st[b0 + b] = mfma16x16x32<F16>(f[h][b], qf[j][h], st[b0 + b]);
          if constexpr (n + 1 < PAIRS) next[h][b] = codes8<F16>(k[(n + 1) % QP][b][2 * h], k[(n + 1) % QP][b][2 * h + 1]);
          __builtin_amdgcn_sched_barrier(0);
        }
      if constexpr (n + 1 < PAIRS) {
        issue(std::integral_constant<int, n + 1 + QP>{});
#pragma unroll
        for (int h = 0; h < QH; ++h)
#pragma unroll
          for (int b = 0; b < 2; ++b) f[h][b] = next[h][b];
      }
      beside(NC);
    });
    }
    asm volatile("s_waitcnt lgkmcnt(0)" : "+v"(s4[0]), "+v"(s4[1]));
    if constexpr (MB == 4) asm volatile("" : "+v"(s4[MB - 2]), "+v"(s4[MB - 1]));
#pragma unroll
    for (int mb = 0; mb < MB; ++mb) sc[mb] = __builtin_bit_cast(f32x4, s4[mb]);
  };

  int all1lo = win_lo(a, pb), all1hi = nrows == M ? win_hi(a, pa) : -1;
  int all2hi = nrows == M ? ent_hi(a, pa) : -1;
  int window = a.window, cap1 = a.c1.keys, cap2 = a.c2.keys, ratio = a.ratio;
  scalar_tie(window);
  scalar_tie(cap1);
  scalar_tie(cap2);
  scalar_tie(ratio);
  auto ent_end = [&](int p) __attribute__((always_inline)) {
    return p < 0 ? 0 : min(static_cast<int>(static_cast<uint32_t>(p + 1) / static_cast<uint32_t>(ratio)), cap2);
  };
  scalar_tie(all1lo);
  scalar_tie(all1hi);
  scalar_tie(all2hi);

  // ---- softmax -----------------------------------------------------------------
  // Weights are 2^(score - m_ref), and their products with the scales go to P V.  bf16: the 16-bit kernel's references, from 2^-32
  // to 1, the products having fp32's range: scales from 2^-64 on keep those of weights down to 2^-30 of the largest, and up to 2^100
  // their sums over 2^19 keys stay finite.  fp16: 2^11 to 2^15 is where the largest product with a scale lies, so that 2^-25
  // of it keeps its 11 bits; the reference is that of the scores plus the exponents of their scales (from 2^-80 on: the weights'
  // sum stays in range).
  constexpr float kHead = F16 ? 11.0f : -32.0f, kLazy = F16 ? 4.0f : 32.0f;
  auto above = [&](float x, float scale) __attribute__((always_inline)) {  // what the reference counts of a score
    return F16 ? x + static_cast<float>(max(__builtin_amdgcn_frexp_expf(scale), -80)) : x;
  };
  float m_ref = kNever, l_run = 0.f;
  int skey = 0;
  auto softmax_begin = [&](int t, uint64_t okmask, f32x4 (&st)[MB], f32x4 (&sc)[MB], float& ref, int pbuf) __attribute__((always_inline)) {
    mfma_result_fence(st[0], st[1]);
    if constexpr (MB == 4) mfma_result_fence(st[MB - 2], st[MB - 1]);
    if (t == n1) skey = 0;
    const bool second = t >= n1;
    const bool full = (TK == 64 ? okmask == ~0ull : static_cast<uint32_t>(okmask) == ~0u) && (second ? skey <= all2hi - TK : skey >= all1lo && skey <= all1hi - TK);
    int flags = 0;
    float lmax = kNever;
    if (!full) {
      bool odd = false;
      const int end2 = second ? ent_end(rpos) : max(min(rpos + 1, cap1), 0);
      const int begin2 = second ? 0 : max(max(rpos + 1, 0) - window, 0);
      const int lo = skey - begin2, cnt = max(end2 - begin2, 0);
      const int g4 = 4 * (lane_now() >> 4);
      const uint64_t mine = okmask >> g4;
#pragma unroll
      for (int mb = 0; mb < MB; ++mb)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const bool ok = static_cast<uint32_t>(16 * mb + g4 + r + lo) < static_cast<uint32_t>(cnt) && ((mine >> (16 * mb + r)) & 1);
          odd = odd || (!ok && !(__builtin_fabsf(st[mb][r]) < __builtin_inff()));
          sc[mb][r] = ok ? sc[mb][r] : 0.f;  // (a masked key's scale may be anything)
          st[mb][r] = ok ? st[mb][r] * (sc[mb][r] * rscale) : kNever;
          lmax = __builtin_fmaxf(lmax, above(st[mb][r], sc[mb][r]));
        }
      flags = __builtin_amdgcn_ballot_w64(odd) ? kOdd : 0;
    } else {
#pragma unroll
      for (int mb = 0; mb < MB; ++mb)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          st[mb][r] = st[mb][r] * (sc[mb][r] * rscale);
          lmax = __builtin_fmaxf(lmax, above(st[mb][r], sc[mb][r]));
        }
    }
    skey = static_cast<int>(static_cast<uint32_t>(skey) + static_cast<uint32_t>(TK));
    if (__builtin_expect(__builtin_amdgcn_ballot_w64(lmax > m_ref + (kHead + kLazy)) != 0, 0)) {
      const auto r16 = __builtin_amdgcn_permlane16_swap(__float_as_uint(lmax), __float_as_uint(lmax), false, false);
      float tmax = __builtin_fmaxf(__uint_as_float(r16[0]), __uint_as_float(r16[1]));
      const SwapPair r32 = permlane32_swap(__float_as_uint(tmax), __float_as_uint(tmax));
      tmax = __builtin_fmaxf(__uint_as_float(r32.x), __uint_as_float(r32.y));
      const bool raise = tmax > m_ref + (kHead + kLazy), first = m_ref == kNever;
      const float alpha = raise && !first ? __builtin_amdgcn_exp2f(m_ref - (tmax - kHead)) : 1.0f;
      if (raise) m_ref = tmax - kHead;
      l_run *= alpha;
      const uint32_t adst = lds_addr(reinterpret_cast<const char*>(&alpha_lds[pbuf][wave * 16 + (lane_now() & 15)]));
      asm volatile("ds_write_b32 %0, %1" ::"v"(adst), "v"(alpha) : "memory");
      if (__builtin_amdgcn_ballot_w64(alpha != 1.0f)) flags |= kMoved;
    }
    ref = m_ref == kNever ? 0.f : m_ref;
    const uint32_t fdst = lds_addr(reinterpret_cast<const char*>(&flag_lds[pbuf][wave]));
    asm volatile("ds_write_b32 %0, %1" ::"v"(fdst), "v"(flags) : "memory");
  };
  auto softmax_exp = [&](int i, f32x4 (&st)[MB], float ref) __attribute__((always_inline)) {  // i of 4 MB weights
    st[i >> 2][i & 3] = __builtin_amdgcn_exp2f(st[i >> 2][i & 3] - ref);
  };
  auto softmax_end = [&](const f32x4 (&p)[MB], const f32x4 (&sc)[MB], int pbuf) __attribute__((always_inline)) {
    const int ln16 = (wave * 64 + lane_now()) * 16;
#pragma unroll
    for (int mb = 0; mb < MB; ++mb) l_run += (p[mb][0] + p[mb][1]) + (p[mb][2] + p[mb][3]);
    // P^T B-fragment of k-step s: k-slots 8g+0..3 <-> keys 32s + 4g+0..3, 8g+4..7 <-> keys 32s + 16 + 4g+0..3
#pragma unroll
    for (int s = 0; s < KSTEPS; ++s) {
      const f32x4 x = p[2 * s] * sc[2 * s], y = p[2 * s + 1] * sc[2 * s + 1];
      const u32x4 w = u32x4{pack2<F16>(x[0], x[1]), pack2<F16>(x[2], x[3]), pack2<F16>(y[0], y[1]), pack2<F16>(y[2], y[3])};
      asm volatile("ds_write_b128 %0, %1" ::"v"(lds_addr(&p_lds[pbuf][s][ln16])), "v"(w) : "memory");
    }
  };

  // ---- O^T += V^T P^T -------------------------------------------------------------
  f32x4 oacc[MBW][NB];
#pragma unroll
  for (int j = 0; j < MBW; ++j)
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) oacc[j][nb] = f32x4{0.f, 0.f, 0.f, 0.f};
  // V^T reads: source lane (g, i16) points at key 4g + (x & 3) + 16 (x >> 2), x = i16 >> 1, half i16 & 1 of chunk 4 j + wave
  constexpr int VQ0 = PAIR ? 2 : 3, VQ = VQ0 < MBW ? VQ0 : MBW;
  auto pv = [&](int slot, int pbuf, auto&& between) __attribute__((always_inline)) {
    const int ln = lane_now();
    uint32_t vbase[2];
    {
      const int x = (ln & 15) >> 1, key = 4 * (ln >> 4) + (x & 3) + 16 * (x >> 2), f = q_swz<D>(key);
      const uint32_t at = lds_addr(ring(slot)) + key * ROW + 16 * ((wave ^ (f & 3)) & (SH::CPR < 4 ? SH::CPR - 1 : 3)) + 8 * (ln & 1);
      vbase[0] = at + 64 * (f >> 2);
      vbase[1] = at - 64 * (f >> 2);
    }
    bf16x8 pf[KSTEPS][NB];
    const uint32_t psrc = lds_addr(&p_lds[pbuf][0][0]) + ln * 16;
    attn_static_for<0, KSTEPS * NB>([&](auto NC) {
      constexpr int n = decltype(NC)::value;
      pf[n / NB][n % NB] = ld128<1024 * n>(psrc);
    });
    i32x2 v[VQ][KSTEPS];
    auto issue = [&](auto JC) __attribute__((always_inline)) {
      constexpr int j = decltype(JC)::value;
      attn_static_for<0, KSTEPS>([&](auto SC) {
        constexpr int s = decltype(SC)::value;
        v[j % VQ][s] = tr_read8<64 * j + 32 * ROW * s>(vbase[j & 1]);
      });
    };
    auto wait = [&](auto JC) __attribute__((always_inline)) {  // for block j, where those up to j - 1 + VQ have been asked for
      constexpr int j = decltype(JC)::value, last = j == 0 ? VQ - 1 : j - 1 + VQ;
      constexpr int later = KSTEPS * ((last < MBW - 1 ? last : MBW - 1) - j);
      if constexpr (KSTEPS == 2) lds_wait_for<later>(v[j % VQ][0], v[j % VQ][KSTEPS - 1]);
      else lds_wait_one<later>(v[j % VQ][0]);
    };
    attn_static_for<0, VQ>(issue);
    wait(std::integral_constant<int, 0>{});
#pragma unroll
    for (int s = 0; s < KSTEPS; ++s)
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) reg_tie(pf[s][nb]);
    bf16x8 vf[KSTEPS];
    auto convert = [&](int slot) __attribute__((always_inline)) {
#pragma unroll
      for (int s = 0; s < KSTEPS; ++s) vf[s] = codes8<F16>(v[slot][s][0], v[slot][s][1]);
    };
    constexpr bool AHEAD_OF = !PAIR;  // the codes of block j + 1 are converted among the MFMAs of block j
    if constexpr (AHEAD_OF) {
      convert(0);
      if constexpr (VQ < MBW) issue(std::integral_constant<int, VQ>{});
    }
    attn_static_for<0, MBW>([&](auto JC) {
      constexpr int j = decltype(JC)::value;
      if constexpr (!AHEAD_OF) {
        if constexpr (j > 0) wait(JC);
        convert(j % VQ);
        if constexpr (j + VQ < MBW) issue(std::integral_constant<int, j + VQ>{});
      } else if constexpr (j + 1 < MBW) {
        wait(std::integral_constant<int, j + 1>{});
      }
      u32x4 next[KSTEPS];
#pragma unroll
      for (int s = 0; s < KSTEPS; ++s)
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
          oacc[j][nb] = mfma16x16x32<F16>(vf[s], pf[s][nb], oacc[j][nb]);
          if constexpr (AHEAD_OF && j + 1 < MBW) next[s][nb] = codes2<F16>(v[(j + 1) % VQ][s][nb >> 1], nb & 1);
        }
      static_assert(NB == 4, "a conversion beside each MFMA");
      if constexpr (AHEAD_OF && j + 1 + VQ < MBW) issue(std::integral_constant<int, j + 1 + VQ>{});
      between(JC);
#pragma unroll
      for (int i = 0; i < (AHEAD_OF ? KSTEPS * NB : 0); ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);  // an MFMA, then
        __builtin_amdgcn_sched_group_barrier(0x002, 3, 0);  // vector instructions
      }
      if constexpr (AHEAD_OF && j + 1 < MBW) {
#pragma unroll
        for (int s = 0; s < KSTEPS; ++s) vf[s] = __builtin_bit_cast(bf16x8, next[s]);
      }
    });
  };
  // A masked key has a score that is not finite: the tile's NaN codes become zero, in LDS, where every wave has done with its
  // scores.  The rows that see such a key have a weight of NaN for it.
  auto clean_tile = [&](int slot) __attribute__((always_inline)) {
    const uint32_t tile = lds_addr(ring(slot));
    for (int e = threadIdx.x; e < TK * SH::CPR; e += kPagedThreads) {
      u32x4 x;
      asm volatile("ds_read_b128 %0, %1\n\ts_waitcnt lgkmcnt(0)" : "=v"(x) : "v"(tile + e * 16));
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const uint32_t nan = ((x[c] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;  // bit 7 of the bytes 0x7f, 0xff
        x[c] &= ~((nan >> 7) * 0xffu);
      }
      asm volatile("ds_write_b128 %0, %1" ::"v"(tile + e * 16), "v"(x) : "memory");
    }
  };
  auto settle = [&](int flags, int pbuf, int slot) __attribute__((always_inline)) {
    if (flags & kMoved) {
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
        float al;
        int f;
        asm volatile("ds_read_b32 %0, %2\n\tds_read_b32 %1, %3\n\ts_waitcnt lgkmcnt(0)"
                     : "=&v"(al), "=&v"(f)
                     : "v"(lds_addr(reinterpret_cast<const char*>(&alpha_lds[pbuf][nb * 16 + i16]))),
                       "v"(lds_addr(reinterpret_cast<const char*>(&flag_lds[pbuf][nb]))));
        al = f & kMoved ? al : 1.0f;
#pragma unroll
        for (int j = 0; j < MBW; ++j) oacc[j][nb] = oacc[j][nb] * al;
      }
    }
    if (flags & kOdd) {
      clean_tile(slot);
      attn_tile_barrier();
    }
  };

  // ---- the tiles -------------------------------------------------------------
  // Iteration t: S^T of tile t + 1, then P V of tile t beside the softmax of tile t + 1; one barrier.  Tile t lives in slot
  // t - tbeg mod NS, its P in p_lds[t & 1].  The copies of tile t + AHEAD go out at the start, into the slot of tile t - 1.
  if (tbeg >= tend) {
    sink_to_lds();
  } else if constexpr (!PAIR) {
    skey = tbeg < n1 ? k1lo + tbeg * TK : (tbeg - n1) * TK;
    if (tbeg + AHEAD <= tend) __builtin_amdgcn_s_waitcnt(vm_lgkm0((AHEAD - 1) * (LANDED + 1)));
    else __builtin_amdgcn_s_waitcnt(vm_lgkm0(0));
    attn_tile_barrier();  // the first tile landed
    f32x4 st[MB], sc[MB];
    float ref;
    sink_to_lds();
    qk(0, st, sc, [] {}, [](auto) {});
    softmax_begin(tbeg, okq[0], st, sc, ref, tbeg & 1);
#pragma unroll
    for (int i = 0; i < 4 * MB; ++i) softmax_exp(i, st, ref);
    softmax_end(st, sc, tbeg & 1);
    int slot = 0;  // of tile t
    auto iteration = [&](int t, auto MORE, auto COPY) __attribute__((always_inline)) {
      constexpr bool more = decltype(MORE)::value, ahead = decltype(COPY)::value;
      // tile t + 1 and the page numbers of tile t + AHEAD have landed; what was issued for tile t + AHEAD - 1 behind them, its
      // scales and copies, may be in flight with three tiles ahead
      if constexpr (ahead && AHEAD == 3) __builtin_amdgcn_s_waitcnt(vm_lgkm0(LANDED + 1));
      else __builtin_amdgcn_s_waitcnt(vm_lgkm0(0));
      attn_tile_barrier();
      const int next = slot + 1 == NS ? 0 : slot + 1, last_slot = slot == 0 ? NS - 1 : slot - 1;
      int flags = 0;
      uint64_t ok_new = 0;
      char* dst = ring(last_slot);
      auto start = [&]() __attribute__((always_inline)) {
        u32x4 fl;
        int page;
        asm volatile("ds_read_b32 %0, %2\n\tds_read_b128 %1, %3\n\ts_waitcnt lgkmcnt(0)"
                     : "=&v"(page), "=&v"(fl)
                     : "v"(page_addr(t + AHEAD)), "v"(lds_addr(reinterpret_cast<const char*>(&flag_lds[t & 1][0]))));
        flags = __builtin_amdgcn_readfirstlane(static_cast<int>(fl[0] | fl[1] | fl[2] | fl[3]));
        if constexpr (ahead) {
          const Within in = in_next;
          in_next = fetch_pages();  // (past the share's end: the same page again, not used)
          ok_new = address_tile(page, in, src, last_slot);
        }
      };
      if constexpr (more) {
        qk(next, st, sc, start, [&](auto UC) {
          constexpr int u = decltype(UC)::value;
          if constexpr (ahead) attn_static_for<u * SH::LPT / PAIRS, (u + 1) * SH::LPT / PAIRS>([&](auto IC) { copy(src, dst, IC); });
        });
      } else {
        start();
      }
      if constexpr (ahead) from = from_next;
      if (__builtin_expect(flags != 0, 0)) settle(flags, t & 1, slot);
      constexpr int SPAN = MBW > 2 ? MBW - 2 : 1, EPB = (16 + SPAN - 1) / SPAN;
      pv(slot, t & 1, [&](auto JC) {
        constexpr int j = decltype(JC)::value;
        if constexpr (more) {
          if constexpr (j == 0) softmax_begin(t + 1, okq[1], st, sc, ref, (t + 1) & 1);
          if constexpr (j > 0 || MBW == 1) {
            constexpr int first = MBW == 1 ? 0 : (j - 1) * EPB;
#pragma unroll
            for (int i = first; i < first + EPB && i < 16; ++i) softmax_exp(i, st, ref);
          }
          if constexpr (j + 1 == MBW) softmax_end(st, sc, (t + 1) & 1);
        }
      });
#pragma unroll
      for (int i = 0; i + 1 < AHEAD; ++i) okq[i] = okq[i + 1];
      okq[AHEAD - 1] = ok_new;
      slot = next;
    };
    int t = tbeg;
    for (; t + AHEAD < tend; ++t) iteration(t, std::true_type{}, std::true_type{});
    for (; t + 1 < tend; ++t) iteration(t, std::true_type{}, std::false_type{});
    iteration(t, std::false_type{}, std::false_type{});
  } else {
    // PAIR: two tiles ahead, two barriers a tile.  Tile t lives in slot t - tbeg mod 3; the copies of tile t + 2 go into the
    // slot of tile t - 1.
    skey = tbeg < n1 ? k1lo + tbeg * TK : (tbeg - n1) * TK;
    sink_to_lds();
    int slot = 0;
    auto step = [&](int t, auto NEXT, auto COPY) __attribute__((always_inline)) {
      constexpr bool next = decltype(NEXT)::value, ahead = decltype(COPY)::value;
      // tile t and the page numbers of tile t + 2 have landed; the scales and copies of tile t + 1 may be in flight
      __builtin_amdgcn_s_waitcnt(vm_lgkm0(next ? LANDED + 1 : 0));
      attn_tile_barrier();  // every wave's, and every wave has left tile t - 1 and its P
      {
        f32x4 st[MB], sc[MB];
        float ref;
        qk(slot, st, sc, [] {}, [](auto) {});
        softmax_begin(t, okq[0], st, sc, ref, 0);
#pragma unroll
        for (int i = 0; i < 4 * MB; ++i) softmax_exp(i, st, ref);
        softmax_end(st, sc, 0);
      }
      okq[0] = okq[1];
      if constexpr (ahead) {
        const int last_slot = slot == 0 ? NS - 1 : slot - 1;
        int page;
        asm volatile("ds_read_b32 %0, %1\n\ts_waitcnt lgkmcnt(0)" : "=v"(page) : "v"(page_addr(t + 2)));
        const Within in = in_next;
        in_next = fetch_pages();  // (past the share's end: the same page again, not used)
        okq[1] = address_tile(page, in, src, last_slot);
        attn_static_for<0, SH::LPT>([&](auto IC) {
          copy(src, ring(last_slot), IC);
          __builtin_amdgcn_sched_barrier(0);  // (one address at a time: registers)
        });
        from = from_next;
      }
      attn_tile_barrier();  // P published
      u32x4 fl;
      asm volatile("ds_read_b128 %0, %1\n\ts_waitcnt lgkmcnt(0)" : "=v"(fl)
                   : "v"(lds_addr(reinterpret_cast<const char*>(&flag_lds[0][0]))));
      const int flags = __builtin_amdgcn_readfirstlane(static_cast<int>(fl[0] | fl[1] | fl[2] | fl[3]));
      if (__builtin_expect(flags != 0, 0)) settle(flags, 0, slot);
      pv(slot, 0, [](auto) {});
      slot = slot + 1 == NS ? 0 : slot + 1;
    };
    int t = tbeg;
    for (; t + 2 < tend; ++t) step(t, std::true_type{}, std::true_type{});
    if (t + 1 < tend) step(t++, std::true_type{}, std::false_type{});
    step(t, std::false_type{}, std::false_type{});
  }
  asm volatile("s_nop 7\n\ts_nop 7\n\ts_nop 3" ::: "memory");  // (the last MFMAs' wait states, see mfma_result_fence)

  // ---- the result ----------------------------------------------------------------
  const auto r16 = __builtin_amdgcn_permlane16_swap(__float_as_uint(l_run), __float_as_uint(l_run), false, false);
  float l_tot = __uint_as_float(r16[0]) + __uint_as_float(r16[1]);
  const SwapPair r32 = permlane32_swap(__float_as_uint(l_tot), __float_as_uint(l_tot));
  l_tot = __uint_as_float(r32.x) + __uint_as_float(r32.y);
  const int64_t flat0 = static_cast<int64_t>(item.first) * a.H + row0;  // first row of o
  if (shares > 1) {
    const int64_t slot = item.slot;
    if (g == 0) a.part_ml[slot * M + wave * 16 + i16] = float2{m_ref, l_tot};
    float* po = a.part_o + slot * M * D;
#pragma unroll
    for (int j = 0; j < MBW; ++j) {
      const int mbi = j * kAttnWaves + wave;
      if (SH::MBT % kAttnWaves == 0 || mbi < SH::MBT) {
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
          if (nb * 16 < nrows) *reinterpret_cast<f32x4*>(po + ((nb * SH::MBT + mbi) * 64 + lane) * 4) = oacc[j][nb];
      }
    }
    if (share == 0 && threadIdx.x == 0) {
      int32_t* rec = a.rec + 4 + 4 * static_cast<int64_t>(item.rec);
      *reinterpret_cast<int4*>(rec) = int4{static_cast<int>(slot), shares, static_cast<int>(flat0), nrows};
    }
    return;
  }
  float* out_scale = alpha_lds[0];
  __syncthreads();  // every wave has left the last tile and its alpha
  const float sink = sink_lds[lrow];
  const float sink2 = sink_log2(sink);
  const float m_fin = __builtin_fmaxf(m_ref, sink2);
  const float top = m_fin == kNever ? 0.f : m_fin;
  const float resc = __builtin_amdgcn_exp2f(m_ref - top), keys = l_tot * resc;
  const float l_fin = keys + __builtin_amdgcn_exp2f(sink2 - top);
  if (g == 0) {
    out_scale[lrow] = keys == 0.f ? 0.f : resc / l_fin;
    if (live) a.lse[flat0 + lrow] = keys == 0.f ? lse_of_sink(sink) : (__builtin_amdgcn_logf(l_fin) + top) * kLn2;
  }
  __syncthreads();  // scales published
  // staged in the tiles' LDS, then written in one piece: the rows follow each other in o
  char* obase = reinterpret_cast<char*>(a.o + flat0 * D);
#pragma unroll
  for (int part = 0; part < PARTS; ++part) {
    constexpr int R = M / PARTS;  // rows of a part
    if (part > 0) {
      if (part * R >= nrows) return;
      __syncthreads();  // the part before has been read
    }
#pragma unroll
    for (int nb = part * (NB / PARTS); nb < (part + 1) * (NB / PARTS); ++nb) {
      const float osc = out_scale[nb * 16 + i16];
#pragma unroll
      for (int j = 0; j < MBW; ++j) {
        const int mbi = j * kAttnWaves + wave;
        if (SH::MBT % kAttnWaves == 0 || mbi < SH::MBT) {
          const f32x4 v = oacc[j][nb] * osc;
          uint2 w;
          w.x = pack2<F16>(v[0], v[1]);
          w.y = pack2<F16>(v[2], v[3]);
          *reinterpret_cast<uint2*>(kv_lds + kv_off<D>(nb * 16 + i16 - part * R, 2 * mbi + (g >> 1)) + 8 * (g & 1)) = w;
        }
      }
    }
    __syncthreads();
    for (int e = threadIdx.x; e < min(nrows - part * R, R) * (D / 8); e += kPagedThreads)
      *reinterpret_cast<u32x4*>(obase + static_cast<int64_t>(e + part * R * (D / 8)) * 16) =
          *reinterpret_cast<const u32x4*>(kv_lds + kv_off<D>(e / (D / 8), e % (D / 8)));
  }
}

// Row blocks from which PAIR is taken: where two workgroups a CU have work.  PAIR / not, D = 576: 64 heads, five chunks of 300 to 4,096
// tokens, window 128 and compressed entries (5 to 17 tiles a row block) 495 / 603 us; 1,024 new tokens behind 8,192 (1,024 row blocks,
// 144 tiles) 1,560 / 1,561; D = 512 the same 1,308 / 1,425; of few row blocks, 32 single tokens behind 20,000 keys 168 / 144, 64 behind
// 40,000 with a window and compressed entries 41 / 30.  Fewer dimensions have two workgroups a CU and more without it: D = 256
// (2,048 row blocks) 1,607 / 1,290, 128 1,017 / 785.
constexpr int64_t q_pair_from(int64_t D) { return D >= 512 ? 257 : INT64_MAX; }

// Sizes of a call, from what the host knows.
struct PagedQSizes {
  bool pair;             // the kernel with PAIR
  int64_t blocks;        // row blocks of a workgroup at most
  int64_t want;          // workgroups that run at once
  int64_t grid;          // workgroups
  int64_t items;         // partial outputs at most, 0: no row block is split
  int64_t split_blocks;  // split row blocks at most
  int64_t bytes;         // scratch
  int behind;            // tokens of a row block before its last one at most
};
static PagedQSizes q_sizes(int64_t N, int64_t H, int64_t D, int64_t R, int64_t window, int64_t keys1, int64_t keys2) {
  PagedQSizes p{};
  const int64_t M = kRows;
  // a request's last row block is part empty unless M divides n H
  int64_t g = M;
  while (H % g) g /= 2;
  p.blocks = (N * H + (R < N ? R : N) * (M - g)) / M;
  p.pair = p.blocks >= q_pair_from(D);
  const int64_t want = p.want = 256 * q_per_cu(static_cast<int>(D), p.pair), tile = p.pair ? 32 : 64;
  p.grid = 2 * p.blocks <= want ? want : p.blocks + want;
  const int64_t span = M / H + 1 + window;
  p.behind = static_cast<int>((M - 1 + H - g) / H);  // (a row block begins at any multiple of g heads of a token)
  const int64_t tiles = ((window < keys1 && span < keys1 ? span : keys1) + tile - 1) / tile + (keys2 + tile - 1) / tile;
  // Where no cut can win back the second launch that joins the shares, none is made.
  if (tiles <= (D >= 512 ? 8 : 14) + p.blocks / 8) {
    p.grid = p.blocks;
    return p;
  }
  p.items = 2 * want;
  const int64_t each = p.blocks * ((tiles + kLeastTiles - 1) / kLeastTiles);
  if (each < p.items) p.items = each;
  p.split_blocks = p.items / 2;
  if (p.blocks < p.split_blocks) p.split_blocks = p.blocks;
  if (2 * p.blocks <= want && each < p.grid) p.grid = each;
  p.bytes = p.items * M * (D * 4 + 8) + 16 * (p.split_blocks + 1);
  return p;
}

template <int D>
static int launch_paged_attn_q(bool f16, const PagedAttnQArgs& a, const PagedQSizes& p, hipStream_t st) {
  const int64_t most = 0xffffffffLL / kPagedThreads;  // (a launch has fewer than 2^32 threads)
  if (p.grid + 7 > most) return set_error(SI_ERR_UNSUPPORTED, "too many rows for one launch");
  // (whole rounds of the XCDs: see paged_item_number)
  const dim3 grid(static_cast<unsigned>(((p.grid < 1 ? 1 : p.grid) + 7) & ~int64_t{7})), block(kPagedThreads);
  auto launch = [&](auto F16) {
    constexpr bool half = decltype(F16)::value;
    if constexpr (q_pair_from(D) < INT64_MAX) {
      if (p.pair) {
        hipLaunchKernelGGL((paged_attn_q_kernel<D, half, true>), grid, block, 0, st, a);
        return;
      }
    }
    hipLaunchKernelGGL((paged_attn_q_kernel<D, half, false>), grid, block, 0, st, a);
  };
  if (f16) launch(std::true_type{});
  else launch(std::false_type{});
  const int rc = check_launch("paged_attn_q_kernel");
  if (rc || !a.a.part_o) return rc;
  return launch_paged_combine(f16, a.a, D, p.split_blocks, st);
}

static int set_scales(QScales& s, const float* scales, int64_t stride, int64_t block, int64_t pages, int64_t ps, int64_t P,
                      const char* name) {
  const std::string n(name);
  if (block <= 0 || ps % block) return set_error(SI_ERR_INVALID, n + ": the block must divide the page size");
  if (stride < 0) return set_error(SI_ERR_INVALID, n + ": negative scale stride");
  if (pages > 0 && P > 0 && !scales) return set_error(SI_ERR_INVALID, n + ": null scales");
  s.base = scales;
  s.pstride = stride;
  s.per_page = static_cast<uint32_t>(ps / block);
  s.magic = 0;
  s.shift = 0;
  s.one = block == 1 ? ~0u : 0u;
  if (block > 1) {  // as in set_paged_cache
    int l = 1;
    while ((int64_t{1} << l) < block) ++l;
    s.magic = static_cast<uint32_t>(((uint64_t{1} << (31 + l)) + static_cast<uint64_t>(block) - 1) / static_cast<uint64_t>(block));
    s.shift = static_cast<uint32_t>(l - 1);
  }
  return SI_OK;
}

}  // namespace si

using namespace si;

extern "C" int64_t si_paged_attn_q_fwd_scratch_bytes(int64_t N, int64_t H, int64_t D, int64_t R, int64_t window, int64_t keys,
                                                     int64_t keys2) {
  const int64_t lim = 0x7fffffff;
  if (N <= 0 || H <= 0 || R <= 0 || window < 0 || keys < 0 || keys2 < 0 || !paged_attn_served(D) || N > lim || H > lim ||
      N * H > lim || R > lim)
    return 0;
  return q_sizes(N, H, D, R, window == 0 || window > lim ? lim : window, keys < lim ? keys : lim,
                 keys2 < lim ? keys2 : lim).bytes;
}

extern "C" int si_paged_attn_q_fwd(const void* q, const int64_t* q_strides, const void* kv, const int64_t* kv_strides,
                                   const float* scales, int64_t scale_stride, int64_t block, int64_t pages, int64_t page_size,
                                   const int32_t* block_table, int64_t table_stride, int64_t P, const void* kv2,
                                   const int64_t* kv2_strides, const float* scales2, int64_t scale_stride2, int64_t block2,
                                   int64_t pages2, int64_t page_size2, const int32_t* block_table2, int64_t table_stride2,
                                   int64_t P2, int64_t window, int64_t ratio, const int32_t* cu_q, const int32_t* seq_lens,
                                   const float* attn_sink, int64_t N, int64_t H, int64_t D, int64_t R, float softmax_scale,
                                   int qkv_dtype, void* o, float* lse, void* scratch, int64_t scratch_bytes, void* stream) {
  if (qkv_dtype != SI_DTYPE_BF16 && qkv_dtype != SI_DTYPE_F16)
    return set_error(SI_ERR_INVALID, "qkv_dtype must be SI_DTYPE_BF16 (0) or SI_DTYPE_F16 (1)");
  if (N < 0 || H <= 0 || D <= 0 || R < 0 || window < 0 || ratio < 0) return set_error(SI_ERR_INVALID, "bad dimension");
  if (!paged_attn_served(D))
    return set_error(SI_ERR_UNSUPPORTED,
                     "unsupported head dim D=" + std::to_string(D) + " (supported: 32, 64, 128, 256, 512, 576)");
  if (N > 0x7fffffff || H > 0x7fffffff || R > 0x7fffffff || N * H > 0x7fffffff || ratio > 0x7fffffff)
    return set_error(SI_ERR_UNSUPPORTED, "dimension exceeds int32");
  // (a thread's share of the requests ends within 31 bits)
  if (R > int64_t{1} << 30) return set_error(SI_ERR_UNSUPPORTED, "more than 2^30 requests");
  if (!q_strides) return set_error(SI_ERR_INVALID, "null stride argument");
  if (N > 0 && (!q || !attn_sink || !o || !lse || !cu_q || (R > 0 && !seq_lens)))
    return set_error(SI_ERR_INVALID, "null pointer argument");
  if (q_strides[2] != 1 || (q_strides[0] | q_strides[1]) % 8)
    return set_error(SI_ERR_INVALID, "q needs a contiguous last dimension and strides that are multiples of 8 elements");
  if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(o) | reinterpret_cast<uintptr_t>(scratch)) & 15)
    return set_error(SI_ERR_INVALID, "q, o and scratch must be 16-byte aligned");
  PagedAttnQArgs x{};
  PagedAttnArgs& a = x.a;
  int rc = set_paged_cache(a.c1, 1, kv, kv_strides, pages, page_size, D, block_table, table_stride, P, R, "kv");
  if (!rc) rc = set_scales(x.s1, scales, scale_stride, block, pages, page_size, R > 0 ? P : 0, "kv");
  if (!rc && ratio > 0) {
    rc = set_paged_cache(a.c2, 1, kv2, kv2_strides, pages2, page_size2, D, block_table2, table_stride2, P2, R, "kv2");
    if (!rc) rc = set_scales(x.s2, scales2, scale_stride2, block2, pages2, page_size2, R > 0 ? P2 : 0, "kv2");
  }
  if (rc || N == 0) return rc;
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
  const bool f16 = qkv_dtype == SI_DTYPE_F16;
  PagedQSizes p = q_sizes(N, H, D, R > 0 ? R : 1, a.window, paged_cache_keys(pages, P, page_size),
                          ratio > 0 ? paged_cache_keys(pages2, P2, page_size2) : 0);
  a.want = static_cast<int>(p.want);
  a.behind = p.behind;
  a.part_cost = static_cast<float>(N * H) / (24.f * kRows * static_cast<float>(p.blocks));
  if (p.bytes > 0 && scratch && scratch_bytes >= p.bytes) {
    const int64_t M = kRows;
    a.part_o = static_cast<float*>(scratch);
    a.part_ml = reinterpret_cast<float2*>(a.part_o + p.items * M * D);
    a.rec = reinterpret_cast<int32_t*>(a.part_ml + p.items * M);
  } else {
    p.grid = p.blocks;
  }
  hipStream_t st = static_cast<hipStream_t>(stream);
  switch (D) {
    case 32: return launch_paged_attn_q<32>(f16, x, p, st);
    case 64: return launch_paged_attn_q<64>(f16, x, p, st);
    case 128: return launch_paged_attn_q<128>(f16, x, p, st);
    case 256: return launch_paged_attn_q<256>(f16, x, p, st);
    case 512: return launch_paged_attn_q<512>(f16, x, p, st);
    default: return launch_paged_attn_q<576>(f16, x, p, st);
  }
}
