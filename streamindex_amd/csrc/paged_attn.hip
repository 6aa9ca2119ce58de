// Kernels of the paged attention (formulas in paged_attn.h).
//
// A workgroup of four waves takes 64 rows, a row being one head of one token: with 64 heads one token, with 16 heads
// four neighbouring tokens, so every key row that is fetched serves 64 query rows whatever the head count.  It walks
// the keys that any of its rows sees, 32 at a time, the window's first:
//   * the tile's rows are copied from their pages straight into LDS (global_load_lds, 16 bytes a lane, no staging
//     registers), the page numbers fetched a tile before their copies;
//   * S^T = K Q^T on 16x16x32 MFMAs, keys on M: wave w takes rows 16w .. 16w+15, Q^T stays in registers;
//   * the online softmax is in-lane (a lane holds eight keys of one row) plus two lane exchanges when a maximum moves,
//     which it does only once a weight exceeds the first by 2^32 (fp16: 2^4), so the accumulator is rarely rescaled;
//   * P^T goes through LDS, and O^T += V^T P^T with the output dimensions dealt to the waves.
// P is rounded to the element type for the matrix core, the denominator sums the unrounded values in fp32.
//
// Two ways through the tiles.  With four tiles in LDS (one workgroup a CU at D >= 512, two at 256, three at 128, four
// below), the softmax of tile t + 1 runs among the MFMAs of tile t's P V, its copies three tiles ahead, one barrier a tile.
// PAIR: two tiles in LDS, a tile's steps one after the other, one workgroup more a CU, whose copies, prologues and ends
// fall behind each other's MFMAs: for many row blocks, from D = 128 on (pair_from below).
//
// Bound, long keys: the LDS, which every K tile leaves four times (each wave's S^T) and once more as V, beside its copy: one
// request of 8,192 earlier tokens, 64 heads, 1,024 new ones at D = 576 1,130 TFLOP/s, at 512 1,055, 2,048 at 256 941, at 128 714,
// 4,096 at 64 616, where a library product reaches 1,279 (below 256 the softmax's vector work weighs more).  Few keys a row:
// Q in, O out and the prologue.
//
// A key that only some of the 64 rows see is masked for the others by a weight of zero; the matrix core would still
// turn 0 x inf into NaN.  Keys and values being the same rows, such a value makes the key's raw score non-finite as
// well, so on a masked non-finite score the tile's values that are not finite are zeroed in LDS before P V; a row that
// does see such a key gets a weight of NaN there, and with it its output.  A score of -inf from finite values, a key of the
// type's lowest ones say, is a weight of zero.
//
// Few rows over many keys: each workgroup works out from the requests' lengths how many shares a row block's tiles are
// cut into (Schedule below) and which share is its own; shares leave fp32 partial outputs that a second kernel joins.
// Nothing of the lengths is read on the host.
#include <cstdint>
#include <string>
#include <type_traits>

#include "paged_attn_sched.h"
#include "si_status.h"

namespace si {

// Resident workgroups of a CU: LDS sets them, and Q^T and O^T take 216 registers of a wave at D = 576, 96 at D = 256.
constexpr int per_cu(int D, bool PAIR) { return (D >= 512 ? 1 : D == 256 ? 2 : D == 128 ? 3 : 4) + (PAIR ? 1 : 0); }
// Row blocks from which PAIR is taken (us, PAIR and not, rows of 250 to 290 tiles and of 12: D = 576, 256 row blocks 330 and 346,
// 66 and 33, 320 of them 549 and 661, 44 and 57, 1,024 1,171 and 1,411, 84 and 109; D = 256, 1,024 689 and 650, 46 and 46, 1,536
// 933 and 982, 58 and 65, 4,096 2,755 and 2,926, 144 and 162; D = 128, 1,536 653 and 644, 41 and 43, 2,048 842 and 877, 50 and
// 54; D = 64, 4,096 1,150 and 1,113, 63 and 67).
constexpr int64_t pair_from(int64_t D) { return D >= 512 ? 257 : D == 256 ? 1025 : D == 128 ? 1537 : INT64_MAX; }

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

// PAIR: the steps of a tile one after the other, for one workgroup more on a CU.
template <int D, bool F16, bool PAIR>
__global__ __launch_bounds__(kPagedThreads, per_cu(D, PAIR)) void paged_attn_kernel(PagedAttnArgs a) {
  using SH = AttnShape<D>;
  constexpr int KS = SH::KS, MBW = SH::MBW, ROW = SH::ROW;
  constexpr int M = kRows, NB = M / 16;             // rows of the workgroup, and blocks of 16
  constexpr int NS = PAIR ? 2 : 4, AHEAD = NS - 1;  // tiles in LDS, and copied ahead of P V
  constexpr int NP = PAIR ? 1 : 2, PAGES = PAIR ? 2 : 4;  // P's and page numbers' buffers
  constexpr float kLn2 = 0.6931471805599453f;
  static_assert(NS * SH::TILE >= M * ROW, "the output is staged in the tiles' LDS");
  __shared__ __attribute__((aligned(16))) char kv_lds[NS * SH::TILE];
  __shared__ __attribute__((aligned(16))) char p_lds[NP][NB * 64 * 16];
  __shared__ __attribute__((aligned(16))) float alpha_lds[NP][M];
  __shared__ float sink_lds[M];  // of each row, for the end
  __shared__ __attribute__((aligned(16))) int flag_lds[NP][4];  // kOdd, kMoved of this tile, by wave
  __shared__ __attribute__((aligned(16))) int page_lds[kAttnWaves][PAGES][64];  // page numbers of the next tiles, by wave

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  __builtin_assume(wave >= 0 && wave < 4);
  const int g = lane >> 4, i16 = lane & 15;
  // rows [begin, end) are the requests'
  int begin = a.R > 0 ? min(max(a.cu[0], 0), a.N) : 0, end = a.R > 0 ? min(max(a.cu[a.R], 0), a.N) : 0;
  PagedItem item;
  bool down;
  const bool work = a.R <= kWave ? paged_schedule_wave<kAttnTK>(a, item, down) : paged_schedule<kAttnTK>(a, item, down);
  if (down) begin = end = 0;
  // Rows of no request: as a row without a key.
  for (int64_t i = blockIdx.x; i < begin + static_cast<int64_t>(a.N - end); i += gridDim.x) {
    const int64_t t = i < begin ? i : end + i - begin;
    u32x4* orow = reinterpret_cast<u32x4*>(a.o + t * a.H * D);
    for (int64_t e = threadIdx.x; e < static_cast<int64_t>(a.H) * SH::CPR; e += kPagedThreads) orow[e] = u32x4{0, 0, 0, 0};
    for (int h = threadIdx.x; h < a.H; h += kPagedThreads) {
      a.lse[t * a.H + h] = lse_of_sink(a.sink[h]);
    }
  }
  if (!work) return;

  // (scalars from here on: as the vector registers they come in they would stay there to the end)
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
  // tiles of this row block: the window's, then the second cache's; and this share of them
  const int k1lo = win_lo(a, pa), k1hi = win_hi(a, pb);
  const int k2hi = ent_hi(a, pb);
  const int n1 = k1hi > k1lo ? key_tiles<kAttnTK>(k1hi - k1lo) : 0;
  const int ntiles = n1 + key_tiles<kAttnTK>(k2hi);
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
  // Lanes l and l + 32 resolve key l of a tile; a key past the tile's last one stands in for by that one (it is masked,
  // and a tile always has a first key).  A key without a page reads row 0 of the cache and is masked.  Each wave fetches
  // the page numbers for its own copies into LDS (as registers they would make the compiler wait for every copy in
  // flight before their use), a tile ahead of the copies; `within` is what the key's place in its page adds.  What
  // a tile asks of its cache is held in scalars that every path sets: as vector registers, which a value that only some
  // paths set becomes, they were spilled and read back between a tile's steps, with a wait for its copies each time
  // (7,149 row blocks of up to 17 tiles, D = 576: 540 us, 476 without).  Five registers are still
  // spilled with PAIR at D = 576: four are read back in a rescale of the accumulator only, one behind the last tile.
  CacheView view1, view2;
  CacheBase base1, base2;
  view_cache(a.c1, req, view1, base1);
  view_cache(a.c2, req, view2, base2);
  CacheView view;            // of the next tile to fetch page numbers for
  CacheBase from, from_next; // of the tile to copy, and of the one after it
  uint32_t fkey = 0, fend = 0;  // (unsigned: a tile past the last key of 2^31 - 1 begins behind 31 bits)
  int ftile = tbeg;
  auto enter = [&](int t) __attribute__((always_inline)) {  // moves the view to tile t
    const bool second = t >= n1;
    view = CacheView{pick(second, view1.table, view2.table), pick(second, view1.ps, view2.ps),
                     pick(second, view1.rstride, view2.rstride), pick(second, view1.magic, view2.magic),
                     pick(second, view1.shift, view2.shift), pick(second, view1.one, view2.one)};
    from_next = CacheBase{pick(second, base1.base, base2.base), pick(second, base1.pstride, base2.pstride),
                          pick(second, base1.pages, base2.pages)};
    fkey = second ? static_cast<uint32_t>(t - n1) * 32u : static_cast<uint32_t>(k1lo) + static_cast<uint32_t>(t) * 32u;
    fend = static_cast<uint32_t>(second ? k2hi : k1hi);
    scalar_tie(view.table);
    scalar_tie(view.ps);
    scalar_tie(view.rstride);
    scalar_tie(view.magic);
    scalar_tie(view.shift);
    scalar_tie(view.one);
    scalar_tie(from_next.base);
    scalar_tie(from_next.pstride);
    scalar_tie(from_next.pages);
    scalar_tie(fkey);
    scalar_tie(fend);
  };
  auto fetch_pages = [&]() __attribute__((always_inline)) {
    if (__builtin_expect(ftile == n1, 0) && ntiles > n1) enter(n1);
    const uint32_t key = min(fkey + static_cast<uint32_t>(lane_now() & 31), fend - 1);
    const uint32_t col = view.page_of(key);
    __builtin_amdgcn_global_load_lds(reinterpret_cast<const uint32_t*>(view.table + col),
                                     (lds_void_t*)&page_lds[wave][ftile % PAGES][0], 4, 0, 0);
    ++ftile;
    fkey += 32;
    return (key - col * view.ps) * view.rstride;
  };
  // A tile's copies, LPT of a wave.  At D >= 256 wave w copies keys 8w .. 8w + 7, 64 chunks of 16 bytes at a time: copy i
  // holds the end of key A(i) and, from lane B(i) on, the start of the next, so the two rows are scalars; the swizzle of key
  // 8w + j is j.  Below, a copy spans more keys and each lane gets its row by a lane exchange; copies go over the waves.
  constexpr bool BY_WAVE = D >= 256;
  constexpr int FSWZ = SH::FMASK;
  constexpr int CPR = SH::CPR, LPT = SH::LPT;
  static_assert(!BY_WAVE || LPT * 64 == 8 * CPR, "a wave's copies are its eight rows");
  struct Sources {
    uint32_t row[LPT < 8 ? 8 : LPT];  // rows of the wave's keys, or of this lane's copies, in 16-byte units
  };
  // Sources of the tile whose page numbers are `page`; returns which of its keys have a page.
  auto address_tile = [&](int page, uint32_t within, Sources& y) __attribute__((always_inline)) {
    const bool ok = static_cast<uint32_t>(page) < from.pages;
    const uint32_t row = ok ? static_cast<uint32_t>(page) * from.pstride + within : 0u;
    if constexpr (BY_WAVE) {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        y.row[j] = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(row), wave * 8 + j));
    } else {
#pragma unroll
      for (int i = 0; i < LPT; ++i)
        y.row[i] = static_cast<uint32_t>(__builtin_amdgcn_ds_bpermute(
            ((i * SH::NT + wave * 64 + lane_now()) / CPR & 31) * 4, static_cast<int>(row)));
    }
    return static_cast<uint32_t>(__builtin_amdgcn_ballot_w64(ok));
  };
  auto copy = [&](const Sources& y, char* tile, auto IC) __attribute__((always_inline)) {
    constexpr int i = decltype(IC)::value;
    uint32_t src;
    char* dst;
    if constexpr (BY_WAVE) {
      constexpr int A = 64 * i / CPR, OFF = 64 * i - CPR * A, B = CPR - OFF;  // lanes [0, B): key A, the others the next
      const int ln = lane_now();
      if constexpr (B >= 64) {
        src = y.row[A] + static_cast<uint32_t>((ln + OFF) ^ (FSWZ & A));
      } else {
        const uint32_t one = y.row[A] + static_cast<uint32_t>((ln + OFF) ^ (FSWZ & A));
        const uint32_t two = y.row[A + 1 < 8 ? A + 1 : 7] + static_cast<uint32_t>((ln - B) ^ (FSWZ & (A + 1)));
        src = ln < B ? one : two;
      }
      dst = tile + wave * (LPT * 1024) + i * 1024;
    } else {
      const int e = i * SH::NT + wave * 64 + lane_now();
      src = y.row[i] + static_cast<uint32_t>((e % CPR) ^ kv_swz<D>(e / CPR));
      dst = tile + wave * 1024 + i * (SH::NT * 16);
    }
    if (BY_WAVE || SH::CH % SH::NT == 0 || i + 1 < LPT || i * SH::NT + wave * 64 < SH::CH)
      __builtin_amdgcn_global_load_lds(reinterpret_cast<const uint16_t*>(from.base + (static_cast<uint64_t>(src) << 4)),
                                       (lds_void_t*)dst, 16, 0, 0);
  };
  auto ring = [&](int slot) __attribute__((always_inline)) { return kv_lds + slot * SH::TILE; };
  auto page_addr = [&](int t) __attribute__((always_inline)) {
    return lds_addr(reinterpret_cast<const char*>(&page_lds[wave][t % PAGES][0])) + lane_now() * 4;
  };
  // (the first tiles' page numbers are on their way while Q is addressed; tiles past the share's end are not used)
  uint32_t within[AHEAD + 1];
  CacheBase froms[AHEAD + 1];
  enter(tbeg);
#pragma unroll
  for (int i = 0; i <= AHEAD; ++i) {
    within[i] = 0;
    if (tbeg + i < tend) within[i] = fetch_pages();
    froms[i] = from_next;
  }

  __builtin_amdgcn_sched_barrier(0);

  // ---- this lane's row: its Q^T fragment and the keys it sees ----------------
  bf16x8 qf[KS];
  const int lrow = wave * 16 + i16;
  const bool live = lrow < nrows;
  const int tok = live ? (row0 + lrow) / a.H : 0;
  const int head = live ? row0 + lrow - tok * a.H : 0;
  const int rpos = live ? pos0 + tok : -1;  // position, -1: no row
  const float* sink_at = a.sink + head;
  // (a row past the block's last one reads the first one's Q; nothing of it is used)
  const uint16_t* qrow = a.q + (static_cast<int64_t>(item.first) + tok) * a.qst + head * a.qsh;
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) qf[ks] = *reinterpret_cast<const bf16x8*>(qrow + ks * 32 + g * 8);
  // The page numbers, asked for before these KS loads, have landed; the loads may be in flight.  (The loads return in
  // order; the scheduling barriers keep them between the page numbers and the wait.)
  __builtin_amdgcn_sched_barrier(0);
  __builtin_amdgcn_s_waitcnt(vm_lgkm0(KS));
  __builtin_amdgcn_sched_barrier(0);
  // Sinks, kept in LDS for the end (each row's is read back by the lane that wrote it).
  const float sink_v = *sink_at;
  auto sink_to_lds = [&]() __attribute__((always_inline)) {
    const uint32_t dst = lds_addr(reinterpret_cast<const char*>(&sink_lds[wave * 16 + i16]));
    asm volatile("ds_write_b32 %0, %1" ::"v"(dst), "v"(sink_v) : "memory");  // (the four lanes of a row write the same)
  };

  // ---- S^T -------------------------------------------------------------------
  // A-fragment addresses: key 16mb + i16, chunk 4ks + g; with f = kv_swz(i16), (4ks + g) ^ f = 4 (ks ^ (f >> 2)) +
  // (g ^ (f & 3)), so the offset is a per-lane base (one per parity of ks) plus 64 ks + 16 ROW mb.
  constexpr int QPD0 = PAIR ? 2 : 4, QPD = KS < QPD0 ? KS : QPD0;
  // start() runs behind the first fragments' reads, beside(ks) among the MFMAs of k-step ks.
  auto scale_q = [&]() __attribute__((always_inline)) {  // (scale is positive below)
    if (__builtin_expect(a.scale_log2 <= 0.f, 0)) {
      const uint32_t keep = a.scale_log2 == 0.f ? 0u : ~0u, flip = a.scale_log2 == 0.f ? 0u : 0x80008000u;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
          qf[ks] = __builtin_bit_cast(bf16x8, (__builtin_bit_cast(u32x4, qf[ks]) & keep) ^ flip);
    }
  };
  auto qk = [&](int slot, f32x4 (&st)[2], auto&& start, auto&& beside) __attribute__((always_inline)) {
    const int ln = lane_now(), key = ln & 15, f = kv_swz<D>(key);
    const uint32_t at = lds_addr(ring(slot)) + key * ROW + 16 * ((ln >> 4) ^ (f & 3));
    const uint32_t qa_e = at + 64 * (f >> 2), qa_o = at - 64 * (f >> 2);
    bf16x8 kq[QPD][2];
    auto issue = [&](auto KC) __attribute__((always_inline)) {
      constexpr int ks = decltype(KC)::value;
      const uint32_t base = (ks & 1) ? qa_o : qa_e;
      kq[ks % QPD][0] = ld128<64 * ks>(base);
      kq[ks % QPD][1] = ld128<64 * ks + 16 * ROW>(base);
    };
    attn_static_for<0, QPD>(issue);
    start();
    st[0] = st[1] = f32x4{0.f, 0.f, 0.f, 0.f};
    attn_static_for<0, KS>([&](auto KC) {
      constexpr int ks = decltype(KC)::value;
      constexpr int later = (KS - 1 - ks) < (QPD - 1) ? (KS - 1 - ks) : (QPD - 1);
      lds_wait<2 * later>(kq[ks % QPD][0], kq[ks % QPD][1]);
      st[0] = mfma16x16x32<F16>(kq[ks % QPD][0], qf[ks], st[0]);
      st[1] = mfma16x16x32<F16>(kq[ks % QPD][1], qf[ks], st[1]);
      if constexpr (ks + QPD < KS) issue(std::integral_constant<int, ks + QPD>{});
      beside(KC);
    });
  };

  // Keys that every row sees: [all1lo, all1hi) of the first cache, [0, all2hi) of the second; none where rows are missing.
  int all1lo = win_lo(a, pb), all1hi = nrows == M ? win_hi(a, pa) : -1;
  int all2hi = nrows == M ? ent_hi(a, pa) : -1;
  float scale = a.scale_log2 == 0.f ? 1.0f : __builtin_fabsf(a.scale_log2);
  // (what masks need of the arguments, kept out of the loop as scalar loads)
  int window = a.window, cap1 = a.c1.keys, cap2 = a.c2.keys, ratio = a.ratio;
  scalar_tie(window);
  scalar_tie(cap1);
  scalar_tie(cap2);
  scalar_tie(ratio);
  auto ent_end = [&](int p) __attribute__((always_inline)) {  // as ent_hi; only tiles of the second cache ask
    return p < 0 ? 0 : min(static_cast<int>(static_cast<uint32_t>(p + 1) / static_cast<uint32_t>(ratio)), cap2);
  };
  scalar_tie(all1lo);
  scalar_tie(all1hi);
  scalar_tie(all2hi);
  scalar_tie(scale);

  // ---- softmax -----------------------------------------------------------------
  // In steps that run among the MFMAs of the tile before: scores to log2 units and masks, a new reference maximum where one
  // is due; the weights one by one; their sum and their place in LDS.
  // (scale is positive: a negative one has changed the sign of Q, zero has made Q zero)
  // Weights are 2^(score - m_ref), with m_ref kHead below the row's maximum when it is set: P begins at 2^kHead, and the
  // reference moves when a weight would pass 2^(kHead + kLazy).
  // fp16's normal numbers reach from 2^-14 to 2^15, so a weight of 2^-25 of the largest keeps its 11 bits (with P from 1 to 2^8
  // it was zero in the numerator, 2.6 % of the mass of 2^20 such keys).
  // bf16 has fp32's range: P begins at 2^-32 and never passes 1, so the reference is no lower than the largest weight, whose
  // distance from a sink far above is then in range if the weight is (with P from 1 to 2^64, scores of -90 and -47 beside a sink
  // of 0 gave zero); values below 2^-94 lose bits for it.
  // (us, 131,072 rows over 9,000 keys, D = 128, scores of deviation 1 and 8: fp16 841, 869 with P from 1 to 2^8, 846, 889 now;
  // bf16 831, 833 with P from 1 to 2^64, 837, 840 now, 836, 863 from 2^-16.)
  constexpr float kHead = F16 ? 11.0f : -32.0f, kLazy = F16 ? 4.0f : 32.0f;
  float m_ref = kNever, l_run = 0.f;  // reference (log2 domain) and this lane's share of the denominator
  int skey = 0;  // first key of the next tile to mask
  // This lane's row sees key kk of the tile that begins at key `first` where kk + lo, unsigned, is below cnt.
  auto seen_keys = [&](bool second, int first, int& lo, int& cnt) __attribute__((always_inline)) {
    const int end = second ? ent_end(rpos) : max(min(rpos + 1, cap1), 0);
    const int begin = second ? 0 : max(max(rpos + 1, 0) - window, 0);
    lo = first - begin;
    cnt = max(end - begin, 0);
  };
  auto softmax_begin = [&](int t, uint32_t okmask, f32x4 (&st)[2], float& ref, int pbuf) __attribute__((always_inline)) {
    mfma_result_fence(st[0], st[1]);
    if (t == n1) skey = 0;
    const bool second = t >= n1;
    // every row sees every key of the tile (32-bit sums: skey is below the end of a range that fits 31 bits)
    const bool full = okmask == 0xffffffffu && (second ? skey <= all2hi - 32 : skey >= all1lo && skey <= all1hi - 32);
    int flags = 0;
    if (!full) {
      bool odd = false;
      const int g4 = 4 * (lane_now() >> 4);
      int lo, cnt;
      seen_keys(second, skey, lo, cnt);
#pragma unroll
      for (int mb = 0; mb < 2; ++mb)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int kk = 16 * mb + g4 + r;
          const bool ok = static_cast<uint32_t>(kk + lo) < static_cast<uint32_t>(cnt) && ((okmask >> kk) & 1);
          const bool fin = __builtin_fabsf(st[mb][r]) < __builtin_inff();
          odd = odd || (!ok && !fin);
          st[mb][r] = ok ? st[mb][r] : kNever;
        }
      flags = __builtin_amdgcn_ballot_w64(odd) ? kOdd : 0;
    }
    skey = static_cast<int>(static_cast<uint32_t>(skey) + 32u);  // (may leave 31 bits behind the last tile)
    const f32x4 y0 = st[0], y1 = st[1];
    float lmax = __builtin_fmaxf(__builtin_fmaxf(__builtin_fmaxf(y0[0], y0[1]), __builtin_fmaxf(y0[2], y0[3])),
                                 __builtin_fmaxf(__builtin_fmaxf(y1[0], y1[1]), __builtin_fmaxf(y1[2], y1[3])));
    lmax *= scale;
    // no lane's keys lift its row's maximum: the tile's maximum over the lanes of a row is not needed
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
      asm volatile("ds_write_b32 %0, %1" ::"v"(adst), "v"(alpha) : "memory");  // (the four lanes of a row write the same)
      if (__builtin_amdgcn_ballot_w64(alpha != 1.0f)) flags |= kMoved;
    }
    ref = m_ref == kNever ? 0.f : m_ref;
    const uint32_t fdst = lds_addr(reinterpret_cast<const char*>(&flag_lds[pbuf][wave]));
    asm volatile("ds_write_b32 %0, %1" ::"v"(fdst), "v"(flags) : "memory");
  };
  auto softmax_exp = [&](int i, f32x4 (&st)[2], float ref) __attribute__((always_inline)) {  // i of 8 weights
    const int b = i >> 3, mb = (i >> 2) & 1, r = i & 3;
    st[mb][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(st[mb][r], scale, -ref));
  };
  auto softmax_end = [&](const f32x4 (&p)[2], int pbuf) __attribute__((always_inline)) {
    const uint32_t pdst = lds_addr(&p_lds[pbuf][(wave * 64 + lane_now()) * 16]);
    l_run += ((p[0][0] + p[0][1]) + (p[0][2] + p[0][3])) + ((p[1][0] + p[1][1]) + (p[1][2] + p[1][3]));
    // P^T B-fragment: k-slots 8g+0..3 <-> keys 4g+0..3, 8g+4..7 <-> keys 16+4g+0..3
    const u32x4 w = u32x4{pack2<F16>(p[0][0], p[0][1]), pack2<F16>(p[0][2], p[0][3]),
                          pack2<F16>(p[1][0], p[1][1]), pack2<F16>(p[1][2], p[1][3])};
    asm volatile("ds_write_b128 %0, %1" ::"v"(pdst), "v"(w) : "memory");
  };

  // ---- O^T += V^T P^T -------------------------------------------------------------
  f32x4 oacc[MBW][NB];
#pragma unroll
  for (int j = 0; j < MBW; ++j)
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) oacc[j][nb] = f32x4{0.f, 0.f, 0.f, 0.f};
  // V^T transposing reads: source lane (g, i16) points at key 4g + (i16 >> 2) (+16 for k-slots 4..7), dims d0 + 4 (i16 & 3)
  // with d0 = 16 (4j + wave); chunk 8j + x, x = 2 wave + ((i16 & 3) >> 1) < 8, swizzles to 8j + (x ^ f): a fixed base + 128 j.
  // V^T blocks go through a queue VQ deep; between(j) runs among the MFMAs of output block j.
  constexpr int VQ0 = PAIR ? 2 : 4, VQ = VQ0 < MBW ? VQ0 : MBW;
  auto pv = [&](int slot, int pbuf, auto&& between) __attribute__((always_inline)) {
    const int ln = lane_now();
    const int tkey = 4 * (ln >> 4) + ((ln & 15) >> 2);
    const int tx = 2 * wave + ((ln & 3) >> 1);
    const int tbase = tkey * ROW + 16 * ((tx ^ kv_swz<D>(tkey)) & (SH::CPR - 1)) + 8 * (ln & 1);
    const uint32_t psrc = lds_addr(&p_lds[pbuf][0]) + ln * 16;
    bf16x8 pf[NB];
    attn_static_for<0, NB>([&](auto NC) {
      constexpr int nb = decltype(NC)::value;
      pf[nb] = ld128<1024 * nb>(psrc);
    });
    const uint32_t ta = lds_addr(ring(slot)) + tbase;
    v4i16 lo[VQ], hi[VQ];
    auto issue = [&](auto JC) __attribute__((always_inline)) {
      constexpr int j = decltype(JC)::value;
      lo[j % VQ] = tr_read<128 * j>(ta);
      hi[j % VQ] = tr_read<16 * ROW + 128 * j>(ta);
    };
    attn_static_for<0, VQ>(issue);
    attn_static_for<0, MBW>([&](auto JC) {
      constexpr int j = decltype(JC)::value;
      constexpr int later = (MBW - 1 - j) < (VQ - 1) ? (MBW - 1 - j) : (VQ - 1);
      lds_wait<2 * later>(lo[j % VQ], hi[j % VQ]);
      if constexpr (j == 0) {
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) reg_tie(pf[nb]);
      }
      const bf16x8 vf =
          __builtin_bit_cast(bf16x8, __builtin_shufflevector(lo[j % VQ], hi[j % VQ], 0, 1, 2, 3, 4, 5, 6, 7));
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) oacc[j][nb] = mfma16x16x32<F16>(vf, pf[nb], oacc[j][nb]);
      if constexpr (j + VQ < MBW) issue(std::integral_constant<int, j + VQ>{});
      between(JC);
    });
  };
  // A masked key of the tile has a score that is not finite.  Values that are not finite become zero, in the tile's LDS (every
  // wave has done with its scores), and a row that sees such a key gets a weight of NaN for it (it may be 0 so far, from a
  // score of -inf).  A key of finite values whose score has left fp32's range keeps its weight: 0, or NaN.
  auto clean_tile = [&](int t, uint32_t okmask, int slot, int pbuf) __attribute__((always_inline)) {
    const uint32_t tile = lds_addr(ring(slot));
    const int ln = lane_now(), g4 = 4 * (ln >> 4);
    uint32_t bad = 0;
    for (int c = ln >> 5; c < SH::CPR; c += 2) {  // lanes l and l + 32 look through key l
      bf16x8 x;
      asm volatile("ds_read_b128 %0, %1\n\ts_waitcnt lgkmcnt(0)" : "=v"(x) : "v"(tile + (ln & 31) * ROW + c * 16));
      const u32x4 d = __builtin_bit_cast(u32x4, x) ^ __builtin_bit_cast(u32x4, finite_or_zero<F16>(x));
      bad |= (d[0] | d[1]) | (d[2] | d[3]);
    }
    const uint64_t both = __builtin_amdgcn_ballot_w64(bad != 0);
    const uint32_t keys = (static_cast<uint32_t>(both) | static_cast<uint32_t>(both >> 32)) & okmask;
    const bool second = t >= n1;
    int lo, cnt;
    seen_keys(second, second ? (t - n1) * 32 : k1lo + t * 32, lo, cnt);
    const uint32_t pat = lds_addr(&p_lds[pbuf][(wave * 64 + ln) * 16]);
    u32x4 w;
    asm volatile("ds_read_b128 %0, %1\n\ts_waitcnt lgkmcnt(0)" : "=v"(w) : "v"(pat));
#pragma unroll
    for (int i = 0; i < 8; ++i) {  // (a weight of 0x7fff is NaN in both types)
      const int kk = 16 * (i >> 2) + g4 + (i & 3);
      if (((keys >> kk) & 1) && static_cast<uint32_t>(kk + lo) < static_cast<uint32_t>(cnt)) w[i >> 1] |= i & 1 ? 0x7fff0000u : 0x7fffu;
    }
    asm volatile("ds_write_b128 %0, %1" ::"v"(pat), "v"(w) : "memory");
    attn_tile_barrier();  // every wave has looked through the tile
    for (int e = threadIdx.x; e < SH::CH; e += kPagedThreads) {
      bf16x8 x;
      asm volatile("ds_read_b128 %0, %1\n\ts_waitcnt lgkmcnt(0)" : "=v"(x) : "v"(tile + e * 16));
      x = finite_or_zero<F16>(x);
      asm volatile("ds_write_b128 %0, %1" ::"v"(tile + e * 16), "v"(x) : "memory");
    }
  };

  // What the waves' flags of a tile ask for before its P V.
  auto settle = [&](int flags, int t, uint32_t okmask, int pbuf, int slot) __attribute__((always_inline)) {
    if (flags & kMoved) {
      // a wave's alpha is of this tile where the wave says so
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
      clean_tile(t, okmask, slot, pbuf);
      attn_tile_barrier();
    }
  };

  // ---- the tiles -------------------------------------------------------------
  // Iteration t: P V of tile t beside S^T and softmax of tile t + 1, one barrier.  Tile t lives in slot t - tbeg mod NS,
  // its P in p_lds[t & 1].  The copies of tile t + AHEAD go out at the start, into the slot of tile t - 1, which every
  // wave has left; they land by the start of iteration t + AHEAD - 1.
  if (tbeg >= tend) {
    sink_to_lds();
  } else if constexpr (!PAIR) {
    skey = tbeg < n1 ? k1lo + tbeg * 32 : (tbeg - n1) * 32;
    uint32_t okq[AHEAD];
    Sources src;
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      okq[i] = 0;
      if (tbeg + i < tend) {
        int page;
        asm volatile("ds_read_b32 %0, %1\n\ts_waitcnt lgkmcnt(0)" : "=v"(page) : "v"(page_addr(tbeg + i)));
        from = froms[i];
        okq[i] = address_tile(page, within[i], src);
        attn_static_for<0, SH::LPT>([&](auto IC) { copy(src, ring(i), IC); });
      }
    }
    uint32_t in_next = within[AHEAD];
    from = froms[AHEAD];
    if (tbeg + AHEAD <= tend) __builtin_amdgcn_s_waitcnt(vm_lgkm0((AHEAD - 1) * (SH::CH / SH::NT)));
    else __builtin_amdgcn_s_waitcnt(vm_lgkm0(0));
    attn_tile_barrier();  // the first tile landed
    f32x4 st[2];
    float ref;
    sink_to_lds();
    scale_q();
    qk(0, st, [] {}, [](auto) {});
    softmax_begin(tbeg, okq[0], st, ref, tbeg & 1);
#pragma unroll
    for (int i = 0; i < 8; ++i) softmax_exp(i, st, ref);
    softmax_end(st, tbeg & 1);
    int slot = 0;  // of tile t
    // MORE: a tile t + 1; COPY: a tile t + AHEAD
    auto iteration = [&](int t, auto MORE, auto COPY) __attribute__((always_inline)) {
      constexpr bool more = decltype(MORE)::value, ahead = decltype(COPY)::value;
      // tile t + 1 (and the page numbers of tile t + AHEAD) landed; with three tiles ahead the copies of the last stay in
      // flight.  Behind the barrier: every wave's, and every wave's P of tile t.
      if constexpr (ahead) __builtin_amdgcn_s_waitcnt(vm_lgkm0(SH::CH / SH::NT));
      else __builtin_amdgcn_s_waitcnt(vm_lgkm0(0));
      attn_tile_barrier();
      const int next = slot + 1 == NS ? 0 : slot + 1, last_slot = slot == 0 ? NS - 1 : slot - 1;
      int flags = 0;
      uint32_t ok_new = 0;
      char* dst = ring(last_slot);
      auto start = [&]() __attribute__((always_inline)) {
        u32x4 fl;
        int page;
        asm volatile("ds_read_b32 %0, %2\n\tds_read_b128 %1, %3\n\ts_waitcnt lgkmcnt(0)"
                     : "=&v"(page), "=&v"(fl)
                     : "v"(page_addr(t + AHEAD)), "v"(lds_addr(reinterpret_cast<const char*>(&flag_lds[t & 1][0]))));
        flags = __builtin_amdgcn_readfirstlane(static_cast<int>(fl[0] | fl[1] | fl[2] | fl[3]));
        if constexpr (ahead) {
          ok_new = address_tile(page, in_next, src);
          in_next = fetch_pages();  // (past the share's end: the same page again, not used)
        }
      };
      if constexpr (more) {
        // (the copies spread over the k-steps: in one go each waits for the one before to leave the queue)
        qk(next, st, start, [&](auto KC) {
          constexpr int ks = decltype(KC)::value;
          if constexpr (ahead) {
            constexpr int first = ks * SH::LPT / KS, end = (ks + 1) * SH::LPT / KS;
            attn_static_for<first, end>([&](auto IC) { copy(src, dst, IC); });
          }
        });
      } else {
        start();
      }
      if constexpr (ahead) from = from_next;
      if (__builtin_expect(flags != 0, 0)) settle(flags, t, okq[0], t & 1, slot);
      constexpr int SPAN = MBW > 2 ? MBW - 2 : 1, EPB = (8 + SPAN - 1) / SPAN;  // weights beside one of SPAN output blocks
      pv(slot, t & 1, [&](auto JC) {
        constexpr int j = decltype(JC)::value;
        if constexpr (more) {
          if constexpr (j == 0) softmax_begin(t + 1, okq[1], st, ref, (t + 1) & 1);
          if constexpr (j > 0 || MBW == 1) {
            constexpr int first = MBW == 1 ? 0 : (j - 1) * EPB;
#pragma unroll
            for (int i = first; i < first + EPB && i < 8; ++i) softmax_exp(i, st, ref);
          }
          if constexpr (j + 1 == MBW) softmax_end(st, (t + 1) & 1);
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
    // PAIR: one tile ahead in LDS, a tile's steps one after the other, two barriers; the other workgroups of the CU fill
    // the gaps.
    skey = tbeg < n1 ? k1lo + tbeg * 32 : (tbeg - n1) * 32;
    uint32_t ok;
    {
      int page;
      asm volatile("ds_read_b32 %0, %1\n\ts_waitcnt lgkmcnt(0)" : "=v"(page) : "v"(page_addr(tbeg)));
      from = froms[0];
      Sources src;
      ok = address_tile(page, within[0], src);
      attn_static_for<0, SH::LPT>([&](auto IC) { copy(src, ring(0), IC); });
    }
    uint32_t in_next = within[1];
    from = froms[1];
    sink_to_lds();
    scale_q();
    for (int t = tbeg; t < tend; ++t) {
      const int slot = (t - tbeg) & 1;
      __builtin_amdgcn_s_waitcnt(vm_lgkm0(0));
      attn_tile_barrier();  // tile t landed, every wave has left tile t - 1 and its P
      uint32_t ok_next = 0;
      {
        f32x4 st[2];
        float ref;
        qk(slot, st, [] {}, [](auto) {});
        softmax_begin(t, ok, st, ref, 0);
#pragma unroll
        for (int i = 0; i < 8; ++i) softmax_exp(i, st, ref);
        softmax_end(st, 0);
      }
      if (t + 1 < tend) {
        int page;
        asm volatile("ds_read_b32 %0, %1\n\ts_waitcnt lgkmcnt(0)" : "=v"(page) : "v"(page_addr(t + 1)));
        Sources src;
        ok_next = address_tile(page, in_next, src);
        attn_static_for<0, SH::LPT>([&](auto IC) {
          copy(src, ring(slot ^ 1), IC);
          __builtin_amdgcn_sched_barrier(0);  // (one address at a time: registers)
        });
        in_next = fetch_pages();  // (past the share's end: the same page again, not used)
        from = from_next;
      }
      attn_tile_barrier();  // P published
      u32x4 fl;
      asm volatile("ds_read_b128 %0, %1\n\ts_waitcnt lgkmcnt(0)" : "=v"(fl)
                   : "v"(lds_addr(reinterpret_cast<const char*>(&flag_lds[0][0]))));
      const int flags = __builtin_amdgcn_readfirstlane(static_cast<int>(fl[0] | fl[1] | fl[2] | fl[3]));
      if (__builtin_expect(flags != 0, 0)) settle(flags, t, ok, 0, slot);
      pv(slot, 0, [](auto) {});
      ok = ok_next;
    }
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
  float* scale_lds = alpha_lds[0];
  __syncthreads();  // every wave has left the last tile and its alpha
  const float sink = sink_lds[lrow];
  const float sink2 = sink_log2(sink);
  const float m_fin = __builtin_fmaxf(m_ref, sink2);
  const float top = m_fin == kNever ? 0.f : m_fin;
  const float resc = __builtin_amdgcn_exp2f(m_ref - top), keys = l_tot * resc;
  const float l_fin = keys + __builtin_amdgcn_exp2f(sink2 - top);
  if (g == 0) {
    scale_lds[lrow] = keys == 0.f ? 0.f : resc / l_fin;
    if (live) a.lse[flat0 + lrow] = keys == 0.f ? lse_of_sink(sink) : (__builtin_amdgcn_logf(l_fin) + top) * kLn2;
  }
  __syncthreads();  // scales published
  // staged in the tiles' LDS, chunk c of row r at c ^ (r & 7), then written in one piece: the rows follow each other in o
  float sc[NB];
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) sc[nb] = scale_lds[nb * 16 + i16];
#pragma unroll
  for (int j = 0; j < MBW; ++j) {
    const int mbi = j * kAttnWaves + wave;
    if (SH::MBT % kAttnWaves == 0 || mbi < SH::MBT) {
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
        const f32x4 v = oacc[j][nb] * sc[nb];
        uint2 w;
        w.x = pack2<F16>(v[0], v[1]);
        w.y = pack2<F16>(v[2], v[3]);
        *reinterpret_cast<uint2*>(kv_lds + kv_off<D>(nb * 16 + i16, 2 * mbi + (g >> 1)) + 8 * (g & 1)) = w;
      }
    }
  }
  __syncthreads();
  char* obase = reinterpret_cast<char*>(a.o + flat0 * D);
  for (int e = threadIdx.x; e < nrows * SH::CPR; e += kPagedThreads)
    *reinterpret_cast<u32x4*>(obase + static_cast<int64_t>(e) * 16) =
        *reinterpret_cast<const u32x4*>(kv_lds + kv_off<D>(e / SH::CPR, e % SH::CPR));
}

constexpr int kCombineParts = 4;
// Joins the shares of the split row blocks.  A thread takes four dimensions of a row and every PARTS-th share, up to
// sixteen in flight, with a running maximum; with four parts the four threads of a place join theirs in LDS.  Bound: the
// latency of the launch and of two dependent loads (4 us with nothing split, 6 for 256 partial outputs at D = 576, 38 MB
// that the last-level cache holds).
template <bool F16>
__global__ __launch_bounds__(kPagedThreads) void paged_combine_kernel(PagedAttnArgs a, int D) {
  constexpr float kLn2 = 0.6931471805599453f;
  constexpr int M = kRows, U = 4;
  __shared__ float lds[kCombineParts - 1][6][kPagedThreads / kCombineParts];
  const int count = a.rec[0];
  const bool wide = static_cast<int>(gridDim.x) > D / 16;
  for (int b = blockIdx.y; b < count; b += gridDim.y) {
    const int4 rec = *reinterpret_cast<const int4*>(a.rec + 4 + 4 * static_cast<int64_t>(b));
    const int parts = wide && rec.y > 2 * U ? kCombineParts : 1, places = kPagedThreads / parts;
    if (static_cast<int>(blockIdx.x) * places >= M * D / 4) continue;
    const int at = threadIdx.x % places, part = threadIdx.x / places;
    // block of 16 rows and 16 dimensions (the same in a whole wave), row and dimensions
    const int block = (static_cast<int>(blockIdx.x) * places + at) >> 6, nb = block / (D / 16), mbi = block - nb * (D / 16);
    const int lane = at & 63, row = nb * 16 + (lane & 15), d = mbi * 16 + 4 * (lane >> 4);
    if (nb * 16 >= rec.w) continue;  // (the same in every thread where there are parts)
    const bool live = row < rec.w;
    const int64_t flat = static_cast<int64_t>(rec.z) + row;
    const float sink = live ? a.sink[flat % a.H] : 0.f;
    float m = kNever, l = 0.f;
    f32x4 acc = f32x4{0.f, 0.f, 0.f, 0.f};
    const int64_t first = static_cast<int64_t>(rec.x) * M;
    const float2* ml = a.part_ml + first + (live ? row : 0);
    const float* po = a.part_o + first * D + (block * 64 + lane) * 4;
    for (int i0 = part; i0 < rec.y; i0 += U * parts) {
      float2 v[U];
      f32x4 x[U];
      float top = m;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int i = i0 + u * parts;
        if (i < rec.y) {  // (the same in a whole wave)
          v[u] = ml[static_cast<int64_t>(i) * M];
          x[u] = *reinterpret_cast<const f32x4*>(po + static_cast<int64_t>(i) * M * D);
        } else {
          v[u] = float2{kNever, 0.f};
          x[u] = f32x4{0.f, 0.f, 0.f, 0.f};
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) top = __builtin_fmaxf(top, v[u].x);
      const float ref = top == kNever ? 0.f : top;
      const float s = __builtin_amdgcn_exp2f(m - ref);
      l *= s;
      acc *= s;
      m = top;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const float w = __builtin_amdgcn_exp2f(v[u].x - ref);
        l = __builtin_fmaf(v[u].y, w, l);
#pragma unroll
        for (int c = 0; c < 4; ++c) acc[c] = __builtin_fmaf(x[u][c], w, acc[c]);
      }
    }
    if (parts > 1) {  // (the same in every thread, and nb too)
      __syncthreads();  // (the last block's partial sums have been read)
      if (part > 0) {
        lds[part - 1][0][at] = m;
        lds[part - 1][1][at] = l;
#pragma unroll
        for (int c = 0; c < 4; ++c) lds[part - 1][2 + c][at] = acc[c];
      }
      __syncthreads();
      if (part == 0) {
        float top = m;
#pragma unroll
        for (int q = 0; q + 1 < kCombineParts; ++q) top = __builtin_fmaxf(top, lds[q][0][at]);
        const float ref = top == kNever ? 0.f : top;
        float w = __builtin_amdgcn_exp2f(m - ref);
        l *= w;
        acc *= w;
#pragma unroll
        for (int q = 0; q + 1 < kCombineParts; ++q) {
          w = __builtin_amdgcn_exp2f(lds[q][0][at] - ref);
          l = __builtin_fmaf(lds[q][1][at], w, l);
#pragma unroll
          for (int c = 0; c < 4; ++c) acc[c] = __builtin_fmaf(lds[q][2 + c][at], w, acc[c]);
        }
        m = top;
      }
    }
    if (part > 0 || !live) continue;
    const float sink2 = sink_log2(sink);
    const float top = __builtin_fmaxf(m, sink2);
    const float ref = top == kNever ? 0.f : top;
    const float w = __builtin_amdgcn_exp2f(m - ref);
    const float keys = l * w;
    const float all = keys + __builtin_amdgcn_exp2f(sink2 - ref);
    const float inv = keys == 0.f ? 0.f : w / all;
    uint2 o;
    o.x = pack2<F16>(acc[0] * inv, acc[1] * inv);
    o.y = pack2<F16>(acc[2] * inv, acc[3] * inv);
    *reinterpret_cast<uint2*>(a.o + flat * D + d) = o;
    if (d == 0) a.lse[flat] = keys == 0.f ? lse_of_sink(sink) : (__builtin_amdgcn_logf(all) + ref) * kLn2;
  }
}

int launch_paged_combine(bool f16, const PagedAttnArgs& a, int D, int64_t split_blocks, hipStream_t st) {
  // One thread a place, or up to four for blocks of many shares where the workgroups that others leave idle are few (us, 2
  // shares, D = 576: 24 blocks 5.2 with them and 4.3 without, 33 blocks 6.4 and 4.5; but 32 blocks of up to 59 shares, D = 128, 6
  // and 12).
  const bool wide = D / 16 * kCombineParts * split_blocks < 4096;
  const dim3 block(kPagedThreads), cgrid(static_cast<unsigned>(D / 16 * (wide ? kCombineParts : 1)), static_cast<unsigned>(split_blocks));
  if (f16) hipLaunchKernelGGL(paged_combine_kernel<true>, cgrid, block, 0, st, a, D);
  else hipLaunchKernelGGL(paged_combine_kernel<false>, cgrid, block, 0, st, a, D);
  return check_launch("paged_combine_kernel");
}

bool paged_attn_served(int64_t D) { return D == 32 || D == 64 || D == 128 || D == 256 || D == 512 || D == 576; }

// Sizes of a call, from what the host knows.
struct PagedSizes {
  bool pair;             // the kernel with PAIR
  int64_t blocks;        // row blocks of a workgroup at most
  int64_t want;          // workgroups that run at once
  int64_t grid;          // workgroups
  int64_t items;         // partial outputs at most, 0: no row block is split
  int64_t split_blocks;  // split row blocks at most
  int64_t bytes;         // scratch
  int behind;            // tokens of a row block before its last one at most
};
static PagedSizes paged_sizes(int64_t N, int64_t H, int64_t D, int64_t R, int64_t window, int64_t keys1, int64_t keys2) {
  PagedSizes p{};
  const int64_t M = kRows;
  // a request's last row block is part empty unless M divides n H
  int64_t g = M;
  while (H % g) g /= 2;
  p.blocks = (N * H + (R < N ? R : N) * (M - g)) / M;
  p.pair = p.blocks >= pair_from(D);
  const int64_t want = p.want = 256 * per_cu(static_cast<int>(D), p.pair);
  p.grid = 2 * p.blocks <= want ? want : p.blocks + want;
  // tiles of a row block at most
  const int64_t span = M / H + 1 + window;
  p.behind = static_cast<int>((M - 1 + H - g) / H);  // (a row block begins at any multiple of g heads of a token)
  const int64_t tiles = ((window < keys1 && span < keys1 ? span : keys1) + 31) / 32 + (keys2 + 31) / 32;
  // Where no cut can win back the second launch, 4 us, that joins the shares, none is made (8 tiles at D = 576, 14 at 128, and
  // more of them where many row blocks leave partial outputs; us whole and cut in two: 1 row block of 10 and 16 tiles, D = 576,
  // 21 and 21, 29 and 22; 64 of 16 and 24, 30 and 30, 41 and 34; one of 16 and 24, D = 128, 17 and 20, 23 and 20).
  if (tiles <= (D >= 512 ? 8 : 14) + p.blocks / 8) {
    p.grid = p.blocks;
    return p;
  }
  // shares of split row blocks: sum of ceil(tiles / c) <= 2 sum tiles / c <= 2 want, where tiles > c >= U / want
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
static int launch_paged_attn_d(bool f16, const PagedAttnArgs& a, const PagedSizes& p, hipStream_t st) {
  const int64_t most = 0xffffffffLL / kPagedThreads;  // (a launch has fewer than 2^32 threads)
  if (p.grid + 7 > most) return set_error(SI_ERR_UNSUPPORTED, "too many rows for one launch");
  // (whole rounds of the XCDs: see paged_item_number)
  const dim3 grid(static_cast<unsigned>(((p.grid < 1 ? 1 : p.grid) + 7) & ~int64_t{7})), block(kPagedThreads);
  auto launch = [&](auto PAIR) {
    constexpr bool pair = decltype(PAIR)::value;
    if (f16) hipLaunchKernelGGL((paged_attn_kernel<D, true, pair>), grid, block, 0, st, a);
    else hipLaunchKernelGGL((paged_attn_kernel<D, false, pair>), grid, block, 0, st, a);
  };
  if constexpr (pair_from(D) < INT64_MAX) {
    if (p.pair) launch(std::true_type{});
    else launch(std::false_type{});
  } else {
    launch(std::false_type{});
  }
  const int rc = check_launch("paged_attn_kernel");
  if (rc || !a.part_o) return rc;
  return launch_paged_combine(f16, a, D, p.split_blocks, st);
}

int64_t paged_cache_keys(int64_t pages, int64_t P, int64_t ps) {
  const int64_t k = pages > 0 ? P * ps : 0;
  return k < 0x7fffffff ? k : 0x7fffffff;
}

int set_paged_cache(PagedCache& c, int size, const void* base, const int64_t* strides, int64_t pages, int64_t ps, int64_t D,
                    const int32_t* table, int64_t tstride, int64_t P, int64_t R, const char* name) {
  const std::string n(name);
  if (!strides) return set_error(SI_ERR_INVALID, n + ": null stride argument");
  if (pages < 0 || ps <= 0 || P < 0) return set_error(SI_ERR_INVALID, n + ": bad dimension");
  if (pages > 0x7fffffff || ps > 0x7fffffff || P > 0x7fffffff) return set_error(SI_ERR_UNSUPPORTED, n + ": dimension exceeds int32");
  if (R == 0) P = 0;
  if (pages > 0 && P > 0 && (!base || !table)) return set_error(SI_ERR_INVALID, n + ": null pointer argument");
  if (R > 1 && tstride < 0) return set_error(SI_ERR_INVALID, n + ": negative block table stride");
  if (strides[2] != 1 || strides[0] < 0 || strides[1] < 0 || (strides[0] | strides[1]) % (16 / size) ||
      (reinterpret_cast<uintptr_t>(base) & 15))
    return set_error(SI_ERR_INVALID, n + " needs a contiguous last dimension, 16-byte rows and alignment");
  // (each factor below 2^31: no product overflows 64 bits before it is compared)
  const int64_t lim = (int64_t{1} << 36) / size;  // 64 GiB in elements
  if (pages > 0 && (strides[0] >= lim || strides[1] >= lim || (pages - 1) > (lim - 1) / (strides[0] > 0 ? strides[0] : 1) ||
                    (ps - 1) > (lim - 1) / (strides[1] > 0 ? strides[1] : 1) ||
                    (pages - 1) * strides[0] + (ps - 1) * strides[1] + D > lim))
    return set_error(SI_ERR_UNSUPPORTED, n + " larger than 64 GiB");
  c.base = static_cast<const uint16_t*>(base);
  c.table = table;
  c.tstride = tstride;
  c.pstride = static_cast<uint32_t>(strides[0] / (16 / size));
  c.rstride = static_cast<uint32_t>(strides[1] / (16 / size));
  c.pages = P > 0 ? static_cast<int>(pages) : 0;
  c.keys = static_cast<int>(paged_cache_keys(pages, P, ps));
  c.ps = static_cast<uint32_t>(ps);
  c.magic = 0;
  c.shift = 0;
  c.one = ps == 1 ? ~0u : 0u;
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

}  // namespace si

using namespace si;

extern "C" int64_t si_paged_attn_fwd_scratch_bytes(int64_t N, int64_t H, int64_t D, int64_t R, int64_t window,
                                                   int64_t keys, int64_t keys2) {
  const int64_t lim = 0x7fffffff;
  if (N <= 0 || H <= 0 || R <= 0 || window < 0 || keys < 0 || keys2 < 0 || !paged_attn_served(D) || N > lim || H > lim ||
      N * H > lim || R > lim)
    return 0;
  return paged_sizes(N, H, D, R, window == 0 || window > lim ? lim : window, keys < lim ? keys : lim,
                       keys2 < lim ? keys2 : lim).bytes;
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
  PagedAttnArgs a{};
  int rc = set_paged_cache(a.c1, 2, kv, kv_strides, pages, page_size, D, block_table, table_stride, P, R, "kv");
  if (rc) return rc;
  if (ratio > 0) {
    rc = set_paged_cache(a.c2, 2, kv2, kv2_strides, pages2, page_size2, D, block_table2, table_stride2, P2, R, "kv2");
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
  PagedSizes p = paged_sizes(N, H, D, R > 0 ? R : 1, a.window, paged_cache_keys(pages, P, page_size),
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
  const bool f16 = qkv_dtype == SI_DTYPE_F16;
  switch (D) {
    case 32: return launch_paged_attn_d<32>(f16, a, p, st);
    case 64: return launch_paged_attn_d<64>(f16, a, p, st);
    case 128: return launch_paged_attn_d<128>(f16, a, p, st);
    case 256: return launch_paged_attn_d<256>(f16, a, p, st);
    case 512: return launch_paged_attn_d<512>(f16, a, p, st);
    default: return launch_paged_attn_d<576>(f16, a, p, st);
  }
}
