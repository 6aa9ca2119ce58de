// Paged-cache bookkeeping for gfx950: block tables and slots from request lengths, rows written to slots, and the token
// compressor over paged streams.
//
// A page holds page_size consecutive entries of one request; block_table[r, i] is the page of entries i * page_size and
// on, negative where there is none; slot = page * page_size + offset names a row of the cache.  No counterpart in the
// reference (its operators take whole sequences); the compressor's formula is flash_sparse/reference.py:176-272.
#include <hip/hip_fp16.h>

#include <string>

#include "si_common.h"
#include "si_status.h"

namespace si {

constexpr int64_t kMostBlocks = 0xffffffffLL / 256;  // of 256 threads: a launch has fewer than 2^32

// ---------------------------------------------------------------------------
// Plan
//
//   old = ctx / m, want = (ctx + new) / m - old, cu[r+1] = min(rows, want[0] + .. + want[r]), seq = old + cu[r+1] - cu[r]
//   have = min(ceil(old / ps), P), more = max(0, min(ceil(seq / ps), P) - have), base = start + more[0] + .. + more[r-1]
//   block_table[r, have + j] = free[base + j], or -1 past the list's end, for j < more
//
// One launch: every workgroup sums the lengths itself (R of them, L2-resident after the first) and then takes its share of
// the rows and of the new pages, which it finds in the sums by bisection.  A row whose page is new computes that page
// from the free list as well, so no workgroup reads what another one writes.  Bound: the latency of one chain of loads
// and scans, 3.7 us for 64 rows of 64 requests and 9.2 for 79,134 of 301; a kernel for the sums and one for the rows would pay a
// second launch.
// ---------------------------------------------------------------------------
struct PlanArgs {
  const int32_t* ctx;
  const int32_t* add;
  int32_t* table;
  int64_t tstride;
  const int32_t* free_pages;
  const int32_t* free_start;  // optional
  int32_t *cu, *seq, *request, *pos, *next;
  int64_t* slots;
  int R, P, F, rows;
  int64_t m, ps;
  int per;  // requests per thread in the sums
};

constexpr int kPlanThreads = 256;

struct PlanReq {  // lengths of one request in entries
  int64_t old, want;
};
__device__ __forceinline__ PlanReq plan_req(const PlanArgs& a, int r) {
  const int64_t ctx = a.ctx[r] > 0 ? a.ctx[r] : 0;
  const int64_t add = a.add[r] > 0 ? a.add[r] : 0;
  if (a.m == 1) return PlanReq{ctx, add};
  const uint32_t m = static_cast<uint32_t>(a.m);  // (ctx + add < 2^32)
  const int64_t old = static_cast<uint32_t>(ctx) / m;
  return PlanReq{old, static_cast<int64_t>(static_cast<uint32_t>(ctx + add) / m) - old};
}
struct PlanPages {
  int64_t have, more;
};
__device__ __forceinline__ PlanPages plan_pages(const PlanArgs& a, int64_t old, int64_t n) {
  auto pages = [&](int64_t len) {  // (len < 2^32: two lengths below 2^31)
    const int64_t p = len > 0 ? static_cast<int64_t>(static_cast<uint32_t>(len - 1) / static_cast<uint32_t>(a.ps)) + 1 : 0;
    return p < a.P ? p : static_cast<int64_t>(a.P);
  };
  const int64_t have = pages(old), need = pages(old + n);
  return PlanPages{have, need - have};
}

// Exclusive prefix sum of x over the workgroup; *total receives the sum.
__device__ __forceinline__ int64_t plan_scan(int64_t x, int64_t* lds, int64_t* total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int64_t v = x;
#pragma unroll
  for (int d = 1; d < kWave; d *= 2) {
    const int64_t y = __shfl_up(v, d);
    if (lane >= d) v += y;
  }
  if (lane == kWave - 1) lds[wave] = v;
  __syncthreads();
  int64_t before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kPlanThreads / kWave; ++w) {
    if (w < wave) before += lds[w];
    all += lds[w];
  }
  __syncthreads();
  *total = all;
  return before + v - x;
}

// The last i in [0, n) with first[i] <= x (first[0] <= x).
__device__ __forceinline__ int plan_find(const int64_t* first, int n, int64_t x) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (first[mid] <= x) lo = mid; else hi = mid;
  }
  return lo;
}

__global__ __launch_bounds__(kPlanThreads) void paged_plan_kernel(PlanArgs a) {
  __shared__ int64_t scan_lds[kPlanThreads / kWave];
  __shared__ int64_t cu_lds[kPlanThreads], page_lds[kPlanThreads];  // rows and pages before each thread's requests
  const int t = threadIdx.x;
  const int r0 = min(t * a.per, a.R), r1 = min(r0 + a.per, a.R);
  int64_t sum = 0, all;
  for (int r = r0; r < r1; ++r) sum += plan_req(a, r).want;
  const int64_t cu0 = plan_scan(sum, scan_lds, &all);
  auto cut = [&](int64_t x) { return x < a.rows ? x : static_cast<int64_t>(a.rows); };
  const int64_t used = cut(all);
  const bool first = blockIdx.x == 0;
  // pages of this thread's requests, and what the first workgroup writes of each request
  int64_t at = cu0, pages = 0, new_pages;
  for (int r = r0; r < r1; ++r) {
    const PlanReq q = plan_req(a, r);
    const int64_t n = cut(at + q.want) - cut(at);
    if (first) {
      a.cu[r] = static_cast<int32_t>(cut(at));
      a.seq[r] = static_cast<int32_t>(q.old + n);
    }
    pages += plan_pages(a, q.old, n).more;
    at += q.want;
  }
  const int64_t page0 = plan_scan(pages, scan_lds, &new_pages);
  cu_lds[t] = cut(cu0);
  page_lds[t] = page0;
  __syncthreads();
  const int64_t start = a.free_start ? (*a.free_start > 0 ? *a.free_start : 0) : 0;
  if (first && t == 0) {
    a.cu[a.R] = static_cast<int32_t>(used);
    const int64_t next = start + new_pages;
    *a.next = static_cast<int32_t>(next < 0x7fffffff ? next : 0x7fffffff);
  }
  auto free_page = [&](int64_t i) { return i < a.F ? a.free_pages[i] : -1; };
  const int64_t step = static_cast<int64_t>(gridDim.x) * kPlanThreads;
  const int64_t self = static_cast<int64_t>(blockIdx.x) * kPlanThreads + t;
  // rows
  for (int64_t row = self; row < a.rows; row += step) {
    int64_t slot = -1;
    int req = -1, pos = -1;
    if (row < used) {
      // (threads without requests start where the last one with some ends: past every used row)
      const int c = plan_find(cu_lds, kPlanThreads, row);
      int64_t begin = cu_lds[c], page = page_lds[c];
      for (int r = c * a.per;; ++r) {  // ends at a request below min((c + 1) per, R): it holds the row
        const PlanReq q = plan_req(a, r);
        const int64_t n = cut(begin + q.want) - begin;
        const PlanPages pp = plan_pages(a, q.old, n);
        if (row < begin + n || r + 1 >= a.R) {
          const int64_t p = q.old + row - begin;
          const int64_t col = static_cast<uint32_t>(p) / static_cast<uint32_t>(a.ps);
          int64_t pg = -1;
          if (col < a.P) pg = col < pp.have ? a.table[r * a.tstride + col] : free_page(start + page + col - pp.have);
          if (pg >= 0) slot = pg * a.ps + (p - col * a.ps);
          req = r;
          pos = static_cast<int>(p);
          break;
        }
        begin += n;
        page += pp.more;
      }
    }
    a.slots[row] = slot;
    a.request[row] = req;
    a.pos[row] = pos;
  }
  // new pages
  for (int64_t i = self; i < new_pages; i += step) {
    const int c = plan_find(page_lds, kPlanThreads, i);
    int64_t begin = cu_lds[c], page = page_lds[c];
    for (int r = c * a.per; r < a.R; ++r) {
      const PlanReq q = plan_req(a, r);
      const int64_t n = cut(begin + q.want) - begin;
      const PlanPages pp = plan_pages(a, q.old, n);
      if (i < page + pp.more) {
        a.table[r * a.tstride + pp.have + i - page] = free_page(start + i);
        break;
      }
      begin += n;
      page += pp.more;
    }
  }
}

// ---------------------------------------------------------------------------
// Write: cache[slot[t]] = rows[t], rows whose slot is outside the cache nowhere.
//
// A copy in pieces of the widest type that every row start allows; a workgroup's threads take consecutive pieces of
// consecutive rows, four each, with all loads of a thread in flight before its stores.  Bound: memory bandwidth (43.8
// MB read and written in 8.4 us, 5.2 TB/s).
// ---------------------------------------------------------------------------
struct WriteArgs {
  const char* rows;
  char* cache;
  const int64_t* slots;
  int64_t rstride, pstride, sstride;  // bytes: row of rows, page and row of the cache
  int64_t total;                      // pieces
  int64_t nslots;
  int64_t ps;
  uint32_t vec;  // pieces of a row
  int flat;      // pages follow each other: a slot is a row number
};

constexpr int kWriteUnroll = 4;

template <typename V>
__global__ __launch_bounds__(256) void paged_write_kernel(WriteArgs a) {
  const int64_t base = static_cast<int64_t>(blockIdx.x) * (256 * kWriteUnroll) + threadIdx.x;
  V v[kWriteUnroll];
  char* dst[kWriteUnroll];
#pragma unroll
  for (int u = 0; u < kWriteUnroll; ++u) {
    const int64_t e = base + u * 256;
    dst[u] = nullptr;
    if (e < a.total) {
      int64_t row, c;
      if (a.total <= 0x7fffffff) {  // (32-bit divisions where they do)
        row = static_cast<uint32_t>(e) / a.vec;
        c = static_cast<uint32_t>(e) % a.vec;
      } else {
        row = e / a.vec;
        c = e % a.vec;
      }
      const int64_t slot = a.slots[row];
      if (slot >= 0 && slot < a.nslots) {
        v[u] = *reinterpret_cast<const V*>(a.rows + row * a.rstride + c * sizeof(V));
        int64_t off;
        if (a.flat) {
          off = slot * a.sstride;
        } else if (a.nslots <= 0x7fffffff) {
          const uint32_t page = static_cast<uint32_t>(slot) / static_cast<uint32_t>(a.ps);
          off = page * a.pstride + (slot - static_cast<int64_t>(page) * a.ps) * a.sstride;
        } else {
          const int64_t page = slot / a.ps;
          off = page * a.pstride + (slot - page * a.ps) * a.sstride;
        }
        dst[u] = a.cache + off + c * sizeof(V);
      }
    }
  }
#pragma unroll
  for (int u = 0; u < kWriteUnroll; ++u)
    if (dst[u]) *reinterpret_cast<V*>(dst[u]) = v[u];
}

template <typename V>
static int launch_write(WriteArgs a, int64_t n, int64_t row_bytes, hipStream_t st) {
  a.vec = static_cast<uint32_t>(row_bytes / static_cast<int64_t>(sizeof(V)));
  a.total = n * a.vec;
  const int64_t blocks = (a.total + 256 * kWriteUnroll - 1) / (256 * kWriteUnroll);
  if (blocks > kMostBlocks) return set_error(SI_ERR_UNSUPPORTED, "tensor too large");
  hipLaunchKernelGGL(paged_write_kernel<V>, dim3(static_cast<unsigned>(blocks)), dim3(256), 0, st, a);
  return check_launch("paged_write_kernel");
}

// ---------------------------------------------------------------------------
// Compress: entry i of request r pools tokens i m .. i m + m - 1 of the streams a (and, with two streams, tokens
// (i - 1) m .. i m - 1 of the streams b),
//   out[c] = sum_j v_j[c] e^(z_j[c] + bias_j[c]) / sum_j e^(z_j[c] + bias_j[c]),
// channel by channel; a token without a page counts as absent.
//
// The workgroup looks up where its tokens' rows are once, into LDS.  Then a thread takes 16 (or 8) bytes of channels and
// every PARTS-th token, keeps the running maximum, denominator and numerator of each channel in fp32 registers, and the
// PARTS threads of a channel group join theirs by lane exchanges and, at 32, one LDS step.  Eight neighbouring threads read
// 128 consecutive bytes of a row.  Bound: the two streams' bytes for 4-byte elements (454 MB in 85 us, 5.3 TB/s).  With 2-byte
// ones as many values come in half the bytes: 149 MB in 40 us, 3.7 TB/s.  Vector instructions, twenty a value with the
// exponential, fill 66 % of the CUs' busy cycles there, and about 9 us do not grow with the entries (113 MB in 31.6 us, 226 MB in
// 54.4: 5.0 TB/s between them): the launch, a chain of lookup, page and rows, and a second round of few workgroups.
// ---------------------------------------------------------------------------
struct CompressArgs {
  const char *ca, *za, *cb, *zb;        // streams, [pages, ps, C]
  int64_t pstride[4], rstride[4];       // elements: page and row of ca, za, cb, zb
  const float *ba, *bb;                 // [m, C]
  const int32_t* table;
  int64_t tstride;
  const int32_t *request, *entry;
  const int64_t* slots;
  char* out;                            // [out_pages, out_ps, C]
  int64_t out_pstride, out_rstride;     // elements
  int64_t nslots, out_ps;
  int64_t E, C, m, ps;
  int R, P, pages, overlap;
  int groups;                           // channel groups of 8 threads
};

template <int DT>
struct Elem;
template <>
struct Elem<0> {
  typedef float T;
};
template <>
struct Elem<1> {
  typedef __bf16 T;
};
template <>
struct Elem<2> {
  typedef _Float16 T;
};
template <int DT, int N>
struct Piece {  // N elements of type DT (0 fp32, 1 bf16, 2 fp16), as they lie in memory
  typedef typename Elem<DT>::T T;
  typedef T vec __attribute__((ext_vector_type(N)));
  vec w;
  __device__ __forceinline__ void load(const char* p) { w = *reinterpret_cast<const vec*>(p); }
  __device__ __forceinline__ void fill(float x) {
#pragma unroll
    for (int e = 0; e < N; ++e) w[e] = static_cast<T>(x);
  }
  __device__ __forceinline__ float at(int e) const { return static_cast<float>(w[e]); }
  static __device__ __forceinline__ void store(char* p, const float (&v)[N]) {  // rounds to nearest even
    vec w;
#pragma unroll
    for (int e = 0; e < N; ++e) w[e] = static_cast<T>(v[e]);
    *reinterpret_cast<vec*>(p) = w;
  }
};

// The value of the lane D away.
template <int D>
__device__ __forceinline__ float lane_away(float x) {
  return __uint_as_float(lane_xor_u32<D>(__float_as_uint(x)));
}

template <int DT, int N, int PARTS>
__global__ __launch_bounds__(256, 4) void paged_compress_kernel(CompressArgs a) {
  static_assert(PARTS == 1 || PARTS == 4 || PARTS == 8 || PARTS == 32, "8 lanes, half a wave, a wave or a workgroup to an entry");
  constexpr int U = 4;                       // tokens of a thread in flight
  constexpr int SIZE = DT == 0 ? 4 : 2;
  constexpr int ITEMS = 32 / PARTS;          // entries of a workgroup
  constexpr int ROWS = 256 / ITEMS;          // tokens of an entry looked up at a time
  constexpr float kLog2e = 1.4426950408889634f;
  __shared__ const char* row_lds[3][256];    // of each token: content and gate (null: no page), bias
  const int vg = threadIdx.x & 7;
  const int part = (threadIdx.x >> 3) % PARTS;
  const int item = (threadIdx.x >> 3) / PARTS;
  const int64_t group = blockIdx.x % a.groups;
  const int64_t e0 = static_cast<int64_t>(blockIdx.x / a.groups) * ITEMS;
  const int64_t c = (group * 8 + vg) * N;
  // entry `i` of the workgroup: its request, or -1
  auto entry = [&](int i, int& ent, int64_t& slot) {
    const int64_t e = e0 + i;
    if (e >= a.E) return -1;
    const int r = a.request[e];
    ent = a.entry[e];
    slot = a.slots[e];
    return r >= 0 && r < a.R && ent >= 0 && slot >= 0 && slot < a.nslots ? r : -1;
  };
  int ent = 0;
  int64_t slot = 0;
  const bool there = entry(item, ent, slot) >= 0;
  if (ITEMS == 1 && !there) return;  // (the same in every thread)
  const bool live = there && c < a.C;
  const int64_t most = a.overlap ? 2 * a.m : a.m;
  const int64_t rows = a.overlap && ent > 0 ? 2 * a.m : a.m;
  // the token that this thread looks up, of entry `look`
  const int look = threadIdx.x / ROWS;
  int lent = 0;
  int64_t lslot = 0;
  const int lreq = ITEMS == 1 ? a.request[e0] : entry(look, lent, lslot);
  if (ITEMS == 1) lent = ent;
  const int64_t lrows = a.overlap && lent > 0 ? 2 * a.m : a.m;
  float mx[N], den[N], num[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    mx[i] = -__builtin_inff();
    den[i] = 0.f;
    num[i] = 0.f;
  }
  bool any = false;
  for (int64_t base = 0; base < most; base += ROWS) {
    if (base > 0) __syncthreads();  // (the last tokens' rows have been read)
    {
      const int64_t j = base + threadIdx.x % ROWS;
      const char *zrow = nullptr, *crow = nullptr, *brow = nullptr;
      if (lreq >= 0 && j < lrows) {
        const bool second = j >= a.m;  // stream b: the block before
        const int64_t jj = second ? j - a.m : j;
        int64_t at = (static_cast<int64_t>(lent) - (second ? 1 : 0)) * a.m + jj;
        int64_t col;
        if (at <= 0x7fffffff) {
          col = static_cast<uint32_t>(at) / static_cast<uint32_t>(a.ps);
        } else {
          col = at / a.ps;
        }
        at -= col * a.ps;
        const int64_t page = col < a.P ? a.table[lreq * a.tstride + col] : -1;
        if (page >= 0 && page < a.pages) {
          const int st = second ? 2 : 0;
          crow = (second ? a.cb : a.ca) + (page * a.pstride[st] + at * a.rstride[st]) * SIZE;
          zrow = (second ? a.zb : a.za) + (page * a.pstride[st + 1] + at * a.rstride[st + 1]) * SIZE;
          brow = reinterpret_cast<const char*>((second ? a.bb : a.ba) + jj * a.C);
        }
      }
      row_lds[0][threadIdx.x] = crow;
      row_lds[1][threadIdx.x] = zrow;
      row_lds[2][threadIdx.x] = brow;
    }
    __syncthreads();
    const int here = live ? static_cast<int>(rows - base < ROWS ? rows - base : ROWS) : 0;
    for (int j0 = part; j0 < here; j0 += PARTS * U) {
      Piece<DT, N> zp[U], vp[U];
      Piece<0, N> bp[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int j = j0 + u * PARTS;
        const char* crow = j < here ? row_lds[0][item * ROWS + (j & (ROWS - 1))] : nullptr;
        if (crow) {
          any = true;
          zp[u].load(row_lds[1][item * ROWS + (j & (ROWS - 1))] + c * SIZE);
          vp[u].load(crow + c * SIZE);
          bp[u].load(row_lds[2][item * ROWS + (j & (ROWS - 1))] + c * 4);
        } else {
          zp[u].fill(-__builtin_inff());
          vp[u].fill(0.f);
          bp[u].fill(0.f);
        }
      }
#pragma unroll
      for (int i = 0; i < N; ++i) {
        float m = mx[i], z[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          z[u] = zp[u].at(i) + bp[u].at(i);
          m = __builtin_fmaxf(m, z[u]);
        }
        // (the difference comes first: m kLog2e overflows for a gate masked with the type's lowest value, and its rounding would
        // differ from part to part)
        const float ref = m == -__builtin_inff() ? 0.f : m;
        const float s = __builtin_amdgcn_exp2f((mx[i] - ref) * kLog2e);
        den[i] *= s;
        num[i] *= s;
        mx[i] = m;
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const float w = __builtin_amdgcn_exp2f((z[u] - ref) * kLog2e);
          den[i] += w;
          num[i] = __builtin_fmaf(w, vp[u].at(i), num[i]);
        }
      }
    }
  }
  // Join the parts: lanes 8, 16, 32 apart, the maxima first, so that a thread rescales its sums once; then the waves of an
  // entry.  (With a rescale in every step, 96 of a thread's 128 exponentials were the joins', with 32 parts.)
  float top[N];
  if constexpr (PARTS > 1) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      top[i] = __builtin_fmaxf(mx[i], lane_away<8>(mx[i]));
      top[i] = __builtin_fmaxf(top[i], lane_away<16>(top[i]));
      if constexpr (PARTS >= 8) top[i] = __builtin_fmaxf(top[i], lane_away<32>(top[i]));
      const float w = top[i] == -__builtin_inff() ? 0.f : __expf(mx[i] - top[i]);
      den[i] *= w;
      num[i] *= w;
      den[i] += lane_away<8>(den[i]);
      num[i] += lane_away<8>(num[i]);
      den[i] += lane_away<16>(den[i]);
      num[i] += lane_away<16>(num[i]);
      if constexpr (PARTS >= 8) {
        den[i] += lane_away<32>(den[i]);
        num[i] += lane_away<32>(num[i]);
      }
    }
    float seen = any ? 1.f : 0.f;
    seen += lane_away<8>(seen);
    seen += lane_away<16>(seen);
    if constexpr (PARTS >= 8) seen += lane_away<32>(seen);
    any = seen != 0.f;
  }
  if constexpr (PARTS > 8) {
    constexpr int WAVES = PARTS / 8;
    __shared__ float lds[WAVES][8][3 * N + 1];
    const int wave = threadIdx.x >> 6;
    if ((threadIdx.x & 63) < 8) {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        lds[wave][vg][i] = top[i];
        lds[wave][vg][N + i] = den[i];
        lds[wave][vg][2 * N + i] = num[i];
      }
      lds[wave][vg][3 * N] = any ? 1.f : 0.f;
    }
    __syncthreads();
    if (threadIdx.x < 8) {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        float m = top[i];
#pragma unroll
        for (int w = 1; w < WAVES; ++w) m = __builtin_fmaxf(m, lds[w][vg][i]);
        const float ref = m == -__builtin_inff() ? 0.f : m;
        const float s = __expf(top[i] - ref);
        den[i] *= s;
        num[i] *= s;
#pragma unroll
        for (int w = 1; w < WAVES; ++w) {
          const float sw = __expf(lds[w][vg][i] - ref);
          den[i] += lds[w][vg][N + i] * sw;
          num[i] += lds[w][vg][2 * N + i] * sw;
        }
      }
#pragma unroll
      for (int w = 1; w < WAVES; ++w) any = any || lds[w][vg][3 * N] != 0.f;
    }
  }
  if (live && part == 0) {
#pragma unroll
    for (int i = 0; i < N; ++i) num[i] = any ? num[i] / den[i] : 0.f;
    const int64_t page = slot / a.out_ps;
    const int64_t off = page * a.out_pstride + (slot - page * a.out_ps) * a.out_rstride + c;
    Piece<DT, N>::store(a.out + off * SIZE, num);
  }
}

template <int DT, int N, int PARTS>
static int launch_paged_compress_p(CompressArgs a, hipStream_t st) {
  constexpr int ITEMS = 32 / PARTS;
  const int64_t groups = (a.C / N + 7) / 8;
  const int64_t blocks = (a.E + ITEMS - 1) / ITEMS * groups;
  if (blocks > kMostBlocks) return set_error(SI_ERR_UNSUPPORTED, "tensor too large");
  a.groups = static_cast<int>(groups);
  hipLaunchKernelGGL((paged_compress_kernel<DT, N, PARTS>), dim3(static_cast<unsigned>(blocks)), dim3(256), 0, st, a);
  return check_launch("paged_compress_kernel");
}
template <int DT, int N>
static int launch_paged_compress_n(const CompressArgs& a, hipStream_t st) {
  // Parts of an entry, that is threads of a channel: the fewer, the less is spent on joining them; the more, the more loads of
  // few entries are in flight (us, C = 576, bf16: 8 tokens, 7,000 entries, 1 and 4 parts 30 and 47; 16, 6,000, 50 and 59; 32,
  // 1,000 entries, fp32, C = 500, 35 and 31).
  const int64_t tokens = (a.overlap ? 2 : 1) * a.m;
  if (tokens <= 16) return launch_paged_compress_p<DT, N, 1>(a, st);
  if (tokens < 64) return launch_paged_compress_p<DT, N, 4>(a, st);
  // 8 or 32: a list of which few entries are there (a decode step's, one row a request) wants 32 at any length, one whose entries
  // all are there 8 from some length on, sooner where entries have few tokens.  Only the length is known here, so the border
  // lies where either choice loses about the same (us with 8 and 32, bf16, all entries there / one in 128: 64 tokens, C = 128,
  // 256 rows 8.3, 8.7 / 6.8, 6.3, 1,024 rows 12.5, 20.2 / 7.4, 6.5; 128 tokens, C = 576, 128 rows 17.1, 16.7 / 10.1, 6.7, 256 rows
  // 21.0, 24.8 / 10.2, 6.8, 512 rows 40.5, 50.1 / 10.9, 6.9; 200 tokens, C = 64, 1,024 rows 20.6, 18.1 / 16.2, 7.9, 4,096 rows 49.8,
  // 63.1 / 16.3, 8.0; 512 tokens, C = 576, 128 rows 56.8, 45.2 / 29.5, 11.4).
  const int64_t many = tokens < 176 ? 32 * (tokens - 48) : 4096;  // workgroups of 32 parts
  return a.E * ((a.C / N + 7) / 8) >= many ? launch_paged_compress_p<DT, N, 8>(a, st) : launch_paged_compress_p<DT, N, 32>(a, st);
}
template <int DT>
static int launch_paged_compress(const CompressArgs& a, hipStream_t st) {
  constexpr int SIZE = DT == 0 ? 4 : 2;
  uintptr_t x = reinterpret_cast<uintptr_t>(a.out);
  int64_t s = (a.C | a.out_pstride | a.out_rstride) * SIZE;
  const char* p[4] = {a.ca, a.za, a.cb, a.zb};
  for (int i = 0; i < (a.overlap ? 4 : 2); ++i) {
    x |= reinterpret_cast<uintptr_t>(p[i]);
    s |= (a.pstride[i] | a.rstride[i]) * SIZE;
  }
  const uintptr_t b = reinterpret_cast<uintptr_t>(a.ba) | (a.overlap ? reinterpret_cast<uintptr_t>(a.bb) : 0);
  const bool bias = a.C % 4 == 0 && (b & 15) == 0;
  if (bias && ((x | static_cast<uintptr_t>(s)) & 15) == 0) return launch_paged_compress_n<DT, 16 / SIZE>(a, st);
  if constexpr (DT != 0) {
    if (bias && ((x | static_cast<uintptr_t>(s)) & 7) == 0) return launch_paged_compress_n<DT, 4>(a, st);
  }
  return launch_paged_compress_n<DT, 1>(a, st);
}

constexpr int64_t kMostRequests = int64_t{1} << 30;  // (a thread's share of the requests ends within 31 bits)
static bool too_big(int64_t x) { return x < 0 || x > 0x7fffffff; }

}  // namespace si

using namespace si;

extern "C" int si_paged_plan(const int32_t* ctx_lens, const int32_t* new_lens, int64_t R, int64_t ratio,
                             int32_t* block_table, int64_t table_stride, int64_t P, const int32_t* free_pages,
                             int64_t F, const int32_t* free_start, int64_t page_size, int64_t rows, int32_t* cu,
                             int32_t* seq_lens, int64_t* slots, int32_t* request, int32_t* positions,
                             int32_t* free_next, void* stream) {
  if (R < 0 || P < 0 || F < 0 || rows < 0 || ratio <= 0 || page_size <= 0)
    return set_error(SI_ERR_INVALID, "bad dimension");
  if (too_big(R) || too_big(P) || too_big(F) || too_big(rows) || too_big(ratio) || too_big(page_size))
    return set_error(SI_ERR_UNSUPPORTED, "dimension exceeds int32");
  if (R > kMostRequests) return set_error(SI_ERR_UNSUPPORTED, "more than 2^30 requests");
  if (!cu || !free_next || (R > 0 && (!ctx_lens || !new_lens || !seq_lens)) || (R > 0 && P > 0 && !block_table) ||
      (F > 0 && !free_pages) || (rows > 0 && (!slots || !request || !positions)))
    return set_error(SI_ERR_INVALID, "null pointer argument");
  if (R > 1 && table_stride < P) return set_error(SI_ERR_INVALID, "block table rows overlap");
  PlanArgs a{ctx_lens, new_lens, block_table, table_stride, free_pages, free_start, cu, seq_lens, request, positions,
             free_next, slots, static_cast<int>(R), static_cast<int>(P), static_cast<int>(F), static_cast<int>(rows),
             ratio, page_size, static_cast<int>((R + kPlanThreads - 1) / kPlanThreads)};
  int64_t blocks = (rows + kPlanThreads - 1) / kPlanThreads;
  blocks = blocks < 1 ? 1 : blocks > 256 ? 256 : blocks;
  hipLaunchKernelGGL(paged_plan_kernel, dim3(static_cast<unsigned>(blocks)), dim3(kPlanThreads), 0,
                     static_cast<hipStream_t>(stream), a);
  return check_launch("paged_plan_kernel");
}

extern "C" int si_paged_write(const void* rows, int64_t row_stride, const int64_t* slots, int64_t n, int64_t row_bytes,
                              void* cache, int64_t page_stride, int64_t slot_stride, int64_t pages, int64_t page_size,
                              void* stream) {
  if (n < 0 || row_bytes < 0 || pages < 0 || page_size <= 0 || row_stride < 0 || page_stride < 0 || slot_stride < 0)
    return set_error(SI_ERR_INVALID, "bad dimension");
  if (n == 0 || row_bytes == 0 || pages == 0) return SI_OK;
  if (!rows || !slots || !cache) return set_error(SI_ERR_INVALID, "null pointer argument");
  if (too_big(n) || too_big(row_bytes) || too_big(pages) || too_big(page_size))
    return set_error(SI_ERR_UNSUPPORTED, "dimension exceeds int32");
  WriteArgs a{static_cast<const char*>(rows), static_cast<char*>(cache), slots, row_stride, page_stride, slot_stride, 0,
              pages * page_size, page_size, 0, page_stride == page_size * slot_stride};
  hipStream_t st = static_cast<hipStream_t>(stream);
  const uint64_t x = reinterpret_cast<uintptr_t>(rows) | reinterpret_cast<uintptr_t>(cache) | static_cast<uint64_t>(row_stride) |
                     static_cast<uint64_t>(page_stride) | static_cast<uint64_t>(slot_stride) | static_cast<uint64_t>(row_bytes);
  if (!(x & 15)) return launch_write<u32x4>(a, n, row_bytes, st);
  if (!(x & 7)) return launch_write<uint64_t>(a, n, row_bytes, st);
  if (!(x & 3)) return launch_write<uint32_t>(a, n, row_bytes, st);
  if (!(x & 1)) return launch_write<uint16_t>(a, n, row_bytes, st);
  return launch_write<uint8_t>(a, n, row_bytes, st);
}

extern "C" int si_paged_compress(const void* c_a, const int64_t* ca_strides, const void* z_a, const int64_t* za_strides,
                                 const float* b_a, const void* c_b, const int64_t* cb_strides, const void* z_b,
                                 const int64_t* zb_strides, const float* b_b, int dtype, int64_t pages,
                                 int64_t page_size, int64_t C, int64_t m, const int32_t* block_table,
                                 int64_t table_stride, int64_t R, int64_t P, const int32_t* request,
                                 const int32_t* positions, const int64_t* slots, int64_t E, void* out,
                                 const int64_t* out_strides, int64_t out_pages, int64_t out_page_size, void* stream) {
  if (pages < 0 || page_size <= 0 || C < 0 || m <= 0 || R < 0 || P < 0 || E < 0 || out_pages < 0 || out_page_size <= 0)
    return set_error(SI_ERR_INVALID, "bad dimension");
  if (too_big(pages) || too_big(page_size) || too_big(C) || too_big(m) || too_big(R) || too_big(P) || too_big(E) ||
      too_big(out_pages) || too_big(out_page_size))
    return set_error(SI_ERR_UNSUPPORTED, "dimension exceeds int32");
  if (dtype < 0 || dtype > 2) return set_error(SI_ERR_UNSUPPORTED, "dtype must be fp32, bf16 or fp16");
  const bool overlap = c_b != nullptr || z_b != nullptr || b_b != nullptr;
  if (!ca_strides || !za_strides || !out_strides || (overlap && (!cb_strides || !zb_strides)))
    return set_error(SI_ERR_INVALID, "null stride argument");
  if (E == 0 || C == 0 || R == 0 || out_pages == 0) return SI_OK;
  if (!b_a || !request || !positions || !slots || !out || (P > 0 && !block_table) || (pages > 0 && (!c_a || !z_a)) ||
      (overlap && (!b_b || (pages > 0 && (!c_b || !z_b)))))
    return set_error(SI_ERR_INVALID, "null pointer argument");
  CompressArgs a{};
  a.ca = static_cast<const char*>(c_a); a.za = static_cast<const char*>(z_a);
  a.cb = static_cast<const char*>(c_b); a.zb = static_cast<const char*>(z_b);
  const int64_t* s[4] = {ca_strides, za_strides, overlap ? cb_strides : ca_strides, overlap ? zb_strides : za_strides};
  for (int i = 0; i < 4; ++i) {
    if (s[i][2] != 1 || s[i][0] < 0 || s[i][1] < 0)
      return set_error(SI_ERR_INVALID, "streams need a contiguous last dimension");
    a.pstride[i] = s[i][0];
    a.rstride[i] = s[i][1];
  }
  if (out_strides[2] != 1 || out_strides[0] < 0 || out_strides[1] < 0)
    return set_error(SI_ERR_INVALID, "the cache needs a contiguous last dimension");
  a.ba = b_a; a.bb = b_b;
  a.table = block_table; a.tstride = table_stride;
  a.request = request; a.entry = positions; a.slots = slots;
  a.out = static_cast<char*>(out);
  a.out_pstride = out_strides[0]; a.out_rstride = out_strides[1];
  a.nslots = out_pages * out_page_size; a.out_ps = out_page_size;
  a.E = E; a.C = C; a.m = m; a.ps = page_size;
  a.R = static_cast<int>(R); a.P = static_cast<int>(P); a.pages = static_cast<int>(pages);
  a.overlap = overlap ? 1 : 0;
  hipStream_t st = static_cast<hipStream_t>(stream);
  switch (dtype) {
    case 0: return launch_paged_compress<0>(a, st);
    case 1: return launch_paged_compress<1>(a, st);
    default: return launch_paged_compress<2>(a, st);
  }
}
