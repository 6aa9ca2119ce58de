// Rows into a paged cache held in 8 bits (e4m3), for gfx950.
//
// A block of tokens shares one scale, a power of two s = 2^e: the smallest with 448 s >= |x| for every finite x of the block's new
// rows, at least 2^-64, and no smaller than the scale of the earlier tokens that the block keeps.  A code is x / s to the
// nearest e4m3 value, ties to even; x / s is exact, so that is the only rounding.  Where s grows, the earlier codes become
// code * s_old / s, which loses what falls below 2^-9 of the new scale and nothing else.  Infinities and NaN become NaN and count
// for no scale.
//
// An earlier scale that another program set need not be a power of two; where it is large enough, it stays.  Quotients by it, and
// products of codes with it, take fp32's last bit as a sign that something is left, so that e4m3 is their only rounding too.
//
// A power of two costs e4m3 at most the lowest bit of its subnormal values, makes every code and its reading exact, and
// lets a block's scale grow without a second rounding of its normal values.
//
// Rows are read once and stay in registers between the maximum and the codes.  With a scale for each token 8 to 64 lanes
// share a row.  With a scale for each block a workgroup takes the blocks that begin in its share of the rows, one after the
// other, whole: a block's rows stand next to each other, as a plan's do.
//
// Bound, many rows: memory, with vector instructions in 52 % of the CUs' busy cycles.  Nine requests' bf16 rows of 576 values, 64
// tokens a page and a scale, 133 MB read and written: 27.6 us, 4.8 TB/s; with a scale for each token 21.4 us.  (Divisions for every piece, rows read a second time: 50;
// 180 registers a lane and half the waves: 38.)  Few rows: latency.  256 single rows into blocks of 16: 5.3 us.
#include <hip/hip_fp16.h>

#include <string>
#include <type_traits>

#include "si_common.h"
#include "si_status.h"

namespace si {

struct WriteQArgs {
  const char* rows;
  int64_t rstride;  // elements
  const int64_t* slots;
  uint8_t* codes;
  int64_t pstride, cstride;  // bytes: page and row
  float* scales;
  int64_t spage;             // floats: page
  int64_t nslots;
  int64_t n;                 // rows
  uint32_t ps, block, pieces;  // tokens of a page and of a block, pieces of a row
  int log_lpr, chunk;
};

constexpr int kLeastExp = -64;
constexpr int kRowThreads = 256;    // kernel of one token a scale
constexpr int kBlockThreads = 512;  // kernel of blocks
constexpr int kHeld = 9;            // pieces of a row that a lane holds in registers; those behind are read twice
constexpr int kHeldRows = 10;       // rows of a block of which a thread holds a piece: 64 of 72 pieces over 512 threads

template <int DT>
struct WqElem;
template <>
struct WqElem<0> {
  typedef float T;
};
template <>
struct WqElem<1> {
  typedef __bf16 T;
};
template <>
struct WqElem<2> {
  typedef _Float16 T;
};
template <int DT, int V>
struct WqPiece {
  typedef typename WqElem<DT>::T T;
  static constexpr int N = V * sizeof(T) > 16 ? 2 : 1, W = V / N;  // loads of up to 16 bytes
  typedef T vec __attribute__((ext_vector_type(W)));
  vec w[N];
  __device__ __forceinline__ void load(const char* p) {
#pragma unroll
    for (int i = 0; i < N; ++i) w[i] = reinterpret_cast<const vec*>(p)[i];
  }
  __device__ __forceinline__ float at(int e) const { return static_cast<float>(w[e / W][e % W]); }
};
template <int DT>
struct WqPiece<DT, 1> {
  typedef typename WqElem<DT>::T T;
  T w;
  __device__ __forceinline__ void load(const char* p) { w = *reinterpret_cast<const T*>(p); }
  __device__ __forceinline__ float at(int) const { return static_cast<float>(w); }
};

// Magnitudes are compared as their bits, 16-bit ones two at a time; a lane's largest is that of both halves.
template <int DT, int V>
__device__ __forceinline__ uint32_t wq_max(const WqPiece<DT, V>& p, uint32_t m) {
  if constexpr (DT == 0) {
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const uint32_t x = __float_as_uint(p.at(e)) & 0x7fffffffu;
      m = x > m ? x : m;
    }
    return m;
  } else {
    typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
    uint32_t w[V == 1 ? 1 : V / 2];
    if constexpr (V == 1) w[0] = __builtin_bit_cast(uint16_t, p.w);
    else __builtin_memcpy(w, &p.w, sizeof(w));
#pragma unroll
    for (uint32_t x : w)
      m = __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, m),
                                                                 __builtin_bit_cast(u16x2, x & 0x7fff7fffu)));
    return m;
  }
}
// The larger half, and the value of such bits.
template <int DT>
__device__ __forceinline__ uint32_t wq_half(uint32_t m) {
  if constexpr (DT == 0) return m;
  const uint32_t lo = m & 0xffffu, hi = m >> 16;
  return lo > hi ? lo : hi;
}
template <int DT>
__device__ __forceinline__ float wq_value(uint32_t bits) {
  if constexpr (DT == 0) return __uint_as_float(bits);
  else if constexpr (DT == 1) return __uint_as_float(bits << 16);
  else return static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(bits)));
}
template <int DT>
constexpr uint32_t kWqInf = DT == 0 ? 0x7f800000u : DT == 1 ? 0x7f80u : 0x7c00u;
// The same of the finite values alone: rows that hold others go through this.
template <int DT, int V>
__device__ __forceinline__ uint32_t wq_max_finite(const WqPiece<DT, V>& p, uint32_t m) {
#pragma unroll
  for (int e = 0; e < V; ++e) {
    uint32_t x;
    if constexpr (DT == 0) x = __float_as_uint(p.at(e));
    else if constexpr (DT == 1) x = __float_as_uint(p.at(e)) >> 16;
    else x = __builtin_bit_cast(uint16_t, static_cast<_Float16>(p.at(e)));
    x &= DT == 0 ? 0x7fffffffu : 0x7fffu;
    m = x < kWqInf<DT> && x > m ? x : m;
  }
  return m;
}
// e of the smallest 2^e, from 2^-64 on, with 448 2^e >= m (448 = 0.875 2^9).
__device__ __forceinline__ int wq_exp(float m) {
  const uint32_t b = __float_as_uint(m);
  // m = f 2^(q - 126), f in [1/2, 1), for normal m; smaller ones need no more than 2^-64
  const int q = static_cast<int>(b >> 23) - 126 - 9;
  const int e = (b & 0x7fffffu) > 0x600000u ? q + 1 : q;  // f > 0.875
  return e > kLeastExp ? e : kLeastExp;
}
__device__ __forceinline__ float wq_pow2(int e) { return __uint_as_float(static_cast<uint32_t>(e + 127) << 23); }

// q, the fp32 value nearest to q + rest, with its last bit set where that is not zero: rounded to fewer bits, this is as q + rest
// rounded once.
__device__ __forceinline__ float wq_odd(float q, float rest) {
  const uint32_t b = __float_as_uint(q);
  const bool more = rest > 0.f || rest < 0.f;
  return more && q != 0.f && !(b & 1) ? __uint_as_float((rest > 0.f) == (q > 0.f) ? b + 1 : b - 1) : q;
}
// x / s and x s for a rounding to e4m3, whatever s > 0.  (Where fma's result falls below fp32's range the code is zero anyway.)
__device__ __forceinline__ float wq_quotient(float x, float s) {
  const float q = x / s;
  return wq_odd(q, __builtin_fmaf(-q, s, x));
}
__device__ __forceinline__ float wq_product(float x, float s) {
  const float q = x * s;
  return wq_odd(q, __builtin_fmaf(x, s, -q));
}

template <int V, typename P>
__device__ __forceinline__ void wq_store(uint8_t* dst, const P& p, float inv) {
  if constexpr (V == 1) {
    *dst = static_cast<uint8_t>(__builtin_amdgcn_cvt_pk_fp8_f32(p.at(0) * inv, 0.f, 0, false));
  } else {
    int w[V / 4];
#pragma unroll
    for (int i = 0; i < V / 4; ++i) {
      int x = __builtin_amdgcn_cvt_pk_fp8_f32(p.at(4 * i) * inv, p.at(4 * i + 1) * inv, 0, false);
      w[i] = __builtin_amdgcn_cvt_pk_fp8_f32(p.at(4 * i + 2) * inv, p.at(4 * i + 3) * inv, x, true);
    }
    if constexpr (V == 8) *reinterpret_cast<uint2*>(dst) = uint2{static_cast<uint32_t>(w[0]), static_cast<uint32_t>(w[1])};
    else *reinterpret_cast<uint32_t*>(dst) = static_cast<uint32_t>(w[0]);
  }
}
struct WqSlot {
  int64_t page;
  uint32_t off;
};
__device__ __forceinline__ WqSlot wq_slot(const WriteQArgs& a, int64_t slot) {
  if (a.nslots <= 0x7fffffff) {
    const uint32_t p = static_cast<uint32_t>(slot) / a.ps;
    return WqSlot{p, static_cast<uint32_t>(slot) - p * a.ps};
  }
  const int64_t p = slot / a.ps;
  return WqSlot{p, static_cast<uint32_t>(slot - p * a.ps)};
}

// One token a scale.
template <int DT, int V>
__global__ __launch_bounds__(kRowThreads) void paged_write_q_rows_kernel(WriteQArgs a) {
  typedef WqPiece<DT, V> P;
  constexpr int SIZE = DT == 0 ? 4 : 2;
  const int lpr = 1 << a.log_lpr, lane = threadIdx.x & (lpr - 1);
  const int64_t row = static_cast<int64_t>(blockIdx.x) * (kRowThreads >> a.log_lpr) + (threadIdx.x >> a.log_lpr);
  if (row >= a.n) return;
  const char* src = a.rows + row * a.rstride * SIZE;
  P held[kHeld];
#pragma unroll
  for (int c = 0; c < kHeld; ++c) {
    const uint32_t i = c * lpr + lane;
    if (i < a.pieces) held[c].load(src + static_cast<int64_t>(i) * (V * SIZE));
  }
  const int64_t slot = a.slots[row];
  if (slot < 0 || slot >= a.nslots) return;
  const WqSlot at = wq_slot(a, slot);
  auto largest = [&](auto&& of) {
    uint32_t m = 0;
#pragma unroll
    for (int c = 0; c < kHeld; ++c)
      if (static_cast<uint32_t>(c * lpr + lane) < a.pieces) m = of(held[c], m);
    for (uint32_t i = kHeld * lpr + lane; i < a.pieces; i += lpr) {
      P p;
      p.load(src + static_cast<int64_t>(i) * (V * SIZE));
      m = of(p, m);
    }
    m = wq_half<DT>(m);
    for (int k = 1; k < lpr; k *= 2) {
      const uint32_t x = __shfl_xor(m, k);
      m = x > m ? x : m;
    }
    return m;
  };
  uint32_t m = largest([](const P& p, uint32_t x) { return wq_max<DT, V>(p, x); });
  if (__builtin_expect(m >= kWqInf<DT>, 0)) m = largest([](const P& p, uint32_t x) { return wq_max_finite<DT, V>(p, x); });
  const int e = wq_exp(wq_value<DT>(m));
  const float inv = wq_pow2(-e);
  uint8_t* dst = a.codes + at.page * a.pstride + at.off * a.cstride;
#pragma unroll
  for (int c = 0; c < kHeld; ++c) {
    const uint32_t i = c * lpr + lane;
    if (i < a.pieces) wq_store<V>(dst + static_cast<int64_t>(i) * V, held[c], inv);
  }
  for (uint32_t i = kHeld * lpr + lane; i < a.pieces; i += lpr) {
    P p;
    p.load(src + static_cast<int64_t>(i) * (V * SIZE));
    wq_store<V>(dst + static_cast<int64_t>(i) * V, p, inv);
  }
  if (lane == 0) a.scales[at.page * a.spage + at.off] = wq_pow2(e);
}

// A scale for each block.
template <int DT, int V>
__global__ __launch_bounds__(kBlockThreads, DT == 0 ? 2 : 4) void paged_write_q_blocks_kernel(WriteQArgs a) {
  typedef WqPiece<DT, V> P;
  constexpr int SIZE = DT == 0 ? 4 : 2, WAVES = kBlockThreads / kWave;
  __shared__ uint32_t max_lds[2][WAVES];
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  const int64_t r0 = static_cast<int64_t>(blockIdx.x) * a.chunk, r1 = r0 + a.chunk < a.n ? r0 + a.chunk : a.n;
  // A thread takes one piece of every step-th row of a run (rows of more pieces than threads: every 512th piece of each row).
  const uint32_t cols = a.pieces < kBlockThreads ? a.pieces : kBlockThreads, step = kBlockThreads / cols;
  const uint32_t tr = t / cols, tc = t - tr * cols;
  auto slot_at = [&](int64_t r) {
    const int64_t s = r >= 0 && r < a.n ? a.slots[r] : -1;
    return s < a.nslots ? s : -1;
  };
  // Two rows are of one run if they stand in one block in rising order with no other slot and fewer than 64 rows between them.
  // Of the row before this lane's that has a slot, among the lanes below or, before them, row `at` with `slot`:
  auto before = [&](int64_t mine, int64_t w, int64_t slot, int64_t at, int64_t& prev) {
    const uint64_t below = __builtin_amdgcn_ballot_w64(mine >= 0) & ((1ull << lane) - 1);
    const int from = below ? 63 - __builtin_clzll(below) : 0;
    const int64_t s = __shfl(mine, from);
    prev = below ? s : slot;
    return w + lane - (below ? w + from : at) <= kWave;  // near enough
  };
  for (int64_t r = r0; r < r1;) {
    // the next row that begins a run, by every wave for itself: all find the same
    const int64_t back = slot_at(r - kWave + lane), mine = r + lane < r1 ? slot_at(r + lane) : -1;
    const uint64_t there = __builtin_amdgcn_ballot_w64(back >= 0);
    const int last_back = there ? 63 - __builtin_clzll(there) : 0;
    const int64_t back_slot = there ? __shfl(back, last_back) : -1;
    int64_t prev;
    const bool near = before(mine, r, back_slot, r - kWave + last_back, prev);
    const uint32_t inside = mine >= 0 ? wq_slot(a, mine).off % a.block : 0;
    const bool goes_on = near && prev >= 0 && prev < mine && mine - prev <= inside;
    const uint64_t begins = __builtin_amdgcn_ballot_w64(mine >= 0 && !goes_on);
    if (begins == 0) {
      r += kWave;
      continue;
    }
    const int k0 = __builtin_ctzll(begins);
    r += k0;
    const int64_t slot = __shfl(mine, k0);
    const WqSlot at = wq_slot(a, slot);
    const uint32_t blk = at.off / a.block, first = at.off - blk * a.block;
    // its rows, up to the last one with a slot
    int run = 1;
    bool gaps = false, apart = false;  // rows without a slot; slots that do not follow each other
    {
      const int64_t end = slot + (a.block - first);
      int64_t last = slot;
      for (int64_t w = r + 1;; w += kWave) {
        const int64_t next = slot_at(w + lane);
        int64_t prev2;
        const bool near2 = before(next, w, last, r + run - 1, prev2);
        const uint64_t stop = __builtin_amdgcn_ballot_w64(next >= 0 && !(near2 && next > prev2 && next < end));
        const uint64_t mask = stop ? (stop & (0 - stop)) - 1 : ~0ull;  // the lanes before the first that is not of the run
        const uint64_t ours = __builtin_amdgcn_ballot_w64(next >= 0) & mask;
        if (ours) {
          const int to = 63 - __builtin_clzll(ours);
          apart = apart || (__builtin_amdgcn_ballot_w64(next >= 0 && next != prev2 + 1) & mask);
          gaps = gaps || w - (r + run) + to + 1 != __builtin_popcountll(ours);
          run = static_cast<int>(w - r) + to + 1;
          last = __shfl(next, to);
        }
        if (stop || !ours) break;
      }
    }
    const float old = first > 0 ? a.scales[at.page * a.spage + blk] : 0.f;  // (in front of joined()'s barrier: it is overwritten behind)
    uint8_t* base = a.codes + at.page * a.pstride + static_cast<int64_t>(blk) * a.block * a.cstride;
    const uint32_t rows = static_cast<uint32_t>(run);
    const bool hold = a.pieces <= kBlockThreads && rows <= kHeldRows * step && !gaps && !apart;  // (the same in every thread)
    auto source = [&](uint32_t row, uint32_t c) { return a.rows + ((r + row) * a.rstride + static_cast<int64_t>(c) * V) * SIZE; };
    auto has_slot = [&](uint32_t row) { return !gaps || slot_at(r + row) >= 0; };
    // rows that are not held, piece by piece
    auto each = [&](auto&& f) {
      if (tr < step)
#pragma unroll 1
        for (uint32_t row = tr; row < rows; row += step) {
          if (!has_slot(row)) continue;
          for (uint32_t c = tc; c < a.pieces; c += kBlockThreads) {
            P p;
            p.load(source(row, c));
            f(row, c, p);
          }
        }
    };
    // (an opaque copy of the first row: what depends on it alone would be kept in registers from run to run)
    uint32_t row0 = tr < step ? tr : 0x7fffffffu;
    asm volatile("" : "+v"(row0));
    P held[kHeldRows];
    if (hold) {
      const char* at0 = source(tr, tc);
      const int64_t rise = step * a.rstride * SIZE;
      uint32_t row = row0;
#pragma unroll
      for (int k = 0; k < kHeldRows; ++k) {
        if (row < rows) held[k].load(at0);
        row += step;
        at0 += rise;
      }
    }
    auto joined = [&](uint32_t x, uint32_t* lds) {  // the largest of all threads
      x = wave_max_u32(x);
      if (lane == 0) lds[wave] = x;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < WAVES; ++w) x = lds[w] > x ? lds[w] : x;
      return x;
    };
    uint32_t m = 0;
    if (hold) {
      uint32_t row = row0;
#pragma unroll
      for (int k = 0; k < kHeldRows; ++k) {
        if (row < rows) m = wq_max<DT, V>(held[k], m);
        row += step;
      }
    } else {
      each([&](uint32_t, uint32_t, const P& p) { m = wq_max<DT, V>(p, m); });
    }
    m = joined(wq_half<DT>(m), max_lds[0]);
    if (__builtin_expect(m >= kWqInf<DT>, 0)) {  // (the same in every thread)
      m = 0;
      each([&](uint32_t, uint32_t, const P& p) { m = wq_max_finite<DT, V>(p, m); });
      m = joined(m, max_lds[1]);
    }
    const float need = wq_pow2(wq_exp(wq_value<DT>(m)));
    const bool kept = old > 0.f && old < __builtin_inff();  // (earlier tokens with a scale that is one)
    const float scale = kept && old > need ? old : need, inv = 1.0f / scale;
    auto place = [&](uint32_t row, uint32_t c) {
      const int64_t s = row ? slot_at(r + row) : slot;
      return base + (first + (s - slot)) * a.cstride + static_cast<int64_t>(c) * V;
    };
    if (__builtin_expect(__float_as_uint(scale) & 0x7fffffu, 0)) {
      // an earlier scale that is no power of two (the same in every thread): value by value, a rare path that takes no registers
      if (tr < step)
#pragma unroll 1
        for (uint32_t row = tr; row < rows; row += step) {
          if (!has_slot(row)) continue;
#pragma unroll 1
          for (uint32_t c = tc; c < a.pieces; c += kBlockThreads) {
            const char* from = source(row, c);
            uint8_t* to = place(row, c);
#pragma unroll 1
            for (int e = 0; e < V; ++e) {
              WqPiece<DT, 1> x;
              x.load(from + e * SIZE);
              to[e] = static_cast<uint8_t>(__builtin_amdgcn_cvt_pk_fp8_f32(wq_quotient(x.at(0), scale), 0.f, 0, false));
            }
          }
        }
    } else if (hold) {
      uint8_t* to = base + (first + tr) * a.cstride + static_cast<int64_t>(tc) * V;
      const int64_t rise = step * a.cstride;
      uint32_t row = row0;
#pragma unroll
      for (int k = 0; k < kHeldRows; ++k) {
        if (row < rows) wq_store<V>(to, held[k], inv);
        row += step;
        to += rise;
      }
    } else {
      each([&](uint32_t row, uint32_t c, const P& p) { wq_store<V>(place(row, c), p, inv); });
    }
    if (kept && scale > old) {  // earlier tokens to the new scale
      const float ratio = old / scale;
      for (uint32_t i = t; i < first * a.pieces; i += kBlockThreads) {
        const uint32_t row = i / a.pieces, c = i - row * a.pieces;
        uint8_t* p = base + row * a.cstride + static_cast<int64_t>(c) * V;
#pragma unroll
        for (int e = 0; e < V; e += V < 4 ? 1 : 4) {
          if constexpr (V == 1) {
            const float x = wq_product(__builtin_amdgcn_cvt_f32_fp8(*p, 0), ratio);
            *p = static_cast<uint8_t>(__builtin_amdgcn_cvt_pk_fp8_f32(x, 0.f, 0, false));
          } else {
            const int w = *reinterpret_cast<const int*>(p + e);
            const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8(w, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8(w, true);
            int x = __builtin_amdgcn_cvt_pk_fp8_f32(wq_product(lo[0], ratio), wq_product(lo[1], ratio), 0, false);
            x = __builtin_amdgcn_cvt_pk_fp8_f32(wq_product(hi[0], ratio), wq_product(hi[1], ratio), x, true);
            *reinterpret_cast<int*>(p + e) = x;
          }
        }
      }
    }
    // (every thread asked for the old scale before joined()'s barrier, which this store stands behind)
    if (t == 0) a.scales[at.page * a.spage + blk] = scale;
    __syncthreads();  // max_lds is free, and a later run of this workgroup sees this one's codes and scale
    r += run;
  }
}

}  // namespace si

using namespace si;

extern "C" int si_paged_write_q(const void* rows, int64_t row_stride, int dtype, const int64_t* slots, int64_t n, int64_t D,
                                void* codes, int64_t page_stride, int64_t slot_stride, float* scales, int64_t scale_stride,
                                int64_t pages, int64_t page_size, int64_t block, void* stream) {
  if (dtype < 0 || dtype > 2) return set_error(SI_ERR_UNSUPPORTED, "dtype must be 0 (fp32), 1 (bf16) or 2 (fp16)");
  if (n < 0 || D <= 0 || pages < 0 || page_size <= 0 || block <= 0 || page_size % block || row_stride < 0)
    return set_error(SI_ERR_INVALID, "bad dimension");
  if (n > 0x7fffffff || page_size > 0x7fffffff || pages > 0x7fffffff || D > (1 << 20))
    return set_error(SI_ERR_UNSUPPORTED, "dimension exceeds int32 or width 2^20");
  if (n > 0 && pages > 0 && (!rows || !slots || !codes || !scales)) return set_error(SI_ERR_INVALID, "null pointer argument");
  if (slot_stride < D || (pages > 1 && (page_stride < slot_stride * (page_size - 1) + D || scale_stride < page_size / block)))
    return set_error(SI_ERR_INVALID, "rows, pages or scales of the cache overlap");
  if (n == 0 || pages == 0) return SI_OK;
  const int size = dtype == 0 ? 4 : 2;
  int vec = 1;
  for (int v = 8; v > 1; v /= 2) {
    if (v == 2) continue;
    const int64_t load = v * size > 16 ? 16 : v * size;
    if (D % v == 0 && row_stride * size % load == 0 && reinterpret_cast<uintptr_t>(rows) % load == 0 && page_stride % v == 0 &&
        slot_stride % v == 0 && reinterpret_cast<uintptr_t>(codes) % v == 0) {
      vec = v;
      break;
    }
  }
  // (a run has at most 64 rows for each of its slots, counted in 31 bits, and a block's pieces are counted in 32)
  if (block > 1 << 24 || block * (D / vec) > 0x7fffffff) return set_error(SI_ERR_UNSUPPORTED, "blocks of more than 2^24 tokens");
  WriteQArgs a{};
  a.rows = static_cast<const char*>(rows);
  a.rstride = row_stride;
  a.slots = slots;
  a.codes = static_cast<uint8_t*>(codes);
  a.pstride = page_stride;
  a.cstride = slot_stride;
  a.scales = scales;
  a.spage = scale_stride;
  a.nslots = pages * page_size;
  a.n = n;
  a.ps = static_cast<uint32_t>(page_size);
  a.block = static_cast<uint32_t>(block);
  a.pieces = static_cast<uint32_t>(D / vec);
  a.log_lpr = 3;
  while (a.log_lpr < 6 && (static_cast<int64_t>(kHeld) << a.log_lpr) < a.pieces) ++a.log_lpr;
  a.chunk = 1;
  while (a.chunk * 2 <= block && n / (a.chunk * 2) >= 1024) a.chunk *= 2;
  hipStream_t st = static_cast<hipStream_t>(stream);
  auto launch = [&](auto DT, auto V) {
    constexpr int dt = decltype(DT)::value, v = decltype(V)::value;
    if (block == 1) {
      const int64_t per = kRowThreads >> a.log_lpr, blocks = (n + per - 1) / per;
      if (blocks > 0xffffffffLL / kRowThreads) return set_error(SI_ERR_UNSUPPORTED, "too many rows for one launch");
      hipLaunchKernelGGL((paged_write_q_rows_kernel<dt, v>), dim3(static_cast<unsigned>(blocks)), dim3(kRowThreads), 0, st, a);
      return check_launch("paged_write_q_rows_kernel");
    }
    const int64_t blocks = (n + a.chunk - 1) / a.chunk;
    if (blocks > 0xffffffffLL / kBlockThreads) return set_error(SI_ERR_UNSUPPORTED, "too many rows for one launch");
    hipLaunchKernelGGL((paged_write_q_blocks_kernel<dt, v>), dim3(static_cast<unsigned>(blocks)), dim3(kBlockThreads), 0, st, a);
    return check_launch("paged_write_q_blocks_kernel");
  };
  using std::integral_constant;
  auto of_type = [&](auto DT) {
    switch (vec) {
      case 8: return launch(DT, integral_constant<int, 8>{});
      case 4: return launch(DT, integral_constant<int, 4>{});
      default: return launch(DT, integral_constant<int, 1>{});
    }
  };
  switch (dtype) {
    case 0: return of_type(integral_constant<int, 0>{});
    case 1: return of_type(integral_constant<int, 1>{});
    default: return of_type(integral_constant<int, 2>{});
  }
}
