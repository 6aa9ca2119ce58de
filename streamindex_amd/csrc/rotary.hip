// Norm and rotation of the heads' rows for gfx950.
//
//   n = x r,  r = (mean(x^2) + eps)^-1/2 over the D values of a row (one head of one token),  z = n w  (without norm z = x),
//   y = z, but in the rotary dimensions, pair by pair, (a', b') = m (a cos t - b sin t, a sin t + b cos t),  t = p f_i,
//
// at position p, with frequencies f_i in radians a position and pairs of neighbours (a, b = z[2i], z[2i + 1]) or of halves
// (z[i], z[i + pairs]).  The gradient turns back, d = m (rotation by -t) dy, and
//
//   dw = sum over the rows of d n,   dx = r (d w - n mean(d w n)).
//
// Everything is fp32, rounded once at the end, but the angle: p f_i and its place within a turn are 64-bit, since 2^31
// positions times a frequency near one leave nothing of the fraction in 32.  No counterpart in the reference, which takes
// rotated queries (flash_sparse/csa.py:184).
//
// LPR lanes share a row, each with CPL pieces of 16 bytes (or the widest that every row start and every pair allows), LPR
// apart, so that neighbouring lanes read neighbouring pieces.  The row stays in registers between the sum of squares and the
// result.  The partner piece of a pair of halves is read again, from the cache.
//
// Bound: memory.  bf16, 4,096 tokens, 64 heads, D = 576 (302 MB in, 302 out): 113 us, 5.3 TB/s, what a large copy reaches; backward
// with dw 195 + 5 us (604 MB in, 302 out, 4.5 TB/s; 27,405 tokens 1,248 + 6 us, 4.8 TB/s).  fp16, 16,001 tokens, 24 heads of 128, rotated in halves (98 MB each way):
// 32.6 us, 6.0 TB/s, some of it from the last-level cache (42 us with cold caches); vector instructions and the LDS fill 70 % of the busy cycles
// there, the latter mostly with bank conflicts, but a table read without them was no faster (32.8 against 33.4).
#include <hip/hip_fp16.h>

#include <string>
#include <type_traits>

#include "rotary_plan.h"
#include "si_common.h"
#include "si_status.h"

namespace si {

struct RotArgs {
  const char* x;   // [T, H, D]; the forward's input
  const char* dy;  // backward: the gradient of y
  char* out;       // y, or dx, contiguous
  int64_t xst, xsh, dst, dsh;  // elements: token and head of x and of dy
  const float* weight;         // [D] or null
  const void* pos;             // [npos]; token t is at pos[t % npos]
  const double* freqs;         // [pairs]
  float* part;                 // backward with a weight: [gridDim.x, D] partial sums of dw
  int64_t rows;                // T * H
  int64_t npos;
  int H, D, pairs, start;      // dimensions [start, start + 2 pairs) are turned
  int pos64, halves, lpr, log_lpr;
  int iters;                   // groups of rows of a workgroup
  int per;                     // of them for each filling of the table
  int tokens;                  // of those at most
  int weight_lds;              // floats of LDS for the weight, in front of the table
  float magnitude, sign, eps;
};

template <int DT>
struct RotElem;
template <>
struct RotElem<0> {
  typedef float T;
};
template <>
struct RotElem<1> {
  typedef __bf16 T;
};
template <>
struct RotElem<2> {
  typedef _Float16 T;
};

template <int DT, int V>
struct RotPiece {
  typedef typename RotElem<DT>::T T;
  typedef T vec __attribute__((ext_vector_type(V)));
  vec w;
  __device__ __forceinline__ void load(const char* base, int64_t element) {
    w = *reinterpret_cast<const vec*>(base + element * static_cast<int64_t>(sizeof(T)));
  }
  __device__ __forceinline__ float at(int e) const { return static_cast<float>(w[e]); }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int e = 0; e < V; ++e) w[e] = static_cast<T>(0.f);
  }
};
template <int DT>
struct RotPiece<DT, 1> {
  typedef typename RotElem<DT>::T T;
  T w;
  __device__ __forceinline__ void load(const char* base, int64_t element) {
    w = *reinterpret_cast<const T*>(base + element * static_cast<int64_t>(sizeof(T)));
  }
  __device__ __forceinline__ float at(int) const { return static_cast<float>(w); }
  __device__ __forceinline__ void zero() { w = static_cast<T>(0.f); }
};
template <int DT, int V>
__device__ __forceinline__ void rot_store(char* base, int64_t element, const float (&v)[V]) {
  typedef typename RotElem<DT>::T T;
  if constexpr (V == 1) {
    *reinterpret_cast<T*>(base + element * static_cast<int64_t>(sizeof(T))) = static_cast<T>(v[0]);
  } else {
    typedef T vec __attribute__((ext_vector_type(V)));
    vec w;
#pragma unroll
    for (int e = 0; e < V; ++e) w[e] = static_cast<T>(v[e]);
    *reinterpret_cast<vec*>(base + element * static_cast<int64_t>(sizeof(T))) = w;
  }
}

// m cos and m sin of pos * freq.  The product is taken in turns with its rounding error, so the fraction of a turn is off
// by 2^-53 of the turns at most.
__device__ __forceinline__ float2 rot_at(const RotArgs& a, int64_t pos, int pair) {
  constexpr double kTurn = 0.15915494309189535, kTurnLow = -9.839338337591243e-18;  // 1 / (2 pi) and what is left of it
  const double angle = static_cast<double>(pos) * a.freqs[pair];
  const double turns = angle * kTurn;
  const double error = __builtin_fma(angle, kTurn, -turns) + angle * kTurnLow;
  const float part = static_cast<float>((turns - __builtin_rint(turns)) + error);
  float s, c;
  sincospif(2.0f * part, &s, &c);
  return float2{c * a.magnitude, s * (a.magnitude * a.sign)};
}
__device__ __forceinline__ int64_t rot_pos(const RotArgs& a, int64_t token) {
  const int64_t i = token < a.npos ? token : (token | a.npos) <= 0x7fffffff
                        ? static_cast<int64_t>(static_cast<uint32_t>(token) % static_cast<uint32_t>(a.npos))
                        : token % a.npos;
  return a.pos64 ? static_cast<const int64_t*>(a.pos)[i] : static_cast<int64_t>(static_cast<const int32_t*>(a.pos)[i]);
}
__device__ __forceinline__ void rot_row(const RotArgs& a, int64_t row, int64_t& token, int& head) {
  if (a.rows <= 0x7fffffff) {
    const uint32_t t = static_cast<uint32_t>(row) / static_cast<uint32_t>(a.H);
    token = t;
    head = static_cast<int>(static_cast<uint32_t>(row) - t * static_cast<uint32_t>(a.H));
  } else {
    token = row / a.H;
    head = static_cast<int>(row - token * a.H);
  }
}
// The sum over the 2^log lanes of a row.
__device__ __forceinline__ float rot_sum(float x, int log) {
  for (int m = 1; m < (1 << log); m *= 2) x += __shfl_xor(x, m);
  return x;
}

// Of the pieces of a row: which dimensions piece c of this lane holds, and whether they are turned.
template <int V>
struct RotPlace {
  int e0;       // first dimension
  bool there, turned, low;
  int partner;  // halves: first dimension of the partner piece
  int pair;     // of dimension e0
  __device__ __forceinline__ RotPlace(const RotArgs& a, int lane, int c) {
    e0 = (c * a.lpr + lane) * V;
    there = e0 < a.D;
    const int i = e0 - a.start;
    turned = there && i >= 0 && i < 2 * a.pairs;
    low = i < a.pairs;
    partner = low ? e0 + a.pairs : e0 - a.pairs;
    pair = a.halves ? (low ? i : i - a.pairs) : i >> 1;
  }
};

// The weights from dimension e0 on.
template <int V>
__device__ __forceinline__ void rot_weights(const RotArgs& a, const float* weight, int e0, float (&w)[V]) {
  if (!a.weight) {
#pragma unroll
    for (int e = 0; e < V; ++e) w[e] = 1.f;
  } else if constexpr (V % 4 == 0) {
#pragma unroll
    for (int i = 0; i < V / 4; ++i) {
      const f32x4 x = reinterpret_cast<const f32x4*>(weight + e0)[i];
#pragma unroll
      for (int e = 0; e < 4; ++e) w[4 * i + e] = x[e];
    }
  } else {
#pragma unroll
    for (int e = 0; e < V; ++e) w[e] = weight[e0 + e];
  }
}

// z turned, in place: v the piece's values; u those of its partner piece (halves).
template <int V, bool PAIRS>
__device__ __forceinline__ void rot_turn(const RotArgs& a, const RotPlace<V>& p, const float2* table, float (&v)[V],
                                         const float (&u)[V]) {
  if (a.halves || !PAIRS) {
#pragma unroll
    for (int e = 0; e < V; ++e) {
      // (one value at a time, neighbours are partners as halves are: the odd one's is in front of it)
      const bool first = a.halves ? p.low : ((p.e0 - a.start) & 1) == 0;
      const float2 t = table[a.halves ? p.pair + e : p.pair];
      v[e] = first ? __builtin_fmaf(v[e], t.x, -u[e] * t.y) : __builtin_fmaf(v[e], t.x, u[e] * t.y);
    }
  } else {
#pragma unroll
    for (int e = 0; e + 1 < V; e += 2) {
      const float2 t = table[p.pair + (e >> 1)];
      const float x = v[e], y = v[e + 1];
      v[e] = __builtin_fmaf(x, t.x, -y * t.y);
      v[e + 1] = __builtin_fmaf(x, t.y, y * t.x);
    }
  }
}

// The weight, at first, and the cosines and sines of the tokens from that of row row0 on, a.tokens of them, to LDS; all threads
// call it.  Returns the first token.
__device__ __forceinline__ int64_t rot_fill(const RotArgs& a, int64_t row0, float* weight, float2* table, bool at_first) {
  const int64_t token0 = row0 / a.H, last = (a.rows - 1) / a.H;
  if (at_first) {
    if (a.weight)
      for (int e = threadIdx.x; e < a.D; e += kRotThreads) weight[e] = a.weight[e];
  } else {
    if (a.pairs == 0) return 0;
    __syncthreads();  // (the table has been used)
  }
  for (int i = threadIdx.x; i < a.tokens * a.pairs; i += kRotThreads) {
    const int64_t token = token0 + static_cast<uint32_t>(i) / static_cast<uint32_t>(a.pairs);
    if (token <= last) table[i] = rot_at(a, rot_pos(a, token), static_cast<int>(static_cast<uint32_t>(i) % static_cast<uint32_t>(a.pairs)));
  }
  __syncthreads();
  return token0;
}

template <int DT, int V, int CPL, bool NORM>
__global__ __launch_bounds__(kRotThreads) void norm_rotary_kernel(RotArgs a) {
  extern __shared__ __attribute__((aligned(16))) float rot_lds[];
  float2* const all = reinterpret_cast<float2*>(rot_lds + a.weight_lds);
  const int lane = threadIdx.x & (a.lpr - 1), group = threadIdx.x >> a.log_lpr, groups = kRotThreads >> a.log_lpr;
  const int64_t row0 = static_cast<int64_t>(blockIdx.x) * a.iters * groups;
  int64_t token0 = 0;
  for (int it = 0; it < a.iters; ++it) {
    const int64_t first = row0 + static_cast<int64_t>(it) * groups, row = first + group;
    const bool live = row < a.rows;  // (the same in every lane of a row)
    int64_t token;
    int head;
    rot_row(a, live ? row : 0, token, head);
    const char* x = a.x;
    const int64_t at = token * a.xst + head * a.xsh;
    RotPiece<DT, V> piece[CPL];
#pragma unroll
    for (int c = 0; c < CPL; ++c) {
      const RotPlace<V> p(a, lane, c);
      if (live && p.there) piece[c].load(x, at + p.e0);
      else piece[c].zero();
    }
    if (it % a.per == 0) token0 = rot_fill(a, first, rot_lds, all, it == 0);
    if (!live) continue;
    float r = 1.f;
    if constexpr (NORM) {
      float sum = 0.f;
#pragma unroll
      for (int c = 0; c < CPL; ++c)
#pragma unroll
        for (int e = 0; e < V; ++e) sum = __builtin_fmaf(piece[c].at(e), piece[c].at(e), sum);
      sum = rot_sum(sum, a.log_lpr);
      r = 1.0f / __builtin_sqrtf(sum / static_cast<float>(a.D) + a.eps);
    }
    const float2* table = all + static_cast<int>(token - token0) * a.pairs;
    const int64_t to = row * a.D;
#pragma unroll
    for (int c = 0; c < CPL; ++c) {
      const RotPlace<V> p(a, lane, c);
      if (!p.there) continue;
      float v[V], u[V], w[V];
      if constexpr (NORM) rot_weights<V>(a, rot_lds, p.e0, w);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        v[e] = piece[c].at(e);
        if constexpr (NORM) v[e] *= r * w[e];
        u[e] = 0.f;
      }
      if (p.turned) {
        if (a.halves || V == 1) {
          const int other = a.halves ? p.partner : p.e0 + (((p.e0 - a.start) & 1) ? -1 : 1);
          RotPiece<DT, V> q;
          q.load(x, at + other);
          if constexpr (NORM) rot_weights<V>(a, rot_lds, other, w);
#pragma unroll
          for (int e = 0; e < V; ++e) {
            u[e] = q.at(e);
            if constexpr (NORM) u[e] *= r * w[e];
          }
        }
        rot_turn<V, (V > 1)>(a, p, table, v, u);
      }
      rot_store<DT, V>(a.out, to + p.e0, v);
    }
  }
}

// The gradients of a normed row.  Partial sums of dw stay in registers over the workgroup's rows; d is formed twice, from dy
// as it was loaded, which costs less than its registers.
template <int DT, int V, int CPL>
__global__ __launch_bounds__(kRotThreads, 2) void norm_rotary_bwd_kernel(RotArgs a) {
  extern __shared__ __attribute__((aligned(16))) float rot_lds[];
  float2* const all = reinterpret_cast<float2*>(rot_lds + a.weight_lds);
  const int lane = threadIdx.x & (a.lpr - 1), group = threadIdx.x >> a.log_lpr, groups = kRotThreads >> a.log_lpr;
  const int64_t row0 = static_cast<int64_t>(blockIdx.x) * a.iters * groups;
  int64_t token0 = 0;
  float dw[CPL][V];
#pragma unroll
  for (int c = 0; c < CPL; ++c)
#pragma unroll
    for (int e = 0; e < V; ++e) dw[c][e] = 0.f;
  for (int it = 0; it < a.iters; ++it) {
    const int64_t first = row0 + static_cast<int64_t>(it) * groups, row = first + group;
    const bool live = row < a.rows;
    int64_t token;
    int head;
    rot_row(a, live ? row : 0, token, head);
    const int64_t at = token * a.xst + head * a.xsh, dat = token * a.dst + head * a.dsh;
    RotPiece<DT, V> piece[CPL], grad[CPL];
#pragma unroll
    for (int c = 0; c < CPL; ++c) {
      const RotPlace<V> p(a, lane, c);
      if (live && p.there) {
        piece[c].load(a.x, at + p.e0);
        grad[c].load(a.dy, dat + p.e0);
      } else {
        piece[c].zero();
        grad[c].zero();
      }
    }
    if (it % a.per == 0) token0 = rot_fill(a, first, rot_lds, all, it == 0);
    if (!live) continue;
    const float2* table = all + static_cast<int>(token - token0) * a.pairs;
    auto gradient = [&](const RotPlace<V>& p, const RotPiece<DT, V>& g, float (&d)[V]) {
      float u[V];
#pragma unroll
      for (int e = 0; e < V; ++e) {
        d[e] = g.at(e);
        u[e] = 0.f;
      }
      if (p.turned) {
        if (a.halves || V == 1) {
          const int other = a.halves ? p.partner : p.e0 + (((p.e0 - a.start) & 1) ? -1 : 1);
          RotPiece<DT, V> q;
          q.load(a.dy, dat + other);
#pragma unroll
          for (int e = 0; e < V; ++e) u[e] = q.at(e);
        }
        rot_turn<V, (V > 1)>(a, p, table, d, u);
      }
    };
    float sum = 0.f, dot = 0.f;
#pragma unroll
    for (int c = 0; c < CPL; ++c) {
      const RotPlace<V> p(a, lane, c);
      if (!p.there) continue;
      float d[V], w[V];
      gradient(p, grad[c], d);
      rot_weights<V>(a, rot_lds, p.e0, w);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float x = piece[c].at(e);
        sum = __builtin_fmaf(x, x, sum);
        dot = __builtin_fmaf(d[e] * w[e], x, dot);
      }
    }
    sum = rot_sum(sum, a.log_lpr);
    dot = rot_sum(dot, a.log_lpr);
    const float inv = 1.0f / static_cast<float>(a.D);
    const float r = 1.0f / __builtin_sqrtf(sum * inv + a.eps), k = (r * dot * inv) * r;  // dx = r (d w - x k)
    const int64_t to = row * a.D;
#pragma unroll
    for (int c = 0; c < CPL; ++c) {
      const RotPlace<V> p(a, lane, c);
      if (!p.there) continue;
      float d[V], w[V], v[V];
      gradient(p, grad[c], d);
      rot_weights<V>(a, rot_lds, p.e0, w);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float x = piece[c].at(e);
        dw[c][e] = __builtin_fmaf(d[e], x * r, dw[c][e]);
        v[e] = r * (d[e] * w[e] - x * k);
      }
      rot_store<DT, V>(a.out, to + p.e0, v);
    }
  }
  if (!a.part) return;
  // over the rows of the wave, then over the waves
  __shared__ float sums[kRotThreads / kWave][kRotMostD];
  const int in_wave = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int c = 0; c < CPL; ++c) {
    const RotPlace<V> p(a, lane, c);
#pragma unroll
    for (int e = 0; e < V; ++e) {
      float s = dw[c][e];
      for (int m = a.lpr; m < kWave; m *= 2) s += __shfl_xor(s, m);
      if (in_wave < a.lpr && p.there) sums[wave][p.e0 + e] = s;
    }
  }
  __syncthreads();
  for (int e = threadIdx.x; e < a.D; e += kRotThreads)
    a.part[static_cast<int64_t>(blockIdx.x) * a.D + e] = (sums[0][e] + sums[1][e]) + (sums[2][e] + sums[3][e]);
}

// dw = the sum of the workgroups' parts, in a fixed order: 16 dimensions a workgroup, every 16th part a thread.
__global__ __launch_bounds__(256) void norm_rotary_dw_kernel(const float* part, int parts, int D, float* dw) {
  __shared__ float lds[16][17];
  const int e = threadIdx.x & 15, k = threadIdx.x >> 4, d = blockIdx.x * 16 + e;
  float s = 0.f;
  if (d < D) {
    constexpr int U = 8;  // in flight
    int i = k;
    for (; i + 16 * (U - 1) < parts; i += 16 * U) {
      float x[U];
#pragma unroll
      for (int u = 0; u < U; ++u) x[u] = part[static_cast<int64_t>(i + 16 * u) * D + d];
#pragma unroll
      for (int u = 0; u < U; ++u) s += x[u];
    }
    for (; i < parts; i += 16) s += part[static_cast<int64_t>(i) * D + d];
  }
  lds[k][e] = s;
  __syncthreads();
  if (k == 0 && d < D) {
    s = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) s += lds[i][e];
    dw[d] = s;
  }
}

}  // namespace si

using namespace si;

static int rot_check(const void* x, const int64_t* xs, const void* pos, int64_t npos, const void* freqs, int64_t pairs,
                     int64_t start, int64_t T, int64_t H, int64_t D, int dtype, const void* out) {
  if (dtype < 0 || dtype > 2) return set_error(SI_ERR_UNSUPPORTED, "dtype must be 0 (fp32), 1 (bf16) or 2 (fp16)");
  if (T < 0 || H <= 0 || D <= 0 || pairs < 0 || start < 0 || npos < 0) return set_error(SI_ERR_INVALID, "bad dimension");
  if (D > kRotMostD) return set_error(SI_ERR_UNSUPPORTED, "heads of more than 1024 dimensions");
  if (pairs > D / 2 || start + 2 * pairs > D) return set_error(SI_ERR_INVALID, "the rotary dimensions must lie within the head");
  if (H > 0x7fffffff || T > (int64_t{1} << 40) / H) return set_error(SI_ERR_UNSUPPORTED, "tensor too large");
  if (!xs) return set_error(SI_ERR_INVALID, "null stride argument");
  if (T > 0 && (!x || !out || (pairs > 0 && (!pos || !freqs)))) return set_error(SI_ERR_INVALID, "null pointer argument");
  if (T > 0 && pairs > 0 && (npos == 0 || T % npos)) return set_error(SI_ERR_INVALID, "the positions must divide the tokens");
  return SI_OK;
}

// Elements of a piece: the largest of 16 bytes that every row start, the row, the rotary part and, in halves, the partner allow.
static int rot_vec(int size, int64_t D, int64_t pairs, int64_t start, int halves, const void* const* ptrs, const int64_t* const* strides,
                   int n) {
  for (int v = 16 / size; v > 1; v /= 2) {
    bool ok = D % v == 0 && (pairs == 0 || (start % v == 0 && (halves ? pairs % v == 0 : 2 * pairs % v == 0)));
    for (int i = 0; i < n; ++i) {
      ok = ok && reinterpret_cast<uintptr_t>(ptrs[i]) % (v * size) == 0;
      if (strides[i]) ok = ok && strides[i][0] % v == 0 && strides[i][1] % v == 0;
    }
    if (ok) return v;
  }
  return 1;
}

template <typename F>
static int rot_dispatch(int dtype, const RotPlan& p, F&& f) {
  using std::integral_constant;
  auto cpl = [&](auto DT, auto V) {
    switch (p.cpl) {
      case 1: return f(DT, V, integral_constant<int, 1>{});
      case 2: return f(DT, V, integral_constant<int, 2>{});
      case 4: return f(DT, V, integral_constant<int, 4>{});
      case 5: return f(DT, V, integral_constant<int, 5>{});
      case 9: return f(DT, V, integral_constant<int, 9>{});
    }
    // (more than 9 pieces only where each is one value: 64 lanes hold 576 pieces)
    if constexpr (decltype(V)::value == 1) return f(DT, V, integral_constant<int, 16>{});
    return set_error(SI_ERR_UNSUPPORTED, "heads of more than 1024 dimensions");
  };
  auto vec = [&](auto DT) {
    if constexpr (decltype(DT)::value != 0) {
      if (p.vec == 8) return cpl(DT, integral_constant<int, 8>{});
    }
    switch (p.vec) {
      case 4: return cpl(DT, integral_constant<int, 4>{});
      case 2: return cpl(DT, integral_constant<int, 2>{});
      default: return cpl(DT, integral_constant<int, 1>{});
    }
  };
  switch (dtype) {
    case 0: return vec(integral_constant<int, 0>{});
    case 1: return vec(integral_constant<int, 1>{});
    default: return vec(integral_constant<int, 2>{});
  }
}

static void rot_args(RotArgs& a, const RotPlan& p, const float* weight, const void* positions, int pos64, int64_t npos,
                     const double* freqs, int64_t pairs, int64_t start, int halves, float magnitude, int inverse, float eps,
                     int64_t T, int64_t H, int64_t D) {
  a.weight = weight;
  a.pos = positions;
  a.pos64 = pos64;
  a.npos = npos;
  a.freqs = freqs;
  a.pairs = static_cast<int>(pairs);
  a.start = static_cast<int>(start);
  a.halves = halves;
  a.magnitude = magnitude;
  a.sign = inverse ? -1.f : 1.f;
  a.eps = eps;
  a.rows = T * H;
  a.H = static_cast<int>(H);
  a.D = static_cast<int>(D);
  a.lpr = p.lpr;
  a.log_lpr = p.log_lpr;
  a.iters = p.iters;
  a.per = p.per;
  a.weight_lds = weight ? static_cast<int>((D + 3) / 4 * 4) : 0;
  a.tokens = p.tokens;
}

extern "C" int si_norm_rotary(const void* x, const int64_t* x_strides, int norm, const float* weight, float eps,
                              const void* positions, int pos64, int64_t npos, const double* freqs, int64_t pairs, int64_t start,
                              int halves, float magnitude, int inverse, int64_t T, int64_t H, int64_t D, int dtype, void* y,
                              void* stream) {
  const int rc = rot_check(x, x_strides, positions, npos, freqs, pairs, start, T, H, D, dtype, y);
  if (rc || T == 0) return rc;
  if (weight && !norm) return set_error(SI_ERR_INVALID, "a weight without norm");
  const void* ptrs[2] = {x, y};
  const int64_t* strides[2] = {x_strides, nullptr};
  const int vec = rot_vec(dtype == 0 ? 4 : 2, D, pairs, start, halves, ptrs, strides, 2);
  const RotPlan p = rot_plan(T * H, H, D, pairs, vec, false);
  if (p.blocks > 0xffffffffLL / kRotThreads) return set_error(SI_ERR_UNSUPPORTED, "tensor too large");
  RotArgs a{};
  rot_args(a, p, weight, positions, pos64, npos, freqs, pairs, start, halves, magnitude, inverse, eps, T, H, D);
  a.x = static_cast<const char*>(x);
  a.xst = x_strides[0];
  a.xsh = x_strides[1];
  a.out = static_cast<char*>(y);
  hipStream_t st = static_cast<hipStream_t>(stream);
  return rot_dispatch(dtype, p, [&](auto DT, auto V, auto CPL) {
    constexpr int dt = decltype(DT)::value, v = decltype(V)::value, cpl = decltype(CPL)::value;
    const dim3 grid(static_cast<unsigned>(p.blocks)), block(kRotThreads);
    const size_t lds = static_cast<size_t>(p.tokens) * pairs * 8 + a.weight_lds * 4;
    if (norm) hipLaunchKernelGGL((norm_rotary_kernel<dt, v, cpl, true>), grid, block, lds, st, a);
    else hipLaunchKernelGGL((norm_rotary_kernel<dt, v, cpl, false>), grid, block, lds, st, a);
    return check_launch("norm_rotary_kernel");
  });
}

extern "C" int64_t si_norm_rotary_bwd_workspace_bytes(int64_t T, int64_t H, int64_t D, int64_t pairs) {
  if (T <= 0 || H <= 0 || D <= 0 || D > kRotMostD || pairs < 0 || pairs > D / 2 || H > 0x7fffffff || T > (int64_t{1} << 40) / H) return 0;
  int64_t most = 0;  // workgroups, whatever the pieces
  for (int vec = 1; vec <= 8; vec *= 2) {
    const int64_t b = rot_plan(T * H, H, D, pairs, vec, true).blocks;
    most = b > most ? b : most;
  }
  return most * D * 4;
}

extern "C" int si_norm_rotary_bwd(const void* dy, const int64_t* dy_strides, const void* x, const int64_t* x_strides,
                                  const float* weight, float eps, const void* positions, int pos64, int64_t npos,
                                  const double* freqs, int64_t pairs, int64_t start, int halves, float magnitude, int inverse,
                                  int64_t T, int64_t H, int64_t D, int dtype, void* dx, float* dweight, void* workspace,
                                  int64_t workspace_bytes, void* stream) {
  int rc = rot_check(x, x_strides, positions, npos, freqs, pairs, start, T, H, D, dtype, dx);
  if (rc) return rc;
  if (!dy_strides) return set_error(SI_ERR_INVALID, "null stride argument");
  if (T > 0 && !dy) return set_error(SI_ERR_INVALID, "null pointer argument");
  hipStream_t st = static_cast<hipStream_t>(stream);
  auto sum = [&](int parts) {
    hipLaunchKernelGGL(norm_rotary_dw_kernel, dim3(static_cast<unsigned>((D + 15) / 16)), dim3(256), 0, st,
                       static_cast<const float*>(workspace), parts, static_cast<int>(D), dweight);
    return check_launch("norm_rotary_dw_kernel");
  };
  if (T == 0) return dweight ? sum(0) : SI_OK;
  const void* ptrs[3] = {x, dy, dx};
  const int64_t* strides[3] = {x_strides, dy_strides, nullptr};
  const int vec = rot_vec(dtype == 0 ? 4 : 2, D, pairs, start, halves, ptrs, strides, 3);
  const RotPlan p = rot_plan(T * H, H, D, pairs, vec, true);
  if (p.blocks > 0xffffffffLL / kRotThreads) return set_error(SI_ERR_UNSUPPORTED, "tensor too large");
  if (dweight && (!workspace || workspace_bytes < p.blocks * D * 4)) return set_error(SI_ERR_INVALID, "workspace too small");
  RotArgs a{};
  // (back: the other way round)
  rot_args(a, p, weight, positions, pos64, npos, freqs, pairs, start, halves, magnitude, !inverse, eps, T, H, D);
  a.x = static_cast<const char*>(x);
  a.xst = x_strides[0];
  a.xsh = x_strides[1];
  a.dy = static_cast<const char*>(dy);
  a.dst = dy_strides[0];
  a.dsh = dy_strides[1];
  a.out = static_cast<char*>(dx);
  a.part = dweight ? static_cast<float*>(workspace) : nullptr;
  rc = rot_dispatch(dtype, p, [&](auto DT, auto V, auto CPL) {
    constexpr int dt = decltype(DT)::value, v = decltype(V)::value, cpl = decltype(CPL)::value;
    hipLaunchKernelGGL((norm_rotary_bwd_kernel<dt, v, cpl>), dim3(static_cast<unsigned>(p.blocks)), dim3(kRotThreads),
                       static_cast<size_t>(p.tokens) * pairs * 8 + a.weight_lds * 4, st, a);
    return check_launch("norm_rotary_bwd_kernel");
  });
  if (rc || !dweight) return rc;
  return sum(static_cast<int>(p.blocks));
}
