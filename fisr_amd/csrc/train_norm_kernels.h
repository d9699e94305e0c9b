// Kernels of the training graph's normalisation and regularisation: group normalisation with an activation and dropout,
// channels last.  x [N, P, C] (P = H * W pixels with a pixel stride of xcs elements), G groups of D = C / G channels:
//
//   mean[n,g], rstd[n,g] = 1 / sqrt(var + eps) over the P * D values of a group (biased variance)
//   xh = (x - mean) * rstd,  z = xh * gamma[c] + beta[c],  y = drop(act(z))
//   backward: dz = drop(dy) * act'(z);  A[n,c] = sum_p dz,  B[n,c] = sum_p dz * xh;  dbeta = sum_n A,  dgamma = sum_n B
//             dx = rstd * (dz * gamma - S1 / (P D) - xh * S2 / (P D)),  S1[n,g] = sum_{c in g} gamma A,  S2 = sum gamma B
//
// Every sum, statistic and intermediate is float32 or more; only y and dx are rounded, once, to the tensors' type.  There are no atomics: partial results go through the workspace and are joined in a fixed order, so a call's
// results are the same bits every time.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

namespace fisr {

typedef _Float16 f16_t;
typedef __bf16 b16_t;
enum { NORM_ACT_NONE = 0, NORM_ACT_RELU = 1, NORM_ACT_SILU = 2, NORM_ACT_GELU = 3 };

// ---- the generator: Philox4x32 with 7 rounds (Salmon, Moraes, Dror, Shaw, "Parallel random numbers: as easy as 1, 2, 3", SC 2011) ----
// 7 rounds are the fewest that the paper reports to pass all of BigCrush.  Block b of call `offset` under key `seed` is four words =
// eight 16-bit numbers; element i of a dense tensor has number i & 7 of block i >> 3 (word (i & 7) >> 1, low half first) and is dropped
// where it is below thresh = round(65536 p).  16 bits an element: a block costs 14 quarter-rate multiplies, which at 32 bits an
// element would take longer than a 16-bit tensor takes to stream; the rate that is realised, thresh / 65536, is what the scale of the
// kept values, 65536 / (65536 - thresh), goes by.
struct DropArgs {
  uint32_t thresh;                   // 0: no dropout
  float scale;
  uint64_t seed, offset;
  const uint64_t* counter;           // nullable, device: its value is added to offset when the kernel runs (captured graphs)
};
struct Philox { uint32_t w[4]; };
__device__ __forceinline__ Philox philox7(uint64_t block, uint64_t offset, uint64_t seed) {
  uint32_t c0 = (uint32_t)block, c1 = (uint32_t)(block >> 32), c2 = (uint32_t)offset, c3 = (uint32_t)(offset >> 32);
  uint32_t k0 = (uint32_t)seed, k1 = (uint32_t)(seed >> 32);
#pragma unroll
  for (int r = 0; r < 7; ++r) {
    const uint64_t p0 = (uint64_t)0xD2511F53u * c0, p1 = (uint64_t)0xCD9E8D57u * c2;
    c0 = (uint32_t)(p1 >> 32) ^ c1 ^ k0;
    c1 = (uint32_t)p1;
    c2 = (uint32_t)(p0 >> 32) ^ c3 ^ k1;
    c3 = (uint32_t)p0;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return Philox{{c0, c1, c2, c3}};
}
__device__ __forceinline__ uint32_t philox_number(const Philox& r, int e) { return (e & 1) ? r.w[e >> 1] >> 16 : r.w[e >> 1] & 0xffffu; }

// v[e] is element i + e of the dense tensor: scaled where it is kept, zero (whatever it was: NaN and infinities too) where not.
// i % V == 0 and V divides 8, so the V elements share a block.
template <int V> __device__ __forceinline__ void drop_apply(float (&v)[V], uint64_t i, const DropArgs& d, uint64_t offset) {
  const Philox r = philox7(i >> 3, offset, d.seed);
  if (V == 8) {
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] = philox_number(r, e) >= d.thresh ? v[e] * d.scale : 0.f;
  } else {
    const int at = (int)(i & 7);
    const uint32_t lo = at & 4 ? r.w[2] : r.w[0], hi = at & 4 ? r.w[3] : r.w[1];      // (selects: an index would go through scratch)
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const int k = (at & 3) + e;                                                         // 0..3 within the pair of words
      const uint32_t w = k & 2 ? hi : lo, number = k & 1 ? w >> 16 : w & 0xffffu;
      v[e] = number >= d.thresh ? v[e] * d.scale : 0.f;
    }
  }
}

// ---- vectors of V channels as they lie in memory.  The caller sees to alignment: 16 bytes, or V elements where that is less ----
// Two and more 16-bit elements are kept as 32-bit words: as an array of elements the compiler takes a loaded vector apart and joins it again.
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
template <typename T, int V> struct alignas(sizeof(T) * V < 16 ? sizeof(T) * V : 16) Pack {
  static constexpr bool WORDS = sizeof(T) * V >= 4;
  typedef typename std::conditional<WORDS, uint32_t, T>::type E;
  static constexpr int N = sizeof(T) * V / sizeof(E);
  E w[N];
  __device__ __forceinline__ float get(int e) const {
    if constexpr (!WORDS) return (float)w[e];
    else if constexpr (sizeof(T) == 4) return __builtin_bit_cast(float, w[e]);
    else if constexpr (std::is_same<T, b16_t>::value) return __builtin_bit_cast(float, e & 1 ? w[e >> 1] & 0xffff0000u : w[e >> 1] << 16);
    else {
      struct H { f16_t h[2]; };
      return (float)__builtin_bit_cast(H, w[e >> 1]).h[e & 1];
    }
  }
  __device__ __forceinline__ void widen(float (&v)[V]) const {
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] = get(e);
  }
  __device__ __forceinline__ void round(const float (&v)[V]) {
    if constexpr (!WORDS) w[0] = (T)v[0];
    else if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int e = 0; e < V; ++e) w[e] = __builtin_bit_cast(uint32_t, v[e]);
    } else {
      struct H { T h[2]; };
#pragma unroll
      for (int e = 0; e < V; e += 2) w[e >> 1] = __builtin_bit_cast(uint32_t, H{{(T)v[e], (T)v[e + 1]}});
    }
  }
  __device__ __forceinline__ void load(const T* p) { *this = *reinterpret_cast<const Pack*>(p); }
  __device__ __forceinline__ void store(T* p) const { *reinterpret_cast<Pack*>(p) = *this; }
  // non-temporal: what is read or written once and is larger than the caches hold
  __device__ __forceinline__ void load_nt(const T* p) {
    if constexpr (N % 4 == 0) {
#pragma unroll
      for (int k = 0; k < N / 4; ++k) {
        const u32x4 u = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(p) + k);
        w[4 * k] = u.x; w[4 * k + 1] = u.y; w[4 * k + 2] = u.z; w[4 * k + 3] = u.w;
      }
    } else if constexpr (N == 2) {
      const u32x2 u = __builtin_nontemporal_load(reinterpret_cast<const u32x2*>(p));
      w[0] = u.x; w[1] = u.y;
    } else if constexpr (WORDS) {
      w[0] = __builtin_nontemporal_load(reinterpret_cast<const uint32_t*>(p));
    } else {
      load(p);
    }
  }
  __device__ __forceinline__ void store_nt(T* p) const {
    if constexpr (N % 4 == 0) {
#pragma unroll
      for (int k = 0; k < N / 4; ++k) __builtin_nontemporal_store(u32x4{w[4 * k], w[4 * k + 1], w[4 * k + 2], w[4 * k + 3]}, reinterpret_cast<u32x4*>(p) + k);
    } else if constexpr (N == 2) {
      __builtin_nontemporal_store(u32x2{w[0], w[1]}, reinterpret_cast<u32x2*>(p));
    } else if constexpr (WORDS) {
      __builtin_nontemporal_store(w[0], reinterpret_cast<uint32_t*>(p));
    } else {
      store(p);
    }
  }
  // Hides from the compiler that a register still holds what it held: it would otherwise keep a 16-bit vector's float32 form from one pass over
  // the registers to the next, at twice the registers.
  __device__ __forceinline__ void keep() {
    if constexpr (sizeof(T) == 2 && WORDS) {
#pragma unroll
      for (int e = 0; e < N; ++e) asm volatile("" : "+v"(w[e]));
    }
  }
};
template <typename T, int V> __device__ __forceinline__ void load_v(const T* p, float (&v)[V]) {
  Pack<T, V> q;
  q.load(p);
  q.widen(v);
}
template <typename T, int V> __device__ __forceinline__ void store_v(T* p, const float (&v)[V]) {
  Pack<T, V> q;
  q.round(v);
  q.store(p);
}
template <typename T, int V> __device__ __forceinline__ void store_nt(T* p, const float (&v)[V]) {
  Pack<T, V> q;
  q.round(v);
  q.store_nt(p);
}
// Between a non-temporal access and a plain one of the same address in two branches: the compiler would make them one access and drop the hint.
#define KEEP_APART(text) asm volatile("; " text)

// ---- activations ----
__device__ __forceinline__ float sigmoid_f(float z) { return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-1.4426950408889634f * z)); }
// The normal distribution's Phi(-|z|) = erfc(|z| / sqrt 2) / 2 by Abramowitz and Stegun 7.1.26 (a polynomial of the fifth degree in
// t = 1 / (1 + 0.3275911 |z| / sqrt 2) times exp(-z^2 / 2), 0.75e-7 off at the most, and as much again by rounding): 9 operations beside one
// exponential, which the gradient needs anyway, and one reciprocal; the library's erf is over twice that.  Halved coefficients.
__device__ __forceinline__ float phi_tail(float z, float gauss) {
  const float t = __builtin_amdgcn_rcpf(1.f + 0.23164189f * fabsf(z));
  return t * (0.127414796f + t * (-0.142248368f + t * (0.7107068705f + t * (-0.7265760135f + t * 0.5307027145f)))) * gauss;
}
__device__ __forceinline__ float gauss_f(float z) { return __builtin_amdgcn_exp2f(-0.72134752f * z * z); }
template <int V> __device__ __forceinline__ void act_apply(float (&z)[V], int act) {
  if (act == NORM_ACT_RELU) {
#pragma unroll
    for (int e = 0; e < V; ++e) z[e] = z[e] < 0.f ? 0.f : z[e];          // NaN stays (a maximum with zero would drop it)
  } else if (act == NORM_ACT_SILU) {
#pragma unroll
    for (int e = 0; e < V; ++e) z[e] *= sigmoid_f(z[e]);
  } else if (act == NORM_ACT_GELU) {
#pragma unroll
    for (int e = 0; e < V; ++e) z[e] = fmaxf(z[e], 0.f) - fabsf(z[e]) * phi_tail(z[e], gauss_f(z[e]));      // z Phi(z) on either side
  }
}
// g[e] *= act'(z[e])
template <int V> __device__ __forceinline__ void act_grad_apply(float (&g)[V], const float (&z)[V], int act) {
  if (act == NORM_ACT_RELU) {
#pragma unroll
    for (int e = 0; e < V; ++e) g[e] = z[e] <= 0.f ? 0.f : g[e];
  } else if (act == NORM_ACT_SILU) {
#pragma unroll
    for (int e = 0; e < V; ++e) { const float s = sigmoid_f(z[e]); g[e] *= s * (1.f + z[e] * (1.f - s)); }
  } else if (act == NORM_ACT_GELU) {
#pragma unroll
    for (int e = 0; e < V; ++e) {                              // Phi = 1/2 + sign(z) (1/2 - Phi(-|z|))
      const float n = gauss_f(z[e]), half = copysignf(0.5f - phi_tail(z[e], n), z[e]);
      g[e] *= 0.5f + (half + z[e] * (0.39894228f * n));
    }
  }
}

// ---- arguments and tiles -----------------------------------------------------------------------------------------------------
// Every kernel below lets a thread keep one vector of V channels (column `col` of its workgroup's) and walk pixels: rows x cb threads.
struct NormArgs {
  const void* x; const void* dy; void* y;              // y: the output (dx in the backward pass)
  const float* gamma; const float* beta;               // nullable
  float* mean; float* rstd;                            // [N][G]
  float2* part;                                        // partial numbers of chunks: see the kernels
  float2* ab; float2* s12;                             // backward: (A, B) by channel, (S1, S2) / (P D) by group
  float* dgamma; float* dbeta;
  size_t xcs, ycs, dycs;                               // pixel strides, elements
  int n, p, c, groups, d;
  int cb, rows, span;                                  // columns and rows of a workgroup's threads, its channels
  int chunks, ppc;                                     // chunks of an image's pixels, pixels of a chunk: chunks = ceil(p / ppc)
  int achunks, appc, join;                             // ... in the second of two launches; whether that joins the first one's numbers
  int slots, per_group, jl;                            // see team_sums
  uint32_t by_d, by_cb, by_rows, by_per_group;               // for div_by
  float eps, inv_m;                                    // inv_m: 1 / (p * d)
  int act, accumulate;
  int team, nt;                                        // the host's variant of the one-launch form; whether reads pass the caches
  DropArgs drop;
};
// x / y for x < 2^16 and y <= 2^16 by the host's ceil(2^32 / y) (0 for y = 1): a division by a number of the launch is some 20 instructions
// otherwise, as many as the work on three channels.
__device__ __forceinline__ int div_by(int x, uint32_t magic) { return magic ? (int)__umulhi((uint32_t)x, magic) : x; }
__device__ __forceinline__ uint64_t drop_offset(const DropArgs& d) { return d.offset + (d.counter ? *d.counter : 0); }
__device__ __forceinline__ float inv_std(float var, float eps) { return 1.f / sqrtf(var + eps); }

struct NormTeam {
  int img, cbase, row, col, c0;
  bool on;
};
template <int V> __device__ __forceinline__ void team_threads(NormTeam& t, const NormArgs& a) {
  t.row = div_by(threadIdx.x, a.by_cb);
  t.col = threadIdx.x - t.row * a.cb;
  t.c0 = t.cbase + t.col * V;
  t.on = t.row < a.rows;
}

// ---- sums over a workgroup's pixels and the channels of each of its groups: tot[group] = last(sum), seen by every thread.  All threads call. ----
// A thread first adds the channels of its vector that share a group (slots numbers are left: 1, V / d or V), a wave its rows where columns
// are a power of two, then 2^jl lanes a group add what is left of all groups at once.  `red`: TH * V floats.
template <int V> __device__ __forceinline__ int fold_slots(const NormArgs& a, float (&v)[V]) {
  if (a.slots < V) {                                         // (groups of one channel or of no divisor's fraction of V stay as they are)
#pragma unroll
    for (int k = V; k > 1; k >>= 1)
      if (a.slots < k) {
#pragma unroll
        for (int e = 0; e < k / 2; ++e) v[e] = v[2 * e] + v[2 * e + 1];
      }
  }
  return a.slots;
}
template <int V, int TH, typename F> __device__ __forceinline__ void team_sums(const NormArgs& a, const NormTeam& t, float (&v)[V], float* red, float* tot, F last) {
  const int slots = fold_slots<V>(a, v), per_row = a.cb * slots;
  const bool pow2 = a.cb <= 64 && (a.cb & (a.cb - 1)) == 0;
  int rows = a.rows;
  if (pow2) {
    rows = TH / 64;
    for (int k = a.cb; k < 64; k <<= 1) {
#pragma unroll
      for (int e = 0; e < V; ++e)
        if (e < slots) v[e] += __shfl_xor(v[e], k);
    }
  }
  const int r = pow2 ? threadIdx.x >> 6 : t.row;
  if (pow2 ? (int)(threadIdx.x & 63) < a.cb : t.on) {
#pragma unroll
    for (int e = 0; e < V; ++e)
      if (e < slots) red[r * per_row + t.col * slots + e] = v[e];
  }
  __syncthreads();
  const int lanes = 1 << a.jl, lane = threadIdx.x & (lanes - 1), groups = a.span / a.d, total = rows * a.per_group;
  for (int j0 = 0; j0 < groups; j0 += TH >> a.jl) {          // (every lane of a wave takes part in the shuffles)
    const int j = j0 + (threadIdx.x >> a.jl);
    float s = 0.f;
    if (j < groups)
      for (int i = lane; i < total; i += lanes) { const int q = div_by(i, a.by_per_group); s += red[q * per_row + j * a.per_group + (i - q * a.per_group)]; }
    for (int k = lanes >> 1; k; k >>= 1) s += __shfl_xor(s, k);
    if (j < groups && lane == 0) tot[j] = last(s);
  }
  __syncthreads();
}

// Two pixels' dropout of a thread with four channels: a generator block is eight, so lanes 2k and 2k + 1 want the same two blocks.  Each
// computes one and they exchange halves.  The span's channels are a multiple of 8, so both lanes are at the same pixels.
template <int V> __device__ __forceinline__ void drop_apply_pair(float (&v0)[V], float (&v1)[V], uint64_t i0, uint64_t i1, const DropArgs& d, uint64_t offset) {
  static_assert(V == 4, "");
  const bool odd = threadIdx.x & 1;
  const Philox r = philox7((odd ? i1 : i0) >> 3, offset, d.seed);
  const uint32_t s0 = odd ? r.w[0] : r.w[2], s1 = odd ? r.w[1] : r.w[3];
  const uint32_t g0 = __builtin_amdgcn_mov_dpp(s0, 0xB1, 0xf, 0xf, true), g1 = __builtin_amdgcn_mov_dpp(s1, 0xB1, 0xf, 0xf, true);   // quad_perm 1, 0, 3, 2
  const uint32_t a0 = odd ? g0 : r.w[0], a1 = odd ? g1 : r.w[1], b0 = odd ? r.w[2] : g0, b1 = odd ? r.w[3] : g1;
#pragma unroll
  for (int e = 0; e < V; ++e) {
    const uint32_t wa = e & 2 ? a1 : a0, wb = e & 2 ? b1 : b0;
    v0[e] = (e & 1 ? wa >> 16 : wa & 0xffffu) >= d.thresh ? v0[e] * d.scale : 0.f;
    v1[e] = (e & 1 ? wb >> 16 : wb & 0xffffu) >= d.thresh ? v1[e] * d.scale : 0.f;
  }
}

// Which elements of a thread's R vectors dropout keeps, found while the vectors are on their way: the generator's numbers need none of them
// (32 x 48 x 48 x 128 bfloat16: 18.7 us against 19.7 with the numbers made where they are used, backward 24.7 and 26.5).  It stands before any other
// load of the kernel: with gamma's and beta's under way the compiler took one of their registers for a product and waited for all loads first.
// Bit (e >> 1) + 16 (e & 1) + 4 (r & 3) of bits[r >> 2] is element e of vector r: a word of the generator is two elements, and packed 16-bit
// operations make both bits at once, max(number - (thresh - 1), 0) and min(that, 1).
template <int V, int R> struct DropMask {
  uint32_t bits[(R + 3) / 4];
  static __device__ __forceinline__ uint32_t two(uint32_t word, uint32_t below) {
    typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
    const u16x2 b = {(unsigned short)below, (unsigned short)below}, one = {1, 1};
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_min(__builtin_elementwise_sub_sat(__builtin_bit_cast(u16x2, word), b), one));
  }
  __device__ __forceinline__ void put(int r, uint32_t m) { bits[r >> 2] |= m << 4 * (r & 3); }
  // vector r is elements i0 + r * di on; pairs: as drop_apply_pair's; `pixel(r)`: whether there is a vector r
  template <typename F> __device__ __forceinline__ void find(bool pairs, uint64_t i0, uint64_t di, const DropArgs& d, uint64_t offset, F pixel) {
    const uint32_t below = d.thresh - 1;
#pragma unroll
    for (int k = 0; k < (R + 3) / 4; ++k) bits[k] = 0;
    if (V == 4 && pairs && R > 1) {
      const bool odd = threadIdx.x & 1;
      uint64_t i = i0 + (odd ? di : 0);
#pragma unroll
      for (int r = 0; r < R; r += 2, i += 2 * di)
        if (pixel(r)) {                                      // (vector r + 1 may be no pixel: nobody uses it)
          const Philox n = philox7(i >> 3, offset, d.seed);
          const uint32_t lo = two(n.w[0], below) | two(n.w[1], below) << 1, hi = two(n.w[2], below) | two(n.w[3], below) << 1;
          const uint32_t got = __builtin_amdgcn_mov_dpp(odd ? lo : hi, 0xB1, 0xf, 0xf, true);               // quad_perm 1, 0, 3, 2
          put(r, odd ? got : lo);
          if (r + 1 < R) put(r + 1, odd ? hi : got);
        }
    } else {
      uint64_t i = i0;
#pragma unroll
      for (int r = 0; r < R; ++r, i += di)
        if (pixel(r)) {
          const Philox n = philox7(i >> 3, offset, d.seed);
          if (V == 8) {
            put(r, two(n.w[0], below) | two(n.w[1], below) << 1 | two(n.w[2], below) << 2 | two(n.w[3], below) << 3);
          } else {
            const int at = (int)(i & 7);
            const uint32_t lo = at & 4 ? n.w[2] : n.w[0], hi = at & 4 ? n.w[3] : n.w[1];
            if (V == 4) put(r, two(lo, below) | two(hi, below) << 1);
            else put(r, two((at & 2 ? hi : lo) >> (V == 1 && (at & 1) ? 16 : 0), below) & (V == 1 ? 1u : ~0u));
          }
        }
    }
#pragma unroll
    for (int k = 0; k < (R + 3) / 4; ++k) asm volatile("" : "+v"(bits[k]));      // (here, not where they are used)
  }
  __device__ __forceinline__ void apply(int r, float (&v)[V], float scale) const {
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const int bit = (e >> 1) + 16 * (e & 1) + 4 * (r & 3);
      v[e] = __builtin_bit_cast(float, __builtin_bit_cast(int, v[e] * scale) & (int)(bits[r >> 2] << (31 - bit)) >> 31);
    }
  }
};

// ---- one launch, one read: a workgroup holds `span` channels (whole groups) of all pixels of an image in registers ----
// Thread (row, col) keeps the vectors of column col at the pixels row + r * rows, r < R, as they were loaded (16-bit tensors packed).
// What a second pass over memory would be is a pass over registers, so the mean comes first and the squares are about it.
// Workgroup b runs on XCD b % 8 (observed; speed only): the workgroups of one image, which share its cache lines where a span is less than a
// line, go to one XCD.
template <int V> __device__ __forceinline__ NormTeam span_team(const NormArgs& a) {
  NormTeam t;
  const int slices = a.c / a.span, b = blockIdx.x, whole = a.n / 8 * 8 * slices;
  int unit = b;
  if (b < whole) { const int k = b >> 3; unit = (k / slices * 8 + (b & 7)) * slices + k % slices; }
  t.img = unit / slices;
  t.cbase = (unit - t.img * slices) * a.span;
  team_threads<V>(t, a);
  return t;
}

// A thread's vectors of one tensor: number r is r * step bytes from its first.  The launch's part of an address stays in scalar registers
// (base, r * step), the thread's is a 32-bit offset (the host sees to that), so a load costs no vector instruction beside itself.
template <typename T, int V> struct Walk {
  char* base;
  uint32_t at;
  size_t step;
  __device__ __forceinline__ Walk(const NormArgs& a, const NormTeam& t, const void* x, size_t cs, int p0)
      : base((char*)x + (((size_t)t.img * a.p + p0) * cs + t.cbase) * sizeof(T)), at((uint32_t)((t.row * (uint32_t)cs + t.col * V) * sizeof(T))),
        step(a.rows * cs * sizeof(T)) {}
  __device__ __forceinline__ T* ptr(int r) const { return reinterpret_cast<T*>(base + (size_t)r * step + at); }
  template <int U> __device__ __forceinline__ void load(Pack<T, V> (&q)[U], int r, int m, int nt) const {      // nt: past the caches
    if (nt) {
      KEEP_APART("past the caches");
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (u < m) q[u].load_nt(ptr(r + u));
      KEEP_APART("end");
    } else {
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (u < m) q[u].load(ptr(r + u));
    }
  }
};
// Bound by the phases, which wait for each other (all loads, two sums over the workgroup, all stores, one workgroup a CU for the largest), and
// by a span being a part of a cache line, which the workgroups of an image read from L2 in turn: 32 x 48 x 48 x 128 bfloat16 in 32 groups, 38 MB, 17.0 us
// without dropout, 17.8 with, 6.3 at the rate of a copy; the two launches below take 24.0 and 25.7.  Twice as large it is 29.0 and 28.8, so up to
// 16 M elements go here.
template <typename T, int V, int R, int TH> __global__ __launch_bounds__(TH) void norm_team_kernel(const NormArgs a) {
  __shared__ float red[TH * V];
  __shared__ float tot[2][TH * V];                           // (as many groups as channels at the most)
  const NormTeam t = span_team<V>(a);
  const Walk<T, V> x(a, t, a.x, a.xcs, 0), y(a, t, a.y, a.ycs, 0);
  Pack<T, V> q[R];
#pragma unroll
  for (int r = 0; r < R; ++r)
    if (t.on && t.row + r * a.rows < a.p) q[r].load(x.ptr(r));
  DropMask<V, R> drop;
  if (a.drop.thresh && t.on)
    drop.find(a.span % 8 == 0, ((uint64_t)t.img * a.p + t.row) * a.c + t.c0, (uint64_t)a.rows * a.c, a.drop, drop_offset(a.drop),
              [&](int r) { return t.row + r * a.rows < a.p; });
  float gamma[V], beta[V];
#pragma unroll
  for (int e = 0; e < V; ++e) {
    gamma[e] = t.on && a.gamma ? a.gamma[t.c0 + e] : 1.f;
    beta[e] = t.on && a.beta ? a.beta[t.c0 + e] : 0.f;
  }
  float s[V];
#pragma unroll
  for (int e = 0; e < V; ++e) s[e] = 0.f;
#pragma unroll
  for (int r = 0; r < R; ++r)
    if (t.on && t.row + r * a.rows < a.p) {
#pragma unroll
      for (int e = 0; e < V; ++e) s[e] += q[r].get(e);
    }
  team_sums<V, TH>(a, t, s, red, tot[0], [&](float v) { return v * a.inv_m; });
#pragma unroll
  for (int r = 0; r < R; ++r) q[r].keep();
  float mean[V];
#pragma unroll
  for (int e = 0; e < V; ++e) { mean[e] = t.on ? tot[0][div_by(t.col * V + e, a.by_d)] : 0.f; s[e] = 0.f; }
#pragma unroll
  for (int r = 0; r < R; ++r)
    if (t.on && t.row + r * a.rows < a.p) {
#pragma unroll
      for (int e = 0; e < V; ++e) { const float dv = q[r].get(e) - mean[e]; s[e] += dv * dv; }
    }
  team_sums<V, TH>(a, t, s, red, tot[1], [&](float v) { return inv_std(v * a.inv_m, a.eps); });
#pragma unroll
  for (int r = 0; r < R; ++r) q[r].keep();
  for (int j = threadIdx.x; j < a.span / a.d; j += TH) {
    const size_t g = (size_t)t.img * a.groups + t.cbase / a.d + j;
    a.mean[g] = tot[0][j];
    a.rstd[g] = tot[1][j];
  }
  if (!t.on) return;
#pragma unroll
  for (int e = 0; e < V; ++e) gamma[e] *= tot[1][div_by(t.col * V + e, a.by_d)];
#pragma unroll
  for (int r = 0; r < R; ++r)
    if (t.row + r * a.rows < a.p) {
      float v[V];
#pragma unroll
      for (int e = 0; e < V; ++e) v[e] = (q[r].get(e) - mean[e]) * gamma[e] + beta[e];
      act_apply<V>(v, a.act);
      if (a.drop.thresh) drop.apply(r, v, a.drop.scale);
      store_v<T, V>(y.ptr(r), v);
    }
}

// ---- two launches, one read each: statistics per group and chunk of pixels, then the output ----
// part[image][group][chunk] = (mean, M2) of a chunk.  The second launch's workgroups join their image's chunks themselves, or, where that is
// much to read for each of them (few images with many chunks), norm_join_kernel joins them once in between.
// Bound by memory where the tensor is beyond the caches: 12 x 544 x 992 x 64 float16, 829 MB, statistics 129 us (6.4 TB/s), output 279 us (5.9 TB/s; the
// best copy of this card 6.0).  Between (75 MB: 15.1 and 23.5 us, 5.0 and 6.4 TB/s) the first launch's ramp and tail count as well, and
// with gelu on 69 MB the arithmetic does (26.5 us for 138 MB).  The parts cannot be one launch without waiting for all workgroups of an image.
template <int V> __device__ __forceinline__ NormTeam chunk_team(const NormArgs& a, int block, int chunks, int ppc, int& chunk, int& p0, int& p1) {
  NormTeam t;
  t.img = block / chunks;
  chunk = block - t.img * chunks;
  p0 = chunk * ppc; p1 = min(a.p, p0 + ppc);
  t.cbase = blockIdx.y * a.span;
  team_threads<V>(t, a);
  return t;
}

// One batch of M <= U pixels joined to the running (mean, M2) of the thread's channels: the batch is reduced about its own mean and joined by
// Chan's formula, so nothing is lost when the mean is large against the spread: no sum of squares about a far point exists anywhere.
template <typename T, int V, int U> __device__ __forceinline__ void stats_batch(Pack<T, V> (&q)[U], int m, float (&mean)[V], float (&m2)[V], float& cnt) {
  float bm[V], b2[V];
  const float fm = (float)m, im = __builtin_amdgcn_rcpf(fm), w = fm * __builtin_amdgcn_rcpf(cnt + fm), nw = cnt * w;      // (1 / 4 is exact)
  cnt += fm;
#pragma unroll
  for (int e = 0; e < V; ++e) bm[e] = b2[e] = 0.f;
#pragma unroll
  for (int u = 0; u < U; ++u)
    if (u < m) {
#pragma unroll
      for (int e = 0; e < V; ++e) bm[e] += q[u].get(e);
    }
#pragma unroll
  for (int e = 0; e < V; ++e) bm[e] *= im;
#pragma unroll
  for (int u = 0; u < U; ++u) q[u].keep();
#pragma unroll
  for (int u = 0; u < U; ++u)
    if (u < m) {
#pragma unroll
      for (int e = 0; e < V; ++e) { const float dv = q[u].get(e) - bm[e]; b2[e] += dv * dv; }
    }
#pragma unroll
  for (int e = 0; e < V; ++e) { const float dm = bm[e] - mean[e]; mean[e] += dm * w; m2[e] += b2[e] + dm * dm * nw; }
}

// The vectors of a thread in a chunk, U at a time, the next ones asked for before these are worked on: two buffers in turn (a copy between
// them would cost as many instructions as a vector's arithmetic).  `load(buffer, r, m)` and `work(buffer, r, m)` take vectors r .. r + m - 1;
// m is U but for the last ones.  fetch() loads the first, finish() does the rest.  As compiled, every other fetch alone is still on its way
// during the work: a whole batch and the last one fill the same buffer on paths that join, after which the number of loads under way is not
// known, and the wait before the work is for all of them.
template <int U, typename B> struct Chunk {
  int full, tail;
  B b0, b1;
  __device__ __forceinline__ Chunk(const NormArgs& a, const NormTeam& t, int len) {
    full = len / (U * a.rows);                               // the same for every thread
    const int left = len - full * U * a.rows - t.row;
    tail = left > 0 ? div_by(left + a.rows - 1, a.by_rows) : 0;
  }
  template <typename L> __device__ __forceinline__ void fetch(B& b, int k, L load) { k < full ? load(b, k * U, U) : load(b, k * U, tail); }
  template <typename L, typename W> __device__ __forceinline__ void finish(L load, W work) {
    int k = 0;
    while (k < full) {
      fetch(b1, k + 1, load);
      work(b0, k * U, U);
      if (++k == full) { b0 = b1; break; }
      fetch(b0, k + 1, load);
      work(b1, k * U, U);
      ++k;
    }
    work(b0, full * U, tail);
  }
};

template <typename T, int V, int U> struct Batch { Pack<T, V> x[U]; };
template <typename T, int V, int TH> __global__ __launch_bounds__(TH, 4) void norm_chunk_stats_kernel(const NormArgs a) {
  constexpr int U = 4;
  typedef Batch<T, V, U> B;
  __shared__ float red[TH * V];
  __shared__ float tot[2][TH * V];
  int chunk, p0, p1;
  const NormTeam t = chunk_team<V>(a, blockIdx.x, a.chunks, a.ppc, chunk, p0, p1);
  float mean[V], m2[V], cnt = 0.f;
#pragma unroll
  for (int e = 0; e < V; ++e) mean[e] = m2[e] = 0.f;
  if (t.on) {
    const Walk<T, V> x(a, t, a.x, a.xcs, p0);
    Chunk<U, B> c(a, t, p1 - p0);
    const auto load = [&](B& b, int r, int m) { x.load(b.x, r, m, a.nt); };
    c.fetch(c.b0, 0, load);
    c.finish(load, [&](B& b, int, int m) { if (m) stats_batch<T, V, U>(b.x, m, mean, m2, cnt); });
  }
  float s[V];
#pragma unroll
  for (int e = 0; e < V; ++e) s[e] = cnt * mean[e];
  const float inv = 1.f / ((float)(p1 - p0) * (float)a.d);
  team_sums<V, TH>(a, t, s, red, tot[0], [&](float v) { return v * inv; });
#pragma unroll
  for (int e = 0; e < V; ++e) { const float dm = t.on ? mean[e] - tot[0][div_by(t.col * V + e, a.by_d)] : 0.f; s[e] = m2[e] + cnt * dm * dm; }
  team_sums<V, TH>(a, t, s, red, tot[1], [](float v) { return v; });
  for (int j = threadIdx.x; j < a.span / a.d; j += TH)
    a.part[((size_t)t.img * a.groups + t.cbase / a.d + j) * a.chunks + chunk] = make_float2(tot[0][j], tot[1][j]);
}

// mean and rstd of `count` groups from the chunks' numbers: 2^jl lanes a group, all groups at once (a wave a group in turn would be two round
// trips to memory for every group after the other: 10 us for 32 groups)
// Up to K numbers a lane stay in registers between the two sums: one trip to memory.
template <int TH, int K> __device__ __forceinline__ void join_groups(const NormArgs& a, size_t first, int count, float* mean, float* rstd) {
  const int lanes = 1 << a.jl, lane = threadIdx.x & (lanes - 1);
  const float m = (float)a.p * (float)a.d, full = (float)a.ppc * (float)a.d, last = (float)(a.p - (a.chunks - 1) * a.ppc) * (float)a.d;
  for (int j0 = 0; j0 < count; j0 += TH >> a.jl) {
    const int j = j0 + (threadIdx.x >> a.jl);
    const float2* part = a.part + (first + j) * a.chunks;
    float2 f[K];
    float s = 0.f, q = 0.f;
    if (j < count) {
#pragma unroll
      for (int i = 0; i < K; ++i) f[i] = lane + i * lanes < a.chunks ? part[lane + i * lanes] : make_float2(0.f, 0.f);
#pragma unroll
      for (int i = 0; i < K; ++i) s += f[i].x * (lane + i * lanes == a.chunks - 1 ? last : full);
      for (int k = lane + K * lanes; k < a.chunks; k += lanes) s += part[k].x * (k == a.chunks - 1 ? last : full);
    }
    for (int k = lanes >> 1; k; k >>= 1) s += __shfl_xor(s, k);
    const float mu = s / m;
    if (j < count) {
#pragma unroll
      for (int i = 0; i < K; ++i)
        if (lane + i * lanes < a.chunks) q += f[i].y + (f[i].x - mu) * (f[i].x - mu) * (lane + i * lanes == a.chunks - 1 ? last : full);
      for (int k = lane + K * lanes; k < a.chunks; k += lanes) {
        const float2 g = part[k];
        q += g.y + (g.x - mu) * (g.x - mu) * (k == a.chunks - 1 ? last : full);
      }
    }
    for (int k = lanes >> 1; k; k >>= 1) q += __shfl_xor(q, k);
    if (j < count && lane == 0) { mean[j] = mu; rstd[j] = inv_std(q / m, a.eps); }
  }
}
// a wave a group of the whole batch (jl = 6)
__global__ __launch_bounds__(64) void norm_join_kernel(const NormArgs a) {
  join_groups<64, 16>(a, blockIdx.x, 1, a.mean + blockIdx.x, a.rstd + blockIdx.x);
}

template <typename T, int V, int TH, bool WHOLE> __global__ __launch_bounds__(TH) void norm_chunk_apply_kernel(const NormArgs a) {
  constexpr int U = 4, W = WHOLE ? 1 : V;
  typedef Batch<T, V, U> B;
  __shared__ float mean_s[TH * V], rstd_s[TH * V];
  int chunk, p0, p1;
  const NormTeam t = chunk_team<V>(a, blockIdx.x, a.achunks, a.appc, chunk, p0, p1);
  const Walk<T, V> x(a, t, a.x, a.xcs, p0), y(a, t, a.y, a.ycs, p0);
  Chunk<U, B> c(a, t, p1 - p0);
  const auto load = [&](B& b, int r, int m) { x.load(b.x, r, m, a.nt); };
  if (t.on) c.fetch(c.b0, 0, load);                          // on its way while the statistics come
  const size_t g0 = (size_t)t.img * a.groups + div_by(t.cbase, a.by_d);
  const float *mg = a.mean + g0, *rg = a.rstd + g0;
  float mean[W], scale[V], beta[V];
#pragma unroll
  for (int e = 0; e < V; ++e) {
    scale[e] = t.on && a.gamma ? a.gamma[t.c0 + e] : 1.f;
    beta[e] = t.on && a.beta ? a.beta[t.c0 + e] : 0.f;
  }
  if (a.join) {
    const int groups = div_by(a.span, a.by_d);
    join_groups<TH, 4>(a, g0, groups, mean_s, rstd_s);
    __syncthreads();
    if (chunk == 0)
      for (int j = threadIdx.x; j < groups; j += TH) { a.mean[g0 + j] = mean_s[j]; a.rstd[g0 + j] = rstd_s[j]; }
  }
  if (!t.on) return;
#pragma unroll
  for (int e = 0; e < V; ++e) {
    const int g = div_by(t.col * V + (WHOLE ? 0 : e), a.by_d);
    if (e < W) mean[e] = a.join ? mean_s[g] : mg[g];
    scale[e] *= a.join ? rstd_s[g] : rg[g];
  }
  const uint64_t offset = a.drop.thresh ? drop_offset(a.drop) : 0;
  const uint64_t i0 = ((uint64_t)t.img * a.p + p0 + t.row) * a.c + t.c0, di = (uint64_t)a.rows * a.c;
  const bool pairs = V == 4 && a.span % 8 == 0;
  c.finish(load, [&](B& b, int r, int m) {
#pragma unroll
    for (int u = 0; u < U; u += 2) {
      float v[2][V];
#pragma unroll
      for (int k = 0; k < 2; ++k)
        if (u + k < m) {
#pragma unroll
          for (int e = 0; e < V; ++e) v[k][e] = (b.x[u + k].get(e) - mean[WHOLE ? 0 : e]) * scale[e] + beta[e];
          act_apply<V>(v[k], a.act);
          if (a.drop.thresh && !pairs) drop_apply<V>(v[k], i0 + (r + u + k) * di, a.drop, offset);
        }
      if constexpr (V == 4) {
        if (a.drop.thresh && pairs && u < m) drop_apply_pair<V>(v[0], v[1], i0 + (r + u) * di, i0 + (r + u + 1) * di, a.drop, offset);   // (the second may be no pixel: not stored)
      }
#pragma unroll
      for (int k = 0; k < 2; ++k)
        if (u + k < m) store_nt<T, V>(y.ptr(r + u + k), v[k]);
    }
  });
}

// ---- backward ----
// What a thread needs of its channels, with t = x - mean: z = t * scale + beta, scale = rstd * gamma.  (x - mean first: scale * x + const would
// round twice at the size of mean * rstd.)  WHOLE: its V channels lie in one group, whose numbers it keeps once: 14 registers of 40 less
// at V = 8.
template <int V, bool WHOLE> struct NormChan {
  static constexpr int W = WHOLE ? 1 : V;
  float mean[W], rstd[W], scale[V], beta[V];
  __device__ __forceinline__ void load(const NormArgs& a, int img, int c0, bool on) {
#pragma unroll
    for (int e = 0; e < W; ++e) {
      const size_t g = (size_t)img * a.groups + (on ? div_by(c0 + e, a.by_d) : 0);
      mean[e] = a.mean[g];
      rstd[e] = a.rstd[g];
    }
#pragma unroll
    for (int e = 0; e < V; ++e) {
      scale[e] = rstd[WHOLE ? 0 : e] * (on && a.gamma ? a.gamma[c0 + e] : 1.f);
      beta[e] = on && a.beta ? a.beta[c0 + e] : 0.f;
    }
  }
};
// v: x -> t; g: dy (already dropped) -> dz
template <int V, bool WHOLE> __device__ __forceinline__ void norm_dz(const NormArgs& a, const NormChan<V, WHOLE>& ch, float (&v)[V], float (&g)[V]) {
  float z[V];
#pragma unroll
  for (int e = 0; e < V; ++e) { v[e] -= ch.mean[WHOLE ? 0 : e]; z[e] = v[e] * ch.scale[e] + ch.beta[e]; }
  act_grad_apply<V>(g, z, a.act);
}
// What takes dz and t to dx = rstd (gamma dz - S1 - xh S2) = scale dz - k1 - t k2, from (S1, S2) by group
template <int V, bool WHOLE> struct NormBack {
  static constexpr int W = WHOLE ? 1 : V;
  float k1[W], k2[W];
  __device__ __forceinline__ void set(int e, float2 s, float rstd) { k1[e] = rstd * s.x; k2[e] = rstd * rstd * s.y; }
  __device__ __forceinline__ void apply(const NormChan<V, WHOLE>& ch, const float (&t)[V], float (&dz)[V]) const {
#pragma unroll
    for (int e = 0; e < V; ++e) dz[e] = (dz[e] * ch.scale[e] - k1[WHOLE ? 0 : e]) - t[e] * k2[WHOLE ? 0 : e];
  }
};
// (A, B) of each of the workgroup's channels from its threads' sums, in sum[0 .. span), seen by every thread.  All threads call.
// sum: TH * V numbers.
template <int V, int TH> __device__ __forceinline__ void team_channels(const NormArgs& a, const NormTeam& t, float (&sa)[V], float (&sb)[V], float2* sum) {
  const bool pow2 = a.cb <= 64 && (a.cb & (a.cb - 1)) == 0;
  if (pow2)
    for (int k = a.cb; k < 64; k <<= 1) {
#pragma unroll
      for (int e = 0; e < V; ++e) { sa[e] += __shfl_xor(sa[e], k); sb[e] += __shfl_xor(sb[e], k); }
    }
  const int rows = pow2 ? TH / 64 : a.rows, r = pow2 ? threadIdx.x >> 6 : t.row;
  if (pow2 ? (int)(threadIdx.x & 63) < a.cb : t.on) {
#pragma unroll
    for (int e = 0; e < V; ++e) sum[r * a.span + t.col * V + e] = make_float2(sa[e], sb[e]);
  }
  __syncthreads();
  for (int c = threadIdx.x; c < a.span; c += TH) {
    float2 s = sum[c];
    for (int k = 1; k < rows; ++k) { const float2 f = sum[k * a.span + c]; s.x += f.x; s.y += f.y; }
    sum[c] = s;                                              // (a column is read and written by one thread)
  }
  __syncthreads();
}
// (sum of gamma A, sum of gamma B) * scale of each of the workgroup's groups.  All threads call.
template <int TH> __device__ __forceinline__ void team_group_sums(const NormArgs& a, const NormTeam& t, const float2* sum, float scale, float2* out) {
  const int lanes = 1 << a.jl, lane = threadIdx.x & (lanes - 1), groups = a.span / a.d;
  for (int j0 = 0; j0 < groups; j0 += TH >> a.jl) {
    const int j = j0 + (threadIdx.x >> a.jl);
    float s1 = 0.f, s2 = 0.f;
    if (j < groups)
      for (int k = lane; k < a.d; k += lanes) {
        const float2 f = sum[j * a.d + k];
        const float gm = a.gamma ? a.gamma[t.cbase + j * a.d + k] : 1.f;
        s1 += gm * f.x; s2 += gm * f.y;
      }
    for (int k = lanes >> 1; k; k >>= 1) { s1 += __shfl_xor(s1, k); s2 += __shfl_xor(s2, k); }
    if (j < groups && lane == 0) out[j] = make_float2(s1 * scale, s2 * scale);
  }
}

// The whole backward pass of a span in registers, x and dy read once: (A, B) of its channels go to ab[image][channel] for the parameters'
// gradients over the images.  dz stays in registers as float32 between the sums and dx (dropout and the activation's gradient are half of the
// arithmetic: 32 x 48 x 48 x 128 bfloat16 took 33 us with both computed twice).  Bound as the forward pass is: 57 MB in 23.3 us, 24.3 with dropout (the
// two launches 38.9 and 40.1), 9.4 at the rate of a copy.
template <typename T, int V, int R, int TH, bool WHOLE> __global__ __launch_bounds__(TH) void norm_team_grad_kernel(const NormArgs a) {
  __shared__ float2 sum[TH * V];
  __shared__ float2 tot[TH * V];
  const NormTeam t = span_team<V>(a);
  const Walk<T, V> x(a, t, a.x, a.xcs, 0), dy(a, t, a.dy, a.dycs, 0), dx(a, t, a.y, a.ycs, 0);
  Pack<T, V> q[R], g[R];
#pragma unroll
  for (int r = 0; r < R; ++r)
    if (t.on && t.row + r * a.rows < a.p) {
      q[r].load(x.ptr(r));
      g[r].load(dy.ptr(r));
    }
  DropMask<V, R> drop;
  if (a.drop.thresh && t.on)
    drop.find(a.span % 8 == 0, ((uint64_t)t.img * a.p + t.row) * a.c + t.c0, (uint64_t)a.rows * a.c, a.drop, drop_offset(a.drop),
              [&](int r) { return t.row + r * a.rows < a.p; });
  NormChan<V, WHOLE> ch;
  ch.load(a, t.img, t.c0, t.on);
  float sa[V], sb[V], dz[R][V];
#pragma unroll
  for (int e = 0; e < V; ++e) sa[e] = sb[e] = 0.f;
#pragma unroll
  for (int r = 0; r < R; ++r)
    if (t.on && t.row + r * a.rows < a.p) {
      float v[V];
      q[r].widen(v);
      g[r].widen(dz[r]);
      if (a.drop.thresh) drop.apply(r, dz[r], a.drop.scale);
      norm_dz<V, WHOLE>(a, ch, v, dz[r]);
#pragma unroll
      for (int e = 0; e < V; ++e) { sa[e] += dz[r][e]; sb[e] += dz[r][e] * v[e]; }
    }
#pragma unroll
  for (int e = 0; e < V; ++e) sb[e] *= ch.rstd[WHOLE ? 0 : e];
  team_channels<V, TH>(a, t, sa, sb, sum);
  team_group_sums<TH>(a, t, sum, a.inv_m, tot);
  for (int c = threadIdx.x; c < a.span; c += TH) a.ab[(size_t)t.img * a.c + t.cbase + c] = sum[c];
  __syncthreads();
#pragma unroll
  for (int r = 0; r < R; ++r) q[r].keep();
  if (!t.on) return;
  NormBack<V, WHOLE> back;
#pragma unroll
  for (int e = 0; e < NormBack<V, WHOLE>::W; ++e) back.set(e, tot[div_by(t.col * V + e, a.by_d)], ch.rstd[e]);
#pragma unroll
  for (int r = 0; r < R; ++r)
    if (t.row + r * a.rows < a.p) {
      float v[V];
      q[r].widen(v);
#pragma unroll
      for (int e = 0; e < V; ++e) v[e] -= ch.mean[WHOLE ? 0 : e];
      back.apply(ch, v, dz[r]);
      store_v<T, V>(dx.ptr(r), dz[r]);
    }
}

// dz (w) and t = x - mean (v) of K vectors of the two-launch form from packed x and dy, elements i and i + di on; K = 2 where a generator
// block is two threads' work, m of them there
template <typename T, int V, bool WHOLE> struct GradPixels {
  static constexpr int K = V == 4 ? 2 : 1;
  float v[K][V], w[K][V];
  __device__ __forceinline__ void get(const NormArgs& a, const NormChan<V, WHOLE>& ch, const Pack<T, V>* q, const Pack<T, V>* g, uint64_t i, uint64_t di, int m,
                                      uint64_t offset) {
    bool pairs = false;
#pragma unroll
    for (int k = 0; k < K; ++k) { q[k].widen(v[k]); g[k].widen(w[k]); }
    if constexpr (K == 2) {
      pairs = a.span % 8 == 0;
      if (a.drop.thresh && pairs) drop_apply_pair<V>(w[0], w[1], i, i + di, a.drop, offset);
    }
#pragma unroll
    for (int k = 0; k < K; ++k)
      if (k < m) {
        if (a.drop.thresh && !pairs) drop_apply<V>(w[k], i + k * di, a.drop, offset);
        norm_dz<V, WHOLE>(a, ch, v[k], w[k]);
      }
  }
};

// Bound by memory: 32 x 96 x 96 x 64 float32, 75 MB a tensor, first launch 30.7 us (4.9 TB/s), second 36.9 us (6.1 TB/s).
// First launch: part[image][chunk][channel] = (A, B) of a chunk, and behind it s12[image][group][chunk] = (sum of gamma A, of gamma B) / (P D).
template <typename T, int V, int U> struct GradBuffer { Pack<T, V> x[U], dy[U]; };
template <typename T, int V, int TH, bool WHOLE> __global__ __launch_bounds__(TH) void norm_chunk_sums_kernel(const NormArgs a) {
  constexpr int U = 2, K = GradPixels<T, V, WHOLE>::K;
  typedef GradBuffer<T, V, U> B;
  __shared__ float2 sum[TH * V];
  __shared__ float2 tot[TH * V];
  int chunk, p0, p1;
  const NormTeam t = chunk_team<V>(a, blockIdx.x, a.chunks, a.ppc, chunk, p0, p1);
  const Walk<T, V> x(a, t, a.x, a.xcs, p0), dy(a, t, a.dy, a.dycs, p0);
  Chunk<U, B> c(a, t, p1 - p0);
  const auto load = [&](B& b, int r, int m) { x.load(b.x, r, m, a.nt); dy.load(b.dy, r, m, a.nt); };
  if (t.on) c.fetch(c.b0, 0, load);
  NormChan<V, WHOLE> ch;
  ch.load(a, t.img, t.c0, t.on);
  const uint64_t offset = a.drop.thresh ? drop_offset(a.drop) : 0;
  const uint64_t i0 = ((uint64_t)t.img * a.p + p0 + t.row) * a.c + t.c0, di = (uint64_t)a.rows * a.c;
  float sa[V], sb[V];
#pragma unroll
  for (int e = 0; e < V; ++e) sa[e] = sb[e] = 0.f;
  if (t.on)
    c.finish(load, [&](B& b, int r, int m) {
#pragma unroll
      for (int u = 0; u < U; u += K)
        if (u < m) {
          GradPixels<T, V, WHOLE> g;
          g.get(a, ch, b.x + u, b.dy + u, i0 + (r + u) * di, di, m - u, offset);
#pragma unroll
          for (int k = 0; k < K; ++k)
            if (u + k < m) {
#pragma unroll
              for (int e = 0; e < V; ++e) { sa[e] += g.w[k][e]; sb[e] += g.w[k][e] * g.v[k][e]; }
            }
        }
    });
#pragma unroll
  for (int e = 0; e < V; ++e) sb[e] *= ch.rstd[WHOLE ? 0 : e];
  team_channels<V, TH>(a, t, sa, sb, sum);
  team_group_sums<TH>(a, t, sum, a.inv_m, tot);
  for (int c = threadIdx.x; c < a.span; c += TH) a.part[((size_t)t.img * a.chunks + chunk) * a.c + t.cbase + c] = sum[c];
  __syncthreads();
  for (int j = threadIdx.x; j < a.span / a.d; j += TH) a.s12[((size_t)t.img * a.groups + t.cbase / a.d + j) * a.chunks + chunk] = tot[j];
}

// dgamma, dbeta of 16 channels: the sum over `rows` rows of (A, B) by channel (float64: a row is a chunk's or an image's sum)
__device__ __forceinline__ void param_grads(const NormArgs& a, const float2* ab, int rows, int block) {
  __shared__ double2 red[256];
  const int ch = block * 16 + (threadIdx.x & 15);
  double sa = 0.0, sb = 0.0;
  if (ch < a.c) {
#pragma unroll 4
    for (int r = threadIdx.x >> 4; r < rows; r += 16) { const float2 f = ab[(size_t)r * a.c + ch]; sa += f.x; sb += f.y; }
  }
  red[threadIdx.x] = make_double2(sa, sb);
  __syncthreads();
  if (threadIdx.x < 16 && ch < a.c) {
    for (int k = 1; k < 16; ++k) { sa += red[16 * k + threadIdx.x].x; sb += red[16 * k + threadIdx.x].y; }
    if (a.dbeta) a.dbeta[ch] = (float)(a.accumulate ? a.dbeta[ch] + sa : sa);
    if (a.dgamma) a.dgamma[ch] = (float)(a.accumulate ? a.dgamma[ch] + sb : sb);
  }
}
__global__ __launch_bounds__(256) void norm_params_kernel(const NormArgs a, const float2* ab, int rows) { param_grads(a, ab, rows, blockIdx.x); }

// Sums over `chunks` numbers of each of `groups` groups: 2^jl lanes a group, all groups at once
template <int TH> __device__ __forceinline__ void join_sums(const float2* part, int chunks, int groups, int jl, float2* out) {
  const int lanes = 1 << jl, lane = threadIdx.x & (lanes - 1);
  for (int j0 = 0; j0 < groups; j0 += TH >> jl) {
    const int j = j0 + (threadIdx.x >> jl);
    float s1 = 0.f, s2 = 0.f;
    if (j < groups) {
#pragma unroll 4
      for (int k = lane; k < chunks; k += lanes) { const float2 f = part[(size_t)j * chunks + k]; s1 += f.x; s2 += f.y; }
    }
    for (int k = lanes >> 1; k; k >>= 1) { s1 += __shfl_xor(s1, k); s2 += __shfl_xor(s2, k); }
    if (j < groups && lane == 0) out[j] = make_float2(s1, s2);
  }
}
// a wave a group of the whole batch, into ab[image][group]
__global__ __launch_bounds__(64) void norm_grad_join_kernel(const NormArgs a) {
  join_sums<64>(a.s12 + (size_t)blockIdx.x * a.chunks, a.chunks, 1, 6, a.ab + blockIdx.x);
}

// Second launch: dx.  Its first `pblocks` workgroups sum the parameters' gradients instead.
template <typename T, int V, int TH, bool WHOLE> __global__ __launch_bounds__(TH) void norm_chunk_grad_kernel(const NormArgs a, int pblocks) {
  static_assert(TH == 256, "param_grads");
  constexpr int U = 2, K = GradPixels<T, V, WHOLE>::K;
  typedef GradBuffer<T, V, U> B;
  __shared__ float2 tot[TH * V];
  if ((int)blockIdx.x < pblocks) {
    if (blockIdx.y == 0) param_grads(a, a.part, a.n * a.chunks, blockIdx.x);
    return;
  }
  int chunk, p0, p1;
  const NormTeam t = chunk_team<V>(a, blockIdx.x - pblocks, a.achunks, a.appc, chunk, p0, p1);
  const Walk<T, V> x(a, t, a.x, a.xcs, p0), dy(a, t, a.dy, a.dycs, p0), dx(a, t, a.y, a.ycs, p0);
  Chunk<U, B> c(a, t, p1 - p0);
  const auto load = [&](B& b, int r, int m) { x.load(b.x, r, m, a.nt); dy.load(b.dy, r, m, a.nt); };
  if (t.on) c.fetch(c.b0, 0, load);
  NormChan<V, WHOLE> ch;
  ch.load(a, t.img, t.c0, t.on);
  const size_t g0 = (size_t)t.img * a.groups + div_by(t.cbase, a.by_d);
  const int groups = div_by(a.span, a.by_d);
  if (a.join) {
    join_sums<TH>(a.s12 + g0 * a.chunks, a.chunks, groups, a.jl, tot);
  } else {
    for (int j = threadIdx.x; j < groups; j += TH) tot[j] = a.ab[g0 + j];
  }
  __syncthreads();
  if (!t.on) return;
  NormBack<V, WHOLE> back;
#pragma unroll
  for (int e = 0; e < NormBack<V, WHOLE>::W; ++e) back.set(e, tot[div_by(t.col * V + e, a.by_d)], ch.rstd[e]);
  const uint64_t offset = a.drop.thresh ? drop_offset(a.drop) : 0;
  const uint64_t i0 = ((uint64_t)t.img * a.p + p0 + t.row) * a.c + t.c0, di = (uint64_t)a.rows * a.c;
  c.finish(load, [&](B& b, int r, int m) {
#pragma unroll
    for (int u = 0; u < U; u += K)
      if (u < m) {
        GradPixels<T, V, WHOLE> g;
        g.get(a, ch, b.x + u, b.dy + u, i0 + (r + u) * di, di, m - u, offset);
#pragma unroll
        for (int k = 0; k < K; ++k)
          if (u + k < m) {
            back.apply(ch, g.v[k], g.w[k]);
            store_nt<T, V>(dx.ptr(r + u + k), g.w[k]);
          }
      }
  });
}

// ---- any shape: workgroups of any channels, three launches (four backward).  What the forms above do not take: pixels of more vectors
// than a workgroup has threads.  4 x 64 x 64 x 1031 float32 (68 MB): 53 us in 1031 groups, 72 in one, where one workgroup an image joins the chunks;
// backward 97 and 96.  Scalar accesses, as the odd channels want them, bound the rest ----
struct NormTile {
  int img, chunk, p0, p1, row, c0;
  bool on;
  template <int V> __device__ __forceinline__ static NormTile get(const NormArgs& a) {
    NormTile t;
    t.img = blockIdx.x / a.chunks; t.chunk = blockIdx.x - t.img * a.chunks;
    t.p0 = t.chunk * a.ppc; t.p1 = min(a.p, t.p0 + a.ppc);
    t.row = threadIdx.x / a.cb;
    t.c0 = (blockIdx.y * a.cb + (threadIdx.x - t.row * a.cb)) * V;
    t.on = t.row < a.rows && t.c0 < a.c;
    return t;
  }
};

// ---- statistics, first half: (mean, M2) of every channel over a chunk ----
template <typename T, int V> __global__ __launch_bounds__(256) void norm_stats_kernel(const NormArgs a) {
  constexpr int U = 4;
  __shared__ float2 red[256 * V];
  const NormTile t = NormTile::get<V>(a);
  float mean[V], m2[V];
#pragma unroll
  for (int e = 0; e < V; ++e) mean[e] = m2[e] = 0.f;
  if (t.on) {
    const T* x = (const T*)a.x + ((size_t)t.img * a.p) * a.xcs + t.c0;
    float cnt = 0.f;
    for (int p = t.p0 + t.row; p < t.p1; p += U * a.rows) {
      const int m = min(U, (t.p1 - p + a.rows - 1) / a.rows);
      Pack<T, V> q[U];
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (u < m) q[u].load(x + (size_t)(p + u * a.rows) * a.xcs);
      stats_batch<T, V, U>(q, m, mean, m2, cnt);
    }
#pragma unroll
    for (int e = 0; e < V; ++e) red[threadIdx.x * V + e] = make_float2(mean[e], m2[e]);
  }
  __syncthreads();
  const int len = t.p1 - t.p0, nch = min(a.cb * V, a.c - (int)blockIdx.y * a.cb * V);
  for (int ch = threadIdx.x; ch < nch; ch += 256) {
    float s = 0.f;
    for (int r = 0; r < min(a.rows, len); ++r) s += red[r * a.cb * V + ch].x * (float)((len - r + a.rows - 1) / a.rows);
    const float m = s / (float)len;
    float q = 0.f;
    for (int r = 0; r < min(a.rows, len); ++r) {
      const float2 f = red[r * a.cb * V + ch];
      q += f.y + (float)((len - r + a.rows - 1) / a.rows) * (f.x - m) * (f.x - m);
    }
    a.part[((size_t)t.img * a.chunks + t.chunk) * a.c + blockIdx.y * a.cb * V + ch] = make_float2(m, q);
  }
}

template <int TH> __device__ __forceinline__ double block_sum(double v, double* red) {            // red: TH / 64 numbers; the same value for every thread
#pragma unroll
  for (int s = 32; s; s >>= 1) v += __shfl_xor(v, s);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  v = 0.0;
#pragma unroll
  for (int k = 0; k < TH / 64; ++k) v += red[k];
  return v;
}

// ---- statistics, second half: one workgroup per (image, group) joins the chunks' (mean, M2) of its channels: nd channels beside each other,
// `lanes` chunks at once.  Bound by its loads' latency where there are few groups: 1024 threads there. ----
template <int TH> __global__ __launch_bounds__(TH) void norm_stats_join_kernel(const NormArgs a) {
  __shared__ double red[TH / 64];
  const int img = blockIdx.x / a.groups, g = blockIdx.x - img * a.groups;
  const float2* part = a.part + (size_t)img * a.chunks * a.c + (size_t)g * a.d;
  const int nd = min(TH, a.d), lanes = TH / nd, k0 = threadIdx.x / nd, ch0 = threadIdx.x - k0 * nd;
  const double m = (double)a.p * a.d;
  double s = 0.0;
  if (k0 < lanes)
    for (int ch = ch0; ch < a.d; ch += nd) {
#pragma unroll 8
      for (int k = k0; k < a.chunks; k += lanes) s += (double)part[(size_t)k * a.c + ch].x * min(a.ppc, a.p - k * a.ppc);
    }
  const double mean = block_sum<TH>(s, red) / m;
  double q = 0.0;
  if (k0 < lanes)
    for (int ch = ch0; ch < a.d; ch += nd) {
#pragma unroll 8
      for (int k = k0; k < a.chunks; k += lanes) {
        const float2 f = part[(size_t)k * a.c + ch];
        q += (double)f.y + ((double)f.x - mean) * ((double)f.x - mean) * min(a.ppc, a.p - k * a.ppc);
      }
    }
  const double var = block_sum<TH>(q, red) / m;
  if (threadIdx.x == 0) {
    a.mean[blockIdx.x] = (float)mean;
    a.rstd[blockIdx.x] = (float)(1.0 / sqrt(var + (double)a.eps));
  }
}

// ---- y = drop(act((x - mean) * rstd * gamma + beta)) ----
template <typename T, int V> __global__ __launch_bounds__(256) void norm_apply_kernel(const NormArgs a) {
  const NormTile t = NormTile::get<V>(a);
  if (!t.on) return;
  NormChan<V, false> ch;
  ch.load(a, t.img, t.c0, true);
  const uint64_t offset = a.drop.thresh ? drop_offset(a.drop) : 0;
  const T* x = (const T*)a.x + (size_t)t.img * a.p * a.xcs + t.c0;
  T* y = (T*)a.y + (size_t)t.img * a.p * a.ycs + t.c0;
  for (int p = t.p0 + t.row; p < t.p1; p += a.rows) {
    float v[V];
    load_v<T, V>(x + (size_t)p * a.xcs, v);
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] = (v[e] - ch.mean[e]) * ch.scale[e] + ch.beta[e];
    act_apply<V>(v, a.act);
    if (a.drop.thresh) drop_apply<V>(v, ((uint64_t)t.img * a.p + p) * a.c + t.c0, a.drop, offset);
    store_v<T, V>(y + (size_t)p * a.ycs, v);
  }
}

// ---- backward, first half: (A, B) of every channel over a chunk ----
template <typename T, int V> __global__ __launch_bounds__(256) void norm_bwd_sums_kernel(const NormArgs a) {
  __shared__ float2 red[256 * V];
  const NormTile t = NormTile::get<V>(a);
  if (t.on) {
    NormChan<V, false> ch;
    ch.load(a, t.img, t.c0, true);
    const uint64_t offset = a.drop.thresh ? drop_offset(a.drop) : 0;
    float sa[V], sb[V];
#pragma unroll
    for (int e = 0; e < V; ++e) sa[e] = sb[e] = 0.f;
    const T* x = (const T*)a.x + (size_t)t.img * a.p * a.xcs + t.c0;
    const T* dy = (const T*)a.dy + (size_t)t.img * a.p * a.dycs + t.c0;
    for (int p = t.p0 + t.row; p < t.p1; p += a.rows) {
      float v[V], g[V];
      load_v<T, V>(x + (size_t)p * a.xcs, v);
      load_v<T, V>(dy + (size_t)p * a.dycs, g);
      if (a.drop.thresh) drop_apply<V>(g, ((uint64_t)t.img * a.p + p) * a.c + t.c0, a.drop, offset);
      norm_dz<V, false>(a, ch, v, g);
#pragma unroll
      for (int e = 0; e < V; ++e) { sa[e] += g[e]; sb[e] += g[e] * v[e]; }
    }
#pragma unroll
    for (int e = 0; e < V; ++e) red[threadIdx.x * V + e] = make_float2(sa[e], sb[e] * ch.rstd[e]);
  }
  __syncthreads();
  const int nch = min(a.cb * V, a.c - (int)blockIdx.y * a.cb * V);
  for (int k = threadIdx.x; k < nch; k += 256) {
    float2 s = make_float2(0.f, 0.f);
    for (int r = 0; r < a.rows; ++r) { const float2 f = red[r * a.cb * V + k]; s.x += f.x; s.y += f.y; }
    a.part[((size_t)t.img * a.chunks + t.chunk) * a.c + blockIdx.y * a.cb * V + k] = s;
  }
}

// ---- backward, join: one workgroup per (image, group): (A, B) of its channels over the chunks, then S1, S2 ----
template <int TH> __global__ __launch_bounds__(TH) void norm_bwd_join_kernel(const NormArgs a) {
  __shared__ double2 sum[TH];
  __shared__ double red[TH / 64];
  const int img = blockIdx.x / a.groups, g = blockIdx.x - img * a.groups;
  double s1 = 0.0, s2 = 0.0;
  for (int cb0 = 0; cb0 < a.d; cb0 += TH) {
    const int nd = min(TH, a.d - cb0), lanes = TH / nd, k0 = threadIdx.x / nd, ch = threadIdx.x - k0 * nd;
    double sa = 0.0, sb = 0.0;
    if (k0 < lanes) {
#pragma unroll 8
      for (int k = k0; k < a.chunks; k += lanes) {
        const float2 f = a.part[((size_t)img * a.chunks + k) * a.c + (size_t)g * a.d + cb0 + ch];
        sa += f.x; sb += f.y;
      }
    }
    __syncthreads();
    sum[threadIdx.x] = make_double2(sa, sb);
    __syncthreads();
    if ((int)threadIdx.x < nd) {
      sa = sb = 0.0;
      for (int k = 0; k < lanes; ++k) { sa += sum[k * nd + threadIdx.x].x; sb += sum[k * nd + threadIdx.x].y; }
      const int c = g * a.d + cb0 + threadIdx.x;
      a.ab[(size_t)img * a.c + c] = make_float2((float)sa, (float)sb);
      const double gm = a.gamma ? (double)a.gamma[c] : 1.0;
      s1 += gm * sa; s2 += gm * sb;
    }
  }
  const double m = (double)a.p * a.d;
  s1 = block_sum<TH>(s1, red); s2 = block_sum<TH>(s2, red);
  if (threadIdx.x == 0) a.s12[blockIdx.x] = make_float2((float)(s1 / m), (float)(s2 / m));
}

// ---- backward, second half: dx ----
template <typename T, int V> __global__ __launch_bounds__(256) void norm_bwd_apply_kernel(const NormArgs a) {
  const NormTile t = NormTile::get<V>(a);
  if (!t.on) return;
  NormChan<V, false> ch;
  ch.load(a, t.img, t.c0, true);
  NormBack<V, false> back;
#pragma unroll
  for (int e = 0; e < V; ++e) back.set(e, a.s12[(size_t)t.img * a.groups + div_by(t.c0 + e, a.by_d)], ch.rstd[e]);
  const uint64_t offset = a.drop.thresh ? drop_offset(a.drop) : 0;
  const T* x = (const T*)a.x + (size_t)t.img * a.p * a.xcs + t.c0;
  const T* dy = (const T*)a.dy + (size_t)t.img * a.p * a.dycs + t.c0;
  T* dx = (T*)a.y + (size_t)t.img * a.p * a.ycs + t.c0;
  for (int p = t.p0 + t.row; p < t.p1; p += a.rows) {
    float v[V], g[V];
    load_v<T, V>(x + (size_t)p * a.xcs, v);
    load_v<T, V>(dy + (size_t)p * a.dycs, g);
    if (a.drop.thresh) drop_apply<V>(g, ((uint64_t)t.img * a.p + p) * a.c + t.c0, a.drop, offset);
    norm_dz<V, false>(a, ch, v, g);
    back.apply(ch, v, g);
    store_v<T, V>(dx + (size_t)p * a.ycs, g);
  }
}

// ---- dropout: y = drop(x) [+ res] ----
// A workgroup takes 256 x DROP_U vectors of 16 bytes that follow each other; float32: a generator block is two lanes' work, see
// drop_apply_pair.  Bound by memory: 13 x 271 x 495 x 29 float32 without a residual in 65 us = 6.3 TB/s, 32 x 96 x 96 x 64 bfloat16 with one in
// 18.2 us = 6.2 TB/s.  Two and four times as much work a workgroup: 67 and 69 us, 18.6 and 18.7 us.
constexpr int DROP_U = 4;
template <typename T, bool NT, bool NT_OUT> __global__ __launch_bounds__(256) void dropout_kernel(const T* x, const T* res, T* y, size_t count, DropArgs d) {
  constexpr int V = 16 / sizeof(T), U = DROP_U;
  const uint64_t offset = d.thresh ? drop_offset(d) : 0;
  const size_t first = (size_t)blockIdx.x * (256 * U * V);
  const T* const xb = x + first;                             // uniform: the threads' parts of the addresses have 32 bits
  const T* const rb = res + first;
  T* const yb = y + first;
  const uint32_t at = threadIdx.x * V;
  if (first + 256 * U * V > count) {                         // the last workgroup
    for (uint32_t e = threadIdx.x; first + e < count; e += 256) {
      float v[1] = {(float)xb[e]};
      if (d.thresh) drop_apply<1>(v, first + e, d, offset);
      yb[e] = (T)(res ? v[0] + (float)rb[e] : v[0]);
    }
    return;
  }
  Pack<T, V> q[U], r[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const T *xp = xb + u * 256 * V + at, *rp = rb + u * 256 * V + at;
    if constexpr (NT) q[u].load_nt(xp);
    else q[u].load(xp);
    if (res) {
      if constexpr (NT) r[u].load_nt(rp);
      else r[u].load(rp);
    }
  }
  float v[2][V];
#pragma unroll
  for (int u = 0; u < U; u += 2) {
    q[u].widen(v[0]);
    q[u + 1].widen(v[1]);
    const uint64_t i = first + u * 256 * V + at;
    if (d.thresh) {
      if constexpr (V == 4) drop_apply_pair<V>(v[0], v[1], i, i + 256 * V, d, offset);
      else { drop_apply<V>(v[0], i, d, offset); drop_apply<V>(v[1], i + 256 * V, d, offset); }
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      if (res) {
#pragma unroll
        for (int e = 0; e < V; ++e) v[k][e] += r[u + k].get(e);
      }
      if constexpr (NT_OUT) store_nt<T, V>(yb + (u + k) * 256 * V + at, v[k]);
      else store_v<T, V>(yb + (u + k) * 256 * V + at, v[k]);
    }
  }
}
// tensors that allow no vector accesses: a thread per generator block
template <typename T> __global__ __launch_bounds__(256) void dropout_any_kernel(const T* x, const T* res, T* y, size_t count, DropArgs d) {
  const size_t blocks = (count + 7) / 8, stride = (size_t)gridDim.x * 256;
  const uint64_t offset = d.thresh ? drop_offset(d) : 0;
  for (size_t b = (size_t)blockIdx.x * 256 + threadIdx.x; b < blocks; b += stride) {
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = 8 * b + e < count ? (float)x[8 * b + e] : 0.f;
    if (d.thresh) drop_apply<8>(v, 8 * b, d, offset);
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (8 * b + e < count) y[8 * b + e] = (T)(res ? v[e] + (float)res[8 * b + e] : v[e]);
  }
}

}  // namespace fisr
