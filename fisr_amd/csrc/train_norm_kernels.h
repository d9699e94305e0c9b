// Kernels of the training graph's normalisation and regularisation: group normalisation with an activation and dropout,
// channels last.  x [N, P, C] (P = H * W pixels with a pixel stride of xcs elements), G groups of D = C / G channels:
//
//   mean[n,g], rstd[n,g] = 1 / sqrt(var + eps) over the P * D values of a group (biased variance)
//   xh = (x - mean) * rstd,  z = xh * gamma[c] + beta[c],  y = drop(act(z))
//   backward: dz = drop(dy) * act'(z);  A[n,c] = sum_p dz,  B[n,c] = sum_p dz * xh;  dbeta = sum_n A,  dgamma = sum_n B
//             dx = rstd * (dz * gamma - S1 / (P D) - xh * S2 / (P D)),  S1[n,g] = sum_{c in g} gamma A,  S2 = sum gamma B
//
// Every sum, statistic and intermediate is float32 (the merges over workgroups float64); only y and dx are rounded, once, to the
// tensors' type.  There are no atomics: partial results go through the workspace and are joined in a fixed order, so a call's
// results are the same bits every time.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

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

// ---- loads and stores of V channels as floats.  The caller sees to alignment: 16 bytes, or V elements where that is less ----
template <typename T, int V> struct alignas(sizeof(T) * V < 16 ? sizeof(T) * V : 16) Pack { T e[V]; };
template <typename T, int V> __device__ __forceinline__ void load_v(const T* p, float (&v)[V]) {
  const Pack<T, V> q = *reinterpret_cast<const Pack<T, V>*>(p);
#pragma unroll
  for (int e = 0; e < V; ++e) v[e] = (float)q.e[e];
}
template <typename T, int V> __device__ __forceinline__ void store_v(T* p, const float (&v)[V]) {
  Pack<T, V> q;
#pragma unroll
  for (int e = 0; e < V; ++e) q.e[e] = (T)v[e];
  *reinterpret_cast<Pack<T, V>*>(p) = q;
}

// ---- activations ----
__device__ __forceinline__ float sigmoid_f(float z) { return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-1.4426950408889634f * z)); }
template <int V> __device__ __forceinline__ void act_apply(float (&z)[V], int act) {
  if (act == NORM_ACT_RELU) {
#pragma unroll
    for (int e = 0; e < V; ++e) z[e] = z[e] < 0.f ? 0.f : z[e];          // NaN stays (a maximum with zero would drop it)
  } else if (act == NORM_ACT_SILU) {
#pragma unroll
    for (int e = 0; e < V; ++e) z[e] *= sigmoid_f(z[e]);
  } else if (act == NORM_ACT_GELU) {
#pragma unroll
    for (int e = 0; e < V; ++e) z[e] *= 0.5f + 0.5f * erff(0.70710678f * z[e]);
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
    for (int e = 0; e < V; ++e)
      g[e] *= 0.5f + 0.5f * erff(0.70710678f * z[e]) + z[e] * (0.39894228f * __builtin_amdgcn_exp2f(-0.72134752f * z[e] * z[e]));
  }
}

// ---- work of a launch: a workgroup of 256 threads takes `ppc` pixels of one image and up to cb channel vectors; its threads are
// `rows` rows of cb, a thread keeps its V channels and walks the pixels row, row + rows, ... ----
struct NormArgs {
  const void* x; const void* dy; void* y;              // y: the output (dx in the backward pass)
  const float* gamma; const float* beta;               // nullable
  float* mean; float* rstd;                            // [N][G]
  float2* part;                                        // [N][chunks][C]: (mean, M2) or (A, B) of a chunk
  float2* ab; float2* s12;                             // backward: [N][C] (A, B), [N][G] (S1, S2) / (P D)
  float* dgamma; float* dbeta;
  size_t xcs, ycs, dycs;                               // pixel strides, elements
  int n, p, c, groups, d;
  int cb, rows, chunks, ppc;                           // chunks = ceil(p / ppc)
  float eps; int act, accumulate;
  DropArgs drop;
};
struct NormTile {
  int img, chunk, p0, p1, row, c0;
  bool on;
  template <int V> __device__ __forceinline__ static NormTile get(const NormArgs& a) {
    NormTile t;
    t.img = blockIdx.x / a.chunks; t.chunk = blockIdx.x - t.img * a.chunks;
    t.p0 = t.chunk * a.ppc; t.p1 = min(a.p, t.p0 + a.ppc);                               // (chunks * ppc < 2^31: see norm_tiling)
    t.row = threadIdx.x / a.cb;
    t.c0 = (blockIdx.y * a.cb + (threadIdx.x - t.row * a.cb)) * V;
    t.on = t.row < a.rows && t.c0 < a.c;
    return t;
  }
};

// ---- statistics, first half: (mean, M2) of every channel over a chunk ----
// A batch of U pixels is reduced about its own mean and joined to the running (mean, M2) by Chan's formula, so nothing is lost when the
// mean is large against the spread: no sum of squares about a far point exists anywhere.
template <typename T, int V> __global__ __launch_bounds__(256) void norm_stats_kernel(const NormArgs a) {
  constexpr int U = 4;
  __shared__ float2 red[256 * V];
  const NormTile t = NormTile::get<V>(a);
  float mean[V], m2[V];
#pragma unroll
  for (int e = 0; e < V; ++e) mean[e] = m2[e] = 0.f;
  if (t.on) {
    const T* x = (const T*)a.x + ((size_t)t.img * a.p) * a.xcs + t.c0;
    int p = t.p0 + t.row;
    float cnt = 0.f;
    for (; p + (U - 1) * a.rows < t.p1; p += U * a.rows) {
      float v[U][V];
#pragma unroll
      for (int u = 0; u < U; ++u) load_v<T, V>(x + (size_t)(p + u * a.rows) * a.xcs, v[u]);
      const float w = (float)U / (cnt + (float)U), nw = cnt * w;
      cnt += (float)U;
#pragma unroll
      for (int e = 0; e < V; ++e) {
        float s = v[0][e];
#pragma unroll
        for (int u = 1; u < U; ++u) s += v[u][e];
        const float bm = s * (1.f / U);
        float b2 = 0.f;
#pragma unroll
        for (int u = 0; u < U; ++u) { const float dv = v[u][e] - bm; b2 += dv * dv; }
        const float dm = bm - mean[e];
        mean[e] += dm * w;
        m2[e] += b2 + dm * dm * nw;
      }
    }
    for (; p < t.p1; p += a.rows) {
      float v[V];
      load_v<T, V>(x + (size_t)p * a.xcs, v);
      const float w = 1.f / (cnt + 1.f), nw = cnt * w;
      cnt += 1.f;
#pragma unroll
      for (int e = 0; e < V; ++e) { const float dm = v[e] - mean[e]; mean[e] += dm * w; m2[e] += dm * dm * nw; }
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

__device__ __forceinline__ double block_sum(double v, double* red) {            // 256 threads; the same value for every thread
#pragma unroll
  for (int s = 32; s; s >>= 1) v += __shfl_xor(v, s);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  return (red[0] + red[1]) + (red[2] + red[3]);
}

// ---- statistics, second half: one workgroup per (image, group) joins the chunks' (mean, M2) of its channels ----
__global__ __launch_bounds__(256) void norm_stats_join_kernel(const NormArgs a) {
  __shared__ double red[4];
  const int img = blockIdx.x / a.groups, g = blockIdx.x - img * a.groups;
  const float2* part = a.part + (size_t)img * a.chunks * a.c + (size_t)g * a.d;
  const int total = a.chunks * a.d;
  const double m = (double)a.p * a.d;
  double s = 0.0;
  for (int i = threadIdx.x; i < total; i += 256) {
    const int k = i / a.d, ch = i - k * a.d;
    s += (double)part[(size_t)k * a.c + ch].x * min(a.ppc, a.p - k * a.ppc);
  }
  const double mean = block_sum(s, red) / m;
  double q = 0.0;
  for (int i = threadIdx.x; i < total; i += 256) {
    const int k = i / a.d, ch = i - k * a.d;
    const float2 f = part[(size_t)k * a.c + ch];
    q += (double)f.y + ((double)f.x - mean) * ((double)f.x - mean) * min(a.ppc, a.p - k * a.ppc);
  }
  const double var = block_sum(q, red) / m;
  if (threadIdx.x == 0) {
    a.mean[blockIdx.x] = (float)mean;
    a.rstd[blockIdx.x] = (float)(1.0 / sqrt(var + (double)a.eps));
  }
}

// What a thread needs of its V channels: xh = (x - mean) * rstd, z = xh * gamma + beta.  (x - mean first: rstd * x + const would round
// twice at the size of mean * rstd.)
template <int V> struct NormChan {
  float mean[V], rstd[V], gamma[V], beta[V];
  __device__ __forceinline__ void load(const NormArgs& a, int img, int c0) {
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const int g = (c0 + e) / a.d;
      mean[e] = a.mean[(size_t)img * a.groups + g];
      rstd[e] = a.rstd[(size_t)img * a.groups + g];
      gamma[e] = a.gamma ? a.gamma[c0 + e] : 1.f;
      beta[e] = a.beta ? a.beta[c0 + e] : 0.f;
    }
  }
};

__device__ __forceinline__ uint64_t drop_offset(const DropArgs& d) { return d.offset + (d.counter ? *d.counter : 0); }

// ---- y = drop(act((x - mean) * rstd * gamma + beta)) ----
template <typename T, int V> __global__ __launch_bounds__(256) void norm_apply_kernel(const NormArgs a) {
  const NormTile t = NormTile::get<V>(a);
  if (!t.on) return;
  NormChan<V> ch;
  ch.load(a, t.img, t.c0);
#pragma unroll
  for (int e = 0; e < V; ++e) ch.rstd[e] *= ch.gamma[e];
  const uint64_t offset = a.drop.thresh ? drop_offset(a.drop) : 0;
  const T* x = (const T*)a.x + (size_t)t.img * a.p * a.xcs + t.c0;
  T* y = (T*)a.y + (size_t)t.img * a.p * a.ycs + t.c0;
  for (int p = t.p0 + t.row; p < t.p1; p += a.rows) {
    float v[V];
    load_v<T, V>(x + (size_t)p * a.xcs, v);
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] = (v[e] - ch.mean[e]) * ch.rstd[e] + ch.beta[e];
    act_apply<V>(v, a.act);
    if (a.drop.thresh) drop_apply<V>(v, ((uint64_t)t.img * a.p + p) * a.c + t.c0, a.drop, offset);
    store_v<T, V>(y + (size_t)p * a.ycs, v);
  }
}

// dz and xh of one vector
template <int V> __device__ __forceinline__ void norm_dz(const NormArgs& a, const NormChan<V>& ch, float (&v)[V], float (&g)[V], uint64_t i, uint64_t offset) {
  float z[V];
#pragma unroll
  for (int e = 0; e < V; ++e) { v[e] = (v[e] - ch.mean[e]) * ch.rstd[e]; z[e] = v[e] * ch.gamma[e] + ch.beta[e]; }
  if (a.drop.thresh) drop_apply<V>(g, i, a.drop, offset);
  act_grad_apply<V>(g, z, a.act);
}

// ---- backward, first half: (A, B) of every channel over a chunk ----
template <typename T, int V> __global__ __launch_bounds__(256) void norm_bwd_sums_kernel(const NormArgs a) {
  __shared__ float2 red[256 * V];
  const NormTile t = NormTile::get<V>(a);
  if (t.on) {
    NormChan<V> ch;
    ch.load(a, t.img, t.c0);
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
      norm_dz<V>(a, ch, v, g, ((uint64_t)t.img * a.p + p) * a.c + t.c0, offset);
#pragma unroll
      for (int e = 0; e < V; ++e) { sa[e] += g[e]; sb[e] += g[e] * v[e]; }
    }
#pragma unroll
    for (int e = 0; e < V; ++e) red[threadIdx.x * V + e] = make_float2(sa[e], sb[e]);
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
__global__ __launch_bounds__(256) void norm_bwd_join_kernel(const NormArgs a) {
  __shared__ double2 sum[256];
  __shared__ double red[4];
  const int img = blockIdx.x / a.groups, g = blockIdx.x - img * a.groups;
  double s1 = 0.0, s2 = 0.0;
  for (int cb0 = 0; cb0 < a.d; cb0 += 256) {
    const int nd = min(256, a.d - cb0), lanes = 256 / nd, k0 = threadIdx.x / nd, ch = threadIdx.x - k0 * nd;
    double sa = 0.0, sb = 0.0;
    if (k0 < lanes)
      for (int k = k0; k < a.chunks; k += lanes) {
        const float2 f = a.part[((size_t)img * a.chunks + k) * a.c + (size_t)g * a.d + cb0 + ch];
        sa += f.x; sb += f.y;
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
  s1 = block_sum(s1, red); s2 = block_sum(s2, red);
  if (threadIdx.x == 0) a.s12[blockIdx.x] = make_float2((float)(s1 / m), (float)(s2 / m));
}

// ---- backward: dgamma, dbeta over the images (a thread per channel and quarter of the images) ----
__global__ __launch_bounds__(256) void norm_bwd_params_kernel(const NormArgs a) {
  __shared__ double2 red[256];
  const int c = blockIdx.x * 64 + (threadIdx.x & 63);
  double sa = 0.0, sb = 0.0;
  if (c < a.c)
    for (int n = threadIdx.x >> 6; n < a.n; n += 4) { const float2 f = a.ab[(size_t)n * a.c + c]; sa += f.x; sb += f.y; }
  red[threadIdx.x] = make_double2(sa, sb);
  __syncthreads();
  if (threadIdx.x < 64 && c < a.c) {
    for (int k = 1; k < 4; ++k) { sa += red[64 * k + threadIdx.x].x; sb += red[64 * k + threadIdx.x].y; }
    if (a.dbeta) a.dbeta[c] = (float)(a.accumulate ? a.dbeta[c] + sa : sa);
    if (a.dgamma) a.dgamma[c] = (float)(a.accumulate ? a.dgamma[c] + sb : sb);
  }
}

// ---- backward, second half: dx ----
template <typename T, int V> __global__ __launch_bounds__(256) void norm_bwd_apply_kernel(const NormArgs a) {
  const NormTile t = NormTile::get<V>(a);
  if (!t.on) return;
  NormChan<V> ch;
  ch.load(a, t.img, t.c0);
  float s1[V], s2[V];
#pragma unroll
  for (int e = 0; e < V; ++e) { const float2 s = a.s12[(size_t)t.img * a.groups + (t.c0 + e) / a.d]; s1[e] = s.x; s2[e] = s.y; }
  const uint64_t offset = a.drop.thresh ? drop_offset(a.drop) : 0;
  const T* x = (const T*)a.x + (size_t)t.img * a.p * a.xcs + t.c0;
  const T* dy = (const T*)a.dy + (size_t)t.img * a.p * a.dycs + t.c0;
  T* dx = (T*)a.y + (size_t)t.img * a.p * a.ycs + t.c0;
  for (int p = t.p0 + t.row; p < t.p1; p += a.rows) {
    float v[V], g[V];
    load_v<T, V>(x + (size_t)p * a.xcs, v);
    load_v<T, V>(dy + (size_t)p * a.dycs, g);
    norm_dz<V>(a, ch, v, g, ((uint64_t)t.img * a.p + p) * a.c + t.c0, offset);
#pragma unroll
    for (int e = 0; e < V; ++e) g[e] = ch.rstd[e] * (g[e] * ch.gamma[e] - s1[e] - v[e] * s2[e]);
    store_v<T, V>(dx + (size_t)p * a.ycs, g);
  }
}

// ---- dropout: y = drop(x) [+ res]; a thread per generator block of eight elements ----
template <typename T, bool ALIGNED> __global__ __launch_bounds__(256) void dropout_kernel(const T* x, const T* res, T* y, size_t count, DropArgs d) {
  const size_t blocks = (count + 7) / 8, stride = (size_t)gridDim.x * 256;
  const uint64_t offset = d.thresh ? drop_offset(d) : 0;
  for (size_t b = (size_t)blockIdx.x * 256 + threadIdx.x; b < blocks; b += stride) {
    float v[8], r[8];
    if (ALIGNED && 8 * b + 8 <= count) {
      load_v<T, 8>(x + 8 * b, v);
      if (res) load_v<T, 8>(res + 8 * b, r);
      if (d.thresh) drop_apply<8>(v, 8 * b, d, offset);
      if (res)
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] += r[e];
      store_v<T, 8>(y + 8 * b, v);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = 8 * b + e < count ? (float)x[8 * b + e] : 0.f;
      if (d.thresh) drop_apply<8>(v, 8 * b, d, offset);
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (8 * b + e < count) y[8 * b + e] = (T)(res ? v[e] + (float)res[8 * b + e] : v[e]);
    }
  }
}

}  // namespace fisr
