// Group norm with an activation on gfx950, channels last, forward and backward.
//
//   y = act((x - mean) rstd * gamma + beta),   rstd = 1 / sqrt(var + eps), biased variance,
//
// with mean and variance over the frames inside the length and the C / G channels of a group (one sample = one utterance
// [T][C]), act = none, ReLU or SiLU.  With T = 1 every row is a sample of its own (a frame's heads behind an attention).
// Backward, with xhat = (x - mean) rstd, z = xhat gamma + beta, dz = dy act'(z), n = frames * C / G:
//   dgamma_c = sum dz xhat,  dbeta_c = sum dz                                      (over samples and frames)
//   dx = rstd (gamma dz - (sum_group gamma dz) / n - xhat (sum_group gamma dz xhat) / n).
//
// A thread owns V neighbouring channels of one group (V = what divides C / G, up to 16 bytes), so every load is as wide as
// the group allows and one partial sum serves the V values.
//   rows (T = 1, no lengths): a row's C / V threads hold it in registers -- one read, one write -- and sum a group over its threads by
//     shuffles when they are a power of two, through LDS otherwise.
//   utterances: the frames of an utterance are split over workgroups.  k_gn_stats leaves (count, mean, centred second
//     moment) of each split and group, k_gn_apply joins them and normalises.  The backward does the same with the
//     per-channel sums of dz and dz xhat, from which the group sums and the parameter gradients both follow.
// Sums are 32-bit, second moments about a value of the data, never as a difference of large sums; the moments of
// different threads are joined in 64 bits.  Fixed order, no atomics.  HBM-bound.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "lmufft.h"
#include "lmufft_internal.h"

namespace lmufft {

constexpr int kGnMaxWidth = 1024;
constexpr int kGnMaxSplits = 64;
constexpr int kGnRowBwdBlocks = 1024;  // workgroups of the rows backward: each leaves one partial of the parameter gradients

enum { kGnNone = 0, kGnRelu = 1, kGnSilu = 2 };

__device__ __forceinline__ float gn_act(float z, int act) {
  if (act == kGnRelu) return z > 0.f ? z : (z == z ? 0.f : z);
  if (act == kGnSilu) return z / (1.f + __expf(-z));
  return z;
}
__device__ __forceinline__ float gn_slope(float z, int act) {
  if (act == kGnRelu) return z > 0.f ? 1.f : 0.f;
  if (act == kGnSilu) {
    const float s = 1.f / (1.f + __expf(-z));
    return s * (1.f + z * (1.f - s));
  }
  return 1.f;
}

// V neighbouring values, loaded and stored at once
template <int V>
struct GnVec {
  float f[V];
};
template <bool BF16, int V>
__device__ __forceinline__ GnVec<V> gn_load(const void* base, long idx) {
  GnVec<V> o;
  if (BF16) {
    typedef __bf16 vec __attribute__((ext_vector_type(V)));
    const vec v = *reinterpret_cast<const vec*>(reinterpret_cast<const __bf16*>(base) + idx);
#pragma unroll
    for (int e = 0; e < V; ++e) o.f[e] = (float)v[e];
  } else {
    typedef float vec __attribute__((ext_vector_type(V)));
    const vec v = *reinterpret_cast<const vec*>(reinterpret_cast<const float*>(base) + idx);
#pragma unroll
    for (int e = 0; e < V; ++e) o.f[e] = v[e];
  }
  return o;
}
template <bool BF16, int V>
__device__ __forceinline__ void gn_store(void* base, long idx, const GnVec<V>& v) {
  if (BF16) {
    typedef __bf16 vec __attribute__((ext_vector_type(V)));
    vec o;
#pragma unroll
    for (int e = 0; e < V; ++e) o[e] = (__bf16)v.f[e];
    *reinterpret_cast<vec*>(reinterpret_cast<__bf16*>(base) + idx) = o;
  } else {
    typedef float vec __attribute__((ext_vector_type(V)));
    vec o;
#pragma unroll
    for (int e = 0; e < V; ++e) o[e] = v.f[e];
    *reinterpret_cast<vec*>(reinterpret_cast<float*>(base) + idx) = o;
  }
}

struct GnArgs {
  const void* x;
  const void* dy;
  const float* gamma;
  const float* beta;
  const int* lengths;  // [N] or NULL
  void* out;           // y, or dx
  float* stats;        // [N][G][2]: mean, rstd
  float* part;         // workspace
  float eps;
  long N;
  int T, C, G, act, splits, split_len;
};

// sum over the L neighbouring threads of a group (this thread's first one is g0); red: one float a thread
template <bool POW2>
__device__ __forceinline__ float gn_group_sum(float v, int L, int g0, float* red) {
  if (POW2) {
    for (int o = L >> 1; o > 0; o >>= 1) v += __shfl_xor(v, o);
    return v;
  }
  __syncthreads();
  red[threadIdx.x] = v;
  __syncthreads();
  float s = 0.f;
  for (int i = 0; i < L; ++i) s += red[g0 + i];
  return s;
}

// ---- rows (T = 1).  The workgroup's threads hold blockDim / (C / V) rows side by side.
template <bool XB, bool OB, int V, bool POW2>
__global__ void k_gn_rows(GnArgs a) {
  __shared__ float red[1024];
  const int TR = a.C / V, RB = blockDim.x / TR, cg = a.C / a.G, L = cg / V;
  const int slot = threadIdx.x / TR, c = (threadIdx.x % TR) * V, g0 = threadIdx.x - (threadIdx.x % TR) % L;
  const bool on = slot < RB;
  const float inv_n = 1.f / (float)cg;
  GnVec<V> g, bt;
  if (on) {
    g = gn_load<false, V>(a.gamma, c);
    bt = gn_load<false, V>(a.beta, c);
  }
  for (long r0 = (long)blockIdx.x * RB; r0 < a.N; r0 += (long)gridDim.x * RB) {
    const long row = r0 + slot;
    const bool live = on && row < a.N;
    GnVec<V> x;
    float s = 0.f;
#pragma unroll
    for (int e = 0; e < V; ++e) x.f[e] = 0.f;
    if (live) {
      x = gn_load<XB, V>(a.x, row * a.C + c);
#pragma unroll
      for (int e = 0; e < V; ++e) s += x.f[e];
    }
    const float mean = gn_group_sum<POW2>(s, L, g0, red) * inv_n;
    s = 0.f;
#pragma unroll
    for (int e = 0; e < V; ++e) {
      x.f[e] -= mean;
      s += x.f[e] * x.f[e];
    }
    const float rstd = rsqrtf(gn_group_sum<POW2>(s, L, g0, red) * inv_n + a.eps);
    if (live) {
#pragma unroll
      for (int e = 0; e < V; ++e) x.f[e] = gn_act(x.f[e] * rstd * g.f[e] + bt.f[e], a.act);
      gn_store<OB, V>(a.out, row * a.C + c, x);
    }
  }
}

// Backward of the rows: mean and rstd are recomputed; a thread sums dgamma, dbeta of its channels over the rows it visits,
// the workgroup leaves one partial [2][C] (dgamma, dbeta) in part[blockIdx].
template <bool XB, bool GB, int V, bool POW2>
__global__ void k_gn_rows_bwd(GnArgs a) {
  __shared__ float red[1024 * 2];
  const int TR = a.C / V, RB = blockDim.x / TR, cg = a.C / a.G, L = cg / V;
  const int slot = threadIdx.x / TR, c = (threadIdx.x % TR) * V, g0 = threadIdx.x - (threadIdx.x % TR) % L;
  const bool on = slot < RB;
  const float inv_n = 1.f / (float)cg;
  GnVec<V> g, bt, dg, db;
#pragma unroll
  for (int e = 0; e < V; ++e) dg.f[e] = db.f[e] = g.f[e] = bt.f[e] = 0.f;
  if (on) {
    g = gn_load<false, V>(a.gamma, c);
    bt = gn_load<false, V>(a.beta, c);
  }
  for (long r0 = (long)blockIdx.x * RB; r0 < a.N; r0 += (long)gridDim.x * RB) {
    const long row = r0 + slot;
    const bool live = on && row < a.N;
    GnVec<V> x, dy;
    float s = 0.f;
#pragma unroll
    for (int e = 0; e < V; ++e) x.f[e] = dy.f[e] = 0.f;
    if (live) {
      x = gn_load<XB, V>(a.x, row * a.C + c);
      dy = gn_load<GB, V>(a.dy, row * a.C + c);
#pragma unroll
      for (int e = 0; e < V; ++e) s += x.f[e];
    }
    const float mean = gn_group_sum<POW2>(s, L, g0, red) * inv_n;
    s = 0.f;
#pragma unroll
    for (int e = 0; e < V; ++e) {
      x.f[e] -= mean;
      s += x.f[e] * x.f[e];
    }
    const float rstd = rsqrtf(gn_group_sum<POW2>(s, L, g0, red) * inv_n + a.eps);
    float s1 = 0.f, s2 = 0.f;
    if (live) {
#pragma unroll
      for (int e = 0; e < V; ++e) {
        x.f[e] *= rstd;  // xhat
        const float dz = dy.f[e] * gn_slope(x.f[e] * g.f[e] + bt.f[e], a.act);
        db.f[e] += dz;
        dg.f[e] += dz * x.f[e];
        dy.f[e] = dz * g.f[e];
        s1 += dy.f[e];
        s2 += dy.f[e] * x.f[e];
      }
    }
    s1 = gn_group_sum<POW2>(s1, L, g0, red) * inv_n;
    s2 = gn_group_sum<POW2>(s2, L, g0, red) * inv_n;
    if (live) {
#pragma unroll
      for (int e = 0; e < V; ++e) x.f[e] = (dy.f[e] - s1 - x.f[e] * s2) * rstd;
      gn_store<XB, V>(a.out, row * a.C + c, x);
    }
  }
  // the row slots' sums, one channel element of the vectors at a time (red holds two floats a thread)
#pragma unroll
  for (int e = 0; e < V; ++e) {
    __syncthreads();
    red[2 * threadIdx.x] = dg.f[e];
    red[2 * threadIdx.x + 1] = db.f[e];
    __syncthreads();
    if (on && slot == 0) {
      float t0 = 0.f, t1 = 0.f;
      for (int i = 0; i < RB; ++i) {
        t0 += red[2 * (threadIdx.x + i * TR)];
        t1 += red[2 * (threadIdx.x + i * TR) + 1];
      }
      a.part[(long)blockIdx.x * 2 * a.C + c + e] = t0;
      a.part[(long)blockIdx.x * 2 * a.C + a.C + c + e] = t1;
    }
  }
}

// (count, mean, M2) of a set of values, and of two disjoint sets together.  Joined in 64 bits: a handful of values a
// group, and what they lose would shift every value of the group.
struct GnMoment {
  double n, mean, m2;
};
__device__ __forceinline__ GnMoment gn_join(const GnMoment& p, const GnMoment& q) {
  const double n = p.n + q.n;
  if (n == 0.) return p;
  const double d = q.mean - p.mean, w = q.n / n;
  return GnMoment{n, p.mean + d * w, p.m2 + q.m2 + d * d * p.n * w};
}

__device__ __forceinline__ int gn_len(const GnArgs& a, long n) { return a.lengths ? min(max(a.lengths[n], 0), a.T) : a.T; }

// ---- utterances.  Workgroup (split, n): threads of a row own V channels each, the workgroup's rows of threads take the
// split's frames in turn.
template <bool XB, int V>
__global__ void k_gn_stats(GnArgs a) {
  __shared__ GnMoment red[1024];
  const int TR = a.C / V, RB = blockDim.x / TR, L = a.C / a.G / V;
  const int slot = threadIdx.x / TR, c = (threadIdx.x % TR) * V;
  const long n = blockIdx.y;
  const int t0 = blockIdx.x * a.split_len, t1 = min(t0 + a.split_len, gn_len(a, n));
  const long base = n * a.T * a.C + c;
  float cnt = 0.f, s = 0.f, ss = 0.f, pivot = 0.f;
  if (slot < RB) {
    for (int t = t0 + slot; t < t1; t += RB) {
      const GnVec<V> x = gn_load<XB, V>(a.x, base + (long)t * a.C);
      if (cnt == 0.f) pivot = x.f[0];  // the second moment is taken about a value of the data
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float d = x.f[e] - pivot;
        s += d;
        ss += d * d;
      }
      cnt += V;
    }
  }
  const double m = cnt > 0.f ? (double)s / cnt : 0.;
  const double m2 = (double)ss - s * m;
  red[threadIdx.x] = GnMoment{cnt, pivot + m, m2 < 0. ? 0. : m2};
  __syncthreads();
  // a wave joins a group: its lanes take the RB * L partials in turn, then meet in a tree
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  for (int g = wave; g < a.G; g += blockDim.x >> 6) {
    GnMoment t{0., 0., 0.};
    for (int i = lane; i < RB * L; i += 64) t = gn_join(t, red[(i / L) * TR + g * L + i % L]);
    for (int o = 32; o > 0; o >>= 1) {
      const GnMoment u{__shfl_xor(t.n, o), __shfl_xor(t.mean, o), __shfl_xor(t.m2, o)};
      t = (lane & o) ? gn_join(u, t) : gn_join(t, u);
    }
    if (lane == 0) {
      *(reinterpret_cast<GnMoment*>(a.part) + (n * a.splits + blockIdx.x) * a.G + g) = t;
    }
  }
}

template <bool XB, bool OB, int V>
__global__ void k_gn_apply(GnArgs a) {
  __shared__ float2 st[kGnMaxWidth];  // [G]
  const int TR = a.C / V, RB = blockDim.x / TR, cg = a.C / a.G;
  const int slot = threadIdx.x / TR, c = (threadIdx.x % TR) * V;
  const long n = blockIdx.y;
  for (int g = threadIdx.x; g < a.G; g += blockDim.x) {
    GnMoment t{0., 0., 0.};
    for (int s = 0; s < a.splits; ++s) t = gn_join(t, *(reinterpret_cast<const GnMoment*>(a.part) + (n * a.splits + s) * a.G + g));
    const float rstd = (float)(1. / sqrt((t.n > 0. ? t.m2 / t.n : 0.) + (double)a.eps));
    st[g] = make_float2((float)t.mean, rstd);
    if (a.stats && blockIdx.x == 0) *reinterpret_cast<float2*>(a.stats + (n * a.G + g) * 2) = st[g];
  }
  __syncthreads();
  if (slot >= RB) return;
  const GnVec<V> g = gn_load<false, V>(a.gamma, c), bt = gn_load<false, V>(a.beta, c);
  const float2 ms = st[c / cg];
  const int len = gn_len(a, n), t0 = blockIdx.x * a.split_len, t1 = min(t0 + a.split_len, a.T);
  const long base = n * a.T * a.C + c;
  for (int t = t0 + slot; t < t1; t += RB) {
    GnVec<V> y;
    if (t < len) {
      const GnVec<V> x = gn_load<XB, V>(a.x, base + (long)t * a.C);
#pragma unroll
      for (int e = 0; e < V; ++e) y.f[e] = gn_act((x.f[e] - ms.x) * ms.y * g.f[e] + bt.f[e], a.act);
    } else {
#pragma unroll
      for (int e = 0; e < V; ++e) y.f[e] = 0.f;
    }
    gn_store<OB, V>(a.out, base + (long)t * a.C, y);
  }
}

// part[n][split][2][C]: sums over the split's frames of dz xhat and dz
template <bool XB, bool GB, int V>
__global__ void k_gn_bwd_sums(GnArgs a) {
  __shared__ float red[1024 * 2];
  const int TR = a.C / V, RB = blockDim.x / TR, cg = a.C / a.G;
  const int slot = threadIdx.x / TR, c = (threadIdx.x % TR) * V;
  const long n = blockIdx.y;
  const bool on = slot < RB;
  const int t0 = blockIdx.x * a.split_len, t1 = min(t0 + a.split_len, gn_len(a, n));
  const long base = n * a.T * a.C + c;
  GnVec<V> dg, db;
#pragma unroll
  for (int e = 0; e < V; ++e) dg.f[e] = db.f[e] = 0.f;
  if (on) {
    const GnVec<V> g = gn_load<false, V>(a.gamma, c), bt = gn_load<false, V>(a.beta, c);
    const float2 ms = *reinterpret_cast<const float2*>(a.stats + (n * a.G + c / cg) * 2);
    for (int t = t0 + slot; t < t1; t += RB) {
      const GnVec<V> x = gn_load<XB, V>(a.x, base + (long)t * a.C), dy = gn_load<GB, V>(a.dy, base + (long)t * a.C);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float h = (x.f[e] - ms.x) * ms.y;
        const float dz = dy.f[e] * gn_slope(h * g.f[e] + bt.f[e], a.act);
        db.f[e] += dz;
        dg.f[e] += dz * h;
      }
    }
  }
  float* const out = a.part + (n * a.splits + blockIdx.x) * 2 * a.C;
#pragma unroll
  for (int e = 0; e < V; ++e) {
    __syncthreads();
    red[2 * threadIdx.x] = dg.f[e];
    red[2 * threadIdx.x + 1] = db.f[e];
    __syncthreads();
    if (on && slot == 0) {
      float u0 = 0.f, u1 = 0.f;
      for (int i = 0; i < RB; ++i) {
        u0 += red[2 * (threadIdx.x + i * TR)];
        u1 += red[2 * (threadIdx.x + i * TR) + 1];
      }
      out[c + e] = u0;
      out[a.C + c + e] = u1;
    }
  }
}

// dx of one split of one utterance, from the group sums of all its splits
template <bool XB, bool GB, int V>
__global__ void k_gn_bwd_apply(GnArgs a) {
  __shared__ float sums[2 * kGnMaxWidth];
  __shared__ float2 gs[kGnMaxWidth];
  const int TR = a.C / V, RB = blockDim.x / TR, cg = a.C / a.G;
  const int slot = threadIdx.x / TR, c = (threadIdx.x % TR) * V;
  const long n = blockIdx.y;
  const int len = gn_len(a, n);
  for (int i = threadIdx.x; i < 2 * a.C; i += blockDim.x) {
    float t = 0.f;
    for (int s = 0; s < a.splits; ++s) t += a.part[(n * a.splits + s) * 2 * a.C + i];
    sums[i] = t;
  }
  __syncthreads();
  for (int g = threadIdx.x; g < a.G; g += blockDim.x) {
    float s1 = 0.f, s2 = 0.f;
    for (int i = g * cg; i < (g + 1) * cg; ++i) {
      s1 += a.gamma[i] * sums[a.C + i];
      s2 += a.gamma[i] * sums[i];
    }
    const float inv = len > 0 ? 1.f / ((float)len * (float)cg) : 0.f;
    gs[g] = make_float2(s1 * inv, s2 * inv);
  }
  __syncthreads();
  if (slot >= RB) return;
  const GnVec<V> g = gn_load<false, V>(a.gamma, c), bt = gn_load<false, V>(a.beta, c);
  const float2 ms = *reinterpret_cast<const float2*>(a.stats + (n * a.G + c / cg) * 2);
  const float2 m = gs[c / cg];
  const int t0 = blockIdx.x * a.split_len, t1 = min(t0 + a.split_len, a.T);
  const long base = n * a.T * a.C + c;
  for (int t = t0 + slot; t < t1; t += RB) {
    GnVec<V> d;
    if (t < len) {
      const GnVec<V> x = gn_load<XB, V>(a.x, base + (long)t * a.C), dy = gn_load<GB, V>(a.dy, base + (long)t * a.C);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float h = (x.f[e] - ms.x) * ms.y;
        const float dz = dy.f[e] * gn_slope(h * g.f[e] + bt.f[e], a.act);
        d.f[e] = (dz * g.f[e] - m.x - h * m.y) * ms.y;
      }
    } else {
#pragma unroll
      for (int e = 0; e < V; ++e) d.f[e] = 0.f;
    }
    gn_store<XB, V>(a.out, base + (long)t * a.C, d);
  }
}

// out[i] = sum of the partials, i < C: dgamma, else dbeta; one wave a column, a fixed order
__global__ __launch_bounds__(256) void k_gn_params(const float* __restrict__ part, long count, int C,
                                                   float* __restrict__ dgamma, float* __restrict__ dbeta) {
  const int i = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
  if (i >= 2 * C) return;
  float t = 0.f;
  for (long b = lane; b < count; b += 64) t += part[b * 2 * C + i];
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) t += __shfl_xor(t, o);
  if (lane == 0) (i < C ? dgamma[i] : dbeta[i - C]) = t;
}

// ---- host side
struct GnPlan {
  int V, threads, splits, split_len;
  bool pow2;
  long row_blocks;
};
static bool gn_plan(int64_t N, int32_t T, int32_t C, int32_t G, bool wide, GnPlan* p) {
  const int cg = C / G;
  p->V = wide ? 8 : 4;  // 16 bytes of bf16, or of f32
  while (cg % p->V) p->V /= 2;
  const int tr = C / p->V, L = cg / p->V;
  if (tr > 1024) return false;
  // whole waves that hold whole rows of threads, 256 where a row fits
  p->threads = tr <= 256 ? std::max(64, (256 / tr * tr + 63) / 64 * 64) : (tr + 63) / 64 * 64;
  p->pow2 = (L & (L - 1)) == 0 && L <= 64;
  const int rb = p->threads / tr;
  p->row_blocks = (N + rb - 1) / rb;
  // utterances: about 2048 workgroups in all, each with at least eight frames for a thread
  long s = std::max<long>(1, 2048 / std::max<long>(1, N));
  s = std::min<long>(std::min<long>(s, kGnMaxSplits), std::max<long>(1, T / (8L * rb)));
  p->split_len = (int)((T + s - 1) / s);
  p->splits = p->split_len ? (T + p->split_len - 1) / p->split_len : 1;
  return true;
}

static int gn_check(const char* what, int x_dtype, int other, int64_t N, int32_t T, int32_t C, int32_t G, int act) {
  auto known = [](int d) { return d == LMUFFT_F32 || d == LMUFFT_BF16; };
  if (!known(x_dtype) || !known(other)) return set_error("%s: unknown dtype", what);
  if (N < 0 || T < 0 || C <= 0 || G <= 0 || C % G) return set_error("%s: bad shape (N=%lld T=%d C=%d G=%d)", what, (long long)N, T, C, G);
  if (C > kGnMaxWidth) return set_error("%s: %d channels (at most %d)", what, C, kGnMaxWidth);
  if (act < 0 || act > 2) return set_error("%s: unknown activation %d", what, act);
  return 0;
}
static bool gn_aligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

#define GN_BY_V(V_, CALL)                    \
  do {                                       \
    if (V_ == 8) { constexpr int V = 8; CALL; }      \
    else if (V_ == 4) { constexpr int V = 4; CALL; } \
    else if (V_ == 2) { constexpr int V = 2; CALL; } \
    else { constexpr int V = 1; CALL; }              \
  } while (0)
#define GN_BY_2(A_, B_, CALL)                                                             \
  do {                                                                                    \
    if (A_ && B_) { constexpr bool A = true, B = true; CALL; }                            \
    else if (A_) { constexpr bool A = true, B = false; CALL; }                            \
    else if (B_) { constexpr bool A = false, B = true; CALL; }                            \
    else { constexpr bool A = false, B = false; CALL; }                                   \
  } while (0)

}  // namespace lmufft

using namespace lmufft;

extern "C" size_t lmufft_group_norm_workspace_bytes(int64_t N, int32_t T, int32_t C, int32_t G, int backward) {
  if (N <= 0 || T <= 0 || C <= 0 || G <= 0 || C % G || C > kGnMaxWidth) return 0;
  size_t most = 0;
  for (bool wide : {false, true}) {
    GnPlan p;
    if (!gn_plan(N, T, C, G, wide, &p)) return 0;
    // (one frame: rows, or with lengths the utterances' kernels)
    if (T == 1 && backward) most = std::max(most, sizeof(float) * 2 * C * (size_t)std::min<long>(p.row_blocks, kGnRowBwdBlocks));
    if (T > 1 || N <= 65535) most = std::max(most, (size_t)N * p.splits * (backward ? sizeof(float) * 2 * C : sizeof(GnMoment) * G));
  }
  return most;
}

extern "C" int lmufft_group_norm(const void* x, int x_dtype, const float* gamma, const float* beta, const int32_t* lengths,
                                 int64_t N, int32_t T, int32_t C, int32_t G, float eps, int act, void* out, int out_dtype,
                                 float* stats, void* workspace, size_t workspace_bytes, void* stream) {
  const char* what = "group norm";
  if (gn_check(what, x_dtype, out_dtype, N, T, C, G, act)) return 1;
  if (N == 0 || T == 0) return 0;
  if (!x || !gamma || !beta || !out) return set_error("%s: NULL pointer", what);
  const bool rows = T == 1 && !lengths;  // every row a sample of its own
  if (!rows && N > 65535) return set_error("%s: %lld utterances (at most 65535)", what, (long long)N);
  if (!gn_aligned(x) || !gn_aligned(gamma) || !gn_aligned(beta) || !gn_aligned(out) || (reinterpret_cast<uintptr_t>(stats) & 7))
    return set_error("%s: tensors must start on 16-byte boundaries", what);
  const size_t need = lmufft_group_norm_workspace_bytes(N, T, C, G, 0);
  if (need && (!workspace || workspace_bytes < need || !gn_aligned(workspace)))
    return set_error("%s: workspace of %zu bytes on a 16-byte boundary needed, %zu given", what, need, workspace_bytes);
  GnPlan p;
  const bool xb = x_dtype == LMUFFT_BF16, ob = out_dtype == LMUFFT_BF16;
  if (!gn_plan(N, T, C, G, xb && ob, &p)) return set_error("%s: %d channels in %d groups", what, C, G);
  GnArgs a{x, nullptr, gamma, beta, lengths, out, stats, (float*)workspace, eps, (long)N, T, C, G, act, p.splits, p.split_len};
  hipStream_t st = (hipStream_t)stream;
  if (rows) {
    ProfScope ps("k_gn_rows", st);
    const dim3 grid((unsigned)std::min<long>(p.row_blocks, 256 * 16)), block(p.threads);
    if (p.pow2) GN_BY_2(xb, ob, GN_BY_V(p.V, hipLaunchKernelGGL((k_gn_rows<A, B, V, true>), grid, block, 0, st, a)));
    else GN_BY_2(xb, ob, GN_BY_V(p.V, hipLaunchKernelGGL((k_gn_rows<A, B, V, false>), grid, block, 0, st, a)));
  } else {
    const dim3 grid(p.splits, (unsigned)N), block(p.threads);
    {
      ProfScope ps("k_gn_stats", st);
      GN_BY_2(xb, false, GN_BY_V(p.V, hipLaunchKernelGGL((k_gn_stats<A, V>), grid, block, 0, st, a); (void)B));
    }
    ProfScope ps("k_gn_apply", st);
    GN_BY_2(xb, ob, GN_BY_V(p.V, hipLaunchKernelGGL((k_gn_apply<A, B, V>), grid, block, 0, st, a)));
  }
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return set_error("launch of the group norm failed: %s", hipGetErrorString(e));
  return 0;
}

extern "C" int lmufft_group_norm_bwd(const void* x, int x_dtype, const void* dy, int dy_dtype, const float* gamma,
                                     const float* beta, const int32_t* lengths, const float* stats, int64_t N, int32_t T,
                                     int32_t C, int32_t G, float eps, int act, void* dx, float* dgamma, float* dbeta,
                                     void* workspace, size_t workspace_bytes, void* stream) {
  const char* what = "group norm backward";
  if (gn_check(what, x_dtype, dy_dtype, N, T, C, G, act)) return 1;
  if (!dgamma || !dbeta) return set_error("%s: NULL pointer", what);
  hipStream_t st = (hipStream_t)stream;
  if (N == 0 || T == 0) {  // empty sums
    hipLaunchKernelGGL(k_gn_params, dim3((2 * C + 3) / 4), dim3(256), 0, st, (const float*)nullptr, 0L, C, dgamma, dbeta);
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? 0 : set_error("launch of k_gn_params failed: %s", hipGetErrorString(e));
  }
  if (!x || !dy || !gamma || !beta || !dx || (!(T == 1 && !lengths) && !stats)) return set_error("%s: NULL pointer", what);
  const bool rows = T == 1 && !lengths;  // every row a sample of its own
  if (!rows && N > 65535) return set_error("%s: %lld utterances (at most 65535)", what, (long long)N);
  if (!gn_aligned(x) || !gn_aligned(dy) || !gn_aligned(gamma) || !gn_aligned(beta) || !gn_aligned(dx) ||
      (reinterpret_cast<uintptr_t>(stats) & 7))
    return set_error("%s: tensors must start on 16-byte boundaries", what);
  const size_t need = lmufft_group_norm_workspace_bytes(N, T, C, G, 1);
  if (need && (!workspace || workspace_bytes < need || !gn_aligned(workspace)))
    return set_error("%s: workspace of %zu bytes on a 16-byte boundary needed, %zu given", what, need, workspace_bytes);
  GnPlan p;
  const bool xb = x_dtype == LMUFFT_BF16, gb = dy_dtype == LMUFFT_BF16;
  if (!gn_plan(N, T, C, G, xb && gb, &p)) return set_error("%s: %d channels in %d groups", what, C, G);
  GnArgs a{x,  dy, gamma, beta, lengths, dx, const_cast<float*>(stats), (float*)workspace, eps, (long)N, T, C, G, act,
           p.splits, p.split_len};
  long partials;
  if (rows) {
    ProfScope ps("k_gn_rows_bwd", st);
    partials = std::min<long>(p.row_blocks, kGnRowBwdBlocks);
    const dim3 grid((unsigned)partials), block(p.threads);
    if (p.pow2) GN_BY_2(xb, gb, GN_BY_V(p.V, hipLaunchKernelGGL((k_gn_rows_bwd<A, B, V, true>), grid, block, 0, st, a)));
    else GN_BY_2(xb, gb, GN_BY_V(p.V, hipLaunchKernelGGL((k_gn_rows_bwd<A, B, V, false>), grid, block, 0, st, a)));
  } else {
    partials = (long)N * p.splits;
    const dim3 grid(p.splits, (unsigned)N), block(p.threads);
    {
      ProfScope ps("k_gn_bwd_sums", st);
      GN_BY_2(xb, gb, GN_BY_V(p.V, hipLaunchKernelGGL((k_gn_bwd_sums<A, B, V>), grid, block, 0, st, a)));
    }
    ProfScope ps("k_gn_bwd_apply", st);
    GN_BY_2(xb, gb, GN_BY_V(p.V, hipLaunchKernelGGL((k_gn_bwd_apply<A, B, V>), grid, block, 0, st, a)));
  }
  {
    ProfScope ps("k_gn_params", st);
    hipLaunchKernelGGL(k_gn_params, dim3((2 * C + 3) / 4), dim3(256), 0, st, (const float*)a.part, partials, C, dgamma, dbeta);
  }
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return set_error("launch of the group norm backward failed: %s", hipGetErrorString(e));
  return 0;
}
