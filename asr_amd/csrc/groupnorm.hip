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
//   rows (T = 1, no lengths): a row's C / V threads hold it in registers -- one read, one write -- and sum a group over its
//     threads by shuffles when they are a power of two, through LDS otherwise.
//   utterances, columns: where an utterance's frames of a few groups fit a workgroup's registers, it reads them once, keeps
//     them, and writes the result: one launch, one read, one write.
//   utterances, splits: otherwise the frames are split over workgroups.  k_gn_stats leaves the sums of each split and group,
//     k_gn_apply joins them and normalises, reading x again.  The backward does the same
//     with the per-channel sums of dz and dz xhat, from which the group sums and the parameter gradients both follow.
// Second moments are taken about a value of the data, never as a difference of large sums.  The utterances' statistics are
// summed in 64 bits, everything else in 32.  Fixed order, no atomics.  HBM-bound: 25600 rows x 384 in 6 groups bf16 10 us
// (3.9 TB/s); 64 x 400 x 384 in 32 groups bf16 in columns 13.4 us, backward 23.8 + 4.2 us; 32 x 2999 x 384 in 8 groups f32 in
// splits: statistics 28 us, result 45 us, backward 35 + 9 + 53 us, 780 MB in all at 4.6 TB/s, a large copy's rate (lengths from
// a tenth of the frames up: about half of the frames are read, all are written).
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <initializer_list>

#include "lmufft.h"
#include "lmufft_internal.h"

namespace lmufft {

constexpr int kGnMaxWidth = 1024;
constexpr int kGnMaxSplits = 256;
constexpr int kGnFrames = 16, kGnBwdFrames = 10;  // frames a thread of the column kernels can keep (or eight)
constexpr int kGnRowBwdBlocks = 1024;  // workgroups of the rows backward: each leaves one partial of the parameter gradients

enum { kGnNone = 0, kGnRelu = 1, kGnSilu = 2 };

// 1 / (1 + exp(-z)) by the reciprocal instruction (off by at most one step of 2^-23 of the value): an exact division made the
// kernels bound by their arithmetic.
__device__ __forceinline__ float gn_sigmoid(float z) { return __builtin_amdgcn_rcpf(1.f + __expf(-z)); }
__device__ __forceinline__ float gn_act(float z, int act) {
  if (act == kGnRelu) return z > 0.f ? z : (z == z ? 0.f : z);
  if (act == kGnSilu) return z * gn_sigmoid(z);
  return z;
}
// A group's statistics as the element-wise arithmetic takes them, and in 64 bits.
struct GnStat {
  float mean, rstd;
  double dmean, drstd;
};
__device__ __forceinline__ GnStat gn_stat(const double2& s) { return GnStat{(float)s.x, (float)s.y, s.x, s.y}; }
// act'(z) at z = (x - mean) rstd w + b.  The ReLU's slope jumps at zero, and one element on the wrong side is a whole dy in dx
// and in the sums: a z within the 32-bit arithmetic's error of zero is decided in 64 bits (a few in a million).
__device__ __forceinline__ float gn_slope(float z, float x, float w, float b, const GnStat& s, int act) {
  if (act == kGnRelu) {
    if (fabsf(z) <= 5e-7f * (fabsf(b) + (fabsf(x) + fabsf(s.mean)) * fabsf(s.rstd * w)))
      return ((double)x - s.dmean) * s.drstd * (double)w + (double)b > 0. ? 1.f : 0.f;
    return z > 0.f ? 1.f : 0.f;
  }
  if (act == kGnSilu) {
    const float y = gn_sigmoid(z);
    return y * (1.f + z * (1.f - y));
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

// V neighbouring values as they lie in memory
template <bool BF16, int V>
struct GnRaw;
template <int V>
struct GnRaw<true, V> {
  typedef __bf16 vec __attribute__((ext_vector_type(V)));
  vec v;
  __device__ __forceinline__ void load(const void* base, long idx) {
    v = *reinterpret_cast<const vec*>(reinterpret_cast<const __bf16*>(base) + idx);
  }
  __device__ __forceinline__ GnVec<V> get() const {
    GnVec<V> o;
#pragma unroll
    for (int e = 0; e < V; ++e) o.f[e] = (float)v[e];
    return o;
  }
};
template <int V>
struct GnRaw<false, V> {
  typedef float vec __attribute__((ext_vector_type(V)));
  vec v;
  __device__ __forceinline__ void load(const void* base, long idx) {
    v = *reinterpret_cast<const vec*>(reinterpret_cast<const float*>(base) + idx);
  }
  __device__ __forceinline__ GnVec<V> get() const {
    GnVec<V> o;
#pragma unroll
    for (int e = 0; e < V; ++e) o.f[e] = v[e];
    return o;
  }
};

struct GnArgs {
  const void* x;
  const void* dy;
  const float* gamma;
  const float* beta;
  const int* lengths;  // [N] or NULL
  void* out;           // y, or dx
  double2* stats;      // [N][G]: mean, rstd
  float* part;         // workspace
  float eps;
  long N;
  int T, C, G, act, splits, split_len;
};

// sum over the L neighbouring threads of a group (this thread's first one is g0; `groups` in the workgroup).  POW2: by
// shuffles.  Otherwise through red (one value a thread, one a group behind them): few threads a group are summed by each of
// them, many by a team of lanes (125 threads a group, 3000 x 1000 in 8 groups: 50 us if each thread sums them all).
template <bool POW2, class F>
__device__ __forceinline__ F gn_group_sum(F v, int L, int g0, int groups, F* red) {
  if (POW2) {
    for (int o = L >> 1; o > 0; o >>= 1) v += __shfl_xor(v, o);
    return v;
  }
  __syncthreads();
  red[threadIdx.x] = v;
  __syncthreads();
  F s = 0;
  if (L <= 16) {
    for (int i = 0; i < L; ++i) s += red[g0 + i];
    return s;
  }
  const int lanes = L <= 128 ? 16 : 64, lane = threadIdx.x & (lanes - 1);
  for (int t0 = 0; t0 < groups; t0 += blockDim.x / lanes) {  // uniform: the shuffles need every lane
    const int t = t0 + threadIdx.x / lanes;
    s = 0;
    if (t < groups)
      for (int i = lane; i < L; i += lanes) s += red[t * L + i];
    for (int o = lanes >> 1; o > 0; o >>= 1) s += __shfl_xor(s, o);
    if (t < groups && lane == 0) red[1024 + t] = s;
  }
  __syncthreads();
  return red[1024 + min(g0 / L, groups - 1)];
}

// Sums over the workgroup's row slots of the threads' dgamma, dbeta, four elements of the vectors at a time: through red
// (eight floats a thread), a column's RB values joined by a team of lanes, `put(which, column, sum)` by its first (which: 0
// dgamma, 1 dbeta; columns count from the thread row's first).
template <int V, class F>
__device__ __forceinline__ void gn_channel_sums(const GnVec<V>& dg, const GnVec<V>& db, int TR, int RB, int slot, float* red, F put) {
  constexpr int S = V < 4 ? V : 4;
  const int tr = threadIdx.x % TR, columns = TR * 2 * S;
  int lanes = 1;
  while (lanes < 16 && lanes * 4 < RB) lanes <<= 1;
  const int team = threadIdx.x / lanes, lane = threadIdx.x % lanes;
#pragma unroll
  for (int e0 = 0; e0 < V; e0 += S) {
    __syncthreads();
    if (slot >= 0) {
      float* const p = red + (slot * TR + tr) * 2 * S;
#pragma unroll
      for (int e = 0; e < S; ++e) p[e] = dg.f[e0 + e], p[S + e] = db.f[e0 + e];
    }
    __syncthreads();
    for (int k0 = 0; k0 < columns; k0 += blockDim.x / lanes) {  // uniform: the shuffles need every lane
      const int k = k0 + team;
      float t = 0.f;
      if (k < columns)
        for (int i = lane; i < RB; i += lanes) t += red[i * columns + k];
      for (int o = lanes >> 1; o > 0; o >>= 1) t += __shfl_xor(t, o);
      if (k < columns && lane == 0) put((k % (2 * S)) / S, k / (2 * S) * V + e0 + k % S, t);
    }
  }
}

// ---- rows (T = 1).  The workgroup's threads hold blockDim / (C / V) rows side by side.  One row a thread at a time: with
// four in flight the registers cost more waves than the loads gain (25600 x 384 bf16: 13.0 against 10.9 us, backward 28.8
// against 20.4).
template <bool XB, bool OB, int V, bool POW2>
__global__ __launch_bounds__(1024) void k_gn_rows(GnArgs a) {
  __shared__ float red[POW2 ? 1 : 1024 + 1024];
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
    const float mean = gn_group_sum<POW2>(s, L, g0, RB * a.G, red) * inv_n;
    s = 0.f;
#pragma unroll
    for (int e = 0; e < V; ++e) {
      x.f[e] -= mean;
      s += x.f[e] * x.f[e];
    }
    const float rstd = rsqrtf(gn_group_sum<POW2>(s, L, g0, RB * a.G, red) * inv_n + a.eps);
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
__global__ __launch_bounds__(1024) void k_gn_rows_bwd(GnArgs a) {
  __shared__ double dred[POW2 ? 1 : 1024 + 1024];
  float* const red = reinterpret_cast<float*>(dred);
  extern __shared__ float gn_sums[];
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
#pragma unroll
    for (int e = 0; e < V; ++e) x.f[e] = dy.f[e] = 0.f;
    if (live) {
      x = gn_load<XB, V>(a.x, row * a.C + c);
      dy = gn_load<GB, V>(a.dy, row * a.C + c);
    }
    GnStat st;
    if (a.act == kGnRelu) {  // (whose slope asks for them in 64 bits)
      double s = 0.;
#pragma unroll
      for (int e = 0; e < V; ++e) s += x.f[e];
      const double mean = gn_group_sum<POW2>(s, L, g0, RB * a.G, dred) / cg;
      s = 0.;
#pragma unroll
      for (int e = 0; e < V; ++e) s += (x.f[e] - mean) * (x.f[e] - mean);
      st = gn_stat(make_double2(mean, 1. / sqrt(gn_group_sum<POW2>(s, L, g0, RB * a.G, dred) / cg + (double)a.eps)));
    } else {
      float s = 0.f;
#pragma unroll
      for (int e = 0; e < V; ++e) s += x.f[e];
      st.mean = gn_group_sum<POW2>(s, L, g0, RB * a.G, red) * inv_n;
      s = 0.f;
#pragma unroll
      for (int e = 0; e < V; ++e) s += (x.f[e] - st.mean) * (x.f[e] - st.mean);
      st.rstd = rsqrtf(gn_group_sum<POW2>(s, L, g0, RB * a.G, red) * inv_n + a.eps);
    }
    const float rstd = st.rstd;
    float s1 = 0.f, s2 = 0.f;
    if (live) {
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float h = (x.f[e] - st.mean) * rstd;  // xhat
        const float dz = dy.f[e] * gn_slope(h * g.f[e] + bt.f[e], x.f[e], g.f[e], bt.f[e], st, a.act);
        x.f[e] = h;
        db.f[e] += dz;
        dg.f[e] += dz * h;
        dy.f[e] = dz * g.f[e];
        s1 += dy.f[e];
        s2 += dy.f[e] * h;
      }
    }
    s1 = gn_group_sum<POW2>(s1, L, g0, RB * a.G, red) * inv_n;
    s2 = gn_group_sum<POW2>(s2, L, g0, RB * a.G, red) * inv_n;
    if (live) {
#pragma unroll
      for (int e = 0; e < V; ++e) x.f[e] = (dy.f[e] - s1 - x.f[e] * s2) * rstd;
      gn_store<XB, V>(a.out, row * a.C + c, x);
    }
  }
  float* const out = a.part + (long)blockIdx.x * 2 * a.C;
  gn_channel_sums<V>(dg, db, TR, RB, on ? slot : -1, gn_sums, [&](int which, int i, float s) { out[which * a.C + i] = s; });
}

__device__ __forceinline__ int gn_len(const GnArgs& a, long n) { return a.lengths ? min(max(a.lengths[n], 0), a.T) : a.T; }

// Mean and 1 / standard deviation of cnt values from the sum and the sum of squares of their distances from a pivot.
__device__ __forceinline__ double2 gn_mean_rstd(double cnt, float pivot, double s, double ss, float eps) {
  const double m = cnt > 0. ? s / cnt : 0., var = cnt > 0. ? ss / cnt - m * m : 0.;
  return make_double2(pivot + m, 1. / sqrt((var < 0. ? 0. : var) + (double)eps));
}
// A vector's part of the sums about the pivot, in 64 bits: memory is waited for anyway, and the ReLU's border asks for a mean
// that is exact (gn_slope).
template <int V>
__device__ __forceinline__ void gn_add_moments(const GnVec<V>& x, double pivot, double& s, double& ss) {
#pragma unroll
  for (int e = 0; e < V; ++e) {
    const double d = (double)x.f[e] - pivot;
    s += d;
    ss = fma(d, d, ss);
  }
}
// frames first..last-1 of this thread's channels: zeros
template <bool OB, int V>
__device__ __forceinline__ void gn_zero_frames(const GnArgs& a, long base, int first, int last, int slot, int RB) {
  GnVec<V> z;
#pragma unroll
  for (int e = 0; e < V; ++e) z.f[e] = 0.f;
  for (int t = first + slot; t < last; t += RB) gn_store<OB, V>(a.out, base + (long)t * a.C, z);
}
template <int V>
__device__ __forceinline__ GnVec<V> gn_dx(const GnVec<V>& x, const GnVec<V>& dy, const GnVec<V>& g, const GnVec<V>& bt,
                                          const GnStat& st, const float2& m, int act) {
  GnVec<V> d;
#pragma unroll
  for (int e = 0; e < V; ++e) {
    const float h = (x.f[e] - st.mean) * st.rstd;
    const float dz = dy.f[e] * gn_slope(h * g.f[e] + bt.f[e], x.f[e], g.f[e], bt.f[e], st, act);
    d.f[e] = (dz * g.f[e] - m.x - h * m.y) * st.rstd;
  }
  return d;
}

// ---- utterances.  Threads of a row own V channels each, the workgroup's rows of threads take its frames in turn.
//
// Sums of a group: (sum, sum of squares) of x - pivot over the threads of the group, the pivot being the group's first value in
// the utterance, which all take, so partials simply add up.  red: one double2 a thread.  The threads
// tid / lanes, each team of `lanes` (a power of two up to 64) joining one group at a time, call `put(group, sum, squares)`.
template <class F>
__device__ __forceinline__ void gn_join_groups(double s, double ss, int TR, int RB, int L, int G, double2* red, F put) {
  red[threadIdx.x] = make_double2(s, ss);
  __syncthreads();
  const int parts = RB * L;
  int lanes = 1;
  while (lanes < 64 && lanes * 8 < parts) lanes <<= 1;
  const int team = threadIdx.x / lanes, lane = threadIdx.x % lanes;
  for (int g0 = 0; g0 < G; g0 += blockDim.x / lanes) {  // uniform: the shuffles need every lane
    const int g = g0 + team;
    double a = 0., b = 0.;
    if (g < G)
      for (int i = lane; i < parts; i += lanes) {
        const double2 p = red[(i / L) * TR + g * L + i % L];
        a += p.x;
        b += p.y;
      }
    for (int o = lanes >> 1; o > 0; o >>= 1) {
      a += __shfl_xor(a, o);
      b += __shfl_xor(b, o);
    }
    if (g < G && lane == 0) put(g, a, b);
  }
}

// Workgroup (split, n) of the statistics over several workgroups: each split's sums of each group, part[n][split][G], and the
// pivots behind them, [n][G]: k_gn_apply may write over x, whose first frame they come from.
template <bool XB, int V>
__global__ __launch_bounds__(1024) void k_gn_stats(GnArgs a) {
  __shared__ double2 red[1024];
  const int TR = a.C / V, RB = blockDim.x / TR, cg = a.C / a.G, L = cg / V;
  const int slot = threadIdx.x / TR, c = (threadIdx.x % TR) * V;
  const long n = blockIdx.y;
  const int t0 = blockIdx.x * a.split_len, t1 = min(t0 + a.split_len, gn_len(a, n));
  const long base = n * a.T * a.C;
  double s = 0., ss = 0.;
  if (slot < RB && t0 < t1) {
    const float pivot = gn_load<XB, 1>(a.x, base + c / cg * cg).f[0];
#pragma unroll 4
    for (int t = t0 + slot; t < t1; t += RB) {
      const GnVec<V> x = gn_load<XB, V>(a.x, base + (long)t * a.C + c);
      gn_add_moments<V>(x, pivot, s, ss);
    }
  }
  double2* const out = reinterpret_cast<double2*>(a.part) + (n * a.splits + blockIdx.x) * a.G;
  gn_join_groups(s, ss, TR, RB, L, a.G, red, [&](int g, double u, double v) { out[g] = make_double2(u, v); });
  double* const pivots = reinterpret_cast<double*>(reinterpret_cast<double2*>(a.part) + a.N * a.splits * a.G) + n * a.G;
  if (blockIdx.x == 0)
    for (int g = threadIdx.x; g < a.G; g += blockDim.x) pivots[g] = t1 > 0 ? gn_load<XB, 1>(a.x, base + g * cg).f[0] : 0.f;
}

template <bool XB, bool OB, int V>
__global__ __launch_bounds__(1024) void k_gn_apply(GnArgs a) {
  __shared__ double2 st[kGnMaxWidth];  // [G]
  const int TR = a.C / V, RB = blockDim.x / TR, cg = a.C / a.G;
  const int slot = threadIdx.x / TR, c = (threadIdx.x % TR) * V;
  const long n = blockIdx.y;
  const int len = gn_len(a, n);
  const double* const pivots = reinterpret_cast<const double*>(reinterpret_cast<const double2*>(a.part) + a.N * a.splits * a.G) + n * a.G;
  // a group's splits are summed by a team of lanes (one thread a group took 0.8 us a split)
  int lanes = 1;
  while (lanes < 64 && lanes < a.splits) lanes <<= 1;
  for (int g0 = 0; g0 < a.G; g0 += blockDim.x / lanes) {  // uniform: the shuffles need every lane
    const int g = g0 + threadIdx.x / lanes, lane = threadIdx.x % lanes;
    double s = 0., ss = 0.;
    if (g < a.G)
      for (int i = lane; i < a.splits; i += lanes) {
        const double2 p = reinterpret_cast<const double2*>(a.part)[(n * a.splits + i) * a.G + g];
        s += p.x;
        ss += p.y;
      }
    for (int o = lanes >> 1; o > 0; o >>= 1) {
      s += __shfl_xor(s, o);
      ss += __shfl_xor(ss, o);
    }
    if (g < a.G && lane == 0) {
      st[g] = gn_mean_rstd((double)len * cg, (float)pivots[g], s, ss, a.eps);
      if (a.stats && blockIdx.x == 0) a.stats[n * a.G + g] = st[g];
    }
  }
  __syncthreads();
  if (slot >= RB) return;
  const GnVec<V> g = gn_load<false, V>(a.gamma, c), bt = gn_load<false, V>(a.beta, c);
  const GnStat st_ = gn_stat(st[c / cg]);
  const int t0 = blockIdx.x * a.split_len, t1 = min(t0 + a.split_len, a.T);
  const long base = n * a.T * a.C + c;
#pragma unroll 4
  for (int t = t0 + slot; t < min(t1, len); t += RB) {
    GnVec<V> y = gn_load<XB, V>(a.x, base + (long)t * a.C);
#pragma unroll
    for (int e = 0; e < V; ++e) y.f[e] = gn_act((y.f[e] - st_.mean) * st_.rstd * g.f[e] + bt.f[e], a.act);
    gn_store<OB, V>(a.out, base + (long)t * a.C, y);
  }
  gn_zero_frames<OB, V>(a, base, max(t0, len), t1, slot, RB);
}

// part[n][split][2][C]: sums over the split's frames of dz xhat and dz
template <bool XB, bool GB, int V>
__global__ __launch_bounds__(1024) void k_gn_bwd_sums(GnArgs a) {
  extern __shared__ float gn_sums[];
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
    const GnStat st = gn_stat(a.stats[n * a.G + c / cg]);
#pragma unroll 4
    for (int t = t0 + slot; t < t1; t += RB) {
      const GnVec<V> x = gn_load<XB, V>(a.x, base + (long)t * a.C), dy = gn_load<GB, V>(a.dy, base + (long)t * a.C);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float h = (x.f[e] - st.mean) * st.rstd;
        const float dz = dy.f[e] * gn_slope(h * g.f[e] + bt.f[e], x.f[e], g.f[e], bt.f[e], st, a.act);
        db.f[e] += dz;
        dg.f[e] += dz * h;
      }
    }
  }
  float* const out = a.part + (n * a.splits + blockIdx.x) * 2 * a.C;
  gn_channel_sums<V>(dg, db, TR, RB, on ? slot : -1, gn_sums, [&](int which, int i, float s) { out[which * a.C + i] = s; });
}

// A sample's splits joined, by workgroups of a few groups each: its channel sums in the place of its first split's, and its
// groups' means (sum gamma dz) / n, (sum gamma dz xhat) / n behind all partials.
__global__ __launch_bounds__(1024) void k_gn_bwd_join(GnArgs a) {
  __shared__ float sums[2 * kGnMaxWidth];
  const long n = blockIdx.x;
  const int cg = a.C / a.G, len = gn_len(a, n);
  const int g0 = (int)((long)a.G * blockIdx.y / gridDim.y), g1 = (int)((long)a.G * (blockIdx.y + 1) / gridDim.y);
  const int c0 = g0 * cg, width = (g1 - g0) * cg;
  float* const p = a.part + n * a.splits * 2 * a.C;
  for (int i = threadIdx.x; i < 2 * width; i += blockDim.x) {
    const int c = c0 + (i < width ? i : i - width), at = i < width ? c : a.C + c;
    float t = 0.f;
#pragma unroll 16
    for (int s = 0; s < a.splits; ++s) t += p[(long)s * 2 * a.C + at];
    p[at] = t;
    sums[i] = t * a.gamma[c];
  }
  __syncthreads();
  float2* const out = reinterpret_cast<float2*>(a.part + a.N * a.splits * 2 * a.C) + n * a.G;
  const float inv = len > 0 ? 1.f / ((float)len * (float)cg) : 0.f;
  for (int g = threadIdx.x >> 6; g < g1 - g0; g += blockDim.x >> 6) {
    float s1 = 0.f, s2 = 0.f;
    for (int i = g * cg + (threadIdx.x & 63); i < (g + 1) * cg; i += 64) s1 += sums[width + i], s2 += sums[i];
    for (int o = 32; o > 0; o >>= 1) s1 += __shfl_xor(s1, o), s2 += __shfl_xor(s2, o);
    if ((threadIdx.x & 63) == 0) out[g0 + g] = make_float2(s1 * inv, s2 * inv);
  }
}

// dx of one split of one utterance
template <bool XB, bool GB, int V>
__global__ __launch_bounds__(1024) void k_gn_bwd_apply(GnArgs a) {
  const int TR = a.C / V, RB = blockDim.x / TR, cg = a.C / a.G;
  const int slot = threadIdx.x / TR, c = (threadIdx.x % TR) * V;
  const long n = blockIdx.y;
  const int len = gn_len(a, n);
  if (slot >= RB) return;
  const GnVec<V> g = gn_load<false, V>(a.gamma, c), bt = gn_load<false, V>(a.beta, c);
  const GnStat st = gn_stat(a.stats[n * a.G + c / cg]);
  const float2 m = reinterpret_cast<const float2*>(a.part + a.N * a.splits * 2 * a.C)[n * a.G + c / cg];
  const int t0 = blockIdx.x * a.split_len, t1 = min(t0 + a.split_len, a.T);
  const long base = n * a.T * a.C + c;
#pragma unroll 4
  for (int t = t0 + slot; t < min(t1, len); t += RB) {
    const GnVec<V> x = gn_load<XB, V>(a.x, base + (long)t * a.C), dy = gn_load<GB, V>(a.dy, base + (long)t * a.C);
    gn_store<XB, V>(a.out, base + (long)t * a.C, gn_dx<V>(x, dy, g, bt, st, m, a.act));
  }
  gn_zero_frames<XB, V>(a, base, max(t0, len), t1, slot, RB);
}

// ---- utterances whose group columns fit a workgroup's registers: one read, one write, one launch.  A workgroup owns one
// utterance's `width` channels (whole groups); a thread keeps its up to NV frames as they were read, all loads in flight
// together.  (Kept in LDS instead, 93 KB a workgroup left eight waves a CU: 64 x 400 x 384 bf16 backward 32 us.)
// Workgroups of one utterance stay on one XCD (blocks are dispatched to the eight XCDs in turn): neighbouring columns share
// 128-byte lines.
__device__ __forceinline__ bool gn_column_place(const GnArgs& a, long* n, int* block) {
  const int blocks = a.splits;  // (the plan's count of column blocks)
  const long j = blockIdx.x >> 3;
  *n = (j / blocks) * 8 + (blockIdx.x & 7);
  *block = (int)(j % blocks);
  return *n < a.N;
}

template <bool XB, bool OB, int V, int NV>
__global__ __launch_bounds__(1024) void k_gn_column(GnArgs a) {
  __shared__ double2 red[1024];
  __shared__ double2 st[1024];  // [groups of the block]: no more than its threads of a row
  long n;
  int block;
  if (!gn_column_place(a, &n, &block)) return;
  const int width = a.split_len, TR = width / V, RB = blockDim.x / TR, cg = a.C / a.G, L = cg / V, groups = width / cg;
  const int slot = threadIdx.x / TR, col = (threadIdx.x % TR) * V, c = block * width + col;
  const bool on = slot < RB;
  const int len = on ? gn_len(a, n) : 0;
  const long base = n * a.T * a.C + c, first = n * a.T * a.C + (long)block * width;
  GnRaw<XB, V> x[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int t = slot + i * RB;
    if (t < len) x[i].load(a.x, base + (long)t * a.C);
  }
  double s = 0., ss = 0.;
  const float pivot = len > 0 ? gn_load<XB, 1>(a.x, first + col / cg * cg).f[0] : 0.f;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    if (slot + i * RB < len) {
      gn_add_moments<V>(x[i].get(), pivot, s, ss);
    }
  }
  gn_join_groups(s, ss, TR, RB, L, groups, red, [&](int g, double u, double v) {
    const int frames = gn_len(a, n);
    const float p = frames > 0 ? gn_load<XB, 1>(a.x, first + g * cg).f[0] : 0.f;
    st[g] = gn_mean_rstd((double)frames * cg, p, u, v, a.eps);
    if (a.stats) a.stats[n * a.G + block * groups + g] = st[g];
  });
  __syncthreads();
  if (!on) return;
  const GnVec<V> g = gn_load<false, V>(a.gamma, c), bt = gn_load<false, V>(a.beta, c);
  const GnStat st_ = gn_stat(st[col / cg]);
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int t = slot + i * RB;
    if (t < len) {
      GnVec<V> y = x[i].get();
#pragma unroll
      for (int e = 0; e < V; ++e) y.f[e] = gn_act((y.f[e] - st_.mean) * st_.rstd * g.f[e] + bt.f[e], a.act);
      gn_store<OB, V>(a.out, base + (long)t * a.C, y);
    }
  }
  gn_zero_frames<OB, V>(a, base, len, a.T, slot, RB);
}

// The same for the backward; part[n][2][C] receives the utterance's sums of dz xhat and dz.  dz is kept in place of dy.
template <bool XB, bool GB, int V, int NV>
__global__ __launch_bounds__(1024) void k_gn_column_bwd(GnArgs a) {
  extern __shared__ float gn_sums[];
  __shared__ float sums[2 * kGnMaxWidth];
  __shared__ float2 gs[1024];
  long n;
  int block;
  if (!gn_column_place(a, &n, &block)) return;
  const int width = a.split_len, TR = width / V, RB = blockDim.x / TR, cg = a.C / a.G, groups = width / cg;
  const int slot = threadIdx.x / TR, col = (threadIdx.x % TR) * V, c = block * width + col;
  const bool on = slot < RB;
  const int frames = gn_len(a, n), len = on ? frames : 0;
  const long base = n * a.T * a.C + c;
  GnRaw<XB, V> x[NV];
  GnVec<V> dz[NV];
  {
    GnRaw<GB, V> dy[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int t = slot + i * RB;
      if (t < len) {
        x[i].load(a.x, base + (long)t * a.C);
        dy[i].load(a.dy, base + (long)t * a.C);
      }
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) dz[i] = dy[i].get();
  }
  GnVec<V> dg, db, g;
#pragma unroll
  for (int e = 0; e < V; ++e) dg.f[e] = db.f[e] = 0.f;
  GnStat st{0.f, 0.f, 0., 0.};
  if (on) {
    g = gn_load<false, V>(a.gamma, c);
    const GnVec<V> bt = gn_load<false, V>(a.beta, c);
    st = gn_stat(a.stats[n * a.G + c / cg]);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if (slot + i * RB < len) {
        const GnVec<V> xv = x[i].get();
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const float h = (xv.f[e] - st.mean) * st.rstd;
          dz[i].f[e] *= gn_slope(h * g.f[e] + bt.f[e], xv.f[e], g.f[e], bt.f[e], st, a.act);
          db.f[e] += dz[i].f[e];
          dg.f[e] += dz[i].f[e] * h;
        }
      }
    }
  }
  float* const out = a.part + n * 2 * a.C + block * width;
  gn_channel_sums<V>(dg, db, TR, RB, on ? slot : -1, gn_sums, [&](int which, int i, float s) {
    out[which * a.C + i] = s;
    sums[which * width + i] = s * a.gamma[block * width + i];
  });
  __syncthreads();
  const float inv = frames > 0 ? 1.f / ((float)frames * (float)cg) : 0.f;
  for (int k = threadIdx.x; k < groups; k += blockDim.x) {
    float s1 = 0.f, s2 = 0.f;
    for (int i = k * cg; i < (k + 1) * cg; ++i) s1 += sums[width + i], s2 += sums[i];
    gs[k] = make_float2(s1 * inv, s2 * inv);
  }
  __syncthreads();
  if (!on) return;
  const float2 m = gs[col / cg];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int t = slot + i * RB;
    if (t < len) {
      GnVec<V> d = x[i].get();
#pragma unroll
      for (int e = 0; e < V; ++e) d.f[e] = (dz[i].f[e] * g.f[e] - m.x - (d.f[e] - st.mean) * st.rstd * m.y) * st.rstd;
      gn_store<XB, V>(a.out, base + (long)t * a.C, d);
    }
  }
  gn_zero_frames<XB, V>(a, base, len, a.T, slot, RB);
}

// out[i] = sum of the partials, i < C: dgamma, else dbeta.  A workgroup takes 64 columns, its sixteen waves the partials in
// turn; a fixed order.
__global__ __launch_bounds__(1024) void k_gn_params(const float* __restrict__ part, long count, long stride, int C,
                                                    float* __restrict__ dgamma, float* __restrict__ dbeta) {
  __shared__ float red[1024];
  const int i = blockIdx.x * 64 + (threadIdx.x & 63), wave = threadIdx.x >> 6;
  float t = 0.f;
  if (i < 2 * C) {
#pragma unroll 8
    for (long b = wave; b < count; b += 16) t += part[b * stride + i];
  }
  red[threadIdx.x] = t;
  __syncthreads();
  if (wave == 0 && i < 2 * C) {
#pragma unroll
    for (int w = 1; w < 16; ++w) t += red[w * 64 + threadIdx.x];
    (i < C ? dgamma[i] : dbeta[i - C]) = t;
  }
}

// ---- host side
enum { kGnRows, kGnColumn, kGnSplit };
struct GnPlan {
  int kind, V, threads, splits, split_len;  // kGnColumn: the number of column blocks and their width
  bool pow2;
  long blocks;       // rows: workgroups
  int frames;        // kGnColumn: frames a thread keeps
};

// The smallest workgroup whose threads keep the T frames of `width` channels, eight frames each where that is enough, at most
// what the kernels have room for, or what 64 registers hold (`words`: half registers of a kept value: x as it lies in memory,
// and dz).  False if none does.
static bool gn_column_fits(int T, int width, int V, int words, bool backward, GnPlan* p) {
  const int tc = width / V, most = std::min(backward ? kGnBwdFrames : kGnFrames, 128 / (V * words));
  for (int least : {8, 16})
    for (int threads : {256, 512, 1024}) {
      if (tc > threads) continue;
      const int rb = threads / tc, frames = (T + rb - 1) / rb;
      if (frames > std::min(least, most)) continue;
      p->threads = std::min(threads, (tc * std::min(rb, T) + 63) / 64 * 64);
      p->frames = frames;
      return true;
    }
  return false;
}
static bool gn_plan(int64_t N, int32_t T, int32_t C, int32_t G, bool wide, bool rows, bool backward, int x_bytes, GnPlan* p) {
  const int cg = C / G;
  p->V = wide ? 8 : 4;  // 16 bytes of bf16, or of f32
  while (cg % p->V) p->V /= 2;
  const int L = cg / p->V;
  const int tr = C / p->V;
  if (tr > 1024) return false;
  p->pow2 = (L & (L - 1)) == 0 && L <= 64;
  // whole waves that hold whole rows of threads, 256 where a row fits
  p->threads = tr <= 256 ? std::max(64, (256 / tr * tr + 63) / 64 * 64) : (tr + 63) / 64 * 64;
  const int rb = p->threads / tr;
  if (rows) {
    p->kind = kGnRows;
    p->blocks = std::min<long>((N + rb - 1) / rb, backward ? kGnRowBwdBlocks : 4096);
    return true;
  }
  // Column blocks: whole groups, 64 bytes of a frame at least where the groups allow it, up to 128 while the chip stays
  // full.  Taken when there are workgroups for most CUs, or when the launches are all that counts.
  const int words = x_bytes / 2 + (backward ? 2 : 0);
  const int least = std::max(1, (64 / x_bytes + cg - 1) / cg);
  GnPlan q = *p;
  q.V = std::min(4, p->V);  // (eight values a vector would not leave the registers room)
  int best = 0;
  for (int m = 1; m <= G; ++m) {
    if (G % m) continue;
    const int w = m * cg;
    if (!gn_column_fits(T, w, q.V, words, backward, &q)) break;
    if (m > least && N * (G / m) < 512) break;
    best = m;
    if (m >= least && w * x_bytes >= 128) break;
  }
  // (HIP counts a launch's threads in 32 bits)
  if (best && (N + 8) * (G / best) < (1L << 22) && (N * (G / best) >= 192 || (size_t)T * best * cg <= 16 * 1024)) {
    p->V = q.V;
    gn_column_fits(T, best * cg, p->V, words, backward, p);
    p->kind = kGnColumn;
    p->splits = G / best;
    p->split_len = best * cg;
    return true;
  }
  p->kind = kGnSplit;
  // about 4096 workgroups in all, each with at least eight frames for a thread (32 x 2999 x 384 f32, lengths from a tenth up:
  // 2048 184 us of kernels forward and backward, 4096 177, 8192 178)
  long s = std::max<long>(1, 4096 / std::max<long>(1, N));
  s = std::min<long>(std::min<long>(s, kGnMaxSplits), std::max<long>(1, T / (8L * rb)));
  p->split_len = (int)((T + s - 1) / s);
  p->splits = p->split_len ? (T + p->split_len - 1) / p->split_len : 1;
  return true;
}
static size_t gn_workspace(const GnPlan& p, int64_t N, int32_t C, int32_t G, bool backward) {
  if (p.kind == kGnRows) return backward ? sizeof(float) * 2 * C * (size_t)p.blocks : 0;
  if (p.kind == kGnColumn) return backward ? sizeof(float) * 2 * C * (size_t)N : 0;
  return backward ? sizeof(float) * 2 * ((size_t)N * p.splits * C + (size_t)N * G) : (sizeof(double2) * p.splits + sizeof(double)) * (size_t)N * G;
}
static dim3 gn_column_grid(const GnPlan& p, int64_t N) { return dim3((unsigned)((N + 7) / 8 * 8 * p.splits)); }

static int gn_check(const char* what, int x_dtype, int other, int64_t N, int32_t T, int32_t C, int32_t G, int act) {
  auto known = [](int d) { return d == LMUFFT_F32 || d == LMUFFT_BF16; };
  if (!known(x_dtype) || !known(other)) return set_error("%s: unknown dtype", what);
  if (N < 0 || T < 0 || C <= 0 || G <= 0 || C % G) return set_error("%s: bad shape (N=%lld T=%d C=%d G=%d)", what, (long long)N, T, C, G);
  if (C > kGnMaxWidth) return set_error("%s: %d channels (at most %d)", what, C, kGnMaxWidth);
  if (T > (1 << 30)) return set_error("%s: %d frames (at most 2^30)", what, T);  // (frames are counted in 32 bits, strides on top)
  if (act < 0 || act > 2) return set_error("%s: unknown activation %d", what, act);
  return 0;
}
static bool gn_aligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
// A result over an input is fine where every thread overwrites exactly what it has read: the same place and the same dtype.
static int gn_check_alias(const char* what, const char* out_name, const void* out, int out_dtype, const char* in_name,
                          const void* in, int in_dtype, int64_t rows, int32_t C) {
  auto bytes = [&](int dtype) { return (unsigned __int128)rows * (unsigned)C * (dtype == LMUFFT_F32 ? 4 : 2); };
  const uintptr_t o = reinterpret_cast<uintptr_t>(out), i = reinterpret_cast<uintptr_t>(in);
  const bool apart = o + bytes(out_dtype) <= i || i + bytes(in_dtype) <= o;
  if (apart || (o == i && out_dtype == in_dtype)) return 0;
  return set_error("%s: %s may alias %s only at its start and with the same dtype", what, out_name, in_name);
}

#define GN_BY_V4(V_, CALL)                           \
  do {                                               \
    if (V_ == 4) { constexpr int V = 4; CALL; }      \
    else if (V_ == 2) { constexpr int V = 2; CALL; } \
    else { constexpr int V = 1; CALL; }              \
  } while (0)
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
  size_t most = 0;  // over the dtypes, and for one frame over rows and utterances
  for (bool wide : {false, true})
    for (int bytes : {2, 4})
      for (bool rows : {false, true}) {
        GnPlan p;
        if ((rows && T != 1) || (!rows && N > 65535)) continue;
        if (!gn_plan(N, T, C, G, wide, rows, backward, bytes, &p)) return 0;
        most = std::max(most, gn_workspace(p, N, C, G, backward));
      }
  return most;
}

extern "C" int lmufft_group_norm(const void* x, int x_dtype, const float* gamma, const float* beta, const int32_t* lengths,
                                 int64_t N, int32_t T, int32_t C, int32_t G, float eps, int act, void* out, int out_dtype,
                                 double* stats, void* workspace, size_t workspace_bytes, void* stream) {
  const char* what = "group norm";
  if (gn_check(what, x_dtype, out_dtype, N, T, C, G, act)) return 1;
  if (N == 0 || T == 0) return 0;
  if (!x || !gamma || !beta || !out) return set_error("%s: NULL pointer", what);
  const bool rows = T == 1 && !lengths;  // every row a sample of its own
  if (!rows && N > 65535) return set_error("%s: %lld utterances (at most 65535)", what, (long long)N);
  if (!gn_aligned(x) || !gn_aligned(gamma) || !gn_aligned(beta) || !gn_aligned(out) || !gn_aligned(stats))
    return set_error("%s: tensors must start on 16-byte boundaries", what);
  if (gn_check_alias(what, "out", out, out_dtype, "x", x, x_dtype, N * T, C)) return 1;
  GnPlan p;
  const bool xb = x_dtype == LMUFFT_BF16, ob = out_dtype == LMUFFT_BF16;
  if (!gn_plan(N, T, C, G, xb && ob, rows, false, xb ? 2 : 4, &p)) return set_error("%s: %d channels in %d groups", what, C, G);
  const size_t need = gn_workspace(p, N, C, G, false);
  if (need && (!workspace || workspace_bytes < need || !gn_aligned(workspace)))
    return set_error("%s: workspace of %zu bytes on a 16-byte boundary needed, %zu given", what, need, workspace_bytes);
  GnArgs a{x, nullptr, gamma, beta, lengths, out, (double2*)stats, (float*)workspace, eps, (long)N, T, C, G, act, p.splits, p.split_len};
  hipStream_t st = (hipStream_t)stream;
  const dim3 block(p.threads);
  if (p.kind == kGnRows) {
    ProfScope ps("k_gn_rows", st);
    const dim3 grid((unsigned)p.blocks);
    if (p.pow2) GN_BY_2(xb, ob, GN_BY_V(p.V, hipLaunchKernelGGL((k_gn_rows<A, B, V, true>), grid, block, 0, st, a)));
    else GN_BY_2(xb, ob, GN_BY_V(p.V, hipLaunchKernelGGL((k_gn_rows<A, B, V, false>), grid, block, 0, st, a)));
  } else if (p.kind == kGnColumn) {
    ProfScope ps("k_gn_column", st);
    if (p.frames <= 8) GN_BY_2(xb, ob, GN_BY_V4(p.V, hipLaunchKernelGGL((k_gn_column<A, B, V, 8>), gn_column_grid(p, N), block, 0, st, a)));
    else GN_BY_2(xb, ob, GN_BY_V4(p.V, hipLaunchKernelGGL((k_gn_column<A, B, V, kGnFrames>), gn_column_grid(p, N), block, 0, st, a)));
  } else {
    const dim3 grid(p.splits, (unsigned)N);
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
                                     const float* beta, const int32_t* lengths, const double* stats, int64_t N, int32_t T,
                                     int32_t C, int32_t G, float eps, int act, void* dx, float* dgamma, float* dbeta,
                                     void* workspace, size_t workspace_bytes, void* stream) {
  const char* what = "group norm backward";
  if (gn_check(what, x_dtype, dy_dtype, N, T, C, G, act)) return 1;
  if (!dgamma || !dbeta) return set_error("%s: NULL pointer", what);
  hipStream_t st = (hipStream_t)stream;
  if (N == 0 || T == 0) {  // empty sums
    hipLaunchKernelGGL(k_gn_params, dim3((2 * C + 63) / 64), dim3(1024), 0, st, (const float*)nullptr, 0L, 0L, C, dgamma, dbeta);
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? 0 : set_error("launch of k_gn_params failed: %s", hipGetErrorString(e));
  }
  const bool rows = T == 1 && !lengths;  // every row a sample of its own
  if (!x || !dy || !gamma || !beta || !dx || (!rows && !stats)) return set_error("%s: NULL pointer", what);
  if (!rows && N > 65535) return set_error("%s: %lld utterances (at most 65535)", what, (long long)N);
  if (!gn_aligned(x) || !gn_aligned(dy) || !gn_aligned(gamma) || !gn_aligned(beta) || !gn_aligned(dx) ||
      !gn_aligned(stats))
    return set_error("%s: tensors must start on 16-byte boundaries", what);
  if (gn_check_alias(what, "dx", dx, x_dtype, "x", x, x_dtype, N * T, C) ||
      gn_check_alias(what, "dx", dx, x_dtype, "dy", dy, dy_dtype, N * T, C))
    return 1;
  GnPlan p;
  const bool xb = x_dtype == LMUFFT_BF16, gb = dy_dtype == LMUFFT_BF16;
  if (!gn_plan(N, T, C, G, xb && gb, rows, true, xb ? 2 : 4, &p))
    return set_error("%s: %d channels in %d groups", what, C, G);
  const size_t need = gn_workspace(p, N, C, G, true);
  if (need && (!workspace || workspace_bytes < need || !gn_aligned(workspace)))
    return set_error("%s: workspace of %zu bytes on a 16-byte boundary needed, %zu given", what, need, workspace_bytes);
  GnArgs a{x,  dy, gamma, beta, lengths, dx, (double2*)const_cast<double*>(stats), (float*)workspace, eps, (long)N, T, C, G, act,
           p.splits, p.split_len};
  const dim3 block(p.threads);
  long partials = N, stride = 2 * C;
  const size_t lds = sizeof(float) * p.threads * 2 * std::min(4, p.V);  // gn_channel_sums: at most 32 KB
  if (p.kind == kGnRows) {
    ProfScope ps("k_gn_rows_bwd", st);
    partials = p.blocks;
    const dim3 grid((unsigned)partials);
    if (p.pow2) GN_BY_2(xb, gb, GN_BY_V(p.V, hipLaunchKernelGGL((k_gn_rows_bwd<A, B, V, true>), grid, block, lds, st, a)));
    else GN_BY_2(xb, gb, GN_BY_V(p.V, hipLaunchKernelGGL((k_gn_rows_bwd<A, B, V, false>), grid, block, lds, st, a)));
  } else if (p.kind == kGnColumn) {
    ProfScope ps("k_gn_column_bwd", st);
    if (p.frames <= 8) GN_BY_2(xb, gb, GN_BY_V4(p.V, hipLaunchKernelGGL((k_gn_column_bwd<A, B, V, 8>), gn_column_grid(p, N), block, lds, st, a)));
    else GN_BY_2(xb, gb, GN_BY_V4(p.V, hipLaunchKernelGGL((k_gn_column_bwd<A, B, V, kGnBwdFrames>), gn_column_grid(p, N), block, lds, st, a)));
  } else {
    stride *= p.splits;
    const dim3 grid(p.splits, (unsigned)N);
    {
      ProfScope ps("k_gn_bwd_sums", st);
      GN_BY_2(xb, gb, GN_BY_V(p.V, hipLaunchKernelGGL((k_gn_bwd_sums<A, B, V>), grid, block, lds, st, a)));
    }
    {
      ProfScope ps("k_gn_bwd_join", st);
      hipLaunchKernelGGL(k_gn_bwd_join, dim3((unsigned)N, std::min(G, 8)), dim3(256), 0, st, a);
    }
    ProfScope ps("k_gn_bwd_apply", st);
    GN_BY_2(xb, gb, GN_BY_V(p.V, hipLaunchKernelGGL((k_gn_bwd_apply<A, B, V>), grid, block, 0, st, a)));
  }
  {
    ProfScope ps("k_gn_params", st);
    hipLaunchKernelGGL(k_gn_params, dim3((2 * C + 63) / 64), dim3(1024), 0, st, (const float*)a.part, partials, stride, C, dgamma, dbeta);
  }
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return set_error("launch of the group norm backward failed: %s", hipGetErrorString(e));
  return 0;
}
