// C entry points of the causal decay attention (kernels: decay_core.h), and its single-frame form.
//
// k_decay_step: S <- lambda S + k v^T, o = scale S^T q for one frame of each stream, the state updated in place.
//   One workgroup per (stream, head): DV / 4 threads side by side own four columns each, the workgroup's rows of threads
//   split the DK rows of the state; the partial sums over their rows meet in LDS.  Every element of the state is read and
//   written once, 16 bytes a lane: bound by the states' traffic (8 DK DV bytes a stream and head) when there are many
//   streams, by the launch when there are few.  Six heads of 64 x 64: 1000 streams (90 % of them live) f32 29.5 us, 6.0 TB/s, the
//   states lying partly in the last-level cache; 4 streams 3.3 us.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "decay_core.h"

namespace lmufft {

constexpr int kDecayStepThreads = 256;

template <class T, int DV>
__global__ __launch_bounds__(kDecayStepThreads) void k_decay_step(const T* __restrict__ q, const T* __restrict__ k,
                                                                  const T* __restrict__ v, long ldq, long ldk, long ldv,
                                                                  const float* __restrict__ log_decay,
                                                                  const int* __restrict__ active, int H, int DK,
                                                                  float scale, T* __restrict__ out, long ldo,
                                                                  float* __restrict__ state) {
  constexpr int CV = DV / 4, RG = kDecayStepThreads / CV;  // threads across the columns; rows of threads
  __shared__ __attribute__((aligned(16))) float part[RG * DV];
  const int tid = threadIdx.x, c = (tid % CV) * 4, rg = tid / CV;
  const int b = blockIdx.x / H, h = blockIdx.x - b * H;
  T* const op = out + (long)b * ldo + (long)h * DV;
  if (active && active[b] <= 0) {  // a silent stream: zeros, and its state stays as it is
    if (tid < DV) op[tid] = (T)0.f;
    return;
  }
  const T* const qp = q + (long)b * ldq + (long)h * DK;
  const T* const kp = k + (long)b * ldk + (long)h * DK;
  const T* const vp = v + (long)b * ldv + (long)h * DV + c;
  const float lam = dec_pow(dec_log2(log_decay[h]), 1);
  dec_f4 vv;
#pragma unroll
  for (int e = 0; e < 4; ++e) vv[e] = (float)vp[e];
  dec_f4 o = dec_f4(0.f);
  float* const sp = state + (long)blockIdx.x * DK * DV + c;
#pragma unroll 4
  for (int r = rg; r < DK; r += RG) {
    dec_f4* const e = reinterpret_cast<dec_f4*>(sp + (long)r * DV);
    const dec_f4 s = lam * *e + (float)kp[r] * vv;
    *e = s;
    o += (float)qp[r] * s;
  }
  *reinterpret_cast<dec_f4*>(&part[rg * DV + c]) = o;
  __syncthreads();
  if (tid < DV) {
    float t = 0.f;
#pragma unroll
    for (int i = 0; i < RG; ++i) t += part[i * DV + tid];
    op[tid] = (T)(t * scale);
  }
}

// k_decay_join: a workgroup takes 64 places (16 bytes each) of one head's states, its sixteen waves up to eight consecutive
// segments each, read at once.  A wave first sums its own, the waves' sums meet in LDS.  (Summed by every segment's workgroup for
// itself instead, 62 segments of one head cost 24 us of reads.)  74 segments of six heads 64 x 64: 5.4 us, 14 MB there and back.
constexpr int kJoinEach = kDecayMaxSegments / 16;
__global__ __launch_bounds__(1024) void k_decay_join(float* ws, long role_stride, const float* __restrict__ log_decay,
                                                     const int* __restrict__ lengths, int T, int H, int segments, int seg_len,
                                                     int places) {
  __shared__ dec_f4 sum[16][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, bh = blockIdx.x, b = bh / H;
  const int len = lengths ? min(max(lengths[b], 0), T) : T;
  const int have = min(segments - 1, len > 0 ? (len - 1) / seg_len : 0);  // segments that another one follows left a state
  const int per = (segments - 1 + 15) / 16, from = wave * per, n = min(per, have - from);
  dec_f4* const e = reinterpret_cast<dec_f4*>(ws + blockIdx.z * role_stride) + ((long)bh * segments + from) * places + blockIdx.y * 64 + lane;
  const float a2 = dec_log2(log_decay[bh - b * H]), lam = dec_pow(a2, seg_len);
  dec_f4 x[kJoinEach], acc = dec_f4(0.f);
  if (n > 0) {
#pragma unroll
    for (int i = 0; i < kJoinEach; ++i) x[i] = e[(long)min(i, n - 1) * places];
#pragma unroll
    for (int i = 0; i < kJoinEach; ++i)
      if (i < n) acc = lam * acc + x[i];
  }
  sum[wave][lane] = acc;
  __syncthreads();
  if (n <= 0) return;
  // (the waves before this one are full)
  const float lam_per = dec_pow(a2, per * seg_len);
  acc = dec_f4(0.f);
#pragma unroll 4
  for (int w = 0; w < wave; ++w) acc = lam_per * acc + sum[w][lane];
#pragma unroll
  for (int i = 0; i < kJoinEach; ++i)
    if (i < n) {
      acc = lam * acc + x[i];
      e[(long)i * places] = acc;
    }
}

int decay_launch_join(const DecayArgs& a, int roles, int state_elements, hipStream_t st) {
  ProfScope ps("k_decay_join", st);
  const long stride = roles > 1 ? a.role[1].ws - a.role[0].ws : 0;
  hipLaunchKernelGGL(k_decay_join, dim3(a.B * a.H, state_elements / 256, roles), dim3(1024), 0, st, a.role[0].ws, stride,
                     a.log_decay, a.lengths, a.T, a.H, a.segments, a.seg_len, state_elements / 4);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? 0 : set_error("launch of k_decay_join failed: %s", hipGetErrorString(e));
}

// Workgroups from which on they take the utterances from the longest to the shortest (up to 64 of them, those a wave can rank):
// a CU's second workgroups are then the short ones, and none starts late.  Kernel times, lengths from a tenth up, in the batch's
// order and in this one: 64 x 400 x 6 heads bf16 22.0 and 19.0 us, backward 42 and 38; backward of 16 x 400 f32 51 and 44; 32 x
// 3000 bf16 66 and 57, backward 144 and 122.  With a workgroup a CU or fewer the order changes nothing, and the ranking costs
// 0.3 us.  Batches above 64 keep their own order.
constexpr long kDecayOrderFrom = 256;

static bool decay_width(int d) { return d == 32 || d == 64 || d == 128; }

static int decay_check(const char* what, int dtype, int32_t B, int32_t T, int32_t H, int32_t dk, int32_t dv) {
  if (dtype != LMUFFT_F32 && dtype != LMUFFT_BF16) return set_error("%s: unknown dtype %d", what, dtype);
  if (B < 0 || T < 0 || H <= 0) return set_error("%s: bad shape (B=%d T=%d H=%d)", what, B, T, H);
  if (!decay_width(dk) || !decay_width(dv)) return set_error("%s: head widths %d, %d (supported: 32, 64, 128)", what, dk, dv);
  // (HIP counts a launch's threads in 32 bits, 512 for each head and role; and the kernels an utterance's 16-byte pieces)
  if ((long)B * H > (1 << 21) || T > (1 << 25)) return set_error("%s: too large (B=%d T=%d H=%d)", what, B, T, H);
  return 0;
}

// Segments an utterance's frames are split into when there are few heads in all (counted over utterances and roles).  A split
// costs a second read of k and v and a launch, from kDecayJoinFrom segments on another one, and pays while CUs are idle or the
// longest utterance's chunks are what is waited for.  Heads of up to 64 columns leave a CU room for two workgroups, and long
// utterances are split into about that many, 480; wider heads have a CU each, and short utterances are in so few chunks that the
// launches weigh: 320.  Measured, whole call in us (all utterances full / lengths from a tenth up), by segments:
//   480 or fewer  f32 96 heads of 3000 frames 5: 123 / 120, 3: 162 / 119; bf16 24 heads of 3000 16: 27 / 27, 12: 29 / 26; one
//                 utterance of 24000 bf16 of 24 heads 20: 103, 13: 133, of 17 27: 74, 18: 97; 192 heads of 3000 bf16 2: 92 / 75,
//                 whole: 85 / 84, 240 heads 2: 102 / 90, whole: 94 / 85; backward of 144 (3 x 48) heads of 3000 bf16 3: 68 / 63,
//                 2: 88 / 69, of 288 whole: 122 / 86, 2: 128 / 89
//   480 or more   one utterance of 24000 bf16 of 6 heads 75: 36, 125: 40, of 16 29: 69, 47: 70; of 8000 of 12 32: 30, 42: 28
//   32 chunks     f32 96 heads of 1000 3: 62 / 47, 5: 58 / 56; 72 (3 x 24) heads' backward 4: 50 / 38, 6: 50 / 50; above (47 and
//                 94 chunks) see the first lines
//   128 columns   bf16 24 heads of 3000 12: 74 / 49, 16: 66 / 63, 10: 54 / 52; 96 heads 3: 184 / 113, 5: 157 / 148, 2: 160 / 159
static int decay_segments(int dtype, int32_t B, int32_t T, int32_t H, int32_t dk, int32_t dv, int roles, int* seg_len) {
  const int chunk = dtype == LMUFFT_BF16 ? decay_chunk_bf16(dk, dv) : decay_chunk_f32(dk, dv);
  const long heads = std::max<long>(1, (long)B * H * roles), chunks = std::max<long>(1, (T + (long)chunk - 1) / chunk);
  const long workgroups = chunks > 32 && std::max(dk, dv) <= 64 ? 480 : 320;
  long n = std::min<long>(workgroups / heads, chunks / 2);  // (no segment of a single chunk)
  n = std::max<long>(std::min<long>(n, kDecayMaxSegments), 1);
  const long per = (chunks + n - 1) / n;
  *seg_len = (int)(per * chunk);
  return (int)((chunks + per - 1) / per);
}

// Rows of [B][T][H * width] tensors have to start on 16-byte boundaries (the kernels load 16 bytes a lane).
static int decay_tensor(const char* what, const char* name, const void* p, int dtype, int64_t ld, int64_t bs, int32_t B,
                        int32_t T, long width, bool written, DecayTensor* out) {
  if (!p) return set_error("%s: `%s` is NULL", what, name);
  const int64_t unit = dtype == LMUFFT_F32 ? 4 : 8;
  if ((reinterpret_cast<uintptr_t>(p) & 15) || ld % unit || bs % unit)
    return set_error("%s: rows of `%s` must start on 16-byte boundaries", what, name);
  if (ld < 0 || bs < 0) return set_error("%s: `%s` has a negative stride", what, name);
  if (ld > (1 << 22)) return set_error("%s: rows of `%s` are %lld elements apart (at most 2^22)", what, name, (long long)ld);
  if (written && ((T > 1 && ld < width) || (B > 1 && bs < (T - 1) * ld + width)))
    return set_error("%s: rows of `%s` overlap", what, name);
  out->p = p;
  out->ld = ld;
  out->bs = bs;
  return 0;
}

static int decay_launch_any(int dtype, DecayArgs a, int roles, int dk, int dv, hipStream_t st) {
  a.roles = roles;
  a.order = a.lengths && a.B > 1 && a.B <= 64 && (long)a.B * a.H * roles * a.segments > kDecayOrderFrom;
  return dtype == LMUFFT_BF16 ? decay_launch_bf16(a, roles, dk, dv, st) : decay_launch_f32(a, roles, dk, dv, st);
}

}  // namespace lmufft

using namespace lmufft;

extern "C" size_t lmufft_decay_workspace_bytes(int dtype, int32_t B, int32_t T, int32_t H, int32_t dk, int32_t dv,
                                               int backward) {
  if (decay_check("decay attention", dtype, B, T, H, dk, dv)) return 0;
  int seg_len = 0;
  const int n = decay_segments(dtype, B, T, H, dk, dv, backward ? 3 : 1, &seg_len);
  return n > 1 ? sizeof(float) * (backward ? 3 : 1) * (size_t)B * H * n * dk * dv : 0;
}

extern "C" int lmufft_decay_attention(const void* q, const void* k, const void* v, int dtype, int64_t ldq, int64_t bsq,
                                      int64_t ldk, int64_t bsk, int64_t ldv, int64_t bsv, const float* log_decay,
                                      const int32_t* lengths, int32_t B, int32_t T, int32_t H, int32_t dk, int32_t dv,
                                      float scale, void* out, int64_t ldo, int64_t bso, float* state, void* workspace,
                                      size_t workspace_bytes, void* stream) {
  const char* what = "decay attention";
  if (decay_check(what, dtype, B, T, H, dk, dv)) return 1;
  if (B == 0 || T == 0) return 0;
  DecayArgs a{};
  DecayRole& r = a.role[0];
  if (decay_tensor(what, "q", q, dtype, ldq, bsq, B, T, (long)H * dk, false, &r.q) ||
      decay_tensor(what, "k", k, dtype, ldk, bsk, B, T, (long)H * dk, false, &r.k) ||
      decay_tensor(what, "v", v, dtype, ldv, bsv, B, T, (long)H * dv, false, &r.v) ||
      decay_tensor(what, "out", out, dtype, ldo, bso, B, T, (long)H * dv, true, &r.out))
    return 1;
  if (!log_decay) return set_error("%s: `log_decay` is NULL", what);
  if (reinterpret_cast<uintptr_t>(state) & 15) return set_error("%s: `state` must be 16-byte aligned", what);
  a.segments = decay_segments(dtype, B, T, H, dk, dv, 1, &a.seg_len);
  const size_t need = lmufft_decay_workspace_bytes(dtype, B, T, H, dk, dv, 0);
  if (need && (!workspace || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 15)))
    return set_error("%s: workspace of %zu bytes on a 16-byte boundary needed, %zu given", what, need, workspace_bytes);
  r.ws = (float*)workspace;
  a.log_decay = log_decay;
  a.lengths = lengths;
  a.state = state;
  a.scale = scale;
  a.B = B, a.T = T, a.H = H;
  a.joined = a.segments >= kDecayJoinFrom;
  return decay_launch_any(dtype, a, 1, dk, dv, (hipStream_t)stream);
}

extern "C" int lmufft_decay_attention_bwd(const void* q, const void* k, const void* v, const void* dout, int dtype,
                                          int64_t ldq, int64_t bsq, int64_t ldk, int64_t bsk, int64_t ldv, int64_t bsv,
                                          int64_t ldd, int64_t bsd, const float* log_decay, const int32_t* lengths,
                                          int32_t B, int32_t T, int32_t H, int32_t dk, int32_t dv, float scale, void* dq,
                                          void* dkey, void* dval, int64_t ld_gq, int64_t bs_gq, int64_t ld_gk,
                                          int64_t bs_gk, int64_t ld_gv, int64_t bs_gv, void* workspace,
                                          size_t workspace_bytes, void* stream) {
  const char* what = "decay attention backward";
  if (decay_check(what, dtype, B, T, H, dk, dv)) return 1;
  if (B == 0 || T == 0) return 0;
  DecayTensor tq, tk, tv, td, gq, gk, gv;
  if (decay_tensor(what, "q", q, dtype, ldq, bsq, B, T, (long)H * dk, false, &tq) ||
      decay_tensor(what, "k", k, dtype, ldk, bsk, B, T, (long)H * dk, false, &tk) ||
      decay_tensor(what, "v", v, dtype, ldv, bsv, B, T, (long)H * dv, false, &tv) ||
      decay_tensor(what, "dout", dout, dtype, ldd, bsd, B, T, (long)H * dv, false, &td) ||
      decay_tensor(what, "dq", dq, dtype, ld_gq, bs_gq, B, T, (long)H * dk, true, &gq) ||
      decay_tensor(what, "dk", dkey, dtype, ld_gk, bs_gk, B, T, (long)H * dk, true, &gk) ||
      decay_tensor(what, "dv", dval, dtype, ld_gv, bs_gv, B, T, (long)H * dv, true, &gv))
    return 1;
  if (!log_decay) return set_error("%s: `log_decay` is NULL", what);
  DecayArgs a{};
  a.segments = decay_segments(dtype, B, T, H, dk, dv, 3, &a.seg_len);
  const size_t need = lmufft_decay_workspace_bytes(dtype, B, T, H, dk, dv, 1);
  if (need && (!workspace || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 15)))
    return set_error("%s: workspace of %zu bytes on a 16-byte boundary needed, %zu given", what, need, workspace_bytes);
  a.log_decay = log_decay;
  a.lengths = lengths;
  a.scale = scale;
  a.B = B, a.T = T, a.H = H;
  a.joined = a.segments >= kDecayJoinFrom;
  const size_t part = (size_t)B * H * a.segments * dk * dv;
  float* const ws = (float*)workspace;
  // dq = A(do, v, k); dk = A_reversed(v, do, q); dv = A_reversed(k, q, do): one launch when the head widths agree
  const DecayRole rq = {td, tv, tk, gq, ws, 0}, rk = {tv, td, tq, gk, ws ? ws + part : ws, 1},
                  rv = {tk, tq, td, gv, ws ? ws + 2 * part : ws, 1};
  a.role[0] = rq, a.role[1] = rk, a.role[2] = rv;
  if (dk == dv) return decay_launch_any(dtype, a, 3, dk, dv, (hipStream_t)stream);
  // the other way round the operator's DK is dv; the chunks the segments were chosen for depend on the sum of the widths
  if (decay_launch_any(dtype, a, 2, dv, dk, (hipStream_t)stream)) return 1;
  a.role[0] = rv;
  return decay_launch_any(dtype, a, 1, dk, dv, (hipStream_t)stream);
}

extern "C" int lmufft_decay_attention_step(const void* q, const void* k, const void* v, int dtype, int64_t ldq, int64_t ldk,
                                           int64_t ldv, const float* log_decay, const int32_t* active, int32_t B, int32_t H,
                                           int32_t dk, int32_t dv, float scale, void* out, int64_t ldo, float* state,
                                           void* stream) {
  const char* what = "decay attention step";
  if (decay_check(what, dtype, B, 1, H, dk, dv)) return 1;
  if (B == 0) return 0;
  if (!q || !k || !v || !log_decay || !out || !state) return set_error("%s: NULL pointer", what);
  if (ldq < 0 || ldk < 0 || ldv < 0 || (B > 1 && ldo < (int64_t)H * dv)) return set_error("%s: bad row stride", what);
  if (reinterpret_cast<uintptr_t>(state) & 15) return set_error("%s: `state` must be 16-byte aligned", what);
  hipStream_t st = (hipStream_t)stream;
  const dim3 grid((unsigned)(B * H)), block(kDecayStepThreads);
  {
    ProfScope ps("k_decay_step", st);
#define DECAY_STEP(TT, DVV)                                                                                              \
  hipLaunchKernelGGL((k_decay_step<TT, DVV>), grid, block, 0, st, (const TT*)q, (const TT*)k, (const TT*)v, (long)ldq,    \
                     (long)ldk, (long)ldv, log_decay, active, H, dk, scale, (TT*)out, (long)ldo, state)
    if (dtype == LMUFFT_BF16) {
      if (dv == 32) DECAY_STEP(__bf16, 32);
      else if (dv == 64) DECAY_STEP(__bf16, 64);
      else DECAY_STEP(__bf16, 128);
    } else {
      if (dv == 32) DECAY_STEP(float, 32);
      else if (dv == 64) DECAY_STEP(float, 64);
      else DECAY_STEP(float, 128);
    }
#undef DECAY_STEP
  }
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return set_error("launch of k_decay_step failed: %s", hipGetErrorString(e));
  return 0;
}
