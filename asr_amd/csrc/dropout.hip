// Residual dropout on gfx950: out = res + keep x / (1 - p), the keep decisions recomputed from the element's place and the
// call's two seeds (HashDropout, lmufft_internal.h), nothing stored.  The backward is the same kernel on the output's
// gradient without a residual.  A thread takes eight neighbouring elements (16 bytes of bf16): one hash serves two of them.
// HBM-bound: reads x and res once, writes out once (25600 x 384 bf16 onto f32: 19 us, 5.2 TB/s; its backward to bf16 12.5 us,
// 4.7 TB/s).
//
// Rows of an even width below 2^32 pairs in all: a pair's hash index is its place in the whole tensor, no division.  Else
// the row and column of a thread's first element come from one division and the others are counted on.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "lmufft.h"
#include "lmufft_internal.h"

namespace lmufft {

constexpr int kDropThreads = 256;
typedef float drop_f4 __attribute__((ext_vector_type(4)));
typedef __bf16 drop_b8 __attribute__((ext_vector_type(8)));

template <bool BF16>
__device__ __forceinline__ void drop_load8(const void* base, long i, float v[8]) {
  if (BF16) {
    const drop_b8 x = *reinterpret_cast<const drop_b8*>(reinterpret_cast<const __bf16*>(base) + i);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = (float)x[e];
  } else {
    const drop_f4* p = reinterpret_cast<const drop_f4*>(reinterpret_cast<const float*>(base) + i);
    const drop_f4 a = p[0], b = p[1];
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = a[e], v[4 + e] = b[e];
  }
}
template <bool BF16>
__device__ __forceinline__ float drop_load1(const void* base, long i) {
  return BF16 ? (float)reinterpret_cast<const __bf16*>(base)[i] : reinterpret_cast<const float*>(base)[i];
}

// RES: 0 none, 1 f32, 2 bf16.  EVEN: see above.
template <bool XB, int RES, bool OB, bool EVEN>
__global__ __launch_bounds__(kDropThreads) void k_dropout_add(const void* x, const void* res, long total, unsigned C,
                                                              void* out, HashDropout dr) {
  hash_resolve_epoch(dr);
  const unsigned pairs = (C + 1) >> 1;
  for (long i = ((long)blockIdx.x * kDropThreads + threadIdx.x) * 8; i < total; i += (long)gridDim.x * kDropThreads * 8) {
    bool keep[8];
    if (EVEN) {
      const HashRow hr = hash_row(dr, 0, pairs);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t h = hash_pair(hr, (uint32_t)(i >> 1) + e);
        keep[2 * e] = hash_keep_lo(dr, h);
        keep[2 * e + 1] = hash_keep_hi(dr, h);
      }
    } else {
      unsigned long long row = (unsigned long long)i / C;
      unsigned col = (unsigned)(i - (long)row * C);
      HashRow hr = hash_row(dr, row, pairs);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        keep[e] = hash_keep(dr, hr, col);
        if (++col == C) col = 0, hr = hash_row(dr, ++row, pairs);
      }
    }
    if (i + 8 <= total) {
      float v[8], r[8];
      drop_load8<XB>(x, i, v);
      if (RES) drop_load8<RES == 2>(res, i, r);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = (keep[e] ? v[e] * dr.inv_keep : 0.f) + (RES ? r[e] : 0.f);
      if (OB) {
        drop_b8 o;
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e] = (__bf16)v[e];
        *reinterpret_cast<drop_b8*>(reinterpret_cast<__bf16*>(out) + i) = o;
      } else {
        drop_f4* p = reinterpret_cast<drop_f4*>(reinterpret_cast<float*>(out) + i);
        p[0] = drop_f4{v[0], v[1], v[2], v[3]};
        p[1] = drop_f4{v[4], v[5], v[6], v[7]};
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        if (i + e >= total) continue;
        const float v = (keep[e] ? drop_load1<XB>(x, i + e) * dr.inv_keep : 0.f) +
                        (RES ? drop_load1<RES == 2>(res, i + e) : 0.f);
        if (OB) reinterpret_cast<__bf16*>(out)[i + e] = (__bf16)v;
        else reinterpret_cast<float*>(out)[i + e] = v;
      }
    }
  }
}

}  // namespace lmufft

using namespace lmufft;

extern "C" int lmufft_dropout_add(const void* x, int x_dtype, const void* res, int res_dtype, int64_t rows, int32_t C,
                                  float p_drop, uint32_t seed0, uint32_t seed1, void* out, int out_dtype, void* stream) {
  const char* what = "dropout";
  auto known = [](int d) { return d == LMUFFT_F32 || d == LMUFFT_BF16; };
  if (!(p_drop >= 0.f && p_drop < 1.f)) return set_error("%s: probability %g outside [0, 1)", what, (double)p_drop);
  if (!known(x_dtype) || !known(out_dtype) || (res && !known(res_dtype))) return set_error("%s: unknown dtype", what);
  if (rows < 0 || C <= 0 || (rows && rows > INT64_MAX / 16 / C)) return set_error("%s: bad shape (rows=%lld C=%d)", what, (long long)rows, C);
  if (rows == 0) return 0;
  if (!x || !out) return set_error("%s: NULL pointer", what);
  auto aligned = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; };
  if (!aligned(x) || !aligned(out) || !aligned(res)) return set_error("%s: tensors must start on 16-byte boundaries", what);
  // in place is fine when the element sizes agree (a thread overwrites exactly what it has read)
  if ((out == x && out_dtype != x_dtype) || (res && out == res && out_dtype != res_dtype))
    return set_error("%s: out may alias x or res only with the same dtype", what);
  const long total = (long)rows * C;
  const HashDropout dr = make_hash_dropout(p_drop, seed0, seed1);
  const bool even = C % 2 == 0 && total / 2 <= 0xffffffffL;
  const dim3 grid((unsigned)std::min<long>((total + kDropThreads * 8 - 1) / (kDropThreads * 8), 256 * 64)), block(kDropThreads);
  hipStream_t st = (hipStream_t)stream;
  {
    ProfScope ps("k_dropout_add", st);
#define DROP_GO(XB, RES, OB)                                                                                              \
  do {                                                                                                                    \
    if (even) hipLaunchKernelGGL((k_dropout_add<XB, RES, OB, true>), grid, block, 0, st, x, res, total, (unsigned)C, out, dr); \
    else hipLaunchKernelGGL((k_dropout_add<XB, RES, OB, false>), grid, block, 0, st, x, res, total, (unsigned)C, out, dr);  \
  } while (0)
#define DROP_RES(XB, OB)                                   \
  do {                                                     \
    if (!res) DROP_GO(XB, 0, OB);                          \
    else if (res_dtype == LMUFFT_F32) DROP_GO(XB, 1, OB);  \
    else DROP_GO(XB, 2, OB);                               \
  } while (0)
    const bool xb = x_dtype == LMUFFT_BF16, ob = out_dtype == LMUFFT_BF16;
    if (xb && ob) DROP_RES(true, true);
    else if (xb) DROP_RES(true, false);
    else if (ob) DROP_RES(false, true);
    else DROP_RES(false, false);
#undef DROP_RES
#undef DROP_GO
  }
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return set_error("launch of k_dropout_add failed: %s", hipGetErrorString(e));
  return 0;
}
