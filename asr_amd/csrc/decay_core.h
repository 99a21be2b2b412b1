// Causal linear attention with one decay per head: the chunk kernels (templates; decay_bf16.hip and decay_f32.hip
// instantiate them, decay.hip holds the C entry points and the single-frame kernel).
//
// Per head, with decay lambda in [0, 1] and a state S [DK][DV]:
//   S_t = lambda S_(t-1) + k_t v_t^T,      o_t = scale S_t^T q_t.
// A chunk of C frames that starts from the state S (rows i, j of the chunk):
//   P_ij = lambda^(i-j) (q_i . k_j)  for j <= i, else 0
//   O    = scale (P V + diag(lambda^(i+1)) Q S)
//   S'   = lambda^C S + sum_j lambda^(C-1-j) k_j v_j^T
// The gradients are the same operator with its operands exchanged, two of them run from the last frame to the first:
//   dq = A(do, v, k),   dk = A_reversed(v, do, q),   dv = A_reversed(k, q, do),
// so one kernel serves both directions and a launch takes up to three such roles.
//
// A workgroup owns one (utterance, head, segment of frames) and walks the segment's chunks with the state in
// registers.  Its waves split the DV columns: a wave holds S[all DK][its columns] as MFMA accumulators and computes
// O^T[its columns][all frames of the chunk].  With transposed products every intermediate stays in registers, because
// the accumulator layout of a 16 x 16 tile (lane = column, four consecutive rows) is, two tiles side by side, the operand
// layout of the next product up to a permutation of the contraction index -- and that permutation is baked into how the
// operands from memory are stored in LDS:
//   P^T = K Q^T          A = K rows, B = Q rows            (contraction over DK, permuted in 32s)
//   O^T = S^T Q^T + V^T P^T     A = S^T from S's accumulators, B = Q rows;  A = V^T columns, B = P^T's accumulators
//   S  += K^T (w V)      A = K^T columns, B = V^T columns scaled by lambda^(C-1-j)
// Only q, k, v go through LDS (k both by rows and by columns); the next chunk's rows are fetched into registers while
// the present one is computed.  Every wave computes all of P^T: sharing it through LDS would cost a barrier per tile.
//
// Rounding: products accumulate in 32 bits and the state is held in 32 bits.  bf16 tensors: P and the copy of S that
// multiplies q are rounded to bf16 once (what a bf16 operand of the matrix cores costs; each is below the rounding of the
// output); the scaled v that enters the state is split into three bf16 terms, so the state keeps 24 bits.
// f32 tensors: the exact-f32 matrix instruction throughout.
#pragma once
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include "lmufft.h"
#include "lmufft_internal.h"

namespace lmufft {

typedef float dec_f4 __attribute__((ext_vector_type(4)));
typedef __bf16 dec_b8 __attribute__((ext_vector_type(8)));
typedef __bf16 dec_b4 __attribute__((ext_vector_type(4)));
typedef unsigned int dec_u4 __attribute__((ext_vector_type(4)));

constexpr int kDecayMaxSegments = 32;
constexpr int kDecayMaxRoles = 3;

// One tensor [B][T][H * width] with unit column stride: element strides of a frame and of an utterance.
struct DecayTensor {
  const void* p;
  long ld, bs;
};
// One application of the operator: out = A(q, k, v), from the last frame to the first when `reverse`.
struct DecayRole {
  DecayTensor q, k, v, out;
  float* ws;  // [B * H][segments][DK * DV]: states at the segments' ends (and the initial state), segments > 1 only
  int reverse;
};
struct DecayArgs {
  DecayRole role[kDecayMaxRoles];
  const float* log_decay;  // [H]
  const int* lengths;      // [B] or NULL
  float* state;            // [B][H][DK][DV]: read at the start, replaced at the end; or NULL
  float scale;
  int B, T, H, segments, seg_len;
};

int decay_chunk_bf16(int dk, int dv);  // frames per chunk
int decay_chunk_f32(int dk, int dv);
int decay_launch_bf16(const DecayArgs& a, int roles, int dk, int dv, hipStream_t st);
int decay_launch_f32(const DecayArgs& a, int roles, int dk, int dv, hipStream_t st);

template <class T>
struct DecTraits;
template <>
struct DecTraits<__bf16> {
  typedef dec_b8 frag;                     // eight values of the contraction index of one row
  static constexpr int kVec = 8;           // elements of a 16-byte load
};
template <>
struct DecTraits<float> {
  struct frag {
    dec_f4 a, b;
  };
  static constexpr int kVec = 4;
};

__device__ __forceinline__ dec_f4 dec_mma(const dec_b8& a, const dec_b8& b, const dec_f4& c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
// The 4-deep f32 product gives lane group g the contraction index g; element e of both fragments is taken by step e,
// so the eight steps cover the same 32 indices as one bf16 product, in the same fragment layout.
__device__ __forceinline__ dec_f4 dec_mma(const DecTraits<float>::frag& a, const DecTraits<float>::frag& b, dec_f4 c) {
#pragma unroll
  for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a.a[e], b.a[e], c, 0, 0, 0);
#pragma unroll
  for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a.b[e], b.b[e], c, 0, 0, 0);
  return c;
}
__device__ __forceinline__ void dec_pack(dec_b8& f, const dec_f4& lo, const dec_f4& hi) {
#pragma unroll
  for (int e = 0; e < 4; ++e) f[e] = (__bf16)lo[e], f[4 + e] = (__bf16)hi[e];
}
__device__ __forceinline__ void dec_pack(DecTraits<float>::frag& f, const dec_f4& lo, const dec_f4& hi) {
  f.a = lo;
  f.b = hi;
}
__device__ __forceinline__ void dec_lds_frag(dec_b8& f, const __bf16* p) { f = *reinterpret_cast<const dec_b8*>(p); }
__device__ __forceinline__ void dec_lds_frag(DecTraits<float>::frag& f, const float* p) {
  f.a = *reinterpret_cast<const dec_f4*>(p);
  f.b = *reinterpret_cast<const dec_f4*>(p + 4);
}
__device__ __forceinline__ void dec_store4(__bf16* p, const dec_f4& v) {
  dec_b4 o;
#pragma unroll
  for (int e = 0; e < 4; ++e) o[e] = (__bf16)v[e];
  *reinterpret_cast<dec_b4*>(p) = o;
}
__device__ __forceinline__ void dec_store4(float* p, const dec_f4& v) { *reinterpret_cast<dec_f4*>(p) = v; }

// lambda^n for n >= 0 from log2 lambda (which is -inf for lambda = 0: lambda^0 is 1 all the same)
__device__ __forceinline__ float dec_pow(float a2, int n) { return n == 0 ? 1.f : exp2f(a2 * (float)n); }

// Position, inside its 32, of contraction index x in a stored operand: the accumulator pair (tiles 2b, 2b + 1) gives lane
// group g the indices 4g..4g+3 and 16+4g..16+4g+3, which are stored side by side.
__device__ __forceinline__ constexpr int dec_perm(int x) { return ((x & 15) >> 2) * 8 + (x >> 4) * 4 + (x & 3); }

// A fetched 16-byte piece of a row goes to LDS by rows: quads of columns at their permuted places.
__device__ __forceinline__ void dec_put_row(__bf16* row, int c0, const dec_u4& v) {
  const int base = c0 & ~31, x = c0 & 31;
  *reinterpret_cast<uint2*>(row + base + dec_perm(x)) = make_uint2(v[0], v[1]);
  *reinterpret_cast<uint2*>(row + base + dec_perm(x + 4)) = make_uint2(v[2], v[3]);
}
__device__ __forceinline__ void dec_put_row(float* row, int c0, const dec_u4& v) {
  *reinterpret_cast<dec_u4*>(row + (c0 & ~31) + dec_perm(c0 & 31)) = v;
}
// Four rows' pieces (rows j0..j0+3, j0 a multiple of four) go to LDS by columns: tile[column][permuted row].
template <int PITCH>
__device__ __forceinline__ void dec_put_cols(__bf16* tile, int c0, int j0, const dec_u4 v[4]) {
  __bf16* dst = tile + c0 * PITCH + (j0 & ~31) + dec_perm(j0 & 31);
#pragma unroll
  for (int e = 0; e < 4; ++e) {  // columns c0 + 2e and c0 + 2e + 1 share a 32-bit word of each row
    const uint2 even = make_uint2(__builtin_amdgcn_perm(v[1][e], v[0][e], 0x05040100u),
                                  __builtin_amdgcn_perm(v[3][e], v[2][e], 0x05040100u));
    const uint2 odd = make_uint2(__builtin_amdgcn_perm(v[1][e], v[0][e], 0x07060302u),
                                 __builtin_amdgcn_perm(v[3][e], v[2][e], 0x07060302u));
    *reinterpret_cast<uint2*>(dst + (2 * e) * PITCH) = even;
    *reinterpret_cast<uint2*>(dst + (2 * e + 1) * PITCH) = odd;
  }
}
template <int PITCH>
__device__ __forceinline__ void dec_put_cols(float* tile, int c0, int j0, const dec_u4 v[4]) {
  float* dst = tile + c0 * PITCH + (j0 & ~31) + dec_perm(j0 & 31);
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    dec_u4 t;
#pragma unroll
    for (int r = 0; r < 4; ++r) t[r] = v[r][e];
    *reinterpret_cast<dec_u4*>(dst + e * PITCH) = t;
  }
}

// acc += A^T-free product with B = w * v in the state's precision
__device__ __forceinline__ void dec_split(const dec_b8& v, const float w[8], dec_b8 s[3]) {
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float x = (float)v[e] * w[e];
    const __bf16 h = (__bf16)x;
    const float r = x - (float)h;  // exact
    const __bf16 m = (__bf16)r;
    s[0][e] = h;
    s[1][e] = m;
    s[2][e] = (__bf16)(r - (float)m);
  }
}

// Geometry of the kernels for one (type, DK, DV).
template <class T, int DK, int DV>
struct DecGeo {
  static constexpr int NW = DV >= 64 ? 4 : 2;       // waves; each owns DV / NW columns of S and O
  static constexpr int MT = DV / NW / 16;           // 16-column tiles of a wave
  static constexpr int C = sizeof(T) == 2 ? 64 : 32;  // frames per chunk
  static constexpr int PAD = 16 / sizeof(T);        // rows 16 bytes longer than 64 words: sixteen rows hit different banks
  static constexpr int PR = DK + PAD;               // pitch of the tiles stored by rows
  static constexpr int PC = C + PAD;                // pitch of the tiles stored by columns
  static constexpr int VEC = DecTraits<T>::kVec;
  static constexpr int THREADS = 64 * NW;
  static constexpr int UK = (C / 4) * (DK / VEC), UV = (C / 4) * (DV / VEC);  // units: four rows x 16 bytes
  static constexpr int NK = (UK + THREADS - 1) / THREADS, NV = (UV + THREADS - 1) / THREADS;
  static constexpr size_t kLdsState = sizeof(T) * ((size_t)DK * PC + (size_t)DV * PC);
  static constexpr size_t kLdsOut = kLdsState + sizeof(T) * 2 * (size_t)C * PR;
};

// OUT: the outputs and, in the last segment, the final state.  !OUT: the states at the ends of all segments but the
// last (which the OUT kernel joins), from zero or, in the first segment, from the initial state.
template <class T, int DK, int DV, bool OUT>
__global__ __launch_bounds__(64 * (DV >= 64 ? 4 : 2)) void k_decay(DecayArgs args) {
  typedef DecGeo<T, DK, DV> G;
  typedef typename DecTraits<T>::frag Frag;
  constexpr int C = G::C, MT = G::MT, KT = DK / 16, KB = DK / 32, JB = C / 32, IT = C / 16, VEC = G::VEC;
  extern __shared__ __attribute__((aligned(16))) unsigned char dec_lds[];
  T* const kcol = reinterpret_cast<T*>(dec_lds);  // [DK][C]
  T* const vcol = kcol + DK * G::PC;              // [DV][C]
  T* const krow = vcol + DV * G::PC;              // [C][DK]
  T* const qrow = krow + C * G::PR;               // [C][DK]

  const DecayRole& R = args.role[blockIdx.z];
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, l16 = lane & 15, g = lane >> 4;
  const int bh = blockIdx.x, b = bh / args.H, h = bh - b * args.H, seg = blockIdx.y;
  const int T_ = args.T;
  const int len = args.lengths ? min(max(args.lengths[b], 0), T_) : T_;
  const int s0 = seg * args.seg_len, s1 = min(s0 + args.seg_len, T_);
  const int end = min(s1, len);  // frames s0..end-1 are computed, end..s1-1 (of the padding) get zeros
  const bool first = s0 == 0, single = args.segments == 1;
  const bool rev = R.reverse != 0;
  const int col0 = wave * (DV / G::NW);  // this wave's first column

  if (!OUT) {
    // the last segment's copy of the state has a slot of its own: it may be replaced while others still read it
    if (first && args.state) {
      const float* src = args.state + (long)bh * DK * DV;
      float* dst = R.ws + ((long)bh * args.segments + args.segments - 1) * (DK * DV);
      for (int i = tid * 4; i < DK * DV; i += G::THREADS * 4)
        *reinterpret_cast<dec_f4*>(dst + i) = *reinterpret_cast<const dec_f4*>(src + i);
    }
    if (s0 + args.seg_len >= len) return;  // nobody needs the state behind this segment
  }

  const T* const qp = (const T*)R.q.p + (long)b * R.q.bs + (long)h * DK;
  const T* const kp = (const T*)R.k.p + (long)b * R.k.bs + (long)h * DK;
  const T* const vp = (const T*)R.v.p + (long)b * R.v.bs + (long)h * DV;
  const float a2 = args.log_decay[h] * 1.4426950408889634f;

  // ---- the state this segment starts from; tile t = rows 16t..16t+15, this lane: column col0 + 16 m + l16, rows 4g..4g+3
  dec_f4 S[KT][MT];
#pragma unroll
  for (int t = 0; t < KT; ++t)
#pragma unroll
    for (int m = 0; m < MT; ++m) S[t][m] = dec_f4(0.f);
  if (first && args.state && s0 <= len) {
    // (with several segments the copy is read, see above)
    const float* sp = OUT && !single ? R.ws + ((long)bh * args.segments + args.segments - 1) * (DK * DV)
                                     : args.state + (long)bh * DK * DV;
#pragma unroll
    for (int t = 0; t < KT; ++t)
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int r = 0; r < 4; ++r) S[t][m][r] = sp[(16 * t + 4 * g + r) * DV + col0 + 16 * m + l16];
  }
  if (OUT && !first && s0 < len) {
    // joined from the states at the ends of the earlier segments: sum over s' < seg of lambda^((seg-1-s') seg_len) E_s'
    float w = 1.f;
    const float lamL = dec_pow(a2, args.seg_len);
    for (int s = seg - 1; s >= 0 && w != 0.f; --s, w *= lamL) {
      const dec_f4* e = reinterpret_cast<const dec_f4*>(R.ws + ((long)bh * args.segments + s) * (DK * DV)) +
                        wave * (KT * MT * 64) + lane;
#pragma unroll
      for (int t = 0; t < KT; ++t)
#pragma unroll
        for (int m = 0; m < MT; ++m) S[t][m] += w * e[(t * MT + m) * 64];
    }
  }

  // ---- powers of the decay
  float wdiag[4], woff[4], wfar[IT], fq[IT];
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const int d = l16 - (4 * g + r);  // i - j inside a tile
    wdiag[r] = d >= 0 ? dec_pow(a2, max(d, 0)) : 0.f;
    woff[r] = dec_pow(a2, 16 + d);
  }
#pragma unroll
  for (int t = 0; t < IT; ++t) {
    wfar[t] = t ? dec_pow(a2, 16 * (t - 1)) : 1.f;
    fq[t] = dec_pow(a2, 16 * t + l16 + 1);
  }
  float wv[JB][8];

  // ---- staging
  dec_u4 kf[G::NK][4], vf[G::NV][4], qf[G::NK][4];
  auto fetch_rows = [&](const T* p, long ld, int c0, int j0, int t0, dec_u4 out[4]) {
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int t = t0 + j0 + r;
      dec_u4 x = dec_u4(0u);
      if (t < end) x = *reinterpret_cast<const dec_u4*>(p + (long)(rev ? len - 1 - t : t) * ld + c0);
      out[r] = x;
    }
  };
  auto fetch = [&](int t0) {
#pragma unroll
    for (int n = 0; n < G::NK; ++n) {
      const int u = tid + n * G::THREADS, c0 = (u % (DK / VEC)) * VEC, j0 = (u / (DK / VEC)) * 4;
      if (G::UK % G::THREADS != 0 && u >= G::UK) continue;
      fetch_rows(kp, R.k.ld, c0, j0, t0, kf[n]);
      if (OUT) fetch_rows(qp, R.q.ld, c0, j0, t0, qf[n]);
    }
#pragma unroll
    for (int n = 0; n < G::NV; ++n) {
      const int u = tid + n * G::THREADS, c0 = (u % (DV / VEC)) * VEC, j0 = (u / (DV / VEC)) * 4;
      if (G::UV % G::THREADS != 0 && u >= G::UV) continue;
      fetch_rows(vp, R.v.ld, c0, j0, t0, vf[n]);
    }
  };
  auto stage = [&]() {
#pragma unroll
    for (int n = 0; n < G::NK; ++n) {
      const int u = tid + n * G::THREADS, c0 = (u % (DK / VEC)) * VEC, j0 = (u / (DK / VEC)) * 4;
      if (G::UK % G::THREADS != 0 && u >= G::UK) continue;
      dec_put_cols<G::PC>(kcol, c0, j0, kf[n]);
      if (OUT) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          dec_put_row(krow + (j0 + r) * G::PR, c0, kf[n][r]);
          dec_put_row(qrow + (j0 + r) * G::PR, c0, qf[n][r]);
        }
      }
    }
#pragma unroll
    for (int n = 0; n < G::NV; ++n) {
      const int u = tid + n * G::THREADS, c0 = (u % (DV / VEC)) * VEC, j0 = (u / (DV / VEC)) * 4;
      if (G::UV % G::THREADS != 0 && u >= G::UV) continue;
      dec_put_cols<G::PC>(vcol, c0, j0, vf[n]);
    }
  };

  T* const op = (T*)R.out.p + (long)b * R.out.bs + (long)h * DV + col0;
  if (s0 < end) fetch(s0);
  for (int t0 = s0; t0 < end; t0 += C) {
    const int n = min(C, end - t0);  // frames of this chunk
    __syncthreads();                 // everybody has finished with the previous one
    stage();
    __syncthreads();
    if (t0 + C < end) fetch(t0 + C);

    if (t0 == s0 || n < C) {  // lambda^(n-1-j) of this lane's contraction indices (frames behind the end hold zeros)
#pragma unroll
      for (int jb = 0; jb < JB; ++jb)
#pragma unroll
        for (int e = 0; e < 8; ++e) wv[jb][e] = dec_pow(a2, max(n - 1 - (jb * 32 + (e >> 2) * 16 + 4 * g + (e & 3)), 0));
    }
    Frag vt[MT][JB];  // V^T: row = column of v, contraction over frames
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int jb = 0; jb < JB; ++jb) dec_lds_frag(vt[m][jb], vcol + (col0 + 16 * m + l16) * G::PC + jb * 32 + g * 8);

    if (OUT) {
      Frag st[MT][KB];  // S^T
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) dec_pack(st[m][kb], S[2 * kb][m], S[2 * kb + 1][m]);
#pragma unroll
      for (int it = 0; it < IT; ++it) {
        Frag qx[KB];
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) dec_lds_frag(qx[kb], qrow + (16 * it + l16) * G::PR + kb * 32 + g * 8);
        dec_f4 o[MT];
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          o[m] = dec_f4(0.f);
#pragma unroll
          for (int kb = 0; kb < KB; ++kb) o[m] = dec_mma(st[m][kb], qx[kb], o[m]);
          o[m] *= fq[it];
        }
#pragma unroll
        for (int jb = 0; jb <= it / 2; ++jb) {
          dec_f4 p[2];
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const int jt = 2 * jb + x;
            p[x] = dec_f4(0.f);
            if (jt > it) continue;
#pragma unroll
            for (int kb = 0; kb < KB; ++kb) {
              Frag kx;
              dec_lds_frag(kx, krow + (16 * jt + l16) * G::PR + kb * 32 + g * 8);
              p[x] = dec_mma(kx, qx[kb], p[x]);
            }
            if (jt == it) {  // masked by selection: a frame behind this one contributes nothing, whatever it holds
#pragma unroll
              for (int r = 0; r < 4; ++r) p[x][r] = l16 >= 4 * g + r ? p[x][r] * wdiag[r] : 0.f;
            } else {
#pragma unroll
              for (int r = 0; r < 4; ++r) p[x][r] *= woff[r] * wfar[it - jt];
            }
          }
          Frag pf;
          dec_pack(pf, p[0], p[1]);
#pragma unroll
          for (int m = 0; m < MT; ++m) o[m] = dec_mma(vt[m][jb], pf, o[m]);
        }
        const int t = t0 + 16 * it + l16;
        if (t < end) {
          T* dst = op + (long)(rev ? len - 1 - t : t) * R.out.ld + 4 * g;
#pragma unroll
          for (int m = 0; m < MT; ++m) dec_store4(dst + 16 * m, o[m] * args.scale);
        }
      }
    }

    // ---- the state behind the chunk
    const float lam = dec_pow(a2, n);
#pragma unroll
    for (int t = 0; t < KT; ++t)
#pragma unroll
      for (int m = 0; m < MT; ++m) S[t][m] *= lam;
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int jb = 0; jb < JB; ++jb) {
        if constexpr (sizeof(T) == 2) {
          dec_b8 s[3];
          dec_split(vt[m][jb], wv[jb], s);
#pragma unroll
          for (int t = 0; t < KT; ++t) {
            Frag kx;
            dec_lds_frag(kx, kcol + (16 * t + l16) * G::PC + jb * 32 + g * 8);
#pragma unroll
            for (int x = 2; x >= 0; --x) S[t][m] = dec_mma(kx, s[x], S[t][m]);
          }
        } else {
          Frag s;
#pragma unroll
          for (int e = 0; e < 4; ++e) s.a[e] = vt[m][jb].a[e] * wv[jb][e], s.b[e] = vt[m][jb].b[e] * wv[jb][4 + e];
#pragma unroll
          for (int t = 0; t < KT; ++t) {
            Frag kx;
            dec_lds_frag(kx, kcol + (16 * t + l16) * G::PC + jb * 32 + g * 8);
            S[t][m] = dec_mma(kx, s, S[t][m]);
          }
        }
      }
  }

  if (!OUT) {
    dec_f4* e = reinterpret_cast<dec_f4*>(R.ws + ((long)bh * args.segments + seg) * (DK * DV)) + wave * (KT * MT * 64) + lane;
#pragma unroll
    for (int t = 0; t < KT; ++t)
#pragma unroll
      for (int m = 0; m < MT; ++m) e[(t * MT + m) * 64] = S[t][m];
    return;
  }
  // zeros behind the utterance's end
  for (int i = max(s0, len) * (DV / VEC) + tid; i < s1 * (DV / VEC); i += G::THREADS) {
    const int t = i / (DV / VEC), c = (i % (DV / VEC)) * VEC;
    *reinterpret_cast<dec_u4*>((T*)R.out.p + (long)b * R.out.bs + (long)t * R.out.ld + (long)h * DV + c) = dec_u4(0u);
  }
  // the final state, by the segment that holds the last frame (an empty utterance keeps what it had)
  if (args.state && s0 < len && s1 >= len) {
    float* sp = args.state + (long)bh * DK * DV;
#pragma unroll
    for (int t = 0; t < KT; ++t)
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int r = 0; r < 4; ++r) sp[(16 * t + 4 * g + r) * DV + col0 + 16 * m + l16] = S[t][m][r];
  }
}

template <class T, int DK, int DV>
static int decay_launch(const DecayArgs& a, int roles, hipStream_t st) {
  typedef DecGeo<T, DK, DV> G;
  static_assert(G::kLdsOut <= 160 * 1024, "a workgroup's tiles fit the CU's LDS");
  if (G::kLdsOut > 64 * 1024) {  // above the default limit of dynamic LDS
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(&k_decay<T, DK, DV, true>),
                                             hipFuncAttributeMaxDynamicSharedMemorySize, (int)G::kLdsOut);
    if (e != hipSuccess) return set_error("decay attention: %zu bytes of LDS refused: %s", G::kLdsOut, hipGetErrorString(e));
  }
  if (a.segments > 1) {
    ProfScope ps("k_decay_states", st);
    hipLaunchKernelGGL((k_decay<T, DK, DV, false>), dim3(a.B * a.H, a.segments - 1, roles), dim3(G::THREADS), G::kLdsState,
                       st, a);
  }
  {
    ProfScope ps("k_decay", st);
    hipLaunchKernelGGL((k_decay<T, DK, DV, true>), dim3(a.B * a.H, a.segments, roles), dim3(G::THREADS), G::kLdsOut, st, a);
  }
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return set_error("launch of k_decay failed: %s", hipGetErrorString(e));
  return 0;
}

#define DECAY_FOR_WIDTHS(T, DK_, DV_, RESULT, EXPR)                        \
  do {                                                                     \
    auto for_dv = [&](auto dk_tag) {                                       \
      constexpr int DK = decltype(dk_tag)::value;                          \
      if (DV_ == 32) { constexpr int DV = 32; RESULT = EXPR; }             \
      else if (DV_ == 64) { constexpr int DV = 64; RESULT = EXPR; }        \
      else { constexpr int DV = 128; RESULT = EXPR; }                      \
    };                                                                     \
    if (DK_ == 32) for_dv(std::integral_constant<int, 32>{});              \
    else if (DK_ == 64) for_dv(std::integral_constant<int, 64>{});         \
    else for_dv(std::integral_constant<int, 128>{});                       \
  } while (0)

}  // namespace lmufft
