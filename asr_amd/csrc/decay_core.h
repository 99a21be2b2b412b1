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
// A workgroup of four waves owns one (utterance, head, segment of frames) and walks the segment's chunks.  For the outputs
// a wave owns sixteen frames of the chunk (and, in chunks of 32, half of the columns); the state is held as MFMA accumulators,
// its tiles split over the waves.  With transposed products a wave's intermediates stay in its registers, because the
// accumulator layout of a 16 x 16 tile (lane = column, four consecutive rows) is, two tiles side by side, the operand layout
// of the next product up to a permutation of the contraction index, which the reads of the other operand follow:
//   P^T = K Q^T          A = K rows, B = Q rows
//   O^T = S^T Q^T + V^T P^T     A = S^T rows, B = Q rows;  A = V^T columns, B = P^T's accumulators
//   S  += K^T (w V)      A = K^T columns, B = V^T columns scaled by lambda^(C-1-j)
// q, k, v go through LDS by rows, as they lie in memory, and the state in the products' type; columns are read from there by
// the transposing LDS read (bf16) or element by element (f32).  The next chunk's rows are fetched into registers while the
// present one is computed, and the state is handed over at the barriers that the tiles need anyway.
//
// Rounding: products accumulate in 32 bits and the state is held in 32 bits.  bf16 tensors: P and the copy of S that
// multiplies q are rounded to bf16 once (what a bf16 operand of the matrix cores costs; each is below the rounding of the
// output); the scaled v that enters the state is split into bf16 terms, three where the state is returned (24 bits are kept).
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
__device__ __forceinline__ void dec_store8(__bf16* p, const dec_f4& v, const dec_f4& w) {
  dec_b8 o;
  dec_pack(o, v, w);
  *reinterpret_cast<dec_b8*>(p) = o;
}
__device__ __forceinline__ void dec_store8(float* p, const dec_f4& v, const dec_f4& w) {
  dec_store4(p, v);
  dec_store4(p + 4, w);
}

// lambda^n for n >= 0 from log2 lambda, which is held above -2^100 so that lambda = 0 gives lambda^0 = 1 (and 0 behind it)
__device__ __forceinline__ float dec_log2(float log_decay) {
  const float a2 = log_decay * 1.4426950408889634f;
  return a2 < -0x1p100f ? -0x1p100f : a2;
}
__device__ __forceinline__ float dec_pow(float a2, int n) { return __builtin_amdgcn_exp2f(a2 * (float)n); }
__device__ __forceinline__ float dec_uniform(float x) {
  return __int_as_float(__builtin_amdgcn_readfirstlane(__float_as_int(x)));
}

// Column fragments of a tile that lies in LDS by rows (pitch P): a lane's eight values are one column of the rows 4g..4g+3 and
// 16+4g..16+4g+3 behind `tile`, as the accumulators of two tiles hold them.  Lane i of sixteen has the column i.
// dec_cols_spread: it has the column 8 (i / 4) + i % 4 (of 32; the other sixteen lie four columns on): the accumulators of two
// such tiles hold eight columns side by side.
template <int P>
__device__ __forceinline__ void dec_cols_at(dec_b8& f, const __bf16* a) {
  typedef dec_b4 __attribute__((address_space(3))) * lds4;
  const dec_b4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds4)a);
  const dec_b4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds4)(a + 16 * P));
#pragma unroll
  for (int e = 0; e < 4; ++e) f[e] = lo[e], f[4 + e] = hi[e];
}
// (the transposing read: of sixteen lanes, lane 4 q + p addresses four columns, piece p, of row q; lane i receives the four
// rows' values of the i-th column of the four pieces side by side)
template <int P>
__device__ __forceinline__ void dec_cols(dec_b8& f, const __bf16* tile, int l16, int g) {
  dec_cols_at<P>(f, tile + (4 * g + (l16 >> 2)) * P + 4 * (l16 & 3));
}
template <int P>
__device__ __forceinline__ void dec_cols_spread(dec_b8& f, const __bf16* tile, int l16, int g) {
  dec_cols_at<P>(f, tile + (4 * g + (l16 >> 2)) * P + 8 * (l16 & 3));
}
template <int P>
__device__ __forceinline__ void dec_cols(DecTraits<float>::frag& f, const float* tile, int l16, int g) {
  const float* a = tile + 4 * g * P + l16;
#pragma unroll
  for (int e = 0; e < 4; ++e) f.a[e] = a[e * P], f.b[e] = a[(16 + e) * P];
}
template <int P>
__device__ __forceinline__ void dec_cols_spread(DecTraits<float>::frag& f, const float* tile, int l16, int g) {
  dec_cols<P>(f, tile, 8 * (l16 >> 2) + (l16 & 3), g);
}

// w v in TERMS bf16 terms: what is left behind the last is below 2^(-9 TERMS) of the value
template <int TERMS>
__device__ __forceinline__ void dec_split(const dec_b8& v, const float w[8], dec_b8 s[TERMS]) {
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    float x = (float)v[e] * w[e];
#pragma unroll
    for (int i = 0; i < TERMS; ++i) {
      s[i][e] = (__bf16)x;
      x -= (float)s[i][e];  // exact
    }
  }
}

// Geometry of the kernels for one (type, DK, DV).
template <class T, int DK, int DV>
struct DecGeo {
  // frames per chunk: 64, or 32 where the tiles would leave room for one workgroup a CU, and for f32, whose products cost more
  static constexpr int C = sizeof(T) == 2 && DK + DV < 256 ? 64 : 32;
  static constexpr int THREADS = 256;
  static constexpr int WQ = C / 16, WD = 4 / WQ;      // waves over the chunk's frames, over the columns of the outputs
  static constexpr int MO = DV / 16 / WD;             // column tiles of a wave's outputs
  static constexpr int MS = DV >= 64 ? DV / 64 : 1;   // column tiles of a wave's part of the state
  static constexpr int KS = DV >= 64 ? 1 : 2;         // waves over the rows of the state
  static constexpr int KT = DK / 16 / KS;             // row tiles of a wave's part
  static constexpr int PAD = 16 / sizeof(T);          // rows 16 bytes longer than their data: sixteen rows hit different banks
  static constexpr int PK = DK + PAD, PV = DV + PAD;  // pitches of the k, q and state tiles, and of the v tile
  static constexpr int VEC = DecTraits<T>::kVec;
  static constexpr int NK = C * DK / VEC / THREADS, NV = C * DV / VEC / THREADS;  // 16-byte pieces a thread stages
  static_assert(NK * VEC * THREADS == C * DK && NV * VEC * THREADS == C * DV, "whole pieces for every thread");
  static constexpr size_t kLdsState = sizeof(T) * (size_t)C * (PK + PV);
  static constexpr size_t kLdsOut = kLdsState + sizeof(T) * (size_t)(C + DV) * PK;
  static constexpr int WAVES = kLdsOut <= 52 * 1024 ? 3 : 2;  // a SIMD: as many workgroups as the LDS holds, and no spills
};

// OUT: the outputs and, in the last segment, the final state.  !OUT: the states at the ends of all segments but the
// last (which the OUT kernel joins), from zero or, in the first segment, from the initial state.
// TERMS: bf16 terms of the scaled v that enters the state (see above): three where the state is returned, two where it only
// serves outputs that are rounded to bf16 themselves.
template <class T, int DK, int DV, bool OUT, int TERMS>
__global__ __launch_bounds__(256, (DecGeo<T, DK, DV>::WAVES)) void k_decay(DecayArgs args) {
  typedef DecGeo<T, DK, DV> G;
  typedef typename DecTraits<T>::frag Frag;
  constexpr int C = G::C, MS = G::MS, KT = G::KT, MO = G::MO, KB = DK / 32, JB = C / 32, VEC = G::VEC, PK = G::PK, PV = G::PV;
  extern __shared__ __attribute__((aligned(16))) unsigned char dec_lds[];
  T* const ktile = reinterpret_cast<T*>(dec_lds);  // [C][DK]
  T* const vtile = ktile + C * PK;                 // [C][DV]
  T* const qtile = vtile + C * PV;                 // [C][DK]
  T* const stile = qtile + C * PK;                 // [DV][DK]: S^T

  const DecayRole& R = args.role[blockIdx.z];
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, l16 = lane & 15, g = lane >> 4;
  const int bh = blockIdx.x, b = bh / args.H, h = bh - b * args.H, seg = blockIdx.y;
  const int T_ = args.T;
  const int len = args.lengths ? min(max(args.lengths[b], 0), T_) : T_;
  const int s0 = seg * args.seg_len, s1 = min(s0 + args.seg_len, T_);
  const int end = min(s1, len);  // frames s0..end-1 are computed, end..s1-1 (of the padding) get zeros
  const bool first = s0 == 0, single = args.segments == 1;
  const bool rev = R.reverse != 0;
  // this wave's part of the state: rows srow.., columns scol..; and of the outputs: frames 16 it.., column tiles mo0..
  const int srow = G::KS == 1 ? 0 : (wave >> 1) * KT * 16, scol = G::KS == 1 ? wave * MS * 16 : (wave & 1) * 16;
  const int it = wave % G::WQ, mo0 = wave / G::WQ * MO;

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

  // ---- staging: thread -> 16-byte pieces (row, columns) of the chunk's tiles.  A chunk's rows lie at a uniform address, which
  // is that of its lowest row in memory, plus 32-bit offsets that do not change.
  auto head = [&](const DecayTensor& x, int width) {
    return reinterpret_cast<const char*>(x.p) + ((long)b * x.bs + (long)h * width) * (long)sizeof(T);
  };
  const char *const kbase = head(R.k, DK), *const vbase = head(R.v, DV), *const qbase = OUT ? head(R.q, DK) : nullptr;
  unsigned koff[G::NK], qoff[OUT ? G::NK : 1], voff[G::NV];
#pragma unroll
  for (int n = 0; n < G::NK; ++n) {
    const int u = tid + n * G::THREADS, row = u / (DK / VEC), c = u % (DK / VEC) * VEC, m = rev ? C - 1 - row : row;
    koff[n] = (unsigned)((m * R.k.ld + c) * (long)sizeof(T));
    if (OUT) qoff[n] = (unsigned)((m * R.q.ld + c) * (long)sizeof(T));
  }
#pragma unroll
  for (int n = 0; n < G::NV; ++n) {
    const int u = tid + n * G::THREADS, row = u / (DV / VEC), c = u % (DV / VEC) * VEC, m = rev ? C - 1 - row : row;
    voff[n] = (unsigned)((m * R.v.ld + c) * (long)sizeof(T));
  }
  dec_u4 kf[G::NK], qf[G::NK], vf[G::NV];
  auto fetch = [&](int t0) {
    const long low = rev ? len - t0 - C : t0;  // (below zero only where the lanes of those rows do not load)
    const char* const ka = kbase + low * R.k.ld * (long)sizeof(T);
    const char* const va = vbase + low * R.v.ld * (long)sizeof(T);
    const char* const qa = OUT ? qbase + low * R.q.ld * (long)sizeof(T) : nullptr;
    const int n_rows = end - t0;
    if (n_rows >= C) {
#pragma unroll
      for (int n = 0; n < G::NK; ++n) {
        kf[n] = *reinterpret_cast<const dec_u4*>(ka + koff[n]);
        if (OUT) qf[n] = *reinterpret_cast<const dec_u4*>(qa + qoff[n]);
      }
#pragma unroll
      for (int n = 0; n < G::NV; ++n) vf[n] = *reinterpret_cast<const dec_u4*>(va + voff[n]);
    } else {
#pragma unroll
      for (int n = 0; n < G::NK; ++n) {
        const bool in = (tid + n * G::THREADS) / (DK / VEC) < n_rows;
        kf[n] = dec_u4(0u);
        if (in) kf[n] = *reinterpret_cast<const dec_u4*>(ka + koff[n]);
        if (OUT) {
          qf[n] = dec_u4(0u);
          if (in) qf[n] = *reinterpret_cast<const dec_u4*>(qa + qoff[n]);
        }
      }
#pragma unroll
      for (int n = 0; n < G::NV; ++n) {
        vf[n] = dec_u4(0u);
        if ((tid + n * G::THREADS) / (DV / VEC) < n_rows) vf[n] = *reinterpret_cast<const dec_u4*>(va + voff[n]);
      }
    }
  };
  auto stage = [&]() {
#pragma unroll
    for (int n = 0; n < G::NK; ++n) {
      const int u = tid + n * G::THREADS, at = u / (DK / VEC) * PK + u % (DK / VEC) * VEC;
      *reinterpret_cast<dec_u4*>(ktile + at) = kf[n];
      if (OUT) *reinterpret_cast<dec_u4*>(qtile + at) = qf[n];
    }
#pragma unroll
    for (int n = 0; n < G::NV; ++n) {
      const int u = tid + n * G::THREADS;
      *reinterpret_cast<dec_u4*>(vtile + u / (DV / VEC) * PV + u % (DV / VEC) * VEC) = vf[n];
    }
  };
  if (s0 < end) fetch(s0);

  // ---- powers of the decay: lambda^(i-j) is, tile by tile, the one of the places inside the tiles times a uniform one
  const float a2 = dec_log2(args.log_decay[h]);
  auto upow = [&](int n) { return dec_uniform(dec_pow(a2, n)); };
  float wdiag[4], woff[4], wend[4];
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const int d = l16 - (4 * g + r);
    wdiag[r] = dec_pow(a2, max(d, 0));
    woff[r] = dec_pow(a2, 16 + d);
    wend[r] = dec_pow(a2, 15 - (4 * g + r));
  }
  const float fq = dec_pow(a2, 16 * it + l16 + 1);

  // ---- the state this segment starts from: tile (t, m), this lane: column scol + 16 m + l16, rows srow + 16 t + 4 g + r
  dec_f4 S[KT][MS];
#pragma unroll
  for (int t = 0; t < KT; ++t)
#pragma unroll
    for (int m = 0; m < MS; ++m) S[t][m] = dec_f4(0.f);
  const int splace = (srow + 4 * g) * DV + scol + l16;
  const int wplace = wave * (KT * MS * 64) + lane;  // in the workspace the accumulators lie as they are
  if (first && args.state) {
    // (with several segments the copy is read, see above)
    const float* sp = (OUT && !single ? R.ws + ((long)bh * args.segments + args.segments - 1) * (DK * DV)
                                      : args.state + (long)bh * DK * DV) + splace;
#pragma unroll
    for (int t = 0; t < KT; ++t)
#pragma unroll
      for (int m = 0; m < MS; ++m)
#pragma unroll
        for (int r = 0; r < 4; ++r) S[t][m][r] = sp[(16 * t + r) * DV + 16 * m];
  }
  if (OUT && !first && s0 < len) {
    // joined from the states at the ends of the earlier segments: sum over s' < seg of lambda^((seg-1-s') seg_len) E_s'
    float w = 1.f;
    const float lamL = upow(args.seg_len);
    for (int s = seg - 1; s >= 0 && w != 0.f; --s, w *= lamL) {
      const dec_f4* e = reinterpret_cast<const dec_f4*>(R.ws + ((long)bh * args.segments + s) * (DK * DV)) + wplace;
#pragma unroll
      for (int t = 0; t < KT; ++t)
#pragma unroll
        for (int m = 0; m < MS; ++m) S[t][m] += w * e[(t * MS + m) * 64];
    }
  }

  T* const op = (T*)R.out.p + (long)b * R.out.bs + (long)h * DV + 8 * g;
  for (int t0 = s0; t0 < end; t0 += C) {
    const int n = min(C, end - t0);  // frames of this chunk
    __syncthreads();                 // everybody has finished with the previous one
    stage();
    if (OUT) {
#pragma unroll
      for (int t = 0; t < KT; ++t)
#pragma unroll
        for (int m = 0; m < MS; ++m) dec_store4(stile + (scol + 16 * m + l16) * PK + srow + 16 * t + 4 * g, S[t][m]);
    }
    __syncthreads();
    if (t0 + C < end) fetch(t0 + C);

    if (OUT && 16 * it < n) {
      Frag qx[KB];
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) dec_lds_frag(qx[kb], qtile + (16 * it + l16) * PK + kb * 32 + g * 8);
      dec_f4 o[MO];
#pragma unroll
      for (int i = 0; i < MO; ++i) {  // column tile mo: columns 32 (mo / 2) + 4 (mo % 2) + 8 (row / 4) + row % 4
        const int mo = mo0 + i;
        const T* const sr = stile + (32 * (mo >> 1) + 4 * (mo & 1) + 8 * (l16 >> 2) + (l16 & 3)) * PK + g * 8;
        o[i] = dec_f4(0.f);
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
          Frag sx;
          dec_lds_frag(sx, sr + kb * 32);
          o[i] = dec_mma(sx, qx[kb], o[i]);
        }
        o[i] *= fq;
      }
#pragma unroll 1
      for (int jb = 0; jb <= it >> 1; ++jb) {
        dec_f4 p[2];
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const int jt = 2 * jb + x;
          p[x] = dec_f4(0.f);
          if (jt > it) continue;
#pragma unroll
          for (int kb = 0; kb < KB; ++kb) {
            Frag kx;
            dec_lds_frag(kx, ktile + (16 * jt + l16) * PK + kb * 32 + g * 8);
            p[x] = dec_mma(kx, qx[kb], p[x]);
          }
          if (jt == it) {  // masked by selection: a frame behind this one contributes nothing, whatever it holds
#pragma unroll
            for (int r = 0; r < 4; ++r) p[x][r] = l16 >= 4 * g + r ? p[x][r] * wdiag[r] : 0.f;
          } else {
            const float far = upow(16 * (it - jt - 1));
#pragma unroll
            for (int r = 0; r < 4; ++r) p[x][r] *= woff[r] * far;
          }
        }
        Frag pf;
        dec_pack(pf, p[0], p[1]);
#pragma unroll
        for (int i = 0; i < MO; ++i) {
          const int mo = mo0 + i;
          Frag vx;
          dec_cols_spread<PV>(vx, vtile + jb * 32 * PV + 32 * (mo >> 1) + 4 * (mo & 1), l16, g);
          o[i] = dec_mma(vx, pf, o[i]);
        }
      }
      const int t = t0 + 16 * it + l16;
      if (t < end) {
        T* const dst = op + (long)(rev ? len - 1 - t : t) * R.out.ld;
        if constexpr (MO == 1) {
          dec_store4(dst + 32 * (mo0 >> 1) + 4 * (mo0 & 1), o[0] * args.scale);
        } else {
#pragma unroll
          for (int i = 0; i < MO; i += 2) dec_store8(dst + 16 * (mo0 + i), o[i] * args.scale, o[i + 1] * args.scale);
        }
      }
    }

    // ---- the state behind the chunk
    const float lam = upow(n);
#pragma unroll
    for (int t = 0; t < KT; ++t)
#pragma unroll
      for (int m = 0; m < MS; ++m) S[t][m] *= lam;
#pragma unroll
    for (int jb = 0; jb < JB; ++jb) {
      float w[8];  // lambda^(n-1-j) of this lane's frames (those behind the end hold zeros)
      if (n == C) {
        const float w0 = upow(C - 16 - 32 * jb), w1 = upow(C - 32 - 32 * jb);
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = wend[e] * w0, w[4 + e] = wend[e] * w1;
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) w[e] = dec_pow(a2, max(n - 1 - (jb * 32 + (e >> 2) * 16 + 4 * g + (e & 3)), 0));
      }
      Frag wv[MS][sizeof(T) == 2 ? TERMS : 1];
#pragma unroll
      for (int m = 0; m < MS; ++m) {
        Frag vx;
        dec_cols<PV>(vx, vtile + jb * 32 * PV + scol + 16 * m, l16, g);
        if constexpr (sizeof(T) == 2) {
          dec_split<TERMS>(vx, w, wv[m]);
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e) wv[m][0].a[e] = vx.a[e] * w[e], wv[m][0].b[e] = vx.b[e] * w[4 + e];
        }
      }
#pragma unroll
      for (int t = 0; t < KT; ++t) {
        Frag kx;
        dec_cols<PK>(kx, ktile + jb * 32 * PK + srow + 16 * t, l16, g);
#pragma unroll
        for (int m = 0; m < MS; ++m)
#pragma unroll
          for (int x = (sizeof(T) == 2 ? TERMS : 1) - 1; x >= 0; --x) S[t][m] = dec_mma(kx, wv[m][x], S[t][m]);
      }
    }
  }

  if (!OUT) {
    dec_f4* e = reinterpret_cast<dec_f4*>(R.ws + ((long)bh * args.segments + seg) * (DK * DV)) + wplace;
#pragma unroll
    for (int t = 0; t < KT; ++t)
#pragma unroll
      for (int m = 0; m < MS; ++m) e[(t * MS + m) * 64] = S[t][m];
    return;
  }
  // zeros behind the utterance's end
  for (int i = max(s0, len) * (DV / VEC) + tid; i < s1 * (DV / VEC); i += G::THREADS) {
    const int t = i / (DV / VEC), c = (i % (DV / VEC)) * VEC;
    *reinterpret_cast<dec_u4*>((T*)R.out.p + (long)b * R.out.bs + (long)t * R.out.ld + (long)h * DV + c) = dec_u4(0u);
  }
  // the final state, by the segment that holds the last frame (an empty utterance keeps what it had)
  if (args.state && s0 < len && s1 >= len) {
    float* sp = args.state + (long)bh * DK * DV + splace;
#pragma unroll
    for (int t = 0; t < KT; ++t)
#pragma unroll
      for (int m = 0; m < MS; ++m)
#pragma unroll
        for (int r = 0; r < 4; ++r) sp[(16 * t + r) * DV + 16 * m] = S[t][m][r];
  }
}

template <class T, int DK, int DV, int TERMS>
static int decay_launch_terms(const DecayArgs& a, int roles, hipStream_t st) {
  typedef DecGeo<T, DK, DV> G;
  static_assert(G::kLdsOut <= 160 * 1024, "a workgroup's tiles fit the CU's LDS");
  if (G::kLdsOut > 48 * 1024) {  // more dynamic LDS than the default limit has to be asked for
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(&k_decay<T, DK, DV, true, TERMS>),
                                             hipFuncAttributeMaxDynamicSharedMemorySize, (int)G::kLdsOut);
    if (e != hipSuccess) return set_error("decay attention: %zu bytes of LDS refused: %s", G::kLdsOut, hipGetErrorString(e));
  }
  if (a.segments > 1) {
    ProfScope ps("k_decay_states", st);
    hipLaunchKernelGGL((k_decay<T, DK, DV, false, TERMS>), dim3(a.B * a.H, a.segments - 1, roles), dim3(G::THREADS),
                       G::kLdsState, st, a);
  }
  {
    ProfScope ps("k_decay", st);
    hipLaunchKernelGGL((k_decay<T, DK, DV, true, TERMS>), dim3(a.B * a.H, a.segments, roles), dim3(G::THREADS), G::kLdsOut,
                       st, a);
  }
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return set_error("launch of k_decay failed: %s", hipGetErrorString(e));
  return 0;
}
template <class T, int DK, int DV>
static int decay_launch(const DecayArgs& a, int roles, hipStream_t st) {
  if constexpr (sizeof(T) == 4) return decay_launch_terms<T, DK, DV, 1>(a, roles, st);
  else return a.state ? decay_launch_terms<T, DK, DV, 3>(a, roles, st) : decay_launch_terms<T, DK, DV, 2>(a, roles, st);
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
