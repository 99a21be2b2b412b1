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
// A workgroup of eight waves owns one (utterance, head, segment of frames) and walks the segment's chunks.  Four waves make
// the outputs, each of sixteen frames of the chunk (in chunks of 32, of half of the columns); four hold the state as MFMA
// accumulators, its tiles split between them, and bring it behind the chunk meanwhile -- the two halves of a chunk are
// independent, and side by side the chain of a chunk is half as long.  With transposed products a wave's intermediates stay
// in its registers, because the accumulator layout of a 16 x 16 tile (lane = column, four consecutive rows) is, two tiles side
// by side, the operand layout of the next product up to a permutation of the contraction index, which the reads of the other
// operand follow:
//   P^T = K Q^T          A = K rows, B = Q rows
//   O^T = S^T Q^T + V^T P^T     A = S^T rows, B = Q rows;  A = V^T columns, B = P^T's accumulators
//   S  += K^T (w V)      A = K^T columns, B = V^T columns scaled by lambda^(C-1-j)
// q, k, v go through LDS by rows, as they lie in memory, and the state in the products' type; columns are read from there by
// the transposing LDS read (bf16) or element by element (f32).  Rows are stored without padding, their 16-byte pieces in an
// order that depends on the row, so that writes, row and column reads all spread over the banks (DecTile; conflict cycles
// counted per LDS instruction: none in the states' kernel of bf16, 1.8-1.9 in the outputs', 2.5 in f32).  The next chunk's rows
// are fetched into registers while the present one is computed.
//
// What bounds it: the chain of a chunk (stage, two products, the state's update between two barriers), 1.7 us for 64 frames when
// a workgroup has a CU to itself, 2.6-2.9 us when two share it.  Batches of full length, bf16: 128 x 400 x 6 heads of 64 36 us,
// 4.3 TB/s; 64 x 3000 x 6 171 us, 3.4 TB/s (a large copy: 4.76).  Lengths from a tenth of the frames up: 64 x 400 x 6 bf16 18.8 us
// forward, 38 us backward; 32 x 3000 x 6 29 + 58 and 124 us; one utterance of 23999 frames 39 us in 75 segments (states 12, join
// 5.5, outputs 21); 16 x 400 x 6 f32 9.6 + 17.5 and 44 us: 13 chunks of 32 frames in the chain, 3.3 us each, of which a SIMD's
// exact-f32 products are 2800 cycles (64 operations a cycle), 1.2 us.
//
// Rounding: products accumulate in 32 bits and the state is held in 32 bits.  bf16 tensors: P and the copy of S that multiplies
// q enter their products in two bf16 terms each, so 2^-16 of a value is lost: an output may hang on a single P, at the start of
// an utterance or under a fast decay, or on the state alone, and one term would cost it as much as the rounding of the result
// (0.0023 of the results' norm in error, 0.0017 with two).  Measured at 64 x 400 x 6: one term each 16.9 us forward and 34.1
// backward, P in two 17.7 and 36.4, both 19.0 and 38.5; 32 x 3000 x 6 76 and 111, 81 and 114, 87 and 119.  The scaled v that
// enters the state is split into two terms, three where the state is returned (24 bits are kept).
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

constexpr int kDecayMaxSegments = 128;
constexpr int kDecayJoinFrom = 5;  // segments from which on their states are joined by a launch of its own
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
  int B, T, H, segments, seg_len, joined, roles;
  int order;  // workgroups take the utterances from the longest to the shortest
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
// what dec_pack's rounding leaves of lo, hi (a NaN of an infinity)
__device__ __forceinline__ void dec_rest(dec_b8& f, const dec_b8& packed, const dec_f4& lo, const dec_f4& hi) {
#pragma unroll
  for (int e = 0; e < 4; ++e) f[e] = (__bf16)(lo[e] - (float)packed[e]), f[4 + e] = (__bf16)(hi[e] - (float)packed[4 + e]);
}
__device__ __forceinline__ void dec_store4(__bf16* p, const dec_f4& v) {
  dec_b4 o;
#pragma unroll
  for (int e = 0; e < 4; ++e) o[e] = (__bf16)v[e];
  *reinterpret_cast<dec_b4*>(p) = o;
}
__device__ __forceinline__ void dec_store4(float* p, const dec_f4& v) { *reinterpret_cast<dec_f4*>(p) = v; }

// A tile of rows of D elements in LDS.  Sixteen 16-byte pieces lie side by side over the banks: the pieces of a row are stored
// at their place xor a key of the row, such that one piece of sixteen consecutive rows (the row reads), and two neighbouring
// pieces of eight (the column reads, 32 lanes at a time), all lie apart.
template <class T, int D>
struct DecTile {
  typedef typename DecTraits<T>::frag Frag;
  static constexpr int VEC = DecTraits<T>::kVec, NP = D / VEC, RP = NP < 16 ? 16 / NP : 1, KEYS = NP < 16 ? NP : 16;
  T* base;
  static __device__ __forceinline__ int key(int row) {  // the row's number among those that would collide, its top bit last
    const int k = row / RP % KEYS;
    return (2 * k + 2 * k / KEYS) % KEYS;
  }
  __device__ __forceinline__ T* piece(int row, int p) const { return base + row * D + (p ^ key(row)) * VEC; }
  // eight elements of a row from column 32 kb + 8 g on
  __device__ __forceinline__ Frag row_frag(int row, int kb, int g) const {
    Frag f;
    if constexpr (VEC == 8) {
      f = *reinterpret_cast<const dec_b8*>(piece(row, 4 * kb + g));
    } else {
      f.a = *reinterpret_cast<const dec_f4*>(piece(row, 8 * kb + 2 * g));
      f.b = *reinterpret_cast<const dec_f4*>(piece(row, 8 * kb + 2 * g + 1));
    }
    return f;
  }
  // column c0 + l16 of the rows r0 + 4g..4g+3 and r0 + 16+4g..16+4g+3, as the accumulators of two tiles hold them (c0, r0
  // multiples of sixteen).  The transposing read: of sixteen lanes, lane 4 q + p addresses four columns, piece p, of row q, and
  // lane i receives the four rows' values of the i-th of the sixteen columns.
  __device__ __forceinline__ Frag col_frag(int r0, int c0, int l16, int g) const {
    Frag f;
    if constexpr (VEC == 8) {
      typedef dec_b4 __attribute__((address_space(3))) * lds4;
      const int row = 4 * g + (l16 >> 2);
      const T* const a = base + (r0 + row) * D + ((c0 / 8 + ((l16 >> 1) & 1)) ^ key(row)) * 8 + (l16 & 1) * 4;
      const dec_b4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds4)a);
      const dec_b4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds4)(a + 16 * D));
#pragma unroll
      for (int e = 0; e < 4; ++e) f[e] = lo[e], f[4 + e] = hi[e];
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const T* const a = piece(4 * g + e, c0 / 4 + (l16 >> 2)) + r0 * D + (l16 & 3);
        f.a[e] = a[0];
        f.b[e] = a[16 * D];
      }
    }
    return f;
  }
  // where four elements of a row lie, from a column that is a multiple of four on
  __device__ __forceinline__ T* four(int row, int c) const { return piece(row, c / VEC) + c % VEC; }
};

// lambda^n for n >= 0 from log2 lambda, which is held above -2^100 so that lambda = 0 gives lambda^0 = 1 (and 0 behind it)
__device__ __forceinline__ float dec_log2(float log_decay) {
  const float a2 = log_decay * 1.4426950408889634f;
  return a2 < -0x1p100f ? -0x1p100f : a2;
}
__device__ __forceinline__ float dec_pow(float a2, int n) { return __builtin_amdgcn_exp2f(a2 * (float)n); }
__device__ __forceinline__ float dec_uniform(float x) {
  return __int_as_float(__builtin_amdgcn_readfirstlane(__float_as_int(x)));
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

// Which of up to 64 utterances is the rank-th longest (equal ones in their order), n: this lane's length, zero and more.  A
// selection bit by bit from the highest: `left` are the utterances that share the bits so far with the one looked for.
__device__ __forceinline__ int dec_ranked(int n, unsigned long long left, int rank, int most) {
  for (int bit = 31 - __builtin_clz(most | 1); bit >= 0; --bit) {
    const unsigned long long one = __ballot((n >> bit) & 1) & left;
    const int c = __popcll(one);
    left = rank < c ? one : left & ~one;
    rank -= rank < c ? 0 : c;
  }
  const int before = __builtin_amdgcn_mbcnt_hi((unsigned)(left >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)left, 0));
  return __ffsll((unsigned long long)__ballot(before == rank) & left) - 1;
}

// Geometry of the kernels for one (type, DK, DV).
template <class T, int DK, int DV>
struct DecGeo {
  // frames per chunk: 64, or 32 where the tiles would leave room for one workgroup a CU, and for f32, whose products cost more
  static constexpr int C = sizeof(T) == 2 && DK + DV < 256 ? 64 : 32;
  static constexpr int WQ = C / 16, WD = 4 / WQ;      // output waves over the chunk's frames, over the columns
  static constexpr int MO = DV / 16 / WD;             // column tiles of a wave's outputs
  static constexpr int MS = DV >= 64 ? DV / 64 : 1;   // column tiles of a wave's part of the state
  static constexpr int KS = DV >= 64 ? 1 : 2;         // waves over the rows of the state
  static constexpr int KT = DK / 16 / KS;             // row tiles of a wave's part
  static constexpr int VEC = DecTraits<T>::kVec;
  static constexpr size_t kLdsState = sizeof(T) * (size_t)C * (DK + DV);
  static constexpr int STERMS = sizeof(T) == 2 ? 2 : 1;  // terms of the state's copy
  static constexpr size_t kLdsOut = kLdsState + sizeof(T) * (size_t)(C + STERMS * DV) * DK;
  static constexpr int WAVES = kLdsOut <= 40 * 1024 && DV <= 64 ? 4 : 2;  // a SIMD: two workgroups of eight waves a CU, or one
};

// OUT (eight waves): the outputs and, in the last segment, the final state.  !OUT (the four waves of the state alone): the
// states at the ends of all segments but the last (which the OUT kernel joins), from zero or, in the first segment, from the
// initial state.
// TERMS: bf16 terms of the scaled v that enters the state (see above): three where the state is returned, two where it only
// serves outputs that are rounded to bf16 themselves.
template <class T, int DK, int DV, bool OUT, int TERMS>
__global__ __launch_bounds__(OUT ? 512 : 256, (DecGeo<T, DK, DV>::WAVES)) void k_decay(DecayArgs args) {
  typedef DecGeo<T, DK, DV> G;
  typedef typename DecTraits<T>::frag Frag;
  constexpr int THREADS = OUT ? 512 : 256;
  constexpr int C = G::C, MS = G::MS, KT = G::KT, MO = G::MO, KB = DK / 32, JB = C / 32, VEC = G::VEC;
  constexpr int PIECES_K = C * DK / VEC, PIECES_V = C * DV / VEC;  // 16-byte pieces of the tiles, and how many a thread stages
  constexpr int NK = (PIECES_K + THREADS - 1) / THREADS, NV = (PIECES_V + THREADS - 1) / THREADS;
  extern __shared__ __attribute__((aligned(16))) unsigned char dec_lds[];
  // OUT: from which frame on a column is NaN, because v holds an infinity or a NaN there
  __shared__ int odd_from[DV], odd_any;
  const DecTile<T, DK> ktile{reinterpret_cast<T*>(dec_lds)};  // [C][DK]
  const DecTile<T, DV> vtile{ktile.base + C * DK};            // [C][DV]
  const DecTile<T, DK> qtile{vtile.base + C * DV};            // [C][DK]
  const DecTile<T, DK> stile{qtile.base + C * DK};            // [DV][DK]: S^T
  const DecTile<T, DK> srest{stile.base + DV * DK};           // bf16: what its rounding left

  const int tid = threadIdx.x, lane = tid & 63, l16 = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6) & 3;             // among those of its kind
  const bool holds = !OUT || __builtin_amdgcn_readfirstlane(tid >> 8) != 0;  // a wave of the state
  // Eight heads of one role, then the same eight of the next: workgroups go round the eight XCDs, so a head's roles meet in one
  // XCD's L2, where two of them read the same rows of two tensors at about the same time (the backward of 32 x 3000 x 6 heads
  // 113.5 -> 108.5 us).
  const unsigned group = blockIdx.x / (8u * args.roles), place = blockIdx.x - group * (8u * args.roles);
  const unsigned wide = min(8u, (unsigned)(args.B * args.H) - group * 8), role = place / wide;
  const int ranked = group * 8 + (place - role * wide), seg = blockIdx.y;
  int b = ranked / args.H;
  const int h = ranked - b * args.H;
  const DecayRole& R = args.role[role];
  const int T_ = args.T;
  int len = T_;
  if (args.order) {  // (every wave for itself)
    const int n = lane < args.B ? min(max(args.lengths[lane], 0), T_) : 0;
    b = dec_ranked(n, ~0ull >> (64 - args.B), b, T_);
    len = __builtin_amdgcn_readlane(n, b);
  } else if (args.lengths) {
    len = min(max(args.lengths[b], 0), T_);
  }
  const int bh = b * args.H + h;
  const int s0 = seg * args.seg_len, s1 = min(s0 + args.seg_len, T_);
  const int end = min(s1, len);  // frames s0..end-1 are computed, end..s1-1 (of the padding) get zeros
  const bool first = s0 == 0, single = args.segments == 1;
  const bool rev = R.reverse != 0;
  // this wave's part of the state: rows srow.., columns scol..; or of the outputs: frames 16 it.., column tiles mo0..
  const int srow = G::KS == 1 ? 0 : (wave >> 1) * KT * 16, scol = G::KS == 1 ? wave * MS * 16 : (wave & 1) * 16;
  const int it = wave % G::WQ, mo0 = wave / G::WQ * MO;

  if (!OUT) {
    // the last segment's copy of the state has a slot of its own: it may be replaced while others still read it
    if (first && args.state) {
      const float* src = args.state + (long)bh * DK * DV;
      float* dst = R.ws + ((long)bh * args.segments + args.segments - 1) * (DK * DV);
      for (int i = tid * 4; i < DK * DV; i += THREADS * 4)
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
  auto krow = [&](int n) { return (tid + n * THREADS) / (DK / VEC); };
  auto kpiece = [&](int n) { return (tid + n * THREADS) % (DK / VEC); };
  auto vrow = [&](int n) { return (tid + n * THREADS) / (DV / VEC); };
  auto vpiece = [&](int n) { return (tid + n * THREADS) % (DV / VEC); };
  auto offset = [&](int row, int p, long ld) {
    return ((unsigned)(rev ? C - 1 - row : row) * (unsigned)ld + (unsigned)(p * VEC)) * (unsigned)sizeof(T);
  };
  unsigned koff[NK], qoff[OUT ? NK : 1], voff[NV];
#pragma unroll
  for (int n = 0; n < NK; ++n) {
    koff[n] = offset(krow(n), kpiece(n), R.k.ld);
    if (OUT) qoff[n] = offset(krow(n), kpiece(n), R.q.ld);
  }
#pragma unroll
  for (int n = 0; n < NV; ++n) voff[n] = offset(vrow(n), vpiece(n), R.v.ld);
  struct Rows {  // a chunk's pieces on their way from memory
    dec_u4 k[NK], q[OUT ? NK : 1], v[NV];
  };
  auto fetch = [&](int t0, Rows& f) {
    const long low = rev ? len - t0 - C : t0;  // (below zero only where the lanes of those rows do not load)
    const char* const ka = kbase + low * R.k.ld * (long)sizeof(T);
    const char* const va = vbase + low * R.v.ld * (long)sizeof(T);
    const char* const qa = OUT ? qbase + low * R.q.ld * (long)sizeof(T) : nullptr;
    const int rows = min(end - t0, C);  // (a thread without a piece of its own has a row behind the chunk)
    if (rows == C && PIECES_K % THREADS == 0 && PIECES_V % THREADS == 0) {
#pragma unroll
      for (int n = 0; n < NK; ++n) {
        f.k[n] = *reinterpret_cast<const dec_u4*>(ka + koff[n]);
        if (OUT) f.q[n] = *reinterpret_cast<const dec_u4*>(qa + qoff[n]);
      }
#pragma unroll
      for (int n = 0; n < NV; ++n) f.v[n] = *reinterpret_cast<const dec_u4*>(va + voff[n]);
    } else {
#pragma unroll
      for (int n = 0; n < NK; ++n) {
        const bool in = krow(n) < rows;
        f.k[n] = dec_u4(0u);
        if (in) f.k[n] = *reinterpret_cast<const dec_u4*>(ka + koff[n]);
        if (OUT) {
          f.q[n] = dec_u4(0u);
          if (in) f.q[n] = *reinterpret_cast<const dec_u4*>(qa + qoff[n]);
        }
      }
#pragma unroll
      for (int n = 0; n < NV; ++n) {
        f.v[n] = dec_u4(0u);
        if (vrow(n) < rows) f.v[n] = *reinterpret_cast<const dec_u4*>(va + voff[n]);
      }
    }
  };
  auto stage = [&](const Rows& f) {
#pragma unroll
    for (int n = 0; n < NK; ++n) {
      if (PIECES_K % THREADS != 0 && krow(n) >= C) continue;
      *reinterpret_cast<dec_u4*>(ktile.piece(krow(n), kpiece(n))) = f.k[n];
      if (OUT) *reinterpret_cast<dec_u4*>(qtile.piece(krow(n), kpiece(n))) = f.q[n];
    }
#pragma unroll
    for (int n = 0; n < NV; ++n) {
      if (PIECES_V % THREADS != 0 && vrow(n) >= C) continue;
      *reinterpret_cast<dec_u4*>(vtile.piece(vrow(n), vpiece(n))) = f.v[n];
    }
  };
  if (OUT) {
    if (tid == 0) odd_any = 0;
    for (int i = tid; i < DV; i += THREADS) odd_from[i] = 0x7fffffff;
  }
  Rows rows;  // one chunk ahead (two ahead measured the same, in twice the registers)

  const float a2 = dec_log2(args.log_decay[h]);
  auto upow = [&](int n) { return dec_uniform(dec_pow(a2, n)); };
  // A chunk's tiles: staged once everybody has finished with the previous ones, `hand_over` by the waves of the state.  The two
  // kinds of waves run loops of their own (each keeps its own values in registers) that meet at the same barriers.
  auto begin = [&](int t0, auto hand_over) {
    __syncthreads();
    stage(rows);
    hand_over();
    __syncthreads();
    if (t0 + C < end) fetch(t0 + C, rows);
  };

  if (s0 < end) fetch(s0, rows);
  if (!holds) {
    float wdiag[4], woff[4];  // lambda^(i-j) inside a tile, and 16 more: tile by tile times a uniform power
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int d = l16 - (4 * g + r);
      wdiag[r] = dec_pow(a2, max(d, 0));
      woff[r] = dec_pow(a2, 16 + d);
    }
    const float fq = dec_pow(a2, 16 * it + l16 + 1);
    T* const op = (T*)R.out.p + (long)b * R.out.bs + (long)h * DV + 16 * mo0 + 4 * g;
    for (int t0 = s0; t0 < end; t0 += C) {
      begin(t0, [] {});
      if (t0 + 16 * it >= end) continue;
      Frag qx[KB];
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) qx[kb] = qtile.row_frag(16 * it + l16, kb, g);
      // The products carry an infinity or a NaN in v to the frames before it, too (zero times infinity).  A wave that finds such
      // an output puts zeros in their place in the tile, notes from where on their columns are NaN (these are written at the
      // end) and computes the chunk once more.  What another wave reads meanwhile does not matter: its outputs are finite, or it
      // does the same, and the state's column is one of those noted.
      dec_f4 o[MO];
      for (bool again = false;; again = true) {
#pragma unroll
        for (int i = 0; i < MO; ++i) o[i] = dec_f4(0.f);
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
#pragma unroll
          for (int i = 0; i < (G::STERMS == 2 ? MO : 0); ++i) o[i] = dec_mma(srest.row_frag(16 * (mo0 + i) + l16, kb, g), qx[kb], o[i]);
#pragma unroll
          for (int i = 0; i < MO; ++i) o[i] = dec_mma(stile.row_frag(16 * (mo0 + i) + l16, kb, g), qx[kb], o[i]);
        }
#pragma unroll
        for (int i = 0; i < MO; ++i) o[i] *= fq;
#pragma unroll 1
        for (int jb = 0; jb <= it >> 1; ++jb) {
          dec_f4 p[2];
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const int jt = 2 * jb + x;
            p[x] = dec_f4(0.f);
            if (jt > it) continue;
#pragma unroll
            for (int kb = 0; kb < KB; ++kb) p[x] = dec_mma(ktile.row_frag(16 * jt + l16, kb, g), qx[kb], p[x]);
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
          if constexpr (sizeof(T) == 2) {
            Frag low, vx[MO];
            dec_rest(low, pf, p[0], p[1]);
#pragma unroll
            for (int i = 0; i < MO; ++i) o[i] = dec_mma(vx[i] = vtile.col_frag(32 * jb, 16 * (mo0 + i), l16, g), low, o[i]);
#pragma unroll
            for (int i = 0; i < MO; ++i) o[i] = dec_mma(vx[i], pf, o[i]);
          } else {
#pragma unroll
            for (int i = 0; i < MO; ++i) o[i] = dec_mma(vtile.col_frag(32 * jb, 16 * (mo0 + i), l16, g), pf, o[i]);
          }
        }
        dec_f4 odd = dec_f4(0.f);
#pragma unroll
        for (int i = 0; i < MO; ++i)
#pragma unroll
          for (int r = 0; r < 4; ++r) odd[r] = fmaf(o[i][r], 0.f, odd[r]);
        if (again || __builtin_expect(!__any((odd[0] + odd[1]) + (odd[2] + odd[3]) != 0.f), 1)) break;
#pragma unroll 1
        for (int e = lane; e < C * DV; e += 64) {
          T* const v = vtile.piece(e / DV, e % DV / VEC) + e % VEC;
          if (__builtin_isfinite((float)*v)) continue;
          *v = (T)0.f;
          atomicMin(&odd_from[e % DV], t0 + e / DV);
          odd_any = 1;
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
      }
      const int t = t0 + 16 * it + l16;
      if (t < end) {
        T* const dst = op + (long)(rev ? len - 1 - t : t) * R.out.ld;
#pragma unroll
        for (int i = 0; i < MO; ++i) dec_store4(dst + 16 * i, o[i] * args.scale);
      }
    }
    __syncthreads();
  } else {
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
      // sum over s' < seg of lambda^((seg-1-s') seg_len) E_s' of the states E at the ends of the segments before; where there
      // are many, k_decay_join has summed them
      const float lamL = upow(args.seg_len);
      float w = 1.f;
      const int from = args.joined ? seg - 1 : 0;
      for (int s = seg - 1; s >= from; --s, w *= lamL) {
        const dec_f4* e = reinterpret_cast<const dec_f4*>(R.ws + ((long)bh * args.segments + s) * (DK * DV)) + wplace;
#pragma unroll
        for (int t = 0; t < KT; ++t)
#pragma unroll
          for (int m = 0; m < MS; ++m) S[t][m] += w * e[(t * MS + m) * 64];
      }
    }

    float wend[4];  // lambda^(15-j) inside a tile
#pragma unroll
    for (int r = 0; r < 4; ++r) wend[r] = dec_pow(a2, 15 - (4 * g + r));
    for (int t0 = s0; t0 < end; t0 += C) {
      const int n = min(C, end - t0);  // frames of this chunk
      // the state's copy, rounded before the barrier (between the two there is only its way to LDS)
      constexpr bool TWO = OUT && G::STERMS == 2;
      dec_b4 copy[TWO ? KT : 1][MS], rest[TWO ? KT : 1][MS];
      if constexpr (TWO) {
#pragma unroll
        for (int t = 0; t < KT; ++t)
#pragma unroll
          for (int m = 0; m < MS; ++m)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              copy[t][m][r] = (__bf16)S[t][m][r];
              rest[t][m][r] = (__bf16)(S[t][m][r] - (float)copy[t][m][r]);
            }
      }
      begin(t0, [&] {
#pragma unroll
        for (int t = 0; t < (OUT ? KT : 0); ++t)
#pragma unroll
          for (int m = 0; m < MS; ++m) {
            const int row = scol + 16 * m + l16, c = srow + 16 * t + 4 * g;
            if constexpr (TWO) {
              *reinterpret_cast<dec_b4*>(stile.four(row, c)) = copy[t][m];
              *reinterpret_cast<dec_b4*>(srest.four(row, c)) = rest[t][m];
            } else {
              dec_store4(stile.four(row, c), S[t][m]);
            }
          }
      });
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
          const Frag vx = vtile.col_frag(32 * jb, scol + 16 * m, l16, g);
          if constexpr (sizeof(T) == 2) {
            dec_split<TERMS>(vx, w, wv[m]);
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) wv[m][0].a[e] = vx.a[e] * w[e], wv[m][0].b[e] = vx.b[e] * w[4 + e];
          }
        }
#pragma unroll
        for (int t = 0; t < KT; ++t) {
          const Frag kx = ktile.col_frag(32 * jb, srow + 16 * t, l16, g);
#pragma unroll
          for (int m = 0; m < MS; ++m)
#pragma unroll
            for (int x = (sizeof(T) == 2 ? TERMS : 1) - 1; x >= 0; --x) S[t][m] = dec_mma(kx, wv[m][x], S[t][m]);
        }
      }
    }

    if (OUT) __syncthreads();
    if (!OUT) {
      dec_f4* e = reinterpret_cast<dec_f4*>(R.ws + ((long)bh * args.segments + seg) * (DK * DV)) + wplace;
#pragma unroll
      for (int t = 0; t < KT; ++t)
#pragma unroll
        for (int m = 0; m < MS; ++m) e[(t * MS + m) * 64] = S[t][m];
    } else if (args.state && s0 < len && s1 >= len) {
      // the final state, by the segment that holds the last frame (an empty utterance keeps what it had)
      float* sp = args.state + (long)bh * DK * DV + splace;
#pragma unroll
      for (int t = 0; t < KT; ++t)
#pragma unroll
        for (int m = 0; m < MS; ++m)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            sp[(16 * t + r) * DV + 16 * m] = odd_from[scol + 16 * m + l16] < end ? __builtin_nanf("") : S[t][m][r];
    }
  }
  if (!OUT) return;
  if (odd_any) {
    for (int i = tid; i < (end - s0) * DV; i += THREADS) {
      const int t = s0 + i / DV, c = i % DV;
      if (t >= odd_from[c])
        ((T*)R.out.p)[(long)b * R.out.bs + (long)(rev ? len - 1 - t : t) * R.out.ld + (long)h * DV + c] = (T)__builtin_nanf("");
    }
  }
  // zeros behind the utterance's end
  for (int i = max(s0, len) * (DV / VEC) + tid; i < s1 * (DV / VEC); i += THREADS) {
    const int t = i / (DV / VEC), c = (i % (DV / VEC)) * VEC;
    *reinterpret_cast<dec_u4*>((T*)R.out.p + (long)b * R.out.bs + (long)t * R.out.ld + (long)h * DV + c) = dec_u4(0u);
  }
}

// The states at the ends of the segments (decay.hip): E_s becomes sum over s' <= s of lambda^((s-s') seg_len) E_s'.
int decay_launch_join(const DecayArgs& a, int roles, int state_elements, hipStream_t st);

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
    hipLaunchKernelGGL((k_decay<T, DK, DV, false, TERMS>), dim3(a.B * a.H * a.roles, a.segments - 1), dim3(256),
                       G::kLdsState, st, a);
    if (a.joined && decay_launch_join(a, roles, DK * DV, st)) return 1;
  }
  {
    ProfScope ps("k_decay", st);
    hipLaunchKernelGGL((k_decay<T, DK, DV, true, TERMS>), dim3(a.B * a.H * a.roles, a.segments), dim3(512), G::kLdsOut,
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
