// What the forward and the backward kernel of the residual block's norms share (rownorm_fwd.hip, rownorm_bwd.hip).
//
//   n(v; w, b) = (v - mu) r w + b,   r = 1 / sqrt(mean((v - mu)^2) + eps),   mu = mean(v) (layer) or 0 (rms), over the C channels
//   u = n(y; weight, bias)  (y itself without a weight),   a = gate | sigmoid(gate) | 1
//   out = x + scale a u   (x itself without y),            normed = n(out; next_weight, next_bias)
//
// A row is held by L lanes, eight channels each, from its one load to its one store: L = 8 .. 64 lanes inside a wave (row sums by
// DPP and lane swaps), 128 .. 512 lanes = several waves (sums through LDS, one barrier each).  All arithmetic is fp32.
#pragma once
#include "rows16.h"

#define CPFN_NORM_MAX_C 4096        // (512 lanes: with 1024 the backward kernel's registers do not fit)

// (rows of several waves have a workgroup of their own: its barriers then wait for nobody else)
template <typename T, int L> struct NormShape {
  enum { THREADS = L <= 64 ? 256 : L, ROWS = THREADS / L, VN = cpfn_piece<T>::N, NP = 8 / VN, WAVES = THREADS / 64 };
};

// channel of element i (0..7) of lane `lane` of its row
template <typename T, int L> __device__ __forceinline__ int norm_col(int lane, int i) {
  constexpr int VN = cpfn_piece<T>::N;
  return ((i / VN) * L + lane) * VN + i % VN;
}

template <typename T, int L> struct RowRaw { typename cpfn_piece<T>::vec p[8 / cpfn_piece<T>::N]; };

// RAGGED: C is no multiple of a piece; `mask`: what of this lane's pieces lies in the row
template <typename T, int L, bool RAGGED> __device__ __forceinline__ RowRaw<T, L> row_mask(int lane, int C) {
  RowRaw<T, L> m;
#pragma unroll
  for (int q = 0; q < 8 / cpfn_piece<T>::N; ++q) {
    if (RAGGED) m.p[q] = cpfn_piece_mask<T>(C - (q * L + lane) * cpfn_piece<T>::N);
    else m.p[q] = {};
  }
  return m;
}
// row r of P rows
template <typename T, int L, bool RAGGED>
__device__ __forceinline__ void row_load(RowRaw<T, L> &raw, const T *__restrict__ base, long long r, long long P, int lane, int C, const RowRaw<T, L> &mask) {
  const T *__restrict__ row = base + r * C;
#pragma unroll
  for (int q = 0; q < 8 / cpfn_piece<T>::N; ++q) {
    const int at = (q * L + lane) * cpfn_piece<T>::N;
    if (RAGGED) raw.p[q] = cpfn_load_ragged(row, at, C, (P - r) * C, mask.p[q]);
    else if (at < C) raw.p[q] = *(const typename cpfn_piece<T>::vec *)(row + at);
    else raw.p[q] = {};
  }
}
template <typename T, int L> __device__ __forceinline__ void row_zero(RowRaw<T, L> &raw) {
#pragma unroll
  for (int q = 0; q < 8 / cpfn_piece<T>::N; ++q) raw.p[q] = {};
}
template <typename T, int L> __device__ __forceinline__ void row_unpack(const RowRaw<T, L> &raw, float *f) {
#pragma unroll
  for (int q = 0; q < 8 / cpfn_piece<T>::N; ++q) cpfn_unpack(raw.p[q], f + q * cpfn_piece<T>::N, (T *)nullptr);
}
template <typename T, int L, bool RAGGED> __device__ __forceinline__ void row_store(T *__restrict__ row, int lane, int C, const float *f) {
#pragma unroll
  for (int q = 0; q < 8 / cpfn_piece<T>::N; ++q) {
    const int at = (q * L + lane) * cpfn_piece<T>::N;
    if (RAGGED) cpfn_store_piece(row, at, C, f + q * cpfn_piece<T>::N);
    else if (at < C) *(typename cpfn_piece<T>::vec *)(row + at) = cpfn_pack(f + q * cpfn_piece<T>::N, (T *)nullptr);
  }
}
// a parameter vector (fp32, any 4-byte alignment: parameters live inside a flat buffer), `fill` where there is none
template <typename T, int L> __device__ __forceinline__ void param_load(float *f, const float *__restrict__ p, int lane, int C, float fill) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int c = norm_col<T, L>(lane, i);
    f[i] = p ? (c < C ? p[c] : 0.f) : fill;
  }
}

// Sums of two values over a row's lanes.  L > 64: the waves of a row exchange their sums through LDS; the two halves of `slots`
// take turns, so one barrier per call is enough (a half is rewritten only behind the NEXT call's barrier).
template <int L> __device__ __forceinline__ void row_sum2(float &a, float &b, float2 *slots, int &turn) {
  constexpr int LW = L < 64 ? L : 64;
  a = cpfn_lanes_sum<LW>(a);
  b = cpfn_lanes_sum<LW>(b);
  if (L > 64) {
    constexpr int W = L / 64;
    const int wave = threadIdx.x >> 6;
    float2 *s = slots + turn * 16;
    turn ^= 1;
    if ((threadIdx.x & 63) == 0) s[wave] = make_float2(a, b);
    __syncthreads();
    a = 0.f; b = 0.f;
#pragma unroll
    for (int i = 0; i < W; ++i) {
      const float2 v = s[(wave & ~(W - 1)) + i];
      a += v.x; b += v.y;
    }
  }
}
template <int L> __device__ __forceinline__ float row_sum(float a, float2 *slots, int &turn) {
  float z = 0.f;
  row_sum2<L>(a, z, slots, turn);
  return a;
}

// v -> its normalised form (v - mu) r; returns r.  Two passes over the registers for `layer` (mean, then centred squares): no
// cancellation.  Channels behind C hold zero and stay out of the centred squares; a row slot without a row is called with a positive
// eps, so that its zeros stay zeros.
template <typename T, int L, bool RAGGED>
__device__ __forceinline__ float row_normalise(float *v, int lane, int C, float inv_c, bool layer, float eps, float2 *slots, int &turn) {
  if (layer) {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) s += v[i];
    const float mu = row_sum<L>(s, slots, turn) * inv_c;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = norm_col<T, L>(lane, RAGGED ? i : i & -cpfn_piece<T>::N) < C ? v[i] - mu : 0.f;
  }
  float q = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) q = fmaf(v[i], v[i], q);
  const float r = rsqrtf(fmaf(row_sum<L>(q, slots, turn), inv_c, eps));
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] *= r;
  return r;
}

// 1 / (1 + exp(-v)).  fp32 rows: exp within 2 units in the last place.  16-bit rows: exp2(-v log2 e) with the product rounded, off by
// |v| 2^-24 relative on top (2^-18 at |v| = 64; the results are rounded to 2^-9), a third of the instructions.
template <typename T> __device__ __forceinline__ float norm_sigmoid(float v) {
  return __builtin_amdgcn_rcpf(1.f + (sizeof(T) == 4 ? expf(-v) : __builtin_amdgcn_exp2f(v * -1.44269504f)));
}

// the gate's row for row r (a 64-bit division only where 32 bits do not hold the rows)
__device__ __forceinline__ long long norm_gate_row(long long r, long long rows_per_gate, long long P) {
  if (rows_per_gate == 1) return r;
  if (P <= 0xffffffffll) return (unsigned)r / (unsigned)rows_per_gate;
  return r / rows_per_gate;
}

// the number of lanes for a row of C channels
static inline int norm_lanes(int C) {
  int L = 8;
  while (L * 8 < C) L *= 2;
  return L;
}
