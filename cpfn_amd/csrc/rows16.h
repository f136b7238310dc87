// 16-byte pieces of rows of fp32 / bf16 / fp16 values, computed on in fp32, for kernels whose rows may have any length and start
// anywhere (norms, routed rows, gradient lists).  The vector types carry the ELEMENT's alignment: the compiler still emits one
// 16-byte access (the target reads and writes global memory at any alignment), so that an odd number of channels, a slice of a
// buffer or a parameter inside a flat buffer takes the same path as an aligned tensor.
//
// Figures in the comments of these kernels: "measured" are kernel durations of a trace (profiles/block_operators_kernels.txt); "a -> b" and
// other comparisons of two choices are calls in a row between two events, which hold the launches' gaps too, in one run of both sides.
#pragma once
#include "common.h"

struct cpfn_bf16 { unsigned short bits; };
struct cpfn_f16 { _Float16 v; };

__device__ __forceinline__ float cpfn_to_f32(float v) { return v; }
__device__ __forceinline__ float cpfn_to_f32(cpfn_bf16 v) { return __uint_as_float((unsigned)v.bits << 16); }
__device__ __forceinline__ float cpfn_to_f32(cpfn_f16 v) { return (float)v.v; }
template <typename T> __device__ __forceinline__ T cpfn_from_f32(float v);
template <> __device__ __forceinline__ float cpfn_from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ cpfn_bf16 cpfn_from_f32<cpfn_bf16>(float v) {       // nearest, ties to even
  return cpfn_bf16{__builtin_bit_cast(unsigned short, (__bf16)v)};
}
template <> __device__ __forceinline__ cpfn_f16 cpfn_from_f32<cpfn_f16>(float v) { return cpfn_f16{(_Float16)v}; }

template <typename T> struct cpfn_piece;                 // one 16-byte access: N elements
template <> struct cpfn_piece<float> {
  enum { N = 4 };
  typedef float vec __attribute__((ext_vector_type(4), aligned(4)));
};
template <> struct cpfn_piece<cpfn_bf16> {
  enum { N = 8 };
  typedef unsigned vec __attribute__((ext_vector_type(4), aligned(2)));
};
template <> struct cpfn_piece<cpfn_f16> {
  enum { N = 8 };
  typedef unsigned vec __attribute__((ext_vector_type(4), aligned(2)));
};

// raw 16 bytes <-> N floats (no dynamically indexed arrays: everything below is unrolled)
__device__ __forceinline__ void cpfn_unpack(const cpfn_piece<float>::vec &r, float *f, float *) {
  f[0] = r.x; f[1] = r.y; f[2] = r.z; f[3] = r.w;
}
template <typename T> __device__ __forceinline__ float cpfn_half_lo(unsigned u);                // a word's two 16-bit elements
template <typename T> __device__ __forceinline__ float cpfn_half_hi(unsigned u);
template <> __device__ __forceinline__ float cpfn_half_lo<cpfn_bf16>(unsigned u) { return __uint_as_float(u << 16); }
template <> __device__ __forceinline__ float cpfn_half_hi<cpfn_bf16>(unsigned u) { return __uint_as_float(u & 0xffff0000u); }
template <> __device__ __forceinline__ float cpfn_half_lo<cpfn_f16>(unsigned u) { return (float)__builtin_bit_cast(_Float16, (unsigned short)u); }
template <> __device__ __forceinline__ float cpfn_half_hi<cpfn_f16>(unsigned u) { return (float)__builtin_bit_cast(_Float16, (unsigned short)(u >> 16)); }
template <> __device__ __forceinline__ float cpfn_half_lo<float>(unsigned u) { return 0.f; }    // (never called)
template <> __device__ __forceinline__ float cpfn_half_hi<float>(unsigned u) { return 0.f; }
__device__ __forceinline__ void cpfn_unpack(const cpfn_piece<cpfn_bf16>::vec &r, float *f, cpfn_bf16 *) {
  const unsigned u[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) { f[2 * i] = cpfn_half_lo<cpfn_bf16>(u[i]); f[2 * i + 1] = cpfn_half_hi<cpfn_bf16>(u[i]); }
}
__device__ __forceinline__ void cpfn_unpack(const cpfn_piece<cpfn_f16>::vec &r, float *f, cpfn_f16 *) {
  const unsigned u[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) { f[2 * i] = cpfn_half_lo<cpfn_f16>(u[i]); f[2 * i + 1] = cpfn_half_hi<cpfn_f16>(u[i]); }
}
__device__ __forceinline__ cpfn_piece<float>::vec cpfn_pack(const float *f, float *) {
  cpfn_piece<float>::vec r;
  r.x = f[0]; r.y = f[1]; r.z = f[2]; r.w = f[3];
  return r;
}
typedef float cpfn_f32x2_ __attribute__((ext_vector_type(2)));
typedef __bf16 cpfn_bf16x2_ __attribute__((ext_vector_type(2)));
typedef _Float16 cpfn_f16x2_ __attribute__((ext_vector_type(2)));
template <typename T> __device__ __forceinline__ unsigned cpfn_pair16(float lo, float hi);      // two roundings, one instruction (bf16)
template <> __device__ __forceinline__ unsigned cpfn_pair16<cpfn_bf16>(float lo, float hi) {
  const cpfn_f32x2_ v = {lo, hi};
  return __builtin_bit_cast(unsigned, __builtin_convertvector(v, cpfn_bf16x2_));
}
template <> __device__ __forceinline__ unsigned cpfn_pair16<cpfn_f16>(float lo, float hi) {
  const cpfn_f32x2_ v = {lo, hi};
  return __builtin_bit_cast(unsigned, __builtin_convertvector(v, cpfn_f16x2_));
}
template <typename T> __device__ __forceinline__ typename cpfn_piece<T>::vec cpfn_pack16(const float *f) {
  typename cpfn_piece<T>::vec r;
  r.x = cpfn_pair16<T>(f[0], f[1]);
  r.y = cpfn_pair16<T>(f[2], f[3]);
  r.z = cpfn_pair16<T>(f[4], f[5]);
  r.w = cpfn_pair16<T>(f[6], f[7]);
  return r;
}
__device__ __forceinline__ cpfn_piece<cpfn_bf16>::vec cpfn_pack(const float *f, cpfn_bf16 *) { return cpfn_pack16<cpfn_bf16>(f); }
__device__ __forceinline__ cpfn_piece<cpfn_f16>::vec cpfn_pack(const float *f, cpfn_f16 *) { return cpfn_pack16<cpfn_f16>(f); }

// piece at element `at` of a row of C elements that starts at p: whole, or element by element where the row ends inside it
// (values behind the end: zero, never read; never written)
template <typename T> __device__ __forceinline__ typename cpfn_piece<T>::vec cpfn_load_piece(const T *__restrict__ p, int at, int C) {
  typedef typename cpfn_piece<T>::vec V;
  constexpr int N = cpfn_piece<T>::N;
  V r = {};
  if (at + N <= C) {
    r = *(const V *)(p + at);
  } else if (at < C) {
    float f[N];
#pragma unroll
    for (int i = 0; i < N; ++i) f[i] = at + i < C ? cpfn_to_f32(p[at + i]) : 0.f;
    r = cpfn_pack(f, (T *)nullptr);                      // (exact: the values come from T)
  }
  return r;
}
// (a vector's element goes through a value: __builtin_bit_cast of the element itself reads element 0 with this compiler)
__device__ __forceinline__ unsigned cpfn_word(float v) { return __float_as_uint(v); }
__device__ __forceinline__ unsigned cpfn_word(unsigned v) { return v; }
// 16 bytes, or the first C % N elements of them in one to three stores (which ones is the same for a whole launch)
template <typename T> __device__ __forceinline__ void cpfn_store_piece(T *__restrict__ p, int at, int C, const float *f) {
  typedef typename cpfn_piece<T>::vec V;
  constexpr int N = cpfn_piece<T>::N;
  const V v = cpfn_pack(f, (T *)nullptr);
  if (at + N <= C) {
    *(V *)(p + at) = v;
  } else if (at < C) {
    typedef unsigned two __attribute__((ext_vector_type(2), aligned(2)));
    typedef unsigned one __attribute__((aligned(2)));
    const unsigned w[4] = {cpfn_word(v.x), cpfn_word(v.y), cpfn_word(v.z), cpfn_word(v.w)};
    char *o = (char *)(p + at);
    const int bytes = (C % N) * (int)sizeof(T);
    if (bytes & 8) {
      *(two *)o = two{w[0], w[1]};
      if (bytes & 4) {
        *(one *)(o + 8) = w[2];
        if (bytes & 2) *(unsigned short *)(o + 12) = (unsigned short)w[3];
      } else if (bytes & 2) {
        *(unsigned short *)(o + 8) = (unsigned short)w[2];
      }
    } else if (bytes & 4) {
      *(one *)o = w[0];
      if (bytes & 2) *(unsigned short *)(o + 4) = (unsigned short)w[1];
    } else if (bytes & 2) {
      *(unsigned short *)o = (unsigned short)w[0];
    }
  }
}

// Sum over groups of L consecutive lanes (L a power of two, <= 64), the same value in every lane of the group: pairs, quads,
// eights and sixteens by DPP, the halves of 32 and of 64 by lane swaps — no LDS traffic, ~6 instructions for a whole wave.
template <int CTRL> __device__ __forceinline__ float cpfn_dpp(float v) {
  return __uint_as_float((unsigned)__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(v), CTRL, 0xf, 0xf, false));
}
template <int L> __device__ __forceinline__ float cpfn_lanes_sum(float v) {
  if (L >= 2) v += cpfn_dpp<0xB1>(v);                    // quad_perm 1,0,3,2
  if (L >= 4) v += cpfn_dpp<0x4E>(v);                    // quad_perm 2,3,0,1
  if (L >= 8) v += cpfn_dpp<0x141>(v);                   // row_half_mirror
  if (L >= 16) v += cpfn_dpp<0x140>(v);                  // row_mirror
  if (L >= 32) {
    const auto s = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(s[0]) + __uint_as_float(s[1]);
  }
  if (L >= 64) {
    const auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(s[0]) + __uint_as_float(s[1]);
  }
  return v;
}
