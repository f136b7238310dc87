// What the forward and the backward kernel of the residual block's norms share (rownorm_fwd.hip, rownorm_bwd.hip).
//
//   n(v; w, b) = (v - mu) r w + b,   r = 1 / sqrt(mean((v - mu)^2) + eps),   mu = mean(v) (layer) or 0 (rms), over the C channels
//   u = n(y; weight, bias)  (y itself without a weight),   a = gate | sigmoid(gate) | 1
//   out = x + scale a u   (x itself without y),            normed = n(out; next_weight, next_bias)
//
// A row is held by L lanes, W = 8 channels each (or 16), from its one load to its one store: L = 8 .. 64 lanes inside a wave (row sums by
// DPP and lane swaps), 128 .. 512 lanes = several waves (sums through LDS, one barrier each).  All arithmetic is fp32.
//
// Loads run one row set ahead of the arithmetic, and no branch stands around a load or a store: then the compiler can count what is
// in flight and waits for the one row set it needs, not for everything.  What a row, a tensor or a lane does not have is expressed in
// the buffer descriptors and offsets instead: a load outside a descriptor's bytes gives zero, a store outside is dropped.
#pragma once
#include "rows16.h"

#define CPFN_NORM_MAX_C 4096        // (512 lanes: with 1024 the backward kernel's registers do not fit)

// How the 16-byte pieces of a row lie: WHOLE: C is a multiple of a piece; RAGGED: the last piece of a row reaches into the next one;
// EACH: element by element (the whole tensor is smaller than a piece)
enum NormMode { WHOLE, RAGGED, EACH };

// What a launch has to do.  ANY: whatever pointers it is given, asked for step by step.  The whole block (y, its norm and the next norm)
// has kernels of its own, without those branches, and without the registers of a gate where rows share one or there is none (BLOCK).
// FRONT: no y (backward only; the forward kernel is as fast with its branches).
enum NormForm { ANY, BLOCK, BLOCK_OWN, FRONT };

// (rows of several waves have a workgroup of their own: its barriers then wait for nobody else)
template <typename T, int L, int W> struct NormShape {
  enum { THREADS = L <= 64 ? 256 : L, ROWS = THREADS / L, VN = cpfn_piece<T>::N, NP = W / VN };
};

// channel of element i (0..W-1) of lane `lane` of its row
template <typename T, int L, int W> __device__ __forceinline__ int norm_col(int lane, int i) {
  constexpr int VN = cpfn_piece<T>::N;
  return ((i / VN) * L + lane) * VN + i % VN;
}

typedef unsigned cpfn_u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned cpfn_u32x2 __attribute__((ext_vector_type(2)));

template <typename T, int L, int W> struct RowRaw { cpfn_u32x4 p[W / cpfn_piece<T>::N]; };

template <typename T, int L, int W> __device__ __forceinline__ void row_unpack(const RowRaw<T, L, W> &raw, float *f) {
#pragma unroll
  for (int q = 0; q < W / cpfn_piece<T>::N; ++q) {
    const unsigned u[4] = {raw.p[q].x, raw.p[q].y, raw.p[q].z, raw.p[q].w};
    float *o = f + q * cpfn_piece<T>::N;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (sizeof(T) == 4) {
        o[i] = __uint_as_float(u[i]);
      } else {
        o[2 * i] = cpfn_half_lo<T>(u[i]);
        o[2 * i + 1] = cpfn_half_hi<T>(u[i]);
      }
    }
  }
}
template <typename T> __device__ __forceinline__ cpfn_u32x4 piece_pack(const float *f) {
  cpfn_u32x4 r;
  if constexpr (sizeof(T) == 4) {
    r.x = __float_as_uint(f[0]); r.y = __float_as_uint(f[1]); r.z = __float_as_uint(f[2]); r.w = __float_as_uint(f[3]);
  } else {
    r.x = cpfn_pair16<T>(f[0], f[1]); r.y = cpfn_pair16<T>(f[2], f[3]); r.z = cpfn_pair16<T>(f[4], f[5]); r.w = cpfn_pair16<T>(f[6], f[7]);
  }
  return r;
}

// Where a lane finds its pieces in a chunk of rows [row0, row1) of tensors [P, C].  Offsets are bytes from the chunk's start.
constexpr unsigned OUTSIDE = 0xC0000000u;            // (chunks stay below 2^30 bytes: every step from here is outside too)
template <typename T, int L, int W, NormMode MODE> struct RowChunk {
  static constexpr int VN = cpfn_piece<T>::N, NP = W / VN;
  int lane, C;
  long long row0, row1, P;
  unsigned off[NP];                  // first row set
  unsigned bytes;                    // of the chunk
  // RAGGED: the descriptor of a load reaches 16 bytes behind the chunk where the tensor does (the last row's last piece), and begins
  // `back` bytes in front of it where fewer than 16 bytes are left; a piece that would pass the tensor's end starts at `limit` instead
  // and is shifted down when it is used
  unsigned back, limit, load_bytes;
  cpfn_u32x4 mask[MODE == RAGGED && sizeof(T) == 2 ? NP : 1];      // 16-bit rows; fp32 rows compare (four registers less a piece)
  unsigned tail[MODE == RAGGED ? NP : 1];              // offset of the row's last, partial piece (OUTSIDE elsewhere), for stores

  __device__ __forceinline__ void begin(long long r0, long long r1, long long P_, int C_, int lane_, int slot) {
    lane = lane_; C = C_; P = P_; row0 = r0; row1 = r1;
    bytes = (unsigned)((r1 - r0) * C * (long long)sizeof(T));
#pragma unroll
    for (int q = 0; q < NP; ++q) {
      const int at = (q * L + lane) * VN;
      const unsigned here = (unsigned)(slot * C + at) * (unsigned)sizeof(T);
      if (MODE == RAGGED) {
        off[q] = at + VN <= C ? here : OUTSIDE;          // whole pieces (stores)
        tail[q] = at < C && at + VN > C ? here : OUTSIDE;
        if (sizeof(T) == 2) {
          const int n = C - at;
          unsigned m[4];
#pragma unroll
          for (int w = 0; w < 4; ++w) m[w] = n >= 2 * w + 2 ? 0xffffffffu : n == 2 * w + 1 ? 0xffffu : 0u;
          mask[q] = cpfn_u32x4{m[0], m[1], m[2], m[3]};
        }
      } else {
        off[q] = at < C ? here : OUTSIDE;
      }
    }
    if (MODE == RAGGED) {
      const long long left = (P - r0) * C * (long long)sizeof(T);
      back = left < 16 ? 16u - (unsigned)left : 0u;
      load_bytes = left < (long long)bytes + 16 ? (unsigned)left + back : bytes + 16u;
      limit = load_bytes - 16u;
    }
  }

  __device__ __forceinline__ __amdgpu_buffer_rsrc_t source(const T *p) const {
    const char *at = (const char *)p + row0 * C * (long long)sizeof(T);
    if (MODE == RAGGED) return __builtin_amdgcn_make_buffer_rsrc((void *)(at - back), 0, p ? (int)load_bytes : 0, 0x00020000);
    return __builtin_amdgcn_make_buffer_rsrc((void *)at, 0, p ? (int)bytes : 0, 0x00020000);
  }
  __device__ __forceinline__ __amdgpu_buffer_rsrc_t target(T *p) const {
    return __builtin_amdgcn_make_buffer_rsrc((void *)((char *)p + row0 * C * (long long)sizeof(T)), 0, p ? (int)bytes : 0, 0x00020000);
  }

  // the offsets of a row set `step` bytes behind the first one (there: the row belongs to the chunk); RAGGED: `shift` takes by how many
  // bytes each piece has to be moved down
  __device__ __forceinline__ void at(unsigned *o, unsigned *shift, unsigned step, bool there) const {
#pragma unroll
    for (int q = 0; q < NP; ++q) {
      if (MODE == RAGGED) {
        const unsigned first = tail[q] == OUTSIDE ? off[q] : tail[q];
        o[q] = first == OUTSIDE || !there ? OUTSIDE : first + step + back;
        const unsigned over = o[q] - limit;
        shift[q] = over - 1u < 15u ? over : 0u;
        o[q] -= shift[q];
      } else {
        o[q] = off[q] + step;
      }
    }
  }
  // STREAM: the values are not kept in the caches (the last reader of whole rows; ragged rows share their cache lines)
  template <bool STREAM = false> __device__ __forceinline__ void load(RowRaw<T, L, W> &raw, __amdgpu_buffer_rsrc_t rs, const unsigned *o) const {
#pragma unroll
    for (int q = 0; q < NP; ++q) raw.p[q] = __builtin_amdgcn_raw_buffer_load_b128(rs, o[q], 0, STREAM && MODE == WHOLE ? 2 : 0);
  }
  // what was loaded -> the row's values, zero behind its end
  __device__ __forceinline__ void settle(RowRaw<T, L, W> &raw, const unsigned *shift) const {
    if (MODE != RAGGED) return;
#pragma unroll
    for (int q = 0; q < NP; ++q) {
      if (shift[q]) {                                    // (the last piece of the tensor, once in a launch)
        unsigned w[4] = {raw.p[q].x, raw.p[q].y, raw.p[q].z, raw.p[q].w};
        for (unsigned n = shift[q]; n >= 4; n -= 4) { w[0] = w[1]; w[1] = w[2]; w[2] = w[3]; w[3] = 0u; }
        if (shift[q] & 2) { w[0] = w[0] >> 16 | w[1] << 16; w[1] = w[1] >> 16 | w[2] << 16; w[2] = w[2] >> 16 | w[3] << 16; w[3] >>= 16; }
        raw.p[q] = cpfn_u32x4{w[0], w[1], w[2], w[3]};
      }
      if (sizeof(T) == 2) {
        raw.p[q] &= mask[q];
      } else {
        const int n = C - (q * L + lane) * VN;
        raw.p[q] = cpfn_u32x4{n > 0 ? raw.p[q].x : 0u, n > 1 ? raw.p[q].y : 0u, n > 2 ? raw.p[q].z : 0u, n > 3 ? raw.p[q].w : 0u};
      }
    }
  }
  __device__ __forceinline__ void store(__amdgpu_buffer_rsrc_t rs, unsigned step, const float *f) const {
#pragma unroll
    for (int q = 0; q < NP; ++q) {
      const cpfn_u32x4 v = piece_pack<T>(f + q * VN);
      __builtin_amdgcn_raw_buffer_store_b128(v, rs, off[q] + step, 0, 2);       // (2: non-temporal)
      if (MODE == RAGGED) {                              // 8, 4 and 2 bytes of the partial piece, as C % VN says (the same for all rows)
        const unsigned n = (unsigned)(C % VN) * (unsigned)sizeof(T), t = tail[q] + step;
        const bool b8 = n & 8, b4 = n & 4, b2 = n & 2;
        __builtin_amdgcn_raw_buffer_store_b64(cpfn_u32x2{v.x, v.y}, rs, b8 ? t : OUTSIDE, 0, 0);
        __builtin_amdgcn_raw_buffer_store_b32(b8 ? v.z : v.x, rs, b4 ? t + (b8 ? 8u : 0u) : OUTSIDE, 0, 0);
        if (sizeof(T) == 2) {
          const unsigned last = b8 ? (b4 ? v.w : v.z) : (b4 ? v.y : v.x);
          __builtin_amdgcn_raw_buffer_store_b16((unsigned short)last, rs, b2 ? t + (n & 12u) : OUTSIDE, 0, 0);
        }
      }
    }
  }
};

// EACH: every element an access of its own
template <typename T, int L, int W> __device__ __forceinline__ void each_load(RowRaw<T, L, W> &raw, const T *p, long long r, int lane, int C, bool there) {
  float f[W];
#pragma unroll
  for (int i = 0; i < W; ++i) f[i] = p && there && norm_col<T, L, W>(lane, i) < C ? cpfn_to_f32(p[r * C + norm_col<T, L, W>(lane, i)]) : 0.f;
#pragma unroll
  for (int q = 0; q < W / cpfn_piece<T>::N; ++q) raw.p[q] = piece_pack<T>(f + q * cpfn_piece<T>::N);
}
template <typename T, int L, int W> __device__ __forceinline__ void each_store(T *p, long long r, int lane, int C, bool there, const float *f) {
#pragma unroll
  for (int i = 0; i < W; ++i)
    if (p && there && norm_col<T, L, W>(lane, i) < C) p[r * C + norm_col<T, L, W>(lane, i)] = cpfn_from_f32<T>(f[i]);
}

// one row of a tensor by itself (a gate that a group of rows shares), element by element where its end is not whole
template <typename T, int L, int W> __device__ __forceinline__ void single_load(RowRaw<T, L, W> &raw, const T *__restrict__ row, int lane, int C) {
#pragma unroll
  for (int q = 0; q < W / cpfn_piece<T>::N; ++q) {
    const auto v = cpfn_load_piece(row, (q * L + lane) * cpfn_piece<T>::N, C);
    raw.p[q] = cpfn_u32x4{cpfn_word(v.x), cpfn_word(v.y), cpfn_word(v.z), cpfn_word(v.w)};
  }
}

// A value has arrived where this stands.  In front of a loop: without it every step of the loop waits for whatever was requested last,
// which is the next step's rows.  At the end of a step, on the next step's rows: there the number of stores behind them is known (where
// the loop begins it is not: with or without a step before it), and only the loads are waited for.
template <int W> __device__ __forceinline__ void arrived(float (&f)[W]) {
#pragma unroll
  for (int i = 0; i < W; ++i) asm volatile("" : "+v"(f[i]));
}

template <typename T, int L, int W> __device__ __forceinline__ void arrived(RowRaw<T, L, W> &raw) {
#pragma unroll
  for (int q = 0; q < W / cpfn_piece<T>::N; ++q) asm volatile("" : "+v"(raw.p[q]));
}

// a parameter vector (fp32, any 4-byte alignment: parameters live inside a flat buffer), `fill` where there is none.  16 bytes a load:
// word by word the five vectors cost a launch over 131072 x 128 rows 15 of its 50 us
template <typename T, int L, int W, bool PARTIAL> __device__ __forceinline__ void param_load(float *f, const float *__restrict__ p, int lane, int C, float fill) {
  if (!p) {
#pragma unroll
    for (int i = 0; i < W; ++i) f[i] = fill;
    return;
  }
#pragma unroll
  for (int i = 0; i < W; i += 4) {
    const int c = norm_col<T, L, W>(lane, i);
    cpfn_piece<float>::vec v = {};
    if (c + 4 <= C) {
      v = *(const cpfn_piece<float>::vec *)(p + c);
    } else if (PARTIAL) {
      v.x = c < C ? p[c] : 0.f;
      v.y = c + 1 < C ? p[c + 1] : 0.f;
      v.z = c + 2 < C ? p[c + 2] : 0.f;
    }
    f[i] = v.x; f[i + 1] = v.y; f[i + 2] = v.z; f[i + 3] = v.w;
  }
}

// scale weight and scale bias of a lane's channels: out = x + a (hat scale weight + scale bias)
template <typename T, int L, int W, bool PARTIAL>
__device__ __forceinline__ void block_params(float *sw, float *sb, const float *weight, const float *bias, const float *scale, int lane, int C) {
  float s[W];
  param_load<T, L, W, PARTIAL>(sw, weight, lane, C, 1.f);
  param_load<T, L, W, PARTIAL>(sb, bias, lane, C, 0.f);
  param_load<T, L, W, PARTIAL>(s, scale, lane, C, 1.f);
#pragma unroll
  for (int i = 0; i < W; ++i) { sw[i] *= s[i]; sb[i] *= s[i]; }
}

// What was read is in registers of its own from here on: the next rows are requested into those that it was loaded into (without this
// the compiler requests them first and moves every register).
__device__ __forceinline__ void unpacked() { __builtin_amdgcn_sched_barrier(0); }

// Sums of two values over a row's lanes.  L > 64: the waves of a row exchange their sums through LDS; the two halves of `slots`
// take turns, so one barrier per call is enough (a half is rewritten only behind the NEXT call's barrier).  The fences are for LDS
// alone: loads and stores of rows stay in flight across the barrier.
template <int L> __device__ __forceinline__ void row_sum2(float &a, float &b, float2 *slots, int &turn) {
  constexpr int LW = L < 64 ? L : 64;
  a = cpfn_lanes_sum<LW>(a);
  b = cpfn_lanes_sum<LW>(b);
  if (L > 64) {
    constexpr int WAVES = L / 64;
    const int wave = threadIdx.x >> 6;
    float2 *s = slots + turn * WAVES;
    turn ^= 1;
    if ((threadIdx.x & 63) == 0) s[wave] = make_float2(a, b);
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
    a = 0.f; b = 0.f;
#pragma unroll
    for (int i = 0; i < WAVES; ++i) {
      const float2 v = s[i];
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
template <typename T, int L, int W, NormMode MODE>
__device__ __forceinline__ float row_normalise(float *v, int lane, int C, float inv_c, bool layer, float eps, float2 *slots, int &turn) {
  if (layer) {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < W; ++i) s += v[i];
    const float mu = row_sum<L>(s, slots, turn) * inv_c;
#pragma unroll
    for (int i = 0; i < W; ++i) v[i] = norm_col<T, L, W>(lane, MODE == WHOLE ? i & -cpfn_piece<T>::N : i) < C ? v[i] - mu : 0.f;
  }
  float q = 0.f;
#pragma unroll
  for (int i = 0; i < W; ++i) q = fmaf(v[i], v[i], q);
  const float r = rsqrtf(fmaf(row_sum<L>(q, slots, turn), inv_c, eps));
#pragma unroll
  for (int i = 0; i < W; ++i) v[i] *= r;
  return r;
}

// 1 / (1 + exp(-v)).  fp32 rows: exp within 2 units in the last place.  16-bit rows: exp2(-v log2 e) with the product rounded, off by
// |v| 2^-23 relative on top (2^-17 at |v| = 64; the results are rounded to 2^-9), a third of the instructions.
template <typename T> __device__ __forceinline__ float norm_sigmoid(float v) {
  return __builtin_amdgcn_rcpf(1.f + (sizeof(T) == 4 ? expf(-v) : __builtin_amdgcn_exp2f(v * -1.44269504f)));
}

template <typename T, int W> __device__ __forceinline__ void gate_act(float (&g)[W], int sigmoid) {
  if (!sigmoid) return;
#pragma unroll
  for (int i = 0; i < W; ++i) g[i] = norm_sigmoid<T>(g[i]);
}
// the gate that all rows of a group share, behind its activation (one without such a gate)
template <typename T, int L, int W> __device__ __forceinline__ void shared_gate(float (&g)[W], const T *row, int lane, int C, int sigmoid) {
#pragma unroll
  for (int i = 0; i < W; ++i) g[i] = 1.f;
  if (!row) return;
  RowRaw<T, L, W> raw;
  single_load<T, L, W>(raw, row, lane, C);
  row_unpack(raw, g);
  gate_act<T, W>(g, sigmoid);
  arrived(g);
}

// ---------------------------------------------------------------- how the rows are split over workgroups (host)
// Channels of a lane: 8, and 16 where that keeps a whole row of 16-bit values in one wave (32768 x 1024, layer, shared gate: forward 56 ->
// 51 us, backward 101 -> 94; norm in front 24 -> 22, 52 -> 48; 50000 x 520 54 -> 45, 110 -> 90).  Elsewhere 16 are slower, for their
// registers (131072 x 128 backward 56 -> 64, 16384 x 2048 94 -> 107), for idle lanes (fp32 20528 x 259 36 -> 47) or for the masks of
// ragged rows (40000 x 601 forward 45 -> 47).
static inline int norm_width(int C, size_t element) { return element == 2 && C % 8 == 0 && C > 512 && C <= 1024 ? 16 : 8; }
// lanes for a row of C channels
static inline int norm_lanes(int C, int W) {
  int L = 8;
  while (L * W < C) L *= 2;
  return L;
}
// Rows are cut at the borders of gate groups (rows that share a gate row; one group without such a gate), then into chunks: a
// workgroup has one chunk of a group (blocks_per_group > 1) or whole groups.
struct NormSplit { long long groups, rows_per_gate, chunk; int nblk, blocks_per_group, groups_per_block; };
// waves: as many as are resident together; sets: row sets that a workgroup should have at least
static inline NormSplit norm_split(long long P, int C, int W, long long gate_rows, long long waves, int sets_at_least) {
  const int L = norm_lanes(C, W), threads = L <= 64 ? 256 : L, rows = threads / L;
  const bool shared = gate_rows > 0 && gate_rows < P;
  NormSplit s;
  s.groups = shared ? gate_rows : 1;
  s.rows_per_gate = P / s.groups;
  const long long sets = (s.rows_per_gate + rows - 1) / rows;             // row sets of a group
  const long long want = waves * 64 / threads;
  long long bpg = (want + s.groups - 1) / s.groups;
  if (bpg > (sets + sets_at_least - 1) / sets_at_least) bpg = (sets + sets_at_least - 1) / sets_at_least;
  const long long big = (s.rows_per_gate * C + (1ll << 27) - 1) >> 27;    // chunks below 2^29 bytes: offsets are 32 bits
  if (bpg < big) bpg = big;
  if (bpg < 1) bpg = 1;
  s.chunk = (sets + bpg - 1) / bpg * rows;
  bpg = (s.rows_per_gate + s.chunk - 1) / s.chunk;
  s.blocks_per_group = (int)bpg;
  s.groups_per_block = 1;
  if (bpg == 1) {
    const long long per = (s.groups + want - 1) / want;
    s.groups_per_block = (int)per;
    s.nblk = (int)((s.groups + per - 1) / per);
  } else {
    s.nblk = (int)(bpg * s.groups);
  }
  return s;
}
template <typename T> static inline NormMode norm_mode(long long P, int C) {
  if (C % cpfn_piece<T>::N == 0) return WHOLE;
  return P * C * (long long)sizeof(T) < 16 ? EACH : RAGGED;
}
