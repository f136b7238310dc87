// The norm over all gradients of a model, and their clipping, for lists of tensors of mixed types and lengths.  Launches: one of pass 1 for
// each 186 tensors, one of scaling for each 130, and one in between that adds the partial sums, for a norm alone and where every scaling
// workgroup doing so would be too many loads (partial sums x scaling workgroups > 2^20: from about 6M values in place, 3M elsewhere).
//
//   norm = (sum |g|^p)^(1/p), p = 1, 2 or infinity (the largest |g|);   coef = min(1, max_norm / (norm + 1e-6));   out = coef g
//
// The tensors travel as a table in the kernel's arguments (nothing is copied to the device, so a captured graph replays it as it is).
// Pass 1: a workgroup takes a share of ONE tensor and leaves one partial sum.  Sums are fp64: the squares of fp32 values cover
// 1e-90 .. 1e77, and one lane adds thousands of them.  Pass 2: every workgroup of the scaling launch adds the partial sums itself (in
// one fixed order: all agree, and runs repeat bit for bit; long lists: one workgroup does, in a launch in between), forms the factor and
// scales its share, from the list's end backwards: the values that pass 1 read last are still in the last-level cache.  A NaN in any gradient makes the norm NaN, an
// infinity makes it infinite; the factor follows by the formula (0 for an infinite norm, NaN for NaN).
#include "gradnorm.h"

#include <algorithm>
#include <vector>

namespace {

constexpr int GN_THREADS = 256;
// Elements of a workgroup before the workgroups are limited (1.4M values in 60 tensors, both launches: 4096 10.8 us, 16384 13.1) ...
constexpr int SHARE = 4096;
// ... to about so many in a call, one more for a tensor's last share: up to 48 long tensors stay within the 2048 that run at once, 8 on
// each of 256 CUs (67M fp32 elements 38.2 us, 5.5 TB/s, 2048: 39.8; 271M bf16 elements 86.3, 6.3 TB/s, 2048: 90.2)
constexpr int MOST_BLOCKS = 2000;
// Bytes at the list's end that pass 1 leaves in the last-level cache (of 256 MB; the rest is not kept): 271M bf16 to fp32, both passes, none
// 383 us, 96 MB 375, 240 MB 360
constexpr long long KEPT = 240ll << 20;
// The scaling launch has many short workgroups, whose stretches of memory follow each other closely: 271M values bf16 to fp32 268 us
// measured, 6.1 TB/s; in a comparison 284, shares of 4096 292, of 1024 397, 2000 workgroups with strides through whole tensors 357.  In
// place a workgroup that finds nothing to do should not be one of too many: 200M bf16 scaled, 35M fp32 left alone: 8192 157 and 4.9 us
// (4096: 153, 6; 16384: 161, 5).
constexpr int SCALE_SHARE = 2048, SCALE_SHARE_IN_PLACE = 8192;
constexpr long long MOST_SCALE_BLOCKS = 1 << 22;         // (a launch has fewer than 2^32 lanes)
// The partial sums are added by every scaling workgroup, or, where that would be more loads than these, by one launch in between
constexpr long long DIRECT_LOADS = 1 << 20;

// What a launch's arguments hold of a list.  Pass 1 takes more tensors (301 short ones: 23.7 -> 20.4 us).
struct Sources {
  enum { MAX = 186 };
  const void *src[MAX];
  long long n[MAX];
  int block0[MAX + 1];                     // first workgroup of each tensor
  unsigned char from[MAX];
  int count;
};
struct Moves {
  enum { MAX = 130 };
  const void *src[MAX];
  long long n[MAX];
  int block0[MAX + 1];
  unsigned char from[MAX];
  int count;
  void *dst[MAX];
  unsigned char to[MAX];
};
static_assert(sizeof(Sources) <= 4032 && sizeof(Moves) <= 4032, "4 KB of kernel arguments");
// Where the elements begin that pass 1 leaves in the last-level cache: element `at` of the launch's tensor `tensor`
struct Kept { int tensor; long long at; };

template <typename List> __device__ __forceinline__ int list_find(const List &a, int blk) {              // the last tensor with block0 <= blk
  int lo = 0, hi = a.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (a.block0[mid] <= blk) lo = mid; else hi = mid - 1;
  }
  return lo;
}

template <int P> __device__ __forceinline__ double gn_add(double acc, float v) {
  if (P == 1) return acc + fabs((double)v);
  return fma((double)v, (double)v, acc);
}
template <> __device__ __forceinline__ double gn_add<0>(double acc, float v) {  // the maximum; a NaN stays
  const double m = fabs((double)v);
  return (m > acc || m != m) ? m : acc;
}
template <int P> __device__ __forceinline__ double gn_join(double a, double b) {
  if (P == 0) return (b > a || b != b) ? b : a;
  return a + b;
}
template <int P> __device__ __forceinline__ double gn_block(double v, double *lds) {     // over a workgroup of GN_THREADS lanes
#pragma unroll
  for (int d = 32; d; d >>= 1) v = gn_join<P>(v, __shfl_xor(v, d, 64));
  __syncthreads();
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  v = lds[0];
#pragma unroll
  for (int w = 1; w < GN_THREADS / 64; ++w) v = gn_join<P>(v, lds[w]);
  return v;
}

// this lane's 16-byte pieces [first, end) of a tensor in steps of `step`, four in flight; ONCE: not kept in the caches
template <int P, bool ONCE, typename T>
__device__ __forceinline__ long long gn_pieces(const T *__restrict__ p, long long i, long long end, long long step, double (&acc)[4]) {
  constexpr int N = cpfn_piece<T>::N;
  typedef typename cpfn_piece<T>::vec V;
  for (; i + 3 * step < end; i += 4 * step) {
    V v[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const V *at = (const V *)(p + (i + q * step) * N);
      v[q] = ONCE ? __builtin_nontemporal_load(at) : *at;
    }
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      float f[N];
      cpfn_unpack(v[q], f, (T *)nullptr);
#pragma unroll
      for (int j = 0; j < N; ++j) acc[q] = gn_add<P>(acc[q], f[j]);
    }
  }
  if (ONCE) return i;
  for (; i < end; i += step) {
    float f[N];
    cpfn_unpack(*(const V *)(p + i * N), f, (T *)nullptr);
#pragma unroll
    for (int j = 0; j < N; ++j) acc[0] = gn_add<P>(acc[0], f[j]);
  }
  return i;
}
// keep: elements from here on are read a second time soon (the scaling pass), those before it are not kept
template <int P, typename T> __device__ __forceinline__ double gn_share(const T *__restrict__ p, long long n, long long keep, long long first, long long step) {
  constexpr int N = cpfn_piece<T>::N;
  double acc[4] = {0.0, 0.0, 0.0, 0.0};
  const long long whole = n / N;
  const long long i = gn_pieces<P, true>(p, first, keep / N, step, acc);
  gn_pieces<P, false>(p, i, whole, step, acc);
  if (whole * N + first < n) acc[1] = gn_add<P>(acc[1], cpfn_to_f32(p[whole * N + first]));      // the last n % N
  return gn_join<P>(gn_join<P>(acc[0], acc[1]), gn_join<P>(acc[2], acc[3]));
}

template <int P> __global__ __launch_bounds__(GN_THREADS, 8) void grad_norm_kernel(const Sources a, const Kept kept, double *__restrict__ part) {
  __shared__ double lds[GN_THREADS / 64];
  const int d = list_find(a, blockIdx.x);
  const long long first = (long long)(blockIdx.x - a.block0[d]) * GN_THREADS + threadIdx.x;
  const long long step = (long long)(a.block0[d + 1] - a.block0[d]) * GN_THREADS;
  const long long n = a.n[d], keep = d < kept.tensor ? n : d > kept.tensor ? 0 : kept.at;
  double v = 0.0;
  if (a.from[d] == CPFN_F32) v = gn_share<P>((const float *)a.src[d], n, keep, first, step);
  else if (a.from[d] == CPFN_BF16) v = gn_share<P>((const cpfn_bf16 *)a.src[d], n, keep, first, step);
  else v = gn_share<P>((const cpfn_f16 *)a.src[d], n, keep, first, step);
  v = gn_block<P>(v, lds);
  if (threadIdx.x == 0) part[blockIdx.x] = v;
}

// the norm from the partial sums: the same order in every workgroup
template <int P> __device__ __forceinline__ double gn_total(const double *__restrict__ part, int parts, double *lds) {
  double v = 0.0;
  for (int i = threadIdx.x; i < parts; i += GN_THREADS) v = gn_join<P>(v, part[i]);
  v = gn_block<P>(v, lds);
  return P == 2 ? sqrt(v) : v;
}
template <int P> __global__ __launch_bounds__(GN_THREADS) void grad_norm_finish_kernel(const double *__restrict__ part, int parts,
                                                                                       double *__restrict__ total, float *__restrict__ norm) {
  __shared__ double lds[GN_THREADS / 64];
  const double v = gn_total<P>(part, parts, lds);
  if (threadIdx.x == 0) {
    if (total) *total = v;
    if (norm) *norm = (float)v;
  }
}

// Elements [begin, end) of a tensor (begin: a multiple of 16).  Of a lane and step: 16 bytes on the wider side, so that the lanes of an
// access lie next to each other on both; two steps in flight, from the end (in place: T = U, every element is read before it is written).
template <typename T, typename U>
__device__ __forceinline__ void scale_share(const T *__restrict__ p, U *__restrict__ o, long long begin, long long end, float coef) {
  constexpr int N = cpfn_piece<T>::N < cpfn_piece<U>::N ? cpfn_piece<T>::N : cpfn_piece<U>::N, AHEAD = 2;
  constexpr bool narrow = N * sizeof(T) == 8;                        // 8 bytes in, 16 out
  typedef unsigned half __attribute__((ext_vector_type(2), aligned(2)));
  typedef typename cpfn_piece<T>::vec V;
  typedef typename cpfn_piece<U>::vec W;
  const long long whole = end / N, first = begin / N;
  const auto one = [&](const V &v, long long i) {
    float f[8];
    cpfn_unpack(v, f, (T *)nullptr);
#pragma unroll
    for (int j = 0; j < N; ++j) f[j] *= coef;
    __builtin_nontemporal_store(cpfn_pack(f, (U *)nullptr), (W *)(o + i * N));
  };
  const auto get = [&](long long i) {
    V v = {};
    if (narrow) {
      const half h = __builtin_nontemporal_load((const half *)(p + i * N));
      v.x = h.x; v.y = h.y;
    } else {
      v = __builtin_nontemporal_load((const V *)(p + i * N));
    }
    return v;
  };
  long long i = whole - 1 - threadIdx.x;
  for (; i - (AHEAD - 1) * GN_THREADS >= first; i -= AHEAD * GN_THREADS) {
    V v[AHEAD];
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) v[k] = get(i - k * GN_THREADS);
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) one(v[k], i - k * GN_THREADS);
  }
  for (; i >= first; i -= GN_THREADS) one(get(i), i);
  const long long last = whole * N + threadIdx.x;                    // (the tensor's last end % N: no other workgroup has them)
  if (last < end) o[last] = cpfn_from_f32<U>(cpfn_to_f32(p[last]) * coef);
}

// parts == 0: `part` is the norm itself.  elsewhere: the results go to other tensors (always written); in place nothing is to be done
// where the factor is 1.
template <int P>
__global__ __launch_bounds__(GN_THREADS) void grad_scale_kernel(const Moves a, const double *__restrict__ part, int parts, double max_norm,
                                                                int elsewhere, int share, float *__restrict__ norm) {
  __shared__ double lds[GN_THREADS / 64];
  const double total = parts ? gn_total<P>(part, parts, lds) : *part;
  if (norm && blockIdx.x == 0 && threadIdx.x == 0) *norm = (float)total;
  const float coef = grad_clip_factor(total, max_norm);
  if (coef == 1.f && !elsewhere) return;
  const int blk = a.block0[a.count] - 1 - (int)blockIdx.x;                       // (backwards, see above)
  const int d = list_find(a, blk);
  const long long begin = (long long)(blk - a.block0[d]) * share, end = begin + share < a.n[d] ? begin + share : a.n[d];
  if (a.from[d] == CPFN_F32) scale_share((const float *)a.src[d], (float *)a.dst[d], begin, end, coef);
  else if (a.from[d] == CPFN_BF16 && a.to[d] == CPFN_BF16) scale_share((const cpfn_bf16 *)a.src[d], (cpfn_bf16 *)a.dst[d], begin, end, coef);
  else if (a.from[d] == CPFN_BF16) scale_share((const cpfn_bf16 *)a.src[d], (float *)a.dst[d], begin, end, coef);
  else if (a.to[d] == CPFN_F16) scale_share((const cpfn_f16 *)a.src[d], (cpfn_f16 *)a.dst[d], begin, end, coef);
  else scale_share((const cpfn_f16 *)a.src[d], (float *)a.dst[d], begin, end, coef);
}

// workgroups of a tensor: one for each `share` elements
int blocks_of(long long n, long long share) { return (int)((n + share - 1) / share); }
// elements of a workgroup: SHARE, more where that would be more than about MOST_BLOCKS workgroups
long long share_of(const long long *n, int count) {
  long long sum = 0;
  for (int i = 0; i < count; ++i) sum += n[i];
  const long long even = (sum + MOST_BLOCKS - 1) / MOST_BLOCKS;
  return even > SHARE ? even : SHARE;
}

bool bad_list(const void *const *src, const long long *n, const int *type, int count) {
  if (count < 0 || (count > 0 && (!src || !n || !type))) return true;
  long long sum = 0;
  for (int i = 0; i < count; ++i) {
    if (n[i] < 0 || n[i] > (1ll << 48) || (n[i] > 0 && !src[i]) || type[i] < CPFN_F32 || type[i] > CPFN_F16) return true;
    sum += n[i];
    if (sum > (1ll << 48)) return true;
  }
  return false;
}

// Does a tensor that is written share memory with another one of the list (its own source excepted, where they are the same tensor)?
// Two workgroups would then read and write it in no order.
bool overlapping(const void *const *src, void *const *dst, const long long *n, const int *from, const int *to, int count) {
  struct Range { uintptr_t begin, end; bool written; };
  std::vector<Range> r;
  r.reserve(2 * (size_t)count);
  for (int i = 0; i < count; ++i) {
    if (n[i] == 0) continue;
    const uintptr_t s = (uintptr_t)src[i], d = (uintptr_t)dst[i];
    r.push_back({d, d + (uintptr_t)n[i] * (to[i] == CPFN_F32 ? 4 : 2), true});
    if (s != d || from[i] != to[i]) r.push_back({s, s + (uintptr_t)n[i] * (from[i] == CPFN_F32 ? 4 : 2), false});
  }
  std::sort(r.begin(), r.end(), [](const Range &a, const Range &b) { return a.begin < b.begin; });
  uintptr_t any = 0, written = 0;                        // the ends of what lies before
  for (const Range &x : r) {
    if (x.begin < (x.written ? any : written)) return true;
    any = std::max(any, x.end);
    if (x.written) written = std::max(written, x.end);
  }
  return false;
}

void set_target(Sources &, int, void *, int) {}
void set_target(Moves &a, int c, void *dst, int to) { a.dst[c] = dst; a.to[c] = (unsigned char)to; }

// tensors base.. of the list into `a`; returns the index behind the last one taken.  Empty tensors take no place.
template <typename List>
int fill(List &a, int base, const void *const *src, void *const *dst, const long long *n, const int *from, const int *to, int count, long long share) {
  a.count = 0;
  a.block0[0] = 0;
  int i = base;
  for (; i < count && a.count < List::MAX; ++i) {
    if (n[i] == 0) continue;
    const int c = a.count++;
    a.src[c] = src[i];
    a.n[c] = n[i];
    a.from[c] = (unsigned char)from[i];
    a.block0[c + 1] = a.block0[c] + blocks_of(n[i], share);
    set_target(a, c, dst ? dst[i] : nullptr, to ? to[i] : from[i]);
  }
  return i;
}

// kept: so many bytes from the list's end are read again soon
template <int P>
int norm_pass(const void *const *src, const long long *n, const int *type, int count, long long share, long long kept, double *part, hipStream_t st) {
  int parts = 0;
  const auto size = [](int t) { return t == CPFN_F32 ? 4 : 2; };
  long long streamed = -kept;                           // bytes in front of those
  for (int i = 0; i < count; ++i) streamed += n[i] * size(type[i]);
  for (int base = 0; base < count;) {
    Sources a;
    base = fill(a, base, src, nullptr, n, type, nullptr, count, share);
    if (a.count == 0) break;
    Kept k = {0, 0};
    for (; k.tensor < a.count && streamed >= a.n[k.tensor] * size(a.from[k.tensor]); ++k.tensor) streamed -= a.n[k.tensor] * size(a.from[k.tensor]);
    if (k.tensor < a.count && streamed > 0) {
      k.at = streamed / size(a.from[k.tensor]);
      streamed = 0;
    }
    grad_norm_kernel<P><<<a.block0[a.count], GN_THREADS, 0, st>>>(a, k, part + parts);
    parts += a.block0[a.count];
  }
  return parts;
}

template <int P>
int run(const void *const *src, void *const *dst, const long long *n, const int *from, const int *to, int count, double max_norm,
        bool clip, bool elsewhere, float *norm, double *ws, hipStream_t st) {
  const long long share = share_of(n, count);
  int scale_share = elsewhere ? SCALE_SHARE : SCALE_SHARE_IN_PLACE;
  long long sum = 0;
  for (int i = 0; i < count; ++i) sum += n[i];
  while (sum / scale_share > MOST_SCALE_BLOCKS) scale_share *= 2;
  double *part = ws + 1;
  int parts = norm_pass<P>(src, n, from, count, share, clip ? KEPT : 0, part, st);
  long long scale_blocks = 0;
  for (int i = 0; i < count; ++i) scale_blocks += (n[i] + scale_share - 1) / scale_share;
  if (!clip || parts == 0 || parts * scale_blocks > DIRECT_LOADS) {
    grad_norm_finish_kernel<P><<<1, GN_THREADS, 0, st>>>(part, parts, ws, norm);
    norm = nullptr;                                     // (written)
    part = ws;
    if (!clip || parts == 0) return cpfn_launch_status();
    parts = 0;
  }
  for (int base = 0; base < count;) {
    Moves a;
    base = fill(a, base, src, dst, n, from, to, count, scale_share);
    if (a.count == 0) break;
    grad_scale_kernel<P><<<a.block0[a.count], GN_THREADS, 0, st>>>(a, part, parts, max_norm, elsewhere ? 1 : 0, scale_share, norm);
    norm = nullptr;
  }
  return cpfn_launch_status();
}

int any(const void *const *src, void *const *dst, const long long *n, const int *from, const int *to, int count, int p, double max_norm,
        bool clip, bool elsewhere, float *norm, void *ws, hipStream_t st) {
  switch (p) {
    case 0: return run<0>(src, dst, n, from, to, count, max_norm, clip, elsewhere, norm, (double *)ws, st);
    case 1: return run<1>(src, dst, n, from, to, count, max_norm, clip, elsewhere, norm, (double *)ws, st);
    case 2: return run<2>(src, dst, n, from, to, count, max_norm, clip, elsewhere, norm, (double *)ws, st);
  }
  return CPFN_EINVAL;
}

}  // namespace

extern "C" long long cpfn_grad_norm_workspace(const long long *n, int count) {
  if (count < 0 || (count > 0 && !n)) return -1;
  const long long share = share_of(n, count);
  long long parts = 1;
  for (int i = 0; i < count; ++i) parts += blocks_of(n[i] < 0 ? 0 : n[i], share);
  return parts * (long long)sizeof(double);
}

extern "C" int cpfn_grad_norm(const void *const *grads, const long long *n, const int *type, int count, int p, float *norm,
                              void *workspace, void *stream) {
  if (bad_list(grads, n, type, count) || !norm || !workspace || ((uintptr_t)workspace & 7)) return CPFN_EINVAL;
  return any(grads, nullptr, n, type, nullptr, count, p, 0.0, false, false, norm, workspace, (hipStream_t)stream);
}

extern "C" int cpfn_grad_clip(const void *const *grads, void *const *out, const long long *n, const int *type, const int *out_type,
                              int count, int p, double max_norm, float *norm, void *workspace, void *stream) {
  if (bad_list(grads, n, type, count) || !norm || !workspace || ((uintptr_t)workspace & 7) || !(max_norm >= 0.0)) return CPFN_EINVAL;
  if (out) {
    if (!out_type) return CPFN_EINVAL;
    for (int i = 0; i < count; ++i)
      if (n[i] > 0 && (!out[i] || (out_type[i] != type[i] && out_type[i] != CPFN_F32))) return CPFN_EINVAL;
  }
  void *const *dst = out ? out : (void *const *)grads;
  const int *to = out ? out_type : type;
  try {
    if (overlapping(grads, dst, n, type, to, count)) return CPFN_EOVERLAP;
  } catch (...) {
    return CPFN_EINVAL;
  }
  return any(grads, dst, n, type, to, count, p, max_norm, true, out != nullptr, norm, workspace, (hipStream_t)stream);
}

extern "C" int cpfn_grad_sumsq_blocks(long long n) { return n < 0 || n > (1ll << 48) ? -1 : blocks_of(n, share_of(&n, 1)); }

extern "C" int cpfn_grad_sumsq(const float *g, long long n, double *parts, void *stream) {
  if (n < 0 || n > (1ll << 48) || (n > 0 && (!g || !parts)) || ((uintptr_t)parts & 7)) return CPFN_EINVAL;
  const void *src = g;
  const int type = CPFN_F32;
  norm_pass<2>(&src, &n, &type, 1, share_of(&n, 1), 4 * n, parts, (hipStream_t)stream);
  return cpfn_launch_status();
}
