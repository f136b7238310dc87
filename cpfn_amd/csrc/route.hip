// Rows sorted by expert and back (routed layers): the order (a stable counting sort of expert indices), the move into it, the
// weighted sum out of it, and their adjoints.
//
//   place[r, j] = position of row r's j-th choice among all choices sorted by expert (stable; -1: an index outside [0, E))
//   gather:   sorted[place[r, j]] = rows[r]                      (rows behind the last expert's: zero)
//   combine:  out[r] = sum_j w[r, j] sorted[place[r, j]]         (no weights: w = 1, the adjoint of gather)
//   adjoint of combine:  d_sorted[place[r, j]] = w[r, j] g[r],   d_w[r, j] = <g[r], sorted[place[r, j]]>
//
// Every move walks the UNSORTED rows r: the tensor with one row per r is read or written once, the one with k rows per r by whole
// rows, and each output row has one writer: no atomics, no zero fill in front.  Products and sums in fp32, one rounding at the store.
#include "rows16.h"

namespace {

// ---------------------------------------------------------------- the order
// A workgroup ranks TILE consecutive choices; a wave takes a contiguous part of them, 64 at a time.  Rank inside 64: the lanes with
// the same expert are found by one ballot for each bit of the index; the first such lane adds their number to the wave's own LDS
// counter of that expert: no atomics, so the order is the input's order by construction.
constexpr int RANK_WAVES = 8, RANK_ITEMS = 8, RANK_TILE = RANK_WAVES * RANK_ITEMS * 64;
constexpr int ROUTE_MAX_E = 2048;                 // a 16-bit counter for each wave (a tile has 4096 choices) and a base: 40 KB of LDS
// up to so many tiles and experts every workgroup sums the tiles' counts by itself, instead of a launch that does it once
constexpr int DIRECT_TILES = 64, DIRECT_E = 256;

template <typename I> __device__ __forceinline__ int expert_of(const I *__restrict__ choice, long long i, long long n, int E) {
  if (i >= n) return -1;
  const I v = choice[i];
  return v >= 0 && v < (I)E ? (int)v : -1;
}

// mask of the lanes of this wave whose expert is this lane's (of lanes that have one)
__device__ __forceinline__ unsigned long long same_expert(int e, int bits) {
  unsigned long long m = __ballot(e >= 0);
  for (int b = 0; b < bits; ++b) {
    const bool one = (e >> b) & 1;
    const unsigned long long v = __ballot(one);
    m &= one ? v : ~v;
  }
  return m;
}

// the ranks of a wave's choices among the wave's own; `mine`: the wave's counters, zero before, the wave's counts afterwards
__device__ __forceinline__ void wave_ranks(const int *e, int *rank, unsigned short *mine, int bits, int lane) {
#pragma unroll
  for (int t = 0; t < RANK_ITEMS; ++t) {
    const unsigned long long m = same_expert(e[t], bits);
    rank[t] = 0;
    if (e[t] >= 0) {
      const int before = mine[e[t]];
      rank[t] = before + __popcll(m & ((1ull << lane) - 1ull));
      if (__builtin_ctzll(m) == lane) mine[e[t]] = (unsigned short)(before + __popcll(m));
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");      // the next 64 read what these wrote
    __builtin_amdgcn_wave_barrier();
  }
}

__device__ __forceinline__ void zero_counters(unsigned short *cnt, int E) {       // (E counters of RANK_WAVES waves: whole words)
  for (int i = threadIdx.x; i < RANK_WAVES * E / 2; i += RANK_WAVES * 64) ((unsigned *)cnt)[i] = 0u;
  __syncthreads();
}

// counts[e][tile] (several tiles only): a histogram by LDS additions, whose order does not show in an integer
template <typename I>
__global__ __launch_bounds__(RANK_WAVES * 64) void route_count_kernel(const I *__restrict__ choice, long long n, int E, int tiles,
                                                                      int *__restrict__ counts) {
  extern __shared__ unsigned lds[];               // [E]
  for (int x = threadIdx.x; x < E; x += RANK_WAVES * 64) lds[x] = 0u;
  const long long i0 = (long long)blockIdx.x * RANK_TILE + threadIdx.x;
  int e[RANK_ITEMS];
#pragma unroll
  for (int t = 0; t < RANK_ITEMS; ++t) e[t] = expert_of(choice, i0 + t * (RANK_WAVES * 64), n, E);
  __syncthreads();
#pragma unroll
  for (int t = 0; t < RANK_ITEMS; ++t)
    if (e[t] >= 0) atomicAdd(&lds[e[t]], 1u);
  __syncthreads();
  for (int x = threadIdx.x; x < E; x += RANK_WAVES * 64) counts[(long long)x * tiles + blockIdx.x] = (int)lds[x];
}

__device__ __forceinline__ int wave_scan(int v, int lane) {                       // inclusive
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int u = __shfl_up(v, d, 64);
    if (lane >= d) v += u;
  }
  return v;
}

// counts[e][0..tiles) -> exclusive sums over the tiles, totals[e]: one wave for each expert
__global__ __launch_bounds__(256) void route_scan_kernel(int *__restrict__ counts, int *__restrict__ totals, int E, int tiles) {
  const int e = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
  if (e >= E) return;
  int *row = counts + (long long)e * tiles;
  int carry = 0;
  for (int b = 0; b < tiles; b += 64) {
    const int v = b + lane < tiles ? row[b + lane] : 0;
    const int s = wave_scan(v, lane);
    if (b + lane < tiles) row[b + lane] = carry + s - v;
    carry += __shfl(s, 63, 64);
  }
  if (lane == 0) totals[e] = carry;
}

// mode 0: one tile (its own counts are all there is); 1: sums the tiles' counts itself; 2: counts are exclusive sums, totals given
template <typename I>
__global__ __launch_bounds__(RANK_WAVES * 64) void route_rank_kernel(const I *__restrict__ choice, long long n, int E, int bits, int tiles,
                                                                     int mode, const int *__restrict__ counts,
                                                                     const int *__restrict__ totals, int *__restrict__ offsets,
                                                                     int *__restrict__ place) {
  extern __shared__ unsigned lds[];               // [waves][E] 16-bit counters | [E] first position of this tile's
  __shared__ int wsum[RANK_WAVES], d_before[DIRECT_E], d_total[DIRECT_E];
  constexpr int THREADS = RANK_WAVES * 64;
  unsigned short *cnt = (unsigned short *)lds;
  int *base = (int *)(lds + RANK_WAVES * E / 2);
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const long long i0 = (long long)blockIdx.x * RANK_TILE + wave * (RANK_ITEMS * 64) + lane;
  unsigned short *mine = cnt + wave * E;
  int e[RANK_ITEMS], rank[RANK_ITEMS];
#pragma unroll
  for (int t = 0; t < RANK_ITEMS; ++t) e[t] = expert_of(choice, i0 + t * 64, n, E);
  if (mode == 1) {                                // tiles <= 64: a lane for each tile, a wave for each expert
    for (int x = wave; x < E; x += RANK_WAVES) {
      const int v = lane < tiles ? counts[x * tiles + lane] : 0;
      const int s = wave_scan(v, lane);
      if (lane == (int)blockIdx.x) d_before[x] = s - v;
      if (lane == 63) d_total[x] = s;
    }
  }
  zero_counters(cnt, E);
  wave_ranks(e, rank, mine, bits, lane);
  __syncthreads();
  // per expert: exclusive sums over the waves (in place), the tiles before this one, and the total; the totals' exclusive sum over
  // the experts is the expert's first position (a carry from one THREADS-wide step to the next)
  int carry = 0;
  for (int x0 = 0; x0 < E; x0 += THREADS) {
    const int x = x0 + tid;
    int before = 0, total = 0;
    if (x < E) {
      int s = 0;
#pragma unroll
      for (int w = 0; w < RANK_WAVES; ++w) {
        const int v = cnt[w * E + x];
        cnt[w * E + x] = (unsigned short)s;
        s += v;
      }
      total = mode == 0 ? s : mode == 1 ? d_total[x] : totals[x];
      before = mode == 0 ? 0 : mode == 1 ? d_before[x] : counts[(long long)x * tiles + blockIdx.x];
    }
    const int s = wave_scan(total, lane);
    if (lane == 63) wsum[wave] = s;
    __syncthreads();
    int pre = carry;
#pragma unroll
    for (int w = 0; w < RANK_WAVES; ++w) {
      const int v = wsum[w];
      if (w < wave) pre += v;
      carry += v;
    }
    if (x < E) {
      const int first = pre + s - total;
      base[x] = first + before;
      if (blockIdx.x == 0) offsets[x] = first;
    }
    __syncthreads();
  }
  if (blockIdx.x == 0 && tid == 0) offsets[E] = carry;
#pragma unroll
  for (int t = 0; t < RANK_ITEMS; ++t) {
    const long long i = i0 + t * 64;
    if (i < n) place[i] = e[t] >= 0 ? base[e[t]] + mine[e[t]] + rank[t] : -1;
  }
}

// ---------------------------------------------------------------- the moves
constexpr int MOVE_THREADS = 256;

// rows behind the last expert's, [offsets[E], n): zero, shared out over all row slots of the launch
template <typename T>
__device__ __forceinline__ void zero_tail(T *__restrict__ out, const int *__restrict__ end, long long n, int C, int lane, int lanes,
                                          long long slot, long long slots) {
  float z[cpfn_piece<T>::N];
#pragma unroll
  for (int i = 0; i < cpfn_piece<T>::N; ++i) z[i] = 0.f;
  for (long long p = *end + slot; p < n; p += slots)
    for (int c = lane * cpfn_piece<T>::N; c < C; c += lanes * cpfn_piece<T>::N) cpfn_store_piece(out + p * C, c, C, z);
}

// LANES lanes per row, 16 bytes each and step
template <typename T>
__global__ __launch_bounds__(MOVE_THREADS) void route_gather_kernel(const T *__restrict__ rows, const int *__restrict__ place,
                                                                    const int *__restrict__ end, long long R, int k, int C, int lanes_log2,
                                                                    T *__restrict__ out) {
  constexpr int N = cpfn_piece<T>::N;
  typedef typename cpfn_piece<T>::vec V;                // (bits are moved, not values: NaNs keep theirs)
  const int lanes = 1 << lanes_log2, lane = threadIdx.x & (lanes - 1);
  const long long slot = (long long)blockIdx.x * (MOVE_THREADS >> lanes_log2) + (threadIdx.x >> lanes_log2);
  const long long slots = (long long)gridDim.x * (MOVE_THREADS >> lanes_log2);
  for (long long r = slot; r < R; r += slots) {
    for (int c = lane * N; c < C; c += lanes * N) {
      if (c + N <= C) {
        const V v = *(const V *)(rows + r * C + c);
        for (int j = 0; j < k; ++j) {
          const int p = place[r * k + j];
          if (p >= 0) *(V *)(out + (long long)p * C + c) = v;
        }
      } else {                                          // the row ends inside this piece
        for (int q = c; q < C; ++q) {
          const T v = rows[r * C + q];
          for (int j = 0; j < k; ++j) {
            const int p = place[r * k + j];
            if (p >= 0) out[(long long)p * C + q] = v;
          }
        }
      }
    }
  }
  zero_tail(out, end, R * k, C, lane, lanes, slot, slots);
}

template <typename T>
__global__ __launch_bounds__(MOVE_THREADS) void route_combine_kernel(const T *__restrict__ sorted, const float *__restrict__ weights,
                                                                     const int *__restrict__ place, long long R, int k, int C,
                                                                     int lanes_log2, T *__restrict__ out) {
  constexpr int N = cpfn_piece<T>::N, AHEAD = 4;        // rows of one sum in flight
  const int lanes = 1 << lanes_log2, lane = threadIdx.x & (lanes - 1);
  const long long slot = (long long)blockIdx.x * (MOVE_THREADS >> lanes_log2) + (threadIdx.x >> lanes_log2);
  const long long slots = (long long)gridDim.x * (MOVE_THREADS >> lanes_log2);
  for (long long r = slot; r < R; r += slots) {
    for (int c = lane * N; c < C; c += lanes * N) {
      float acc[N];
#pragma unroll
      for (int i = 0; i < N; ++i) acc[i] = 0.f;
      for (int j0 = 0; j0 < k; j0 += AHEAD) {
        typename cpfn_piece<T>::vec v[AHEAD];
        float w[AHEAD];
        bool there[AHEAD];
#pragma unroll
        for (int t = 0; t < AHEAD; ++t) {
          const int p = j0 + t < k ? place[r * k + j0 + t] : -1;
          there[t] = p >= 0;
          v[t] = {};
          w[t] = 1.f;
          if (there[t]) {
            v[t] = cpfn_load_piece(sorted + (long long)p * C, c, C);
            if (weights) w[t] = weights[r * k + j0 + t];
          }
        }
#pragma unroll
        for (int t = 0; t < AHEAD; ++t) {
          if (there[t]) {                                // (a choice that is not there adds nothing, whatever its weight)
            float f[N];
            cpfn_unpack(v[t], f, (T *)nullptr);
#pragma unroll
            for (int i = 0; i < N; ++i) acc[i] = fmaf(w[t], f[i], acc[i]);
          }
        }
      }
      cpfn_store_piece(out + r * C, c, C, acc);
    }
  }
}

// LANES <= 64: the products of a row meet inside a wave
template <typename T, int LANES>
__global__ __launch_bounds__(MOVE_THREADS) void route_combine_bwd_kernel(const T *__restrict__ g, const T *__restrict__ sorted,
                                                                         const float *__restrict__ weights, const int *__restrict__ place,
                                                                         const int *__restrict__ end, long long R, int k, int C,
                                                                         T *__restrict__ d_sorted, float *__restrict__ d_weights) {
  constexpr int N = cpfn_piece<T>::N, AHEAD = 4, ROWS = MOVE_THREADS / LANES;
  const int lane = threadIdx.x & (LANES - 1);
  const long long slot = (long long)blockIdx.x * ROWS + threadIdx.x / LANES, slots = (long long)gridDim.x * ROWS;
  // (whole row sets: the lanes of a wave stay together for the row sums)
  for (long long r0 = (long long)blockIdx.x * ROWS; r0 < R; r0 += slots) {
    const long long r = r0 + threadIdx.x / LANES;
    const bool row = r < R;
    for (int j0 = 0; j0 < k; j0 += AHEAD) {
      int p[AHEAD];
      float w[AHEAD], dot[AHEAD];
#pragma unroll
      for (int t = 0; t < AHEAD; ++t) {
        p[t] = row && j0 + t < k ? place[r * k + j0 + t] : -1;
        w[t] = p[t] >= 0 && weights ? weights[r * k + j0 + t] : 1.f;
        dot[t] = 0.f;
      }
      if (row) {
        for (int c = lane * N; c < C; c += LANES * N) {
          float gf[N];
          cpfn_unpack(cpfn_load_piece(g + r * C, c, C), gf, (T *)nullptr);
          typename cpfn_piece<T>::vec v[AHEAD];
#pragma unroll
          for (int t = 0; t < AHEAD; ++t) {
            v[t] = {};
            if (d_weights && p[t] >= 0) v[t] = cpfn_load_piece(sorted + (long long)p[t] * C, c, C);
          }
#pragma unroll
          for (int t = 0; t < AHEAD; ++t) {
            if (p[t] < 0) continue;
            if (d_weights) {
              float f[N];
              cpfn_unpack(v[t], f, (T *)nullptr);
#pragma unroll
              for (int i = 0; i < N; ++i) dot[t] = fmaf(gf[i], f[i], dot[t]);
            }
            if (d_sorted) {
              float f[N];
#pragma unroll
              for (int i = 0; i < N; ++i) f[i] = w[t] * gf[i];
              cpfn_store_piece(d_sorted + (long long)p[t] * C, c, C, f);
            }
          }
        }
      }
      if (d_weights) {
#pragma unroll
        for (int t = 0; t < AHEAD; ++t) {
          const float s = cpfn_lanes_sum<LANES>(dot[t]);
          if (row && lane == 0 && j0 + t < k) d_weights[r * k + j0 + t] = p[t] >= 0 ? s : 0.f;
        }
      }
    }
  }
  if (d_sorted) zero_tail(d_sorted, end, R * k, C, lane, LANES, slot, slots);
}

int lanes_log2_for(int C, int per_lane, int most) {
  int l = 0;
  while (l < most && (per_lane << l) < C) ++l;
  return l;
}
unsigned move_blocks(long long R, int lanes_log2) {
  const long long rows = MOVE_THREADS >> lanes_log2, b = (R + rows - 1) / rows;
  return (unsigned)(b < 8192 ? b : 8192);
}

template <typename I>
int plan(const I *choice, long long n, int E, int *offsets, int *place, int *ws, hipStream_t st) {
  const int tiles = n > RANK_TILE ? (int)((n + RANK_TILE - 1) / RANK_TILE) : 1;
  int bits = 0;
  while ((1 << bits) < E) ++bits;
  const size_t lds_rank = (size_t)RANK_WAVES * E * 2 + (size_t)E * 4;
  const int mode = tiles == 1 ? 0 : tiles <= DIRECT_TILES && E <= DIRECT_E ? 1 : 2;
  int *counts = ws, *totals = ws + (size_t)tiles * E;
  if (mode) route_count_kernel<I><<<tiles, RANK_WAVES * 64, (size_t)E * 4, st>>>(choice, n, E, tiles, counts);
  if (mode == 2) route_scan_kernel<<<cpfn_cdiv(E, 4), 256, 0, st>>>(counts, totals, E, tiles);
  route_rank_kernel<I><<<tiles, RANK_WAVES * 64, lds_rank, st>>>(choice, n, E, bits, tiles, mode, counts, totals, offsets, place);
  return cpfn_launch_status();
}

template <typename T> int gather(const void *rows, const int *place, const int *offsets, long long R, int k, int E, int C, void *out, hipStream_t st) {
  const int l = lanes_log2_for(C, cpfn_piece<T>::N, 8);
  route_gather_kernel<T><<<move_blocks(R, l), MOVE_THREADS, 0, st>>>((const T *)rows, place, offsets + E, R, k, C, l, (T *)out);
  return cpfn_launch_status();
}
template <typename T> int combine(const void *sorted, const float *weights, const int *place, long long R, int k, int C, void *out, hipStream_t st) {
  const int l = lanes_log2_for(C, cpfn_piece<T>::N, 8);
  route_combine_kernel<T><<<move_blocks(R, l), MOVE_THREADS, 0, st>>>((const T *)sorted, weights, place, R, k, C, l, (T *)out);
  return cpfn_launch_status();
}
template <typename T, int L>
void combine_bwd_launch(const void *g, const void *sorted, const float *weights, const int *place, const int *end, long long R, int k, int C,
                        void *d_sorted, float *d_weights, int l, hipStream_t st) {
  route_combine_bwd_kernel<T, L><<<move_blocks(R, l), MOVE_THREADS, 0, st>>>((const T *)g, (const T *)sorted, weights, place, end, R, k, C,
                                                                            (T *)d_sorted, d_weights);
}
template <typename T>
int combine_bwd(const void *g, const void *sorted, const float *weights, const int *place, const int *offsets, long long R, int k, int E, int C,
                void *d_sorted, float *d_weights, hipStream_t st) {
  const int l = lanes_log2_for(C, cpfn_piece<T>::N, 6);
  const int *end = offsets + E;
  switch (l < 2 ? 2 : l) {
    case 2: combine_bwd_launch<T, 4>(g, sorted, weights, place, end, R, k, C, d_sorted, d_weights, 2, st); break;
    case 3: combine_bwd_launch<T, 8>(g, sorted, weights, place, end, R, k, C, d_sorted, d_weights, 3, st); break;
    case 4: combine_bwd_launch<T, 16>(g, sorted, weights, place, end, R, k, C, d_sorted, d_weights, 4, st); break;
    case 5: combine_bwd_launch<T, 32>(g, sorted, weights, place, end, R, k, C, d_sorted, d_weights, 5, st); break;
    default: combine_bwd_launch<T, 64>(g, sorted, weights, place, end, R, k, C, d_sorted, d_weights, 6, st); break;
  }
  return cpfn_launch_status();
}

bool bad_sizes(long long R, int k, int E, int C) {
  return R < 0 || k < 1 || E < 1 || E > ROUTE_MAX_E || C < 1 || R > 0x7fffffffll / k;
}

}  // namespace

extern "C" long long cpfn_route_workspace(long long n, int E) {
  if (n < 0 || n > 0x7fffffffll || E < 1 || E > ROUTE_MAX_E) return -1;
  const long long tiles = (n + RANK_TILE - 1) / RANK_TILE;
  return tiles <= 1 ? 0 : (tiles + 1) * E * (long long)sizeof(int);
}

extern "C" int cpfn_route_plan(const void *choice, int wide, long long n, int E, int *offsets, int *place, void *workspace, void *stream) {
  if (bad_sizes(n, 1, E, 1) || !offsets || (n > 0 && (!choice || !place)) || (n > RANK_TILE && !workspace)) return CPFN_EINVAL;
  hipStream_t st = (hipStream_t)stream;
  return wide ? plan((const long long *)choice, n, E, offsets, place, (int *)workspace, st)
              : plan((const int *)choice, n, E, offsets, place, (int *)workspace, st);
}

extern "C" int cpfn_route_gather(const void *rows, const int *place, const int *offsets, long long R, int k, int E, int C, int dtype,
                                 void *out, void *stream) {
  if (bad_sizes(R, k, E, C) || (R > 0 && (!rows || !place || !offsets || !out))) return CPFN_EINVAL;
  if (R == 0) return 0;
  hipStream_t st = (hipStream_t)stream;
  switch (dtype) {
    case CPFN_F32: return gather<float>(rows, place, offsets, R, k, E, C, out, st);
    case CPFN_BF16: return gather<cpfn_bf16>(rows, place, offsets, R, k, E, C, out, st);
    case CPFN_F16: return gather<cpfn_f16>(rows, place, offsets, R, k, E, C, out, st);
  }
  return CPFN_EINVAL;
}

extern "C" int cpfn_route_combine(const void *sorted, const float *weights, const int *place, long long R, int k, int C, int dtype,
                                  void *out, void *stream) {
  if (bad_sizes(R, k, 1, C) || (R > 0 && (!sorted || !place || !out))) return CPFN_EINVAL;
  if (R == 0) return 0;
  hipStream_t st = (hipStream_t)stream;
  switch (dtype) {
    case CPFN_F32: return combine<float>(sorted, weights, place, R, k, C, out, st);
    case CPFN_BF16: return combine<cpfn_bf16>(sorted, weights, place, R, k, C, out, st);
    case CPFN_F16: return combine<cpfn_f16>(sorted, weights, place, R, k, C, out, st);
  }
  return CPFN_EINVAL;
}

extern "C" int cpfn_route_combine_bwd(const void *g, const void *sorted, const float *weights, const int *place, const int *offsets,
                                      long long R, int k, int E, int C, int dtype, void *d_sorted, float *d_weights, void *stream) {
  if (bad_sizes(R, k, E, C) || (!d_sorted && !d_weights) || (R > 0 && (!g || !place || !offsets || (d_weights && !sorted))))
    return CPFN_EINVAL;
  if (R == 0) return 0;
  hipStream_t st = (hipStream_t)stream;
  switch (dtype) {
    case CPFN_F32: return combine_bwd<float>(g, sorted, weights, place, offsets, R, k, E, C, d_sorted, d_weights, st);
    case CPFN_BF16: return combine_bwd<cpfn_bf16>(g, sorted, weights, place, offsets, R, k, E, C, d_sorted, d_weights, st);
    case CPFN_F16: return combine_bwd<cpfn_f16>(g, sorted, weights, place, offsets, R, k, E, C, d_sorted, d_weights, st);
  }
  return CPFN_EINVAL;
}
