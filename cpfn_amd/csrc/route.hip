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

// mask of the lanes of this wave whose expert is this lane's (of lanes that have one): a lane keeps the lanes whose bit is its own
__device__ __forceinline__ unsigned long long same_expert(int e, int bits) {
  const unsigned long long valid = __ballot(e >= 0);
  unsigned lo = (unsigned)valid, hi = (unsigned)(valid >> 32);
  for (int b = 0; b < bits; ++b) {
    const unsigned mine = (unsigned)((e << (31 - b)) >> 31);                      // all ones: my bit is set
    const unsigned long long v = __ballot(mine != 0u);
    lo &= ~((unsigned)v ^ mine);
    hi &= ~((unsigned)(v >> 32) ^ mine);
  }
  return (unsigned long long)hi << 32 | lo;
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

// counts[e][0..tiles) -> exclusive sums over the tiles, totals[e]: a workgroup for each expert, four tiles a lane and step
__global__ __launch_bounds__(256) void route_scan_kernel(int *__restrict__ counts, int *__restrict__ totals, int tiles) {
  __shared__ int wsum[2][4];
  const int e = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  int *row = counts + (long long)e * tiles;
  int carry = 0, turn = 0;
  for (int b = 0; b < tiles; b += 1024, turn ^= 1) {
    const int at = b + tid * 4;
    int v[4], s = 0;
#pragma unroll
    for (int q = 0; q < 4; ++q) v[q] = at + q < tiles ? row[at + q] : 0;
#pragma unroll
    for (int q = 0; q < 4; ++q) s += v[q];
    const int up_to = wave_scan(s, lane);
    if (lane == 63) wsum[turn][wave] = up_to;
    __syncthreads();
    int before = carry + up_to - s;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const int x = wsum[turn][w];
      if (w < wave) before += x;
      carry += x;
    }
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      if (at + q < tiles) row[at + q] = before;
      before += v[q];
    }
  }
  if (tid == 0) totals[e] = carry;
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
constexpr int MOVE_THREADS = 256, MOVE_BLOCKS = 2048;

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

// How a launch walks its rows: 1 << lanes_log2 lanes for a row, 16 bytes each and step; ROWS rows of a lane group in flight.
struct Walk {
  int lanes, lane;
  long long slot, slots;
  __device__ __forceinline__ explicit Walk(int lanes_log2) {
    lanes = 1 << lanes_log2;
    lane = threadIdx.x & (lanes - 1);
    slot = (long long)blockIdx.x * (MOVE_THREADS >> lanes_log2) + (threadIdx.x >> lanes_log2);
    slots = (long long)gridDim.x * (MOVE_THREADS >> lanes_log2);
  }
};

// KT: choices of a row that are taken at once (their places in flight together)
template <typename T, int KT>
__global__ __launch_bounds__(MOVE_THREADS) void route_gather_kernel(const T *__restrict__ rows, const int *__restrict__ place,
                                                                    const int *__restrict__ end, long long R, int k, int C, int lanes_log2,
                                                                    T *__restrict__ out) {
  constexpr int N = cpfn_piece<T>::N, ROWS = KT <= 2 ? 4 : 2;
  typedef typename cpfn_piece<T>::vec V;                // (bits are moved, not values: NaNs keep theirs)
  const Walk w(lanes_log2);
  for (long long r0 = w.slot; r0 < R; r0 += ROWS * w.slots) {
    for (int j0 = 0; j0 < k; j0 += KT) {
      int p[ROWS][KT];
#pragma unroll
      for (int u = 0; u < ROWS; ++u)
#pragma unroll
        for (int t = 0; t < KT; ++t) {
          const long long r = r0 + u * w.slots;
          p[u][t] = r < R && j0 + t < k ? place[r * k + j0 + t] : -1;
        }
      for (int c = w.lane * N; c < C; c += w.lanes * N) {
        if (c + N <= C) {
          V v[ROWS];
#pragma unroll
          for (int u = 0; u < ROWS; ++u) {
            const long long r = r0 + u * w.slots;
            v[u] = *(const V *)(rows + (r < R ? r : R - 1) * C + c);
          }
#pragma unroll
          for (int u = 0; u < ROWS; ++u)
#pragma unroll
            for (int t = 0; t < KT; ++t)
              if (p[u][t] >= 0) __builtin_nontemporal_store(v[u], (V *)(out + (long long)p[u][t] * C + c));
        } else {                                        // the row ends inside this piece
          for (int q = c; q < C; ++q)
#pragma unroll
            for (int u = 0; u < ROWS; ++u) {
              const long long r = r0 + u * w.slots;
              const T v = rows[(r < R ? r : R - 1) * C + q];
#pragma unroll
              for (int t = 0; t < KT; ++t)
                if (p[u][t] >= 0) out[(long long)p[u][t] * C + q] = v;
            }
        }
      }
    }
  }
  zero_tail(out, end, R * k, C, w.lane, w.lanes, w.slot, w.slots);
}

template <typename T, int KT>
__global__ __launch_bounds__(MOVE_THREADS) void route_combine_kernel(const T *__restrict__ sorted, const float *__restrict__ weights,
                                                                     const int *__restrict__ place, long long R, int k, int C,
                                                                     int lanes_log2, T *__restrict__ out) {
  constexpr int N = cpfn_piece<T>::N, ROWS = KT <= 2 ? 4 : 2;
  typedef typename cpfn_piece<T>::vec V;
  const Walk walk(lanes_log2);
  for (long long r0 = walk.slot; r0 < R; r0 += ROWS * walk.slots) {
    int p[ROWS][KT];
    float w[ROWS][KT];
    const auto choices = [&](int j0) {
#pragma unroll
      for (int u = 0; u < ROWS; ++u)
#pragma unroll
        for (int t = 0; t < KT; ++t) {
          const long long r = r0 + u * walk.slots;
          const bool is = r < R && j0 + t < k;
          const long long at = is ? r * k + j0 + t : 0;
          p[u][t] = is ? place[at] : -1;
          w[u][t] = weights ? weights[at] : 1.f;
        }
    };
    choices(0);
    for (int c = walk.lane * N; c < C; c += walk.lanes * N) {
      float acc[ROWS][N];
#pragma unroll
      for (int u = 0; u < ROWS; ++u)
#pragma unroll
        for (int i = 0; i < N; ++i) acc[u][i] = 0.f;
      for (int j0 = 0; j0 < k; j0 += KT) {
        if (k > KT) choices(j0);
        V v[ROWS][KT];
#pragma unroll
        for (int u = 0; u < ROWS; ++u)
#pragma unroll
          for (int t = 0; t < KT; ++t) v[u][t] = cpfn_load_piece(sorted + (long long)(p[u][t] < 0 ? 0 : p[u][t]) * C, c, C);
#pragma unroll
        for (int u = 0; u < ROWS; ++u)
#pragma unroll
          for (int t = 0; t < KT; ++t) {
            float f[N];
            cpfn_unpack(v[u][t], f, (T *)nullptr);
            const bool is = p[u][t] >= 0;               // (a choice that is not there adds nothing, whatever stands in its places)
#pragma unroll
            for (int i = 0; i < N; ++i) acc[u][i] = is ? fmaf(w[u][t], f[i], acc[u][i]) : acc[u][i];
          }
      }
#pragma unroll
      for (int u = 0; u < ROWS; ++u) {
        const long long r = r0 + u * walk.slots;
        if (r < R) cpfn_store_piece(out + r * C, c, C, acc[u]);
      }
    }
  }
}

// LANES <= 64: the products of a row meet inside a wave
template <typename T, int LANES, int KT>
__global__ __launch_bounds__(MOVE_THREADS) void route_combine_bwd_kernel(const T *__restrict__ g, const T *__restrict__ sorted,
                                                                         const float *__restrict__ weights, const int *__restrict__ place,
                                                                         const int *__restrict__ end, long long R, int k, int C,
                                                                         T *__restrict__ d_sorted, float *__restrict__ d_weights) {
  constexpr int N = cpfn_piece<T>::N, GROUPS = MOVE_THREADS / LANES, ROWS = KT <= 2 ? 2 : 1;
  typedef typename cpfn_piece<T>::vec V;
  const int lane = threadIdx.x & (LANES - 1);
  const long long slot = (long long)blockIdx.x * GROUPS + threadIdx.x / LANES, slots = (long long)gridDim.x * GROUPS;
  // (whole row sets: the lanes of a wave stay together for the row sums)
  for (long long s0 = (long long)blockIdx.x * GROUPS; s0 < R; s0 += ROWS * slots) {
    const long long r0 = s0 + threadIdx.x / LANES;
    for (int j0 = 0; j0 < k; j0 += KT) {
      int p[ROWS][KT];
      float w[ROWS][KT], dot[ROWS][KT];
#pragma unroll
      for (int u = 0; u < ROWS; ++u)
#pragma unroll
        for (int t = 0; t < KT; ++t) {
          const long long r = r0 + u * slots;
          const bool is = r < R && j0 + t < k;
          const long long at = is ? r * k + j0 + t : 0;
          p[u][t] = is ? place[at] : -1;
          w[u][t] = weights ? weights[at] : 1.f;
          dot[u][t] = 0.f;
        }
      for (int c = lane * N; c < C; c += LANES * N) {
        V gv[ROWS], v[ROWS][KT];
#pragma unroll
        for (int u = 0; u < ROWS; ++u) {
          const long long r = r0 + u * slots;
          gv[u] = cpfn_load_piece(g + (r < R ? r : R - 1) * C, c, C);
        }
        if (d_weights) {
#pragma unroll
          for (int u = 0; u < ROWS; ++u)
#pragma unroll
            for (int t = 0; t < KT; ++t) v[u][t] = cpfn_load_piece(sorted + (long long)(p[u][t] < 0 ? 0 : p[u][t]) * C, c, C);
        }
#pragma unroll
        for (int u = 0; u < ROWS; ++u) {
          float gf[N];
          cpfn_unpack(gv[u], gf, (T *)nullptr);
#pragma unroll
          for (int t = 0; t < KT; ++t) {
            if (d_weights) {                            // (of a choice that is not there the sum is not used)
              float f[N];
              cpfn_unpack(v[u][t], f, (T *)nullptr);
#pragma unroll
              for (int i = 0; i < N; ++i) dot[u][t] = fmaf(gf[i], f[i], dot[u][t]);
            }
            if (d_sorted && p[u][t] >= 0) {
              float f[N];
#pragma unroll
              for (int i = 0; i < N; ++i) f[i] = w[u][t] * gf[i];
              cpfn_store_piece(d_sorted + (long long)p[u][t] * C, c, C, f);
            }
          }
        }
      }
      if (d_weights) {
#pragma unroll
        for (int u = 0; u < ROWS; ++u)
#pragma unroll
          for (int t = 0; t < KT; ++t) {
            const long long r = r0 + u * slots;
            const float sum = cpfn_lanes_sum<LANES>(dot[u][t]);
            if (r < R && lane == 0 && j0 + t < k) d_weights[r * k + j0 + t] = p[u][t] >= 0 ? sum : 0.f;
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
// as many workgroups as are resident together, or one row for each lane group
unsigned move_blocks(long long R, int lanes_log2) {
  const long long rows = MOVE_THREADS >> lanes_log2, b = (R + rows - 1) / rows;
  return (unsigned)(b < MOVE_BLOCKS ? b : MOVE_BLOCKS);
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
  if (mode == 2) route_scan_kernel<<<E, 256, 0, st>>>(counts, totals, tiles);
  route_rank_kernel<I><<<tiles, RANK_WAVES * 64, lds_rank, st>>>(choice, n, E, bits, tiles, mode, counts, totals, offsets, place);
  return cpfn_launch_status();
}

template <typename T> int gather(const void *rows, const int *place, const int *offsets, long long R, int k, int E, int C, void *out, hipStream_t st) {
  const int l = lanes_log2_for(C, cpfn_piece<T>::N, 8);
  const unsigned b = move_blocks(R, l);
  if (k == 1) route_gather_kernel<T, 1><<<b, MOVE_THREADS, 0, st>>>((const T *)rows, place, offsets + E, R, k, C, l, (T *)out);
  else if (k == 2) route_gather_kernel<T, 2><<<b, MOVE_THREADS, 0, st>>>((const T *)rows, place, offsets + E, R, k, C, l, (T *)out);
  else route_gather_kernel<T, 4><<<b, MOVE_THREADS, 0, st>>>((const T *)rows, place, offsets + E, R, k, C, l, (T *)out);
  return cpfn_launch_status();
}
template <typename T> int combine(const void *sorted, const float *weights, const int *place, long long R, int k, int C, void *out, hipStream_t st) {
  const int l = lanes_log2_for(C, cpfn_piece<T>::N, 8);
  const unsigned b = move_blocks(R, l);
  if (k == 1) route_combine_kernel<T, 1><<<b, MOVE_THREADS, 0, st>>>((const T *)sorted, weights, place, R, k, C, l, (T *)out);
  else if (k == 2) route_combine_kernel<T, 2><<<b, MOVE_THREADS, 0, st>>>((const T *)sorted, weights, place, R, k, C, l, (T *)out);
  else route_combine_kernel<T, 4><<<b, MOVE_THREADS, 0, st>>>((const T *)sorted, weights, place, R, k, C, l, (T *)out);
  return cpfn_launch_status();
}
template <typename T, int L>
void combine_bwd_launch(const void *g, const void *sorted, const float *weights, const int *place, const int *end, long long R, int k, int C,
                        void *d_sorted, float *d_weights, int l, hipStream_t st) {
  const unsigned b = move_blocks(R, l);
  if (k <= 2)
    route_combine_bwd_kernel<T, L, 2><<<b, MOVE_THREADS, 0, st>>>((const T *)g, (const T *)sorted, weights, place, end, R, k, C, (T *)d_sorted, d_weights);
  else
    route_combine_bwd_kernel<T, L, 4><<<b, MOVE_THREADS, 0, st>>>((const T *)g, (const T *)sorted, weights, place, end, R, k, C, (T *)d_sorted, d_weights);
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
