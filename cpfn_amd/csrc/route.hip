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
// A workgroup ranks a tile of consecutive choices; a wave takes a contiguous part of them, 64 at a time.  Rank inside 64: the lanes with
// the same expert are found by one ballot for each bit of the index; the first such lane adds their number to the wave's own LDS
// counter of that expert: no atomics, so the order is the input's order by construction.
// ITEMS: 64-choice steps of a wave.  4 up to RANK_SMALL choices (more workgroups: 60000 choices, 28 experts 10.6 -> 8.3 us), 8 above (fewer
// counts to scan: 4000000 choices, 2000 experts 57 -> 44 us; 4194304, 128: 30.9 -> 30.5).
//
// Measured: 4194304 choices, 128 experts 28 us (count 8, scan 5.5, ranks 14.5), 1.8 TB/s of choices and places (a choice is read twice; the
// ranks' arithmetic is 4 of a call's 26); 4000000, 2000 experts 37 us (6, 11, 21); 60000, 28 experts 8.2 us, two launches.
constexpr int RANK_WAVES = 8;
constexpr long long RANK_SMALL = 1 << 19;
constexpr int rank_tile(int items) { return RANK_WAVES * items * 64; }
int rank_items(long long n) { return n <= RANK_SMALL ? 4 : 8; }
constexpr int ROUTE_MAX_E = 2048;                 // a 16-bit counter for each wave (a tile has 4096 choices at most) and a base: 40 KB of LDS
// Every workgroup sums the tiles' counts by itself, instead of a launch that does it once, where a wave loads up to 8 times for it (64
// tiles of an expert each time; of 8 waves): 262144 choices, 8 experts 7.5 us (launch: 9.6), 64 experts 11.0 (10.2); 130000, 128 11.7 (10.0)
constexpr int DIRECT_LOADS = 64;

template <typename I> __device__ __forceinline__ int expert_of(const I *__restrict__ choice, long long i, long long n, int E) {
  if (i >= n) return -1;
  const I v = choice[i];
  return v >= 0 && v < (I)E ? (int)v : -1;
}

// the ranks of a wave's choices among the wave's own; `mine`: the wave's counters, zero before, the wave's counts afterwards
template <int RANK_ITEMS> __device__ __forceinline__ void wave_ranks(const int *e, int *rank, unsigned short *mine, int bits) {
#pragma unroll
  for (int t = 0; t < RANK_ITEMS; ++t) {
    // the lanes whose expert is this lane's: for each bit, those whose bit is its own (of lanes that have an expert)
    const unsigned long long valid = __ballot(e[t] >= 0);
    unsigned lo = (unsigned)valid, hi = (unsigned)(valid >> 32);
    for (int b = 0; b < bits; ++b) {
      const unsigned own = (unsigned)__builtin_amdgcn_sbfe(e[t], b, 1);           // all ones: my bit is set
      const unsigned long long v = __ballot(own != 0u);
      lo &= ~((unsigned)v ^ own);
      hi &= ~((unsigned)(v >> 32) ^ own);
    }
    const int ahead = (int)__builtin_amdgcn_mbcnt_hi(hi, __builtin_amdgcn_mbcnt_lo(lo, 0u));      // of them, those before this lane
    rank[t] = 0;
    if (e[t] >= 0) {
      const int before = mine[e[t]];
      rank[t] = before + ahead;
      if (ahead == 0) mine[e[t]] = (unsigned short)(before + __popc(lo) + __popc(hi));
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");      // the next 64 read what these wrote
    __builtin_amdgcn_wave_barrier();
  }
}

__device__ __forceinline__ void zero_counters(unsigned short *cnt, int E) {       // (E counters of RANK_WAVES waves: whole words)
  for (int i = threadIdx.x; i < RANK_WAVES * E / 2; i += RANK_WAVES * 64) ((unsigned *)cnt)[i] = 0u;
  __syncthreads();
}

// counts[tile][e] (several tiles only): a histogram by LDS additions, whose order does not show in an integer
template <typename I, int RANK_ITEMS>
__global__ __launch_bounds__(RANK_WAVES * 64) void route_count_kernel(const I *__restrict__ choice, long long n, int E,
                                                                      int *__restrict__ counts) {
  extern __shared__ unsigned lds[];               // [E]
  for (int x = threadIdx.x; x < E; x += RANK_WAVES * 64) lds[x] = 0u;
  const long long i0 = (long long)blockIdx.x * rank_tile(RANK_ITEMS) + threadIdx.x;
  int e[RANK_ITEMS];
#pragma unroll
  for (int t = 0; t < RANK_ITEMS; ++t) e[t] = expert_of(choice, i0 + t * (RANK_WAVES * 64), n, E);
  __syncthreads();
#pragma unroll
  for (int t = 0; t < RANK_ITEMS; ++t)
    if (e[t] >= 0) atomicAdd(&lds[e[t]], 1u);
  __syncthreads();
  for (int x = threadIdx.x; x < E; x += RANK_WAVES * 64) counts[(long long)blockIdx.x * E + x] = (int)lds[x];
}

// inclusive sums over a wave (in registers: six exchanges through LDS cost 0.5 to 3 us of a list's order): inside rows of 16 lanes, then each row's last sum into the rows behind it
template <int CTRL, int ROWS> __device__ __forceinline__ int moved_up(int v) { return __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xf, false); }
__device__ __forceinline__ int wave_scan(int v) {
  v += moved_up<0x111, 0xf>(v);                   // row_shr 1, 2, 4, 8
  v += moved_up<0x112, 0xf>(v);
  v += moved_up<0x114, 0xf>(v);
  v += moved_up<0x118, 0xf>(v);
  v += moved_up<0x142, 0xa>(v);                   // lane 15 to row 1, lane 47 to row 3
  v += moved_up<0x143, 0xc>(v);                   // lane 31 to rows 2 and 3
  return v;
}

// counts[0..tiles)[e] -> exclusive sums over the tiles, totals[e]: 16 experts x 64 stretches of tiles for each workgroup
__global__ __launch_bounds__(1024) void route_scan_kernel(int *__restrict__ counts, int *__restrict__ totals, int E, int tiles) {
  __shared__ int part[64][17];
  const int x = threadIdx.x & 15, q = threadIdx.x >> 4, e = blockIdx.x * 16 + x;
  const int per = (tiles + 63) / 64, t0 = q * per, t1 = t0 + per < tiles ? t0 + per : tiles;
  int s = 0;
  if (e < E) {
#pragma unroll 16
    for (int t = t0; t < t1; ++t) s += counts[(long long)t * E + e];
  }
  part[q][x] = s;
  __syncthreads();
  {                                                // a wave for each expert: the stretches' sums -> exclusive
    const int lane = threadIdx.x & 63, wx = threadIdx.x >> 6;
    const int v = part[lane][wx], up_to = wave_scan(v);
    part[lane][wx] = up_to - v;
    if (lane == 63 && blockIdx.x * 16 + wx < E) totals[blockIdx.x * 16 + wx] = up_to;
  }
  __syncthreads();
  if (e >= E) return;
  s = part[q][x];
  for (int t = t0; t < t1; t += 16) {
    int v[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = t + i < t1 ? counts[(long long)(t + i) * E + e] : 0;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      if (t + i < t1) counts[(long long)(t + i) * E + e] = s;
      s += v[i];
    }
  }
}

// mode 0: one tile (its own counts are all there is); 1: sums the tiles' counts itself; 2: counts are exclusive sums, totals given
template <typename I, int RANK_ITEMS>
__global__ __launch_bounds__(RANK_WAVES * 64) void route_rank_kernel(const I *__restrict__ choice, long long n, int E, int bits, int tiles,
                                                                     int mode, const int *__restrict__ counts,
                                                                     const int *__restrict__ totals, int *__restrict__ offsets,
                                                                     int *__restrict__ place) {
  extern __shared__ unsigned lds[];               // [waves][E] 16-bit counters | [E] first position of this tile's
  __shared__ int wsum[RANK_WAVES], d_before[DIRECT_LOADS], d_total[DIRECT_LOADS];
  constexpr int THREADS = RANK_WAVES * 64;
  unsigned short *cnt = (unsigned short *)lds;
  int *base = (int *)(lds + RANK_WAVES * E / 2);
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const long long i0 = (long long)blockIdx.x * rank_tile(RANK_ITEMS) + wave * (RANK_ITEMS * 64) + lane;
  unsigned short *mine = cnt + wave * E;
  int e[RANK_ITEMS], rank[RANK_ITEMS];
#pragma unroll
  for (int t = 0; t < RANK_ITEMS; ++t) e[t] = expert_of(choice, i0 + t * 64, n, E);
  if (mode == 1) {                                // a wave for each expert, its lanes share out the tiles
    for (int x = wave; x < E; x += RANK_WAVES) {
      int before = 0, total = 0;
#pragma unroll 4
      for (int t = lane; t < tiles; t += 64) {
        const int v = counts[t * E + x];
        total += v;
        before += t < (int)blockIdx.x ? v : 0;
      }
      total = wave_scan(total);
      before = wave_scan(before);
      if (lane == 63) { d_total[x] = total; d_before[x] = before; }
    }
  }
  zero_counters(cnt, E);
  wave_ranks<RANK_ITEMS>(e, rank, mine, bits);
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
      before = mode == 0 ? 0 : mode == 1 ? d_before[x] : counts[(long long)blockIdx.x * E + x];
    }
    const int s = wave_scan(total);
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
// One row for each group of lanes of a launch (up to MOVE_BLOCKS workgroups; several rows in flight for a group, with fewer
// workgroups, measured 0 to 40 % slower at 131072 x 128 .. 50000 x 1024 rows: the chip holds enough groups).  A row is walked in
// 16-byte pieces; the last piece of a row whose length is no multiple of one ENDS with the row and overlaps the piece before it: its
// lane moves (or computes) a few elements that another lane moves too, to the same value.  Rows shorter than a piece go element by element.
// Memory bound.  Measured (bf16): 131072 x 128 to 2 of 8: gather 20 us, combine 21, its adjoint 30 (5.2, 5.0, 5.7 TB/s); 50000 x 1024 to 4
// of 64: 91, 90, 173 us (5.6, 5.7, 5.3); fp32 30000 x 259 to 3 of 64: 33, 32, 47 (3.8, 3.9, 4.6).
constexpr int MOVE_THREADS = 256;
constexpr long long MOVE_BLOCKS = 1 << 20;
constexpr int MOVE_MAX_C = 1 << 30;               // (a row is walked with 32-bit steps of up to 2048 elements)

struct Walk {                     // 1 << lanes_log2 lanes for a row
  int lanes, lane;
  long long slot, slots;
  __device__ __forceinline__ explicit Walk(int lanes_log2) {
    lanes = 1 << lanes_log2;
    lane = threadIdx.x & (lanes - 1);
    slot = (long long)blockIdx.x * (MOVE_THREADS >> lanes_log2) + (threadIdx.x >> lanes_log2);
    slots = (long long)gridDim.x * (MOVE_THREADS >> lanes_log2);
  }
};
template <typename T> __device__ __forceinline__ int piece_at(int c, int C) { return c + cpfn_piece<T>::N <= C ? c : C - cpfn_piece<T>::N; }

// rows behind the last expert's, [offsets[E], n): zero, shared out over all row slots of the launch
template <typename T>
__device__ __forceinline__ void zero_tail(T *__restrict__ out, const int *__restrict__ end, long long n, int C, int lane, int lanes,
                                          long long slot, long long slots) {
  constexpr int N = cpfn_piece<T>::N;
  const typename cpfn_piece<T>::vec z = {};
  for (long long p = (*end < 0 ? 0 : *end) + slot; p < n; p += slots)
    for (int c = lane * N; c < C; c += lanes * N) {
      if (C >= N) *(typename cpfn_piece<T>::vec *)(out + p * C + piece_at<T>(c, C)) = z;
      else
        for (int q = 0; q < C; ++q) out[p * C + q] = cpfn_from_f32<T>(0.f);
    }
}

// A place that is not one of the n sorted rows (-1; anything else only in tensors that no plan left) is a choice that is not there.
__device__ __forceinline__ int place_of(const int *__restrict__ place, long long at, long long n) {
  const int p = place[at];
  return (unsigned)p < (unsigned)n ? p : -1;
}

// KT: choices of a row that are taken at once (their places in flight together)
template <typename T, int KT>
__global__ __launch_bounds__(MOVE_THREADS) void route_gather_kernel(const T *__restrict__ rows, const int *__restrict__ place,
                                                                    const int *__restrict__ end, long long R, int k, int C, int lanes_log2,
                                                                    T *__restrict__ out) {
  constexpr int N = cpfn_piece<T>::N;
  typedef typename cpfn_piece<T>::vec V;                // (bits are moved, not values: NaNs keep theirs)
  const Walk w(lanes_log2);
  for (long long r = w.slot; r < R; r += w.slots) {
    for (int j0 = 0; j0 < k; j0 += KT) {
      int p[KT];
#pragma unroll
      for (int t = 0; t < KT; ++t) p[t] = j0 + t < k ? place_of(place, r * k + j0 + t, R * k) : -1;
      for (int c = w.lane * N; c < C; c += w.lanes * N) {
        if (C >= N) {
          const int at = piece_at<T>(c, C);
          const V v = *(const V *)(rows + r * C + at);
#pragma unroll
          for (int t = 0; t < KT; ++t)
            if (p[t] >= 0) __builtin_nontemporal_store(v, (V *)(out + (long long)p[t] * C + at));
        } else {
          for (int q = 0; q < C; ++q) {
            const T v = rows[r * C + q];
#pragma unroll
            for (int t = 0; t < KT; ++t)
              if (p[t] >= 0) out[(long long)p[t] * C + q] = v;
          }
        }
      }
    }
  }
  zero_tail(out, end, R * k, C, w.lane, w.lanes, w.slot, w.slots);
}

// a piece as floats, zeros behind a row shorter than a piece
template <typename T> __device__ __forceinline__ void piece_get(const T *__restrict__ row, int at, int C, typename cpfn_piece<T>::vec &v) {
  if (C >= cpfn_piece<T>::N) v = *(const typename cpfn_piece<T>::vec *)(row + at);
  else v = cpfn_load_piece(row, 0, C);
}
template <typename T> __device__ __forceinline__ void piece_put(T *__restrict__ row, int at, int C, const float *f) {
  if (C >= cpfn_piece<T>::N) __builtin_nontemporal_store(cpfn_pack(f, (T *)nullptr), (typename cpfn_piece<T>::vec *)(row + at));
  else cpfn_store_piece(row, 0, C, f);
}

template <typename T, int KT>
__global__ __launch_bounds__(MOVE_THREADS) void route_combine_kernel(const T *__restrict__ sorted, const float *__restrict__ weights,
                                                                     const int *__restrict__ place, long long R, int k, int C,
                                                                     int lanes_log2, T *__restrict__ out) {
  constexpr int N = cpfn_piece<T>::N;
  const Walk walk(lanes_log2);
  for (long long r = walk.slot; r < R; r += walk.slots) {
    int p[KT];
    float w[KT];
    const auto choices = [&](int j0) {
#pragma unroll
      for (int t = 0; t < KT; ++t) {
        const bool is = j0 + t < k;
        const long long at = r * k + (is ? j0 + t : 0);
        p[t] = is ? place_of(place, at, R * k) : -1;
        w[t] = weights ? weights[at] : 1.f;
      }
    };
    choices(0);
    for (int c = walk.lane * N; c < C; c += walk.lanes * N) {
      const int here = C >= N ? piece_at<T>(c, C) : 0;
      float acc[N];
#pragma unroll
      for (int i = 0; i < N; ++i) acc[i] = 0.f;
      for (int j0 = 0; j0 < k; j0 += KT) {
        if (k > KT) choices(j0);
        typename cpfn_piece<T>::vec v[KT];
#pragma unroll
        for (int t = 0; t < KT; ++t) piece_get(sorted + (long long)(p[t] < 0 ? 0 : p[t]) * C, here, C, v[t]);
#pragma unroll
        for (int t = 0; t < KT; ++t) {
          float f[N];
          cpfn_unpack(v[t], f, (T *)nullptr);
          const bool is = p[t] >= 0;                    // (a choice that is not there adds nothing, whatever stands in its places)
#pragma unroll
          for (int i = 0; i < N; ++i) acc[i] = is ? fmaf(w[t], f[i], acc[i]) : acc[i];
        }
      }
      piece_put(out + r * C, here, C, acc);
    }
  }
}

// LANES <= 64: the products of a row meet inside a wave.  A lane has two pieces of a row in flight: against one, with twice the lanes,
// fp32 30000 x 259 to 3 of 64 69 -> 56 us, fp32 8000 x 1100 48 -> 43, 262144 x 256 to one 77 -> 73, 131072 x 128 31.9 -> 30.2 (30000 x 512
// to 8 of 64 105.5 -> 107.6).
constexpr int STEPS = 2;
template <typename T, int LANES, int KT>
__global__ __launch_bounds__(MOVE_THREADS) void route_combine_bwd_kernel(const T *__restrict__ g, const T *__restrict__ sorted,
                                                                         const float *__restrict__ weights, const int *__restrict__ place,
                                                                         const int *__restrict__ end, long long R, int k, int C,
                                                                         T *__restrict__ d_sorted, float *__restrict__ d_weights) {
  constexpr int N = cpfn_piece<T>::N, GROUPS = MOVE_THREADS / LANES;
  typedef typename cpfn_piece<T>::vec V;
  const int lane = threadIdx.x & (LANES - 1);
  const long long slot = (long long)blockIdx.x * GROUPS + threadIdx.x / LANES, slots = (long long)gridDim.x * GROUPS;
  // (whole row sets: the lanes of a wave stay together for the row sums)
  for (long long s0 = (long long)blockIdx.x * GROUPS; s0 < R; s0 += slots) {
    const long long r = s0 + threadIdx.x / LANES;
    const bool row = r < R;
    for (int j0 = 0; j0 < k; j0 += KT) {
      int p[KT];
      float w[KT], dot[KT];
#pragma unroll
      for (int t = 0; t < KT; ++t) {
        const bool is = row && j0 + t < k;
        const long long at = is ? r * k + j0 + t : 0;
        p[t] = is ? place_of(place, at, R * k) : -1;
        w[t] = weights ? weights[at] : 1.f;
        dot[t] = 0.f;
      }
      for (int c0 = lane * N; c0 < C; c0 += STEPS * LANES * N) {
        int here[STEPS], skip[STEPS];                     // skip: first elements, which the lane before has too (all: a step behind the row)
        V gv[STEPS], v[STEPS][KT];
#pragma unroll
        for (int u = 0; u < STEPS; ++u) {
          const int c = c0 + u * LANES * N;
          here[u] = C >= N ? piece_at<T>(c, C) : 0;
          skip[u] = c < C ? c - here[u] : N;
          piece_get(g + (row ? r : 0) * C, here[u], C, gv[u]);
          if (d_weights) {
#pragma unroll
            for (int t = 0; t < KT; ++t) piece_get(sorted + (long long)(p[t] < 0 ? 0 : p[t]) * C, here[u], C, v[u][t]);
          }
        }
#pragma unroll
        for (int u = 0; u < STEPS; ++u) {
          float gf[N];
          cpfn_unpack(gv[u], gf, (T *)nullptr);
#pragma unroll
          for (int t = 0; t < KT; ++t) {
            if (d_weights) {                              // (of a choice that is not there the sum is not used)
              float f[N];
              cpfn_unpack(v[u][t], f, (T *)nullptr);
#pragma unroll
              for (int i = 0; i < N; ++i) dot[t] = i >= skip[u] ? fmaf(gf[i], f[i], dot[t]) : dot[t];
            }
            if (d_sorted && p[t] >= 0 && skip[u] < N) {
              float f[N];
#pragma unroll
              for (int i = 0; i < N; ++i) f[i] = w[t] * gf[i];
              piece_put(d_sorted + (long long)p[t] * C, here[u], C, f);
            }
          }
        }
      }
      if (d_weights) {
#pragma unroll
        for (int t = 0; t < KT; ++t) {
          const float sum = cpfn_lanes_sum<LANES>(dot[t]);
          if (row && lane == 0 && j0 + t < k) d_weights[r * k + j0 + t] = p[t] >= 0 ? sum : 0.f;
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
// The same for the sums over a row's choices, whose lanes hold several pieces at once: fewer lanes and more steps where a last, nearly
// empty step would leave half of the lanes idle (fp32 259 channels 40 -> 29 us, bf16 520 21 -> 18, fp32 131 12.3 -> 11.3).  The copies are
// slower for it (fp32 131 11 -> 16 us), the adjoints as fast or slower.
int lanes_log2_sparing(int C, int per_lane, int most) {
  const int l = lanes_log2_for(C, per_lane, most), pieces = (C + per_lane - 1) / per_lane;
  for (int m = l; m >= 4; --m)
    if (((long long)(pieces + (1 << m) - 1) >> m << m) * 2 <= 3ll * pieces) return m;
  return l;
}
unsigned move_blocks(long long R, int lanes_log2) {
  const long long rows = MOVE_THREADS >> lanes_log2, b = (R + rows - 1) / rows;
  return (unsigned)(b < MOVE_BLOCKS ? b : MOVE_BLOCKS);
}

int tiles_of(long long n) {
  const int tile = rank_tile(rank_items(n));
  return n > tile ? (int)((n + tile - 1) / tile) : 1;
}

template <typename I, int ITEMS>
int plan(const I *choice, long long n, int E, int *offsets, int *place, int *ws, hipStream_t st) {
  const int tiles = tiles_of(n);
  int bits = 0;
  while ((1 << bits) < E) ++bits;
  const size_t lds_rank = (size_t)RANK_WAVES * E * 2 + (size_t)E * 4;
  const int mode = tiles == 1 ? 0 : (long long)E * ((tiles + 63) / 64) <= DIRECT_LOADS ? 1 : 2;
  int *counts = ws, *totals = ws + (size_t)tiles * E;
  if (mode) route_count_kernel<I, ITEMS><<<tiles, RANK_WAVES * 64, (size_t)E * 4, st>>>(choice, n, E, counts);
  if (mode == 2) route_scan_kernel<<<cpfn_cdiv(E, 16), 1024, 0, st>>>(counts, totals, E, tiles);
  route_rank_kernel<I, ITEMS><<<tiles, RANK_WAVES * 64, lds_rank, st>>>(choice, n, E, bits, tiles, mode, counts, totals, offsets, place);
  return cpfn_launch_status();
}
template <typename I> int plan(const I *choice, long long n, int E, int *offsets, int *place, int *ws, hipStream_t st) {
  return rank_items(n) == 4 ? plan<I, 4>(choice, n, E, offsets, place, ws, st) : plan<I, 8>(choice, n, E, offsets, place, ws, st);
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
  const int l = lanes_log2_sparing(C, cpfn_piece<T>::N, 8);
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
  const int l = lanes_log2_for(C, cpfn_piece<T>::N * STEPS, 6);
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
  return R < 0 || k < 1 || E < 1 || E > ROUTE_MAX_E || C < 1 || C > MOVE_MAX_C || R > 0x7fffffffll / k;
}

}  // namespace

extern "C" long long cpfn_route_workspace(long long n, int E) {
  if (n < 0 || n > 0x7fffffffll || E < 1 || E > ROUTE_MAX_E) return -1;
  const long long tiles = tiles_of(n);
  return tiles <= 1 ? 0 : (tiles + 1) * E * (long long)sizeof(int);
}

extern "C" int cpfn_route_plan(const void *choice, int wide, long long n, int E, int *offsets, int *place, void *workspace, void *stream) {
  if (bad_sizes(n, 1, E, 1) || !offsets || (n > 0 && (!choice || !place)) || (tiles_of(n) > 1 && !workspace)) return CPFN_EINVAL;
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
