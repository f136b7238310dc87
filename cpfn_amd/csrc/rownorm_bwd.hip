// Backward pass of the residual block's norms, gate and residual scale (rownorm.h), in one pass over the rows.
//
// Nothing of the forward pass is kept but its inputs: out and both norms' statistics are formed again from x, y and the gate, which
// the gradients need anyway (out in fp32, as the forward pass had it).  With D = d loss / d out (its own gradient and the one through
// the next norm), hats for normalised values and means over the channels:
//   dh = d_normed next_weight,  D = d_out + r1 (dh - [mean dh] - hat1 mean(dh hat1)),   d_x = D
//   du = D scale a,  e = du weight,  d_y = r2 (e - [mean e] - hat2 mean(e hat2))   (d_y = du without a post-norm)
//   d_gate = D scale u  (times a (1 - a) behind a sigmoid), summed over the rows that share it
// [..] for layer norms only.  The parameters' gradients are column sums of four products:
//   S1 = sum D a hat2,  S2 = sum D a,  S3 = sum d_normed hat1,  S4 = sum d_normed
//   d_weight = scale S1,  d_bias = scale S2,  d_scale = weight S1 + bias S2,  d_next_weight = S3,  d_next_bias = S4
// (hat2 = y without a post-norm).  A lane owns its channels for every row of its workgroup, so a column sum is a register until
// the workgroup ends, or for SEGMENT row sets: equal terms (a mean's gradient) are rounded the same way at each of n fp32 additions, off by
// up to n 2^-24, so longer sums go to LDS in between.  The workgroups' sums are added by a second small launch in fp64, in a fixed order:
// no atomics, bit-reproducible.
// d_gate of rows that share one: the factor of the sigmoid is the same for all of them and comes after the sum.
//
// Memory bound up to 512 channels; above, registers (1024: one wave on a SIMD), the barriers of the row sums (up to six a row) and the
// workgroups' sums (16 MB) show.
// Measured (bf16, both launches):
//   131072 x 128, layer, sigmoid gate for each row    50 us   5.3 TB/s      262144 x 64, rms, no gate      39 us   5.1 TB/s
//   65536 x 512, rms, gate for each row               90 us   5.9 TB/s      100003 x 131, rms, no gate     49 us   3.2 TB/s
//   32768 x 1024, layer, gate for 2048 rows           80 us   5.0 TB/s      fp32 20528 x 259, shared gate  36 us   3.5 TB/s
//   262144 x 128, layer, gate for 32 rows             82 us   4.9 TB/s      8192 x 4096, layer, no gate    93 us   4.4 TB/s
// The kernels of the whole block without branches, against the one with them: 32768 x 1024 110 -> 100 us, 8192 x 4096 134 -> 109,
// fp32 20528 x 259 44 -> 36; of the norm in front: 32768 x 1024 57 -> 52.
#include "rownorm.h"

namespace {

template <typename T> struct NormBwd {
  const T *x, *y, *gate, *d_out, *d_normed;
  const float *weight, *bias, *scale, *next_weight;
  long long P, rows_per_gate;      // rows that share a gate row (1: a gate for every row; P with no gate)
  long long chunk;                 // rows of a workgroup (blocks_per_group > 1) ...
  int blocks_per_group;            // ... of which so many cover one gate group,
  int groups_per_block;            // or whole groups of a workgroup
  long long groups;
  int C, layer, sigmoid;
  float eps;
  T *d_x, *d_y, *d_gate;
  float *part;                     // [workgroup][4 (+ 1)][C]
  int shared_gate, sums12, sums34; // which sums are wanted
};

// sum over the row slots of a workgroup, element by element; lane `i` order of the registers -> dst[channel]
template <typename T, int L, int W, typename F> __device__ __forceinline__ void slots_sum(const float *v, float *lds, int C, F store) {
  constexpr int THREADS = NormShape<T, L, W>::THREADS, ROWS = NormShape<T, L, W>::ROWS;
  const int lane = threadIdx.x & (L - 1), slot = threadIdx.x / L;
  if (ROWS == 1) {
#pragma unroll
    for (int i = 0; i < W; ++i) {
      const int c = norm_col<T, L, W>(lane, i);
      if (c < C) store(c, v[i]);
    }
    return;
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < W; ++i) lds[slot * (L * W) + i * L + lane] = v[i];
  __syncthreads();
  for (int e = threadIdx.x; e < L * W; e += THREADS) {
    float t = 0.f;
#pragma unroll
    for (int q = 0; q < ROWS; ++q) t += lds[q * (L * W) + e];
    const int c = norm_col<T, L, W>(e & (L - 1), e / L);
    if (c < C) store(c, t);
  }
}

constexpr int SEGMENT = 128;         // row sets whose sums are added in registers (workgroups of 16 to 32 sets are what the usual sizes give)

template <typename T, int L, int W, NormMode MODE, NormForm FORM>
__global__ __launch_bounds__((NormShape<T, L, W>::THREADS)) void norm_residual_bwd_kernel(const NormBwd<T> a) {
  constexpr int ROWS = NormShape<T, L, W>::ROWS, THREADS = NormShape<T, L, W>::THREADS, NP = NormShape<T, L, W>::NP;
  __shared__ float2 slots[16];
  __shared__ float comb[ROWS > 1 ? THREADS * W : 1];
  __shared__ float held[5][THREADS * W];             // each lane's own: what its sums were before the present ones
  int turn = 0, summed = 0;                            // summed: row sets in the registers
  bool holds = false, holds_gate = false;
  const int lane = threadIdx.x & (L - 1), slot = threadIdx.x / L, C = a.C;
  const float inv_c = 1.f / (float)C;
  const bool layer = a.layer != 0, post = FORM != ANY || a.weight != nullptr, next = FORM != ANY || a.d_normed != nullptr;
  const bool has_y = FORM == FRONT ? false : FORM != ANY || a.y != nullptr;
  constexpr bool may_y = FORM != FRONT, may_own = FORM == ANY || FORM == BLOCK_OWN;       // rows that may be there
  const bool own = FORM == ANY ? a.gate != nullptr && !a.shared_gate : FORM == BLOCK_OWN;
  float sw[W], sb[W], nw[W], s1[W], s2[W], s3[W], s4[W], sg[W];
  block_params<T, L, W, MODE != WHOLE>(sw, sb, a.weight, a.bias, a.scale, lane, C);
  param_load<T, L, W, MODE != WHOLE>(nw, a.next_weight, lane, C, 1.f);
#pragma unroll
  for (int i = 0; i < W; ++i) { s1[i] = s2[i] = s3[i] = s4[i] = sg[i] = 0.f; }
  const long long g0 = a.blocks_per_group > 1 ? blockIdx.x / a.blocks_per_group : (long long)blockIdx.x * a.groups_per_block;
  long long g1 = a.blocks_per_group > 1 ? g0 + 1 : g0 + a.groups_per_block;
  if (g1 > a.groups) g1 = a.groups;
  const int nsums = 4 + (a.shared_gate && a.blocks_per_group > 1);
  const unsigned set_bytes = (unsigned)(ROWS * C) * (unsigned)sizeof(T);
  const auto hold = [&](int k, float *v, bool more) {
#pragma unroll
    for (int i = 0; i < W; ++i) {
      float *h = &held[k][i * THREADS + threadIdx.x];
      *h = more ? *h + v[i] : v[i];
      v[i] = 0.f;
    }
  };
  const auto whole = [&](int k, float *v) {
#pragma unroll
    for (int i = 0; i < W; ++i) v[i] += held[k][i * THREADS + threadIdx.x];
  };
  for (long long g = g0; g < g1; ++g) {
    long long first = g * a.rows_per_gate, last = first + a.rows_per_gate;
    if (a.blocks_per_group > 1) {
      first += (long long)(blockIdx.x % a.blocks_per_group) * a.chunk;
      if (first + a.chunk < last) last = first + a.chunk;
    }
    float gs[W];
    shared_gate<T, L, W>(gs, a.shared_gate ? a.gate + g * C : nullptr, lane, C, a.sigmoid);
    for (long long row0 = first; row0 < last; row0 += SEGMENT * ROWS) {
      const long long row1 = row0 + SEGMENT * ROWS < last ? row0 + SEGMENT * ROWS : last;
      const int sets = (int)((row1 - row0 + ROWS - 1) / ROWS);
      if (summed + sets > SEGMENT) {
        hold(0, s1, holds); hold(1, s2, holds); hold(2, s3, holds); hold(3, s4, holds);
        holds = true;
        summed = 0;
        if (row0 > first) {                              // (a gate's sum begins with its group)
          hold(4, sg, holds_gate);
          holds_gate = true;
        }
      }
      summed += sets;
      RowChunk<T, L, W, MODE> ch;
      ch.begin(row0, row1, a.P, C, lane, slot);
      const T *own_gate = own ? a.gate : nullptr;
      T *d_own_gate = own ? a.d_gate : nullptr;
      const auto bx = ch.source(next ? a.x : nullptr), by = ch.source(a.y), bg = ch.source(own_gate), bd = ch.source(a.d_out), bn = ch.source(a.d_normed);
      const auto tx = ch.target(a.d_x), ty = ch.target(a.d_y), tg = ch.target(d_own_gate);
      RowRaw<T, L, W> rx, ry, rg, rd, rn;
      unsigned o[NP], sh[NP];
      const auto request = [&](unsigned step, long long r) {
        if (MODE == EACH) {
          each_load(rx, next ? a.x : nullptr, r, lane, C, r < row1);
          if (may_y) each_load(ry, a.y, r, lane, C, r < row1);
          if (may_own) each_load(rg, own_gate, r, lane, C, r < row1);
          each_load(rd, a.d_out, r, lane, C, r < row1);
          each_load(rn, a.d_normed, r, lane, C, r < row1);
        } else {
          ch.at(o, sh, step, r < row1);
          ch.template load<true>(rx, bx, o);
          if (may_y) ch.template load<true>(ry, by, o);
          if (may_own) ch.template load<true>(rg, bg, o);
          ch.template load<true>(rd, bd, o);
          ch.template load<true>(rn, bn, o);
        }
      };
      const auto requested = [&] {
        arrived(rx);
        if (may_y) arrived(ry);
        if (may_own) arrived(rg);
        arrived(rd); arrived(rn);
      };
      arrived(sw); arrived(sb); arrived(nw);
      request(0, row0 + slot);
      requested();
      unsigned step = 0;
      for (long long base = row0; base < row1; base += ROWS, step += set_bytes) {
        const long long r = base + slot;
        const bool there = r < row1;
        const float eps = there ? a.eps : 1.f;
        float h[W], hat2[W], ga[W], D[W], dn[W], r2 = 0.f;
        ch.settle(rx, sh); ch.settle(rd, sh); ch.settle(rn, sh);
        row_unpack(rx, h);
        row_unpack(rd, D);
        row_unpack(rn, dn);
        if (may_y) {
          ch.settle(ry, sh);
          row_unpack(ry, hat2);
        }
        if (may_own) {
          ch.settle(rg, sh);
          row_unpack(rg, ga);
        }
        unpacked();
        request(step + set_bytes, r + ROWS);
        if (has_y && post) r2 = row_normalise<T, L, W, MODE>(hat2, lane, C, inv_c, layer, eps, slots, turn);
        if (own) gate_act<T, W>(ga, a.sigmoid);
        const auto gate = [&](int i) { return own ? ga[i] : gs[i]; };
        if (next) {
          if (has_y) {
#pragma unroll
            for (int i = 0; i < W; ++i) h[i] = fmaf(gate(i), fmaf(hat2[i], sw[i], sb[i]), h[i]);
          }
          const float r1 = row_normalise<T, L, W, MODE>(h, lane, C, inv_c, layer, eps, slots, turn);
          float m1 = 0.f, m2 = 0.f;
#pragma unroll
          for (int i = 0; i < W; ++i) {
            s3[i] = fmaf(dn[i], h[i], s3[i]);
            s4[i] += dn[i];
            dn[i] *= nw[i];
            m1 += dn[i];
            m2 = fmaf(dn[i], h[i], m2);
          }
          row_sum2<L>(m1, m2, slots, turn);
          m1 = layer ? m1 * inv_c : 0.f;
          m2 *= inv_c;
#pragma unroll
          for (int i = 0; i < W; ++i) D[i] = fmaf(r1, dn[i] - m1 - h[i] * m2, D[i]);
        }
        if (MODE == EACH) each_store<T, L, W>(a.d_x, r, lane, C, there, D);
        else ch.store(tx, step, D);
        float e[W], dg[W];
        if (has_y) {
          if (a.d_gate) {
#pragma unroll
            for (int i = 0; i < W; ++i) {
              dg[i] = D[i] * fmaf(hat2[i], sw[i], sb[i]);
              if (own) dg[i] *= a.sigmoid ? ga[i] * (1.f - ga[i]) : 1.f;
              else sg[i] += dg[i];
            }
          }
          float m1 = 0.f, m2 = 0.f;
#pragma unroll
          for (int i = 0; i < W; ++i) {
            const float da = D[i] * gate(i);
            s1[i] = fmaf(da, hat2[i], s1[i]);
            s2[i] += da;
            e[i] = da * sw[i];                             // (sw = scale without a post-norm: e = du)
            m1 += e[i];
            m2 = fmaf(e[i], hat2[i], m2);
          }
          if (post) {
            row_sum2<L>(m1, m2, slots, turn);
            m1 = layer ? m1 * inv_c : 0.f;
            m2 *= inv_c;
#pragma unroll
            for (int i = 0; i < W; ++i) e[i] = r2 * (e[i] - m1 - hat2[i] * m2);
          }
        }
        if (MODE == EACH) {
          if (may_own) each_store<T, L, W>(d_own_gate, r, lane, C, there, dg);
          if (may_y) each_store<T, L, W>(a.d_y, r, lane, C, there, e);
        } else {
          if (may_own) ch.store(tg, step, dg);
          if (may_y) ch.store(ty, step, e);
        }
        requested();
      }
    }
    if (a.shared_gate && a.d_gate) {
      if (holds_gate) whole(4, sg);
      holds_gate = false;
      if (a.sigmoid) {
#pragma unroll
        for (int i = 0; i < W; ++i) sg[i] *= gs[i] * (1.f - gs[i]);
      }
      if (a.blocks_per_group == 1) {                     // this workgroup has seen all rows of the gate's row
        slots_sum<T, L, W>(sg, comb, C, [&](int c, float v) { a.d_gate[g * C + c] = cpfn_from_f32<T>(v); });
#pragma unroll
        for (int i = 0; i < W; ++i) sg[i] = 0.f;
      }
    }
  }
  if (holds) { whole(0, s1); whole(1, s2); whole(2, s3); whole(3, s4); }
  float *part = a.part + (size_t)blockIdx.x * nsums * C;
  if (a.sums12) {
    slots_sum<T, L, W>(s1, comb, C, [&](int c, float v) { part[c] = v; });
    slots_sum<T, L, W>(s2, comb, C, [&](int c, float v) { part[C + c] = v; });
  }
  if (a.sums34) {
    slots_sum<T, L, W>(s3, comb, C, [&](int c, float v) { part[2 * C + c] = v; });
    slots_sum<T, L, W>(s4, comb, C, [&](int c, float v) { part[3 * C + c] = v; });
  }
  if (nsums == 5) slots_sum<T, L, W>(sg, comb, C, [&](int c, float v) { part[4 * C + c] = v; });
}

// The workgroups' sums -> gradients of the parameters (grid.y 0: S1, S2; 1: S3, S4) and of a shared gate (grid.y 2 + group).
// 16 channels x 64 subsets of workgroups: subset q adds workgroups q, q + 64, ... in fp64, then the subsets are added in order.
struct NormReduce {
  const float *part;
  int nblk, nsums, C, blocks_per_group;
  const float *weight, *bias, *scale;
  float *d_weight, *d_bias, *d_scale, *d_next_weight, *d_next_bias;
  void *d_gate;
  int wants12, wants34;
};
template <typename T> __global__ __launch_bounds__(1024) void norm_residual_reduce_kernel(const NormReduce a) {
  __shared__ double acc[64][16][2];
  const int c = blockIdx.x * 16 + (threadIdx.x & 15), q = threadIdx.x >> 4;
  const bool gate = blockIdx.y >= 2;
  if ((blockIdx.y == 0 && !a.wants12) || (blockIdx.y == 1 && !a.wants34)) return;
  const int first = gate ? (int)(blockIdx.y - 2) * a.blocks_per_group : 0, last = gate ? first + a.blocks_per_group : a.nblk;
  const int k = gate ? 4 : blockIdx.y * 2;
  double t1 = 0.0, t2 = 0.0;
  if (c < a.C) {
#pragma unroll 8
    for (int i = first + q; i < last; i += 64) {
      const float *p = a.part + ((size_t)i * a.nsums + k) * a.C + c;
      t1 += (double)p[0];
      if (!gate) t2 += (double)p[a.C];
    }
  }
  acc[q][threadIdx.x & 15][0] = t1;
  acc[q][threadIdx.x & 15][1] = t2;
  __syncthreads();
  if (q != 0 || c >= a.C) return;
  t1 = t2 = 0.0;
#pragma unroll 8
  for (int i = 0; i < 64; ++i) { t1 += acc[i][threadIdx.x][0]; t2 += acc[i][threadIdx.x][1]; }
  if (gate) {
    ((T *)a.d_gate)[(size_t)(blockIdx.y - 2) * a.C + c] = cpfn_from_f32<T>((float)t1);
  } else if (blockIdx.y == 0) {
    const double sc = a.scale ? (double)a.scale[c] : 1.0;
    if (a.d_weight) a.d_weight[c] = (float)(sc * t1);
    if (a.d_bias) a.d_bias[c] = (float)(sc * t2);
    if (a.d_scale) a.d_scale[c] = (float)((a.weight ? (double)a.weight[c] : 1.0) * t1 + (a.bias ? (double)a.bias[c] * t2 : 0.0));
  } else {
    if (a.d_next_weight) a.d_next_weight[c] = (float)t1;
    if (a.d_next_bias) a.d_next_bias[c] = (float)t2;
  }
}

// Two waves on each SIMD run at once (one with 16 channels a lane); at least four row sets for each workgroup, or its sums cost as much
// as its rows.  (Where three waves fit the registers they measured 0 to 30 % slower: more workgroups' sums, and two keep enough rows in
// flight.)
NormSplit split(long long P, int C, int W, long long gate_rows) { return norm_split(P, C, W, gate_rows, 2048, 4); }

template <typename T, int L, int W, NormForm FORM> void launch_form(const NormBwd<T> &a, int nblk, NormMode mode, hipStream_t st) {
  constexpr int THREADS = NormShape<T, L, W>::THREADS;
  if (W == 16 || mode == WHOLE) norm_residual_bwd_kernel<T, L, W, WHOLE, FORM><<<nblk, THREADS, 0, st>>>(a);
  else if constexpr (W == 8) norm_residual_bwd_kernel<T, L, W, RAGGED, FORM><<<nblk, THREADS, 0, st>>>(a);
}
template <typename T, int L, int W> void launch(const NormBwd<T> &a, int nblk, NormMode mode, hipStream_t st) {
  if (!a.d_normed || (a.y && !a.weight)) launch_form<T, L, W, ANY>(a, nblk, mode, st);
  else if (!a.y) launch_form<T, L, W, FRONT>(a, nblk, mode, st);
  else if (a.gate && !a.shared_gate) launch_form<T, L, W, BLOCK_OWN>(a, nblk, mode, st);
  else launch_form<T, L, W, BLOCK>(a, nblk, mode, st);
}

struct Grads { float *d_weight, *d_bias, *d_scale, *d_next_weight, *d_next_bias; };

template <typename T>
int backward(const void *x, const void *y, const void *gate, const float *weight, const float *bias, const float *scale,
             const float *next_weight, const void *d_out, const void *d_normed, long long P, int C, long long gate_rows, int layer,
             int sigmoid, float eps, void *d_x, void *d_y, void *d_gate, const Grads &d, float *workspace, hipStream_t st) {
  const int W = norm_width(C, sizeof(T));
  const NormSplit s = split(P, C, W, gate_rows);
  NormBwd<T> a;
  a.x = (const T *)x; a.y = (const T *)y; a.gate = (const T *)gate; a.d_out = (const T *)d_out; a.d_normed = (const T *)d_normed;
  a.weight = weight; a.bias = bias; a.scale = scale; a.next_weight = next_weight;
  a.P = P; a.rows_per_gate = s.rows_per_gate; a.chunk = s.chunk; a.blocks_per_group = s.blocks_per_group;
  a.groups_per_block = s.groups_per_block; a.groups = s.groups;
  a.C = C; a.layer = layer; a.sigmoid = sigmoid; a.eps = eps;
  a.d_x = (T *)d_x; a.d_y = (T *)d_y; a.d_gate = (T *)d_gate;
  a.part = workspace;
  a.shared_gate = gate && gate_rows < P;
  a.sums12 = d.d_weight || d.d_bias || d.d_scale;
  a.sums34 = d.d_next_weight || d.d_next_bias;
  const NormMode mode = norm_mode<T>(P, C);
  if (mode == EACH) {
    norm_residual_bwd_kernel<T, 8, 8, EACH, ANY><<<s.nblk, 256, 0, st>>>(a);
  } else if (W == 16) {
    if constexpr (sizeof(T) == 2) launch<T, 64, 16>(a, s.nblk, mode, st);
  } else {
    switch (norm_lanes(C, W)) {
      case 8: launch<T, 8, 8>(a, s.nblk, mode, st); break;
      case 16: launch<T, 16, 8>(a, s.nblk, mode, st); break;
      case 32: launch<T, 32, 8>(a, s.nblk, mode, st); break;
      case 64: launch<T, 64, 8>(a, s.nblk, mode, st); break;
      case 128: launch<T, 128, 8>(a, s.nblk, mode, st); break;
      case 256: launch<T, 256, 8>(a, s.nblk, mode, st); break;
      default: launch<T, 512, 8>(a, s.nblk, mode, st); break;
    }
  }
  const bool gate_part = a.shared_gate && d_gate && s.blocks_per_group > 1;
  if (a.sums12 || a.sums34 || gate_part) {
    NormReduce r;
    r.part = workspace; r.nblk = s.nblk; r.nsums = 4 + (a.shared_gate && s.blocks_per_group > 1); r.C = C;
    r.blocks_per_group = s.blocks_per_group;
    r.weight = weight; r.bias = bias; r.scale = scale;
    r.d_weight = d.d_weight; r.d_bias = d.d_bias; r.d_scale = d.d_scale; r.d_next_weight = d.d_next_weight; r.d_next_bias = d.d_next_bias;
    r.d_gate = d_gate; r.wants12 = a.sums12; r.wants34 = a.sums34;
    norm_residual_reduce_kernel<T><<<dim3(cpfn_cdiv(C, 16), 2 + (gate_part ? (unsigned)s.groups : 0)), 1024, 0, st>>>(r);
  }
  return cpfn_launch_status();
}

}  // namespace

extern "C" long long cpfn_norm_residual_workspace(long long P, int C, long long gate_rows) {
  if (P < 0 || C < 1 || C > CPFN_NORM_MAX_C || gate_rows < 0 || (gate_rows > 0 && P % gate_rows != 0)) return -1;
  if (P == 0) return 0;
  const int a = split(P, C, norm_width(C, 2), gate_rows).nblk, b = split(P, C, norm_width(C, 4), gate_rows).nblk;
  return (long long)(a > b ? a : b) * 5 * C * (long long)sizeof(float);
}

extern "C" int cpfn_norm_residual_bwd(const void *x, const void *y, const void *gate, const float *weight, const float *bias,
                                      const float *scale, const float *next_weight, const void *d_out, const void *d_normed,
                                      long long P, int C, long long gate_rows, int dtype, int layer, int sigmoid, float eps, void *d_x,
                                      void *d_y, void *d_gate, float *d_weight, float *d_bias, float *d_scale, float *d_next_weight,
                                      float *d_next_bias, void *workspace, void *stream) {
  if (P < 0 || C < 1 || C > CPFN_NORM_MAX_C || !(eps >= 0.f) || (d_normed && (!next_weight || !x)) || (bias && !weight) ||
      (!y && (gate || weight || scale || d_y || d_weight || d_scale)) || (d_weight && !weight) || (d_bias && !weight) ||
      (d_scale && !scale) || ((d_next_weight || d_next_bias) && !d_normed) || (d_gate && !gate))
    return CPFN_EINVAL;
  if (gate && (gate_rows < 1 || P % gate_rows != 0)) return CPFN_EINVAL;
  if (P == 0 || (!d_out && !d_normed) || !workspace) return CPFN_EINVAL;
  const Grads d = {d_weight, d_bias, d_scale, d_next_weight, d_next_bias};
  if (!gate) gate_rows = 0;
  hipStream_t st = (hipStream_t)stream;
  float *ws = (float *)workspace;
  switch (dtype) {
    case CPFN_F32: return backward<float>(x, y, gate, weight, bias, scale, next_weight, d_out, d_normed, P, C, gate_rows, layer, sigmoid, eps, d_x, d_y, d_gate, d, ws, st);
    case CPFN_BF16: return backward<cpfn_bf16>(x, y, gate, weight, bias, scale, next_weight, d_out, d_normed, P, C, gate_rows, layer, sigmoid, eps, d_x, d_y, d_gate, d, ws, st);
    case CPFN_F16: return backward<cpfn_f16>(x, y, gate, weight, bias, scale, next_weight, d_out, d_normed, P, C, gate_rows, layer, sigmoid, eps, d_x, d_y, d_gate, d, ws, st);
  }
  return CPFN_EINVAL;
}
