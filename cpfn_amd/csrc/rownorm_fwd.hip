// Norms before and after a residual block, its gate and its residual scale in one pass over the rows (forward; the formulas are in
// rownorm.h).  Memory bound: x, y and the gate are read once, out and normed written once; the op-by-op form moves each of the ~12
// intermediate tensors through memory.  Measured (bf16; a copy of gigabytes reaches 4.9 TB/s, one that fits the last-level cache 8.6):
//   131072 x 128, layer, sigmoid gate for each row    33 us   5.1 TB/s      262144 x 64, rms, no gate      26 us   5.1 TB/s
//   65536 x 512, rms, gate for each row               61 us   5.5 TB/s      100003 x 131, rms, no gate     30 us   3.5 TB/s
//   32768 x 1024, layer, gate for 2048 rows           51 us   5.3 TB/s      fp32 20528 x 259, shared gate  20 us   4.2 TB/s
//   262144 x 128, layer, gate for 32 rows             52 us   5.2 TB/s      8192 x 4096, layer, no gate    51 us   5.3 TB/s
// Ragged rows cost instructions (masks of the last piece, three more stores).
#include "rownorm.h"

namespace {

template <typename T> struct NormFwd {
  const T *x, *y, *gate;
  const float *weight, *bias, *scale, *next_weight, *next_bias;
  long long P, rows_per_gate, groups, chunk;
  int blocks_per_group, groups_per_block, shared_gate;
  int C, layer, sigmoid;
  float eps;
  T *out, *normed;
};

template <typename T, int L, int W, NormMode MODE, NormForm FORM>
__global__ __launch_bounds__((NormShape<T, L, W>::THREADS)) void norm_residual_fwd_kernel(const NormFwd<T> a) {
  constexpr int ROWS = NormShape<T, L, W>::ROWS, NP = NormShape<T, L, W>::NP;
  __shared__ float2 slots[16];
  int turn = 0;
  const int lane = threadIdx.x & (L - 1), slot = threadIdx.x / L, C = a.C;
  const float inv_c = 1.f / (float)C;
  const bool layer = a.layer != 0, post = FORM != ANY || a.weight != nullptr, has_y = FORM != ANY || a.y != nullptr, next = FORM != ANY || a.normed != nullptr;
  const bool own = FORM == ANY ? a.gate != nullptr && !a.shared_gate : FORM == BLOCK_OWN;
  float sw[W], sb[W], nw[W], nb[W];
  block_params<T, L, W, MODE != WHOLE>(sw, sb, a.weight, a.bias, a.scale, lane, C);
  param_load<T, L, W, MODE != WHOLE>(nw, a.next_weight, lane, C, 1.f);
  param_load<T, L, W, MODE != WHOLE>(nb, a.next_bias, lane, C, 0.f);
  const long long g0 = a.blocks_per_group > 1 ? blockIdx.x / a.blocks_per_group : (long long)blockIdx.x * a.groups_per_block;
  long long g1 = a.blocks_per_group > 1 ? g0 + 1 : g0 + a.groups_per_block;
  if (g1 > a.groups) g1 = a.groups;
  const unsigned set_bytes = (unsigned)(ROWS * C) * (unsigned)sizeof(T);
  for (long long g = g0; g < g1; ++g) {
    long long row0 = g * a.rows_per_gate, row1 = row0 + a.rows_per_gate;
    if (a.blocks_per_group > 1) {
      row0 += (long long)(blockIdx.x % a.blocks_per_group) * a.chunk;
      if (row0 + a.chunk < row1) row1 = row0 + a.chunk;
    }
    RowChunk<T, L, W, MODE> ch;
    ch.begin(row0, row1, a.P, C, lane, slot);
    const T *own_gate = own ? a.gate : nullptr;
    const auto sx = ch.source(a.x), sy = ch.source(a.y), sg = ch.source(own_gate);
    const auto to = ch.target(a.out), tn = ch.target(a.normed);
    RowRaw<T, L, W> rx, ry, rg;
    unsigned o[NP], sh[NP];
    const auto request = [&](unsigned step, long long r) {
      if (MODE == EACH) {
        each_load(rx, a.x, r, lane, C, r < row1);
        each_load(ry, a.y, r, lane, C, r < row1);
        if (FORM != BLOCK) each_load(rg, own_gate, r, lane, C, r < row1);
      } else {
        ch.at(o, sh, step, r < row1);
        ch.load(rx, sx, o);
        ch.load(ry, sy, o);
        if (FORM != BLOCK) ch.load(rg, sg, o);
      }
    };
    float gs[W];
    shared_gate<T, L, W>(gs, a.shared_gate ? a.gate + g * C : nullptr, lane, C, a.sigmoid);
    arrived(sw); arrived(sb); arrived(nw); arrived(nb);
    request(0, row0 + slot);
    arrived(rx); arrived(ry);
    if (FORM != BLOCK) arrived(rg);
    unsigned step = 0;
    // (every row slot of a workgroup takes part in the barriers of row_sum: the loop runs over whole row sets)
    for (long long base = row0; base < row1; base += ROWS, step += set_bytes) {
      const long long r = base + slot;
      const bool there = r < row1;
      const float eps = there ? a.eps : 1.f;
      float v[W], u[W], ga[W];
      ch.settle(rx, sh);
      row_unpack(rx, v);
      ch.settle(ry, sh);
      row_unpack(ry, u);
      if (FORM != BLOCK) {
        ch.settle(rg, sh);
        row_unpack(rg, ga);
      }
      unpacked();
      request(step + set_bytes, r + ROWS);
      if (has_y) {
        if (post) row_normalise<T, L, W, MODE>(u, lane, C, inv_c, layer, eps, slots, turn);
        if (own) gate_act<T, W>(ga, a.sigmoid);
#pragma unroll
        for (int i = 0; i < W; ++i) v[i] = fmaf(own ? ga[i] : gs[i], fmaf(u[i], sw[i], sb[i]), v[i]);
      }
      if (MODE == EACH) each_store<T, L, W>(a.out, r, lane, C, there, v);
      else ch.store(to, step, v);
      if (next) {
        // (of the fp32 sum, not of its rounded copy in `out`)
        row_normalise<T, L, W, MODE>(v, lane, C, inv_c, layer, eps, slots, turn);
#pragma unroll
        for (int i = 0; i < W; ++i) v[i] = fmaf(v[i], nw[i], nb[i]);
      }
      if (MODE == EACH) each_store<T, L, W>(a.normed, r, lane, C, there, v);
      else ch.store(tn, step, v);
      arrived(rx); arrived(ry);
      if (FORM != BLOCK) arrived(rg);
    }
  }
}

template <typename T, int L, int W, NormForm FORM> void launch_form(const NormFwd<T> &a, int nblk, NormMode mode, hipStream_t st) {
  constexpr int THREADS = NormShape<T, L, W>::THREADS;
  if (W == 16 || mode == WHOLE) norm_residual_fwd_kernel<T, L, W, WHOLE, FORM><<<nblk, THREADS, 0, st>>>(a);
  else if constexpr (W == 8) norm_residual_fwd_kernel<T, L, W, RAGGED, FORM><<<nblk, THREADS, 0, st>>>(a);
}
template <typename T, int L, int W> void launch(const NormFwd<T> &a, int nblk, NormMode mode, hipStream_t st) {
  if (!(a.y && a.weight && a.normed)) launch_form<T, L, W, ANY>(a, nblk, mode, st);
  else if (a.gate && !a.shared_gate) launch_form<T, L, W, BLOCK_OWN>(a, nblk, mode, st);
  else launch_form<T, L, W, BLOCK>(a, nblk, mode, st);
}

template <typename T>
int forward(const void *x, const void *y, const void *gate, const float *weight, const float *bias, const float *scale,
            const float *next_weight, const float *next_bias, long long P, int C, long long gate_rows, int layer, int sigmoid, float eps,
            void *out, void *normed, hipStream_t st) {
  if (!gate) gate_rows = 0;
  const int W = norm_width(C, sizeof(T));
  // Four waves on each of the 1024 SIMDs run at once (87 to 129 registers; three with 16 channels a lane); twice as many are launched, and
  // those that come second start as the first end: 65536 x 512 64 -> 61 us, fp32 65536 x 256 65 -> 60, 8192 x 4096 56 -> 53.  Four and
  // more times as many load the parameters too often: 131072 x 128 31 to 35 (33), 100003 x 131 26 to 44 (24), 8192 x 4096 52 to 87.
  const NormSplit s = norm_split(P, C, W, gate_rows, 8 * 1024, 1);
  NormFwd<T> a;
  a.x = (const T *)x; a.y = (const T *)y; a.gate = (const T *)gate;
  a.weight = weight; a.bias = bias; a.scale = scale; a.next_weight = next_weight; a.next_bias = next_bias;
  a.P = P; a.rows_per_gate = s.rows_per_gate; a.groups = s.groups; a.chunk = s.chunk;
  a.blocks_per_group = s.blocks_per_group; a.groups_per_block = s.groups_per_block; a.shared_gate = gate && gate_rows < P;
  a.C = C; a.layer = layer; a.sigmoid = sigmoid; a.eps = eps;
  a.out = (T *)out; a.normed = (T *)normed;
  const NormMode mode = norm_mode<T>(P, C);
  if (mode == EACH) {
    norm_residual_fwd_kernel<T, 8, 8, EACH, ANY><<<s.nblk, 256, 0, st>>>(a);
    return cpfn_launch_status();
  }
  if (W == 16) {
    if constexpr (sizeof(T) == 2) launch<T, 64, 16>(a, s.nblk, mode, st);
    return cpfn_launch_status();
  }
  switch (norm_lanes(C, W)) {
    case 8: launch<T, 8, 8>(a, s.nblk, mode, st); break;
    case 16: launch<T, 16, 8>(a, s.nblk, mode, st); break;
    case 32: launch<T, 32, 8>(a, s.nblk, mode, st); break;
    case 64: launch<T, 64, 8>(a, s.nblk, mode, st); break;
    case 128: launch<T, 128, 8>(a, s.nblk, mode, st); break;
    case 256: launch<T, 256, 8>(a, s.nblk, mode, st); break;
    default: launch<T, 512, 8>(a, s.nblk, mode, st); break;
  }
  return cpfn_launch_status();
}

}  // namespace

extern "C" int cpfn_norm_residual_fwd(const void *x, const void *y, const void *gate, const float *weight, const float *bias,
                                      const float *scale, const float *next_weight, const float *next_bias, long long P, int C,
                                      long long gate_rows, int dtype, int layer, int sigmoid, float eps, void *out, void *normed,
                                      void *stream) {
  if (P < 0 || C < 1 || C > CPFN_NORM_MAX_C || !(eps >= 0.f) || (normed && !next_weight) || (!y && (weight || gate || scale || !normed)) ||
      (y && !out) || (bias && !weight) || (next_bias && !next_weight))
    return CPFN_EINVAL;
  if (gate && (gate_rows < 1 || P % gate_rows != 0)) return CPFN_EINVAL;
  if (P == 0) return 0;
  if (!x) return CPFN_EINVAL;
  hipStream_t st = (hipStream_t)stream;
  switch (dtype) {
    case CPFN_F32: return forward<float>(x, y, gate, weight, bias, scale, next_weight, next_bias, P, C, gate_rows, layer, sigmoid, eps, out, normed, st);
    case CPFN_BF16: return forward<cpfn_bf16>(x, y, gate, weight, bias, scale, next_weight, next_bias, P, C, gate_rows, layer, sigmoid, eps, out, normed, st);
    case CPFN_F16: return forward<cpfn_f16>(x, y, gate, weight, bias, scale, next_weight, next_bias, P, C, gate_rows, layer, sigmoid, eps, out, normed, st);
  }
  return CPFN_EINVAL;
}
