// Norms before and after a residual block, its gate and its residual scale in one pass over the rows (forward; the formulas are in
// rownorm.h).  Memory bound: x, y and the gate are read once, out and normed written once; the op-by-op form moves each of the ~12
// intermediate tensors through memory.
#include "rownorm.h"

namespace {

constexpr long long FWD_WAVES = 4096;         // waves of a launch: what is resident together

template <typename T> struct NormFwd {
  const T *x, *y, *gate;
  const float *weight, *bias, *scale, *next_weight, *next_bias;
  long long P, rows_per_gate, gate_rows;
  int C, layer, sigmoid;
  float eps;
  T *out, *normed;
};

template <typename T, int L, bool RAGGED>
__global__ __launch_bounds__((NormShape<T, L>::THREADS)) void norm_residual_fwd_kernel(const NormFwd<T> a) {
  constexpr int ROWS = NormShape<T, L>::ROWS;
  __shared__ float2 slots[32];
  int turn = 0;
  const int lane = threadIdx.x & (L - 1), slot = threadIdx.x / L, C = a.C;
  const float inv_c = 1.f / (float)C;
  const bool layer = a.layer != 0, post = a.weight != nullptr, has_y = a.y != nullptr;
  const RowRaw<T, L> mask = row_mask<T, L, RAGGED>(lane, C);
  // the rows of the NEXT step are requested before this one's are worked on
  RowRaw<T, L> rx, ry, rg;
  row_zero(rx); row_zero(ry); row_zero(rg);
  const auto request = [&](long long r) {
    if (r < a.P) {
      row_load<T, L, RAGGED>(rx, a.x, r, a.P, lane, C, mask);
      if (has_y) row_load<T, L, RAGGED>(ry, a.y, r, a.P, lane, C, mask);
      if (a.gate) row_load<T, L, RAGGED>(rg, a.gate, norm_gate_row(r, a.rows_per_gate, a.P), a.gate_rows, lane, C, mask);
    } else {
      row_zero(rx); row_zero(ry); row_zero(rg);
    }
  };
  const long long step = (long long)gridDim.x * ROWS;
  long long base = (long long)blockIdx.x * ROWS;
  request(base + slot);
  float w[8], b[8], s[8], nw[8], nb[8];
  param_load<T, L>(w, a.weight, lane, C, 1.f);
  param_load<T, L>(b, a.bias, lane, C, 0.f);
  param_load<T, L>(s, a.scale, lane, C, 1.f);
  param_load<T, L>(nw, a.next_weight, lane, C, 1.f);
  param_load<T, L>(nb, a.next_bias, lane, C, 0.f);
  // (every row slot of a workgroup takes part in the barriers of row_sum: the loop runs over whole row sets)
  for (; base < a.P; base += step) {
    const long long r = base + slot;
    const bool there = r < a.P;
    const float eps = there ? a.eps : 1.f;
    const RowRaw<T, L> cx = rx, cy = ry, cg = rg;
    request(r + step);
    float o[8];
    row_unpack(cx, o);
    if (has_y) {
      float u[8];
      row_unpack(cy, u);
      if (post) {
        row_normalise<T, L, RAGGED>(u, lane, C, inv_c, layer, eps, slots, turn);
#pragma unroll
        for (int i = 0; i < 8; ++i) u[i] = fmaf(u[i], w[i], b[i]);
      }
      if (a.gate) {
        float g[8];
        row_unpack(cg, g);
        if (a.sigmoid) {
#pragma unroll
          for (int i = 0; i < 8; ++i) g[i] = norm_sigmoid<T>(g[i]);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) u[i] *= g[i];
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) o[i] = fmaf(s[i], u[i], o[i]);
      if (there) row_store<T, L, RAGGED>(a.out + r * C, lane, C, o);
    }
    if (a.normed) {
      // (of the fp32 sum, not of its rounded copy in `out`)
      row_normalise<T, L, RAGGED>(o, lane, C, inv_c, layer, eps, slots, turn);
#pragma unroll
      for (int i = 0; i < 8; ++i) o[i] = fmaf(o[i], nw[i], nb[i]);
      if (there) row_store<T, L, RAGGED>(a.normed + r * C, lane, C, o);
    }
  }
}

template <typename T, int L> int launch(const NormFwd<T> &a, hipStream_t st) {
  const long long sets = (a.P + NormShape<T, L>::ROWS - 1) / NormShape<T, L>::ROWS;
  const long long most = FWD_WAVES * 64 / NormShape<T, L>::THREADS;
  const unsigned blocks = (unsigned)(sets < most ? sets : most);
  if (a.C % cpfn_piece<T>::N) norm_residual_fwd_kernel<T, L, true><<<blocks, NormShape<T, L>::THREADS, 0, st>>>(a);
  else norm_residual_fwd_kernel<T, L, false><<<blocks, NormShape<T, L>::THREADS, 0, st>>>(a);
  return cpfn_launch_status();
}

template <typename T>
int forward(const void *x, const void *y, const void *gate, const float *weight, const float *bias, const float *scale,
            const float *next_weight, const float *next_bias, long long P, int C, long long gate_rows, int layer, int sigmoid, float eps,
            void *out, void *normed, hipStream_t st) {
  NormFwd<T> a;
  a.x = (const T *)x; a.y = (const T *)y; a.gate = (const T *)gate;
  a.weight = weight; a.bias = bias; a.scale = scale; a.next_weight = next_weight; a.next_bias = next_bias;
  a.P = P; a.rows_per_gate = gate ? P / gate_rows : 1; a.gate_rows = gate_rows;
  a.C = C; a.layer = layer; a.sigmoid = sigmoid; a.eps = eps;
  a.out = (T *)out; a.normed = (T *)normed;
  switch (norm_lanes(C)) {
    case 8: return launch<T, 8>(a, st);
    case 16: return launch<T, 16>(a, st);
    case 32: return launch<T, 32>(a, st);
    case 64: return launch<T, 64>(a, st);
    case 128: return launch<T, 128>(a, st);
    case 256: return launch<T, 256>(a, st);
    default: return launch<T, 512>(a, st);
  }
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
