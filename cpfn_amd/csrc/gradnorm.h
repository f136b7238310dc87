// The factor by which gradients of norm `total` are clipped to `max_norm` (gradnorm.hip; the optimizer's own step: optim.hip).
#pragma once
#include "rows16.h"

// min(1, max_norm / (total + 1e-6)); NaN for a NaN norm
__device__ __forceinline__ float grad_clip_factor(double total, double max_norm) {
  const double f = max_norm / (total + 1e-6);
  return f < 1.0 ? (float)f : (f != f ? (float)f : 1.f);
}
