// The update of one element that sparc_adam_step and the clipped steps share, in float32 with the step's scalars prepared in
// float64 on the host (the formulas of torch.optim.Adam, amsgrad = False, maximize = False), for the gradient coef g:
//     g' = coef g + weight_decay p;   m = m + (1 - beta1) (g' - m);   v = beta2 v + (1 - beta2) g' g'
//     p = p - (lr / (1 - beta1^t)) m / (sqrt(v) / sqrt(1 - beta2^t) + eps)
#pragma once
#include <math.h>

#include "common.h"

struct AdamFactors {
    float step_size, bc2_rsqrt, beta2, one_minus_beta1, one_minus_beta2, eps, weight_decay;
};

inline AdamFactors adam_factors(const double lr, const double beta1, const double beta2, const double eps, const double weight_decay, const int64_t step) {
    const double bc1 = 1.0 - pow(beta1, static_cast<double>(step)), bc2 = 1.0 - pow(beta2, static_cast<double>(step));
    AdamFactors a;
    a.step_size = static_cast<float>(lr / bc1);
    a.bc2_rsqrt = static_cast<float>(1.0 / sqrt(bc2));
    a.beta2 = static_cast<float>(beta2);
    a.one_minus_beta1 = static_cast<float>(1.0 - beta1);
    a.one_minus_beta2 = static_cast<float>(1.0 - beta2);
    a.eps = static_cast<float>(eps);
    a.weight_decay = static_cast<float>(weight_decay);
    return a;
}

__device__ __forceinline__ void adam_one(float& p, const float g0, float& m, float& v, const AdamFactors& a, const float coef) {
    float g = coef * g0;
    if (a.weight_decay != 0.f) g = fmaf(a.weight_decay, p, g);
    m = fmaf(a.one_minus_beta1, g - m, m);
    v = fmaf(a.beta2, v, a.one_minus_beta2 * g * g);
    p -= a.step_size * (m / (sqrtf(v) * a.bc2_rsqrt + a.eps));
}
