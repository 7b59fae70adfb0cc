// adam.h -- the Adam update of one value, for every kernel that takes a step (elementwise.hip, gradnorm.hip).
//
// Its two fused products are written out -- left to the compiler they differ from kernel to kernel -- so that a bound on the gradient's norm that is
// never reached changes no bit of a step.  The constants come from the betas in 64 bits and are rounded once each: 1 - 0.999 formed from an
// fp32 0.999 would be 1.3e-5 of itself too small, and so would every new term of the second moment.  The bias corrections are folded into two of them,
// lr / (1 - beta1^t) and sqrt(1 - beta2^t), as torch.optim.Adam does: two divisions a value instead of three.
#ifndef FDGAN_ADAM_H
#define FDGAN_ADAM_H

#include <math.h>

struct AdamUpdate {
  float b1, a1, b2, a2, eps, step, root;      // a = 1 - beta; step = lr / (1 - beta1^t), root = sqrt(1 - beta2^t)
};

inline AdamUpdate adam_constants(float lr, double beta1, double beta2, float eps, int64_t step) {
  return AdamUpdate{(float)beta1, (float)(1.0 - beta1), (float)beta2, (float)(1.0 - beta2), eps, (float)(lr / (1.0 - pow(beta1, (double)step))),
                    (float)sqrt(1.0 - pow(beta2, (double)step))};
}

__device__ __forceinline__ void adam_update(const AdamUpdate& a, float g, float& p, float& m, float& v) {
#pragma clang fp contract(off)
  m = fmaf(a.b1, m, a.a1 * g);
  v = fmaf(a.b2, v, a.a2 * g * g);
  p -= a.step * m / (sqrtf(v) / a.root + a.eps);
}

#endif
