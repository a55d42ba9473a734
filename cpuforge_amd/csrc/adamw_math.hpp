// AdamW's arithmetic, shared by the kernels over 32-bit and 8-bit states.
#pragma once
#include <hip/hip_runtime.h>

namespace cfattn {

// optim.rs:21-29 with every product and sum rounded on its own (correctly
// rounded, as hipcc's default f32 division and sqrt are; HIP's own __fadd_rn
// and __fmul_rn could still be fused after inlining):
//   m = b1*m + (1-b1)*g,  v = b2*v + ((1-b2)*g)*g,
//   p -= lr * ((m/bc1) / (sqrt(v/bc2) + eps) + wd*p).
__device__ __forceinline__ void adamw_one(float& p, float g, float& m, float& v, float lr, float b1, float b2, float ob1,
                                          float ob2, float eps, float wd, float bc1, float bc2) {
#pragma clang fp contract(off)
    m = b1 * m + ob1 * g;
    v = b2 * v + (ob2 * g) * g;
    const float mhat = m / bc1;
    const float vhat = v / bc2;
    const float upd = mhat / (sqrtf(vhat) + eps) + wd * p;
    p = p - lr * upd;
}

}  // namespace cfattn
