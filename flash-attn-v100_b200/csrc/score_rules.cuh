// What the tensor-core kernels do to a score under rules (fa_b200_rules): the cap's tanh for pairs of scores.
#pragma once
#include "sm100_ptx.cuh"

namespace fa {

// tanh(u) for |u| <= 1 on the FMA pipes, z = u * u: an odd polynomial with the least largest relative error there, 5.9e-7
// (fitted by reweighted least squares).  A score of size s is off by 5.9e-7 s: the rounding of a sum of products of size s.
// The special-function unit, which the softmax keeps busiest, would be asked twice for each score.
constexpr float kTanhPolyMax = 1.f;
__device__ __forceinline__ uint64_t f2_tanh_poly(uint64_t u, uint64_t z) {
    using namespace ptx;
    const uint64_t c0 = f2_pack(0.999999414f, 0.999999414f), c1 = f2_pack(-0.333290423f, -0.333290423f);
    const uint64_t c2 = f2_pack(0.132814332f, 0.132814332f), c3 = f2_pack(-0.0516056576f, -0.0516056576f);
    const uint64_t c4 = f2_pack(0.0167430985f, 0.0167430985f), c5 = f2_pack(-0.00306705425f, -0.00306705425f);
    uint64_t r = f2_fma(c5, z, c4);
    r = f2_fma(r, z, c3);
    r = f2_fma(r, z, c2);
    r = f2_fma(r, z, c1);
    r = f2_fma(r, z, c0);
    return f2_mul(r, u);
}
// tanh of any u: 1 - 2 / (1 + e^2u), off by at most 2^-22; 1 and -1 far out, a NaN stays one.
__device__ __forceinline__ float tanh_any(float u) {
    const float e = ptx::ex2(u * 2.8853900817779268f);           // 2 log2 e
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.f + e));
    return fmaf(-2.f, r, 1.f);
}

}  // namespace fa
