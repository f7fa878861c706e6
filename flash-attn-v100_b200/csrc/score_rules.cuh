// What the tensor-core kernels do to a score under rules (fa_b200_rules): the cap's tanh for pairs of scores.
#pragma once
#include "sm100_ptx.cuh"

namespace fa {

// tanh(u) on the FMA pipes, z = u * u: odd polynomials with the least largest relative error (fitted by reweighted least
// squares), four terms for |u| <= 1/2, 5.5e-7, six for |u| <= 1, 5.9e-7.  A score of size s is off by 6e-7 s: the rounding of
// a sum of products of size s.  The special-function unit, which the softmax keeps busiest, would be asked twice for each.
constexpr float kTanhShortMax = 0.5f, kTanhLongMax = 1.f;
template <bool LONG>
__device__ __forceinline__ uint64_t f2_tanh_poly(uint64_t u, uint64_t z) {
    using namespace ptx;
    constexpr float c[6] = {LONG ? 0.999999414f : 0.999999456f, LONG ? -0.333290423f : -0.333263176f, LONG ? 0.132814332f : 0.13190294f,
                            LONG ? -0.0516056576f : -0.0444021663f, 0.0167430985f, -0.00306705425f};
    uint64_t r = LONG ? f2_fma(f2_pack(c[5], c[5]), z, f2_pack(c[4], c[4])) : f2_pack(c[3], c[3]);
    if (LONG) r = f2_fma(r, z, f2_pack(c[3], c[3]));
    r = f2_fma(r, z, f2_pack(c[2], c[2]));
    r = f2_fma(r, z, f2_pack(c[1], c[1]));
    r = f2_fma(r, z, f2_pack(c[0], c[0]));
    return f2_mul(r, u);
}
// The same for several pairs step by step, so that no step waits for the one before it; u is replaced.
constexpr int kTanhAtOnce = 8;
template <bool LONG>
__device__ __forceinline__ void f2_tanh_poly(uint64_t (&u)[kTanhAtOnce], const uint64_t (&z)[kTanhAtOnce]) {
    using namespace ptx;
    constexpr float c[6] = {LONG ? 0.999999414f : 0.999999456f, LONG ? -0.333290423f : -0.333263176f, LONG ? 0.132814332f : 0.13190294f,
                            LONG ? -0.0516056576f : -0.0444021663f, 0.0167430985f, -0.00306705425f};
    constexpr int n = LONG ? 6 : 4;
    uint64_t r[kTanhAtOnce];
#pragma unroll
    for (int e = 0; e < kTanhAtOnce; ++e) r[e] = f2_fma(f2_pack(c[n - 1], c[n - 1]), z[e], f2_pack(c[n - 2], c[n - 2]));
#pragma unroll
    for (int k = n - 3; k >= 0; --k)
#pragma unroll
        for (int e = 0; e < kTanhAtOnce; ++e) r[e] = f2_fma(r[e], z[e], f2_pack(c[k], c[k]));
#pragma unroll
    for (int e = 0; e < kTanhAtOnce; ++e) u[e] = f2_mul(r[e], u[e]);
}
// tanh of any u: 1 - 2 / (1 + e^2u), off by at most 2^-22; 1 and -1 far out, a NaN stays one.
__device__ __forceinline__ float tanh_any(float u) {
    const float e = ptx::ex2(u * 2.8853900817779268f);           // 2 log2 e
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.f + e));
    return fmaf(-2.f, r, 1.f);
}

}  // namespace fa
