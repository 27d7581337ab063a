// Arithmetic that every group norm kernel shares.
//
// These kernels stand or fall with the number of vector instructions per element: a wave's instruction takes four cycles, so 256
// compute units do 39e12 of them a second, and at 16-bit storage memory asks for an element every 0.7 ps forward (4 bytes) and 1.1 ps
// backward (6 bytes): 27 and 43 instructions.
#pragma once
#include "layer_common.hpp"

// ---- normalisation -----------------------------------------------------------------------------------------------------------
// Per channel, from the group's (mean, r) and (gamma, beta): z(x) and the deviation from the mean.  The deviation is formed first: for values
// near the mean it is exact, and z is beta where a group holds one value.  (With the mean in the shift, z = x (gamma r) + (beta - mean gamma r),
// z is off by |mean| r gamma 2^-24: 0.02 at a mean of 1000 beside r = 316 = eps^-1/2.  One instruction less: 16 x 608 x 608 x 32 f16 174.5 us
// for 178.6, 32 x 76 x 76 x 256 bf16 with a shortcut 64.2 for 65.3, backward the same.)
//
// LEAKY: d = x - mean, xh = d r, z = gamma xh + beta, every operation rounded (no contraction): which side of the kink a value falls on
// is then a function of the inputs and the statistics alone, the same in the forward and the backward pass and in every kernel.
// Smooth activations at 16-bit storage: z = d (gamma r) + beta, a subtraction and a multiply-add.
template <typename T, int ACT>
struct Norm {
    static constexpr bool SCALED = sizeof(T) == 2 && ACT != CY_ACT_LEAKY;
    float mean, r, ga, be;      // SCALED: ga = gamma r
    __device__ __forceinline__ void set(float2 stat, float gamma, float beta) {
#pragma clang fp contract(off)
        mean = stat.x;
        r = stat.y;
        ga = SCALED ? gamma * stat.y : gamma;
        be = beta;
    }
    __device__ __forceinline__ float z(float x) const {
#pragma clang fp contract(off)
        float d = x - mean;
        if constexpr (SCALED && !__is_same(T, bf16)) {      // (the same number: 1 x - mean, which takes the stored half as it is)
            float one = 1.f;
            asm("" : "+s"(one));
            d = fmaf(x, one, -mean);
        }
        if constexpr (SCALED) return ACT == CY_ACT_LINEAR ? rounded(fmaf(d, ga, be)) : fmaf(d, ga, be);
        const float xh = d * r;
        const float g = xh * ga;
        return g + be;
    }
};

// dx = r (gamma dz - S1 - xh S2) = dz (gamma r) + (x - mean) k1 + k0, with (k0, k1) = (-r S1, -r^2 S2) of the group
__device__ __forceinline__ float2 gn_k01(float r, double s1, double s2) {
#pragma clang fp contract(off)
    return make_float2(-r * (float)s1, -r * (r * (float)s2));
}
template <typename T, int ACT>
__device__ __forceinline__ float gn_dx(const Norm<T, ACT>& nm, float2 k, float x, float dz) {
#pragma clang fp contract(off)
    const float k2 = Norm<T, ACT>::SCALED ? nm.ga : nm.ga * nm.r;
    return rounded(fmaf(dz, k2, fmaf(x - nm.mean, k.y, k.x)));
}

// ---- activations -------------------------------------------------------------------------------------------------------------
// mish(z) = z tanh(log(1 + e^z)).  With n = e^z, w = n (n + 2): tanh = w / (w + 2).  FAST (16-bit storage): hardware exponential and
// reciprocal, 1 - 2 e each.  The exponent is cut at 20, where w / (w + 2) is 1 in 32 bits and w finite, so no value needs a branch.
// Derivative: with q = 2 / (w + 2) = 1 - tanh it is tanh + z q^2 (w - n): one exponential, one reciprocal.  tanh is formed by itself, 1 - q
// cancels for large negative z (0.04 % of the derivative at z = -12, 2 % at -16).  The second term takes the cut z, too: q no longer
// falls beyond 20, and z q^2 (w - n) would grow again from 10^16 on.  (The cut lets a NaN through.)
// (No contraction is left to the compiler anywhere in this file: a value comes out the same wherever it is computed, by the block that
// holds it or by the one that finishes for it.)
//
// 32 bits: e^z = 2^h (1 + l ln 2) with h + l = z log2(e) in two words; 1 / a by the hardware's reciprocal and one Newton step (a >= 2,
// finite).  Within 2 e and 1 e, in 16 issue slots less per element than the library's exponential and an IEEE division:
// 16 x 38 x 38 x 512 f32 backward 38.5 -> 34.1 us, forward 26.5 -> 22.2.
constexpr float LOG2E = 1.44269504088896341f, LOG2E_REST = (float)(1.4426950408889634074 - (double)LOG2E), LN2 = 0.69314718055994531f;
template <bool FAST>
__device__ __forceinline__ float gn_cut(float z) {
    z = __builtin_elementwise_minimum(z, 20.f);
    return FAST ? z : __builtin_elementwise_maximum(z, -120.f);      // (2^h, which is 0 below 2^-126, is 0 there; the residual finite)
}
template <bool FAST>
__device__ __forceinline__ float gn_exp(float z) {      // e^z of a cut z
#pragma clang fp contract(off)
    const float h = z * LOG2E, n = __builtin_amdgcn_exp2f(h);
    if constexpr (FAST) return n;
    const float l = fmaf(z, LOG2E_REST, fmaf(z, LOG2E, -h));
    return fmaf(n, l * LN2, n);
}
template <bool FAST>
__device__ __forceinline__ float gn_rcp(float a) {
#pragma clang fp contract(off)
    const float r = __builtin_amdgcn_rcpf(a);
    return FAST ? r : fmaf(fmaf(-a, r, 1.f), r, r);
}
template <int ACT, bool FAST>
__device__ __forceinline__ float gn_act(float z) {
#pragma clang fp contract(off)
    if constexpr (ACT == CY_ACT_MISH) {
        const float n = gn_exp<FAST>(gn_cut<FAST>(z));
        const float w = n * (n + 2.f);
        return z * (w * gn_rcp<FAST>(w + 2.f));
    }
    return ACT == CY_ACT_LEAKY && !(z > 0.f) ? 0.1f * z : z;
}
template <int ACT, bool FAST>
__device__ __forceinline__ float gn_act_grad(float z) {
#pragma clang fp contract(off)
    if constexpr (ACT == CY_ACT_MISH) {
        z = gn_cut<FAST>(z);
        const float n = gn_exp<FAST>(z);
        if constexpr (FAST) {      // z q^2 (w - n) = z t (t + q), tanh = t h  with h = n / 2 + 1, t = n q
            const float h = fmaf(n, 0.5f, 1.f), q = gn_rcp<true>(fmaf(n, h, 1.f)), t = n * q;
            return fmaf(z * t, t + q, t * h);
        }
        const float w = n * (n + 2.f), i = gn_rcp<false>(w + 2.f), q = 2.f * i;
        return fmaf(z * (w - n), q * q, w * i);
    }
    return ACT == CY_ACT_LEAKY && !(z > 0.f) ? 0.1f : 1.f;
}

__device__ __forceinline__ float gn_rstd(double var, float eps) {
    if (var < 0.0) var = 0.0;
    return (float)(1.0 / sqrt(var + (double)eps));
}

// ---- statistics --------------------------------------------------------------------------------------------------------------
// How many sums a thread keeps for the V channels of a chunk: 1 -- they lie in one group (Cg % V == 0); V / Cg -- one for each of the whole
// groups in the chunk; V -- one per channel.
template <int V>
static inline int gn_sums(int Cg) {
    return Cg % V == 0 ? 1 : V % Cg == 0 ? V / Cg : V;
}
// columns (thread sums side by side) of a group
template <int V>
__device__ __host__ static inline int gn_cols(int Cg) {
    return Cg % V == 0 ? Cg / V : V % Cg == 0 ? 1 : Cg;
}
