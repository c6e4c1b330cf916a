// Element arithmetic of the gated activations and of RMSNorm, shared by the stand-alone kernels and by the quantizer's
// fused prologue, so that "activation, then quantize" and the fused kernel produce the same bits.
//
// Formulas of the reference (all in fp32, result rounded to the tensor's type):
//   SwiGLU  out = (a / (1 + exp(-a))) * b * p        primus_turbo/triton/activation/swiglu_kernel.py:51-57
//   GeGLU   out = (0.5 * a * (1 + erf(a / sqrt 2))) * b * p   geglu_kernel.py:53, triton/utils/gelu.py:21-25
//   RMSNorm y = x * rstd * g, rstd = rsqrt(mean(x^2) + eps), g = gamma (or 1 + gamma)   normalization/rmsnorm_kernel.py:68-75
// with a = first half of the row ("up" in the reference's kernels), b = second half, p = the row's probability.
#pragma once
#include <cuda_runtime.h>

namespace ptb {

// the first two are also the gated activations'; the rest are epilogue activations of gemm_bias_act
enum { PT_ACT_SILU = 0, PT_ACT_GELU = 1, PT_ACT_NONE = 2, PT_ACT_RELU = 3, PT_ACT_GELU_TANH = 4 };

template <int ACT> __device__ __forceinline__ float act_value(float a) {
    if constexpr (ACT == PT_ACT_SILU) return __fdividef(a, 1.0f + __expf(-a));
    else if constexpr (ACT == PT_ACT_RELU) return a < 0.0f ? 0.0f : a;   // a NaN stays
    // tanh form of the GELU, 0.5 a (1 + tanh u) with u = sqrt(2 / pi) (a + 0.044715 a^3), as a / (1 + exp(-2 u)): no cancellation
    else if constexpr (ACT == PT_ACT_GELU_TANH) return __fdividef(a, 1.0f + __expf(-1.5957691216f * a * (1.0f + 0.044715f * a * a)));
    else if constexpr (ACT == PT_ACT_NONE) return a;
    else return 0.5f * a * (1.0f + erff(a * 0.7071067811f));
}
// d act(a) / d a
template <int ACT> __device__ __forceinline__ float act_grad(float a) {
    if constexpr (ACT == PT_ACT_SILU) {
        const float s = __fdividef(1.0f, 1.0f + __expf(-a));
        return s * (1.0f + a * (1.0f - s));
    } else if constexpr (ACT == PT_ACT_RELU) {
        return a > 0.0f ? 1.0f : 0.0f;
    } else if constexpr (ACT == PT_ACT_GELU_TANH) {
        const float s = __fdividef(1.0f, 1.0f + __expf(-1.5957691216f * a * (1.0f + 0.044715f * a * a)));
        return s + a * s * (1.0f - s) * 1.5957691216f * (1.0f + 0.134145f * a * a);
    } else if constexpr (ACT == PT_ACT_NONE) {
        return 1.0f;
    } else {
        return 0.3989422803f * a * __expf(-(0.7071067811f * a) * (0.7071067811f * a)) + 0.5f * erff(0.7071067811f * a) + 0.5f;
    }
}
// The slope at a pre-activation that was saved in 16 bits.  Beyond 65504 fp16 holds an infinity, and the square of a large bf16 value is one;
// either would meet a factor that has become zero.  At +-100 every slope has long reached its limit in fp32, 0 or 1, so further values
// take that (a NaN stays one).
template <int ACT> __device__ __forceinline__ float act_grad_saved(float z) {
    return act_grad<ACT>(fabsf(z) > 100.0f ? copysignf(100.0f, z) : z);
}
template <int ACT> __device__ __forceinline__ float glu_value(float a, float b, float p) { return act_value<ACT>(a) * b * p; }

// GELU (erf form) of the epilogues: z Phi(z) = max(z, 0) - |z| R(|z|) exp(-z^2 / 2) with R(x) = erfc(x / sqrt 2) exp(x^2 / 2) / 2.  R is smooth
// and falls like 1 / x: a polynomial in t = 1 / (1 + 0.3 x), without a constant term, fitted here for the least relative error on [0, 14.5]
// (1.7e-7).  So the error is relative in the negative tail too, where 1 + erf(z / sqrt 2) cancels: at most 8e-7 from -3 on, 3e-6 from -8
// on (exp's argument is rounded).  About 16 instructions where erff takes 40; the epilogue of a short product is bound by their number
// (8192 x 4096 x 64: 49.5 us, with erff 67).
__device__ __forceinline__ float gelu_epilogue(float z) {
    const float x = fminf(fabsf(z), 20.0f);   // the second term is zero from there on
    float t, e, positive;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(t) : "f"(1.0f + 0.3f * x));
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(-0.7213475204f * (x * x)));   // exp(-x^2 / 2)
    asm("max.NaN.f32 %0, %1, 0f00000000;" : "=f"(positive) : "f"(z));              // a NaN stays one
    const float r = 0.119632007f + t * (0.120712136f + t * (0.100175949f + t * (0.127691767f + t * (-0.0520340042f + t * (0.204556767f +
                    t * (-0.156158435f + t * 0.0354237315f))))));
    return positive - x * t * r * e;
}

// The activation chosen at run time (uniform over the launch), for a lane's values under one branch.
template <int ROWS> __device__ __forceinline__ void act_any_all(int act, float (&v)[ROWS][4]) {
    auto all = [&](auto f) {
#pragma unroll
        for (int r = 0; r < ROWS; ++r)
#pragma unroll
            for (int i = 0; i < 4; ++i) v[r][i] = f(v[r][i]);
    };
    switch (act) {
    case PT_ACT_SILU: all([](float x) { return act_value<PT_ACT_SILU>(x); }); break;
    case PT_ACT_GELU: all([](float x) { return gelu_epilogue(x); }); break;
    case PT_ACT_RELU: all([](float x) { return act_value<PT_ACT_RELU>(x); }); break;
    case PT_ACT_GELU_TANH: all([](float x) { return act_value<PT_ACT_GELU_TANH>(x); }); break;
    default: break;
    }
}

__device__ __forceinline__ float rmsnorm_value(float x, float rstd, float g) { return x * rstd * g; }

}  // namespace ptb
