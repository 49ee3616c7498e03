// Activations behind a dense layer's product, and their derivatives.
//   relu: max(z, 0)    gelu: z P(z), P the normal distribution function    silu: z / (1 + exp(-z))
//
// P by the error function's rational approximation 7.1.26 of Abramowitz and Stegun's Handbook (absolute error 1.5e-7, so that P is off by 0.75e-7): the
// exponential in it is the derivative's too, and one reciprocal and five products go with it, where a library's erf branches.  Below zero P is the
// small term itself, with no difference taken.  Exponentials and reciprocals are the instructions', 2^-23 or so, and an
// exponential's argument v is rounded before: |v| 2^-23 of the result at most (2^-17 at the ends of the range, where the result is next to nothing).
#pragma once

#include "fgl_common.hpp"
#include "fgl_keep8.hpp"

namespace fgl {

// Derivatives are kept in fp16 beside bf16 values, times 2^15: they are at most 1.13, and so have eleven bits down to 2^-29 (silu's at -23) and are off by 2^-40 at
// most below that.
constexpr float kSlopeScale = 0x1p15f;

constexpr int kActNone = 0, kActRelu = 1, kActGelu = 2, kActSilu = 3;

#if defined(__HIPCC__)

__device__ __forceinline__ float act_exp(float v) { return __builtin_amdgcn_exp2f(v * 1.44269504089f); }

// P(z), and exp(-z^2 / 2)
__device__ __forceinline__ float act_normal(float z, float& e)
{
    const float x = fabsf(z) * 0.70710678119f;
    const float t = __builtin_amdgcn_rcpf(fmaf(0.3275911f, x, 1.0f));
    e = act_exp(-0.5f * z * z);
    float p = fmaf(1.061405429f, t, -1.453152027f);
    p = fmaf(p, t, 1.421413741f);
    p = fmaf(p, t, -0.284496736f);
    p = fmaf(p, t, 0.254829592f);
    const float q = 0.5f * p * t * e;
    return z < 0.0f ? q : 1.0f - q;
}

__device__ __forceinline__ bool act_passes(float z) { return !(z <= 0.0f); }  // (what is not a number stays it)

template <int N, int V, typename F>
__device__ __forceinline__ void act_each(float (&v)[N][V], F&& f)
{
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
        for (int t = 0; t < V; ++t) v[i][t] = f(v[i][t]);
}
template <int N, int V>
__device__ __forceinline__ void act_apply(int act, float (&v)[N][V])
{
    if (act == kActRelu) {
        act_each(v, [](float z) { return act_passes(z) ? z : 0.0f; });
    } else if (act == kActGelu) {
        act_each(v, [](float z) {
            float unused;
            return z * act_normal(z, unused);
        });
    } else if (act == kActSilu) {
        act_each(v, [](float z) { return z * __builtin_amdgcn_rcpf(1.0f + act_exp(-z)); });
    }
}

// gelu or silu of v, and their derivatives
template <int N, int V>
__device__ __forceinline__ void act_with_slope(int act, float (&v)[N][V], float (&slope)[N][V])
{
    if (act == kActGelu) {
#pragma unroll
        for (int i = 0; i < N; ++i)
#pragma unroll
            for (int t = 0; t < V; ++t) {
                float e;
                const float z = v[i][t], p = act_normal(z, e);
                slope[i][t] = fmaf(z * 0.39894228040f, e, p);
                v[i][t] = z * p;
            }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i)
#pragma unroll
            for (int t = 0; t < V; ++t) {
                const float z = v[i][t], p = __builtin_amdgcn_rcpf(1.0f + act_exp(-z));
                slope[i][t] = p * fmaf(z, 1.0f - p, 1.0f);
                v[i][t] = z * p;
            }
    }
}

#endif  // __HIPCC__

}  // namespace fgl
