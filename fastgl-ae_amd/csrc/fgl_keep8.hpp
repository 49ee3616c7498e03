// Rows held in 8 bits a value for a backward pass.  32 neighbouring columns of a row share a step, a power of two:
//   step = 2^(max(floor(log2(largest magnitude)), -120) - 6),   code = clamp(nearest whole number to v / step, -127, 127), a signed byte
// so a value is off by half a step, 2^-7 of its neighbours' largest at most (by a whole one where that lies in the last half step below a power of
// two).  A step is held as the exponent of an fp32 value, 255 where one of the 32 is infinite or not a number; all of them are not a number then.
//
// Why powers of two: which code is nearest needs no rounded quotient, so that it is the same whoever forms it; and a code times a step is a
// bf16 value, exactly (seven bits and a sign), which the matrix instructions take as it is: an fp32 product with it is three bf16 products instead of six.
// The price is up to a bit of the eight, against a step of a 127th of the largest.
#pragma once

#include "fgl_common.hpp"

namespace fgl {

inline int64_t k8_columns(int64_t d) { return (d + 31) / 32 * 32; }  // of the codes, those past the end zero

#if defined(__HIPCC__)

// Lanes of a row of 16 exchange what they hold with their neighbour, their neighbouring pair, four or eight.
template <int CTRL>
__device__ __forceinline__ uint32_t dpp_u32(uint32_t v) { return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xF, 0xF, true); }
constexpr int kDppXor1 = 0xB1, kDppXor2 = 0x4E, kDppHalfMirror = 0x141, kDppMirror = 0x140;

// Over groups of GROUP neighbouring lanes (4, 8, 16: those that hold what one step is shared by), the largest of a whole number
template <int GROUP>
__device__ __forceinline__ uint32_t group_max(uint32_t v)
{
    static_assert(GROUP == 4 || GROUP == 8 || GROUP == 16, "");
    uint32_t o = dpp_u32<kDppXor1>(v);
    v = v > o ? v : o;
    o = dpp_u32<kDppXor2>(v);
    v = v > o ? v : o;
    if constexpr (GROUP >= 8) {
        o = dpp_u32<kDppHalfMirror>(v);
        v = v > o ? v : o;
    }
    if constexpr (GROUP >= 16) {
        o = dpp_u32<kDppMirror>(v);
        v = v > o ? v : o;
    }
    return v;
}

// The same lanes' bits (8 or 16 lanes), together
template <int GROUP>
__device__ __forceinline__ uint32_t group_or(uint32_t v)
{
    static_assert(GROUP == 8 || GROUP == 16, "");
    v |= dpp_u32<kDppXor1>(v);
    v |= dpp_u32<kDppXor2>(v);
    v |= dpp_u32<kDppHalfMirror>(v);
    if constexpr (GROUP == 16) v |= dpp_u32<kDppMirror>(v);
    return v;
}

// the exponent that stands for the step, from floor(log2) of the largest magnitude
__device__ __forceinline__ uint32_t k8_step(int log2_most) { return (uint32_t)((log2_most < -120 ? -120 : log2_most) + 121); }
constexpr uint32_t kStepNone = 255;

// 1 / step, by which a value is multiplied without rounding (a result below fp32's normal range is below half a step)
__device__ __forceinline__ float k8_inverse(uint32_t step) { return __uint_as_float((254u - step) << 23); }
__device__ __forceinline__ double k8_inverse64(uint32_t step) { return __hiloint2double((int)((1023u + 127u - step) << 20), 0); }

// the code of v plus 128: its sum with 1.5 2^23 + 128 is rounded to a whole number, the nearest, in its lower bits (64 bits: 1.5 2^52).  Four of them at a time become signed
// bytes by their upper bits.
constexpr uint32_t kSigned = 0x80808080u;
__device__ __forceinline__ uint32_t k8_clamp(int r) { return (uint32_t)(r < 1 ? 1 : r > 255 ? 255 : r); }
__device__ __forceinline__ uint32_t k8_code(float v, float inverse) { return k8_clamp((int)__float_as_uint(fmaf(v, inverse, 0x1.8p23f + 128.0f)) - 0x4B400000); }
__device__ __forceinline__ uint32_t k8_code(double v, double inverse) { return k8_clamp(__double2loint(fma(v, inverse, 0x1.8p52 + 128.0))); }

// the step that an exponent stands for, exactly (255: no number, which infinity times zero is)
__device__ __forceinline__ float k8_step_value(uint32_t step)
{
    const float s = __uint_as_float(step << 23);
    return fmaf(s, 0.0f, s);
}
// code number c of a word, exactly.  Signed bytes, so that a value is one product: next to the largest finite values 128 steps, which an offset would take off, are infinite.
__device__ __forceinline__ float k8_code_value(uint32_t word, int c) { return (float)(int)__builtin_amdgcn_sbfe((int)word, 8 * c, 8); }

#endif  // __HIPCC__

}  // namespace fgl
