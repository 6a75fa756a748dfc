// Element types of the token kernels (layernorm.hip, act8.hip, crossattn.hip): `dtype` 0 float32, 1 bfloat16, 2 float16, as md_bn_*.
#pragma once
#include "md_common.hpp"

using bf16_t = __bf16;     // conversions from float round to nearest even (v_cvt_pk_bf16_f32)
using f16_t = _Float16;

// Runs `...` with the alias T set to the element type; anything else is the caller's error.
#define MD_DISPATCH_DTYPE(dtype, what, ...)                                        \
    do {                                                                           \
        if ((dtype) == 0) { using T = float; __VA_ARGS__; }                        \
        else if ((dtype) == 1) { using T = bf16_t; __VA_ARGS__; }                  \
        else if ((dtype) == 2) { using T = f16_t; __VA_ARGS__; }                   \
        else MD_REQUIRE(false, "%s: unknown dtype %d (0 f32, 1 bf16, 2 f16)", what, (int)(dtype)); \
    } while (0)

static inline size_t md_dtype_bytes(int dtype) { return dtype == 0 ? 4 : 2; }

__device__ __forceinline__ float md_wave_max(float v) {
#pragma unroll
    for (int o = 32; o; o >>= 1) v = fmaxf(v, __shfl_xor(v, o));
    return v;
}

// ---------------------------------------------------------------- 8-bit activations
// 32 neighbours of a row share one scale 2^e: value = n 2^e, n a whole number of [-127, 127].  e is the least exponent for which the
// group's largest magnitude a rounds to 127 or less.  With a = m 2^E, 1 <= m < 2: a 2^-(E-6) = 64 m lies in [64, 128) and rounds to
// 128 exactly when m >= 255/128, i.e. when the seven leading mantissa bits are all ones -- adding 2^16 to the bit pattern then carries
// into the exponent field, so e + 6 is read straight from it.  A power of two makes the scaling and its inverse exact: the whole number
// is a correctly rounded x 2^-e (ties to even) and n 2^e is representable in x's own type, so nothing is rounded when it comes back.
// The range of e is where that holds: below emin the step would be subnormal (fp32 / bf16: 2^-126; fp16: 2^-24, its smallest value),
// above emax 127 2^e would overflow (fp16: 127 2^9 = 65024), and n is cut off at 127 there.
// A group with an infinity or a NaN is stored as MD_ACT8_NAN and comes back as NaN: an overflow must not turn into a plausible number.
#define MD_ACT8_GROUP 32
#define MD_ACT8_NAN (-128)

template <class T> struct Act8Range { static constexpr int lo = -126, hi = 121; };
template <> struct Act8Range<f16_t> { static constexpr int lo = -24, hi = 9; };

// scale code of a group from the bit pattern of its largest magnitude (NaN and infinity have the largest patterns)
template <class T> __device__ __forceinline__ int md_act8_code(unsigned amax_bits) {
    if (amax_bits >= 0x7F800000u) return MD_ACT8_NAN;
    const int e = (int)((amax_bits + 0x10000u) >> 23) - 133;
    return e < Act8Range<T>::lo ? Act8Range<T>::lo : e > Act8Range<T>::hi ? Act8Range<T>::hi : e;
}
__device__ __forceinline__ float md_act8_inv(int code) {       // 2^-e
    return code == MD_ACT8_NAN ? 0.f : __uint_as_float((unsigned)(127 - code) << 23);
}
__device__ __forceinline__ float md_act8_scale(int code) {     // 2^e, NaN for a group that held one
    return code == MD_ACT8_NAN ? __uint_as_float(0x7FC00000u) : __uint_as_float((unsigned)(127 + code) << 23);
}
__device__ __forceinline__ int md_act8_round(float x, float inv) {
    const float r = rintf(x * inv);
    return (int)fminf(fmaxf(r, -127.f), 127.f);
}
