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

// ---------------------------------------------------------------- 16 bytes of T, or as many 8-bit codes, at any element's address
// (global memory takes 16-byte accesses at every alignment; rows of odd length then run like the others)
using md_u32x4 = unsigned __attribute__((ext_vector_type(4)));
template <class T> struct Wide {
    static constexpr int n = 16 / (int)sizeof(T);
    struct __attribute__((packed, aligned(sizeof(T)))) Mem { md_u32x4 v; };
    struct __attribute__((packed, aligned(1))) Codes { unsigned char b[n]; };
};

// elements at .. at + n - 1 of a row of `len`, zeros behind its end; as they are in memory, and as floats
template <class T> __device__ __forceinline__ md_u32x4 md_load_raw(const T *row, int at, int len) {
    constexpr int n = Wide<T>::n;
    if (at + n <= len) return ((const typename Wide<T>::Mem *)(row + at))->v;
    T raw[n];
#pragma unroll
    for (int j = 0; j < n; ++j) raw[j] = at + j < len ? row[at + j] : (T)0.f;
    md_u32x4 w;
    __builtin_memcpy(&w, raw, 16);
    return w;
}
template <class T> __device__ __forceinline__ void md_floats(md_u32x4 w, float (&v)[Wide<T>::n]) {
    T raw[Wide<T>::n];
    __builtin_memcpy(raw, &w, 16);
#pragma unroll
    for (int j = 0; j < Wide<T>::n; ++j) v[j] = (float)raw[j];
}
template <class T> __device__ __forceinline__ void md_load_wide(const T *row, int at, int len, float (&v)[Wide<T>::n]) {
    md_floats<T>(md_load_raw<T>(row, at, len), v);
}
template <class T> __device__ __forceinline__ void md_store_wide(T *row, int at, int len, const float (&v)[Wide<T>::n]) {
    constexpr int n = Wide<T>::n;
    T raw[n];
#pragma unroll
    for (int j = 0; j < n; ++j) raw[j] = (T)v[j];
    if (at + n <= len) {
        md_u32x4 w;
        __builtin_memcpy(&w, raw, 16);
        ((typename Wide<T>::Mem *)(row + at))->v = w;
    } else {
#pragma unroll
        for (int j = 0; j < n; ++j)
            if (at + j < len) row[at + j] = raw[j];
    }
}

// largest bit pattern of a group's magnitudes, over the 32 / n lanes that hold it
template <int n> __device__ __forceinline__ unsigned md_act8_group_max(const float (&v)[n]) {
    int m = 0;
#pragma unroll
    for (int j = 0; j < n; ++j) m = max(m, (int)(__float_as_uint(v[j]) & 0x7FFFFFFFu));
    m = max(m, __builtin_amdgcn_update_dpp(m, m, 0xB1, 0xF, 0xF, false));           // lane ^ 1
    m = max(m, __builtin_amdgcn_update_dpp(m, m, 0x4E, 0xF, 0xF, false));           // lane ^ 2
    if (n == 4) m = max(m, __builtin_amdgcn_update_dpp(m, m, 0x141, 0xF, 0xF, false));   // the other half of 8
    return (unsigned)m;
}
// n codes into a register pair, lowest byte first
template <int n> __device__ __forceinline__ void md_act8_encode(const float (&v)[n], int code, unsigned (&w)[n / 4]) {
    const float inv = md_act8_inv(code);
#pragma unroll
    for (int j = 0; j < n; ++j) {
        const unsigned q = code == MD_ACT8_NAN ? 0u : (unsigned)md_act8_round(v[j], inv) & 0xFFu;
        w[j / 4] = j % 4 ? w[j / 4] | q << (8 * (j % 4)) : q;
    }
}
template <class T> __device__ __forceinline__ void md_store_codes(signed char *row, int at, int len, const unsigned (&w)[Wide<T>::n / 4]) {
    constexpr int n = Wide<T>::n;
    if (at + n <= len) {
        typename Wide<T>::Codes c;
        __builtin_memcpy(&c, w, n);
        *(typename Wide<T>::Codes *)(row + at) = c;
    } else {
#pragma unroll
        for (int j = 0; j < n; ++j)
            if (at + j < len) row[at + j] = (signed char)(w[j / 4] >> (8 * (j % 4)));
    }
}
template <class T> __device__ __forceinline__ void md_load_codes(const signed char *row, int at, int len, float scale, float (&v)[Wide<T>::n]) {
    constexpr int n = Wide<T>::n;
    unsigned w[n / 4];
    if (at + n <= len) {
        const typename Wide<T>::Codes c = *(const typename Wide<T>::Codes *)(row + at);
        __builtin_memcpy(w, &c, n);
    } else {
#pragma unroll
        for (int j = 0; j < n; ++j) {
            const unsigned q = at + j < len ? (unsigned)(unsigned char)row[at + j] : 0u;
            w[j / 4] = j % 4 ? w[j / 4] | q << (8 * (j % 4)) : q;
        }
    }
#pragma unroll
    for (int j = 0; j < n; ++j) v[j] = (float)(signed char)(w[j / 4] >> (8 * (j % 4))) * scale;
}
