// 8-bit activation checkpoints: what a forward pass keeps for its backward pass, in 1 + 1/32 byte per element.  Format: md_types.hpp.
// Both kernels only move bytes: a lane takes 16 bytes of the tensor (4 or 8 elements), the 8 or 4 lanes of a group find its largest magnitude
// with in-register exchanges, and a few such pieces per lane are in flight together.
#include <algorithm>

#include "md_types.hpp"

namespace {

// pieces per lane: writing a quarter of what is read, packing gains nothing from more than one (70.8 M floats: 74 us, with four 84; 4.8 TB/s); unpacking does
// (69 us against 74; 5.2 TB/s)
constexpr int PACK = 1, UNPACK = 4;
constexpr long long CHUNK = 1LL << 32;        // elements per launch, which has fewer than 2^32 threads

template <class T>
__global__ __launch_bounds__(256) void act8_pack_kernel(const T *__restrict__ x, long long n, signed char *__restrict__ codes,
                                                        signed char *__restrict__ scales) {
    constexpr int W = Wide<T>::n, BLOCK = 256 * W * PACK;
    const long long base = (long long)blockIdx.x * BLOCK;
    const int len = (int)(n - base < BLOCK ? n - base : BLOCK);
    x += base, codes += base, scales += base / MD_ACT8_GROUP;
    float v[PACK][W];
#pragma unroll
    for (int u = 0; u < PACK; ++u) md_load_wide<T>(x, (u * 256 + threadIdx.x) * W, len, v[u]);
#pragma unroll
    for (int u = 0; u < PACK; ++u) {
        const int at = (u * 256 + threadIdx.x) * W;
        const int code = md_act8_code<T>(md_act8_group_max(v[u]));
        unsigned w[W / 4];
        md_act8_encode(v[u], code, w);
        md_store_codes<T>(codes, at, len, w);
        if (at % MD_ACT8_GROUP == 0 && at < len) scales[at / MD_ACT8_GROUP] = (signed char)code;
    }
}

template <class T>
__global__ __launch_bounds__(256) void act8_unpack_kernel(const signed char *__restrict__ codes, const signed char *__restrict__ scales,
                                                          long long n, T *__restrict__ x) {
    constexpr int W = Wide<T>::n, BLOCK = 256 * W * UNPACK;
    const long long base = (long long)blockIdx.x * BLOCK;
    const int len = (int)(n - base < BLOCK ? n - base : BLOCK);
    x += base, codes += base, scales += base / MD_ACT8_GROUP;
    float v[UNPACK][W];
#pragma unroll
    for (int u = 0; u < UNPACK; ++u) {
        const int at = (u * 256 + threadIdx.x) * W;
        md_load_codes<T>(codes, at, len, at < len ? md_act8_scale(scales[at / MD_ACT8_GROUP]) : 0.f, v[u]);
    }
#pragma unroll
    for (int u = 0; u < UNPACK; ++u) md_store_wide<T>(x, (u * 256 + threadIdx.x) * W, len, v[u]);
}

}  // namespace

extern "C" int md_act8_pack(const void *x, int dtype, long long n, void *codes, void *scales, md_stream_t stream) {
    MD_REQUIRE(n >= 0, "md_act8_pack: negative size");
    if (n == 0) return MD_OK;
    MD_REQUIRE(x && codes && scales, "md_act8_pack: null pointer");
    MD_REQUIRE(n <= (1LL << 38), "md_act8_pack: more than 2^38 elements");
    hipStream_t s = (hipStream_t)stream;
    MD_DISPATCH_DTYPE(dtype, "md_act8_pack", {
        for (long long at = 0; at < n; at += CHUNK) {
            const long long m = std::min(n - at, CHUNK);
            act8_pack_kernel<T><<<md_cdiv(m, 256 * Wide<T>::n * PACK), 256, 0, s>>>((const T *)x + at, m, (signed char *)codes + at,
                                                                                    (signed char *)scales + at / MD_ACT8_GROUP);
        }
    });
    MD_CHECK_LAUNCH("md_act8_pack");
    return MD_OK;
}

extern "C" int md_act8_unpack(const void *codes, const void *scales, int dtype, long long n, void *x, md_stream_t stream) {
    MD_REQUIRE(n >= 0, "md_act8_unpack: negative size");
    if (n == 0) return MD_OK;
    MD_REQUIRE(x && codes && scales, "md_act8_unpack: null pointer");
    MD_REQUIRE(n <= (1LL << 38), "md_act8_unpack: more than 2^38 elements");
    hipStream_t s = (hipStream_t)stream;
    MD_DISPATCH_DTYPE(dtype, "md_act8_unpack", {
        for (long long at = 0; at < n; at += CHUNK) {
            const long long m = std::min(n - at, CHUNK);
            act8_unpack_kernel<T><<<md_cdiv(m, 256 * Wide<T>::n * UNPACK), 256, 0, s>>>((const signed char *)codes + at,
                                                                                        (const signed char *)scales + at / MD_ACT8_GROUP, m, (T *)x + at);
        }
    });
    MD_CHECK_LAUNCH("md_act8_unpack");
    return MD_OK;
}
