// 8-bit activation checkpoints: what a forward pass keeps for its backward pass, in 1 + 1/32 byte per element.  Format: md_types.hpp.
#include "md_types.hpp"

namespace {

template <class T>
__global__ __launch_bounds__(256) void act8_pack_kernel(const T *__restrict__ x, long long n, signed char *__restrict__ codes,
                                                        signed char *__restrict__ scales) {
    const long long g = (long long)blockIdx.x * 256 + threadIdx.x;
    const long long at = g * MD_ACT8_GROUP;
    if (at >= n) return;
    const int len = (int)(n - at < MD_ACT8_GROUP ? n - at : MD_ACT8_GROUP);
    unsigned amax = 0;
    for (int i = 0; i < len; ++i) {
        const unsigned b = __float_as_uint((float)x[at + i]) & 0x7FFFFFFFu;
        amax = b > amax ? b : amax;
    }
    const int code = md_act8_code<T>(amax);
    const float inv = md_act8_inv(code);
    for (int i = 0; i < len; ++i) codes[at + i] = code == MD_ACT8_NAN ? 0 : (signed char)md_act8_round((float)x[at + i], inv);
    scales[g] = (signed char)code;
}

template <class T>
__global__ __launch_bounds__(256) void act8_unpack_kernel(const signed char *__restrict__ codes, const signed char *__restrict__ scales,
                                                          long long n, T *__restrict__ x) {
    const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
    if (i < n) x[i] = (T)((float)codes[i] * md_act8_scale(scales[i / MD_ACT8_GROUP]));
}

}  // namespace

extern "C" int md_act8_pack(const void *x, int dtype, long long n, void *codes, void *scales, md_stream_t stream) {
    MD_REQUIRE(n >= 0, "md_act8_pack: negative size");
    if (n == 0) return MD_OK;
    MD_REQUIRE(x && codes && scales, "md_act8_pack: null pointer");
    MD_REQUIRE(n <= (1LL << 38), "md_act8_pack: more than 2^38 elements");
    hipStream_t s = (hipStream_t)stream;
    MD_DISPATCH_DTYPE(dtype, "md_act8_pack",
                      act8_pack_kernel<T><<<md_cdiv(md_cdiv(n, MD_ACT8_GROUP), 256), 256, 0, s>>>((const T *)x, n, (signed char *)codes,
                                                                                                (signed char *)scales));
    MD_CHECK_LAUNCH("md_act8_pack");
    return MD_OK;
}

extern "C" int md_act8_unpack(const void *codes, const void *scales, int dtype, long long n, void *x, md_stream_t stream) {
    MD_REQUIRE(n >= 0, "md_act8_unpack: negative size");
    if (n == 0) return MD_OK;
    MD_REQUIRE(x && codes && scales, "md_act8_unpack: null pointer");
    MD_REQUIRE(n <= (1LL << 38), "md_act8_unpack: more than 2^38 elements");
    hipStream_t s = (hipStream_t)stream;
    MD_DISPATCH_DTYPE(dtype, "md_act8_unpack",
                      act8_unpack_kernel<T><<<md_cdiv(n, 256), 256, 0, s>>>((const signed char *)codes, (const signed char *)scales, n, (T *)x));
    MD_CHECK_LAUNCH("md_act8_unpack");
    return MD_OK;
}
