// Layer norm over the last axis, forward and backward.  m = mean x, r = (mean (x - m)^2 + eps)^(-1/2), n = (x - m) r, y = w n + b;
// h = g w:  dx = r (h - mean h - n mean(h n)),  dw = sum_rows g n,  db = sum_rows g.
// Every sum is held in 32 bits; the mean is taken off before squaring, so a large common offset costs no digits of the variance.
// With 8-bit codes (md_types.hpp) in place of x the backward's n is (x8 - m) r, with m and r those of x itself.
#include "md_types.hpp"

namespace {

template <class T>
__global__ __launch_bounds__(64) void ln_fwd_kernel(const T *__restrict__ x, long long ldx, const float *__restrict__ w,
                                                    const float *__restrict__ b, int C, float eps, T *__restrict__ y,
                                                    float *__restrict__ stat, signed char *__restrict__ codes,
                                                    signed char *__restrict__ scales) {
    const long long row = blockIdx.x;
    const int t = threadIdx.x;
    x += row * ldx;
    y += row * C;
    float s = 0.f;
    for (int c = t; c < C; c += 64) s += (float)x[c];
    const float mean = md_wave_sum(s) / (float)C;
    s = 0.f;
    for (int c = t; c < C; c += 64) {
        const float d = (float)x[c] - mean;
        s = fmaf(d, d, s);
    }
    const float rstd = 1.f / sqrtf(md_wave_sum(s) / (float)C + eps);
    for (int c = t; c < C; c += 64) {
        const float v = ((float)x[c] - mean) * rstd;
        y[c] = (T)fmaf(v, w ? w[c] : 1.f, b ? b[c] : 0.f);
    }
    if (stat && t == 0) {
        stat[2 * row] = mean;
        stat[2 * row + 1] = rstd;
    }
    if (codes) {
        const int groups = (C + MD_ACT8_GROUP - 1) / MD_ACT8_GROUP;
        for (int g = t; g < groups; g += 64) {
            const int hi = min(C, (g + 1) * MD_ACT8_GROUP);
            unsigned amax = 0;
            for (int c = g * MD_ACT8_GROUP; c < hi; ++c) amax = max(amax, __float_as_uint((float)x[c]) & 0x7FFFFFFFu);
            const int code = md_act8_code<T>(amax);
            const float inv = md_act8_inv(code);
            for (int c = g * MD_ACT8_GROUP; c < hi; ++c)
                codes[row * C + c] = code == MD_ACT8_NAN ? 0 : (signed char)md_act8_round((float)x[c], inv);
            scales[row * groups + g] = (signed char)code;
        }
    }
}

template <class T>
__device__ __forceinline__ float ln_value(const T *x, long long ldx, const signed char *codes, const signed char *scales, long long row, int C, int c) {
    if (!codes) return (float)x[row * ldx + c];
    const int groups = (C + MD_ACT8_GROUP - 1) / MD_ACT8_GROUP;
    return (float)codes[row * C + c] * md_act8_scale(scales[row * groups + c / MD_ACT8_GROUP]);
}

template <class T>
__global__ __launch_bounds__(64) void ln_dx_kernel(const T *__restrict__ g, long long ldg, const T *__restrict__ x, long long ldx,
                                                   const signed char *__restrict__ codes, const signed char *__restrict__ scales,
                                                   const float *__restrict__ stat, const float *__restrict__ w, int C, T *__restrict__ dx) {
    const long long row = blockIdx.x;
    const int t = threadIdx.x;
    const float mean = stat[2 * row], rstd = stat[2 * row + 1];
    float sh = 0.f, shn = 0.f;
    for (int c = t; c < C; c += 64) {
        const float h = (float)g[row * ldg + c] * (w ? w[c] : 1.f);
        const float n = (ln_value(x, ldx, codes, scales, row, C, c) - mean) * rstd;
        sh += h;
        shn = fmaf(h, n, shn);
    }
    sh = md_wave_sum(sh) / (float)C;
    shn = md_wave_sum(shn) / (float)C;
    for (int c = t; c < C; c += 64) {
        const float h = (float)g[row * ldg + c] * (w ? w[c] : 1.f);
        const float n = (ln_value(x, ldx, codes, scales, row, C, c) - mean) * rstd;
        dx[row * C + c] = (T)(rstd * (h - sh - n * shn));
    }
}

// one thread per column and slice of rows: partial sums [slice][2][C]
template <class T>
__global__ __launch_bounds__(64) void ln_dwdb_kernel(const T *__restrict__ g, long long ldg, const T *__restrict__ x, long long ldx,
                                                     const signed char *__restrict__ codes, const signed char *__restrict__ scales,
                                                     const float *__restrict__ stat, long long rows, int C, float *__restrict__ part) {
    const int c = blockIdx.x * 64 + threadIdx.x;
    if (c >= C) return;
    float dw = 0.f, db = 0.f;
    for (long long row = blockIdx.y; row < rows; row += gridDim.y) {
        const float v = (float)g[row * ldg + c];
        dw = fmaf(v, (ln_value(x, ldx, codes, scales, row, C, c) - stat[2 * row]) * stat[2 * row + 1], dw);
        db += v;
    }
    part[(size_t)blockIdx.y * 2 * C + c] = dw;
    part[(size_t)blockIdx.y * 2 * C + C + c] = db;
}

__global__ __launch_bounds__(64) void ln_dwdb_sum_kernel(const float *__restrict__ part, int slices, int C, float *__restrict__ dw,
                                                         float *__restrict__ db) {
    const int c = blockIdx.x * 64 + threadIdx.x;
    if (c >= 2 * C) return;
    double s = 0.;
    for (int i = 0; i < slices; ++i) s += part[(size_t)i * 2 * C + c];
    if (c < C) {
        if (dw) dw[c] = (float)s;
    } else if (db) db[c - C] = (float)s;
}

constexpr int LN_SLICES = 512;

}  // namespace

#define LN_CHECK(what)                                                                                                        \
    MD_REQUIRE(rows >= 0 && C >= 1 && C <= (1 << 20), "%s: %lld rows of %d columns (1 .. 2^20 columns)", what, rows, C);      \
    MD_REQUIRE(rows <= 0x7FFFFFFF, "%s: more than 2^31 - 1 rows", what);                                                      \
    MD_REQUIRE((codes == nullptr) == (scales == nullptr), "%s: codes and scales come together", what)

extern "C" int md_layer_norm_fwd(const void *x, int dtype, long long rows, int C, long long ldx, const float *w, const float *b, float eps,
                                 void *y, float *stat, void *codes, void *scales, md_stream_t stream) {
    LN_CHECK("md_layer_norm_fwd");
    MD_REQUIRE(eps >= 0.f, "md_layer_norm_fwd: eps = %g", (double)eps);
    if (rows == 0) return MD_OK;
    MD_REQUIRE(x && y, "md_layer_norm_fwd: null pointer");
    MD_REQUIRE(ldx >= C || rows == 1, "md_layer_norm_fwd: row stride %lld below %d columns", ldx, C);
    hipStream_t s = (hipStream_t)stream;
    MD_DISPATCH_DTYPE(dtype, "md_layer_norm_fwd",
                      ln_fwd_kernel<T><<<(unsigned)rows, 64, 0, s>>>((const T *)x, ldx, w, b, C, eps, (T *)y, stat, (signed char *)codes,
                                                                     (signed char *)scales));
    MD_CHECK_LAUNCH("md_layer_norm_fwd");
    return MD_OK;
}

extern "C" size_t md_layer_norm_bwd_ws_bytes(long long rows, int C) {
    if (rows < 1 || C < 1) return 0;
    return (size_t)(rows < LN_SLICES ? rows : LN_SLICES) * 2 * C * sizeof(float);
}

extern "C" int md_layer_norm_bwd(const void *g, long long ldg, const void *x, long long ldx, const void *codes, const void *scales, int dtype,
                                 const float *stat, const float *w, long long rows, int C, void *dx, float *dw, float *db, void *ws,
                                 size_t ws_bytes, md_stream_t stream) {
    LN_CHECK("md_layer_norm_bwd");
    hipStream_t s = (hipStream_t)stream;
    if (rows > 0) {
        MD_REQUIRE(g && stat && (x || codes), "md_layer_norm_bwd: null pointer");
        MD_REQUIRE((ldg >= C || rows == 1) && (codes || ldx >= C || rows == 1), "md_layer_norm_bwd: row stride below %d columns", C);
        MD_REQUIRE(!(dw || db) || (ws && ws_bytes >= md_layer_norm_bwd_ws_bytes(rows, C)), "md_layer_norm_bwd: workspace of %zu bytes, %zu needed",
                   ws_bytes, md_layer_norm_bwd_ws_bytes(rows, C));
    }
    const signed char *cd = (const signed char *)codes, *sc = (const signed char *)scales;
    if (rows > 0 && dx) {
        MD_DISPATCH_DTYPE(dtype, "md_layer_norm_bwd",
                          ln_dx_kernel<T><<<(unsigned)rows, 64, 0, s>>>((const T *)g, ldg, (const T *)x, ldx, cd, sc, stat, w, C, (T *)dx));
        MD_CHECK_LAUNCH("md_layer_norm_bwd: dx");
    }
    if (dw || db) {
        const int slices = (int)(rows < LN_SLICES ? rows : LN_SLICES);
        if (slices > 0) {
            MD_DISPATCH_DTYPE(dtype, "md_layer_norm_bwd",
                              ln_dwdb_kernel<T><<<dim3(md_cdiv(C, 64), slices), 64, 0, s>>>((const T *)g, ldg, (const T *)x, ldx, cd, sc, stat,
                                                                                            rows, C, (float *)ws));
            MD_CHECK_LAUNCH("md_layer_norm_bwd: partial sums");
        }
        ln_dwdb_sum_kernel<<<md_cdiv(2 * C, 64), 64, 0, s>>>((const float *)ws, slices, C, dw, db);
        MD_CHECK_LAUNCH("md_layer_norm_bwd: sums");
    }
    return MD_OK;
}
