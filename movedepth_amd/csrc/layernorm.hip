// Layer norm over the last axis, forward and backward.  m = mean x, r = (mean (x - m)^2 + eps)^(-1/2), n = (x - m) r, y = w n + b;
// h = g w:  dx = r (h - mean h - n mean(h n)),  dw = sum_rows g n,  db = sum_rows g.
// Every sum is held in 32 bits; the mean is taken off before squaring, so a large common offset costs no digits of the variance.  What the mean's own rounding leaves
// is the deviations' mean: it comes with the sum of their squares and is taken off both (a constant row of 1000.1 would otherwise deviate by its mean's
// rounding, 6e-5, which 1 / sqrt(eps) makes 0.02).
// With 8-bit codes (md_types.hpp) in place of x the backward's n is (x8 - m) r, with m and r those of x itself.
//
// Bound by memory: each row is read once into registers (16 bytes per lane and access at any alignment, so odd row lengths run like the others), and a
// workgroup goes over many rows, so w and b are read, and the columns' sums kept, in registers.  A row takes TPR lanes with NV accesses
// each; the few lanes of a short row leave a wave several rows at once.
#include <algorithm>

#include "md_types.hpp"

namespace {

// sum over the TPR lanes of a row
template <int TPR> __device__ __forceinline__ float lanes_sum(float v) {
#define LN_DPP_ADD(ctrl) v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), ctrl, 0xF, 0xF, true))
    LN_DPP_ADD(0xB1);
    LN_DPP_ADD(0x4E);
    LN_DPP_ADD(0x141);
    if constexpr (TPR >= 16) LN_DPP_ADD(0x140);
#undef LN_DPP_ADD
    if constexpr (TPR >= 32) v += __shfl_xor(v, 16);
    if constexpr (TPR >= 64) v += __shfl_xor(v, 32);
    return v;
}
// ... and of two values (TPR 256: over the workgroup, through shared memory; calls alternate between slots 0 and 1, so that one barrier each is enough)
template <int TPR> __device__ __forceinline__ void row_sum2(float &v, float &w, float *shared, int slot) {
    v = lanes_sum<TPR>(v);
    w = lanes_sum<TPR>(w);
    if constexpr (TPR == 256) {
        float *at = shared + slot * 8;
        if ((threadIdx.x & 63) == 0) at[threadIdx.x >> 6] = v, at[4 + (threadIdx.x >> 6)] = w;
        __syncthreads();
        v = (at[0] + at[1]) + (at[2] + at[3]);
        w = (at[4] + at[5]) + (at[6] + at[7]);
    }
}
template <int TPR> __device__ __forceinline__ float row_sum(float v, float *shared, int slot) {
    v = lanes_sum<TPR>(v);
    if constexpr (TPR == 256) {
        float *at = shared + slot * 8;
        if ((threadIdx.x & 63) == 0) at[threadIdx.x >> 6] = v;
        __syncthreads();
        v = (at[0] + at[1]) + (at[2] + at[3]);
    }
    return v;
}

template <class T, int TPR, int NV, bool ACT8>
__global__ __launch_bounds__(256) void ln_fwd_kernel(const T *__restrict__ x, long long ldx, const float *__restrict__ w, const float *__restrict__ b,
                                                     int rows, int C, float eps, T *__restrict__ y, float *__restrict__ stat,
                                                     signed char *__restrict__ codes, signed char *__restrict__ scales) {
    constexpr int W = Wide<T>::n, RPB = 256 / TPR;
    __shared__ float shared[16];
    const int sub = threadIdx.x % TPR;
    float wv[NV][W], bv[NV][W];
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < W; ++j) {
            const int c = (i * TPR + sub) * W + j;
            wv[i][j] = w && c < C ? w[c] : 1.f;
            bv[i][j] = b && c < C ? b[c] : 0.f;
        }
    const float inv = 1.f / (float)C;
    const int groups = (C + MD_ACT8_GROUP - 1) / MD_ACT8_GROUP;
    // every lane runs the same rounds: sums cross lanes.  The next row is on its way while this one is summed and stored
    const long long step = (long long)gridDim.x * RPB;
    md_u32x4 next[NV];
    auto fetch = [&](long long row) {
        const T *xr = x + (row < rows ? row : 0) * ldx;
#pragma unroll
        for (int i = 0; i < NV; ++i) next[i] = md_load_raw<T>(xr, (i * TPR + sub) * W, C);
    };
    fetch((long long)blockIdx.x * RPB + threadIdx.x / TPR);
    for (long long at = (long long)blockIdx.x * RPB; at < rows; at += step) {
        const long long row = at + threadIdx.x / TPR;
        const bool live = row < rows;
        float v[NV][W];
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i) md_floats<T>(next[i], v[i]);
        if (at + step < rows) fetch(row + step);
        if constexpr (ACT8)
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int c = (i * TPR + sub) * W;
                const int code = md_act8_code<T>(md_act8_group_max(v[i]));
                unsigned q[W / 4];
                md_act8_encode(v[i], code, q);
                if (live) {
                    md_store_codes<T>(codes + row * C, c, C, q);
                    if (c % MD_ACT8_GROUP == 0 && c < C) scales[row * groups + c / MD_ACT8_GROUP] = (signed char)code;
                }
            }
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int j = 0; j < W; ++j) s += v[i][j];
        const float first = row_sum<TPR>(s, shared, 0) * inv;
        float rest = 0.f;
        s = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int j = 0; j < W; ++j) {
                v[i][j] = (i * TPR + sub) * W + j < C ? v[i][j] - first : 0.f;
                s = fmaf(v[i][j], v[i][j], s);
                rest += v[i][j];
            }
        row_sum2<TPR>(s, rest, shared, 1);
        rest *= inv;
        const float mean = first + rest, rstd = 1.f / sqrtf(fmaxf(fmaf(-rest, rest, s * inv), 0.f) + eps);
        if (!live) continue;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
#pragma unroll
            for (int j = 0; j < W; ++j) v[i][j] = fmaf((v[i][j] - rest) * rstd, wv[i][j], bv[i][j]);
            md_store_wide<T>(y + row * C, (i * TPR + sub) * W, C, v[i]);
        }
        if (stat && sub == 0) {
            stat[2 * row] = mean;
            stat[2 * row + 1] = rstd;
        }
    }
}

// dx and, with `part`, this workgroup's column sums [workgroup][2][C]
template <class T, int TPR, int NV, bool ACT8>
__global__ __launch_bounds__(256) void ln_bwd_kernel(const T *__restrict__ g, long long ldg, const T *__restrict__ x, long long ldx,
                                                     const signed char *__restrict__ codes, const signed char *__restrict__ scales,
                                                     const float *__restrict__ stat, const float *__restrict__ w, int rows, int C, T *__restrict__ dx,
                                                     float *__restrict__ part) {
    constexpr int W = Wide<T>::n, RPB = 256 / TPR;
    __shared__ float shared[RPB > 1 ? 256 * W : 16];
    const int sub = threadIdx.x % TPR;
    float wv[NV][W], dw[NV][W], db[NV][W];
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < W; ++j) {
            const int c = (i * TPR + sub) * W + j;
            wv[i][j] = w && c < C ? w[c] : 1.f;
            dw[i][j] = db[i][j] = 0.f;
        }
    const float inv = 1.f / (float)C;
    const int groups = (C + MD_ACT8_GROUP - 1) / MD_ACT8_GROUP;
    for (long long at = (long long)blockIdx.x * RPB; at < rows; at += (long long)gridDim.x * RPB) {
        const long long row = at + threadIdx.x / TPR;
        const bool live = row < rows;
        const long long from = live ? row : 0;
        const float mean = stat[2 * from], rstd = stat[2 * from + 1];
        float gv[NV][W], n[NV][W];
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (i * TPR + sub) * W;
            md_load_wide<T>(g + from * ldg, c, C, gv[i]);
            if constexpr (ACT8) md_load_codes<T>(codes + from * C, c, C, c < C ? md_act8_scale(scales[from * groups + c / MD_ACT8_GROUP]) : 0.f, n[i]);
            else md_load_wide<T>(x + from * ldx, c, C, n[i]);
        }
        float sh = 0.f, shn = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int j = 0; j < W; ++j) {
                n[i][j] = (n[i][j] - mean) * rstd;           // (behind the row's end g is 0: no sum sees it)
                const float h = gv[i][j] * wv[i][j];
                sh += h;
                shn = fmaf(h, n[i][j], shn);
            }
        sh = row_sum<TPR>(sh, shared, 0) * inv;
        shn = row_sum<TPR>(shn, shared, 1) * inv;
        if (live) {
#pragma unroll
            for (int i = 0; i < NV; ++i)
#pragma unroll
                for (int j = 0; j < W; ++j) {
                    dw[i][j] = fmaf(gv[i][j], n[i][j], dw[i][j]);
                    db[i][j] += gv[i][j];
                }
            if (dx)
#pragma unroll
                for (int i = 0; i < NV; ++i) {
#pragma unroll
                    for (int j = 0; j < W; ++j) gv[i][j] = rstd * (fmaf(gv[i][j], wv[i][j], -sh) - n[i][j] * shn);
                    md_store_wide<T>(dx + row * C, (i * TPR + sub) * W, C, gv[i]);
                }
        }
    }
    if (!part) return;
    part += (size_t)blockIdx.x * 2 * C;
    if constexpr (RPB == 1) {
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int j = 0; j < W; ++j) {
                const int c = (i * TPR + sub) * W + j;
                if (c < C) part[c] = dw[i][j], part[C + c] = db[i][j];
            }
    } else {
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                __syncthreads();
#pragma unroll
                for (int j = 0; j < W; ++j) shared[threadIdx.x * W + j] = k ? db[i][j] : dw[i][j];
                __syncthreads();
                for (int e = threadIdx.x; e < TPR * W; e += 256) {
                    const int c = i * TPR * W + e;
                    float s = 0.f;
                    for (int r = 0; r < RPB; ++r) s += shared[r * TPR * W + e];
                    if (c < C) part[k * C + c] = s;
                }
            }
    }
}

// ---------------------------------------------------------------- rows too long for a workgroup's registers: read again for each sum
constexpr int LONG = 1024;
constexpr long long LONG_ROWS = 1 << 20;      // rows per launch, which has fewer than 2^32 threads

__device__ __forceinline__ float block_sum(float v, float *shared) {
    v = md_wave_sum(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) shared[threadIdx.x >> 6] = v;
    __syncthreads();
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < LONG / 64; ++i) s += shared[i];
    return s;
}

template <class T>
__global__ __launch_bounds__(LONG) void ln_long_fwd_kernel(const T *__restrict__ x, long long ldx, const float *__restrict__ w, const float *__restrict__ b,
                                                           int C, float eps, T *__restrict__ y, float *__restrict__ stat,
                                                           signed char *__restrict__ codes, signed char *__restrict__ scales) {
    constexpr int W = Wide<T>::n;
    __shared__ float shared[LONG / 64];
    const long long row = blockIdx.x;
    x += row * ldx;
    float v[W], s = 0.f;
    for (int c = threadIdx.x * W; c < C; c += LONG * W) {
        md_load_wide<T>(x, c, C, v);
#pragma unroll
        for (int j = 0; j < W; ++j) s += v[j];
    }
    const float first = block_sum(s, shared) / (float)C;
    float rest = 0.f;
    s = 0.f;
    for (int c = threadIdx.x * W; c < C; c += LONG * W) {
        md_load_wide<T>(x, c, C, v);
#pragma unroll
        for (int j = 0; j < W; ++j) {
            const float d = c + j < C ? v[j] - first : 0.f;
            s = fmaf(d, d, s);
            rest += d;
        }
    }
    s = block_sum(s, shared) / (float)C;
    rest = block_sum(rest, shared) / (float)C;
    const float mean = first + rest, rstd = 1.f / sqrtf(fmaxf(fmaf(-rest, rest, s), 0.f) + eps);
    const int groups = (C + MD_ACT8_GROUP - 1) / MD_ACT8_GROUP, rounds = (C + LONG * W - 1) / (LONG * W);
    for (int i = 0; i < rounds; ++i) {                    // whole rounds: a group's lanes exchange its maximum
        const int c = (i * LONG + threadIdx.x) * W;
        md_load_wide<T>(x, c, C, v);
        if (codes) {
            const int code = md_act8_code<T>(md_act8_group_max(v));
            unsigned q[W / 4];
            md_act8_encode(v, code, q);
            md_store_codes<T>(codes + row * C, c, C, q);
            if (c % MD_ACT8_GROUP == 0 && c < C) scales[row * groups + c / MD_ACT8_GROUP] = (signed char)code;
        }
#pragma unroll
        for (int j = 0; j < W; ++j)
            if (c + j < C) v[j] = fmaf((v[j] - first - rest) * rstd, w ? w[c + j] : 1.f, b ? b[c + j] : 0.f);
        md_store_wide<T>(y + row * C, c, C, v);
    }
    if (stat && threadIdx.x == 0) {
        stat[2 * row] = mean;
        stat[2 * row + 1] = rstd;
    }
}

template <class T>
__device__ __forceinline__ float ln_value(const T *x, long long ldx, const signed char *codes, const signed char *scales, long long row, int C, int c) {
    if (!codes) return (float)x[row * ldx + c];
    const int groups = (C + MD_ACT8_GROUP - 1) / MD_ACT8_GROUP;
    return (float)codes[row * C + c] * md_act8_scale(scales[row * groups + c / MD_ACT8_GROUP]);
}

template <class T>
__global__ __launch_bounds__(LONG) void ln_long_dx_kernel(const T *__restrict__ g, long long ldg, const T *__restrict__ x, long long ldx,
                                                          const signed char *__restrict__ codes, const signed char *__restrict__ scales,
                                                          const float *__restrict__ stat, const float *__restrict__ w, int C, T *__restrict__ dx) {
    __shared__ float shared[LONG / 64];
    const long long row = blockIdx.x;
    const float mean = stat[2 * row], rstd = stat[2 * row + 1];
    float sh = 0.f, shn = 0.f;
    for (int c = threadIdx.x; c < C; c += LONG) {
        const float h = (float)g[row * ldg + c] * (w ? w[c] : 1.f);
        sh += h;
        shn = fmaf(h, (ln_value(x, ldx, codes, scales, row, C, c) - mean) * rstd, shn);
    }
    sh = block_sum(sh, shared) / (float)C;
    shn = block_sum(shn, shared) / (float)C;
    for (int c = threadIdx.x; c < C; c += LONG) {
        const float h = (float)g[row * ldg + c] * (w ? w[c] : 1.f);
        dx[row * C + c] = (T)(rstd * (h - sh - (ln_value(x, ldx, codes, scales, row, C, c) - mean) * rstd * shn));
    }
}

template <class T>
__global__ __launch_bounds__(256) void ln_long_columns_kernel(const T *__restrict__ g, long long ldg, const T *__restrict__ x, long long ldx,
                                                              const signed char *__restrict__ codes, const signed char *__restrict__ scales,
                                                              const float *__restrict__ stat, long long rows, int C, float *__restrict__ part) {
    const int c = blockIdx.x * 256 + threadIdx.x;
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

// ---------------------------------------------------------------- the workgroups' column sums in a fixed order: 32 columns x 32 shares of the workgroups
__global__ __launch_bounds__(1024) void ln_sum_kernel(const float *__restrict__ part, int slices, int C, float *__restrict__ dw, float *__restrict__ db) {
    __shared__ float shared[32][33];
    const int col = threadIdx.x & 31, share = threadIdx.x >> 5, c = blockIdx.x * 32 + col;
    float s = 0.f;
    if (c < 2 * C)
        for (int i = share; i < slices; i += 32) s += part[(size_t)i * 2 * C + c];
    shared[share][col] = s;
    __syncthreads();
    if (share == 0 && c < 2 * C) {
        s = 0.f;
#pragma unroll
        for (int i = 0; i < 32; ++i) s += shared[i][col];
        if (c < C) {
            if (dw) dw[c] = s;
        } else if (db)
            db[c - C] = s;
    }
}

// ---------------------------------------------------------------- host side
constexpr int CUS = 256;

// lanes per row and accesses per lane for a row of `wide` 16-byte pieces: up to 4 accesses a lane before a row takes more lanes
struct Split { int tpr, nv; };
Split split_of(int wide) {
    if (wide <= 8) return {8, 1};
    if (wide <= 16) return {16, 1};
    if (wide <= 32) return {32, 1};
    if (wide <= 64) return {64, 1};
    if (wide <= 128) return {64, 2};
    if (wide <= 256) return {64, 4};
    if (wide <= 512) return {256, 2};
    if (wide <= 1024) return {256, 4};
    return {0, 0};                                 // too long for registers
}
int pieces(int dtype, int C) { return md_cdiv(C, 16 / (int)md_dtype_bytes(dtype)); }
// workgroups of the forward pass: w and b are read once per workgroup, so no more than keep the loads in flight (32768 x 2048 bf16: 79 us with 8 a CU, 56 with 2;
// 122880 x 64: 16.6 us with 2, 13.1 with 4)
int fwd_blocks(long long rows, Split s) { return (int)std::min<long long>(md_cdiv(rows, 256 / s.tpr), (s.nv == 1 ? 4 : 2) * CUS); }
// workgroups of the backward pass: each leaves 2 C partial sums, so no more than the chip needs to stream
int bwd_blocks(long long rows, int tpr) { return (int)std::min<long long>(md_cdiv(rows, 256 / tpr), 2 * CUS); }
int column_slices(long long rows) { return (int)std::min<long long>(rows, 64); }

#define LN_CONFIG(S, ...)                                                                      \
    switch ((S).tpr * 10 + (S).nv) {                                                           \
        case 81: { constexpr int TPR = 8, NV = 1; __VA_ARGS__; } break;                        \
        case 161: { constexpr int TPR = 16, NV = 1; __VA_ARGS__; } break;                      \
        case 321: { constexpr int TPR = 32, NV = 1; __VA_ARGS__; } break;                      \
        case 641: { constexpr int TPR = 64, NV = 1; __VA_ARGS__; } break;                      \
        case 642: { constexpr int TPR = 64, NV = 2; __VA_ARGS__; } break;                      \
        case 644: { constexpr int TPR = 64, NV = 4; __VA_ARGS__; } break;                      \
        case 2562: { constexpr int TPR = 256, NV = 2; __VA_ARGS__; } break;                    \
        default: { constexpr int TPR = 256, NV = 4; __VA_ARGS__; } break;                      \
    }

}  // namespace

#define LN_CHECK(what)                                                                                                        \
    MD_REQUIRE(rows >= 0 && C >= 1 && C <= (1 << 20), "%s: %lld rows of %d columns (1 .. 2^20 columns)", what, rows, C);      \
    MD_REQUIRE(rows <= 0x7FFFFFFF, "%s: more than 2^31 - 1 rows", what);                                                      \
    MD_REQUIRE(dtype >= 0 && dtype <= 2, "%s: unknown dtype %d (0 f32, 1 bf16, 2 f16)", what, dtype);                         \
    MD_REQUIRE((codes == nullptr) == (scales == nullptr), "%s: codes and scales come together", what)

extern "C" int md_layer_norm_fwd(const void *x, int dtype, long long rows, int C, long long ldx, const float *w, const float *b, float eps,
                                 void *y, float *stat, void *codes, void *scales, md_stream_t stream) {
    LN_CHECK("md_layer_norm_fwd");
    MD_REQUIRE(eps >= 0.f, "md_layer_norm_fwd: eps = %g", (double)eps);
    if (rows == 0) return MD_OK;
    MD_REQUIRE(x && y, "md_layer_norm_fwd: null pointer");
    MD_REQUIRE(ldx >= C || rows == 1, "md_layer_norm_fwd: row stride %lld below %d columns", ldx, C);
    hipStream_t s = (hipStream_t)stream;
    signed char *cd = (signed char *)codes, *sc = (signed char *)scales;
    const Split sp = split_of(pieces(dtype, C));
    if (!sp.tpr) {
        MD_DISPATCH_DTYPE(dtype, "md_layer_norm_fwd", {
            for (long long r = 0; r < rows; r += LONG_ROWS)
                ln_long_fwd_kernel<T><<<(unsigned)std::min(rows - r, LONG_ROWS), LONG, 0, s>>>(
                    (const T *)x + r * ldx, ldx, w, b, C, eps, (T *)y + r * C, stat ? stat + 2 * r : nullptr, cd ? cd + r * C : nullptr,
                    sc ? sc + r * md_cdiv(C, MD_ACT8_GROUP) : nullptr);
        });
    } else {
        const int grid = fwd_blocks(rows, sp);
        MD_DISPATCH_DTYPE(dtype, "md_layer_norm_fwd", LN_CONFIG(sp, {
            if (codes) ln_fwd_kernel<T, TPR, NV, true><<<grid, 256, 0, s>>>((const T *)x, ldx, w, b, (int)rows, C, eps, (T *)y, stat, cd, sc);
            else ln_fwd_kernel<T, TPR, NV, false><<<grid, 256, 0, s>>>((const T *)x, ldx, w, b, (int)rows, C, eps, (T *)y, stat, cd, sc);
        }));
    }
    MD_CHECK_LAUNCH("md_layer_norm_fwd");
    return MD_OK;
}

extern "C" size_t md_layer_norm_bwd_ws_bytes(long long rows, int C) {
    if (rows < 1 || C < 1) return 0;
    // a workgroup per row at the most, and never more than bwd_blocks or column_slices give
    return (size_t)std::min<long long>(rows, 2 * CUS) * 2 * C * sizeof(float);
}

extern "C" int md_layer_norm_bwd(const void *g, long long ldg, const void *x, long long ldx, const void *codes, const void *scales, int dtype,
                                 const float *stat, const float *w, long long rows, int C, void *dx, float *dw, float *db, void *ws,
                                 size_t ws_bytes, md_stream_t stream) {
    LN_CHECK("md_layer_norm_bwd");
    hipStream_t s = (hipStream_t)stream;
    const bool sums = dw || db;
    int slices = 0;
    if (rows > 0) {
        MD_REQUIRE(g && stat && (x || codes), "md_layer_norm_bwd: null pointer");
        MD_REQUIRE((ldg >= C || rows == 1) && (codes || ldx >= C || rows == 1), "md_layer_norm_bwd: row stride below %d columns", C);
        MD_REQUIRE(!sums || (ws && ws_bytes >= md_layer_norm_bwd_ws_bytes(rows, C)), "md_layer_norm_bwd: workspace of %zu bytes, %zu needed",
                   ws_bytes, md_layer_norm_bwd_ws_bytes(rows, C));
        const signed char *cd = (const signed char *)codes, *sc = (const signed char *)scales;
        const Split sp = split_of(pieces(dtype, C));
        if (!sp.tpr) {
            slices = column_slices(rows);
            MD_DISPATCH_DTYPE(dtype, "md_layer_norm_bwd", {
                for (long long r = 0; dx && r < rows; r += LONG_ROWS)
                    ln_long_dx_kernel<T><<<(unsigned)std::min(rows - r, LONG_ROWS), LONG, 0, s>>>(
                        (const T *)g + r * ldg, ldg, x ? (const T *)x + r * ldx : nullptr, ldx, cd ? cd + r * C : nullptr,
                        sc ? sc + r * md_cdiv(C, MD_ACT8_GROUP) : nullptr, stat + 2 * r, w, C, (T *)dx + r * C);
                if (sums) ln_long_columns_kernel<T><<<dim3(md_cdiv(C, 256), slices), 256, 0, s>>>((const T *)g, ldg, (const T *)x, ldx, cd, sc, stat, rows,
                                                                                                   C, (float *)ws);
            });
        } else {
            slices = bwd_blocks(rows, sp.tpr);
            float *part = sums ? (float *)ws : nullptr;
            MD_DISPATCH_DTYPE(dtype, "md_layer_norm_bwd", LN_CONFIG(sp, {
                if (codes) ln_bwd_kernel<T, TPR, NV, true><<<slices, 256, 0, s>>>((const T *)g, ldg, (const T *)x, ldx, cd, sc, stat, w, (int)rows, C, (T *)dx, part);
                else ln_bwd_kernel<T, TPR, NV, false><<<slices, 256, 0, s>>>((const T *)g, ldg, (const T *)x, ldx, cd, sc, stat, w, (int)rows, C, (T *)dx, part);
            }));
        }
        MD_CHECK_LAUNCH("md_layer_norm_bwd");
    }
    if (sums) {
        ln_sum_kernel<<<md_cdiv(2 * C, 32), 1024, 0, s>>>((const float *)ws, slices, C, dw, db);
        MD_CHECK_LAUNCH("md_layer_norm_bwd: sums");
    }
    return MD_OK;
}
