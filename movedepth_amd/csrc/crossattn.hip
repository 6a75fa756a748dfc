// Attention from queries (B, Nq, Hq, d) to another sequence's keys and values (B, Nk, Hk, d), Hq a multiple of Hk (query head i reads key head
// i / (Hq / Hk)), with an optional mask of valid keys (B, Nk):
//   S = scale q k^T over the valid keys, P = softmax S, O = P V;   D = sum g O, dV = P^T g, dS = P (g V^T - D), dQ = scale dS K, dK = scale dS^T Q.
// One pass over the keys: running maximum m and sum l per query, O rescaled when m grows.  A masked key is not read into any product (what stands
// there may be NaN); a query without a valid key gets zeros and gives zero gradients.  `lse` = m + log l per query, in units of log 2; +inf without a key.
#include "md_types.hpp"

namespace {

constexpr float LOG2E = 1.4426950408889634f;

// one wave per query row; a lane holds elements lane and lane + 64 of a row
template <class T>
__global__ __launch_bounds__(64) void xa_fwd_kernel(md_attn_desc a) {
    const int t = threadIdx.x, qi = blockIdx.x, hq = blockIdx.y, b = blockIdx.z, hk = hq / (a.Hq / a.Hk);
    const T *q = (const T *)a.q + b * a.q_sb + qi * a.q_sn + hq * a.q_sh;
    const T *k = (const T *)a.k + b * a.k_sb + hk * a.k_sh, *v = (const T *)a.v + b * a.v_sb + hk * a.v_sh;
    const unsigned char *mask = a.key_mask ? (const unsigned char *)a.key_mask + b * a.mask_sb : nullptr;
    const bool in0 = t < a.d, in1 = t + 64 < a.d;
    const float c = a.scale * LOG2E, q0 = in0 ? (float)q[t] : 0.f, q1 = in1 ? (float)q[t + 64] : 0.f;
    float m = -INFINITY, l = 0.f, o0 = 0.f, o1 = 0.f;
    for (int i = 0; i < a.Nk; ++i) {
        if (mask && !mask[i]) continue;
        const T *kr = k + i * a.k_sn, *vr = v + i * a.v_sn;
        const float s = md_wave_sum(q0 * (in0 ? (float)kr[t] : 0.f) + q1 * (in1 ? (float)kr[t + 64] : 0.f)) * c;
        const float mn = fmaxf(m, s), r = exp2f(m - mn), p = exp2f(s - mn);
        m = mn;
        l = l * r + p;
        o0 = o0 * r + p * (in0 ? (float)vr[t] : 0.f);
        o1 = o1 * r + p * (in1 ? (float)vr[t + 64] : 0.f);
    }
    const float inv = l > 0.f ? 1.f / l : 0.f;
    T *o = (T *)a.o + (((long long)b * a.Nq + qi) * a.Hq + hq) * a.d;
    if (in0) o[t] = (T)(o0 * inv);
    if (in1) o[t + 64] = (T)(o1 * inv);
    if (a.lse && t == 0) a.lse[((long long)b * a.Hq + hq) * a.Nq + qi] = l > 0.f ? m + log2f(l) : INFINITY;
}

template <class T>
__global__ __launch_bounds__(64) void xa_dq_kernel(md_attn_desc a, float *__restrict__ delta) {
    const int t = threadIdx.x, qi = blockIdx.x, hq = blockIdx.y, b = blockIdx.z, hk = hq / (a.Hq / a.Hk);
    const T *q = (const T *)a.q + b * a.q_sb + qi * a.q_sn + hq * a.q_sh, *g = (const T *)a.g + b * a.g_sb + qi * a.g_sn + hq * a.g_sh;
    const T *k = (const T *)a.k + b * a.k_sb + hk * a.k_sh, *v = (const T *)a.v + b * a.v_sb + hk * a.v_sh;
    const long long at = (((long long)b * a.Nq + qi) * a.Hq + hq) * a.d;
    const T *o = (const T *)a.o + at;
    const unsigned char *mask = a.key_mask ? (const unsigned char *)a.key_mask + b * a.mask_sb : nullptr;
    const bool in0 = t < a.d, in1 = t + 64 < a.d;
    const float c = a.scale * LOG2E, q0 = in0 ? (float)q[t] : 0.f, q1 = in1 ? (float)q[t + 64] : 0.f;
    const float g0 = in0 ? (float)g[t] : 0.f, g1 = in1 ? (float)g[t + 64] : 0.f;
    const float D = md_wave_sum(g0 * (in0 ? (float)o[t] : 0.f) + g1 * (in1 ? (float)o[t + 64] : 0.f));
    const float lse = a.lse[((long long)b * a.Hq + hq) * a.Nq + qi];
    if (t == 0) delta[((long long)b * a.Hq + hq) * a.Nq + qi] = D;
    float d0 = 0.f, d1 = 0.f;
    for (int i = 0; i < a.Nk; ++i) {
        if (mask && !mask[i]) continue;
        const T *kr = k + i * a.k_sn, *vr = v + i * a.v_sn;
        const float k0 = in0 ? (float)kr[t] : 0.f, k1 = in1 ? (float)kr[t + 64] : 0.f;
        const float p = exp2f(md_wave_sum(q0 * k0 + q1 * k1) * c - lse);
        const float ds = p * (md_wave_sum(g0 * (in0 ? (float)vr[t] : 0.f) + g1 * (in1 ? (float)vr[t + 64] : 0.f)) - D);
        d0 = fmaf(ds, k0, d0);
        d1 = fmaf(ds, k1, d1);
    }
    if (!a.dq) return;
    T *dq = (T *)a.dq + at;
    if (in0) dq[t] = (T)(d0 * a.scale);
    if (in1) dq[t + 64] = (T)(d1 * a.scale);
}

// one wave per key row, over the queries of every head that shares it
template <class T>
__global__ __launch_bounds__(64) void xa_dkv_kernel(md_attn_desc a, const float *__restrict__ delta) {
    const int t = threadIdx.x, ki = blockIdx.x, hk = blockIdx.y, b = blockIdx.z, G = a.Hq / a.Hk;
    const bool in0 = t < a.d, in1 = t + 64 < a.d;
    const bool valid = !a.key_mask || ((const unsigned char *)a.key_mask)[b * a.mask_sb + ki];
    float dk0 = 0.f, dk1 = 0.f, dv0 = 0.f, dv1 = 0.f;
    if (valid) {
        const T *k = (const T *)a.k + b * a.k_sb + ki * a.k_sn + hk * a.k_sh, *v = (const T *)a.v + b * a.v_sb + ki * a.v_sn + hk * a.v_sh;
        const float c = a.scale * LOG2E, k0 = in0 ? (float)k[t] : 0.f, k1 = in1 ? (float)k[t + 64] : 0.f;
        const float v0 = in0 ? (float)v[t] : 0.f, v1 = in1 ? (float)v[t + 64] : 0.f;
        for (int h = hk * G; h < (hk + 1) * G; ++h)
            for (int i = 0; i < a.Nq; ++i) {
                const T *q = (const T *)a.q + b * a.q_sb + i * a.q_sn + h * a.q_sh, *g = (const T *)a.g + b * a.g_sb + i * a.g_sn + h * a.g_sh;
                const float q0 = in0 ? (float)q[t] : 0.f, q1 = in1 ? (float)q[t + 64] : 0.f;
                const float g0 = in0 ? (float)g[t] : 0.f, g1 = in1 ? (float)g[t + 64] : 0.f;
                const long long r = ((long long)b * a.Hq + h) * a.Nq + i;
                const float p = exp2f(md_wave_sum(q0 * k0 + q1 * k1) * c - a.lse[r]);
                const float ds = p * (md_wave_sum(g0 * v0 + g1 * v1) - delta[r]);
                dk0 = fmaf(ds, q0, dk0);
                dk1 = fmaf(ds, q1, dk1);
                dv0 = fmaf(p, g0, dv0);
                dv1 = fmaf(p, g1, dv1);
            }
    }
    const long long at = (((long long)b * a.Nk + ki) * a.Hk + hk) * a.d;
    T *dk = (T *)a.dk + at, *dv = (T *)a.dv + at;
    if (in0) dk[t] = (T)(dk0 * a.scale), dv[t] = (T)dv0;
    if (in1) dk[t + 64] = (T)(dk1 * a.scale), dv[t + 64] = (T)dv1;
}

int check(const md_attn_desc &a, const char *what) {
    MD_REQUIRE(a.dtype >= 0 && a.dtype <= 2, "%s: unknown dtype %d (0 f32, 1 bf16, 2 f16)", what, a.dtype);
    MD_REQUIRE(a.B >= 0 && a.Nq >= 0 && a.Nk >= 0, "%s: negative size", what);
    MD_REQUIRE(a.d >= 1 && a.d <= MD_ATTN_MAX_D, "%s: head size %d (1 .. %d)", what, a.d, MD_ATTN_MAX_D);
    MD_REQUIRE(a.Hk >= 1 && a.Hq >= 1 && a.Hq % a.Hk == 0, "%s: %d query heads are not a multiple of %d key heads", what, a.Hq, a.Hk);
    MD_REQUIRE(a.Hq <= 65535 && a.B <= 65535, "%s: more than 65535 heads or sequences", what);
    MD_REQUIRE(a.scale == a.scale, "%s: scale is NaN", what);
    return MD_OK;
}

}  // namespace

extern "C" size_t md_attn_desc_bytes(void) { return sizeof(md_attn_desc); }

extern "C" size_t md_cross_attn_ws_bytes(const md_attn_desc *a, int backward) {
    return a && backward && a->B > 0 && a->Nq > 0 && a->Hq > 0 ? (size_t)a->B * a->Hq * a->Nq * sizeof(float) : 0;
}

extern "C" int md_cross_attn_fwd(const md_attn_desc *a, void *ws, size_t ws_bytes, md_stream_t stream) {
    MD_REQUIRE(a, "md_cross_attn_fwd: null descriptor");
    if (int rc = check(*a, "md_cross_attn_fwd")) return rc;
    if (a->B == 0 || a->Nq == 0) return MD_OK;
    MD_REQUIRE(a->q && a->o && (a->Nk == 0 || (a->k && a->v)), "md_cross_attn_fwd: null pointer");
    hipStream_t s = (hipStream_t)stream;
    MD_DISPATCH_DTYPE(a->dtype, "md_cross_attn_fwd", xa_fwd_kernel<T><<<dim3(a->Nq, a->Hq, a->B), 64, 0, s>>>(*a));
    MD_CHECK_LAUNCH("md_cross_attn_fwd");
    return MD_OK;
}

extern "C" int md_cross_attn_bwd(const md_attn_desc *a, void *ws, size_t ws_bytes, md_stream_t stream) {
    MD_REQUIRE(a, "md_cross_attn_bwd: null descriptor");
    if (int rc = check(*a, "md_cross_attn_bwd")) return rc;
    if (a->B == 0) return MD_OK;
    MD_REQUIRE((a->dk == nullptr) == (a->dv == nullptr), "md_cross_attn_bwd: dk and dv come together");
    MD_REQUIRE(a->Nq == 0 || (a->q && a->o && a->g && a->lse), "md_cross_attn_bwd: null pointer");
    MD_REQUIRE(a->Nk == 0 || (a->k && a->v), "md_cross_attn_bwd: null pointer");
    MD_REQUIRE(ws_bytes >= md_cross_attn_ws_bytes(a, 1) && (ws || ws_bytes == 0), "md_cross_attn_bwd: workspace of %zu bytes, %zu needed", ws_bytes,
               md_cross_attn_ws_bytes(a, 1));
    hipStream_t s = (hipStream_t)stream;
    float *delta = (float *)ws;
    if (a->Nq) {
        MD_DISPATCH_DTYPE(a->dtype, "md_cross_attn_bwd", xa_dq_kernel<T><<<dim3(a->Nq, a->Hq, a->B), 64, 0, s>>>(*a, delta));
        MD_CHECK_LAUNCH("md_cross_attn_bwd: dq");
    }
    if (a->Nk && a->dk) {
        MD_DISPATCH_DTYPE(a->dtype, "md_cross_attn_bwd", xa_dkv_kernel<T><<<dim3(a->Nk, a->Hk, a->B), 64, 0, s>>>(*a, delta));
        MD_CHECK_LAUNCH("md_cross_attn_bwd: dk, dv");
    }
    return MD_OK;
}
