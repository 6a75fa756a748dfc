// What a SIMD does beside its matrix instructions: loops of independent v_mfma_f32_32x32x16_bf16, v_fma_f32, v_exp_f32 and v_cvt_pk_bf16_f32, with 1, 2 and 4 waves per SIMD.
// hipcc --offload-arch=gfx950 -O3 token_overlap.hip -o token_overlap && ./token_overlap
#include <hip/hip_runtime.h>
#include <stdio.h>

using bf16x8 = __bf16 __attribute__((ext_vector_type(8)));
using f32x4 = float __attribute__((ext_vector_type(4)));
using f32x16 = float __attribute__((ext_vector_type(16)));

// NM matrix instructions (SMALL: of 16 x 16 x 32, half the work each), NF fma, NE exp and NC conversions an iteration, half of each behind each half of the matrix instructions
template <bool SMALL, int NM, int NF, int NE, int NC> __global__ __launch_bounds__(256) void loop_kernel(float *out, int iterations) {
    bf16x8 a;
    for (int i = 0; i < 8; ++i) a[i] = (__bf16)(threadIdx.x * 0.001f + i);
    f32x16 big[2] = {};
    f32x4 small[4] = {};
    float x[16], e[8];
    for (int i = 0; i < 16; ++i) x[i] = threadIdx.x * 0.01f + i;
    for (int i = 0; i < 8; ++i) e[i] = 0.5f + i * 0.01f;
    const float y = threadIdx.x * 1e-7f;
    unsigned packed = 0;
    for (int it = 0; it < iterations; ++it)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int i = h * NM / 2; i < (h + 1) * NM / 2; ++i)
                if constexpr (SMALL) small[i % 4] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, a, small[i % 4], 0, 0, 0);
                else big[i % 2] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, a, big[i % 2], 0, 0, 0);
#pragma unroll
            for (int i = h * NF / 2; i < (h + 1) * NF / 2; ++i) asm volatile("v_fma_f32 %0, %0, %1, %1" : "+v"(x[i % 16]) : "v"(y));
#pragma unroll
            for (int i = h * NE / 2; i < (h + 1) * NE / 2; ++i) asm volatile("v_exp_f32 %0, %0" : "+v"(e[i % 8]));
#pragma unroll
            for (int i = h * NC / 2; i < (h + 1) * NC / 2; ++i)
                asm volatile("v_cvt_pk_bf16_f32 %0, %1, %2" : "=v"(packed) : "v"(x[i % 16]), "v"(x[(i + 1) % 16]));
        }
    float s = packed;
    for (int i = 0; i < 16; ++i) s += big[0][i] + big[1][i] + x[i];
    for (int i = 0; i < 4; ++i) s += small[0][i] + small[1][i] + small[2][i] + small[3][i];
    for (int i = 0; i < 8; ++i) s += e[i];
    out[blockIdx.x * 256 + threadIdx.x] = s;
}

template <bool SMALL, int NM, int NF, int NE, int NC> void run(const char *name, float *out) {
    const int iterations = 2000;
    hipEvent_t a, b;
    (void)hipEventCreate(&a), (void)hipEventCreate(&b);
    printf("%-36s", name);
    for (int waves : {1, 2, 4}) {
        float ms = 0.f;
        for (int i = 0; i < 2; ++i) {
            (void)hipEventRecord(a);
            loop_kernel<SMALL, NM, NF, NE, NC><<<256 * waves, 256>>>(out, iterations);
            (void)hipEventRecord(b);
            if (hipEventSynchronize(b) != hipSuccess) return;
            (void)hipEventElapsedTime(&ms, a, b);
        }
        printf("  %d: %6.1f", waves, ms * 1e6 / iterations * 2.4 / waves);
    }
    printf("\n");
    fflush(stdout);
}

int main() {
    float *out;
    if (hipMalloc(&out, 256 * 4 * 256 * sizeof(float)) != hipSuccess) return 1;
    printf("cycles at 2.4 GHz an iteration and wave, by waves per SIMD\n");
    run<false, 2, 0, 0, 0>("2 mfma 32x32x16", out);
    run<true, 4, 0, 0, 0>("4 mfma 16x16x32", out);
    run<false, 0, 32, 0, 0>("32 fma", out);
    run<false, 0, 0, 16, 0>("16 exp", out);
    run<false, 0, 0, 0, 16>("16 cvt_pk", out);
    run<false, 2, 16, 0, 0>("2 mfma 32x32x16 + 16 fma", out);
    run<false, 2, 32, 0, 0>("2 mfma 32x32x16 + 32 fma", out);
    run<true, 4, 32, 0, 0>("4 mfma 16x16x32 + 32 fma", out);
    run<false, 2, 0, 16, 0>("2 mfma 32x32x16 + 16 exp", out);
    run<false, 2, 16, 8, 0>("2 mfma 32x32x16 + 16 fma + 8 exp", out);
    run<false, 2, 0, 0, 16>("2 mfma 32x32x16 + 16 cvt_pk", out);
    return 0;
}
