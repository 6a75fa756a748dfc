// Attention from queries (B, Nq, Hq, d) to another sequence's keys and values (B, Nk, Hk, d), Hq a multiple of Hk (query head i reads key head
// i / (Hq / Hk)), with an optional mask of valid keys (B, Nk):
//   S = scale q k^T over the valid keys, P = softmax S, O = P V;   D = sum g O, dV = P^T g, dS = P (g V^T - D), dQ = scale dS K, dK = scale dS^T Q.
//
// The problem is taken as Z = B Hk independent ones of M = (Hq / Hk) Nq query rows (the heads that share a key head, one behind the other) and
// N keys.  Nothing of size M x N is stored: a running maximum m and sum l per query row, O rescaled when m grows, and in the backward
// pass P again from S and the row's log-sum `lse` = m + log2 l (all exponents are in units of log 2; +inf for a row without keys).
//
// Long problems run in three steps: xa_compact lists the valid keys (so a masked key costs nothing and what stands in its row, NaN
// among it, is never touched), xa_pack writes every operand in the order in which the matrix instruction's lanes take it, and the tile kernels
// copy such fragments to shared memory with 1 KB direct loads and read them back without bank conflicts.  A few query rows against long keys
// (serving) are bound by reading K and V once and go to xa_few, which reads them in place.
//
// Fragments of v_mfma_f32_32x32x16 (A, B: lane l holds row / column l % 32 and 8 neighbours of the contraction axis; C: lane l holds column l % 32 and
// rows 8 (r / 4) + 4 (l / 32) + r % 4, r = 0 .. 15):
//   "R": 32 rows x 16 dims, lane l: row l % 32, dims 8 (l / 32) + 0 .. 7.  Both operands of S and g V^T.
//   "T": 32 dims x 16 rows, lane l: dim l % 32, rows 8 (j / 4) + 4 (l / 32) + j % 4, j = 0 .. 7 -- the order in which C leaves its rows in
//        a lane's registers, so P and dS go from the accumulators of one product into the operand of the next without crossing lanes.
// Products run transposed (S^T = K Q^T, O^T = V^T P^T): a lane then owns one query, its softmax is in-lane but for one exchange of halves.
//
// float32 runs on the bf16 instructions too: every operand as the sum of three bf16 pieces (8 + 8 + 8 bits), six products of pieces whose
// magnitudes matter to 2^-24, which is 6 / 16 of what the float32 matrix instruction costs.  2-byte types: P and dS are rounded to
// the type before their products (half a step relative), as the matrix instruction takes them: o, dq, dk and dv then carry two roundings of that size instead of
// one (bf16, norm-wise: 2.5e-3 against 1.7e-3).  Two pieces of P and dS would halve that and cost 35 to 50 % (both passes, bf16: 1.28 to 1.86 ms for 2 x 2 x 20480^2
// heads of 32, 1.40 to 1.90 for 2 x 16 x 4096 x 8192 heads of 64).  l sums P as it is before that rounding, so that `lse`, from which the backward pass takes P again, is that of
// the exact weights; D is formed in 32 bits from o as it was stored.  float16 holds P times 2^7 (forward) or 2^15 (backward) and dS times a power
// of two from |g| |v| (ds_scale), so that the small weights of long rows do not fall below its range.
#include <algorithm>
#include <type_traits>

#include "md_types.hpp"

namespace {

constexpr float LOG2E = 1.4426950408889634f;
constexpr float LAZY = 8.f;     // m is raised only when a score passes it by more than 2^8: the sums stay exact, O is rarely rescaled
// m starts at the lowest finite number: a valid key whose score is -inf then weighs exp2(-inf - m) = 0, wherever it stands, while every finite score raises m or
// (that number itself) weighs exp2(0).  From -inf it would be exp2(-inf + inf).  A row whose scores are all -inf ends with a sum of 0, as one without keys
constexpr float LOWEST = -3.402823466e38f;

using f32x16 = float __attribute__((ext_vector_type(16)));
template <class E> struct Vec { using v8 = E __attribute__((ext_vector_type(8))); };
template <class T> struct Frag { using E = T; static constexpr int NP = 1; };
template <> struct Frag<float> { using E = bf16_t; static constexpr int NP = 3; };

__device__ __forceinline__ f32x16 mfma(Vec<bf16_t>::v8 a, Vec<bf16_t>::v8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x16 mfma(Vec<f16_t>::v8 a, Vec<f16_t>::v8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }

// c + a b for operands of NP pieces, the smallest products first
template <class E, int NP>
__device__ __forceinline__ f32x16 mfma_pieces(const typename Vec<E>::v8 (&a)[NP], const typename Vec<E>::v8 (&b)[NP], f32x16 c) {
    if constexpr (NP == 3) {
        c = mfma(a[2], b[0], c);
        c = mfma(a[1], b[1], c);
        c = mfma(a[0], b[2], c);
        c = mfma(a[1], b[0], c);
        c = mfma(a[0], b[1], c);
    }
    return mfma(a[0], b[0], c);
}

// 8 values as NP pieces each.  Pairs are rounded together (one instruction), and the pair's halves are its values' bits: what is left over is exact
template <class E, int NP> __device__ __forceinline__ void split8(const float (&v)[8], typename Vec<E>::v8 (&out)[NP]) {
    using v2 = E __attribute__((ext_vector_type(2)));
    using f2 = float __attribute__((ext_vector_type(2)));
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
        float x = v[j], y = v[j + 1];
#pragma unroll
        for (int p = 0; p < NP; ++p) {
            const v2 r = __builtin_convertvector((f2){x, y}, v2);
            out[p][j] = r[0], out[p][j + 1] = r[1];
            if (p + 1 < NP) {
                const unsigned w = __builtin_bit_cast(unsigned, r);        // (bf16: the upper halves of two floats)
                x -= __uint_as_float(w << 16);
                y -= __uint_as_float(w & 0xFFFF0000u);
            }
        }
    }
}

__device__ __forceinline__ float swap_halves_max(float v) {
    auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float swap_halves_sum(float v) {
    auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// 1 KB, 16 bytes per lane, from global memory straight to shared memory (lane order); complete after s_waitcnt vmcnt(0)
__device__ __forceinline__ void load_chunk(const char *from, char *to, int lane) {
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)(from + lane * 16),
                                     (__attribute__((address_space(3))) void *)to, 16, 0, 0);
}
__device__ __forceinline__ void wait_loads_and_barrier() {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
}
template <class E, int NP> __device__ __forceinline__ void read_frag(const char *at, int lane, typename Vec<E>::v8 (&out)[NP]) {
#pragma unroll
    for (int p = 0; p < NP; ++p) out[p] = *(const typename Vec<E>::v8 *)(at + p * 1024 + lane * 16);
}

// neighbouring workgroups of a launch go to the 8 dies in turn: give each die a contiguous share of the work, so that the tiles of one z share its cache
__device__ __forceinline__ int die_order(int block, int blocks) {
    const int per = (blocks + 7) / 8;
    return (block % 8) * per + block / 8;
}

// Workgroups of 4 waves that a CU holds at once (registers, and shared memory where it is short), per kernel; also what the compiler is asked to keep to.
template <int NP, int KS, int QT> constexpr int fwd_per_cu() { return NP == 3 ? (KS <= 4 ? 3 : KS == 6 ? 2 : 1) : QT == 2 ? 2 : KS <= 2 ? 4 : KS == 4 ? 3 : 2; }
template <int NP, int KS, int QT> constexpr int dq_per_cu() { return NP == 3 ? (KS <= 2 ? 3 : KS == 4 ? 2 : 1) : QT == 2 ? 2 : KS <= 2 ? 4 : KS == 4 ? 3 : 2; }
template <int NP, int KS> constexpr int dkv_per_cu() { return NP == 3 ? (KS == 1 ? 4 : KS == 2 ? 3 : 1) : KS == 4 ? 3 : 2; }
// query tiles per wave: two read every key fragment once for both (heads of 64: 371 us against 386 in the forward pass of 2 x 16 heads x 4096 x 8192), but
// hold the registers of two, which the smaller heads use better for more waves (heads of 32, 2 x 2 x 20480 x 20480: 430 us against 406)
template <int NP, int KS> constexpr int query_tiles() { return NP == 1 && KS == 4 ? 2 : 1; }
// key tiles per wave of the dk / dv kernel: two halve the fragments read from shared memory, which are what bounds it for small heads (heads of 32: 652 us
// against 602); from 64 on the accumulators of two do not fit
template <int NP, int KS> constexpr int key_tiles() { return NP == 1 && KS <= 2 ? 2 : 1; }

// keys per step of the forward kernel: as many as shared memory has room for beside the other workgroups (two buffers each) -- a step is a barrier, and of its
// parts of 32 keys all but the first have their products under way when their turn comes.  The backward kernels take 32 a step: they need the registers
// that this costs for more waves (dq, heads of 32: 451 us at 4 waves per SIMD, 485 at 2 with the products ahead)
constexpr int DQ_KEYS = 32;
template <int NP, int KS> constexpr int fwd_keys() { return NP == 3 ? (KS <= 2 ? 64 : 32) : KS <= 2 ? 128 : 64; }

// ---------------------------------------------------------------- what the kernels are told
struct Shape {
    int B, Hk, G, Nq, N, M, Hq, d;
    const int *idx, *cnt;          // valid keys of each sequence and their number, or null
};
__device__ __forceinline__ int keys_of(const Shape &s, int z) { return s.cnt ? s.cnt[z / s.Hk] : s.N; }
__device__ __forceinline__ long long q_row(const Shape &s, int z, int r) {      // row r of z in (B, Nq, Hq)
    const int b = z / s.Hk, g = r / s.Nq;
    return ((long long)b * s.Nq + (r - g * s.Nq)) * s.Hq + (z - b * s.Hk) * s.G + g;
}
__device__ __forceinline__ long long k_row(const Shape &s, int z, int i) {      // i-th valid key of z in (B, N, Hk)
    const int b = z / s.Hk;
    return ((long long)b * s.N + (s.idx ? s.idx[(long long)b * s.N + i] : i)) * s.Hk + (z - b * s.Hk);
}

// ---------------------------------------------------------------- the valid keys of each sequence, in order
__global__ __launch_bounds__(1024) void xa_compact_kernel(const unsigned char *__restrict__ mask, long long sb, int N, int *__restrict__ idx,
                                                          int *__restrict__ cnt) {
    __shared__ int wave_sum[16];
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    mask += blockIdx.x * sb;
    idx += (long long)blockIdx.x * N;
    const bool aligned = ((uintptr_t)mask & 15) == 0;
    int base = 0;
    for (long long at = 0; at < N; at += 16384) {
        const long long first = at + t * 16;
        unsigned bits = 0;
        if (aligned && first + 16 <= N) {
            const uint4 w = *(const uint4 *)(mask + first);
            const unsigned word[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
            for (int j = 0; j < 16; ++j) bits |= ((word[j / 4] >> (8 * (j % 4))) & 0xFF ? 1u : 0u) << j;
        } else {
            for (int j = 0; j < 16; ++j)
                if (first + j < N && mask[first + j]) bits |= 1u << j;
        }
        const int mine = __popc(bits);
        int upto = mine;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int v = __shfl_up(upto, o);
            if (lane >= o) upto += v;
        }
        if (lane == 63) wave_sum[wave] = upto;
        __syncthreads();
        int before = 0, all = 0;
#pragma unroll
        for (int w = 0; w < 16; ++w) {
            before += w < wave ? wave_sum[w] : 0;
            all += wave_sum[w];
        }
        int to = base + before + upto - mine;
        for (; bits; bits &= bits - 1) idx[to++] = (int)(first + __ffs(bits) - 1);
        base += all;
        __syncthreads();
    }
    if (t == 0) cnt[blockIdx.x] = base;
}

// ---------------------------------------------------------------- operands into fragment order
// A wave per tile of 32 rows; bound by memory: 2 x 16 heads of 64, 4096 queries and 8192 keys, bf16, takes 56 us on average
// of the forward call's launch (168 MB) and the backward call's (285 MB)
struct PackJob {
    const void *x;
    long long sb, sn, sh;
    char *R, *T;                 // where to, either may be null
    int tiles;                   // of 32 rows, per z; behind the last key are zeros, behind the last query row copies of it
    int query;                   // rows are query rows (else valid keys)
    int vec;                     // 16-byte loads: d and all strides are multiples of 8 elements, x is aligned
    float factor;
    float *norm;                 // no less than the largest |row| (after `factor`) of each tile, or null
};
struct PackArgs {
    PackJob job[4];
    int blocks[5];               // jobs' first workgroups; behind the last job: rows of masked keys to be zeroed in dk, dv
    int jobs, first;             // first: of this launch's workgroups
    Shape s;
    const void *o;               // with `stat`: of job 0 (the gradient g) also -lse, -D = -g . o and (with a norm) |row|, per tile 3 x 32 floats in 1 KB
    const float *lse;
    char *stat;
    const unsigned char *mask;
    long long mask_sb;
    void *dk, *dv;
};

constexpr float LOST_SQUARES = 0x1p-110f;     // more than 128 squares that fall below float32's normal range can add up to

template <class T, int KS>
__global__ __launch_bounds__(64) void xa_pack_kernel(PackArgs a) {
    using E = typename Frag<T>::E;
    constexpr int NP = Frag<T>::NP, DP = 16 * KS, LD = DP + 16 / sizeof(T), DB = (KS + 1) / 2;
    __shared__ __attribute__((aligned(16))) T rows[32 * LD];
    const int lane = threadIdx.x, col = lane & 31, half = lane >> 5;
    const Shape &s = a.s;
    const int block = a.first + (int)blockIdx.x;
    int j = 0;
    while (j < a.jobs && block >= a.blocks[j + 1]) ++j;
    const int local = block - a.blocks[j];
    if (j == a.jobs) {           // 32 rows of one sequence's dk, dv
        const int per = (s.N + 31) / 32, b = local / per, n0 = (local % per) * 32;
        const int len = s.Hk * s.d;
        for (int n = n0; n < n0 + 32 && n < s.N; ++n)
            if (!a.mask[b * a.mask_sb + n])
                for (int i = lane; i < len; i += 64) {
                    ((T *)a.dk)[((long long)b * s.N + n) * len + i] = (T)0.f;
                    ((T *)a.dv)[((long long)b * s.N + n) * len + i] = (T)0.f;
                }
        return;
    }
    const PackJob &job = a.job[j];
    const int z = local / job.tiles, tile = local % job.tiles, b = z / s.Hk, hk = z - b * s.Hk;
    const int count = job.query ? s.M : keys_of(s, z);
#pragma unroll
    for (int c = 0; c < KS; ++c) {
        // a copy of the last query row, its weights 0 by its `lse`, gives keys what that row gives them: a row of zeros would make NaN of an infinite key
        const int chunk = c * 64 + lane, r = chunk / (2 * KS), off = chunk % (2 * KS) * 8, i = job.query ? min(tile * 32 + r, count - 1) : tile * 32 + r;
        T v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = (T)0.f;
        if (i < count) {
            const T *x = (const T *)job.x;
            if (job.query) {
                const int g = i / s.Nq;
                x += b * job.sb + (i - g * s.Nq) * job.sn + (hk * s.G + g) * job.sh;
            } else
                x += b * job.sb + (s.idx ? s.idx[(long long)b * s.N + i] : i) * job.sn + hk * job.sh;
            if (job.vec) {
                if (off < s.d)
#pragma unroll
                    for (int w = 0; w < (int)sizeof(T) / 2; ++w) ((uint4 *)v)[w] = ((const uint4 *)(x + off))[w];
            } else {
                for (int e = 0; e < 8; ++e)
                    if (off + e < s.d) v[e] = x[off + e];
            }
        }
#pragma unroll
        for (int w = 0; w < (int)sizeof(T) / 2; ++w) ((uint4 *)(rows + r * LD + off))[w] = ((uint4 *)v)[w];
    }
    __syncthreads();
    const long long at = (long long)z * job.tiles + tile;
    if (job.R)
#pragma unroll
        for (int k = 0; k < KS; ++k) {
            float v[8];
            typename Vec<E>::v8 p[NP];
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = (float)rows[col * LD + 16 * k + 8 * half + e] * job.factor;
            split8<E, NP>(v, p);
#pragma unroll
            for (int n = 0; n < NP; ++n) *(typename Vec<E>::v8 *)(job.R + ((at * KS + k) * NP + n) * 1024 + lane * 16) = p[n];
        }
    if (job.T)
#pragma unroll
        for (int f = 0; f < 2 * DB; ++f) {
            const int dim = 32 * (f / 2) + col;
            float v[8];
            typename Vec<E>::v8 p[NP];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int r = 16 * (f % 2) + 8 * (e / 4) + 4 * half + e % 4;
                v[e] = dim < DP ? (float)rows[r * LD + (dim < DP ? dim : 0)] * job.factor : 0.f;
            }
            split8<E, NP>(v, p);
#pragma unroll
            for (int n = 0; n < NP; ++n) *(typename Vec<E>::v8 *)(job.T + ((at * 2 * DB + f) * NP + n) * 1024 + lane * 16) = p[n];
        }
    if (j == 0 && a.stat) {
        const int i = tile * 32 + col;
        float D = 0.f;
        if (i < s.M) {
            const T *o = (const T *)a.o + q_row(s, z, i) * s.d;
            for (int e = half * 8 * KS; e < (half + 1) * 8 * KS && e < s.d; ++e) D = fmaf((float)rows[col * LD + e], (float)o[e], D);
        }
        D = swap_halves_sum(D);
        float *st = (float *)(a.stat + at * 1024);
        if (half == 0) st[col] = i < s.M ? -a.lse[(long long)z * s.M + i] : -INFINITY;
        else st[32 + col] = -D;
    }
    if (job.norm) {
        // NaN elements do not count: what they meet is NaN whatever the bound
        float q = 0.f;
        for (int e = half * 8 * KS; e < (half + 1) * 8 * KS; ++e) {
            const float x = (float)rows[col * LD + e], more = fmaf(x, x, q);
            q = more == more ? more : q;
        }
        q = sqrtf(swap_halves_sum(q) + LOST_SQUARES) * fabsf(job.factor);
        if (j == 0 && a.stat && half == 0) ((float *)(a.stat + at * 1024))[64 + col] = q;
        q = md_wave_max(q);
        if (lane == 0) job.norm[at] = q;
    }
}

// ---------------------------------------------------------------- accumulators to memory
// A lane holds 4 neighbouring dims of its row in each 4 registers: one 8- or 16-byte store where the rows allow it.
template <class T, int DB> __device__ __forceinline__ void store_row(T *row, int d, int half, const f32x16 (&x)[DB], float f) {
#pragma unroll
    for (int b = 0; b < DB; ++b)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const int dim = 32 * b + 8 * g + 4 * half;
            T v[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = (T)(x[b][4 * g + e] * f);
            if (d % 4 == 0) {
                if (dim < d) __builtin_memcpy(__builtin_assume_aligned(row + dim, 4 * sizeof(T)), v, 4 * sizeof(T));
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (dim + e < d) row[dim + e] = v[e];
            }
        }
}
// a part of 32 rows, as it stands in the registers: [b][g][lane][4 floats], 1 KB each
using f32x4 = float __attribute__((ext_vector_type(4)));
template <int DB> __device__ __forceinline__ void store_part(float *to, int lane, const f32x16 (&x)[DB], float f) {
#pragma unroll
    for (int b = 0; b < DB; ++b)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            f32x4 v;
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = x[b][4 * g + e] * f;
            *(f32x4 *)(to + ((b * 4 + g) * 64 + lane) * 4) = v;
        }
}
template <int DB> __device__ __forceinline__ void add_part(const float *from, int lane, f32x16 (&x)[DB], float f) {
#pragma unroll
    for (int b = 0; b < DB; ++b)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const f32x4 v = *(const f32x4 *)(from + ((b * 4 + g) * 64 + lane) * 4);
#pragma unroll
            for (int e = 0; e < 4; ++e) x[b][4 * g + e] = fmaf(f, v[e], x[b][4 * g + e]);
        }
}

// ---------------------------------------------------------------- the tile kernels' share of the work
// The work of a launch is a line of units: blocks of rows (`rows` query rows, or keys in the dk / dv kernel) of each z, one behind the other, and of each
// block the steps over the other axis.  Every worker (workgroup) takes an equal stretch of it, so the chip is filled evenly whatever the
// sizes.  A block that lies within one stretch is written at once; of the others each worker leaves its part in a slot (at most two: its
// first block and its last) and xa_join / xa_sum put the parts together in the order of the line: the same bits every time.
struct TileArgs {
    Shape s;
    const char *Qr, *Kr, *Vt;                          // forward
    const float *qn, *kn, *vn, *gn;                    // largest row norm of each tile of 32
    const char *Qt, *Kt, *Vr, *Gr, *Gt, *stat;         // backward
    int q_tiles, k_tiles, workers, rows, step;          // `step`: keys per step; 0: blocks are of keys, a step is a tile of 32 queries
    long long units;                                    // all of them; with a mask the device counts
    float c, scale, down;                               // 2^-down times the weights of all keys is 1 at the most (P is up to 2^LAZY)
    void *o, *dq, *dk, *dv;
    int4 *first;                                         // each worker's first piece: z (-1: idle), block, step -- for who joins the parts
    float *lse, *part, *part2, *ml;                      // parts: [slot][tile of the block][store_part], [slot][row of the block][2]
};

struct Line {                                          // of one sequence: blocks of a z, steps of a block
    int blocks, steps;
    __device__ long long units(int Hk) const { return (long long)Hk * blocks * steps; }
};
__device__ __forceinline__ Line line_of(const TileArgs &a, int b) {
    const int n = a.s.cnt ? a.s.cnt[b] : a.s.N;
    Line l;
    l.blocks = ((a.step ? a.s.M : n) + a.rows - 1) / a.rows;
    l.steps = max(1, a.step ? (n + a.step - 1) / a.step : a.q_tiles);     // (a block without steps is still written)
    return l;
}
__device__ __forceinline__ long long uniform(long long v) {
    return (long long)((unsigned long long)(unsigned)__builtin_amdgcn_readfirstlane((int)(v >> 32)) << 32 | (unsigned)__builtin_amdgcn_readfirstlane((int)v));
}
// all units, and those ahead of sequence `b`; every lane of a wave calls it
__device__ __forceinline__ long long units_before(const TileArgs &a, int b, long long &all) {
    if (!a.s.cnt) {
        all = a.units;
        return line_of(a, 0).units(a.s.Hk) * b;
    }
    const int lane = threadIdx.x & 63;
    long long before = 0, sum = 0;
    for (int b0 = 0; b0 < a.s.B; b0 += 64) {
        const long long mine = b0 + lane < a.s.B ? line_of(a, b0 + lane).units(a.s.Hk) : 0;
        long long x = mine, y = b0 + lane < b ? mine : 0;
#pragma unroll
        for (int o = 32; o; o >>= 1) {
            x += __shfl_xor(x, o);
            y += __shfl_xor(y, o);
        }
        sum += x;
        before += y;
    }
    all = uniform(sum);
    return uniform(before);
}
// a / b of non-negative numbers, in 32 bits where they fit (64-bit division is ~100 instructions)
__device__ __forceinline__ long long quotient(long long a, long long b) {
    return ((a | b) >> 32) == 0 ? (long long)((unsigned)a / (unsigned)b) : a / b;
}
__device__ __forceinline__ long long stretch_start(long long all, int worker, int workers) {     // all * worker / workers
    const long long q = quotient(all, workers);
    return q * worker + quotient((all - q * workers) * worker, workers);
}

struct Piece { int z, block, first, last, slot; bool whole; };
struct Walk {
    long long left;
    int b, hk, block, first, slot, part;
    Line line;
    __device__ __forceinline__ Walk(const TileArgs &a, int worker) {
        long long all;
        units_before(a, 0, all);
        const int workers = (int)min((long long)a.workers, all);      // (a mask may leave fewer units than workers: the others are idle)
        long long at = 0;
        left = 0;
        if (worker < workers) {
            at = stretch_start(all, worker, workers);
            left = stretch_start(all, worker + 1, workers) - at;
        }
        b = hk = block = first = 0;
        line = {};
        if (left > 0) {
            if (!a.s.cnt) {
                line = line_of(a, 0);
                const long long per = line.units(a.s.Hk);
                b = (int)quotient(at, per);
                at -= per * b;
            } else {
                const int lane = threadIdx.x & 63;         // 64 sequences at a time
                for (;; b += 64) {
                    long long upto = b + lane < a.s.B ? line_of(a, b + lane).units(a.s.Hk) : 0;
#pragma unroll
                    for (int o = 1; o < 64; o <<= 1) {
                        const long long v = __shfl_up(upto, o);
                        if (lane >= o) upto += v;
                    }
                    const unsigned long long behind = __ballot(upto > at);
                    if (behind) {
                        const int i = __ffsll(behind) - 1;
                        if (i > 0) at -= __shfl(upto, i - 1);
                        b += i;
                        break;
                    }
                    at -= __shfl(upto, 63);
                }
                at = uniform(at);
                b = __builtin_amdgcn_readfirstlane(b);
                line = line_of(a, b);
            }
            const long long per = (long long)line.blocks * line.steps;
            hk = (int)quotient(at, per);
            at -= hk * per;
            block = (int)quotient(at, line.steps);
            first = (int)(at - (long long)block * line.steps);
        }
        // the same in every lane: scalar registers
        left = uniform(left);
        b = __builtin_amdgcn_readfirstlane(b), hk = __builtin_amdgcn_readfirstlane(hk), block = __builtin_amdgcn_readfirstlane(block);
        first = __builtin_amdgcn_readfirstlane(first);
        line.blocks = __builtin_amdgcn_readfirstlane(line.blocks), line.steps = __builtin_amdgcn_readfirstlane(line.steps);
        slot = 2 * worker;
        part = 0;
        if (a.first && threadIdx.x == 0) a.first[worker] = make_int4(left > 0 ? b * a.s.Hk + hk : -1, block, first, 0);
    }
    __device__ __forceinline__ bool next(const TileArgs &a, Piece &p) {
        if (left <= 0) return false;
        p.z = b * a.s.Hk + hk, p.block = block, p.first = first;
        p.last = (int)min((long long)line.steps, first + left);
        p.whole = p.last - p.first == line.steps;
        p.slot = slot + (part ? 1 : 0);
        part = 1;
        left -= p.last - p.first;
        first = 0;
        if (++block == line.blocks) {
            block = 0;
            if (++hk == a.s.Hk) {
                hk = 0;
                if (left > 0)
                    do line = line_of(a, ++b);
                    while (!line.blocks);
            }
        }
        return true;
    }
};

template <class E> struct Shift { static constexpr float fwd = 0.f, bwd = 0.f; };
template <> struct Shift<f16_t> { static constexpr float fwd = 7.f, bwd = 15.f; };

// largest of the norms of tiles `from` .. `to` - 1 (a NaN, of an infinite row times a factor of 0, stays): every lane of a wave calls it
__device__ __forceinline__ float row_norm(const float *norm, int from, int to) {
    float x = 0.f;
    bool nan = false;
    for (int i = from + (threadIdx.x & 63); i < to; i += 64) {
        x = fmaxf(x, norm[i]);
        nan |= norm[i] != norm[i];
    }
    return __any(nan) ? NAN : __int_as_float(__builtin_amdgcn_readfirstlane(__float_as_int(md_wave_max(x))));
}

// ---------------------------------------------------------------- forward: 32 QT queries per wave, NW waves, steps of TK keys
// Where |q| |k| scale of a piece's rows bounds its scores by 48 either way, and |v| is below 2^40, m is 0 throughout: no maximum, no rescaling, and the step is
// straight-line code in which the products of one half run beside the exponentials of the other.  P stays within 2^+-48 then, and O's sums within 2^88 times the
// row length (bf16 has float32's exponents; float16 has not and always takes the running maximum).  Beside a running maximum values above 2^80 take P
// times a smaller power of two, so that sums of values near the range's end stay in it.
// 2 x 2 x 20480^2 heads of 32, bf16: 351 us (with the running maximum 425), 0.61 PFLOP/s: 20 cycles of vector and 8 of matrix instructions per 64 pairs and
// SIMD, 25 to 28 in all at the 2.0 GHz the clock falls to.  2 x 16 x 4096 x 8192 heads of 64: 330 us, 0.83 PFLOP/s
template <class T, int KS, int QT, int TK, int NW>
__global__ __launch_bounds__(64 * NW, (NW == 4 ? fwd_per_cu<Frag<T>::NP, KS, QT>() : 1)) void xa_fwd_kernel(TileArgs a) {
    using E = typename Frag<T>::E;
    using v8 = typename Vec<E>::v8;
    constexpr int NP = Frag<T>::NP, DB = (KS + 1) / 2, SUB = TK / 32;
    constexpr int KC = SUB * KS * NP, VC = SUB * DB * 2 * NP;       // 1 KB chunks per step
    __shared__ __attribute__((aligned(1024))) char lds[2][(KC + VC) * 1024];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = lane & 31, half = lane >> 5;
    const int worker = die_order(blockIdx.x, gridDim.x);
    if (worker >= a.workers) return;
    Piece w;
    for (Walk walk(a, worker); walk.next(a, w);) {
        const int z = w.z, n = keys_of(a.s, z), last = min(w.last, (n + TK - 1) / TK);
        const int q0 = (w.block * NW + wave) * QT;          // this wave's first query tile

        v8 q[QT][KS][NP];
        f32x16 o[QT][DB];
        float m[QT], l[QT];
#pragma unroll
        for (int t = 0; t < QT; ++t) {
            const int tile = q0 + t < a.q_tiles ? q0 + t : a.q_tiles - 1;
#pragma unroll
            for (int k = 0; k < KS; ++k) read_frag<E, NP>(a.Qr + (((long long)z * a.q_tiles + tile) * KS + k) * NP * 1024, lane, q[t][k]);
#pragma unroll
            for (int b = 0; b < DB; ++b) o[t][b] = (f32x16)0.f;
            m[t] = LOWEST;
            l[t] = 0.f;
        }
        const float c = NP == 3 ? 1.f : a.c;               // (float32: in q's fragments)
        constexpr float BOUND = Shift<E>::fwd == 0.f ? 48.f : 0.f, V_BOUND = 0x1p40f, V_LARGE = 0x1p80f;
        float shift = -Shift<E>::fwd;                      // P is held times 2^-shift
        const char *Kz = a.Kr + (long long)z * a.k_tiles * KS * NP * 1024, *Vz = a.Vt + (long long)z * a.k_tiles * DB * 2 * NP * 1024;
        auto fetch = [&](int step) {
            char *to = lds[step & 1];
            for (int i = wave; i < KC + VC; i += NW)
                load_chunk(i < KC ? Kz + ((long long)step * KC + i) * 1024 : Vz + ((long long)step * VC + i - KC) * 1024, to + i * 1024, lane);
        };
        // BOUNDED: no score of this piece can pass BOUND either way, m stays 0.  TAIL: rows behind the last key
        auto run = [&](auto bounded, auto tail, int step) {
            constexpr bool BOUNDED = decltype(bounded)::value, TAIL = decltype(tail)::value;
            wait_loads_and_barrier();
            if (step + 1 < last) fetch(step + 1);
            const char *K = lds[step & 1], *V = K + KC * 1024;
            f32x16 s[2][QT];
            auto scores = [&](int u, f32x16 (&to)[QT]) {
#pragma unroll
                for (int t = 0; t < QT; ++t) to[t] = (f32x16)0.f;
#pragma unroll
                for (int k = 0; k < KS; ++k) {
                    v8 f[NP];
                    read_frag<E, NP>(K + (u * KS + k) * NP * 1024, lane, f);
#pragma unroll
                    for (int t = 0; t < QT; ++t) to[t] = mfma_pieces<E, NP>(f, q[t][k], to[t]);
                }
            };
            scores(0, s[0]);
#pragma unroll
            for (int u = 0; u < SUB; ++u) {
                f32x16 (&x)[QT] = s[u & 1];
                if constexpr (TAIL)
#pragma unroll
                    for (int r = 0; r < 16; ++r)
                        if (step * TK + u * 32 + 8 * (r / 4) + 4 * half + r % 4 >= n)
#pragma unroll
                            for (int t = 0; t < QT; ++t) x[t][r] = -INFINITY;
                if constexpr (!BOUNDED)
#pragma unroll
                    for (int t = 0; t < QT; ++t) {
                        float top = x[t][0];
#pragma unroll
                        for (int r = 1; r < 16; ++r) top = fmaxf(top, x[t][r]);
                        top = swap_halves_max(top) * c;
                        if (__any(top > m[t] + LAZY)) {
                            const float up = fmaxf(m[t], top), f = __builtin_amdgcn_exp2f(m[t] - up);
                            m[t] = up;
                            l[t] *= f;
#pragma unroll
                            for (int b = 0; b < DB; ++b) o[t][b] *= f;
                        }
                    }
                // the next half's products and this one's fragments are under way while the exponentials run
                constexpr bool EARLY = DB * NP <= 4;           // (registers)
                v8 vf[2][DB][NP];
                if constexpr (EARLY)
#pragma unroll
                    for (int h = 0; h < 2; ++h)
#pragma unroll
                        for (int b = 0; b < DB; ++b) read_frag<E, NP>(V + ((u * DB + b) * 2 + h) * NP * 1024, lane, vf[h][b]);
                if (u + 1 < SUB) scores(u + 1, s[(u + 1) & 1]);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    v8 f[QT][NP];
#pragma unroll
                    for (int t = 0; t < QT; ++t) {
                        float p[8];
                        const float base = m[t] + shift;
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            const float y = x[t][8 * h + e];
                            p[e] = __builtin_amdgcn_exp2f(BOUNDED ? (NP == 3 ? y : y * c) : fmaf(y, c, -base));
                            l[t] += p[e];
                        }
                        split8<E, NP>(p, f[t]);
                    }
#pragma unroll
                    for (int b = 0; b < DB; ++b) {
                        if constexpr (!EARLY) read_frag<E, NP>(V + ((u * DB + b) * 2 + h) * NP * 1024, lane, vf[h][b]);
#pragma unroll
                        for (int t = 0; t < QT; ++t) o[t][b] = mfma_pieces<E, NP>(vf[h][b], f[t], o[t][b]);
                    }
                }
            }
        };
        const std::true_type yes;
        const std::false_type no;
        __syncthreads();                                   // the last piece's tiles have been read
        if (w.first < last) fetch(w.first);
        const int whole = min(last, n / TK);               // steps without rows behind the last key
        int step = w.first;
        const float v_norm = BOUND > 0.f ? row_norm(a.vn + (long long)z * a.k_tiles, w.first * SUB, last * SUB) : 0.f;
        if (BOUND > 0.f && row_norm(a.qn + (long long)z * a.q_tiles, w.block * NW * QT, min((w.block + 1) * NW * QT, a.q_tiles)) *
                                   row_norm(a.kn + (long long)z * a.k_tiles, w.first * SUB, last * SUB) * c <= BOUND && v_norm <= V_BOUND) {
#pragma unroll
            for (int t = 0; t < QT; ++t) m[t] = 0.f;
            for (; step < whole; ++step) run(yes, no, step);
            if (step < last) run(yes, yes, step);
        } else {
            if (BOUND > 0.f && v_norm > V_LARGE) shift = a.down;     // sums of large values stay in range
            for (; step < whole; ++step) run(no, no, step);
            if (step < last) run(no, yes, step);
        }
#pragma unroll
        for (int t = 0; t < QT; ++t) {
            const int row = (q0 + t) * 32 + col;
            const float sum = swap_halves_sum(l[t]), base = m[t] + shift;
            if (!w.whole) {
                const long long tile = (long long)w.slot * (NW * QT) + wave * QT + t;
                if (half == 0) {
                    a.ml[2 * (tile * 32 + col)] = base;
                    a.ml[2 * (tile * 32 + col) + 1] = sum;
                }
                store_part<DB>(a.part + tile * DB * 1024, lane, o[t], 1.f);
            } else if (row < a.s.M) {
                const float inv = sum > 0.f ? 1.f / sum : (sum == 0.f ? 0.f : sum);     // (NaN stays NaN)
                if (half == 0 && a.lse) a.lse[(long long)z * a.s.M + row] = sum == 0.f ? INFINITY : base + __log2f(sum);
                store_row<T, DB>((T *)a.o + q_row(a.s, z, row) * a.s.d, a.s.d, half, o[t], inv);
            }
        }
    }
}

// The block that the start of stretch `worker` falls into, and who has parts of it: workers `from` .. `to` - 1, from what each worker noted of its first piece.
// Found once, by the first worker that starts inside the block: for the others find() is false.
struct Joint {
    int z, block, from, to;
    bool tail;                   // `from` has a piece ahead of this one: its part is in its second slot
    __device__ __forceinline__ bool find(const TileArgs &a, int worker) {
        const int4 me = a.first[worker];
        if (worker == 0 || me.x < 0 || me.z == 0) return false;        // idle, or it starts with a block of its own
        const int4 last = a.first[worker - 1];
        const bool same = last.x == me.x && last.y == me.y;
        if (same && last.z > 0) return false;
        z = me.x, block = me.y, from = worker - 1, tail = !same;
        for (to = worker + 1; to < a.workers; to += 64) {              // 64 notes at a time; every lane calls this
            const int i = to + (threadIdx.x & 63);
            const int4 next = a.first[i < a.workers ? i : worker];
            const unsigned long long other = __ballot(i >= a.workers || next.x != z || next.y != block || next.z == 0);
            if (other) {
                to += __ffsll(other) - 1;
                break;
            }
        }
        to = min(to, a.workers);
        return true;
    }
    __device__ __forceinline__ int slot(int i) const { return 2 * i + (tail && i == from ? 1 : 0); }
};

// The four waves of a workgroup add up one tile's parts, each every fourth of them, in their order; then wave g holds registers 4 g .. 4 g + 3 of each b.
template <int DB> __device__ __forceinline__ void sum_waves(float *shared, int wave, int lane, const f32x16 (&x)[DB], const float (&f)[4], f32x4 (&out)[DB]) {
#pragma unroll
    for (int b = 0; b < DB; ++b) {
        __syncthreads();
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            f32x4 v;
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = x[b][4 * g + e];
            *(f32x4 *)(shared + ((wave * 4 + g) * 64 + lane) * 4) = v;
        }
        __syncthreads();
        out[b] = (f32x4)0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) out[b] += *(const f32x4 *)(shared + ((i * 4 + wave) * 64 + lane) * 4) * f[i];
    }
}
template <class T, int DB> __device__ __forceinline__ void store_quarter(T *row, int d, int half, int g, const f32x4 (&x)[DB], float f) {
#pragma unroll
    for (int b = 0; b < DB; ++b) {
        const int dim = 32 * b + 8 * g + 4 * half;
        T v[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = (T)(x[b][e] * f);
        if (d % 4 == 0) {
            if (dim < d) __builtin_memcpy(__builtin_assume_aligned(row + dim, 4 * sizeof(T)), v, 4 * sizeof(T));
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (dim + e < d) row[dim + e] = v[e];
        }
    }
}

// O = sum 2^(m_i - m) O_i / sum 2^(m_i - m) l_i, m = max m_i; a workgroup per tile of 32 rows
template <class T, int DB>
__global__ __launch_bounds__(256) void xa_join_kernel(TileArgs a) {
    __shared__ float shared[4096], sm[4][2][32];
    Joint j;
    if (!j.find(a, blockIdx.x)) return;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = lane & 31, half = lane >> 5;
    const int tiles = a.rows / 32, row = j.block * a.rows + blockIdx.y * 32 + col;
    f32x16 o[DB];
#pragma unroll
    for (int b = 0; b < DB; ++b) o[b] = (f32x16)0.f;
    float m = -INFINITY, sum = 0.f;
    for (int i = j.from + wave; i < j.to; i += 4) {
        const long long tile = (long long)j.slot(i) * tiles + blockIdx.y;
        const float mi = a.ml[2 * (tile * 32 + col)], li = a.ml[2 * (tile * 32 + col) + 1];
        const float up = fmaxf(m, mi), f = m == -INFINITY ? 0.f : exp2f(m - up), fi = li == 0.f ? 0.f : exp2f(mi - up);     // (0: no keys there)
        m = up;
        sum = sum * f + li * fi;
        if (__any(f != 1.f))
#pragma unroll
            for (int b = 0; b < DB; ++b) o[b] *= f;
        add_part<DB>(a.part + tile * DB * 1024, lane, o, fi);
    }
    if (half == 0) sm[wave][0][col] = m, sm[wave][1][col] = sum;
    __syncthreads();
    float f[4], top = -INFINITY, total = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) top = fmaxf(top, sm[i][0][col]);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        f[i] = sm[i][1][col] == 0.f ? 0.f : exp2f(sm[i][0][col] - top);
        total = fmaf(f[i], sm[i][1][col], total);
    }
    f32x4 out[DB];
    sum_waves<DB>(shared, wave, lane, o, f, out);
    if (row >= a.s.M) return;
    store_quarter<T, DB>((T *)a.o + q_row(a.s, j.z, row) * a.s.d, a.s.d, half, wave, out, total == 0.f ? 0.f : 1.f / total);
    if (threadIdx.x < 32 && a.lse) a.lse[(long long)j.z * a.s.M + row] = total == 0.f ? INFINITY : top + log2f(total);
}

// dq, or dk and dv: the parts' sums
template <class T, int DB>
__global__ __launch_bounds__(256) void xa_sum_kernel(TileArgs a) {
    __shared__ float shared[4096];
    Joint j;
    if (!j.find(a, blockIdx.x)) return;
    const bool keys = a.step == 0;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = lane & 31, half = lane >> 5;
    const int tiles = a.rows / 32, row = j.block * a.rows + blockIdx.y * 32 + col;
    const bool live = row < (keys ? keys_of(a.s, j.z) : a.s.M);
    const long long to = live ? (keys ? k_row(a.s, j.z, row) : q_row(a.s, j.z, row)) * a.s.d : 0;
    const float one[4] = {1.f, 1.f, 1.f, 1.f};
    for (int which = 0; which < (keys ? 2 : 1); ++which) {
        f32x16 x[DB];
#pragma unroll
        for (int b = 0; b < DB; ++b) x[b] = (f32x16)0.f;
        for (int i = j.from + wave; i < j.to; i += 4)
            add_part<DB>((which ? a.part2 : a.part) + ((long long)j.slot(i) * tiles + blockIdx.y) * DB * 1024, lane, x, 1.f);
        f32x4 out[DB];
        sum_waves<DB>(shared, wave, lane, x, one, out);
        if (live) store_quarter<T, DB>((T *)(which ? a.dv : keys ? a.dk : a.dq) + to, a.s.d, half, wave, out, 1.f);
    }
}

// the splits of a few rows (xa_few): [split][z][row][d]
struct FewArgs {
    Shape s;
    const void *q, *k, *v;
    long long q_sb, q_sn, q_sh, k_sb, k_sn, k_sh, v_sb, v_sn, v_sh, mask_sb;
    const unsigned char *mask;
    int splits;
    float c, down, up;           // O is summed times `down`, a power of two that keeps sums of large values in range, and taken back by `up`
    void *o;
    float *lse, *part, *ml;
};
template <class T>
__global__ __launch_bounds__(64) void xa_few_join_kernel(FewArgs a) {
    const int lane = threadIdx.x, z = blockIdx.x / a.s.M, row = blockIdx.x % a.s.M;
    const long long rows = (long long)a.s.B * a.s.Hk * a.s.M, at = blockIdx.x;
    // a lane holds one split's m and l (there are at most 64), then the weights go round
    const bool on = lane < a.splits;
    const float mi = on ? a.ml[2 * (lane * rows + at)] : -INFINITY, li = on ? a.ml[2 * (lane * rows + at) + 1] : 0.f;
    const float m = md_wave_max(mi), f = li == 0.f ? 0.f : exp2f(mi - m);
    const float sum = md_wave_sum(f * li);
    float o0 = 0.f, o1 = 0.f;
    constexpr int U = 8;           // parts in flight
    for (int i0 = 0; i0 < a.splits; i0 += U) {
        float x0[U], x1[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = i0 + u < a.splits ? i0 + u : i0;
            const float *p = a.part + (i * rows + at) * a.s.d;
            x0[u] = lane < a.s.d ? p[lane] : 0.f;
            x1[u] = lane + 64 < a.s.d ? p[lane + 64] : 0.f;
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const float fi = i0 + u < a.splits ? __shfl(f, i0 + u) : 0.f;
            if (fi != 0.f) o0 = fmaf(fi, x0[u], o0), o1 = fmaf(fi, x1[u], o1);
        }
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    T *to = (T *)a.o + q_row(a.s, z, row) * a.s.d;
    if (lane < a.s.d) to[lane] = (T)(o0 * inv * a.up);
    if (lane + 64 < a.s.d) to[lane + 64] = (T)(o1 * inv * a.up);
    if (lane == 0 && a.lse) a.lse[at] = sum == 0.f ? INFINITY : m + log2f(sum);
}

// ---------------------------------------------------------------- backward
// float16: dS times 2^k, |dS| 2^k < 2^15: |dS| <= |g v - D| <= 2 |g| |v|, with the largest |v| of the z's keys and the |g| of the query (dq, where a lane owns
// one) or the largest of the piece's queries (dk and dv, whose sums run over them).  So a query's dq, and a sequence's dk and dv, are as exact beside gradients
// of any other size: with one k for the call, rows 2^-20 of the largest came out 2 % off.
template <class E> __device__ __forceinline__ float ds_scale(float g, float v) {
    if constexpr (Shift<E>::bwd == 0.f) return 1.f;
    const float most = 2.f * g * v;
    if (!(most > 0.f) || most > 1e30f) return 1.f;
    int k = 14 - ((int)(__float_as_uint(most) >> 23) - 127);           // 2^(14 - k) <= most < 2^(15 - k)
    k = k < -60 ? -60 : k > 60 ? 60 : k;
    return __uint_as_float((unsigned)(127 + k) << 23);
}

// dq: 32 QT queries per wave, steps of 32 keys.  S and g V^T again, dS from both, dQ^T += K^T dS.  -D is what the accumulators of g V^T start from.
// 2 x 2 x 20480^2 heads of 32, bf16: 458 us (64 % of the vector pipe's and 36 % of the matrix pipe's cycles; a matrix instruction
// takes about half of its own from the vector pipe);
// 2 x 16 x 4096 x 8192 heads of 64: 468 us, 0.88 PFLOP/s
template <class T, int KS, int QT, int NW>
__global__ __launch_bounds__(64 * NW, (NW == 4 ? dq_per_cu<Frag<T>::NP, KS, QT>() : 1)) void xa_dq_kernel(TileArgs a) {
    using E = typename Frag<T>::E;
    using v8 = typename Vec<E>::v8;
    constexpr int NP = Frag<T>::NP, DB = (KS + 1) / 2, TK = DQ_KEYS, RC = KS * NP, TC = DB * 2 * NP;
    __shared__ __attribute__((aligned(1024))) char lds[2][(2 * RC + TC) * 1024];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = lane & 31, half = lane >> 5;
    const int worker = die_order(blockIdx.x, gridDim.x);
    if (worker >= a.workers) return;
    Piece w;
    for (Walk walk(a, worker); walk.next(a, w);) {
        const int z = w.z, n = keys_of(a.s, z), first = w.first, last = min(w.last, (n + TK - 1) / TK);
        const float v_norm = Shift<E>::bwd != 0.f ? row_norm(a.vn + (long long)z * a.k_tiles, 0, a.k_tiles) : 0.f;
        const int q0 = (w.block * NW + wave) * QT;

        v8 q[QT][KS][NP], g[QT][KS][NP];
        f32x16 dq[QT][DB];
        float lse[QT], D[QT], up[QT];                      // the first two negated
#pragma unroll
        for (int t = 0; t < QT; ++t) {
            const long long tile = (long long)z * a.q_tiles + (q0 + t < a.q_tiles ? q0 + t : a.q_tiles - 1);
#pragma unroll
            for (int k = 0; k < KS; ++k) {
                read_frag<E, NP>(a.Qr + (tile * KS + k) * NP * 1024, lane, q[t][k]);
                read_frag<E, NP>(a.Gr + (tile * KS + k) * NP * 1024, lane, g[t][k]);
            }
#pragma unroll
            for (int b = 0; b < DB; ++b) dq[t][b] = (f32x16)0.f;
            lse[t] = ((const float *)(a.stat + tile * 1024))[col];
            D[t] = ((const float *)(a.stat + tile * 1024))[32 + col];
            up[t] = Shift<E>::bwd != 0.f ? ds_scale<E>(((const float *)(a.stat + tile * 1024))[64 + col], v_norm) : 1.f;
        }
        const char *Kz = a.Kr + (long long)z * a.k_tiles * KS * NP * 1024, *Vz = a.Vr + (long long)z * a.k_tiles * KS * NP * 1024;
        const char *Tz = a.Kt + (long long)z * a.k_tiles * DB * 2 * NP * 1024;
        auto fetch = [&](int step) {
            char *to = lds[step & 1];
            for (int i = wave; i < 2 * RC + TC; i += NW)
                load_chunk(i < RC ? Kz + ((long long)step * RC + i) * 1024 : i < 2 * RC ? Vz + ((long long)step * RC + i - RC) * 1024
                                                                                         : Tz + ((long long)step * TC + i - 2 * RC) * 1024,
                           to + i * 1024, lane);
        };
        auto run = [&](auto tail, int step) {
            constexpr bool TAIL = decltype(tail)::value;
            wait_loads_and_barrier();
            if (step + 1 < last) fetch(step + 1);
            const char *K = lds[step & 1], *V = K + RC * 1024, *KT = V + RC * 1024;
            f32x16 s[QT], dp[QT];
#pragma unroll
            for (int t = 0; t < QT; ++t) s[t] = (f32x16)0.f, dp[t] = (f32x16)D[t];
#pragma unroll
            for (int k = 0; k < KS; ++k) {
                v8 f[NP];
                read_frag<E, NP>(K + k * NP * 1024, lane, f);
#pragma unroll
                for (int t = 0; t < QT; ++t) s[t] = mfma_pieces<E, NP>(f, q[t][k], s[t]);
                read_frag<E, NP>(V + k * NP * 1024, lane, f);
#pragma unroll
                for (int t = 0; t < QT; ++t) dp[t] = mfma_pieces<E, NP>(f, g[t][k], dp[t]);
            }
            if constexpr (TAIL)
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    if (step * TK + 8 * (r / 4) + 4 * half + r % 4 >= n)
#pragma unroll
                        for (int t = 0; t < QT; ++t) s[t][r] = -INFINITY, dp[t][r] = 0.f;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                v8 f[QT][NP];
#pragma unroll
                for (int t = 0; t < QT; ++t) {
                    float ds[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        ds[e] = __builtin_amdgcn_exp2f(fmaf(s[t][8 * h + e], a.c, lse[t])) * dp[t][8 * h + e];
                        if constexpr (Shift<E>::bwd != 0.f) ds[e] *= up[t];
                    }
                    split8<E, NP>(ds, f[t]);
                }
#pragma unroll
                for (int b = 0; b < DB; ++b) {
                    v8 x[NP];
                    read_frag<E, NP>(KT + (b * 2 + h) * NP * 1024, lane, x);
#pragma unroll
                    for (int t = 0; t < QT; ++t) dq[t][b] = mfma_pieces<E, NP>(x, f[t], dq[t][b]);
                }
            }
        };
        __syncthreads();                                   // the last piece's tiles have been read
        if (first < last) fetch(first);
        const int whole = min(last, n / TK);               // steps without rows behind the last key
        int step = first;
        for (; step < whole; ++step) run(std::false_type(), step);
        if (step < last) run(std::true_type(), step);
#pragma unroll
        for (int t = 0; t < QT; ++t) {
            const int row = (q0 + t) * 32 + col;
            const float back = a.scale / up[t];
            if (!w.whole) store_part<DB>(a.part + ((long long)w.slot * (NW * QT) + wave * QT + t) * DB * 1024, lane, dq[t], back);
            else if (row < a.s.M) store_row<T, DB>((T *)a.dq + q_row(a.s, z, row) * a.s.d, a.s.d, half, dq[t], back);
        }
    }
}

// dk, dv: 32 KT keys per wave, steps of 32 queries.  A lane owns a key here: S = Q K^T, dV^T += g^T P, dK^T += Q^T dS; lse and D of a step's queries lie
// across a lane's registers and come from LDS with the fragments.  2 x 2 x 20480^2 heads of 32, bf16: 563 us (57 % of the vector and 40 % of the matrix pipe's
// cycles); 2 x 16 x 4096 x 8192 heads of 64: 659 us, 0.83 PFLOP/s, with no pipe full (matrix 43 %, vector 36 %, LDS 32 % of the cycles): three waves a SIMD, and within a wave
// S and g V^T, the exponentials and the products behind them follow one another, for a second key tile to run beside them spills or leaves one wave (945 us)
template <class T, int KS>
struct DkvLds {
    static constexpr int NP = Frag<T>::NP, DB = (KS + 1) / 2, CHUNKS = 2 * KS * NP + 4 * DB * NP + 1;
    static constexpr int BUFFERS = CHUNKS <= 80 ? 2 : 1;
};

template <class T, int KS, int KT, int NW>
__global__ __launch_bounds__(64 * NW, (NW == 4 ? dkv_per_cu<Frag<T>::NP, KS>() : 1)) void xa_dkv_kernel(TileArgs a) {
    using E = typename Frag<T>::E;
    using v8 = typename Vec<E>::v8;
    using L = DkvLds<T, KS>;
    constexpr int NP = L::NP, DB = L::DB, RC = KS * NP, TC = DB * 2 * NP, NB = L::BUFFERS;
    extern __shared__ __attribute__((aligned(1024))) char lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = lane & 31, half = lane >> 5;
    const int worker = die_order(blockIdx.x, gridDim.x);
    if (worker >= a.workers) return;
    Piece w;
    for (Walk walk(a, worker); walk.next(a, w);) {
        const int z = w.z, n = keys_of(a.s, z), first = w.first, last = min(w.last, a.q_tiles);
        float up = 1.f;
        if constexpr (Shift<E>::bwd != 0.f)
            up = ds_scale<E>(row_norm(a.gn + (long long)z * a.q_tiles, first, last), row_norm(a.vn + (long long)z * a.k_tiles, 0, a.k_tiles));
        const int k0 = (w.block * NW + wave) * KT;

        v8 kf[KT][KS][NP], vf[KT][KS][NP];
        f32x16 dk[KT][DB], dv[KT][DB];
#pragma unroll
        for (int t = 0; t < KT; ++t) {
            const long long tile = (long long)z * a.k_tiles + (k0 + t < a.k_tiles ? k0 + t : a.k_tiles - 1);
#pragma unroll
            for (int k = 0; k < KS; ++k) {
                read_frag<E, NP>(a.Kr + (tile * KS + k) * NP * 1024, lane, kf[t][k]);
                read_frag<E, NP>(a.Vr + (tile * KS + k) * NP * 1024, lane, vf[t][k]);
            }
#pragma unroll
            for (int b = 0; b < DB; ++b) dk[t][b] = dv[t][b] = (f32x16)0.f;
        }
        const long long qz = (long long)z * a.q_tiles;
        auto fetch = [&](int step) {
            char *to = lds + (NB == 2 ? (step & 1) * L::CHUNKS * 1024 : 0);
            const long long tile = qz + step;
            for (int i = wave; i < L::CHUNKS; i += NW) {
                const char *from = i < RC ? a.Qr + (tile * RC + i) * 1024 : i < 2 * RC ? a.Gr + (tile * RC + i - RC) * 1024
                                 : i < 2 * RC + TC ? a.Qt + (tile * TC + i - 2 * RC) * 1024
                                 : i < 2 * (RC + TC) ? a.Gt + (tile * TC + i - 2 * RC - TC) * 1024 : a.stat + tile * 1024;
                load_chunk(from, to + i * 1024, lane);
            }
        };
        __syncthreads();                                   // the last piece's tiles have been read
        if (first < last) fetch(first);
        for (int step = first; step < last; ++step) {
            wait_loads_and_barrier();
            if (NB == 2 && step + 1 < last) fetch(step + 1);
            const char *Q = lds + (NB == 2 ? (step & 1) * L::CHUNKS * 1024 : 0), *G = Q + RC * 1024, *QT = G + RC * 1024, *GT = QT + TC * 1024;
            const float *st = (const float *)(GT + TC * 1024);
            f32x16 s[KT], dp[KT];
            float lse[16];                                      // -lse
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                lse[r] = st[8 * (r / 4) + 4 * half + r % 4];
                if constexpr (Shift<E>::bwd != 0.f) lse[r] += Shift<E>::bwd;
            }
            auto scores = [&](int t) {
                s[t] = (f32x16)0.f;
#pragma unroll
                for (int r = 0; r < 16; ++r) dp[t][r] = st[32 + 8 * (r / 4) + 4 * half + r % 4];    // -D
#pragma unroll
                for (int k = 0; k < KS; ++k) {
                    v8 f[NP];
                    read_frag<E, NP>(Q + k * NP * 1024, lane, f);
                    s[t] = mfma_pieces<E, NP>(f, kf[t][k], s[t]);
                    read_frag<E, NP>(G + k * NP * 1024, lane, f);
                    dp[t] = mfma_pieces<E, NP>(f, vf[t][k], dp[t]);
                }
            };
            scores(0);
#pragma unroll
            for (int t = 0; t < KT; ++t) {
                // the next tile's products and this one's fragments are under way while the exponentials run
                constexpr bool EARLY = DB * NP <= 2 && KT > 1;           // (registers)
                v8 gf[2][DB][NP], qf[2][DB][NP];
                if constexpr (EARLY)
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int b = 0; b < DB; ++b) {
                        read_frag<E, NP>(GT + (b * 2 + h) * NP * 1024, lane, gf[h][b]);
                        read_frag<E, NP>(QT + (b * 2 + h) * NP * 1024, lane, qf[h][b]);
                    }
                if (t + 1 < KT) scores(t + 1);
                if constexpr (EARLY) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    float p[8], ds[8];
                    v8 f[NP];
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        p[e] = __builtin_amdgcn_exp2f(fmaf(s[t][8 * h + e], a.c, lse[8 * h + e]));
                        ds[e] = p[e] * dp[t][8 * h + e];
                        if constexpr (Shift<E>::bwd != 0.f) ds[e] *= up * (1.f / 32768.f);
                    }
                    split8<E, NP>(p, f);
#pragma unroll
                    for (int b = 0; b < DB; ++b) {
                        if constexpr (!EARLY) read_frag<E, NP>(GT + (b * 2 + h) * NP * 1024, lane, gf[h][b]);
                        dv[t][b] = mfma_pieces<E, NP>(gf[h][b], f, dv[t][b]);
                    }
                    split8<E, NP>(ds, f);
#pragma unroll
                    for (int b = 0; b < DB; ++b) {
                        if constexpr (!EARLY) read_frag<E, NP>(QT + (b * 2 + h) * NP * 1024, lane, qf[h][b]);
                        dk[t][b] = mfma_pieces<E, NP>(qf[h][b], f, dk[t][b]);
                    }
                }
            }
            if (NB == 1) {
                __syncthreads();
                if (step + 1 < last) fetch(step + 1);
            }
        }
        const float back_k = a.scale / up, back_v = Shift<E>::bwd != 0.f ? 1.f / 32768.f : 1.f;
#pragma unroll
        for (int t = 0; t < KT; ++t) {
            const int i = (k0 + t) * 32 + col;
            if (!w.whole) {
                const long long tile = (long long)w.slot * (NW * KT) + wave * KT + t;
                store_part<DB>(a.part + tile * DB * 1024, lane, dk[t], back_k);
                store_part<DB>(a.part2 + tile * DB * 1024, lane, dv[t], back_v);
            } else if (i < n) {
                const long long to = k_row(a.s, z, i) * a.s.d;
                store_row<T, DB>((T *)a.dk + to, a.s.d, half, dk[t], back_k);
                store_row<T, DB>((T *)a.dv + to, a.s.d, half, dv[t], back_v);
            }
        }
    }
}

// ---------------------------------------------------------------- a few query rows: K and V read once, in place
// A key row is spread over LPR lanes (8 dims each), so 64 / LPR keys per wave and load; every lane group keeps its own m, l and O for all R query
// rows and they are joined at the end: first within the workgroup, then, over the splits of the key axis, by xa_join.
template <int LPR> __device__ __forceinline__ float group_sum(float v) {
#define XA_DPP_ADD(ctrl) v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), ctrl, 0xF, 0xF, true))
    if constexpr (LPR >= 2) XA_DPP_ADD(0xB1);
    if constexpr (LPR >= 4) XA_DPP_ADD(0x4E);
    if constexpr (LPR >= 8) XA_DPP_ADD(0x141);
    if constexpr (LPR >= 16) XA_DPP_ADD(0x140);
#undef XA_DPP_ADD
    return v;
}

template <class T, bool VEC> __device__ __forceinline__ void few_load(const T *x, int off, int d, float (&v)[8]) {
    T raw[8];
    if constexpr (VEC) {
#pragma unroll
        for (int w = 0; w < (int)sizeof(T) / 2; ++w) ((uint4 *)raw)[w] = off < d ? ((const uint4 *)(x + off))[w] : make_uint4(0, 0, 0, 0);
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) raw[e] = off + e < d ? x[off + e] : (T)0.f;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = (float)raw[e];
}

template <class T, int R, int LPR, bool VEC>
__global__ __launch_bounds__(256) void xa_few_kernel(FewArgs a) {
    constexpr int GROUPS = 64 / LPR, U = 2;             // lane groups per wave, keys in flight per group
    __shared__ float sm[4][R][2], so[4][R][LPR * 8];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, off = (lane % LPR) * 8, group = wave * GROUPS + lane / LPR;
    const int split = blockIdx.x % a.splits, z = blockIdx.x / a.splits, b = z / a.s.Hk, hk = z - b * a.s.Hk;
    const T *k = (const T *)a.k + b * a.k_sb + hk * a.k_sh, *v = (const T *)a.v + b * a.v_sb + hk * a.v_sh;
    const unsigned char *mask = a.mask ? a.mask + b * a.mask_sb : nullptr;
    const int n0 = (int)((long long)a.s.N * split / a.splits), n1 = (int)((long long)a.s.N * (split + 1) / a.splits);
    float q[R][8], o[R][8], m[R], l[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int g = r / a.s.Nq;
        if (r < a.s.M) few_load<T, false>((const T *)a.q + b * a.q_sb + (r - g * a.s.Nq) * a.q_sn + (hk * a.s.G + g) * a.q_sh, off, a.s.d, q[r]);
        else
#pragma unroll
            for (int e = 0; e < 8; ++e) q[r][e] = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            q[r][e] *= a.c;
            o[r][e] = 0.f;
        }
        m[r] = LOWEST;
        l[r] = 0.f;
    }
    // every lane of a wave runs the same number of rounds: the row sums cross lanes
    for (long long i0 = n0; i0 < n1; i0 += 4 * GROUPS * U) {
        float kv[U][8], vv[U][8];
        bool on[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const long long i = i0 + u * 4 * GROUPS + group;
            on[u] = i < n1 && (!mask || mask[i < n1 ? i : n0]);
            const long long at = i < n1 ? i : n0;
            few_load<T, VEC>(k + at * a.k_sn, off, a.s.d, kv[u]);
            few_load<T, VEC>(v + at * a.v_sn, off, a.s.d, vv[u]);
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (!on[u])
#pragma unroll
                for (int e = 0; e < 8; ++e) vv[u][e] = 0.f;         // what stands in a masked row may be NaN
#pragma unroll
        for (int r = 0; r < R; ++r) {
            float s[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                s[u] = 0.f;
#pragma unroll
                for (int e = 0; e < 8; ++e) s[u] = fmaf(q[r][e], kv[u][e], s[u]);
                s[u] = group_sum<LPR>(s[u]);
                s[u] = on[u] ? s[u] : -INFINITY;
            }
            float top = s[0];
#pragma unroll
            for (int u = 1; u < U; ++u) top = fmaxf(top, s[u]);
            if (__any(top > m[r] + LAZY)) {
                const float up = fmaxf(m[r], top), f = __builtin_amdgcn_exp2f(m[r] - up);
                m[r] = up;
                l[r] *= f;
#pragma unroll
                for (int e = 0; e < 8; ++e) o[r][e] *= f;
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const float p = on[u] ? __builtin_amdgcn_exp2f(s[u] - m[r]) : 0.f, pd = p * a.down;
                l[r] += p;
#pragma unroll
                for (int e = 0; e < 8; ++e) o[r][e] = fmaf(pd, vv[u][e], o[r][e]);
            }
        }
    }
    // join the lane groups of the wave, then the four waves
#pragma unroll
    for (int x = LPR; x < 64; x <<= 1)
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const float m2 = __shfl_xor(m[r], x), l2 = __shfl_xor(l[r], x), up = fmaxf(m[r], m2);
            const float f = exp2f(m[r] - up), f2 = exp2f(m2 - up);
            m[r] = up;
            l[r] = l[r] * f + l2 * f2;
#pragma unroll
            for (int e = 0; e < 8; ++e) o[r][e] = o[r][e] * f + __shfl_xor(o[r][e], x) * f2;
        }
    if (lane < LPR)
#pragma unroll
        for (int r = 0; r < R; ++r) {
            if (lane == 0) {
                sm[wave][r][0] = m[r];
                sm[wave][r][1] = l[r];
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) so[wave][r][off + e] = o[r][e];
        }
    __syncthreads();
    for (int i = threadIdx.x; i < R * LPR * 8; i += 256) {
        const int r = i / (LPR * 8), dim = i % (LPR * 8);
        if (r >= a.s.M || dim >= a.s.d) continue;
        float up = sm[0][r][0], sum = 0.f, x = 0.f;
#pragma unroll
        for (int w = 1; w < 4; ++w) up = fmaxf(up, sm[w][r][0]);
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const float f = exp2f(sm[w][r][0] - up);
            sum = fmaf(f, sm[w][r][1], sum);
            x = fmaf(f, so[w][r][dim], x);
        }
        const long long zr = (long long)z * a.s.M + r;
        if (a.splits > 1) {
            const long long at = (long long)split * a.s.B * a.s.Hk * a.s.M + zr;
            a.part[at * a.s.d + dim] = x;
            if (dim == 0) {
                a.ml[2 * at] = up;
                a.ml[2 * at + 1] = sum;
            }
        } else {
            ((T *)a.o)[q_row(a.s, z, r) * a.s.d + dim] = (T)(sum == 0.f ? 0.f : x / sum * a.up);
            if (dim == 0 && a.lse) a.lse[zr] = sum == 0.f ? INFINITY : up + log2f(sum);
        }
    }
}

// ---------------------------------------------------------------- float32 beyond the pieces
// Three bf16 pieces hold a float32 up to 3.39e38 and not infinity, whose remainder is inf - inf, and the six products of two operands overflow one by one, with
// either sign, where the sum of their exact values would not.  Rows of the tile kernels' operands up to 2^36 keep every product and sum of both passes finite (dS K:
// 2^36 to the third, times 2, times 2^17 rows); a z with a row beyond, an infinite one among them, is computed again here, from the formula in
// float32 arithmetic and from the tensors themselves.  Such rows are not met in earnest, so this is the simplest kernel: a wave takes a row, its lanes
// 64 rows of the other side and then the row's dims (6 x 2 x 7680^2 heads of 16, both passes: 0.2 s).  Otherwise a workgroup reads the tiles' norms of its z and
// ends: 5 us forward and 6 backward, of 1480.
struct BeyondArgs {
    Shape s;
    const float *q, *k, *v, *g;
    long long q_sb, q_sn, q_sh, k_sb, k_sn, k_sh, v_sb, v_sn, v_sh, g_sb, g_sn, g_sh;
    const float *qn, *kn, *vn, *gn;      // gn: backward
    const char *stat;                    // -lse and -D, as xa_pack left them
    int q_tiles, k_tiles, blocks;        // blocks: workgroups of a z
    float c, scale;                      // c: of the exponents, in units of log 2
    float *o, *lse, *dq, *dk, *dv;
};
constexpr float PIECES_BOUND = 0x1p36f;
__device__ __forceinline__ bool beyond(const BeyondArgs &a, int z) {       // every lane of a wave calls it
    const long long q0 = (long long)z * a.q_tiles, k0 = (long long)z * a.k_tiles;
    bool out = false;
    for (int i = threadIdx.x & 63; i < a.k_tiles; i += 64) out |= !(fmaxf(a.kn[k0 + i], a.vn[k0 + i]) <= PIECES_BOUND);
    for (int i = threadIdx.x & 63; i < a.q_tiles; i += 64) out |= !(a.qn[q0 + i] <= PIECES_BOUND) || (a.gn && !(a.gn[q0 + i] <= PIECES_BOUND));
    return __any(out);
}
__device__ __forceinline__ float beyond_dot(const float *x, const float *y, int d, float f) {
    float s = 0.f;
#pragma unroll 8
    for (int e = 0; e < d; ++e) s = fmaf(x[e] * f, y[e], s);
    return s;
}
struct BeyondRows {                      // of one z
    const float *q, *k, *v, *g;
    int b, Nq;
    __device__ __forceinline__ BeyondRows(const BeyondArgs &a, int z) {
        b = z / a.s.Hk, Nq = a.s.Nq;
        const int hk = z - b * a.s.Hk;
        q = a.q + b * a.q_sb + hk * a.s.G * a.q_sh, k = a.k + b * a.k_sb + hk * a.k_sh, v = a.v + b * a.v_sb + hk * a.v_sh;
        g = a.g ? a.g + b * a.g_sb + hk * a.s.G * a.g_sh : nullptr;
    }
    __device__ __forceinline__ const float *query(const float *x, long long sn, long long sh, int r) const { return x + (r % Nq) * sn + (r / Nq) * sh; }
    __device__ __forceinline__ long long key(const Shape &s, int i) const { return s.idx ? s.idx[(long long)b * s.N + i] : i; }
};

__global__ __launch_bounds__(256) void xa_beyond_fwd_kernel(BeyondArgs a) {
    const int z = blockIdx.x / a.blocks, lane = threadIdx.x & 63, n = keys_of(a.s, z), d = a.s.d;
    if (!beyond(a, z)) return;
    const BeyondRows at(a, z);
    for (int r = (blockIdx.x % a.blocks) * 4 + (threadIdx.x >> 6); r < a.s.M; r += a.blocks * 4) {
        const float *q = at.query(at.q, a.q_sn, a.q_sh, r);
        auto score = [&](int i) { return beyond_dot(q, at.k + at.key(a.s, i) * a.k_sn, d, a.c); };
        float m = LOWEST, l = 0.f, o0 = 0.f, o1 = 0.f;
        for (int i = lane; i < n; i += 64) m = fmaxf(m, score(i));
        m = md_wave_max(m);
        for (int i = lane; i < n; i += 64) l += exp2f(score(i) - m);
        l = md_wave_sum(l);
        const float inv = l == 0.f ? 0.f : 1.f / l;
        for (int i0 = 0; i0 < n; i0 += 64) {
            const float p = i0 + lane < n ? exp2f(score(i0 + lane) - m) * inv : 0.f;     // normalised first: sums of large values stay in range
            const int some = min(64, n - i0);
#pragma unroll 8
            for (int i = 0; i < some; ++i) {
                const float pi = __shfl(p, i), *v = at.v + at.key(a.s, i0 + i) * a.v_sn;
                if (lane < d) o0 = fmaf(pi, v[lane], o0);
                if (lane + 64 < d) o1 = fmaf(pi, v[lane + 64], o1);
            }
        }
        float *o = a.o + q_row(a.s, z, r) * d;
        if (lane < d) o[lane] = l == 0.f ? 0.f : o0;
        if (lane + 64 < d) o[lane + 64] = l == 0.f ? 0.f : o1;
        if (lane == 0 && a.lse) a.lse[(long long)z * a.s.M + r] = l == 0.f ? INFINITY : m + log2f(l);
    }
}

// rows of dq, then of dk and dv
__global__ __launch_bounds__(256) void xa_beyond_bwd_kernel(BeyondArgs a) {
    const int z = blockIdx.x / a.blocks, lane = threadIdx.x & 63, n = keys_of(a.s, z), d = a.s.d;
    if (!beyond(a, z)) return;
    const BeyondRows at(a, z);
    // weight and scale dS of a pair (scaled first: sums of large values stay in range): `st` are the query row's -lse and -D
    auto pair = [&](const float *q, const float *g, int r, int i, float &p, float &ds) {
        const float *st = (const float *)(a.stat + ((long long)z * a.q_tiles + r / 32) * 1024) + r % 32;
        const long long key = at.key(a.s, i);
        p = exp2f(beyond_dot(q, at.k + key * a.k_sn, d, a.c) + st[0]);
        ds = p * (beyond_dot(g, at.v + key * a.v_sn, d, 1.f) + st[32]) * a.scale;
    };
    const int queries = a.dq ? a.s.M : 0, keys = a.dk ? n : 0;
    for (long long row = (blockIdx.x % a.blocks) * 4 + (threadIdx.x >> 6); row < (long long)queries + keys; row += a.blocks * 4) {
        float x0 = 0.f, x1 = 0.f, y0 = 0.f, y1 = 0.f;
        if (row < queries) {
            const int r = (int)row;
            const float *q = at.query(at.q, a.q_sn, a.q_sh, r), *g = at.query(at.g, a.g_sn, a.g_sh, r);
            for (int i0 = 0; i0 < n; i0 += 64) {
                float p = 0.f, ds = 0.f;
                if (i0 + lane < n) pair(q, g, r, i0 + lane, p, ds);
                const int some = min(64, n - i0);
#pragma unroll 8
                for (int i = 0; i < some; ++i) {
                    const float di = __shfl(ds, i), *k = at.k + at.key(a.s, i0 + i) * a.k_sn;
                    if (lane < d) x0 = fmaf(di, k[lane], x0);
                    if (lane + 64 < d) x1 = fmaf(di, k[lane + 64], x1);
                }
            }
            float *dq = a.dq + q_row(a.s, z, r) * d;
            if (lane < d) dq[lane] = x0;
            if (lane + 64 < d) dq[lane + 64] = x1;
        } else {
            const int i = (int)(row - queries);
            for (int r0 = 0; r0 < a.s.M; r0 += 64) {
                float p = 0.f, ds = 0.f;
                if (r0 + lane < a.s.M)
                    pair(at.query(at.q, a.q_sn, a.q_sh, r0 + lane), at.query(at.g, a.g_sn, a.g_sh, r0 + lane), r0 + lane, i, p, ds);
                const int some = min(64, a.s.M - r0);
#pragma unroll 4
                for (int r = 0; r < some; ++r) {
                    const float di = __shfl(ds, r), pi = __shfl(p, r);
                    const float *q = at.query(at.q, a.q_sn, a.q_sh, r0 + r), *g = at.query(at.g, a.g_sn, a.g_sh, r0 + r);
                    if (lane < d) x0 = fmaf(di, q[lane], x0), y0 = fmaf(pi, g[lane], y0);
                    if (lane + 64 < d) x1 = fmaf(di, q[lane + 64], x1), y1 = fmaf(pi, g[lane + 64], y1);
                }
            }
            const long long to = k_row(a.s, z, i) * d;
            if (lane < d) a.dk[to + lane] = x0, a.dv[to + lane] = y0;
            if (lane + 64 < d) a.dk[to + lane + 64] = x1, a.dv[to + lane + 64] = y1;
        }
    }
}

// ---------------------------------------------------------------- host side
// Query rows per key head up to which K and V are read in place.  8 rows on 8 x 20480 keys of 4 heads of 64 (bf16): 73 us, through the tiles 129 us, most of it
// packing; 16 rows would take two such passes (128 us through the tiles).  1 row: 43 us, 3.9 TB/s of K and V
constexpr int FEW_ROWS = 8;
constexpr int CUS = 256;

int check(const md_attn_desc &a, const char *what) {
    MD_REQUIRE(a.dtype >= 0 && a.dtype <= 2, "%s: unknown dtype %d (0 f32, 1 bf16, 2 f16)", what, a.dtype);
    MD_REQUIRE(a.B >= 0 && a.Nq >= 0 && a.Nk >= 0, "%s: negative size", what);
    MD_REQUIRE(a.d >= 1 && a.d <= MD_ATTN_MAX_D, "%s: head size %d (1 .. %d)", what, a.d, MD_ATTN_MAX_D);
    MD_REQUIRE(a.Hk >= 1 && a.Hq >= 1 && a.Hq % a.Hk == 0, "%s: %d query heads are not a multiple of %d key heads", what, a.Hq, a.Hk);
    MD_REQUIRE(a.Hq <= 65535 && a.B <= 65535, "%s: more than 65535 heads or sequences", what);
    MD_REQUIRE((long long)a.B * a.Hq < (1LL << 31) - 65536, "%s: 2^31 heads of sequences or more", what);
    MD_REQUIRE((long long)a.B * a.Hq * a.Nq < (1LL << 31) - 65536 && (long long)a.B * a.Hk * a.Nk < (1LL << 31) - 65536 &&
                   a.Nk < (1 << 30) && (long long)a.Hq / a.Hk * a.Nq < (1 << 30),
               "%s: 2^31 rows or more", what);
    MD_REQUIRE((long long)a.B * a.Hk < 1 << 24, "%s: 2^24 key heads of sequences or more", what);          // a launch has fewer than 2^32 threads
    MD_REQUIRE(a.scale - a.scale == 0.f, "%s: scale is not finite", what);
    return MD_OK;
}

int ks_of(int d) { return d <= 16 ? 1 : d <= 32 ? 2 : d <= 64 ? 4 : d <= 96 ? 6 : 8; }
size_t align256(size_t n) { return (n + 255) & ~(size_t)255; }

// One launch of a tile kernel: `nw` waves of `t` tiles of 32 rows each in a workgroup, `workers` workgroups, and where their parts go.
struct Tiles {
    int nw, t, rows, step, workers;
    long long units;
    bool join;
    size_t part, part2, ml, first;
};
// How a call is run, and where its workspace's parts begin; the same for the size query and the launch.
struct Plan {
    int M, Z, KS, NP, DB, q_tiles, k_tiles;
    bool few;
    int splits;                                   // few rows: of the keys
    Tiles fwd, dq, dkv;
    size_t idx, cnt, qn, kn, vn, gn, Qr, Kr, Vt, Qt, Kt, Vr, Gr, Gt, stat, part, ml, bytes;
};

// Workgroups that the chip holds at once, so that they all run to the end together -- unless that left them fewer than `least` steps: then one block of rows
// each at the least.  `step` as in TileArgs; the number of keys is what it is without a mask.
Tiles tiles_for(int Z, int tiles, int t, int step, long long steps, int least, int per_cu, bool masked) {
    Tiles r{};
    r.nw = tiles <= 1 ? 1 : 4;
    r.t = r.nw == 1 ? 1 : t;
    r.rows = 32 * r.t * r.nw;
    r.step = step;
    const long long blocks = (long long)Z * ((tiles + r.t * r.nw - 1) / (r.t * r.nw)), units = blocks * (steps < 1 ? 1 : steps);
    const long long most = (r.nw == 1 ? 8 : per_cu) * CUS, want = std::max(blocks, units / least);
    r.workers = (int)std::max<long long>(1, std::min(most, want));
    r.units = units;
    r.join = blocks && (masked || units % r.workers || units / r.workers % (steps < 1 ? 1 : steps));
    return r;
}

template <int NP, int KS> Plan plan_of(const md_attn_desc &a, bool backward) {
    Plan p{};
    p.M = a.Hq / a.Hk * a.Nq;
    p.Z = a.B * a.Hk;
    p.KS = KS;
    p.NP = NP;
    p.DB = (KS + 1) / 2;
    p.q_tiles = (p.M + 31) / 32;
    p.k_tiles = (a.Nk + 127) / 128 * 4;                       // whole steps of every kernel
    p.few = !backward && p.M <= FEW_ROWS;
    size_t at = 0;
    auto take = [&](size_t n) { const size_t r = at; at = align256(at + n); return r; };
    const size_t kb = 1024;
    if (p.few) {
        // as many workgroups as the chip holds at once (registers: 7, 3, 2 a CU for 1, 4, 8 rows), 128 keys each at the least
        const long long want = (p.M <= 1 ? 7 : p.M <= 4 ? 3 : 2) * CUS / std::max(1, p.Z), most = a.Nk / 128;
        p.splits = (int)std::max<long long>(1, std::min<long long>(std::min(want, most), 64));
        if (p.splits > 1) {
            p.part = take((size_t)p.Z * p.M * p.splits * a.d * 4);
            p.ml = take((size_t)p.Z * p.M * p.splits * 8);
        }
        p.bytes = at;
        return p;
    }
    const bool masked = a.key_mask != nullptr;
    if (masked) {
        p.idx = take((size_t)a.B * a.Nk * 4);
        p.cnt = take((size_t)a.B * 4);
    }
    const size_t qR = (size_t)p.Z * p.q_tiles * p.KS * p.NP * kb, qT = (size_t)p.Z * p.q_tiles * p.DB * 2 * p.NP * kb;
    const size_t kR = (size_t)p.Z * p.k_tiles * p.KS * p.NP * kb, kT = (size_t)p.Z * p.k_tiles * p.DB * 2 * p.NP * kb;
    const int qt = p.q_tiles >= 8 ? query_tiles<NP, KS>() : 1;
    p.Qr = take(qR);
    p.Kr = take(kR);
    p.qn = take((size_t)p.Z * p.q_tiles * 4);
    p.kn = take((size_t)p.Z * p.k_tiles * 4);
    p.vn = take((size_t)p.Z * p.k_tiles * 4);
    if (!backward) {
        const int tk = fwd_keys<NP, KS>();
        p.Vt = take(kT);
        p.fwd = tiles_for(p.Z, p.q_tiles, qt, tk, (a.Nk + tk - 1) / tk, 256 / tk, qt == 2 ? fwd_per_cu<NP, KS, 2>() : fwd_per_cu<NP, KS, 1>(), masked);
        if (p.fwd.join) {
            p.fwd.part = take((size_t)2 * p.fwd.workers * p.fwd.rows * p.DB * 32 * 4);
            p.fwd.ml = take((size_t)2 * p.fwd.workers * p.fwd.rows * 8);
            p.fwd.first = take((size_t)p.fwd.workers * 16);
        }
    } else {
        p.gn = take((size_t)p.Z * p.q_tiles * 4);
        p.Vr = take(kR);
        p.Kt = take(kT);
        p.Qt = take(qT);
        p.Gr = take(qR);
        p.Gt = take(qT);
        p.stat = take((size_t)p.Z * p.q_tiles * kb);
        p.dq = tiles_for(p.Z, p.q_tiles, qt, DQ_KEYS, (a.Nk + DQ_KEYS - 1) / DQ_KEYS, 256 / DQ_KEYS, qt == 2 ? dq_per_cu<NP, KS, 2>() : dq_per_cu<NP, KS, 1>(), masked);
        p.dkv = tiles_for(p.Z, (a.Nk + 31) / 32, key_tiles<NP, KS>(), 0, p.q_tiles, 8, dkv_per_cu<NP, KS>(), masked);
        const size_t nq = p.dq.join ? (size_t)2 * p.dq.workers * p.dq.rows * p.DB * 32 * 4 : 0, nk = p.dkv.join ? (size_t)2 * p.dkv.workers * p.dkv.rows * p.DB * 32 * 4 : 0;
        p.dq.part = p.dkv.part = take(std::max(nq, nk));            // dq's are summed before dk's are written (and `first` likewise)
        p.dkv.part2 = take(nk);
        p.dq.first = p.dkv.first = take((size_t)std::max(p.dq.workers, p.dkv.workers) * 16);
    }
    p.bytes = at;
    return p;
}

Plan make_plan(const md_attn_desc &a, bool backward) {
    const int ks = ks_of(a.d);
    if (a.dtype == 0)
        return ks == 1 ? plan_of<3, 1>(a, backward) : ks == 2 ? plan_of<3, 2>(a, backward) : ks == 4 ? plan_of<3, 4>(a, backward)
             : ks == 6 ? plan_of<3, 6>(a, backward) : plan_of<3, 8>(a, backward);
    return ks == 1 ? plan_of<1, 1>(a, backward) : ks == 2 ? plan_of<1, 2>(a, backward) : ks == 4 ? plan_of<1, 4>(a, backward)
         : ks == 6 ? plan_of<1, 6>(a, backward) : plan_of<1, 8>(a, backward);
}

bool aligned_rows(const void *x, size_t size, int d, long long sb, long long sn, long long sh) {
    const long long e = 16 / (long long)size;
    return d % 8 == 0 && ((uintptr_t)x & 15) == 0 && sb % e == 0 && sn % e == 0 && sh % e == 0;
}

template <class K> int set_lds(K kernel, int bytes) {
    if (bytes > 64 * 1024) MD_CHECK_HIP(hipFuncSetAttribute((const void *)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes));
    return MD_OK;
}

float down_of(int keys) { return LAZY + ceilf(log2f((float)std::max(1, keys))); }
unsigned grid8(long long blocks) { return (unsigned)((blocks + 7) / 8 * 8); }

template <class T, int R> int launch_few(const FewArgs &f, int d, bool vec, hipStream_t s) {
    const unsigned grid = (unsigned)f.s.B * f.s.Hk * f.splits;
#define XA_FEW(LPR) \
    if (vec) xa_few_kernel<T, R, LPR, true><<<grid, 256, 0, s>>>(f); else xa_few_kernel<T, R, LPR, false><<<grid, 256, 0, s>>>(f)
    if (d <= 16) { XA_FEW(2); }
    else if (d <= 32) { XA_FEW(4); }
    else if (d <= 64) { XA_FEW(8); }
    else { XA_FEW(16); }
#undef XA_FEW
    return MD_OK;
}

template <class T> int run_few(const md_attn_desc &a, const Plan &p, const Shape &sh, char *ws, hipStream_t s) {
    FewArgs f{};
    f.s = sh;
    f.q = a.q, f.k = a.k, f.v = a.v;
    f.q_sb = a.q_sb, f.q_sn = a.q_sn, f.q_sh = a.q_sh, f.k_sb = a.k_sb, f.k_sn = a.k_sn, f.k_sh = a.k_sh;
    f.v_sb = a.v_sb, f.v_sn = a.v_sn, f.v_sh = a.v_sh, f.mask_sb = a.mask_sb;
    f.mask = (const unsigned char *)a.key_mask;
    f.splits = p.splits;
    f.c = a.scale * LOG2E;
    f.down = exp2f(-down_of(a.Nk)), f.up = exp2f(down_of(a.Nk));
    f.o = a.o, f.lse = a.lse;
    f.part = (float *)(ws + p.part), f.ml = (float *)(ws + p.ml);
    const bool vec = aligned_rows(a.k, sizeof(T), a.d, a.k_sb, a.k_sn, a.k_sh) && aligned_rows(a.v, sizeof(T), a.d, a.v_sb, a.v_sn, a.v_sh);
    const int rc = p.M <= 1 ? launch_few<T, 1>(f, a.d, vec, s) : p.M <= 4 ? launch_few<T, 4>(f, a.d, vec, s) : launch_few<T, 8>(f, a.d, vec, s);
    if (rc) return rc;
    MD_CHECK_LAUNCH("md_cross_attn_fwd: few rows");
    if (p.splits > 1) {
        xa_few_join_kernel<T><<<(unsigned)p.Z * p.M, 64, 0, s>>>(f);
        MD_CHECK_LAUNCH("md_cross_attn_fwd: join");
    }
    return MD_OK;
}

// descriptor -> kernels' shape, and the list of valid keys where there is a mask
int start(const md_attn_desc &a, const Plan &p, char *ws, hipStream_t s, Shape &sh) {
    sh.B = a.B, sh.Hk = a.Hk, sh.G = a.Hq / a.Hk, sh.Nq = a.Nq, sh.N = a.Nk, sh.M = p.M, sh.Hq = a.Hq, sh.d = a.d;
    if (a.key_mask && !p.few) {
        sh.idx = (const int *)(ws + p.idx), sh.cnt = (const int *)(ws + p.cnt);
        xa_compact_kernel<<<a.B, 1024, 0, s>>>((const unsigned char *)a.key_mask, a.mask_sb, a.Nk, (int *)(ws + p.idx), (int *)(ws + p.cnt));
        MD_CHECK_LAUNCH("md_cross_attn: key list");
    }
    return MD_OK;
}

PackJob job_of(const void *x, long long sb, long long sn, long long sh, size_t size, int d, char *R, char *T, int tiles, int query, float factor) {
    PackJob j{};
    j.x = x, j.sb = sb, j.sn = sn, j.sh = sh, j.R = R, j.T = T, j.tiles = tiles, j.query = query, j.factor = factor;
    j.vec = aligned_rows(x, size, d, sb, sn, sh);
    return j;
}

constexpr int MAX_PACK = 1 << 25;             // a launch has fewer than 2^32 threads

template <class T, int KS> int launch_pack(PackArgs &k, const Plan &p, long long more, hipStream_t s) {
    long long n = 0;
    for (int i = 0; i < k.jobs; ++i) {
        k.blocks[i] = (int)n;
        n += (long long)p.Z * k.job[i].tiles;
    }
    k.blocks[k.jobs] = (int)n;
    n += more;
    MD_REQUIRE(n < (1LL << 31), "md_cross_attn: too many tiles");
    for (long long at = 0; at < n; at += MAX_PACK) {
        k.first = (int)at;
        xa_pack_kernel<T, KS><<<(unsigned)std::min<long long>(n - at, MAX_PACK), 64, 0, s>>>(k);
    }
    MD_CHECK_LAUNCH("md_cross_attn: pack");
    return MD_OK;
}

TileArgs tile_args(const Shape &sh, const Plan &p, const Tiles &w, char *ws) {
    TileArgs t{};
    t.s = sh;
    t.q_tiles = p.q_tiles, t.k_tiles = p.k_tiles, t.workers = w.workers, t.rows = w.rows, t.step = w.step, t.units = w.units;
    t.part = (float *)(ws + w.part), t.part2 = (float *)(ws + w.part2), t.ml = (float *)(ws + w.ml);
    t.first = w.join ? (int4 *)(ws + w.first) : nullptr;
    return t;
}

// what the float32 kernels beyond the pieces are told, and their workgroups: as many as keep the chip busy should they have work, one for each z at the least
BeyondArgs beyond_args(const md_attn_desc &a, const Plan &p, const Shape &sh, char *ws, long long rows) {
    BeyondArgs b{};
    b.s = sh;
    b.q = (const float *)a.q, b.k = (const float *)a.k, b.v = (const float *)a.v;
    b.q_sb = a.q_sb, b.q_sn = a.q_sn, b.q_sh = a.q_sh, b.k_sb = a.k_sb, b.k_sn = a.k_sn, b.k_sh = a.k_sh, b.v_sb = a.v_sb, b.v_sn = a.v_sn, b.v_sh = a.v_sh;
    b.qn = (const float *)(ws + p.qn), b.kn = (const float *)(ws + p.kn), b.vn = (const float *)(ws + p.vn);
    b.q_tiles = p.q_tiles, b.k_tiles = p.k_tiles;
    b.blocks = (int)std::max<long long>(1, std::min<long long>((rows + 3) / 4, 4 * CUS / p.Z));
    b.c = a.scale * LOG2E, b.scale = a.scale;
    return b;
}

template <class T, int KS> int run_fwd(const md_attn_desc &a, const Plan &p, const Shape &sh, char *ws, hipStream_t s) {
    constexpr int NP = Frag<T>::NP, TK = fwd_keys<NP, KS>();
    // c > 0 in the kernels: a negative scale goes into q's sign.  In float32 q takes all of it (2^-24 like every other product of the sums)
    const float factor = NP == 3 ? a.scale * LOG2E : a.scale < 0.f ? -1.f : 1.f;
    PackArgs k{};
    k.s = sh, k.jobs = 3;
    k.job[0] = job_of(a.q, a.q_sb, a.q_sn, a.q_sh, sizeof(T), a.d, ws + p.Qr, nullptr, p.q_tiles, 1, factor);
    k.job[1] = job_of(a.k, a.k_sb, a.k_sn, a.k_sh, sizeof(T), a.d, ws + p.Kr, nullptr, p.k_tiles, 0, 1.f);
    k.job[2] = job_of(a.v, a.v_sb, a.v_sn, a.v_sh, sizeof(T), a.d, nullptr, ws + p.Vt, p.k_tiles, 0, 1.f);
    if (Shift<typename Frag<T>::E>::fwd == 0.f) k.job[0].norm = (float *)(ws + p.qn), k.job[1].norm = (float *)(ws + p.kn), k.job[2].norm = (float *)(ws + p.vn);
    if (int rc = launch_pack<T, KS>(k, p, 0, s)) return rc;
    TileArgs t = tile_args(sh, p, p.fwd, ws);
    t.qn = (float *)(ws + p.qn), t.kn = (float *)(ws + p.kn), t.vn = (float *)(ws + p.vn);
    t.Qr = ws + p.Qr, t.Kr = ws + p.Kr, t.Vt = ws + p.Vt;
    t.c = fmaxf(fabsf(a.scale) * LOG2E, 1.2e-38f);         // not 0: the scores of rows behind the last key are -inf
    t.down = down_of(a.Nk);
    t.o = a.o, t.lse = a.lse;
    const unsigned grid = grid8(t.workers);
    if (p.fwd.nw == 1) xa_fwd_kernel<T, KS, 1, TK, 1><<<grid, 64, 0, s>>>(t);
    else if constexpr (query_tiles<NP, KS>() == 2) {
        if (p.fwd.t == 2) xa_fwd_kernel<T, KS, 2, TK, 4><<<grid, 256, 0, s>>>(t);
        else xa_fwd_kernel<T, KS, 1, TK, 4><<<grid, 256, 0, s>>>(t);
    } else
        xa_fwd_kernel<T, KS, 1, TK, 4><<<grid, 256, 0, s>>>(t);
    MD_CHECK_LAUNCH("md_cross_attn_fwd");
    if (p.fwd.join) {
        xa_join_kernel<T, (KS + 1) / 2><<<dim3(t.workers, t.rows / 32), 256, 0, s>>>(t);
        MD_CHECK_LAUNCH("md_cross_attn_fwd: join");
    }
    if constexpr (NP == 3) {
        BeyondArgs b = beyond_args(a, p, sh, ws, p.M);
        b.o = (float *)a.o, b.lse = a.lse;
        xa_beyond_fwd_kernel<<<(unsigned)p.Z * b.blocks, 256, 0, s>>>(b);
        MD_CHECK_LAUNCH("md_cross_attn_fwd: rows beyond the pieces");
    }
    return MD_OK;
}

template <class T, int KS> int run_bwd(const md_attn_desc &a, const Plan &p, const Shape &sh, char *ws, hipStream_t s) {
    constexpr int NP = Frag<T>::NP;
    const float sign = a.scale < 0.f ? -1.f : 1.f;
    PackArgs k{};
    k.s = sh;
    k.jobs = 4;
    k.job[0] = job_of(a.g, a.g_sb, a.g_sn, a.g_sh, sizeof(T), a.d, ws + p.Gr, ws + p.Gt, p.q_tiles, 1, 1.f);
    k.job[1] = job_of(a.q, a.q_sb, a.q_sn, a.q_sh, sizeof(T), a.d, ws + p.Qr, ws + p.Qt, p.q_tiles, 1, sign);
    k.job[2] = job_of(a.k, a.k_sb, a.k_sn, a.k_sh, sizeof(T), a.d, ws + p.Kr, ws + p.Kt, p.k_tiles, 0, 1.f);
    k.job[3] = job_of(a.v, a.v_sb, a.v_sn, a.v_sh, sizeof(T), a.d, ws + p.Vr, nullptr, p.k_tiles, 0, 1.f);
    k.o = a.o, k.lse = a.lse, k.stat = ws + p.stat;
    if (NP == 3 || Shift<typename Frag<T>::E>::bwd != 0.f) k.job[0].norm = (float *)(ws + p.gn), k.job[3].norm = (float *)(ws + p.vn);
    if (NP == 3) k.job[1].norm = (float *)(ws + p.qn), k.job[2].norm = (float *)(ws + p.kn);
    long long zero = 0;
    if (a.key_mask && a.dk) {
        k.mask = (const unsigned char *)a.key_mask, k.mask_sb = a.mask_sb, k.dk = a.dk, k.dv = a.dv;
        zero = (long long)a.B * ((a.Nk + 31) / 32);
    }
    if (int rc = launch_pack<T, KS>(k, p, zero, s)) return rc;
    auto args = [&](const Tiles &w) {
        TileArgs t = tile_args(sh, p, w, ws);
        t.Qr = ws + p.Qr, t.Kr = ws + p.Kr, t.Vr = ws + p.Vr, t.Qt = ws + p.Qt, t.Kt = ws + p.Kt, t.Gr = ws + p.Gr, t.Gt = ws + p.Gt, t.stat = ws + p.stat;
        t.c = fmaxf(fabsf(a.scale) * LOG2E, 1.2e-38f);
        t.dq = a.dq, t.dk = a.dk, t.dv = a.dv;
        t.vn = (const float *)(ws + p.vn), t.gn = (const float *)(ws + p.gn);
        return t;
    };
    if (a.dq && p.M) {
        TileArgs t = args(p.dq);
        t.scale = a.scale;
        const unsigned grid = grid8(t.workers);
        if (p.dq.nw == 1) xa_dq_kernel<T, KS, 1, 1><<<grid, 64, 0, s>>>(t);
        else if constexpr (query_tiles<NP, KS>() == 2) {
            if (p.dq.t == 2) xa_dq_kernel<T, KS, 2, 4><<<grid, 256, 0, s>>>(t);
            else xa_dq_kernel<T, KS, 1, 4><<<grid, 256, 0, s>>>(t);
        } else
            xa_dq_kernel<T, KS, 1, 4><<<grid, 256, 0, s>>>(t);
        MD_CHECK_LAUNCH("md_cross_attn_bwd: dq");
        if (p.dq.join) {
            xa_sum_kernel<T, (KS + 1) / 2><<<dim3(t.workers, t.rows / 32), 256, 0, s>>>(t);
            MD_CHECK_LAUNCH("md_cross_attn_bwd: dq sums");
        }
    }
    if (a.dk && a.Nk) {
        TileArgs t = args(p.dkv);
        t.scale = fabsf(a.scale);                          // Q's fragments carry the sign
        const unsigned grid = grid8(t.workers);
        using L = DkvLds<T, KS>;
        const int lds = L::BUFFERS * L::CHUNKS * 1024;
        if (p.dkv.nw == 1) {
            if (int rc = set_lds(xa_dkv_kernel<T, KS, 1, 1>, lds)) return rc;
            xa_dkv_kernel<T, KS, 1, 1><<<grid, 64, lds, s>>>(t);
        } else {
            constexpr int KT = key_tiles<NP, KS>();
            if (int rc = set_lds(xa_dkv_kernel<T, KS, KT, 4>, lds)) return rc;
            xa_dkv_kernel<T, KS, KT, 4><<<grid, 256, lds, s>>>(t);
        }
        MD_CHECK_LAUNCH("md_cross_attn_bwd: dk, dv");
        if (p.dkv.join) {
            xa_sum_kernel<T, (KS + 1) / 2><<<dim3(t.workers, t.rows / 32), 256, 0, s>>>(t);
            MD_CHECK_LAUNCH("md_cross_attn_bwd: dk, dv sums");
        }
    }
    if constexpr (NP == 3) {
        BeyondArgs b = beyond_args(a, p, sh, ws, (a.dq ? (long long)p.M : 0) + (a.dk ? a.Nk : 0));
        b.g = (const float *)a.g, b.g_sb = a.g_sb, b.g_sn = a.g_sn, b.g_sh = a.g_sh;
        b.gn = (const float *)(ws + p.gn), b.stat = ws + p.stat;
        b.dq = (float *)a.dq, b.dk = (float *)a.dk, b.dv = (float *)a.dv;
        xa_beyond_bwd_kernel<<<(unsigned)p.Z * b.blocks, 256, 0, s>>>(b);
        MD_CHECK_LAUNCH("md_cross_attn_bwd: rows beyond the pieces");
    }
    return MD_OK;
}

#define XA_DISPATCH(what, KSV, CALL)                                     \
    MD_DISPATCH_DTYPE(a->dtype, what, switch (KSV) {                     \
        case 1: rc = CALL<T, 1>(*a, p, sh, w, s); break;                 \
        case 2: rc = CALL<T, 2>(*a, p, sh, w, s); break;                 \
        case 4: rc = CALL<T, 4>(*a, p, sh, w, s); break;                 \
        case 6: rc = CALL<T, 6>(*a, p, sh, w, s); break;                 \
        default: rc = CALL<T, 8>(*a, p, sh, w, s); break;                \
    })

}  // namespace

extern "C" size_t md_attn_desc_bytes(void) { return sizeof(md_attn_desc); }

extern "C" size_t md_cross_attn_ws_bytes(const md_attn_desc *a, int backward) {
    if (!a || check(*a, "md_cross_attn_ws_bytes") || a->B == 0) return 0;
    return make_plan(*a, backward != 0).bytes;
}

extern "C" int md_cross_attn_fwd(const md_attn_desc *a, void *ws, size_t ws_bytes, md_stream_t stream) {
    MD_REQUIRE(a, "md_cross_attn_fwd: null descriptor");
    if (int rc = check(*a, "md_cross_attn_fwd")) return rc;
    if (a->B == 0 || a->Nq == 0) return MD_OK;
    MD_REQUIRE(a->q && a->o && (a->Nk == 0 || (a->k && a->v)), "md_cross_attn_fwd: null pointer");
    const Plan p = make_plan(*a, false);
    MD_REQUIRE(ws_bytes >= p.bytes && (ws || p.bytes == 0), "md_cross_attn_fwd: workspace of %zu bytes, %zu needed", ws ? ws_bytes : (size_t)0, p.bytes);
    MD_REQUIRE(((uintptr_t)ws & 255) == 0, "md_cross_attn_fwd: workspace is not aligned to 256 bytes");
    hipStream_t s = (hipStream_t)stream;
    char *w = (char *)ws;
    Shape sh{};
    int rc = start(*a, p, w, s, sh);
    if (rc) return rc;
    if (p.few) MD_DISPATCH_DTYPE(a->dtype, "md_cross_attn_fwd", rc = run_few<T>(*a, p, sh, w, s));
    else XA_DISPATCH("md_cross_attn_fwd", p.KS, run_fwd);
    return rc;
}

extern "C" int md_cross_attn_bwd(const md_attn_desc *a, void *ws, size_t ws_bytes, md_stream_t stream) {
    MD_REQUIRE(a, "md_cross_attn_bwd: null descriptor");
    if (int rc = check(*a, "md_cross_attn_bwd")) return rc;
    if (a->B == 0) return MD_OK;
    MD_REQUIRE((a->dk == nullptr) == (a->dv == nullptr), "md_cross_attn_bwd: dk and dv come together");
    MD_REQUIRE(a->Nq == 0 || (a->q && a->o && a->g && a->lse), "md_cross_attn_bwd: null pointer");
    MD_REQUIRE(a->Nk == 0 || (a->k && a->v), "md_cross_attn_bwd: null pointer");
    const Plan p = make_plan(*a, true);
    MD_REQUIRE(ws_bytes >= p.bytes && (ws || p.bytes == 0), "md_cross_attn_bwd: workspace of %zu bytes, %zu needed", ws ? ws_bytes : (size_t)0, p.bytes);
    MD_REQUIRE(((uintptr_t)ws & 255) == 0, "md_cross_attn_bwd: workspace is not aligned to 256 bytes");
    hipStream_t s = (hipStream_t)stream;
    char *w = (char *)ws;
    Shape sh{};
    int rc = start(*a, p, w, s, sh);
    if (rc) return rc;
    XA_DISPATCH("md_cross_attn_bwd", p.KS, run_bwd);
    return rc;
}
