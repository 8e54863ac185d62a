// distill_rows.h -- the pass over the index of rag_flat_distill_dev for one to four queries.
//
// One query needs 4 d flops for the d elements of a row: nothing but the rows' bytes counts (1M x 384 float32: 1.54 GB).  So no
// LDS, no barrier and no matrix tile: LPR lanes hold a row in registers (NP pieces of 16 bytes each, the next rows on
// their way while these are used), multiply it with the queries' registers, add the LPR parts with DPP, and put the row
// straight into their own columns of the row sum.  Every group of LPR lanes keeps its own maximum, sum and row sum
// (rows of one group: some hundred, so no sum is long); they are joined once, at the end.
// Measured, 1 query, 1M x 384 float32: 229 us = 6.7 TB/s, 241 with the join (the search's stream of the same bytes: 7.2 TB/s).
#pragma once
#include "distill_tile.h"

namespace rag {
namespace distill {

__device__ __forceinline__ float bf_to_f(unsigned short v) { return __uint_as_float((unsigned)v << 16); }

template <typename T> struct RowPiece;
template <> struct RowPiece<float> {
    static constexpr int E = 4;
    typedef f32x4 raw;
    static __device__ __forceinline__ void widen(const raw& r, float* v) {
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = r[e];
    }
};
template <> struct RowPiece<unsigned short> {
    static constexpr int E = 8;
    typedef unsigned raw __attribute__((ext_vector_type(4)));
    static __device__ __forceinline__ void widen(const raw& r, float* v) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            v[2 * e] = __uint_as_float(r[e] << 16);
            v[2 * e + 1] = __uint_as_float(r[e] & 0xffff0000u);
        }
    }
};
__device__ __forceinline__ float query_at(const float* q, int j) { return q[j]; }
__device__ __forceinline__ float query_at(const unsigned short* q, int j) { return bf_to_f(q[j]); }

template <int N>
__device__ __forceinline__ float rotate_add(float v) {   // v + v of the lane N back in its group of 16
    return v + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x120 + N, 0xf, 0xf, false));
}
// Sum over groups of LPR lanes, the same bits in each of them (a + b on one side is b + a on the other).
template <int LPR>
__device__ __forceinline__ float group_sum(float v) {
    v = rotate_add<8>(v);
    v = rotate_add<4>(v);
    v = rotate_add<2>(v);
    v = rotate_add<1>(v);
    if (LPR >= 32) {
        const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    }
    return v;
}

constexpr int ROWS_WAVES = 8;

template <typename T, int LPR, int NP, int MQ, bool GRAD, bool L2>
__global__ __launch_bounds__(64 * ROWS_WAVES) void rows_kernel(TileCall c) {
    typedef RowPiece<T> P;
    typedef typename P::raw raw;
    constexpr int E = P::E, RPW = 64 / LPR, STEP = RPW * ROWS_WAVES;
    extern __shared__ __align__(16) float lds[];   // GRAD: ROWS_WAVES x ld
    __shared__ float ml[ROWS_WAVES][MQ][2];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, grp = lane / LPR, li = lane % LPR;
    const long long r0 = (long long)blockIdx.x * c.rows_per_split, r1 = min(c.n, r0 + c.rows_per_split);
    const T* x = static_cast<const T*>(c.x);

    float q[MQ][NP * E];
    bool mine[NP];                                  // pieces that the row has
    int col[NP];
#pragma unroll
    for (int i = 0; i < NP; ++i) {
        col[i] = (li + LPR * i) * E;
        mine[i] = col[i] < c.ld;
        if (!mine[i]) col[i] = c.ld - E;            // (its last piece again, with zero queries)
    }
#pragma unroll
    for (int a = 0; a < MQ; ++a) {
        const T* qp = static_cast<const T*>(c.q) + min((long long)a, c.m - 1) * c.ldq;
#pragma unroll
        for (int i = 0; i < NP; ++i)
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const float v = query_at(qp, min(col[i] + e, c.d - 1));
                q[a][i * E + e] = __uint_as_float(__float_as_uint(v) & (mine[i] && col[i] + e < c.d ? ~0u : 0u));
            }
    }
    float m[MQ], l[MQ], o[MQ][GRAD ? NP * E : 1];
#pragma unroll
    for (int a = 0; a < MQ; ++a) {
        m[a] = -INFINITY;
        l[a] = 0.f;
#pragma unroll
        for (int j = 0; j < (GRAD ? NP * E : 1); ++j) o[a][j] = 0.f;
    }
    auto fetch = [&](long long r, raw* to, float* norm) {
        const long long at = min(r + wave * RPW + grp, r1 - 1);
#pragma unroll
        for (int i = 0; i < NP; ++i)
            to[i] = __builtin_nontemporal_load(reinterpret_cast<const raw*>(x + at * c.ld + col[i]));
        if (L2) *norm = c.norms[at];
    };
    auto use = [&](long long r, const raw* from, float norm) {
        float v[NP * E];
#pragma unroll
        for (int i = 0; i < NP; ++i) P::widen(from[i], v + i * E);
        const bool real = r + wave * RPW + grp < r1;
        float s[MQ], top = 0.f;
#pragma unroll
        for (int a = 0; a < MQ; ++a) {
            float part[2] = {0.f, 0.f};
#pragma unroll
            for (int j = 0; j < NP * E; ++j) part[j & 1] = fmaf(q[a][j], v[j], part[j & 1]);
            s[a] = group_sum<LPR>(part[0] + part[1]);
            if (L2) s[a] = fmaf(2.f, s[a], -norm);
            s[a] = real ? s[a] : -INFINITY;
            top = s[a] > m[a] ? 1.f : top;
        }
        if (__any(top != 0.f)) {
#pragma unroll
            for (int a = 0; a < MQ; ++a) {
                const float now = fmaxf(m[a], s[a]);
                const float scale = __builtin_amdgcn_exp2f((m[a] - (now == -INFINITY ? 0.f : now)) * c.k2);
                m[a] = now;
                l[a] *= scale;
                if (GRAD)
#pragma unroll
                    for (int j = 0; j < NP * E; ++j) o[a][j] *= scale;
            }
        }
#pragma unroll
        for (int a = 0; a < MQ; ++a) {
            const float p = __builtin_amdgcn_exp2f((s[a] - (m[a] == -INFINITY ? 0.f : m[a])) * c.k2);
            l[a] += p;
            if (GRAD)
#pragma unroll
                for (int j = 0; j < NP * E; ++j) o[a][j] = fmaf(p, v[j], o[a][j]);
        }
    };
    raw buf[2][NP];
    float norm[2] = {0.f, 0.f};
    fetch(r0, buf[0], &norm[0]);
    for (long long r = r0; r < r1; r += 2 * STEP) {     // (a step behind the end has no real row)
        fetch(r + STEP, buf[1], &norm[1]);
        use(r, buf[0], norm[0]);
        fetch(r + 2 * STEP, buf[0], &norm[0]);
        use(r + STEP, buf[1], norm[1]);
    }
    // join the groups of a wave, then the waves
#pragma unroll
    for (int a = 0; a < MQ; ++a) {
#pragma unroll
        for (int w = LPR; w < 64; w *= 2) {
            const float m2 = __shfl_xor(m[a], w), now = fmaxf(m[a], m2), base = now == -INFINITY ? 0.f : now;
            const float f1 = __builtin_amdgcn_exp2f((m[a] - base) * c.k2), f2 = __builtin_amdgcn_exp2f((m2 - base) * c.k2);
            l[a] = l[a] * f1 + __shfl_xor(l[a], w) * f2;
            m[a] = now;
            if (GRAD)
#pragma unroll
                for (int j = 0; j < NP * E; ++j) o[a][j] = o[a][j] * f1 + __shfl_xor(o[a][j], w) * f2;
        }
        if (lane == 0) {
            ml[wave][a][0] = m[a];
            ml[wave][a][1] = l[a];
        }
    }
    __syncthreads();
#pragma unroll
    for (int a = 0; a < MQ; ++a) {
        if (a >= c.m) break;
        float now = -INFINITY, f[ROWS_WAVES], sum = 0.f;
#pragma unroll
        for (int w = 0; w < ROWS_WAVES; ++w) now = fmaxf(now, ml[w][a][0]);
        const float base = now == -INFINITY ? 0.f : now;
#pragma unroll
        for (int w = 0; w < ROWS_WAVES; ++w) {
            f[w] = __builtin_amdgcn_exp2f((ml[w][a][0] - base) * c.k2);
            sum = fmaf(ml[w][a][1], f[w], sum);
        }
        const long long at = (long long)blockIdx.x * c.m + a;
        if (threadIdx.x == 0) {
            c.part_ml[2 * at] = now;
            c.part_ml[2 * at + 1] = sum;
        }
        if (!GRAD) continue;
        if (a > 0) __syncthreads();
        if (grp == 0)
#pragma unroll
            for (int i = 0; i < NP; ++i)
                if (mine[i])
#pragma unroll
                    for (int e = 0; e < E; ++e) lds[wave * c.ld + col[i] + e] = o[a][i * E + e];
        __syncthreads();
        for (int j = threadIdx.x; j < c.ld; j += 64 * ROWS_WAVES) {
            float t = 0.f;
#pragma unroll
            for (int w = 0; w < ROWS_WAVES; ++w) t = fmaf(lds[w * c.ld + j], f[w], t);
            c.part_o[at * c.ld + j] = t;
        }
    }
}

}  // namespace distill
}  // namespace rag
