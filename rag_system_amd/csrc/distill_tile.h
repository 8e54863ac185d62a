// distill_tile.h -- the pass over the index of rag_flat_distill_dev, float32 rows.
//
// A workgroup holds WQ x QT queries and streams its share of the rows through LDS, RT rows at a time.  Per tile
//     S^T = X Q^T          (rows x queries)     MFMA 32x32x2 (QT = 32) or 16x16x4 (QT = 16), fp32
//     P^T = exp(S^T - m)   running maximum m and sum l per query
//     O^T += X^T P^T       (columns x queries)
// Writing both products transposed keeps a query in ONE lane of every result (lane & (QT-1)): maximum, sum and
// rescaling are per-lane, and register i of S^T, whose lanes hold rows {r, r + 4, ..} of the query, already is the B
// operand of the second product for exactly those rows -- the A operand takes the same rows of X^T.  P never
// leaves its registers.
// WD waves share a group of QT queries, each with CW of the columns (the row sum O and the queries of 384 columns
// fill a wave's registers); their parts of S^T meet in LDS, added in the same order by each of them.
// Each tile's share of O is summed from zero and then added to O: a sum over a million rows of which one has most of
// the weight would otherwise lose the others (added two at a time, each rounded at the large one's last place).
//
// Rows come by LDS-DMA (16 bytes a lane) into a ring of NB tiles, a tile as blocks of 32 columns: [DP / 32][RT][32].
// One instruction fetches 128 bytes of each of eight rows, so a lane's row and piece are the same in all of them and its
// address is one lane offset plus a uniform one.  The 16-byte pieces of a row's 128 bytes are stored at their place
// xor (row & 7): both the 16-byte reads of S (8 rows, one piece) and the 4-byte reads of O (8 pieces of a row) touch
// every bank once.
#pragma once
#include "common.h"

namespace rag {
namespace distill {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

struct TileCall {
    const void* x;             // n x ld
    const float* norms;        // ||x||^2 per row (L2) or NULL
    const void* q;             // m x d, rows ldq apart
    float* part_ml;            // splits x m x 2: maximum in units of the product (L2: 2 <q,x> - ||x||^2), sum
    float* part_o;             // splits x m x ld
    long long n, m, ldq, rows_per_split;
    int ld, d, splits, q_tiles;
    float k2;                  // beta * log2(e)
};

// Host side (distill_tile.hip): the variant and the number of shares for m queries over rows of ld elements; false where
// no tile kernel serves the row length.
struct TilePlan {
    int kind;        // index of the variant, -1: none
    bool few;        // ... among those for one to four queries (distill_rows.h)
    int rows;        // rows per tile
    int splits, q_tiles;
};
bool tile_plan(long long m, int ld, bool bf16, TilePlan* p);
int tile_launch(const TilePlan& p, const TileCall& c, bool grad, hipStream_t st);

__device__ __forceinline__ void glds16(const void* g, void* l) {
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)g,
                                     (__attribute__((address_space(3))) void*)l, 16, 0, 0);
}
// everything but the N youngest loads has landed, all LDS reads have returned; then the workgroup meets
template <int N>
__device__ __forceinline__ void wait_meet() {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(N) : "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// Which part of the work a workgroup has: the workgroups of one share of the rows (all query tiles) follow each
// other on ONE of the eight dies (ids are dealt out round-robin), so that its L2 serves the rows to all of them.
__device__ __forceinline__ bool place(const TileCall& c, int* split, int* q_tile) {
    const int b = blockIdx.x;
    *split = (b & 7) + 8 * ((b >> 3) / c.q_tiles);
    *q_tile = (b >> 3) % c.q_tiles;
    return *split < c.splits;
}

template <int QT> struct Mma32;
template <> struct Mma32<32> {
    typedef f32x16 acc_t;
    static constexpr int KL = 2, ACC = 16;
    static __device__ __forceinline__ acc_t mma(float a, float b, acc_t c) { return __builtin_amdgcn_mfma_f32_32x32x2f32(a, b, c, 0, 0, 0); }
};
template <> struct Mma32<16> {
    typedef f32x4 acc_t;
    static constexpr int KL = 4, ACC = 4;
    static __device__ __forceinline__ acc_t mma(float a, float b, acc_t c) { return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0); }
};

template <int QT, int WQ, int WD, int CW, int RT, int NB, bool GRAD, bool L2>
__global__ __launch_bounds__(64 * WQ * WD, 1) void tile_f32_kernel(TileCall c) {
    typedef Mma32<QT> M;
    typedef typename M::acc_t acc_t;
    constexpr int KL = M::KL, ACC = M::ACC, NW = WQ * WD, DP = CW * WD;
    constexpr int SUBS = RT / QT;              // MFMA tiles along the rows
    constexpr int NG = CW / (4 * KL);          // 16-byte pieces of a lane along the columns (S)
    constexpr int GP = 8 / KL;                 // ... of which GP within 128 bytes
    constexpr int NCT = CW / QT;               // column tiles (O)
    constexpr int PP = 32 / QT;                // ... of which PP within 128 bytes
    constexpr int LOADS = RT * DP / 256 / NW;  // LDS-DMA instructions (1 KiB) per wave and tile
    static_assert(CW % 32 == 0 && RT % QT == 0 && RT % 8 == 0 && RT * DP % (256 * NW) == 0, "tile shape");
    static_assert((NB - 1) * LOADS < 64, "ring too deep for vmcnt");
    constexpr int TILE = RT * DP;              // floats
    extern __shared__ __align__(16) float lds[];
    float* exch = lds + NB * TILE;             // WD > 1: NW x SUBS x ACC x 64

    int split, q_tile;
    if (!place(c, &split, &q_tile)) return;
    const int lane = threadIdx.x & 63, wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int li = lane & (QT - 1), kl = lane / QT, wd = wid % WD, wq = wid / WD;
    const long long r0 = split * c.rows_per_split, r1 = min(c.n, r0 + c.rows_per_split);
    const int tiles = (int)((r1 - r0 + RT - 1) / RT);
    const long long qi = ((long long)q_tile * WQ + wq) * QT + li;
    const float* x = static_cast<const float*>(c.x);

    // queries: B operand of S^T, pieces kl of every 4 KL columns (a lane without a query takes the first one's: its
    // results are not stored); zero behind the row's end
    f32x4 q[NG];
    {
        const float* qp = static_cast<const float*>(c.q) + (qi < c.m ? qi : 0) * c.ldq;
#pragma unroll
        for (int g = 0; g < NG; ++g)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int col = wd * CW + g * 4 * KL + kl * 4 + e;
                q[g][e] = __uint_as_float(__float_as_uint(qp[min(col, c.d - 1)]) & (col < c.d ? ~0u : 0u));
            }
    }
    // places in a tile, in floats
    int off_s[GP], off_p[PP][4];
#pragma unroll
    for (int g = 0; g < GP; ++g) off_s[g] = wd * CW * RT + li * 32 + (((g * KL + kl) ^ (li & 7)) << 2);
#pragma unroll
    for (int j = 0; j < PP; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i)
            off_p[j][i] = wd * CW * RT + (4 * kl + i) * 32 + (((j * (QT / 4) + (li >> 2)) ^ ((4 * kl + i) & 7)) << 2) + (li & 3);

    // Columns behind the row's end come from its last piece (their queries are zero, their sums are not stored), rows
    // behind the index' end from its last row (they are given no weight).
    const int lr = lane >> 3, lc = ((lane & 7) ^ lr) << 2;
    auto fetch = [&](int t, int b) {
        float* to = lds + b * TILE;
        const long long first = r0 + (long long)t * RT;
#pragma unroll
        for (int a = 0; a < LOADS; ++a) {
            const int at = a * NW + wid, blk = at / (RT / 8), rg = at % (RT / 8) * 8;
            int row = rg + lr, col = blk * 32 + lc;
            if (first + RT > c.n) row = (int)min((long long)row, c.n - 1 - first);
            if (blk * 32 + 32 > c.ld) col = min(col, c.ld - 4);
            glds16(x + first * c.ld + (row * c.ld + col), to + at * 256);
        }
    };
    acc_t o[GRAD ? NCT : 1];
    if (GRAD)
#pragma unroll
        for (int j = 0; j < NCT; ++j)
#pragma unroll
            for (int i = 0; i < ACC; ++i) o[j][i] = 0.f;
    float m = -INFINITY, l = 0.f;

#pragma unroll
    for (int t = 0; t < NB - 1; ++t) fetch(t < tiles ? t : 0, t);
    int slot = 0;                               // t % NB
    for (int t = 0; t < tiles; ++t, slot = slot + 1 < NB ? slot + 1 : 0) {
        float nrm[L2 ? SUBS : 1][L2 ? ACC : 1];
        const long long first = r0 + (long long)t * RT;
        if (NB == 1) {
            wait_meet<0>();                     // nobody reads the last tile any more
            fetch(t, 0);
            wait_meet<0>();
        } else {
            wait_meet<(NB > 1 ? (NB - 2) * LOADS : 0)>();   // tile t is there, nobody reads tile t - 1 any more
        }
        if (L2)
#pragma unroll
            for (int s = 0; s < SUBS; ++s)
#pragma unroll
                for (int i = 0; i < ACC; ++i)
                    nrm[s][i] = c.norms[min(first + s * QT + (QT == 32 ? (i & 3) + 8 * (i >> 2) : i) + 4 * kl, c.n - 1)];
        if (NB > 1) fetch(t + NB - 1 < tiles ? t + NB - 1 : 0, slot > 0 ? slot - 1 : NB - 1);   // (one that nobody reads keeps the count)
        const float* xs = lds + slot * TILE;

        acc_t s[SUBS];
#pragma unroll
        for (int u = 0; u < SUBS; ++u)
#pragma unroll
            for (int i = 0; i < ACC; ++i) s[u][i] = 0.f;
        // (the next step's operands are read in front of a step's products: a wave has its SIMD to itself, nobody
        // else fills the time an LDS read takes; sched_barrier keeps the order)
        f32x4 a[2][SUBS];
        auto read_s = [&](int g, f32x4* to) {
#pragma unroll
            for (int u = 0; u < SUBS; ++u)
                to[u] = *reinterpret_cast<const f32x4*>(xs + u * QT * 32 + off_s[g % GP] + (g / GP) * RT * 32);
        };
        read_s(0, a[0]);
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            if (g + 1 < NG) read_s(g + 1, a[(g + 1) & 1]);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
                for (int u = 0; u < SUBS; ++u) s[u] = M::mma(a[g & 1][u][e], q[g][e], s[u]);
            __builtin_amdgcn_sched_barrier(0);
        }
        float p[SUBS][ACC];
#pragma unroll
        for (int u = 0; u < SUBS; ++u)
#pragma unroll
            for (int i = 0; i < ACC; ++i) p[u][i] = s[u][i];
        if (WD > 1) {
            float* mine = exch + wid * SUBS * ACC * 64;
#pragma unroll
            for (int u = 0; u < SUBS; ++u)
#pragma unroll
                for (int i = 0; i < ACC; i += 4)
                    *reinterpret_cast<f32x4*>(mine + (u * ACC + i) * 64 + lane * 4) = f32x4{p[u][i], p[u][i + 1], p[u][i + 2], p[u][i + 3]};
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            __builtin_amdgcn_s_barrier();
            asm volatile("" ::: "memory");
#pragma unroll
            for (int u = 0; u < SUBS; ++u)
#pragma unroll
                for (int i = 0; i < ACC; i += 4) {
                    f32x4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int w = 0; w < WD; ++w)
                        sum += *reinterpret_cast<const f32x4*>(exch + ((wq * WD + w) * SUBS * ACC + u * ACC + i) * 64 + lane * 4);
#pragma unroll
                    for (int e = 0; e < 4; ++e) p[u][i + e] = sum[e];
                }
        }
        if (L2)
#pragma unroll
            for (int u = 0; u < SUBS; ++u)
#pragma unroll
                for (int i = 0; i < ACC; ++i) p[u][i] = fmaf(2.f, p[u][i], -nrm[u][i]);
        if (first + RT > r1)                    // the last tile: rows behind the share's end
#pragma unroll
            for (int u = 0; u < SUBS; ++u)
#pragma unroll
                for (int i = 0; i < ACC; ++i)
                    if (first + u * QT + (QT == 32 ? (i & 3) + 8 * (i >> 2) : i) + 4 * kl >= r1) p[u][i] = -INFINITY;
        float top = p[0][0];
#pragma unroll
        for (int u = 0; u < SUBS; ++u)
#pragma unroll
            for (int i = 0; i < ACC; ++i) top = fmaxf(top, p[u][i]);
#pragma unroll
        for (int w = QT; w < 64; w *= 2) top = fmaxf(top, __shfl_xor(top, w));
        if (__any(top > m)) {                   // (uniform) seldom, once the first tiles are through
            const float now = fmaxf(m, top);
            const float scale = __builtin_amdgcn_exp2f((m - (now == -INFINITY ? 0.f : now)) * c.k2);
            m = now;
            l *= scale;
            if (GRAD)
#pragma unroll
                for (int j = 0; j < NCT; ++j)
#pragma unroll
                    for (int i = 0; i < ACC; ++i) o[j][i] *= scale;
        }
        const float base = m == -INFINITY ? 0.f : m;
        float sum = 0.f;
#pragma unroll
        for (int u = 0; u < SUBS; ++u)
#pragma unroll
            for (int i = 0; i < ACC; ++i) {
                p[u][i] = __builtin_amdgcn_exp2f((p[u][i] - base) * c.k2);
                sum += p[u][i];
            }
        l += sum;                               // this lane's rows; the lanes of a query are added at the end
        if (!GRAD) continue;
        // a step: four rows of every lane, one column tile; STEPS of them are a column tile
        constexpr int STEPS = SUBS * ACC / 4, AHEAD = QT == 32 ? 1 : 2;
        float b[AHEAD + 1][4];
        auto read_o = [&](int st, float* to) {
            const int j = st / STEPS, u = st % STEPS / (ACC / 4), h = st % (ACC / 4);
#pragma unroll
            for (int i = 0; i < 4; ++i) to[i] = xs[(u * QT + 8 * h) * 32 + off_p[j % PP][i] + (j / PP) * RT * 32];
        };
#pragma unroll
        for (int st = 0; st < AHEAD; ++st) read_o(st, b[st]);
#pragma unroll
        for (int j = 0; j < NCT; ++j) {
            acc_t part;
#pragma unroll
            for (int i = 0; i < ACC; ++i) part[i] = 0.f;
#pragma unroll
            for (int k = 0; k < STEPS; ++k) {
                const int st = j * STEPS + k;
                if (st + AHEAD < NCT * STEPS) read_o(st + AHEAD, b[(st + AHEAD) % (AHEAD + 1)]);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int i = 0; i < 4; ++i) part = M::mma(b[st % (AHEAD + 1)][i], p[k / (ACC / 4)][k % (ACC / 4) * 4 + i], part);
            }
#pragma unroll
            for (int i = 0; i < ACC; ++i) o[j][i] += part[i];
        }
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // no LDS-DMA outlives the workgroup
#pragma unroll
    for (int w = QT; w < 64; w *= 2) l += __shfl_xor(l, w);
    if (qi >= c.m) return;
    const long long at = (long long)split * c.m + qi;
    if (kl == 0 && wd == 0) {
        c.part_ml[2 * at] = m;
        c.part_ml[2 * at + 1] = l;
    }
    if (!GRAD) return;
    float* to = c.part_o + at * c.ld;
#pragma unroll
    for (int j = 0; j < NCT; ++j)
#pragma unroll
        for (int i = 0; i < ACC; i += 4) {
            const int col = wd * CW + j * QT + 8 * (i >> 2) + 4 * kl;
            if (col < c.ld) *reinterpret_cast<f32x4*>(to + col) = f32x4{o[j][i], o[j][i + 1], o[j][i + 2], o[j][i + 3]};
        }
}

}  // namespace distill
}  // namespace rag
