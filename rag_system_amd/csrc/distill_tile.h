// distill_tile.h -- the pass over the index of rag_flat_distill_dev with matrix instructions.
//
// A workgroup holds WQ x 16 queries and streams its share of the rows through LDS, RT rows at a time.  Per tile
//     S^T = X Q^T          (rows x queries)     MFMA 16x16x4 (float32) / 16x16x32 (bfloat16)
//     P^T = exp(S^T - m)   reference m and sum l per query
//     O^T += X^T P^T       (columns x queries)
// Writing both products transposed keeps a query in ONE lane of every result (lane & 15): maximum, sum and weights are
// per-lane, and the registers of S^T already are the B operand of the second product -- register i of a lane group kl holds
// row 4 kl + i of the query, so the A operand takes the same rows of X^T.  P never leaves its registers.  (bfloat16: 32
// rows a product, eight of a lane: four of each half of the tile; X^T comes by the transposing LDS read.  The weights are
// float32: each is the sum of three bfloat16, which holds all 24 bits, and has three products.  Where student and teacher agree,
// sum_j P x and sum_k p x nearly cancel, and fewer bits show: two parts, 2^-17 off, took 1.25 ms for 256 queries x 768, 1M rows,
// against 1.40.)
// WD waves share a group of 16 queries, each with CW of the columns (the row sum O and the queries of 384 columns
// fill half of what a wave has with two on a SIMD); their parts of S^T meet in LDS, added in the same order by each.
// The products add to O a few rows at a time, each rounded at O's last place; a sum over many rows of which one has
// most of the weight would lose the others.  So every WINDOW tiles O is put down: added to the workgroup's part in HBM
// and started again from zero.  (Summing each tile from zero and adding it to O in registers is as exact, but those
// additions hold up the next products: 13.4 against 11.2 ms for 1024 queries x 1M x 384.)
// m is not the maximum but a reference that stays until a logit lies more than 2^LIFT above it: weights up to 2^LIFT and
// their sums lose nothing in float32, and O is never rescaled in its registers -- when the reference does move, O is put
// down first.
//
// Rows come by LDS-DMA (16 bytes a lane) into a ring of NB tiles, a tile as blocks of 128 bytes of each row:
// [blocks][RT][128 bytes].  One instruction fetches 128 bytes of each of eight rows, so a lane's row and piece are the same in
// all of them.  The 16-byte pieces of a row's 128 bytes are stored at their place xor a permutation of (row & 7), so
// that the 16-byte reads of S (8 rows, one piece) and the reads of O (float32: 4 pieces of rows r and r + 4; bfloat16: a pair
// of pieces of eight rows) touch every bank once (counted: no conflicts, in either type).
//
// Measured with the join, loss and gradient, 1M rows.  Up to 16 queries the rows' bytes bound it: 16 x 384 float32 302 us = 5.1 TB/s.
// float32 from 64 queries on, the matrix pipes: 1024 x 384 11.05 ms = 142 TFLOP/s (a large library product: 154), busy for 93 % of the
// time.  bfloat16: 256 x 768 1.40 to 1.45 ms = 560 TFLOP/s of the formula's products, twice that with the two more of the weights'
// parts (a large library product: 1261).  The pipes are busy for 54 % of the time: each group of 16 queries reads every tile from LDS
// for S and again for O, and the weights' parts are made between the two.
#pragma once
#include "common.h"

namespace rag {
namespace distill {

typedef float f32x4 __attribute__((ext_vector_type(4)));

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
    bool bf16;
    int rows;        // rows per tile
    int splits, q_tiles;
};
bool tile_plan(long long m, int ld, bool bf16, bool grad, TilePlan* p);
int tile_launch(const TilePlan& p, const TileCall& c, bool grad, hipStream_t st);

// 16 bytes a lane from `off` bytes behind `base` (uniform) into LDS, lane after lane from `l` (uniform) on.  The buffer form: behind
// a global_load_lds, which may count as an LDS access too, the compiler waits for ALL LDS reads in front of each use.
__device__ __forceinline__ void lds_dma16(const void* base, unsigned bytes, int off, void* l) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(__builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), 0, bytes, 0x00027000),
                                             (__attribute__((address_space(3))) void*)l, 16, off, 0, 0, 0);
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

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

// Eight float32 values as the sums of three bfloat16 each, the largest first: the upper 16 bits, of what that leaves the upper 16
// bits, and the rest, eight bits each, so all three are exact.  (Cut off, not rounded: the largest float32 would round to infinity.)
// INF: infinities too, whose rest is zero.
template <bool INF>
__device__ __forceinline__ void three_parts(const float* v, u32x4* part) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        unsigned h[2][3];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            float rest = v[2 * e + i];
#pragma unroll
            for (int a = 0; a < 3; ++a) {
                h[i][a] = __float_as_uint(rest) & 0xffff0000u;
                const float top = __uint_as_float(h[i][a]);
                rest = INF && a == 0 && rest == top ? 0.f : rest - top;
            }
        }
#pragma unroll
        for (int a = 0; a < 3; ++a) part[a][e] = h[0][a] >> 16 | h[1][a];
    }
}

constexpr int WINDOW = 64;      // tiles
constexpr float LIFT = 40.f;    // powers of two
// One group of queries, three tiles: the variant whose four waves are alone on the CU and bound by HBM.
constexpr bool pipelined(int wq, int wd, int cw, int rt, int nb) { return wq == 1 && nb == 3 && rt == 32 && cw <= 96; }

template <typename T, int WQ, int WD, int CW, int RT, int NB, bool GRAD, bool L2>
__global__ __launch_bounds__(64 * WQ * WD, 1) void tile_kernel(TileCall c) {
    constexpr bool BF = sizeof(T) == 2;
    constexpr int ESZ = sizeof(T), PIECE = 16 / ESZ;      // elements of a 16-byte piece
    constexpr int NW = WQ * WD, DP = CW * WD, BLOCK = RT * 128;      // bytes of a block of columns
    constexpr int SUBS = RT / 16;                         // MFMA tiles along the rows
    constexpr int NG = CW / (4 * PIECE);                  // steps of S: 64 bytes of a row
    constexpr int NCT = CW / 16;                          // column tiles of O
    constexpr int PP = 8 * PIECE / 16;                    // ... of which PP within 128 bytes
    constexpr int TILE = RT * DP * ESZ;                   // bytes
    constexpr int LOADS = TILE / 1024 / NW;               // LDS-DMA instructions per wave and tile
    static_assert(CW % (8 * PIECE) == 0 && RT % (BF ? 32 : 16) == 0 && TILE % (1024 * NW) == 0, "tile shape");
    extern __shared__ __align__(16) char lds[];
    float* exch = reinterpret_cast<float*>(lds + NB * TILE);   // WD > 1: NW x SUBS x 64 x 4

    int split, q_tile;
    if (!place(c, &split, &q_tile)) return;
    const int lane = threadIdx.x & 63, wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int li = lane & 15, kl = lane >> 4, wd = wid % WD, wq = wid / WD;
    const long long r0 = split * c.rows_per_split, r1 = min(c.n, r0 + c.rows_per_split);
    const int tiles = (int)((r1 - r0 + RT - 1) / RT);
    const long long qi = ((long long)q_tile * WQ + wq) * 16 + li;
    const T* x = static_cast<const T*>(c.x);
    // where a row's pieces are: place of piece p of row r = p ^ turn(r)
    auto turn = [](int r) __attribute__((always_inline)) { return BF ? (((r & 3) << 1) | ((r >> 2) & 1)) ^ ((r >> 1) & 2) : r & 7; };

    // queries: B operand of S^T, piece kl of every four (a lane without a query takes the first one's: its results are
    // not stored); zero behind the row's end
    u32x4 q[NG];
    {
        const T* qp = static_cast<const T*>(c.q) + (qi < c.m ? qi : 0) * c.ldq;
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            T v[PIECE];
#pragma unroll
            for (int e = 0; e < PIECE; ++e) {
                const int col = wd * CW + (g * 4 + kl) * PIECE + e;
                v[e] = qp[min(col, c.d - 1)];
            }
            __builtin_memcpy(&q[g], v, 16);
            const int end = c.d - (wd * CW + (g * 4 + kl) * PIECE);      // values of this piece that the row has
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if (BF) q[g][e] &= (2 * e < end ? 0xffffu : 0u) | (2 * e + 1 < end ? 0xffff0000u : 0u);
                else q[g][e] &= e < end ? ~0u : 0u;
            }
        }
    }
    // places in a tile, in bytes
    int off_s[2], off_p[PP][BF ? 1 : 4];
#pragma unroll
    for (int g = 0; g < 2; ++g) off_s[g] = wd * (CW / (8 * PIECE)) * BLOCK + li * 128 + (((g * 4 + kl) ^ turn(li)) << 4);
#pragma unroll
    for (int j = 0; j < PP; ++j)
#pragma unroll
        for (int i = 0; i < (BF ? 1 : 4); ++i) {
            // float32: row 4 kl + i, column li of the tile.  bfloat16: this lane's part of the transposing read, row 4 kl + li / 4,
            // columns li % 4 * 4 and on
            const int row = 4 * kl + (BF ? li >> 2 : i), byte = BF ? (li & 3) * 8 : li * 4;
            off_p[j][i] = wd * (CW / (8 * PIECE)) * BLOCK + row * 128 + (((j * (16 / PIECE) + (byte >> 4)) ^ turn(row)) << 4) + (byte & 15);
        }

    // Columns behind the row's end come from its last piece (their queries are zero, their sums are not stored), rows
    // behind the index' end from its last row (they are given no weight).
    const int lr = lane >> 3, lc = ((lane & 7) ^ turn(lr)) * PIECE;
    auto fetch1 = [&](int t, int b, int a) __attribute__((always_inline)) {   // the a-th of this wave's instructions for tile t, into ring place b
        const long long first = r0 + (long long)t * RT;
        const int at = a * NW + wid, blk = at / (RT / 8), rg = at % (RT / 8) * 8;
        const int rows = (int)min((long long)RT, c.n - first), row = min(rg + lr, rows - 1), col = min(blk * 8 * PIECE + lc, c.ld - PIECE);
        lds_dma16(x + first * c.ld, (unsigned)(rows * c.ld) * ESZ, (row * c.ld + col) * ESZ, lds + b * TILE + at * 1024);
    };
    f32x4 o[GRAD ? NCT : 1];
    if (GRAD)
#pragma unroll
        for (int j = 0; j < NCT; ++j) o[j] = f32x4{0.f, 0.f, 0.f, 0.f};
    float m = -INFINITY, m_next = -INFINITY, l = 0.f;
    bool lifted = false;
    f32x4 s[SUBS];                              // S^T of the newest tile, then its weights
    f32x4 nrm[L2 ? SUBS : 1];

    auto norms = [&](int t) __attribute__((always_inline)) {
        const long long first = r0 + (long long)t * RT;
#pragma unroll
        for (int u = 0; u < SUBS; ++u)
#pragma unroll
            for (int i = 0; i < 4; ++i) nrm[L2 ? u : 0][i] = c.norms[min(first + u * 16 + 4 * kl + i, c.n - 1)];
    };
    // S^T of the tile at xs.  The next step's operands are read in front of a step's products (sched_barrier keeps the order),
    // and the wave's LDS-DMA instructions for tile t are spread over the steps: each holds the wave for 60 to 180 cycles.
    auto product = [&](const char* xs, int t, int b) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < SUBS; ++u) s[u] = f32x4{0.f, 0.f, 0.f, 0.f};
        u32x4 a[2][SUBS];
        auto read = [&](int g, u32x4* to) __attribute__((always_inline)) {
#pragma unroll
            for (int u = 0; u < SUBS; ++u)
                to[u] = *reinterpret_cast<const u32x4*>(xs + off_s[g & 1] + u * 16 * 128 + (g >> 1) * BLOCK);
        };
        read(0, a[0]);
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            if (g + 1 < NG) read(g + 1, a[(g + 1) & 1]);
            __builtin_amdgcn_sched_barrier(0);
            if constexpr (BF) {
#pragma unroll
                for (int u = 0; u < SUBS; ++u)
                    s[u] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a[g & 1][u]), __builtin_bit_cast(bf16x8, q[g]), s[u], 0, 0, 0);
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
#pragma unroll
                    for (int u = 0; u < SUBS; ++u)
                        s[u] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a[g & 1][u][e]), __uint_as_float(q[g][e]), s[u], 0, 0, 0);
            }
            if (NB > 1)
#pragma unroll
                for (int f = g * LOADS / NG; f < (g + 1) * LOADS / NG; ++f) fetch1(t, b, f);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    float* mine = exch + wid * SUBS * 256;
    auto give = [&]() __attribute__((always_inline)) {                         // this wave's part of S^T
#pragma unroll
        for (int u = 0; u < SUBS; ++u) *reinterpret_cast<f32x4*>(mine + u * 256 + lane * 4) = s[u];
    };
    auto take = [&]() __attribute__((always_inline)) {                         // the sum of the WD parts, in the same order in each of the waves
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
#pragma unroll
        for (int u = 0; u < SUBS; ++u) {
            f32x4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int w = 0; w < WD; ++w) sum += *reinterpret_cast<const f32x4*>(exch + ((wq * WD + w) * SUBS + u) * 256 + lane * 4);
            s[u] = sum;
        }
    };
    // The softmax of the newest tile, in pieces that the products of the tile before it can hide: 0 the logits and the lane's
    // maximum, 1 the query's maximum, then a weight of each sub-tile at a time.
    constexpr int PIECES = 2 + 4;
    float top = -INFINITY, base = 0.f, sum = 0.f;
    auto softmax = [&](int t, int piece) __attribute__((always_inline)) {
        if (piece == 0) {
            const int left = (int)min((long long)RT, r1 - (r0 + (long long)t * RT)) - 4 * kl;   // rows behind the share's end
            top = -INFINITY;
#pragma unroll
            for (int u = 0; u < SUBS; ++u)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if (L2) s[u][i] = fmaf(2.f, s[u][i], -nrm[L2 ? u : 0][i]);
                    s[u][i] = u * 16 + i < left ? s[u][i] : -INFINITY;
                    top = fmaxf(top, s[u][i]);
                }
        } else if (piece == 1) {
            top = fmaxf(top, __shfl_xor(top, 16));
            top = fmaxf(top, __shfl_xor(top, 32));
            const bool lift = (top - m) * c.k2 > LIFT;         // (m = -inf: nothing but zeros has been added)
            lifted = lift && m != -INFINITY;
            m_next = lift ? top : m;
            base = m_next == -INFINITY ? 0.f : m_next;
            sum = 0.f;
        } else {
#pragma unroll
            for (int u = 0; u < SUBS; ++u) {
                const float p = __builtin_amdgcn_exp2f((s[u][piece - 2] - base) * c.k2);
                s[u][piece - 2] = p;
                sum += p;
            }
        }
    };
    // O^T += of the tile at xs with the weights p; beside it the softmax of tile t (next).  A step is a column tile and
    // sixteen rows (bfloat16: 32).
    constexpr int STEPS = BF ? SUBS / 2 : SUBS, AHEAD = 2, MID = WD > 1 ? NCT / 2 * STEPS : 0;
    auto add_rows = [&](const char* xs, const f32x4* p, int t, bool next) __attribute__((always_inline)) {
        u32x4 b[AHEAD + 1], part[BF ? STEPS : 1][3];       // bfloat16: the weights' parts, the largest first
        if constexpr (BF) {
#pragma unroll
            for (int k = 0; k < STEPS; ++k) {
                float v[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = p[2 * k + (e >> 2)][e & 3];
                three_parts<false>(v, part[k]);          // (no weight is infinite)
            }
        }
        auto read = [&](int st, u32x4* to) __attribute__((always_inline)) {
            const int j = st / STEPS, k = st % STEPS;
            const char* from = xs + (j / PP) * BLOCK;
            if constexpr (BF) {
                s16x4 v[2];
#pragma unroll
                for (int h = 0; h < 2; ++h)
                    v[h] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                        (__attribute__((address_space(3))) s16x4*)(from + off_p[j % PP][0] + (2 * k + h) * 16 * 128));
                *to = __builtin_bit_cast(u32x4, __builtin_shufflevector(v[0], v[1], 0, 1, 2, 3, 4, 5, 6, 7));
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i) (*to)[i] = *reinterpret_cast<const unsigned*>(from + off_p[j % PP][BF ? 0 : i] + k * 16 * 128);
            }
        };
#pragma unroll
        for (int st = 0; st < AHEAD; ++st) read(st < NCT * STEPS ? st : 0, &b[st]);
#pragma unroll
        for (int st = 0; st < NCT * STEPS; ++st) {
            const int j = st / STEPS, k = st % STEPS;
            if (WD > 1 && st == MID && next) take();
            if (st + AHEAD < NCT * STEPS) read(st + AHEAD, &b[(st + AHEAD) % (AHEAD + 1)]);
            __builtin_amdgcn_sched_barrier(0);
            const u32x4 a = b[st % (AHEAD + 1)];
            if constexpr (BF) {
#pragma unroll
                for (int w = 2; w >= 0; --w)
                    o[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, part[k][w]), o[j], 0, 0, 0);
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i) o[j] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a[i]), p[k][i], o[j], 0, 0, 0);
            }
            if (next && st >= MID && st - MID < PIECES) softmax(t, st - MID);
        }
        if (next)
#pragma unroll
            for (int piece = 0; piece < PIECES; ++piece)
                if (piece >= NCT * STEPS - MID) softmax(t, piece);
    };
    // O into the workgroup's part in HBM, which holds what came before for the reference m_part.
    float m_part = 0.f, l_part = 0.f;
    bool fresh = true;
    const long long at = (long long)split * c.m + qi;
    auto put_down = [&]() __attribute__((always_inline)) {
        const float before = fresh ? 0.f : __builtin_amdgcn_exp2f((m_part - (m == -INFINITY ? 0.f : m)) * c.k2);
        l_part = fmaf(l_part, before, l);
        l = 0.f;
        m_part = m;
        if (GRAD) {
            float* to = c.part_o + at * c.ld;
            int col0 = wd * CW + 4 * kl, end = qi < c.m ? c.ld : 0;
            asm volatile("" : "+v"(col0), "+v"(end));    // (else the addresses are kept in registers over the whole loop)
#pragma unroll
            for (int j = 0; j < NCT; ++j) {
                const int col = col0 + j * 16;
                if (col < end) {
                    f32x4 v = o[j];
                    if (!fresh) v += *reinterpret_cast<const f32x4*>(to + col) * before;
                    *reinterpret_cast<f32x4*>(to + col) = v;
                }
                o[j] = f32x4{0.f, 0.f, 0.f, 0.f};
            }
        }
        fresh = false;
    };
    // between the products of tile t and those of tile t + 1, whose softmax has been computed for m_next
    auto advance = [&](int t) __attribute__((always_inline)) {
        if (__any(lifted) || (t > 0 && t % WINDOW == 0)) put_down();     // (uniform)
        m = m_next;
        l += sum;                               // this lane's rows; the lanes of a query are added at the end
    };

    constexpr bool PIPE = pipelined(WQ, WD, CW, RT, NB) && GRAD;
    if (PIPE) {
        // Few waves on a CU: tile t's products for O run beside the softmax of tile t + 1, whose S came first (three tiles in
        // the ring: t, t + 1, and t + 2 on its way).
#pragma unroll
        for (int a = 0; a < LOADS; ++a) fetch1(0, 0, a);
        wait_meet<0>();
        if (L2) norms(0);
        product(lds, 1 < tiles ? 1 : 0, 1);
        if (WD > 1) {
            give();
            take();
        }
#pragma unroll
        for (int piece = 0; piece < PIECES; ++piece) softmax(0, piece);
        advance(0);
        int slot = 0;                           // t % NB
        for (int t = 0; t < tiles; ++t) {
            const int slot1 = slot + 1 < NB ? slot + 1 : 0, slot2 = slot1 + 1 < NB ? slot1 + 1 : 0;
            f32x4 p[SUBS];
#pragma unroll
            for (int u = 0; u < SUBS; ++u) p[u] = s[u];
            if (t + 1 < tiles) {
                wait_meet<0>();                 // tile t + 1 is there, nobody reads tile t - 1 any more
                if (L2) norms(t + 1);
                product(lds + slot1 * TILE, t + 2 < tiles ? t + 2 : 0, slot2);
                if (WD > 1) give();
                add_rows(lds + slot * TILE, p, t + 1, true);
                advance(t + 1);
            } else {
                add_rows(lds + slot * TILE, p, t, false);
            }
            slot = slot1;
        }
    } else {
        // NB == 2, 3: tiles t and, on its way, t + NB - 1; NB == 1: no room for another
#pragma unroll
        for (int b = 0; b < NB - 1; ++b)
#pragma unroll
            for (int a = 0; a < LOADS; ++a) fetch1(b < tiles ? b : 0, b, a);
        int slot = 0;
        for (int t = 0; t < tiles; ++t) {
            wait_meet<(NB > 1 ? (NB - 2) * LOADS : 0)>();   // NB > 1: tile t is there; nobody reads the tile before any more
            if (NB == 1) {
#pragma unroll
                for (int a = 0; a < LOADS; ++a) fetch1(t, 0, a);
                wait_meet<0>();
            }
            if (L2) norms(t);
            product(lds + slot * TILE, t + NB - 1 < tiles ? t + NB - 1 : 0, slot > 0 ? slot - 1 : NB - 1);
            if (WD > 1) {
                give();
                take();
            }
#pragma unroll
            for (int piece = 0; piece < PIECES; ++piece) softmax(t, piece);
            advance(t);
            if (GRAD) add_rows(lds + slot * TILE, s, t, false);
            slot = slot + 1 < NB ? slot + 1 : 0;
        }
    }
    put_down();
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // no LDS-DMA outlives the workgroup
    l_part += __shfl_xor(l_part, 16);
    l_part += __shfl_xor(l_part, 32);
    if (qi < c.m && kl == 0 && wd == 0) {
        c.part_ml[2 * at] = m_part;
        c.part_ml[2 * at + 1] = l_part;
    }
}

}  // namespace distill
}  // namespace rag
