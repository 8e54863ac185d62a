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
// The products add to O two or four rows at a time, each rounded at O's last place; a sum over many rows of which one has
// most of the weight would lose the others.  So every WINDOW tiles O is put down: added to the workgroup's part in HBM
// and started again from zero.  (Summing each tile from zero and adding it to O in registers is as exact, but those
// additions hold up the next products.)
// m is not the maximum but a reference that stays until a logit lies more than 2^LIFT above it: weights up to 2^LIFT and
// their sums lose nothing in float32, and O, which fills the accumulation registers, is never rescaled there -- when the
// reference does move, O is put down first.
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

constexpr int WINDOW = 64;      // tiles
constexpr float LIFT = 40.f;    // powers of two

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
    auto fetch1 = [&](int t, int b, int a) __attribute__((always_inline)) {    // the a-th of this wave's instructions for tile t, into ring place b
        const long long first = r0 + (long long)t * RT;
        const int at = a * NW + wid, blk = at / (RT / 8), rg = at % (RT / 8) * 8;
        const int rows = (int)min((long long)RT, c.n - first), row = min(rg + lr, rows - 1), col = min(blk * 32 + lc, c.ld - 4);
        lds_dma16(x + first * c.ld, (unsigned)(rows * c.ld) * 4, (row * c.ld + col) * 4, lds + b * TILE + at * 256);
    };
    acc_t o[GRAD ? NCT : 1];
    if (GRAD)
#pragma unroll
        for (int j = 0; j < NCT; ++j)
#pragma unroll
            for (int i = 0; i < ACC; ++i) o[j][i] = 0.f;
    float m = -INFINITY, m_next = -INFINITY, l = 0.f;
    bool lifted = false;
    acc_t s[SUBS];                              // S^T of the newest tile, then its weights
    float nrm[L2 ? SUBS : 1][L2 ? ACC : 1];

    auto norms = [&](int t) __attribute__((always_inline)) {
        const long long first = r0 + (long long)t * RT;
#pragma unroll
        for (int u = 0; u < SUBS; ++u)
#pragma unroll
            for (int i = 0; i < ACC; ++i)
                nrm[L2 ? u : 0][L2 ? i : 0] = c.norms[min(first + u * QT + 8 * (i >> 2) + (i & 3) + 4 * kl, c.n - 1)];
    };
    // S^T of the tile at xs.  The next step's operands are read in front of a step's products (a wave has its SIMD to itself:
    // nobody else fills the time an LDS read takes; sched_barrier keeps the order), and the wave's LDS-DMA instructions for
    // tile t are spread over the steps: each holds the wave for 60 to 180 cycles.
    auto product = [&](const float* xs, int t, int b) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < SUBS; ++u)
#pragma unroll
            for (int i = 0; i < ACC; ++i) s[u][i] = 0.f;
        f32x4 a[2][SUBS];
        auto read = [&](int g, f32x4* to) __attribute__((always_inline)) {
#pragma unroll
            for (int u = 0; u < SUBS; ++u)
                to[u] = *reinterpret_cast<const f32x4*>(xs + u * QT * 32 + off_s[g % GP] + (g / GP) * RT * 32);
        };
        read(0, a[0]);
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            if (g + 1 < NG) read(g + 1, a[(g + 1) & 1]);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
                for (int u = 0; u < SUBS; ++u) s[u] = M::mma(a[g & 1][u][e], q[g][e], s[u]);
            if (NB > 1)
#pragma unroll
                for (int f = g * LOADS / NG; f < (g + 1) * LOADS / NG; ++f) fetch1(t, b, f);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    float* mine = exch + wid * SUBS * ACC * 64;
    auto give = [&]() __attribute__((always_inline)) {                         // this wave's part of S^T
#pragma unroll
        for (int u = 0; u < SUBS; ++u)
#pragma unroll
            for (int i = 0; i < ACC; i += 4)
                *reinterpret_cast<f32x4*>(mine + (u * ACC + i) * 64 + lane * 4) = f32x4{s[u][i], s[u][i + 1], s[u][i + 2], s[u][i + 3]};
    };
    auto take = [&]() __attribute__((always_inline)) {                         // the sum of the WD parts, in the same order in each of the waves
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
                for (int e = 0; e < 4; ++e) s[u][i + e] = sum[e];
            }
    };
    // The softmax of the newest tile, in pieces that the products of the tile before it can hide: 0 the logits and the lane's
    // maximum, 1 the query's maximum, then a weight of each sub-tile at a time.
    constexpr int PIECES = 2 + ACC;
    float top = -INFINITY, base = 0.f, sum = 0.f;
    auto softmax = [&](int t, int piece) __attribute__((always_inline)) {
        if (piece == 0) {
            const int left = (int)min((long long)RT, r1 - (r0 + (long long)t * RT)) - 4 * kl;   // rows behind the share's end
            top = -INFINITY;
#pragma unroll
            for (int u = 0; u < SUBS; ++u)
#pragma unroll
                for (int i = 0; i < ACC; ++i) {
                    if (L2) s[u][i] = fmaf(2.f, s[u][i], -nrm[L2 ? u : 0][L2 ? i : 0]);
                    s[u][i] = u * QT + 8 * (i >> 2) + (i & 3) < left ? s[u][i] : -INFINITY;
                    top = fmaxf(top, s[u][i]);
                }
        } else if (piece == 1) {
#pragma unroll
            for (int w = QT; w < 64; w *= 2) top = fmaxf(top, __shfl_xor(top, w));
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
    // O^T += of the tile at xs with the weights p; beside it the softmax of tile t (next).  A step is four rows of every
    // lane and one column tile.
    constexpr int STEPS = SUBS * ACC / 4, AHEAD = QT == 32 ? 1 : 2, MID = WD > 1 ? NCT / 2 * STEPS : 0;
    auto add_rows = [&](const float* xs, const acc_t* p, int t, bool next) __attribute__((always_inline)) {
        float b[AHEAD + 1][4];
        auto read = [&](int st, float* to) __attribute__((always_inline)) {
            const int j = st / STEPS, u = st % STEPS / (ACC / 4), h = st % (ACC / 4);
#pragma unroll
            for (int i = 0; i < 4; ++i) to[i] = xs[(u * QT + 8 * h) * 32 + off_p[j % PP][i] + (j / PP) * RT * 32];
        };
#pragma unroll
        for (int st = 0; st < AHEAD; ++st) read(st, b[st]);
#pragma unroll
        for (int st = 0; st < NCT * STEPS; ++st) {
            const int j = st / STEPS, k = st % STEPS;
            if (WD > 1 && st == MID && next) take();
            if (st + AHEAD < NCT * STEPS) read(st + AHEAD, b[(st + AHEAD) % (AHEAD + 1)]);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int i = 0; i < 4; ++i) o[j] = M::mma(b[st % (AHEAD + 1)][i], p[k / (ACC / 4)][k % (ACC / 4) * 4 + i], o[j]);
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
            asm volatile("" : "+v"(col0), "+v"(end));    // (else 48 addresses are kept in registers over the whole loop)
#pragma unroll
            for (int j = 0; j < NCT; ++j)
#pragma unroll
                for (int i = 0; i < ACC; i += 4) {
                    const int col = col0 + j * QT + 8 * (i >> 2);
                    if (col < end) {
                        f32x4 v = {o[j][i], o[j][i + 1], o[j][i + 2], o[j][i + 3]};
                        if (!fresh) v += *reinterpret_cast<const f32x4*>(to + col) * before;
                        *reinterpret_cast<f32x4*>(to + col) = v;
                    }
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[j][i + e] = 0.f;
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

    constexpr bool PIPE = NB == 3 && GRAD && QT * CW <= 32 * 256;
    if (PIPE) {
        // Tile t's products for O run beside the softmax of tile t + 1, whose S came first: three tiles in the ring (t, t + 1,
        // and t + 2 on its way).
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
            acc_t p[SUBS];
#pragma unroll
            for (int u = 0; u < SUBS; ++u) p[u] = s[u];
            const bool more = t + 1 < tiles;
            if (more) {
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
        int slot = 0;
        if (NB > 1)
#pragma unroll
            for (int a = 0; a < LOADS; ++a) fetch1(0, 0, a);
        for (int t = 0; t < tiles; ++t) {
            wait_meet<0>();                     // NB > 1: tile t is there; nobody reads the tile before any more
            if (NB == 1) {
#pragma unroll
                for (int a = 0; a < LOADS; ++a) fetch1(t, 0, a);
                wait_meet<0>();
            }
            if (L2) norms(t);
            const int next = NB > 1 && slot + 1 < NB ? slot + 1 : 0;
            product(lds + slot * TILE, t + 1 < tiles ? t + 1 : 0, next);
            if (WD > 1) {
                give();
                take();
            }
#pragma unroll
            for (int piece = 0; piece < PIECES; ++piece) softmax(t, piece);
            advance(t);
            if (GRAD) add_rows(lds + slot * TILE, s, t, false);
            slot = next;
        }
    }
    put_down();
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // no LDS-DMA outlives the workgroup
#pragma unroll
    for (int w = QT; w < 64; w *= 2) l_part += __shfl_xor(l_part, w);
    if (qi < c.m && kl == 0 && wd == 0) {
        c.part_ml[2 * at] = m_part;
        c.part_ml[2 * at + 1] = l_part;
    }
}

}  // namespace distill
}  // namespace rag
