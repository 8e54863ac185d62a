// distill_tile.hip -- variants of the pass over the index (distill_tile.h) and the rule that picks one.
#include "distill_rows.h"
#include "distill_tile.h"

#include <algorithm>

namespace rag {
namespace distill {

namespace {

typedef void (*kernel_t)(TileCall);
constexpr int LDS_MAX = 160 * 1024;

struct Variant {
    int qt, wq, wd, cw, rt, lds;
    kernel_t fn[2][2];   // [grad][l2]
};

constexpr int exch_bytes(int qt, int wq, int wd, int rt) {
    return wd > 1 ? wq * wd * (rt / qt) * (qt == 32 ? 16 : 4) * 256 : 0;
}
// tiles of the ring: three where they fit, else what does
constexpr int ring(int qt, int wq, int wd, int cw, int rt, int esz) {
    return std::min(3, (LDS_MAX - exch_bytes(qt, wq, wd, rt)) / (rt * cw * wd * esz));
}

template <int QT, int WQ, int WD, int CW, int RT>
Variant f32_variant() {
    constexpr int NB = ring(QT, WQ, WD, CW, RT, 4);
    static_assert(NB >= 1, "tile does not fit");
    return Variant{QT, WQ, WD, CW, RT, NB * RT * CW * WD * 4 + exch_bytes(QT, WQ, WD, RT),
                   {{tile_f32_kernel<QT, WQ, WD, CW, RT, NB, false, false>, tile_f32_kernel<QT, WQ, WD, CW, RT, NB, false, true>},
                    {tile_f32_kernel<QT, WQ, WD, CW, RT, NB, true, false>, tile_f32_kernel<QT, WQ, WD, CW, RT, NB, true, true>}}};
}

#define RAG_CWS(X, QT, WQ, WD, RT) X(QT, WQ, WD, 32, RT), X(QT, WQ, WD, 64, RT), X(QT, WQ, WD, 96, RT), X(QT, WQ, WD, 128, RT), \
    X(QT, WQ, WD, 192, RT), X(QT, WQ, WD, 256, RT)
#define RAG_F32(QT, WQ, WD, CW, RT) f32_variant<QT, WQ, WD, CW, RT>()

const Variant VARIANTS[] = {
    // up to 16 queries: bound by the rows' bytes
    RAG_CWS(RAG_F32, 16, 1, 4, 32), RAG_F32(16, 1, 4, 384, 16),
    // up to 32, 64 and more queries
    RAG_CWS(RAG_F32, 32, 1, 4, 32),
    RAG_CWS(RAG_F32, 32, 2, 2, 32), RAG_F32(32, 2, 2, 384, 32),
    RAG_CWS(RAG_F32, 32, 4, 1, 32), RAG_F32(32, 4, 1, 384, 32),
};
constexpr int N_VARIANTS = sizeof VARIANTS / sizeof VARIANTS[0];

// One to four queries: [queries: 1, 2, 4][grad][l2]
struct Few {
    int bf16, lpr, np;
    kernel_t fn[3][2][2];
};
template <typename T, int LPR, int NP, int MQ>
void few_fn(kernel_t (*fn)[2]) {
    fn[0][0] = rows_kernel<T, LPR, NP, MQ, false, false>;
    fn[0][1] = rows_kernel<T, LPR, NP, MQ, false, true>;
    fn[1][0] = rows_kernel<T, LPR, NP, MQ, true, false>;
    fn[1][1] = rows_kernel<T, LPR, NP, MQ, true, true>;
}
template <typename T, int LPR, int NP>
Few few() {
    Few f{sizeof(T) == 2, LPR, NP, {}};
    few_fn<T, LPR, NP, 1>(f.fn[0]);
    few_fn<T, LPR, NP, 2>(f.fn[1]);
    few_fn<T, LPR, NP, 4>(f.fn[2]);
    return f;
}
// in order of the row length they serve: LPR x NP pieces of 16 bytes
const Few FEW[] = {
    few<float, 16, 1>(), few<float, 16, 2>(), few<float, 32, 2>(), few<float, 32, 3>(), few<float, 32, 4>(), few<float, 32, 6>(),
    few<float, 32, 8>(),
    few<unsigned short, 16, 1>(), few<unsigned short, 16, 2>(), few<unsigned short, 32, 2>(), few<unsigned short, 32, 3>(),
    few<unsigned short, 32, 4>(),
};
constexpr int N_FEW = sizeof FEW / sizeof FEW[0];

}  // namespace

bool tile_plan(long long m, int ld, bool bf16, TilePlan* p) {
    *p = TilePlan{-1, false, 0, 0, 0};
    if (m <= 4)
        for (int v = 0; v < N_FEW; ++v)
            if ((FEW[v].bf16 != 0) == bf16 && FEW[v].lpr * FEW[v].np * (bf16 ? 8 : 4) >= ld) {
                *p = TilePlan{v, true, 64 / FEW[v].lpr * ROWS_WAVES, num_cus() * 4, 1};
                return true;
            }
    if (bf16) return false;
    const int most = m <= 16 ? 16 : m <= 32 ? 32 : m <= 64 ? 64 : 128;      // queries of a workgroup that are of use
    int best = -1;
    for (int v = 0; v < N_VARIANTS; ++v) {
        const Variant& a = VARIANTS[v];
        if (a.cw * a.wd < ld || a.qt * a.wq > most) continue;
        if (best >= 0) {
            const Variant& b = VARIANTS[best];
            if (a.qt * a.wq < b.qt * b.wq || (a.qt * a.wq == b.qt * b.wq && a.cw * a.wd >= b.cw * b.wd)) continue;
        }
        best = v;
    }
    if (best < 0) return false;
    const Variant& a = VARIANTS[best];
    p->kind = best;
    p->rows = a.rt;
    p->q_tiles = (int)((m + a.qt * a.wq - 1) / (a.qt * a.wq));
    // one workgroup fills a CU: as many shares as leave the fewest CUs idle in the last round; more shares cost
    // their row sums (written once, read once by the join), so the first of equals is taken
    const int cus = num_cus();
    double best_time = 0;
    for (int s = 1; s <= cus; ++s) {
        const long long groups = (long long)s * p->q_tiles, rounds = (groups + cus - 1) / cus;
        if (groups > 4LL * cus && s > 1) break;
        const double time = (double)rounds / s;
        if (p->splits == 0 || time < best_time - 1e-12) {
            best_time = time;
            p->splits = s;
        }
    }
    return true;
}

int tile_launch(const TilePlan& p, const TileCall& c, bool grad, hipStream_t st) {
    if (p.few) {
        const kernel_t fn = FEW[p.kind].fn[c.m == 1 ? 0 : c.m == 2 ? 1 : 2][grad ? 1 : 0][c.norms ? 1 : 0];
        fn<<<(unsigned)c.splits, 64 * ROWS_WAVES, grad ? (size_t)ROWS_WAVES * c.ld * sizeof(float) : 0, st>>>(c);
        RAG_HIP(hipGetLastError());
        return RAG_OK;
    }
    const Variant& a = VARIANTS[p.kind];
    kernel_t fn = a.fn[grad ? 1 : 0][c.norms ? 1 : 0];
    if (a.lds > 48 * 1024)
        RAG_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(fn), hipFuncAttributeMaxDynamicSharedMemorySize, a.lds));
    const unsigned groups = (unsigned)((c.splits + 7) / 8 * 8) * (unsigned)c.q_tiles;
    fn<<<groups, 64 * a.wq * a.wd, a.lds, st>>>(c);
    RAG_HIP(hipGetLastError());
    return RAG_OK;
}

}  // namespace distill
}  // namespace rag
