// distill_tile.hip -- variants of the pass over the index (distill_tile.h) and the rule that picks one.
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

}  // namespace

bool tile_plan(long long m, int ld, bool bf16, TilePlan* p) {
    *p = TilePlan{-1, 0, 0, 0};
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
