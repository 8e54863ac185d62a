// distill_tile.hip -- which kernel makes the pass over the index, and in how many shares.
#include "distill_rows.h"
#include "distill_variants.h"

#include <algorithm>
#include <atomic>
#include <cmath>

namespace rag {
namespace distill {

namespace {

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

const Variants& variants(bool bf16, bool grad) { return (bf16 ? VARIANTS_BF16 : VARIANTS_F32)[grad]; }

// Workgroups of a variant that a CU holds (its LDS and registers; asked of the runtime once per variant).
int resident(bool bf16, bool grad, int v) {
    static std::atomic<int> known[2][2][MAX_VARIANTS];
    int n = known[bf16][grad][v];
    if (n == 0) {
        const Variant& a = variants(bf16, grad).all[v];
        const void* fn = reinterpret_cast<const void*>(a.fn[1]);
        if (hipFuncSetAttribute(fn, hipFuncAttributeMaxDynamicSharedMemorySize, a.lds) != hipSuccess ||
            hipOccupancyMaxActiveBlocksPerMultiprocessor(&n, fn, 64 * a.wq * a.wd, a.lds) != hipSuccess || n < 1) {
            (void)hipGetLastError();
            n = 1;
        }
        known[bf16][grad][v] = n;
    }
    return n;
}

// TFLOP/s that a group of 16, 32, 64, 128 queries reaches (1M rows of 384, float32 and bfloat16, the loss alone and with its gradient).
constexpr double RATE[2][2][4] = {{{48, 71, 118, 131}, {80, 113, 129, 143}}, {{91, 170, 430, 640}, {171, 276, 535, 710}}};

}  // namespace

bool tile_plan(long long m, int ld, bool bf16, bool grad, TilePlan* p) {
    *p = TilePlan{-1, false, bf16, 0, 0, 0};
    if (m <= 4)
        for (int v = 0; v < N_FEW; ++v)
            if ((FEW[v].bf16 != 0) == bf16 && FEW[v].lpr * FEW[v].np * (bf16 ? 8 : 4) >= ld) {
                *p = TilePlan{v, true, bf16, 64 / FEW[v].lpr * ROWS_WAVES, num_cus() * 2, 1};
                return true;
            }
    // The variant with the least work for these queries: whole groups of them, whole columns, over the rate its groups reach.
    const Variants& of = variants(bf16, grad);
    double least = 0;
    int best = -1;
    for (int v = 0; v < of.n; ++v) {
        const Variant& a = of.all[v];
        if (a.cw * a.wd < ld) continue;
        const double rate = RATE[bf16][grad][a.wq == 1 ? 0 : a.wq == 2 ? 1 : a.wq == 4 ? 2 : 3];
        const double cost = (double)((m + 16 * a.wq - 1) / (16 * a.wq)) * a.wq * a.cw * a.wd / rate;
        if (best < 0 || cost < least) {
            best = v;
            least = cost;
        }
    }
    if (best < 0) return false;
    const Variant& a = of.all[best];
    p->kind = best;
    p->rows = a.rt;
    p->q_tiles = (int)((m + 16 * a.wq - 1) / (16 * a.wq));
    // as many shares as leave the fewest places for a workgroup idle in the last round, as if a workgroup could have any place; more
    // shares cost their row sums (written once, read once by the join), so the fewest of equals.  (The workgroups of a share stay on
    // one die: fewer than eight shares, from 4096 float32 queries x 384 on, leave dies idle.)
    const int places = num_cus() * resident(bf16, grad, best);
    p->splits = 1;
    double best_time = INFINITY;
    for (int rounds = 1; rounds <= 4; ++rounds) {
        const long long s = std::min<long long>(places, (long long)rounds * places / p->q_tiles);   // the most that these rounds take
        if (s > 0 && (double)rounds / s < best_time - 1e-12) {
            best_time = (double)rounds / s;
            p->splits = (int)s;
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
    const Variant& a = variants(p.bf16, grad).all[p.kind];
    const kernel_t fn = a.fn[c.norms ? 1 : 0];
    if (a.lds > 48 * 1024)
        RAG_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(fn), hipFuncAttributeMaxDynamicSharedMemorySize, a.lds));
    const unsigned groups = (unsigned)((c.splits + 7) / 8 * 8) * (unsigned)c.q_tiles;
    fn<<<groups, 64 * a.wq * a.wd, a.lds, st>>>(c);
    RAG_HIP(hipGetLastError());
    return RAG_OK;
}

}  // namespace distill
}  // namespace rag
