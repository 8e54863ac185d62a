// distill_variants.h -- the instances of tile_kernel (distill_tile.h) for one storage type (distill_tile_f32.hip, _bf16.hip).
#pragma once
#include "distill_tile.h"

#include <algorithm>

namespace rag {
namespace distill {

typedef void (*kernel_t)(TileCall);
struct Variant {
    int wq, wd, cw, rt, lds;
    kernel_t fn[2];   // [l2]
};
struct Variants {
    const Variant* all;
    int n;
};
extern const Variants VARIANTS_F32[2], VARIANTS_BF16[2];   // [grad]
constexpr int MAX_VARIANTS = 64;      // of a type and form
template <int N>
constexpr Variants list_of(const Variant (&all)[N]) {
    static_assert(N <= MAX_VARIANTS, "what is known of each variant (distill_tile.hip) has no more places");
    return Variants{all, N};
}

constexpr int LDS_MAX = 160 * 1024;
constexpr int exch_bytes(int wq, int wd, int rt) { return wd > 1 ? wq * wd * (rt / 16) * 1024 : 0; }
// tiles of the ring: three where they fit, else what does
constexpr int ring(int wq, int wd, int cw, int rt, int esz) {
    return std::min(3, (LDS_MAX - exch_bytes(wq, wd, rt)) / (rt * cw * wd * esz));
}

template <typename T, bool GRAD, int WQ, int WD, int CW, int RT>
Variant variant() {
    constexpr int E = sizeof(T), NB = ring(WQ, WD, CW, RT, E);
    static_assert(NB >= 1, "tile does not fit");
    return Variant{WQ, WD, CW, RT, NB * RT * CW * WD * E + exch_bytes(WQ, WD, RT),
                   {tile_kernel<T, WQ, WD, CW, RT, NB, GRAD, false>, tile_kernel<T, WQ, WD, CW, RT, NB, GRAD, true>}};
}
template <typename T, int WQ, int WD, int CW, int RT>
Variant grad() { return variant<T, true, WQ, WD, CW, RT>(); }
template <typename T, int WQ, int WD, int CW, int RT>
Variant loss() { return variant<T, false, WQ, WD, CW, RT>(); }

}  // namespace distill
}  // namespace rag
