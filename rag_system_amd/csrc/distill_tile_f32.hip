// distill_tile_f32.hip -- tile_kernel for float32 rows.
#include "distill_variants.h"

namespace rag {
namespace distill {

namespace {
typedef float T;
const Variant GRAD[] = {
    // up to 16 queries, bound by the rows' bytes
    grad<T, 1, 4, 32, 32>(), grad<T, 1, 4, 64, 32>(), grad<T, 1, 4, 96, 32>(), grad<T, 1, 4, 128, 16>(),
    grad<T, 1, 4, 192, 16>(), grad<T, 1, 4, 256, 16>(), grad<T, 1, 4, 384, 16>(),
    // 32 at a time
    grad<T, 2, 2, 32, 16>(), grad<T, 2, 2, 64, 16>(), grad<T, 2, 2, 96, 16>(), grad<T, 2, 2, 128, 16>(),
    grad<T, 2, 2, 192, 16>(), grad<T, 2, 4, 128, 16>(), grad<T, 2, 4, 192, 16>(), grad<T, 2, 4, 256, 16>(),
    grad<T, 2, 4, 384, 16>(),
    // 64 at a time
    grad<T, 4, 2, 32, 32>(), grad<T, 4, 2, 64, 32>(), grad<T, 4, 2, 96, 32>(), grad<T, 4, 2, 128, 32>(),
    grad<T, 4, 2, 192, 32>(), grad<T, 4, 2, 256, 16>(), grad<T, 4, 2, 384, 16>(),
    // 128 at a time
    grad<T, 8, 1, 32, 64>(), grad<T, 8, 1, 64, 32>(), grad<T, 8, 1, 96, 64>(), grad<T, 8, 1, 128, 32>(),
    grad<T, 8, 1, 192, 32>(), grad<T, 8, 1, 256, 32>(), grad<T, 8, 1, 384, 32>(),
};
// The loss alone needs no row sum: without O a wave holds its queries' whole rows, and nothing is exchanged between waves (37
// queries x 100, 200k rows, L2: 52 us with two waves to a query, 42 with one; 64 x 384, 1M rows: 499, 443).
const Variant LOSS[] = {
    loss<T, 1, 1, 32, 16>(), loss<T, 1, 1, 64, 16>(), loss<T, 1, 1, 96, 16>(), loss<T, 1, 1, 128, 16>(),
    loss<T, 1, 1, 192, 16>(), loss<T, 1, 1, 256, 16>(), loss<T, 1, 1, 384, 16>(), loss<T, 1, 4, 128, 16>(), loss<T, 1, 4, 192, 16>(),
    loss<T, 1, 4, 256, 16>(), loss<T, 1, 4, 384, 16>(),
    loss<T, 2, 2, 32, 16>(), loss<T, 2, 2, 64, 16>(), loss<T, 2, 2, 96, 16>(), loss<T, 2, 2, 128, 16>(),
    loss<T, 2, 2, 192, 16>(), loss<T, 2, 4, 128, 16>(), loss<T, 2, 4, 192, 16>(), loss<T, 2, 4, 256, 16>(),
    loss<T, 2, 4, 384, 16>(),
    loss<T, 4, 1, 32, 32>(), loss<T, 4, 1, 64, 16>(), loss<T, 4, 1, 96, 32>(), loss<T, 4, 1, 128, 16>(),
    loss<T, 4, 1, 192, 16>(), loss<T, 4, 1, 256, 16>(), loss<T, 4, 1, 384, 16>(), loss<T, 4, 1, 512, 16>(), loss<T, 4, 1, 768, 16>(),
    loss<T, 8, 1, 64, 32>(), loss<T, 8, 1, 128, 32>(), loss<T, 8, 1, 192, 32>(), loss<T, 8, 1, 256, 32>(), loss<T, 8, 1, 384, 32>(),
};
}  // namespace
const Variants VARIANTS_F32[2] = {list_of(LOSS), list_of(GRAD)};

}  // namespace distill
}  // namespace rag
