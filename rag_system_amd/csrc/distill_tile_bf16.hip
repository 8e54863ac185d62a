// distill_tile_bf16.hip -- tile_kernel for bfloat16 rows.
#include "distill_variants.h"

namespace rag {
namespace distill {

namespace {
typedef unsigned short T;
const Variant GRAD[] = {
    // up to 16 queries, bound by the rows' bytes
    grad<T, 1, 4, 64, 32>(), grad<T, 1, 4, 128, 32>(), grad<T, 1, 4, 192, 32>(), grad<T, 1, 4, 256, 32>(),
    grad<T, 1, 4, 384, 32>(),
    // 32 at a time
    grad<T, 2, 2, 64, 32>(), grad<T, 2, 2, 128, 32>(), grad<T, 2, 2, 192, 32>(), grad<T, 2, 4, 128, 32>(),
    grad<T, 2, 4, 192, 32>(), grad<T, 2, 4, 256, 32>(), grad<T, 2, 4, 384, 32>(),
    // 64 at a time; 64 rows a tile where the ring still has two (256 queries x 512, 1M rows: 1181 us with 32 rows, 1097 with 64)
    grad<T, 4, 2, 64, 64>(), grad<T, 4, 2, 128, 64>(), grad<T, 4, 2, 192, 64>(), grad<T, 4, 2, 256, 64>(),
    grad<T, 4, 2, 384, 32>(),
    // 128 at a time (1024 queries x 384, 1M rows: 2440 us with tiles of 32 rows, 2230 with 64)
    grad<T, 8, 1, 64, 64>(), grad<T, 8, 1, 128, 64>(), grad<T, 8, 1, 192, 64>(), grad<T, 8, 1, 256, 64>(),
    grad<T, 8, 1, 384, 64>(),
};
// The loss alone needs no row sum: without O a wave holds its queries' whole rows, and nothing is exchanged between waves (256
// queries x 768, 1M rows: 916 us with two waves to a query, 593 with one).  Up to 64 queries the rows' bytes
// bound it, and rows of up to 384 values have no smaller group (16 x 384, 1M rows: 136 us with a group of 16, 137 with one of 64).
const Variant LOSS[] = {
    loss<T, 1, 4, 128, 32>(), loss<T, 1, 4, 192, 32>(), loss<T, 1, 4, 256, 32>(), loss<T, 1, 4, 384, 32>(),
    loss<T, 2, 4, 128, 32>(), loss<T, 2, 4, 192, 32>(),
    loss<T, 2, 4, 256, 32>(), loss<T, 2, 4, 384, 32>(),
    loss<T, 4, 1, 64, 32>(), loss<T, 4, 1, 128, 32>(), loss<T, 4, 1, 192, 32>(), loss<T, 4, 1, 256, 32>(), loss<T, 4, 1, 384, 64>(),
    loss<T, 8, 1, 64, 64>(), loss<T, 8, 1, 128, 32>(), loss<T, 8, 1, 192, 64>(), loss<T, 8, 1, 256, 32>(), loss<T, 8, 1, 384, 32>(),
    loss<T, 8, 1, 512, 32>(), loss<T, 8, 1, 768, 32>(),
};
}  // namespace
const Variants VARIANTS_BF16[2] = {list_of(LOSS), list_of(GRAD)};

}  // namespace distill
}  // namespace rag
