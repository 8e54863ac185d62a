// distill_tile_bf16.hip -- tile_kernel for bfloat16 rows.
#include "distill_variants.h"

namespace rag {
namespace distill {

namespace {
typedef unsigned short T;
const Variant ALL[] = {
    // up to 16 queries, bound by the rows' bytes
    variant<T, 1, 4, 64, 32>(), variant<T, 1, 4, 128, 32>(), variant<T, 1, 4, 192, 32>(), variant<T, 1, 4, 256, 32>(),
    variant<T, 1, 4, 384, 32>(),
    // 32 at a time
    variant<T, 2, 2, 64, 32>(), variant<T, 2, 2, 128, 32>(), variant<T, 2, 2, 192, 32>(), variant<T, 2, 4, 128, 32>(),
    variant<T, 2, 4, 192, 32>(), variant<T, 2, 4, 256, 32>(), variant<T, 2, 4, 384, 32>(),
    // 64 at a time; 64 rows a tile where the ring still has two (256 queries x 512, 1M rows: 901 us with 32 rows, 846 with 64)
    variant<T, 4, 2, 64, 64>(), variant<T, 4, 2, 128, 64>(), variant<T, 4, 2, 192, 64>(), variant<T, 4, 2, 256, 64>(),
    variant<T, 4, 2, 384, 32>(),
    // 128 at a time (1024 queries x 384, 1M rows: 2117 us with tiles of 32 rows, 1838 with 64)
    variant<T, 8, 1, 64, 64>(), variant<T, 8, 1, 128, 64>(), variant<T, 8, 1, 192, 64>(), variant<T, 8, 1, 256, 64>(),
    variant<T, 8, 1, 384, 64>(),
};
}  // namespace
const Variant* const VARIANTS_BF16 = ALL;
const int N_VARIANTS_BF16 = sizeof ALL / sizeof ALL[0];

}  // namespace distill
}  // namespace rag
