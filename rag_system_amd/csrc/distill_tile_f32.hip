// distill_tile_f32.hip -- tile_kernel for float32 rows.
#include "distill_variants.h"

namespace rag {
namespace distill {

namespace {
typedef float T;
const Variant ALL[] = {
    // up to 16 queries, bound by the rows' bytes
    variant<T, 1, 4, 32, 32>(), variant<T, 1, 4, 64, 32>(), variant<T, 1, 4, 96, 32>(), variant<T, 1, 4, 128, 16>(),
    variant<T, 1, 4, 192, 16>(), variant<T, 1, 4, 256, 16>(), variant<T, 1, 4, 384, 16>(),
    // 32 at a time
    variant<T, 2, 2, 32, 16>(), variant<T, 2, 2, 64, 16>(), variant<T, 2, 2, 96, 16>(), variant<T, 2, 2, 128, 16>(),
    variant<T, 2, 2, 192, 16>(), variant<T, 2, 4, 128, 16>(), variant<T, 2, 4, 192, 16>(), variant<T, 2, 4, 256, 16>(),
    variant<T, 2, 4, 384, 16>(),
    // 64 at a time
    variant<T, 4, 2, 32, 32>(), variant<T, 4, 2, 64, 32>(), variant<T, 4, 2, 96, 32>(), variant<T, 4, 2, 128, 32>(),
    variant<T, 4, 2, 192, 32>(), variant<T, 4, 2, 256, 16>(), variant<T, 4, 2, 384, 16>(),
    // 128 at a time
    variant<T, 8, 1, 32, 64>(), variant<T, 8, 1, 64, 32>(), variant<T, 8, 1, 96, 64>(), variant<T, 8, 1, 128, 32>(),
    variant<T, 8, 1, 192, 32>(), variant<T, 8, 1, 256, 32>(), variant<T, 8, 1, 384, 32>(),
};
}  // namespace
const Variant* const VARIANTS_F32 = ALL;
const int N_VARIANTS_F32 = sizeof ALL / sizeof ALL[0];

}  // namespace distill
}  // namespace rag
