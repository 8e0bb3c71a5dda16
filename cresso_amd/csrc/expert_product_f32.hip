// The grouped products' kernels for f32 rows.
#include "expert_product.hpp"

namespace cresso {
CRESSO_GROUP_LAUNCH(float)
}  // namespace cresso
