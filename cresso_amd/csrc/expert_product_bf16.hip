// The grouped products' kernels for bf16 rows.
#include "expert_product.hpp"

namespace cresso {
CRESSO_GROUP_LAUNCH(__hip_bfloat16)
}  // namespace cresso
