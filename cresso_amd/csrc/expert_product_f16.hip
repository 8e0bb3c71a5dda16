// The grouped products' kernels for f16 rows.
#include "expert_product.hpp"

namespace cresso {
CRESSO_GROUP_LAUNCH(__half)
}  // namespace cresso
