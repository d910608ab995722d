// The operators of ops.h on f16 tensors.
#include "ops_impl.cuh"

namespace mx {
const OpsTable kOpsF16 = ops_table<__half>();
}
