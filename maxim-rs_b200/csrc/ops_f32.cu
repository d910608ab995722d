// The operators of ops.h on f32 tensors.
#include "ops_impl.cuh"

namespace mx {
const OpsTable kOpsF32 = ops_table<float>();
}
