// The operators of ops.h on bf16 tensors.
#include "ops_impl.cuh"

namespace mx {
const OpsTable kOpsBf16 = ops_table<__nv_bfloat16>();
}
