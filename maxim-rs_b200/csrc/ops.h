// The operators on a caller's device tensors, per element type. ops.cu checks
// the arguments and dispatches; ops_f32.cu, ops_bf16.cu and ops_f16.cu each
// instantiate ops_impl.cuh for one type.
#pragma once

#include <cuda_runtime.h>

#include <cstdint>

#include "maxim_b200.h"

namespace mx {

struct OpsDevice {
  int index, sms;
  int* status;  // the dense kernels' status word of this device, as it sees it
};

// One element type's operators; arguments have been checked.
struct OpsTable {
  void (*layer_norm)(const mx_layer_norm_args& a, const OpsDevice& d, cudaStream_t s);
  int64_t (*layer_norm_backward_workspace)(const mx_layer_norm_backward_args& a, const OpsDevice& d);
  void (*layer_norm_backward)(const mx_layer_norm_backward_args& a, const OpsDevice& d, cudaStream_t s);
  int64_t (*dense_workspace)(const mx_dense_args& a, const OpsDevice& d);
  void (*dense)(const mx_dense_args& a, const OpsDevice& d, cudaStream_t s);
  int64_t (*dense_backward_workspace)(const mx_dense_backward_args& a, const OpsDevice& d);
  void (*dense_backward)(const mx_dense_backward_args& a, const OpsDevice& d, cudaStream_t s);
};
extern const OpsTable kOpsF32, kOpsBf16, kOpsF16;

}  // namespace mx
