// Entry points of the operators on a caller's device tensors
// (include/maxim_b200.h): argument checks and dispatch on the element type.
#include "ops.h"

#include <cstring>
#include <mutex>
#include <string>

#include "common.h"
#include "gpu_common.cuh"
#include "sm100.cuh"
#include "wait_record.h"

namespace mx {
namespace {

const OpsTable& table(const char* who, int dtype) {
  switch (dtype) {
    case MX_DT_F32: return kOpsF32;
    case MX_DT_BF16: return kOpsBf16;
    case MX_DT_F16: return kOpsF16;
  }
  throw Error(fmt("%s: dtype %d is not one of MX_DT_F32, MX_DT_BF16, MX_DT_F16", who, dtype));
}
int64_t size_of(int dtype) { return dtype == MX_DT_F32 ? 4 : 2; }

// Row lengths stay below 2^30, so that a kernel's index may step past the end;
// rows are counted in 64 bits but are a coordinate of the tensor maps.
void check_length(const char* who, const char* what, int64_t v) {
  if (v < 1 || v >= (int64_t(1) << 30))
    throw Error(fmt("%s: %s = %lld is outside 1 .. 2^30-1", who, what, (long long)v));
}
void check_rows(const char* who, const char* what, int64_t v) {
  if (v < 0 || v >= (int64_t(1) << 31) - 512)
    throw Error(fmt("%s: %s = %lld is outside 0 .. 2^31-513", who, what, (long long)v));
}
// A matrix argument: present, aligned to its elements, rows that do not overlap.
void check_matrix(const char* who, const char* what, const void* p, int64_t rows, int64_t cols, int64_t stride,
                  int dtype) {
  if (rows == 0) return;
  if (!p) throw Error(fmt("%s: %s is null", who, what));
  if (reinterpret_cast<uintptr_t>(p) % size_of(dtype))
    throw Error(fmt("%s: %s is not aligned to its elements", who, what));
  if (stride < cols || stride >= (int64_t(1) << 36))
    throw Error(fmt("%s: %s has a row stride of %lld; its rows have %lld elements", who, what, (long long)stride,
                    (long long)cols));
}
void check_vector(const char* who, const char* what, const void* p, int dtype, bool optional) {
  if (!p && !optional) throw Error(fmt("%s: %s is null", who, what));
  if (reinterpret_cast<uintptr_t>(p) % size_of(dtype))
    throw Error(fmt("%s: %s is not aligned to its elements", who, what));
}
void check_workspace(const char* who, const void* p, int64_t have, int64_t need) {
  if (need == 0) return;
  if (!p || have < need)
    throw Error(
        fmt("%s: the workspace has %lld bytes, %lld are needed", who, (long long)(p ? have : 0), (long long)need));
  if (reinterpret_cast<uintptr_t>(p) % 16) throw Error(fmt("%s: the workspace is not 16-byte aligned", who));
}
void check_act(const char* who, int act) {
  if (act < MX_ACT_NONE || act > MX_ACT_SIGMOID) throw Error(fmt("%s: act %d is not one of MX_ACT_*", who, act));
}
void check_param_dtype(const char* who, int dtype, int param) {
  if (param != dtype && param != MX_DT_F32)
    throw Error(fmt("%s: param_dtype %d is neither the tensors' dtype nor MX_DT_F32", who, param));
}

// The status words of the dense kernels, one a device, in page-locked host
// memory that every device can write, so the host reads them without a copy.
struct Status {
  int* words;
  WaitRecords records;
  explicit Status(int* w) : words(w), records(w) {}
};
// While it lives, this thread may make calls that a stream capture under way
// (torch's are of the global mode) would refuse and be spoilt by. What is done
// under it - an allocation kept for good - is no part of any capture.
struct OutsideCapture {
  cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
  OutsideCapture() { MX_CUDA(cudaThreadExchangeStreamCaptureMode(&mode)); }
  ~OutsideCapture() { cudaThreadExchangeStreamCaptureMode(&mode); }
};
Status& status() {
  static std::mutex mu;
  static Status* made = nullptr;  // for the life of the process: kernels write it
  std::lock_guard<std::mutex> lock(mu);
  if (!made) {
    void* p = nullptr;
    constexpr size_t bytes = WaitRecords::kDevices * sizeof(int);
    OutsideCapture outside;
    MX_CUDA(cudaHostAlloc(&p, bytes, cudaHostAllocPortable | cudaHostAllocMapped));
    std::memset(p, 0, bytes);
    made = new Status(static_cast<int*>(p));
  }
  return *made;
}

OpsDevice device() {
  constexpr int kMaxDevices = WaitRecords::kDevices;
  static std::mutex mu;
  static int sms[kMaxDevices] = {};
  int dev = 0;
  MX_CUDA(cudaGetDevice(&dev));
  OpsDevice d;
  {
    std::lock_guard<std::mutex> lock(mu);
    if (dev < 0 || dev >= kMaxDevices)
      throw Error(fmt("device %d is beyond the %d the operators track", dev, kMaxDevices));
    if (!sms[dev]) MX_CUDA(cudaDeviceGetAttribute(&sms[dev], cudaDevAttrMultiProcessorCount, dev));
    d.sms = sms[dev];
  }
  d.index = dev;
  d.status = status().words + dev;  // unified addressing: the host pointer serves the device too
  return d;
}

void check_status(const char* who, const OpsDevice& d) {
  if (const int code = status().records.pending(d.index))
    throw Error(fmt("%s: an earlier dense kernel on device %d gave up a wait in its pipeline (code 0x%x)", who, d.index,
                    code),
                MX_E_DEVICE);
}

// A wait that nothing ends, for mx_dense_wait_check.
constexpr int kErrWaitCheck = 0x2FF;
__global__ void wait_check_kernel(int* status, uint64_t limit_ns) {
  __shared__ uint64_t bar;
  sm100::mbar_init(&bar, 1);
  sm100::fence_mbar_init();
  if (!sm100::mbar_wait(&bar, 0, nullptr, limit_ns)) *static_cast<volatile int*>(status) = kErrWaitCheck;
}

void check(const mx_layer_norm_args& a) {
  const char* who = "mx_layer_norm";
  table(who, a.dtype);
  check_param_dtype(who, a.dtype, a.param_dtype);
  check_rows(who, "rows", a.rows);
  check_length(who, "c", a.c);
  check_matrix(who, "x", a.x, a.rows, a.c, a.x_stride, a.dtype);
  check_matrix(who, "y", a.y, a.rows, a.c, a.y_stride, a.dtype);
  check_vector(who, "scale", a.scale, a.param_dtype, false);
  check_vector(who, "bias", a.bias, a.param_dtype, false);
  check_vector(who, "mean", a.mean, MX_DT_F32, true);
  check_vector(who, "rstd", a.rstd, MX_DT_F32, true);
  if (!(a.eps >= 0.0f)) throw Error(fmt("%s: eps = %g is negative", who, double(a.eps)));
}
void check(const mx_layer_norm_backward_args& a) {
  const char* who = "mx_layer_norm_backward";
  table(who, a.dtype);
  check_param_dtype(who, a.dtype, a.param_dtype);
  check_rows(who, "rows", a.rows);
  check_length(who, "c", a.c);
  check_matrix(who, "dy", a.dy, a.rows, a.c, a.dy_stride, a.dtype);
  check_matrix(who, "x", a.x, a.rows, a.c, a.x_stride, a.dtype);
  if (a.dx) check_matrix(who, "dx", a.dx, a.rows, a.c, a.dx_stride, a.dtype);
  check_vector(who, "scale", a.scale, a.param_dtype, a.dx == nullptr);
  check_vector(who, "mean", a.mean, MX_DT_F32, a.rows == 0);
  check_vector(who, "rstd", a.rstd, MX_DT_F32, a.rows == 0);
  check_vector(who, "dscale", a.dscale, a.param_dtype, true);
  check_vector(who, "dbias", a.dbias, a.param_dtype, true);
}
void check(const mx_dense_args& a) {
  const char* who = "mx_dense";
  table(who, a.dtype);
  check_act(who, a.act);
  check_rows(who, "m", a.m);
  check_length(who, "k", a.k);
  check_length(who, "n", a.n);
  check_matrix(who, "x", a.x, a.m, a.k, a.x_stride, a.dtype);
  check_matrix(who, "w", a.w, a.n, a.k, a.w_stride, a.dtype);
  check_matrix(who, "y", a.y, a.m, a.n, a.y_stride, a.dtype);
  if (a.residual) check_matrix(who, "residual", a.residual, a.m, a.n, a.residual_stride, a.dtype);
  if (a.pre) check_matrix(who, "pre", a.pre, a.m, a.n, a.pre_stride, a.dtype);
  check_vector(who, "bias", a.bias, a.dtype, true);
}
void check(const mx_dense_backward_args& a) {
  const char* who = "mx_dense_backward";
  table(who, a.dtype);
  check_act(who, a.act);
  check_rows(who, "m", a.m);
  check_length(who, "k", a.k);
  check_length(who, "n", a.n);
  check_matrix(who, "dy", a.dy, a.m, a.n, a.dy_stride, a.dtype);
  if (a.act != MX_ACT_NONE) check_matrix(who, "pre", a.pre, a.m, a.n, a.pre_stride, a.dtype);
  if (a.dx) {
    check_matrix(who, "w", a.w, a.n, a.k, a.w_stride, a.dtype);
    check_matrix(who, "dx", a.dx, a.m, a.k, a.dx_stride, a.dtype);
  }
  if (a.dw) {
    check_matrix(who, "x", a.x, a.m, a.k, a.x_stride, a.dtype);
    check_matrix(who, "dw", a.dw, a.n, a.k, a.dw_stride, a.dtype);
  }
  check_vector(who, "db", a.db, a.dtype, true);
}

}  // namespace
}  // namespace mx

using namespace mx;

extern "C" int mx_layer_norm(const mx_layer_norm_args* a, void* stream) {
  return guard([&] {
    if (!a) throw Error("mx_layer_norm: null arguments");
    check(*a);
    if (a->rows == 0) return;
    table("mx_layer_norm", a->dtype).layer_norm(*a, device(), static_cast<cudaStream_t>(stream));
  });
}

extern "C" int mx_layer_norm_backward_workspace(const mx_layer_norm_backward_args* a, int64_t* bytes) {
  return guard([&] {
    if (!a || !bytes) throw Error("mx_layer_norm_backward_workspace: null arguments");
    check(*a);
    *bytes = table("mx_layer_norm_backward", a->dtype).layer_norm_backward_workspace(*a, device());
  });
}

extern "C" int mx_layer_norm_backward(const mx_layer_norm_backward_args* a, void* stream) {
  return guard([&] {
    if (!a) throw Error("mx_layer_norm_backward: null arguments");
    check(*a);
    const OpsDevice d = device();
    const OpsTable& t = table("mx_layer_norm_backward", a->dtype);
    check_workspace("mx_layer_norm_backward", a->workspace, a->workspace_bytes, t.layer_norm_backward_workspace(*a, d));
    t.layer_norm_backward(*a, d, static_cast<cudaStream_t>(stream));
  });
}

extern "C" int mx_dense_workspace(const mx_dense_args* a, int64_t* bytes) {
  return guard([&] {
    if (!a || !bytes) throw Error("mx_dense_workspace: null arguments");
    check(*a);
    *bytes = table("mx_dense", a->dtype).dense_workspace(*a, device());
  });
}

extern "C" int mx_dense(const mx_dense_args* a, void* stream) {
  return guard([&] {
    if (!a) throw Error("mx_dense: null arguments");
    check(*a);
    if (a->m == 0) return;
    const OpsDevice d = device();
    check_status("mx_dense", d);
    const OpsTable& t = table("mx_dense", a->dtype);
    check_workspace("mx_dense", a->workspace, a->workspace_bytes, t.dense_workspace(*a, d));
    t.dense(*a, d, static_cast<cudaStream_t>(stream));
  });
}

extern "C" int mx_dense_backward_workspace(const mx_dense_backward_args* a, int64_t* bytes) {
  return guard([&] {
    if (!a || !bytes) throw Error("mx_dense_backward_workspace: null arguments");
    check(*a);
    *bytes = table("mx_dense_backward", a->dtype).dense_backward_workspace(*a, device());
  });
}

extern "C" int mx_dense_backward(const mx_dense_backward_args* a, void* stream) {
  return guard([&] {
    if (!a) throw Error("mx_dense_backward: null arguments");
    check(*a);
    const OpsDevice d = device();
    check_status("mx_dense_backward", d);
    const OpsTable& t = table("mx_dense_backward", a->dtype);
    check_workspace("mx_dense_backward", a->workspace, a->workspace_bytes, t.dense_backward_workspace(*a, d));
    t.dense_backward(*a, d, static_cast<cudaStream_t>(stream));
  });
}

extern "C" int mx_dense_poll(void) {
  return guard([&] {
    for (int dev = 0; dev < WaitRecords::kDevices; ++dev)
      if (const int code = status().records.take(dev))
        throw Error(
            fmt("mx_dense_poll: a dense kernel on device %d gave up a wait in its pipeline (code 0x%x)", dev, code),
            MX_E_DEVICE);
  });
}

extern "C" int mx_dense_wait_check(int64_t limit_us, void* stream) {
  return guard([&] {
    if (limit_us < 0 || limit_us > 1000000)
      throw Error(fmt("mx_dense_wait_check: limit_us = %lld is outside 0 .. 1000000", (long long)limit_us));
    wait_check_kernel<<<1, 1, 0, static_cast<cudaStream_t>(stream)>>>(device().status, uint64_t(limit_us) * 1000);
    MX_CUDA(cudaGetLastError());
  });
}
