// Element types of the operators on a caller's tensors: fp32, bf16 and fp16
// values held as fp32 in registers, moved 16 bytes at a time where the
// alignment allows it.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "maxim_b200.h"

namespace mx {

// Elements of a 16-byte vector.
template <class T>
constexpr int kVec = 16 / int(sizeof(T));

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
template <class T>
__device__ __forceinline__ T from_f(float v);
template <>
__device__ __forceinline__ float from_f<float>(float v) {
  return v;
}
template <>
__device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}
template <>
__device__ __forceinline__ __half from_f<__half>(float v) {
  return __float2half_rn(v);
}

// V consecutive elements as they lie in memory: one 16-byte word for the
// vector forms, one element for V = 1.
template <class T, int V>
struct Raw {
  uint4 u;
};
template <class T>
struct Raw<T, 1> {
  T u;
};

template <class T, int V>
__device__ __forceinline__ Raw<T, V> raw_load(const T* p) {
  Raw<T, V> r;
  if constexpr (V == 1) {
    r.u = *p;
  } else {
    r.u = *reinterpret_cast<const uint4*>(p);
  }
  return r;
}
// The same for data that is read once: kept out of the L1, fetched into the L2
// by 256 bytes (a token's 134 MB of weights: 26.9 to 25.8 us). Not by the
// read-only path (.nc): that wants memory which nothing writes while the kernel
// lives, and a kernel whose blocks are set up early lives beside the one before
// it, which may be what writes the weights. Volatile, so that it stays after pdl_wait.
template <class T, int V>
__device__ __forceinline__ Raw<T, V> raw_load_once(const T* p) {
  Raw<T, V> r;
  if constexpr (V == 1) {
    r.u = *p;
  } else {
    asm volatile("ld.global.L1::no_allocate.L2::256B.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r.u.x), "=r"(r.u.y), "=r"(r.u.z), "=r"(r.u.w)
                 : "l"(p));
  }
  return r;
}
// Data that is read once, first to leave the L2.
template <class T, int V>
__device__ __forceinline__ Raw<T, V> raw_load_streaming(const T* p) {
  Raw<T, V> r;
  if constexpr (V == 1) {
    r.u = *p;
  } else {
    r.u = __ldcs(reinterpret_cast<const uint4*>(p));
  }
  return r;
}
template <class T, int V>
__device__ __forceinline__ Raw<T, V> raw_zero() {
  Raw<T, V> r;
  if constexpr (V == 1) {
    r.u = from_f<T>(0.0f);
  } else {
    r.u = make_uint4(0, 0, 0, 0);
  }
  return r;
}
template <class T, int V>
__device__ __forceinline__ void raw_unpack(const Raw<T, V>& r, float* v) {
  if constexpr (V == 1) {
    v[0] = to_f(r.u);
  } else if constexpr (sizeof(T) == 4) {
    v[0] = __uint_as_float(r.u.x), v[1] = __uint_as_float(r.u.y);
    v[2] = __uint_as_float(r.u.z), v[3] = __uint_as_float(r.u.w);
  } else {
    const uint32_t w[4] = {r.u.x, r.u.y, r.u.z, r.u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (std::is_same<T, __half>::value) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        v[2 * i] = f.x, v[2 * i + 1] = f.y;
      } else {
        v[2 * i] = __uint_as_float(w[i] << 16);
        v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
      }
    }
  }
}
template <class T, int V>
__device__ __forceinline__ Raw<T, V> raw_pack(const float* v) {
  Raw<T, V> r;
  if constexpr (V == 1) {
    r.u = from_f<T>(v[0]);
  } else if constexpr (sizeof(T) == 4) {
    r.u = make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
  } else {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (std::is_same<T, __half>::value) {
        const __half2 h = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&h);
      } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&h);
      }
    }
    r.u = make_uint4(w[0], w[1], w[2], w[3]);
  }
  return r;
}
template <class T, int V>
__device__ __forceinline__ void raw_store(T* p, const Raw<T, V>& r) {
  if constexpr (V == 1) {
    *p = r.u;
  } else {
    *reinterpret_cast<uint4*>(p) = r.u;
  }
}

// A parameter vector element held as fp32 or in the operator's own type.
template <class T>
__device__ __forceinline__ float param_at(const void* p, int f32, int64_t i) {
  return f32 ? static_cast<const float*>(p)[i] : to_f(static_cast<const T*>(p)[i]);
}
template <class T>
__device__ __forceinline__ void param_put(void* p, int f32, int64_t i, float v) {
  if (f32) {
    static_cast<float*>(p)[i] = v;
  } else {
    static_cast<T*>(p)[i] = from_f<T>(v);
  }
}

}  // namespace mx
