// Layer norm over the rows of a matrix, forward and backward.
//
//   y  = (x - mean) rstd scale + bias,  mean = sum x / c,
//                                       rstd = 1 / sqrt(sum (x - mean)^2 / c + eps)
//   with n = (x - mean) rstd and g = dy scale:
//   dx = rstd (g - mean(g) - n mean(g n)),  dscale = sum_rows dy n,  dbias = sum_rows dy
//
// Both directions are bound by memory: every element is read once (x, and dy)
// and written once (y or dx). A row therefore stays in registers between its
// statistics and its result: L lanes hold a row, NV vectors of V elements
// each, and the next row's vectors are loaded before the current row is
// worked on. A block keeps its columns for all its rows, so the scale and
// bias are read once a block and the backward pass adds the parameter
// gradients up in registers; what a block has summed goes to a partial row,
// and a second kernel adds the partial rows in a fixed order (no atomics, so
// results do not change from run to run). A few rows are one cluster's work,
// whose blocks add their sums up themselves: the second launch would cost more
// (77 x 769 fp16: 17.1 us a call with it, 15.1 without).
#pragma once

#include "gpu_common.cuh"
#include "kernels_vec.cuh"
#include "sm100.cuh"

namespace mx {

struct NormFwd {
  const void *x, *scale, *bias;
  void* y;
  float *mean, *rstd;  // null: not stored
  int64_t rows, x_stride, y_stride;
  int c;
  int param_f32;
  float eps;
};

struct NormBwd {
  const void *dy, *x, *scale;
  const float *mean, *rstd;
  void* dx;     // null: not wanted
  float* part;  // [gridDim.x][2][c] partial sums of dscale and dbias; null: not wanted, or joined in the cluster
  // With `cluster` the grid is one cluster of that many blocks, which add their
  // sums up in one another's shared memory and store dscale and dbias (null:
  // not wanted) themselves.
  int cluster;
  void *dscale, *dbias;
  int64_t rows, dy_stride, x_stride, dx_stride;
  int c;
  int param_f32;
};

// Sum over the L lanes of a row; every lane gets the sums. For L > 32 the
// warps' sums meet in `red` (two slots alternate, so one barrier a sum is
// enough: a warp can only be one sum ahead of another).
template <int L, int K>
__device__ __forceinline__ void row_sum(float (&s)[K], float (*red)[32 * K], int& slot) {
#pragma unroll
  for (int o = (L < 32 ? L : 32) / 2; o > 0; o >>= 1)
#pragma unroll
    for (int k = 0; k < K; ++k) s[k] += __shfl_xor_sync(0xFFFFFFFFu, s[k], o);
  if constexpr (L > 32) {
    constexpr int W = L / 32;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    float* r = red[slot];
    slot ^= 1;
    if (lane == 0)
#pragma unroll
      for (int k = 0; k < K; ++k) r[warp * K + k] = s[k];
    __syncthreads();
#pragma unroll
    for (int k = 0; k < K; ++k) s[k] = r[(lane % W) * K + k];
#pragma unroll
    for (int o = W / 2; o > 0; o >>= 1)
#pragma unroll
      for (int k = 0; k < K; ++k) s[k] += __shfl_xor_sync(0xFFFFFFFFu, s[k], o);
  }
}

template <int L>
constexpr int kNormThreads = L <= 32 ? 256 : L;
// Blocks an SM is asked to hold (0: the compiler's own choice of registers).
// Asking for one lets a row's block have more of them, and fewer blocks share the
// SM. Time with it over time without, 64 to 128 MB of rows: forward 0.92 to 0.99 for 128
// lanes or fewer, 0.83 to 0.97 for fp32 rows of 256, 0.86 to 0.96 for 512 (1.05 at fp32 rows of
// 8192); but 1.05 to 1.12 for 16-bit rows of 256 lanes (2056 to 4096 long, which the
// compiler gives three blocks of fewer registers by itself). Backward 0.91 to 0.97 for 128
// and 512 lanes in 16 bits, 0.95 to 1.01 in fp32.
template <int V, int L, bool BACKWARD>
constexpr int kNormMinBlocks = BACKWARD ? (L == 128 || L == 512) : (V > 1 && L > 32 && !(V == 8 && L == 256));
// Up to 16 values a thread the parameters and the next row fit in registers too.
template <int V, int NV>
constexpr bool kNormHold = V * NV <= 16;

// Rows spread over a block go through a ring in shared memory, filled by
// asynchronous 16-byte copies several rows ahead: every thread copies, waits for
// and reads its own vectors, so the ring needs no barrier. (One row ahead in
// registers left too few bytes in flight: 55 us for 16411 x 4096 bf16, 88 us
// backward.) Short rows, many to a block, have enough in flight in registers.
template <int V, int L>
constexpr bool kNormRing = V > 1 && L > 32;
// Stages of `bytes` each: 3 up to 16 KB (a fourth measured 1 to 3 us slower), else
// 2, else 1 (the next row is on its way while the current one is worked on in
// registers).
constexpr int norm_stages(int bytes) { return bytes <= 16384 ? 3 : (bytes <= 65536 ? 2 : 1); }
template <int V, int L, int NV, int TENSORS>
constexpr int kNormStages = norm_stages(L * NV * 16 * TENSORS);
template <int V, int L, int NV, int TENSORS>
constexpr int kNormSmem = kNormRing<V, L> ? kNormStages<V, L, NV, TENSORS> * L * NV * 16 * TENSORS : 0;

// 16 bytes from src, or 16 zero bytes.
__device__ __forceinline__ void copy_async16(void* dst, const void* src, bool on) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(
                   static_cast<uint32_t>(__cvta_generic_to_shared(dst))),
               "l"(src), "r"(on ? 16 : 0)
               : "memory");
}
__device__ __forceinline__ void copy_async4(void* dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(static_cast<uint32_t>(__cvta_generic_to_shared(dst))),
               "l"(src)
               : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// Values are worked on in pairs (f32x2: the same roundings at half the
// instructions; with 2-byte elements the norm is otherwise bound by its
// instruction issue: 16411 x 4096 bf16 took 57 us in scalar form, 12 us over
// the memory's time). A thread's single value has a zero beside it.
template <int E>
constexpr int kPairs = (E + 1) / 2;
template <class T, int V, int NV>
__device__ __forceinline__ void unpack_pairs(const Raw<T, V> (&q)[NV], uint64_t (&v)[kPairs<V * NV>]) {
  float f[V * NV];
#pragma unroll
  for (int j = 0; j < NV; ++j) raw_unpack<T, V>(q[j], f + j * V);
#pragma unroll
  for (int i = 0; i < kPairs<V * NV>; ++i)
    v[i] = f2_pack(f[2 * i], 2 * i + 1 < V * NV ? f[(2 * i + 1) % (V * NV)] : 0.0f);
}
__device__ __forceinline__ float pair_sum(uint64_t v) {
  float a, b;
  f2_unpack(v, a, b);
  return a + b;
}

template <class T, int V, int L, int NV>
__global__ void __launch_bounds__(kNormThreads<L>, kNormMinBlocks<V, L, false>) layer_norm_kernel(NormFwd p) {
  sm100::pdl_wait();
  constexpr int E = V * NV, P = kPairs<E>;
  constexpr bool HOLD = kNormHold<V, NV>;
  constexpr int GROUPS = kNormThreads<L> / L;
  __shared__ float red[2][64];
  int slot = 0;
  const int lane = threadIdx.x % L;
  const T* x = static_cast<const T*>(p.x);
  T* y = static_cast<T*>(p.y);
  const float inv_c = 1.0f / float(p.c);
  bool in[NV];
#pragma unroll
  for (int j = 0; j < NV; ++j) in[j] = (j * L + lane) * V < p.c;
  // -m where the pair's values exist, 0 where they do not (those stay 0).
  auto minus = [&](float m, int i) {
    const bool a = in[2 * i / V], b = 2 * i + 1 < E && in[(2 * i + 1) % E / V];
    return f2_pack(a ? -m : 0.0f, b ? -m : 0.0f);
  };
  auto param = [&](const void* q, int i) {
    float f[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int e = 2 * i + h;
      f[h] = e < E && in[e % E / V] ? param_at<T>(q, p.param_f32, ((e / V) * L + lane) * V + e % V) : 0.0f;
    }
    return f2_pack(f[0], f[1]);
  };
  uint64_t w[HOLD ? P : 1], b[HOLD ? P : 1];
  if constexpr (HOLD) {
#pragma unroll
    for (int i = 0; i < P; ++i) w[i] = param(p.scale, i), b[i] = param(p.bias, i);
  }
  // L > 32: the values in this warp and in the warp that this lane stands for below.
  constexpr int W = L > 32 ? L / 32 : 1;
  auto warp_values = [&](int k) {
    int n = 0;
#pragma unroll
    for (int j = 0; j < NV; ++j) n += min(max(p.c - (j * L + k * 32) * V, 0), 32 * V);
    return float(n);
  };
  const float n_own = warp_values(threadIdx.x >> 5), n_of = warp_values(threadIdx.x % W);
  const float inv_own = n_own > 0.0f ? 1.0f / n_own : 0.0f, inv_of = n_of > 0.0f ? 1.0f / n_of : 0.0f;

  auto load = [&](int64_t r, Raw<T, V>(&q)[NV]) {
#pragma unroll
    for (int j = 0; j < NV; ++j)
      q[j] = r < p.rows && in[j] ? raw_load<T, V>(x + r * p.x_stride + (j * L + lane) * V) : raw_zero<T, V>();
  };
  const int64_t step = int64_t(gridDim.x) * GROUPS;
  constexpr bool RING = kNormRing<V, L>;
  constexpr int S = kNormStages<V, L, NV, 1>;
  extern __shared__ uint4 ring[];
  auto fill = [&](int64_t r, int stage) {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const bool on = r < p.rows && in[j];
      copy_async16(&ring[(stage * NV + j) * L + lane], on ? x + r * p.x_stride + (j * L + lane) * V : x, on);
    }
    copy_commit();
  };
  Raw<T, V> cur[NV];
  int stage = 0;
  if constexpr (RING) {
#pragma unroll
    for (int k = 0; k < S; ++k) fill(blockIdx.x + k * step, k);
  } else {
    load(int64_t(blockIdx.x) * GROUPS + threadIdx.x / L, cur);
  }
  for (int64_t base = int64_t(blockIdx.x) * GROUPS; base < p.rows; base += step) {
    const int64_t r = base + threadIdx.x / L;
    Raw<T, V> next[HOLD && !RING ? NV : 1];
    if constexpr (RING) {
      copy_wait<S - 1>();
#pragma unroll
      for (int j = 0; j < NV; ++j)
        cur[j] = raw_load<T, V>(reinterpret_cast<const T*>(&ring[(stage * NV + j) * L + lane]));
      fill(r + S * step, stage);
      stage = stage + 1 == S ? 0 : stage + 1;
    } else if constexpr (HOLD) {
      load(r + step, next);
    }
    uint64_t v[P];
    unpack_pairs<T, V, NV>(cur, v);
    // The sum, then the squares about a mean: the row's own where its lanes are
    // in one warp, else the warp's, the warps' squares joined by
    // sum_w [M2_w + n_w (mean_w - mean)^2], so that a row has one barrier.
    auto sum = [&] {
      uint64_t t = v[0];
#pragma unroll
      for (int i = 1; i < P; ++i) t = f2_add(t, v[i]);
      float s = pair_sum(t);
#pragma unroll
      for (int o = (L < 32 ? L : 32) / 2; o > 0; o >>= 1) s += __shfl_xor_sync(0xFFFFFFFFu, s, o);
      return s;
    };
    auto squares = [&](float m, bool keep) {
      uint64_t t = 0;
#pragma unroll
      for (int i = 0; i < P; ++i) {
        const uint64_t d = f2_add(v[i], minus(m, i));
        t = f2_fma(d, d, t);
        if (keep) v[i] = d;
      }
      float q = pair_sum(t);
#pragma unroll
      for (int o = (L < 32 ? L : 32) / 2; o > 0; o >>= 1) q += __shfl_xor_sync(0xFFFFFFFFu, q, o);
      return q;
    };
    float s = sum(), mean, q;
    if constexpr (L <= 32) {
      // Rounded on its own: contracted into the subtractions it would not be the mean that is stored.
      mean = __fmul_rn(s, inv_c);
      q = squares(mean, true);
    } else {
      q = squares(s * inv_own, false);
      float* part = red[slot];
      slot ^= 1;
      if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = s, part[32 + (threadIdx.x >> 5)] = q;
      __syncthreads();
      const float sw = part[threadIdx.x % W];
      q = part[32 + threadIdx.x % W];
      s = sw;
#pragma unroll
      for (int o = W / 2; o > 0; o >>= 1) s += __shfl_xor_sync(0xFFFFFFFFu, s, o);
      mean = __fmul_rn(s, inv_c);
      const float d = fmaf(sw, inv_of, -mean);
      q = fmaf(n_of * d, d, q);
#pragma unroll
      for (int o = W / 2; o > 0; o >>= 1) q += __shfl_xor_sync(0xFFFFFFFFu, q, o);
#pragma unroll
      for (int i = 0; i < P; ++i) v[i] = f2_add(v[i], minus(mean, i));
    }
    const float rstd = 1.0f / sqrtf(fmaf(q, inv_c, p.eps));
    if (r < p.rows) {
      if (lane == 0) {
        if (p.mean) p.mean[r] = mean;
        if (p.rstd) p.rstd[r] = rstd;
      }
      const uint64_t rr = f2_pack(rstd, rstd);
      float o[2 * P];
#pragma unroll
      for (int i = 0; i < P; ++i) {
        const uint64_t wi = HOLD ? w[HOLD ? i : 0] : param(p.scale, i), bi = HOLD ? b[HOLD ? i : 0] : param(p.bias, i);
        f2_unpack(f2_fma(f2_mul(v[i], rr), wi, bi), o[2 * i], o[2 * i + 1]);
      }
#pragma unroll
      for (int j = 0; j < NV; ++j)
        if (in[j]) raw_store<T, V>(y + r * p.y_stride + (j * L + lane) * V, raw_pack<T, V>(o + j * V));
    }
    if constexpr (HOLD && !RING) {
#pragma unroll
      for (int j = 0; j < NV; ++j) cur[j] = next[j];
    } else if constexpr (!RING) {
      load(r + step, cur);
    }
  }
}

// Rows too long for a block's registers: the row is read three times, the
// second and third time from the caches (a block's row is at most a few
// hundred KB of the 126 MB L2).
template <class T, int V>
__global__ void __launch_bounds__(512) layer_norm_long_kernel(NormFwd p) {
  sm100::pdl_wait();
  __shared__ float red[2][32];
  int slot = 0;
  const T* x = static_cast<const T*>(p.x);
  T* y = static_cast<T*>(p.y);
  for (int64_t r = blockIdx.x; r < p.rows; r += gridDim.x) {
    const T* xr = x + r * p.x_stride;
    float v[V], s[1] = {0.0f}, q[1] = {0.0f};
    for (int i = threadIdx.x * V; i < p.c; i += 512 * V) {
      raw_unpack<T, V>(raw_load<T, V>(xr + i), v);
#pragma unroll
      for (int k = 0; k < V; ++k) s[0] += v[k];
    }
    row_sum<512, 1>(s, red, slot);
    const float mean = s[0] / float(p.c);
    for (int i = threadIdx.x * V; i < p.c; i += 512 * V) {
      raw_unpack<T, V>(raw_load<T, V>(xr + i), v);
#pragma unroll
      for (int k = 0; k < V; ++k) q[0] = fmaf(v[k] - mean, v[k] - mean, q[0]);
    }
    row_sum<512, 1>(q, red, slot);
    const float rstd = 1.0f / sqrtf(q[0] / float(p.c) + p.eps);
    if (threadIdx.x == 0) {
      if (p.mean) p.mean[r] = mean;
      if (p.rstd) p.rstd[r] = rstd;
    }
    for (int i = threadIdx.x * V; i < p.c; i += 512 * V) {
      raw_unpack<T, V>(raw_load<T, V>(xr + i), v);
#pragma unroll
      for (int k = 0; k < V; ++k)
        v[k] = fmaf((v[k] - mean) * rstd, param_at<T>(p.scale, p.param_f32, i + k),
                    param_at<T>(p.bias, p.param_f32, i + k));
      raw_store<T, V>(y + r * p.y_stride + i, raw_pack<T, V>(v));
    }
  }
}

template <class T, int V, int L, int NV>
__global__ void __launch_bounds__(kNormThreads<L>, kNormMinBlocks<V, L, true>) layer_norm_backward_kernel(NormBwd p) {
  sm100::pdl_wait();
  constexpr int E = V * NV, P = kPairs<E>;
  constexpr bool HOLD = kNormHold<V, NV>;
  constexpr int GROUPS = kNormThreads<L> / L;
  __shared__ float red[2][64];
  int slot = 0;
  const int lane = threadIdx.x % L;
  const T *x = static_cast<const T*>(p.x), *dy = static_cast<const T*>(p.dy);
  T* dx = static_cast<T*>(p.dx);
  const float inv_c = 1.0f / float(p.c);
  bool in[NV];
#pragma unroll
  for (int j = 0; j < NV; ++j) in[j] = (j * L + lane) * V < p.c;
  // Without dx the scale does not matter (and may be absent).
  auto param = [&](int i) {
    float f[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int e = 2 * i + h;
      f[h] = dx && e < E && in[e % E / V] ? param_at<T>(p.scale, p.param_f32, ((e / V) * L + lane) * V + e % V) : 0.0f;
    }
    return f2_pack(f[0], f[1]);
  };
  // Values past the row's end have dy = 0, so they add nothing anywhere.
  uint64_t w[HOLD ? P : 1], acc_s[P], acc_b[P];
#pragma unroll
  for (int i = 0; i < P; ++i) acc_s[i] = acc_b[i] = 0;
  if constexpr (HOLD) {
#pragma unroll
    for (int i = 0; i < P; ++i) w[i] = param(i);
  }
  auto load = [&](int64_t r, Raw<T, V>(&q)[NV], Raw<T, V>(&d)[NV]) {
    const bool on = r < p.rows;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int col = (j * L + lane) * V;
      q[j] = on && in[j] ? raw_load<T, V>(x + r * p.x_stride + col) : raw_zero<T, V>();
      d[j] = on && in[j] ? raw_load<T, V>(dy + r * p.dy_stride + col) : raw_zero<T, V>();
    }
  };
  auto load_stats = [&](int64_t r, float& mean, float& rstd) {
    mean = r < p.rows ? p.mean[r] : 0.0f;
    rstd = r < p.rows ? p.rstd[r] : 0.0f;
  };
  const int64_t step = int64_t(gridDim.x) * GROUPS;
  constexpr bool RING = kNormRing<V, L>;
  constexpr int S = kNormStages<V, L, NV, 2>;
  extern __shared__ uint4 ring[];
  // A row's statistics travel with it, fetched by the first lane of every warp
  // (a row ahead in registers they were the longest wait).
  __shared__ float2 stats[RING ? S : 1][RING ? L / 32 : 1];
  auto fill = [&](int64_t r, int stage) {
    if ((threadIdx.x & 31) == 0 && r < p.rows) {
      copy_async4(&stats[stage][threadIdx.x >> 5].x, p.mean + r);
      copy_async4(&stats[stage][threadIdx.x >> 5].y, p.rstd + r);
    }
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const bool on = r < p.rows && in[j];
      const int col = (j * L + lane) * V;
      copy_async16(&ring[(2 * stage * NV + j) * L + lane], on ? x + r * p.x_stride + col : x, on);
      copy_async16(&ring[((2 * stage + 1) * NV + j) * L + lane], on ? dy + r * p.dy_stride + col : dy, on);
    }
    copy_commit();
  };
  Raw<T, V> cx[NV], cd[NV];
  float mean, rstd;
  int stage = 0;
  if constexpr (RING) {
#pragma unroll
    for (int k = 0; k < S; ++k) fill(blockIdx.x + k * step, k);
  } else {
    load_stats(int64_t(blockIdx.x) * GROUPS + threadIdx.x / L, mean, rstd);
    load(int64_t(blockIdx.x) * GROUPS + threadIdx.x / L, cx, cd);
  }
  for (int64_t base = int64_t(blockIdx.x) * GROUPS; base < p.rows; base += step) {
    const int64_t r = base + threadIdx.x / L;
    Raw<T, V> nx[HOLD && !RING ? NV : 1], nd[HOLD && !RING ? NV : 1];
    float nmean, nrstd;
    if constexpr (!RING) load_stats(r + step, nmean, nrstd);
    if constexpr (RING) {
      copy_wait<S - 1>();
      __syncwarp();
      mean = stats[stage][threadIdx.x >> 5].x, rstd = stats[stage][threadIdx.x >> 5].y;
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        cx[j] = raw_load<T, V>(reinterpret_cast<const T*>(&ring[(2 * stage * NV + j) * L + lane]));
        cd[j] = raw_load<T, V>(reinterpret_cast<const T*>(&ring[((2 * stage + 1) * NV + j) * L + lane]));
      }
      __syncwarp();  // the warp has read the statistics
      fill(r + S * step, stage);
      stage = stage + 1 == S ? 0 : stage + 1;
    } else if constexpr (HOLD) {
      load(r + step, nx, nd);
    }
    const uint64_t mm = f2_pack(-mean, -mean), rr = f2_pack(rstd, rstd);
    uint64_t n[P], d[P], s0 = 0, s1 = 0;
    unpack_pairs<T, V, NV>(cx, n);
    unpack_pairs<T, V, NV>(cd, d);
#pragma unroll
    for (int i = 0; i < P; ++i) {
      n[i] = f2_mul(f2_add(n[i], mm), rr);
      acc_s[i] = f2_fma(d[i], n[i], acc_s[i]);
      acc_b[i] = f2_add(acc_b[i], d[i]);
      d[i] = f2_mul(d[i], HOLD ? w[HOLD ? i : 0] : param(i));
      s0 = f2_add(s0, d[i]);
      s1 = f2_fma(d[i], n[i], s1);
    }
    if (dx) {
      float s[2] = {pair_sum(s0), pair_sum(s1)};
      row_sum<L, 2>(s, red, slot);
      if (r < p.rows) {
        const float mg = s[0] * -inv_c, mgn = s[1] * -inv_c;
        const uint64_t mg2 = f2_pack(mg, mg), mgn2 = f2_pack(mgn, mgn);
        float o[2 * P];
#pragma unroll
        for (int i = 0; i < P; ++i)
          f2_unpack(f2_mul(f2_fma(n[i], mgn2, f2_add(d[i], mg2)), rr), o[2 * i], o[2 * i + 1]);
#pragma unroll
        for (int j = 0; j < NV; ++j)
          if (in[j]) raw_store<T, V>(dx + r * p.dx_stride + (j * L + lane) * V, raw_pack<T, V>(o + j * V));
      }
    }
    if constexpr (HOLD && !RING) {
#pragma unroll
      for (int j = 0; j < NV; ++j) cx[j] = nx[j], cd[j] = nd[j];
    } else if constexpr (!RING) {
      load(r + step, cx, cd);
    }
    if constexpr (!RING) mean = nmean, rstd = nrstd;
  }
  if (!p.part && !p.cluster) return;
  float* shared_part = reinterpret_cast<float*>(ring + kNormSmem<V, L, NV, 2> / 16);
  float* out = p.cluster ? shared_part : p.part + int64_t(blockIdx.x) * 2 * p.c;
  float as[2 * P], ab[2 * P];
#pragma unroll
  for (int i = 0; i < P; ++i) {
    f2_unpack(acc_s[i], as[2 * i], as[2 * i + 1]);
    f2_unpack(acc_b[i], ab[2 * i], ab[2 * i + 1]);
  }
  if constexpr (GROUPS == 1) {
#pragma unroll
    for (int i = 0; i < E; ++i) {
      if (!in[i / V]) continue;
      const int col = ((i / V) * L + lane) * V + i % V;
      out[col] = as[i];
      out[p.c + col] = ab[i];
    }
  } else {
    // The block's groups hold the same columns: lanes of one warp meet by
    // shuffles, then the eight warps in shared memory.
    constexpr int COLS = L * E;
    __shared__ float sums[8][2 * COLS];
    const int warp = threadIdx.x >> 5;
#pragma unroll
    for (int i = 0; i < E; ++i) {
#pragma unroll
      for (int o = L; o < 32; o <<= 1) {
        as[i] += __shfl_xor_sync(0xFFFFFFFFu, as[i], o);
        ab[i] += __shfl_xor_sync(0xFFFFFFFFu, ab[i], o);
      }
      if ((threadIdx.x & 31) < L) {
        const int col = ((i / V) * L + lane) * V + i % V;
        sums[warp][col] = as[i];
        sums[warp][COLS + col] = ab[i];
      }
    }
    __syncthreads();
    for (int k = threadIdx.x; k < 2 * COLS; k += 256) {
      const int col = k % COLS;
      if (col >= p.c) continue;
      float t = 0.0f;
#pragma unroll
      for (int g = 0; g < 8; ++g) t += sums[g][k];
      out[(k / COLS) * p.c + col] = t;
    }
  }
  if (!p.cluster) return;
  sm100::cluster_sync_all();
  for (int k = int(blockIdx.x * blockDim.x + threadIdx.x); k < 2 * p.c; k += p.cluster * int(blockDim.x)) {
    float t = 0.0f;
    for (int b = 0; b < p.cluster; ++b) t += sm100::cluster_ld(sm100::map_rank(shared_part + k, b));
    void* o = k < p.c ? p.dscale : p.dbias;
    if (o) param_put<T>(o, p.param_f32, k < p.c ? k : k - p.c, t);
  }
  sm100::cluster_sync_all();  // no block leaves while another reads its sums
}

// The input gradient of rows too long for registers (two readings of x and dy).
template <class T, int V>
__global__ void __launch_bounds__(512) layer_norm_dx_long_kernel(NormBwd p) {
  sm100::pdl_wait();
  __shared__ float red[2][64];
  int slot = 0;
  const T *x = static_cast<const T*>(p.x), *dy = static_cast<const T*>(p.dy);
  T* dx = static_cast<T*>(p.dx);
  for (int64_t r = blockIdx.x; r < p.rows; r += gridDim.x) {
    const T *xr = x + r * p.x_stride, *dr = dy + r * p.dy_stride;
    const float mean = p.mean[r], rstd = p.rstd[r];
    float xv[V], dv[V], s[2] = {0.0f, 0.0f};
    for (int i = threadIdx.x * V; i < p.c; i += 512 * V) {
      raw_unpack<T, V>(raw_load<T, V>(xr + i), xv);
      raw_unpack<T, V>(raw_load<T, V>(dr + i), dv);
#pragma unroll
      for (int k = 0; k < V; ++k) {
        const float g = dv[k] * param_at<T>(p.scale, p.param_f32, i + k);
        s[0] += g;
        s[1] = fmaf(g, (xv[k] - mean) * rstd, s[1]);
      }
    }
    row_sum<512, 2>(s, red, slot);
    const float mg = s[0] / float(p.c), mgn = s[1] / float(p.c);
    for (int i = threadIdx.x * V; i < p.c; i += 512 * V) {
      raw_unpack<T, V>(raw_load<T, V>(xr + i), xv);
      raw_unpack<T, V>(raw_load<T, V>(dr + i), dv);
#pragma unroll
      for (int k = 0; k < V; ++k)
        xv[k] = rstd * (fmaf(dv[k], param_at<T>(p.scale, p.param_f32, i + k), -mg) - (xv[k] - mean) * rstd * mgn);
      raw_store<T, V>(dx + r * p.dx_stride + i, raw_pack<T, V>(xv));
    }
  }
}

// The parameter gradients' partial rows for such rows: a block takes 32 V
// columns (32 threads across, 8 rows at a time) of a range of rows.
template <class T, int V>
__global__ void __launch_bounds__(256) layer_norm_param_long_kernel(NormBwd p) {
  sm100::pdl_wait();
  __shared__ float sums[8][2 * 32 * V];
  const int lane = threadIdx.x & 31, sub = threadIdx.x >> 5;
  const int col = (blockIdx.x * 32 + lane) * V;
  const T *x = static_cast<const T*>(p.x), *dy = static_cast<const T*>(p.dy);
  float a[V], b[V];
#pragma unroll
  for (int k = 0; k < V; ++k) a[k] = b[k] = 0.0f;
  if (col < p.c) {
    for (int64_t r = int64_t(blockIdx.y) * 8 + sub; r < p.rows; r += int64_t(gridDim.y) * 8) {
      float xv[V], dv[V];
      raw_unpack<T, V>(raw_load<T, V>(x + r * p.x_stride + col), xv);
      raw_unpack<T, V>(raw_load<T, V>(dy + r * p.dy_stride + col), dv);
      const float mean = p.mean[r], rstd = p.rstd[r];
#pragma unroll
      for (int k = 0; k < V; ++k) {
        a[k] = fmaf(dv[k], (xv[k] - mean) * rstd, a[k]);
        b[k] += dv[k];
      }
    }
  }
#pragma unroll
  for (int k = 0; k < V; ++k) sums[sub][lane * V + k] = a[k], sums[sub][32 * V + lane * V + k] = b[k];
  __syncthreads();
  for (int i = threadIdx.x; i < 2 * 32 * V; i += 256) {
    const int cc = blockIdx.x * 32 * V + i % (32 * V);
    if (cc >= p.c) continue;
    float t = 0.0f;
#pragma unroll
    for (int g = 0; g < 8; ++g) t += sums[g][i];
    p.part[(int64_t(blockIdx.y) * 2 + i / (32 * V)) * p.c + cc] = t;
  }
}

// Add `nb` partial rows of `cols` columns. Columns below `split` go to out0,
// the rest to out1 (a null output's columns are skipped). A block takes 32
// columns; its 8 or 32 rows of threads each add every 8th or 32nd partial row,
// and meet in shared memory: the order of the sum depends on nb alone.
template <class T, int R>
__global__ void __launch_bounds__(32 * R)
    column_join_kernel(const float* part, int nb, int64_t cols, int64_t split, void* out0, void* out1, int out_f32) {
  sm100::pdl_wait();
  __shared__ float sums[R][33];
  const int lane = threadIdx.x & 31, sub = threadIdx.x >> 5;
  const int64_t col = int64_t(blockIdx.x) * 32 + lane;
  float t = 0.0f;
  if (col < cols) {
    int b = sub;
    for (; b + 7 * R < nb; b += 8 * R) {
      float v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = part[int64_t(b + i * R) * cols + col];
      t += ((v[0] + v[1]) + (v[2] + v[3])) + ((v[4] + v[5]) + (v[6] + v[7]));
    }
    float v[7];
#pragma unroll
    for (int i = 0; i < 7; ++i) v[i] = b + i * R < nb ? part[int64_t(b + i * R) * cols + col] : 0.0f;
    t += ((v[0] + v[1]) + (v[2] + v[3])) + ((v[4] + v[5]) + v[6]);
  }
  sums[sub][lane] = t;
  __syncthreads();
#pragma unroll
  for (int h = R / 2; h > 0; h >>= 1) {
    if (sub < h) sums[sub][lane] += sums[sub + h][lane];
    __syncthreads();
  }
  if (sub == 0 && col < cols) {
    void* o = col < split ? out0 : out1;
    if (o) param_put<T>(o, out_f32, col < split ? col : col - split, sums[0][lane]);
  }
}

}  // namespace mx
