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
// results do not change from run to run).
#pragma once

#include "kernels_vec.cuh"

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
  float* part;  // [gridDim.x][2][c] partial sums of dscale and dbias; null: not wanted
  int64_t rows, dy_stride, x_stride, dx_stride;
  int c;
  int param_f32;
};

// Sum over the L lanes of a row. For L > 32 the warps' sums meet in `red`
// (two slots alternate, so one barrier a sum is enough: a warp can only be
// one sum ahead of another).
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
    for (int k = 0; k < K; ++k) {
      float t = lane < W ? r[lane * K + k] : 0.0f;
#pragma unroll
      for (int o = W / 2; o > 0; o >>= 1) t += __shfl_xor_sync(0xFFFFFFFFu, t, o);
      s[k] = __shfl_sync(0xFFFFFFFFu, t, 0);
    }
  }
}

template <int L>
constexpr int kNormThreads = L <= 32 ? 256 : L;
// Up to 16 values a thread the parameters and the next row fit in registers too.
template <int V, int NV>
constexpr bool kNormHold = V * NV <= 16;

template <class T, int V, int L, int NV>
__global__ void __launch_bounds__(kNormThreads<L>) layer_norm_kernel(NormFwd p) {
  constexpr int E = V * NV;
  constexpr bool HOLD = kNormHold<V, NV>;
  constexpr int GROUPS = kNormThreads<L> / L;
  __shared__ float red[2][32];
  int slot = 0;
  const int lane = threadIdx.x % L;
  const T* x = static_cast<const T*>(p.x);
  T* y = static_cast<T*>(p.y);
  const float inv_c = 1.0f / float(p.c);
  bool in[NV];
#pragma unroll
  for (int j = 0; j < NV; ++j) in[j] = (j * L + lane) * V < p.c;
  float w[HOLD ? E : 1], b[HOLD ? E : 1];
  if constexpr (HOLD) {
#pragma unroll
    for (int i = 0; i < E; ++i) {
      const int col = ((i / V) * L + lane) * V + i % V;
      w[i] = in[i / V] ? param_at<T>(p.scale, p.param_f32, col) : 0.0f;
      b[i] = in[i / V] ? param_at<T>(p.bias, p.param_f32, col) : 0.0f;
    }
  }
  auto load = [&](int64_t r, Raw<T, V>(&q)[NV]) {
#pragma unroll
    for (int j = 0; j < NV; ++j)
      q[j] = r < p.rows && in[j] ? raw_load<T, V>(x + r * p.x_stride + (j * L + lane) * V) : raw_zero<T, V>();
  };
  const int64_t step = int64_t(gridDim.x) * GROUPS;
  Raw<T, V> cur[NV];
  load(int64_t(blockIdx.x) * GROUPS + threadIdx.x / L, cur);
  for (int64_t base = int64_t(blockIdx.x) * GROUPS; base < p.rows; base += step) {
    const int64_t r = base + threadIdx.x / L;
    Raw<T, V> next[HOLD ? NV : 1];
    if constexpr (HOLD) load(r + step, next);
    float v[E], s[1] = {0.0f};
#pragma unroll
    for (int j = 0; j < NV; ++j) raw_unpack<T, V>(cur[j], v + j * V);
#pragma unroll
    for (int i = 0; i < E; ++i) s[0] += v[i];
    row_sum<L, 1>(s, red, slot);
    // Rounded on its own: contracted into the subtractions below it would not be the mean that is stored.
    const float mean = __fmul_rn(s[0], inv_c);
    float q[1] = {0.0f};
#pragma unroll
    for (int i = 0; i < E; ++i) {
      v[i] = in[i / V] ? v[i] - mean : 0.0f;
      q[0] = fmaf(v[i], v[i], q[0]);
    }
    row_sum<L, 1>(q, red, slot);
    const float rstd = 1.0f / sqrtf(fmaf(q[0], inv_c, p.eps));
    if (r < p.rows) {
      if (lane == 0) {
        if (p.mean) p.mean[r] = mean;
        if (p.rstd) p.rstd[r] = rstd;
      }
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        if (!in[j]) continue;
        const int col = (j * L + lane) * V;
        float o[V];
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float wi = HOLD ? w[HOLD ? j * V + i : 0] : param_at<T>(p.scale, p.param_f32, col + i);
          const float bi = HOLD ? b[HOLD ? j * V + i : 0] : param_at<T>(p.bias, p.param_f32, col + i);
          o[i] = fmaf(v[j * V + i] * rstd, wi, bi);
        }
        raw_store<T, V>(y + r * p.y_stride + col, raw_pack<T, V>(o));
      }
    }
    if constexpr (HOLD) {
#pragma unroll
      for (int j = 0; j < NV; ++j) cur[j] = next[j];
    } else {
      load(r + step, cur);
    }
  }
}

// Rows too long for a block's registers: the row is read three times, the
// second and third time from the caches (a block's row is at most a few
// hundred KB of the 126 MB L2).
template <class T, int V>
__global__ void __launch_bounds__(512) layer_norm_long_kernel(NormFwd p) {
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
__global__ void __launch_bounds__(kNormThreads<L>) layer_norm_backward_kernel(NormBwd p) {
  constexpr int E = V * NV;
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
  float w[HOLD ? E : 1], acc_s[E], acc_b[E];
#pragma unroll
  for (int i = 0; i < E; ++i) acc_s[i] = acc_b[i] = 0.0f;
  if constexpr (HOLD) {
#pragma unroll
    for (int i = 0; i < E; ++i)
      w[i] = in[i / V] ? param_at<T>(p.scale, p.param_f32, ((i / V) * L + lane) * V + i % V) : 0.0f;
  }
  auto load = [&](int64_t r, Raw<T, V>(&q)[NV], Raw<T, V>(&d)[NV], float& mean, float& rstd) {
    const bool on = r < p.rows;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int col = (j * L + lane) * V;
      q[j] = on && in[j] ? raw_load<T, V>(x + r * p.x_stride + col) : raw_zero<T, V>();
      d[j] = on && in[j] ? raw_load<T, V>(dy + r * p.dy_stride + col) : raw_zero<T, V>();
    }
    // A row past the last has dy = 0 and rstd = 0: it adds nothing.
    mean = on ? p.mean[r] : 0.0f;
    rstd = on ? p.rstd[r] : 0.0f;
  };
  const int64_t step = int64_t(gridDim.x) * GROUPS;
  Raw<T, V> cx[NV], cd[NV];
  float mean, rstd;
  load(int64_t(blockIdx.x) * GROUPS + threadIdx.x / L, cx, cd, mean, rstd);
  for (int64_t base = int64_t(blockIdx.x) * GROUPS; base < p.rows; base += step) {
    const int64_t r = base + threadIdx.x / L;
    Raw<T, V> nx[HOLD ? NV : 1], nd[HOLD ? NV : 1];
    float nmean = 0.0f, nrstd = 0.0f;
    if constexpr (HOLD) load(r + step, nx, nd, nmean, nrstd);
    float s[2] = {0.0f, 0.0f};
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      float xv[V], dv[V];
      raw_unpack<T, V>(cx[j], xv);
      raw_unpack<T, V>(cd[j], dv);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const int e = j * V + i;
        const float n = (xv[i] - mean) * rstd;
        const float we = HOLD ? w[HOLD ? e : 0]
                              : (in[j] ? param_at<T>(p.scale, p.param_f32, (j * L + lane) * V + i) : 0.0f);
        if (in[j]) acc_s[e] = fmaf(dv[i], n, acc_s[e]);
        acc_b[e] += dv[i];
        const float g = dv[i] * we;
        s[0] += g;
        if (in[j]) s[1] = fmaf(g, n, s[1]);
      }
    }
    if (dx) {
      row_sum<L, 2>(s, red, slot);
      const float mg = s[0] * inv_c, mgn = s[1] * inv_c;
      if (r < p.rows) {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
          if (!in[j]) continue;
          float xv[V], dv[V];
          raw_unpack<T, V>(cx[j], xv);
          raw_unpack<T, V>(cd[j], dv);
          const int col = (j * L + lane) * V;
#pragma unroll
          for (int i = 0; i < V; ++i) {
            const float we = HOLD ? w[HOLD ? j * V + i : 0] : param_at<T>(p.scale, p.param_f32, col + i);
            const float n = (xv[i] - mean) * rstd;
            xv[i] = rstd * (fmaf(dv[i], we, -mg) - n * mgn);
          }
          raw_store<T, V>(dx + r * p.dx_stride + col, raw_pack<T, V>(xv));
        }
      }
    }
    if constexpr (HOLD) {
#pragma unroll
      for (int j = 0; j < NV; ++j) cx[j] = nx[j], cd[j] = nd[j];
      mean = nmean, rstd = nrstd;
    } else {
      load(r + step, cx, cd, mean, rstd);
    }
  }
  if (!p.part) return;
  float* out = p.part + int64_t(blockIdx.x) * 2 * p.c;
  if constexpr (GROUPS == 1) {
#pragma unroll
    for (int i = 0; i < E; ++i) {
      if (!in[i / V]) continue;
      const int col = ((i / V) * L + lane) * V + i % V;
      out[col] = acc_s[i];
      out[p.c + col] = acc_b[i];
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
        acc_s[i] += __shfl_xor_sync(0xFFFFFFFFu, acc_s[i], o);
        acc_b[i] += __shfl_xor_sync(0xFFFFFFFFu, acc_b[i], o);
      }
      if ((threadIdx.x & 31) < L) {
        const int col = ((i / V) * L + lane) * V + i % V;
        sums[warp][col] = acc_s[i];
        sums[warp][COLS + col] = acc_b[i];
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
}

// The input gradient of rows too long for registers (two readings of x and dy).
template <class T, int V>
__global__ void __launch_bounds__(512) layer_norm_dx_long_kernel(NormBwd p) {
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
  __shared__ float sums[R][33];
  const int lane = threadIdx.x & 31, sub = threadIdx.x >> 5;
  const int64_t col = int64_t(blockIdx.x) * 32 + lane;
  float t = 0.0f;
  if (col < cols) {
    int b = sub;
    for (; b + 3 * R < nb; b += 4 * R) {
      const float v0 = part[int64_t(b) * cols + col], v1 = part[int64_t(b + R) * cols + col];
      const float v2 = part[int64_t(b + 2 * R) * cols + col], v3 = part[int64_t(b + 3 * R) * cols + col];
      t += (v0 + v1) + (v2 + v3);
    }
    for (; b < nb; b += R) t += part[int64_t(b) * cols + col];
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
