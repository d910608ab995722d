// The dense product of a caller's matrices, forward and backward:
//
//   pre = x w^T + bias,  y = act(pre) + residual        x [m][k], w [n][k], y [m][n]
//   d = dy act'(pre),  dx = d w,  dw = d^T x,  db = sum_rows d
//
// The three products are one tensor-core kernel over D[i][j] = sum_k A(i, k) B(j, k),
// whose operands may each lie k-contiguous (K-major) or i- / j-contiguous
// (MN-major): forward is K-major times K-major, dx takes w MN-major, and dw
// takes both MN-major, so nothing is transposed in memory.
#pragma once

#include <cuda.h>

#include <type_traits>

#include "drain.h"
#include "gpu_common.cuh"
#include "kernels_vec.cuh"
#include "sm100.cuh"

namespace mx {

// ------------------------------------------------------------- activations
__device__ __forceinline__ float act_value(int act, float v, float slope) {
  switch (act) {
    case MX_ACT_GELU: return gelu_f(v);
    case MX_ACT_LRELU: return v >= 0.0f ? v : slope * v;
    case MX_ACT_SIGMOID: return sigmoid_f(v);
    default: return v;
  }
}

// d/dx [x Phi(x)] = Phi(x) + x phi(x). With u = |x|, Phi(-u) = exp(-u^2 / 2) R(u)
// as in gelu_f and phi(x) = c exp(-u^2 / 2), c = 1 / sqrt(2 pi), both terms share
// the exponential: with t = exp(-u^2 / 2) (R(u) - c u) the derivative is t for
// x < 0 and 1 - t otherwise, and R(u) - c u is R's polynomial with another
// linear coefficient. (u is clamped to 5.6 as for R; past it the exponential
// leaves nothing, and an infinite x gives no inf * 0.) On two values at once.
__device__ __forceinline__ void gelu_grad_f2(float a, float b, float& ga, float& gb) {
  const uint64_t x = f2_pack(a, b);
  const uint64_t q = gelu_r2(f2_pack(fmaxf(-fabsf(a), -5.6f), fmaxf(-fabsf(b), -5.6f)), 0.3989422804f);
  float ta, tb;
  f2_unpack(f2_mul(f2_mul(x, f2_pack(-0.72134752f, -0.72134752f)), x), ta, tb);
  f2_unpack(f2_mul(f2_pack(ex2_approx(ta), ex2_approx(tb)), q), ta, tb);
  ga = a < 0.0f ? ta : 1.0f - ta;
  gb = b < 0.0f ? tb : 1.0f - tb;
}
// v[i] *= act'(q[i]).
template <int N>
__device__ __forceinline__ void apply_act_grad(int act, float* v, const float* q, float slope) {
  if (act == MX_ACT_GELU) {
    if constexpr (N > 1) {
#pragma unroll
      for (int i = 0; i < N; i += 2) {
        float a, b;
        gelu_grad_f2(q[i], q[i + 1], a, b);
        v[i] *= a, v[i + 1] *= b;
      }
    } else {
      float g, unused;
      gelu_grad_f2(q[0], 0.0f, g, unused);
      v[0] *= g;
    }
  } else if (act == MX_ACT_LRELU) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] *= q[i] >= 0.0f ? 1.0f : slope;
  } else if (act == MX_ACT_SIGMOID) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float s = sigmoid_f(q[i]);
      v[i] *= s * (1.0f - s);
    }
  }
}

// ----------------------------------------------------------- the epilogue
// What happens to a sum before it is stored. With `part` set the product is
// one of several partial sums over K: they are stored as they are, and
// dense_join_kernel adds them and does the rest.
struct DenseEpi {
  const void* bias;      // [n] or null
  const void* residual;  // [m][n] or null
  void* y;
  void* pre;  // null: not stored
  int64_t residual_stride, y_stride, pre_stride;
  int act;
  float slope;
  int vec_residual, vec_y, vec_pre, vec_bias;  // 16-byte aligned rows
  float* part;                       // [splits][m][ldp] or null
  int64_t ldp;                       // a multiple of 8
};

// Eight consecutive elements of a row, `valid` of which exist.
template <class T>
__device__ __forceinline__ void load8(const T* p, bool vec, int valid, float (&v)[8]) {
  if (vec && valid >= 8) {
#pragma unroll
    for (int h = 0; h < 8; h += kVec<T>) raw_unpack<T, kVec<T>>(raw_load<T, kVec<T>>(p + h), v + h);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < valid ? to_f(p[i]) : 0.0f;
  }
}
template <class T>
__device__ __forceinline__ void store8(T* p, bool vec, int valid, const float (&v)[8]) {
  if (vec && valid >= 8) {
#pragma unroll
    for (int h = 0; h < 8 / kVec<T>; ++h) raw_store<T, kVec<T>>(p + h * kVec<T>, raw_pack<T, kVec<T>>(v + h * kVec<T>));
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < valid) p[i] = from_f<T>(v[i]);
  }
}

// Bias, activation and residual of eight sums of one row, and their stores.
template <class T>
__device__ __forceinline__ void dense_finish(const DenseEpi& e, float (&v)[8], const float (&bias)[8], int64_t row,
                                             int64_t col, int valid) {
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] += bias[i];
  if (e.pre) store8(static_cast<T*>(e.pre) + row * e.pre_stride + col, e.vec_pre, valid, v);
  if (e.act == MX_ACT_GELU) {
#pragma unroll
    for (int i = 0; i < 8; i += 2) gelu_f2(v[i], v[i + 1]);
  } else if (e.act != MX_ACT_NONE) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = act_value(e.act, v[i], e.slope);
  }
  if (e.residual) {
    float r[8];
    load8(static_cast<const T*>(e.residual) + row * e.residual_stride + col, e.vec_residual, valid, r);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] += r[i];
  }
  store8(static_cast<T*>(e.y) + row * e.y_stride + col, e.vec_y, valid, v);
}
template <class T>
__device__ __forceinline__ void load_bias(const DenseEpi& e, int64_t col, int valid, float (&b)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) b[i] = e.bias && i < valid ? to_f(static_cast<const T*>(e.bias)[col + i]) : 0.0f;
}

// Sum of the partial products and the epilogue: a thread per 8 columns of a
// row and, where there are few of those and many splits, `GROUPS` threads that
// each add every GROUPS-th split and meet in shared memory. The order of a sum
// depends on the number of splits alone.
template <class T, int GROUPS>
__global__ void __launch_bounds__(256) dense_join_kernel(DenseEpi e, int splits, int64_t m, int64_t n) {
  sm100::pdl_wait();
  constexpr int PER = 256 / GROUPS;
  __shared__ float sums[GROUPS > 1 ? GROUPS : 1][GROUPS > 1 ? PER * 8 : 1];
  const int64_t cols8 = (n + 7) / 8;
  const int own = threadIdx.x % PER, group = threadIdx.x / PER;
  for (int64_t i0 = int64_t(blockIdx.x) * PER; i0 < m * cols8; i0 += int64_t(gridDim.x) * PER) {
    const int64_t i = i0 + own, row = i / cols8, col = (i % cols8) * 8;
    const int valid = int(n - col < 8 ? n - col : 8);
    float v[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    if (i < m * cols8) {
#pragma unroll 8
      for (int s = group; s < splits; s += GROUPS) {
        const float4* p = reinterpret_cast<const float4*>(e.part + (int64_t(s) * m + row) * e.ldp + col);
        const float4 a = p[0], c = p[1];
        v[0] += a.x, v[1] += a.y, v[2] += a.z, v[3] += a.w;
        v[4] += c.x, v[5] += c.y, v[6] += c.z, v[7] += c.w;
      }
    }
    if constexpr (GROUPS > 1) {
#pragma unroll
      for (int k = 0; k < 8; ++k) sums[group][k * PER + own] = v[k];
      __syncthreads();
      if (group == 0) {
#pragma unroll
        for (int g = 1; g < GROUPS; ++g)
#pragma unroll
          for (int k = 0; k < 8; ++k) v[k] += sums[g][k * PER + own];
      }
      __syncthreads();
    }
    if (group == 0 && i < m * cols8) {
      float b[8];
      load_bias<T>(e, col, valid, b);
      dense_finish<T>(e, v, b, row, col, valid);
    }
  }
}

// ---------------------------------------------------- a few rows (decoding)
// Up to R <= 8 rows of x. Then the weights are nearly all the bytes, each used
// R times: a warp streams CPW weight rows at once (CPW 16-byte loads in
// flight a lane) against the rows of x, which stay in the caches, with fp32
// FMAs. Where there are few columns the KS warps of a group share the same
// columns, each taking every KS-th vector of K, and meet in shared memory.
template <class T, int R, int V, int CPW>
__global__ void __launch_bounds__(256)
    dense_rows_kernel(const T* x, int64_t x_stride, const T* w, int64_t w_stride, DenseEpi e, int m, int n, int k,
                      int ks) {
  sm100::pdl_wait();
  __shared__ float red[8][R * CPW];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int part = warp % ks;
  const int64_t col0 = (int64_t(blockIdx.x) * (blockDim.x / 32 / ks) + warp / ks) * CPW;
  float acc[R][CPW];
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int c = 0; c < CPW; ++c) acc[r][c] = 0.0f;
  if (col0 < n) {
    // Columns past the last and rows past the last read an existing one; their sums are not stored.
    const T* wp[CPW];
#pragma unroll
    for (int c = 0; c < CPW; ++c) wp[c] = w + (col0 + c < n ? col0 + c : int64_t(n) - 1) * w_stride;
#pragma unroll 2
    for (int i = (part * 32 + lane) * V; i < k; i += ks * 32 * V) {
      Raw<T, V> wr[CPW];
#pragma unroll
      for (int c = 0; c < CPW; ++c) wr[c] = raw_load_once<T, V>(wp[c] + i);
      float xv[R][V];
#pragma unroll
      for (int r = 0; r < R; ++r)
        raw_unpack<T, V>(raw_load<T, V>(x + int64_t(r < m ? r : m - 1) * x_stride + i), xv[r]);
#pragma unroll
      for (int c = 0; c < CPW; ++c) {
        float wv[V];
        raw_unpack<T, V>(wr[c], wv);
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
          for (int j = 0; j < V; ++j) acc[r][c] = fmaf(xv[r][j], wv[j], acc[r][c]);
      }
    }
  }
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int c = 0; c < CPW; ++c) {
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) acc[r][c] += __shfl_xor_sync(0xFFFFFFFFu, acc[r][c], o);
      if (lane == 0) red[warp][r * CPW + c] = acc[r][c];
    }
  __syncthreads();
  if (part == 0 && lane < R * CPW) {
    const int r = lane / CPW, c = lane % CPW;
    const int64_t col = col0 + c;
    if (r < m && col < n) {
      float v = 0.0f;
      for (int s = 0; s < ks; ++s) v += red[warp + s][lane];
      if (e.bias) v += to_f(static_cast<const T*>(e.bias)[col]);
      if (e.pre) static_cast<T*>(e.pre)[r * e.pre_stride + col] = from_f<T>(v);
      v = act_value(e.act, v, e.slope);
      if (e.residual) v += to_f(static_cast<const T*>(e.residual)[r * e.residual_stride + col]);
      static_cast<T*>(e.y)[r * e.y_stride + col] = from_f<T>(v);
    }
  }
}

// ------------------------------------------ the pre-activation's gradient
// d = dy act'(pre) and the partial column sums of d (over fp32 values, before
// d is rounded to the operands' type for the two products). A block takes
// lx V columns (lx = 32, or fewer lanes where the matrix is narrow) of a range of
// rows, 256 / lx rows at a time. Without STORE (no product wants d, or act is none and
// d is dy) nothing is written but the sums. GELU's derivative is about 17 instructions an element, which in 16
// bits is as long as the memory's time. Where d is stored, what is read here leaves
// the L2 first, so that more of d is still there for the products (gradients from 1000
// x 256 -> 1024 to 8192 x 4096 -> 4096 in each type: 0.97 to 1.00 of the time with
// ordinary loads, 1.01 for the smallest). The sums alone take 1.02 of their time with
// such loads, and have an instance without: a choice inside the loop costs as much.
template <class T, int V, bool STORE>
__global__ void __launch_bounds__(256, 3)
    dense_grad_kernel(const T* dy, int64_t dy_stride, const T* pre, int64_t pre_stride, T* d, int64_t d_stride,
                      float* part, T* db, int64_t m, int n, int lx_log2, int act, float slope) {
  sm100::pdl_wait();
  __shared__ float sums[256 * V];
  __shared__ float total[32 * V];
  const int lx = 1 << lx_log2, subs = 256 >> lx_log2;
  const int lane = threadIdx.x & (lx - 1), sub = threadIdx.x >> lx_log2;
  const int col = (blockIdx.x * lx + lane) * V;
  float a[V];
#pragma unroll
  for (int k = 0; k < V; ++k) a[k] = 0.0f;
  if (col < n) {
    // AHEAD rows' loads are on their way before the first is worked on.
    constexpr int AHEAD = 4;
    const int64_t step = int64_t(gridDim.y) * subs;
    for (int64_t r0 = int64_t(blockIdx.y) * subs + sub; r0 < m; r0 += AHEAD * step) {
      Raw<T, V> dr[AHEAD], pr[AHEAD];
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) {
        const int64_t r = r0 + i * step;
        if constexpr (STORE) {
          dr[i] = r < m ? raw_load_streaming<T, V>(dy + r * dy_stride + col) : raw_zero<T, V>();
          pr[i] = r < m ? raw_load_streaming<T, V>(pre + r * pre_stride + col) : raw_zero<T, V>();
        } else {
          dr[i] = r < m ? raw_load<T, V>(dy + r * dy_stride + col) : raw_zero<T, V>();
          if (act != MX_ACT_NONE) pr[i] = r < m ? raw_load<T, V>(pre + r * pre_stride + col) : raw_zero<T, V>();
        }
      }
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) {
        const int64_t r = r0 + i * step;
        float v[V];
        raw_unpack<T, V>(dr[i], v);
        if (STORE || act != MX_ACT_NONE) {
          float q[V];
          raw_unpack<T, V>(pr[i], q);
          apply_act_grad<V>(act, v, q, slope);
          if (STORE && r < m) raw_store<T, V>(d + r * d_stride + col, raw_pack<T, V>(v));
        }
#pragma unroll
        for (int k = 0; k < V; ++k) a[k] = __fadd_rn(a[k], v[k]);  // not contracted: the same sums with STORE and without
      }
    }
  }
  if (!part && !db) return;
#pragma unroll
  for (int k = 0; k < V; ++k) sums[sub * lx * V + lane * V + k] = a[k];
  __syncthreads();
  for (int i = threadIdx.x; i < lx * V; i += 256) {
    const int cc = blockIdx.x * lx * V + i;
    if (cc >= n) continue;
    float t = 0.0f;
#pragma unroll 8
    for (int g = 0; g < subs; ++g) t += sums[g * lx * V + i];
    if (part)
      part[int64_t(blockIdx.y) * n + cc] = t;
    else
      total[i] = t;
  }
  if (part) return;
  // A few rows: the row ranges are one cluster, whose first block adds their sums.
  sm100::cluster_sync_all();
  if (blockIdx.y == 0) {
    for (int i = threadIdx.x; i < lx * V; i += 256) {
      const int cc = blockIdx.x * lx * V + i;
      if (cc >= n) continue;
      float t = 0.0f;
      for (unsigned b = 0; b < gridDim.y; ++b) t += sm100::cluster_ld(sm100::map_rank(&total[i], b));
      db[cc] = from_f<T>(t);
    }
  }
  sm100::cluster_sync_all();  // no block leaves while its sums are read
}

// Copies of matrices whose rows are not 16-byte aligned into ones whose rows
// are (what the tensor maps need), all that a call needs in one launch. One
// thread per 16 bytes of a copy; matrix i has the blocks from first[i] on.
struct DenseAlign {
  static constexpr int MAX = 3;
  const void* src[MAX];
  void* dst[MAX];
  int64_t src_stride[MAX], dst_stride[MAX], rows[MAX], cols[MAX];
  unsigned first[MAX + 1];
  int count;
};
template <class T>
__global__ void __launch_bounds__(256) dense_align_kernel(const __grid_constant__ DenseAlign a) {
  sm100::pdl_wait();
  constexpr int V = kVec<T>;
  int m = 0;
  while (m + 1 < a.count && blockIdx.x >= a.first[m + 1]) ++m;
  const T* src = static_cast<const T*>(a.src[m]);
  T* dst = static_cast<T*>(a.dst[m]);
  const int64_t vecs = a.dst_stride[m] / V, total = a.rows[m] * vecs;
  const int64_t step = int64_t(a.first[m + 1] - a.first[m]) * 256;
  for (int64_t i = int64_t(blockIdx.x - a.first[m]) * 256 + threadIdx.x; i < total; i += step) {
    const int64_t r = i / vecs, c = (i % vecs) * V;
    float v[V];
#pragma unroll
    for (int k = 0; k < V; ++k) v[k] = c + k < a.cols[m] ? to_f(src[r * a.src_stride[m] + c + k]) : 0.0f;
    raw_store<T, V>(dst + r * a.dst_stride[m] + c, raw_pack<T, V>(v));
  }
}

// ------------------------------------------------- the tensor-core product
// G CTAs (one, or a pair as cta_group::2) compute a tile of 128 G x BN: each
// loads 128 rows of A and BN / G rows of B and holds 128 accumulator rows. A
// pair reads every B row into shared memory once for 256 rows of A: the
// operands' way through shared memory is what bounds the one-CTA form
// (8192 x 4096 -> 8192 bf16: 418 us with one CTA a tile, 363 with two).
// One CTA per SM, persistent over the tiles. Warp roles:
//   warp 0       TMA producer: 128 bytes of K (64 or 32 elements) a stage
//   warp 1       MMA issuer (one lane, of the pair's leader; the peer's passes on
//                that its lo tiles are written)
//   warp 2       TMEM owner
//   warps 4-19   epilogue: TMEM -> registers -> bias, activation, residual ->
//   (or 4-11)    shared memory -> TMA store; four (two) warps per TMEM lane
//                quarter share the tile's columns
//   then four    fp32 only: the TF32 split (as in the executor's kernels:
//                the fp32 tile itself is hi, read truncated to TF32; these
//                warps write lo = x - hi to a ring beside it)
// Two accumulator sets let the epilogue of one tile overlap the products of
// the next. In fp32 the cross terms hi*lo + lo*hi have a region of their own in
// a set where TMEM has room for it. The epilogue takes a set every CHUNK k-blocks
// and adds it up in registers: the tensor core truncates its accumulator at each
// MMA, about 1e-7 of a sum of one sign. In fp32 a few hundred of them cost more
// than the products' own rounding (the weights' gradient over 71,680 rows was off
// by 2.8e-6 of its size with 1,900 rows to a set, by 6.9e-7 with 256); in 16 bits
// a few thousand do (131,072 positive rows in one set: 7.8e-4 low, against fp16's
// rounding of 4.9e-4), and 256 of them lose 2.4e-5.
// Every wait is bounded in time; one that runs out records a code in the
// status word and raises the abort flag of both CTAs, on which the other roles
// stop. The kernel then lets its MMAs end and its copies land, by waits that the
// flag does not cut short (only their own limit does), frees its TMEM and returns.
struct DenseMm {
  int64_t m, n;
  int kb;          // k-blocks
  int kb_split;    // k-blocks a split takes
  int splits;
  int tiles_m, tiles_n;
  DenseEpi epi;
  int* status;
};

enum : int { kDenseErrProducer = 0x201, kDenseErrSplit, kDenseErrMmaAcc, kDenseErrMmaStage, kDenseErrEpilogue, kDenseErrDrain };

template <class T, int BN, int G>
struct DenseCfg {
  static constexpr bool F32 = sizeof(T) == 4;
  static constexpr int BK = 128 / int(sizeof(T));
  static constexpr int BROWS = BN / G;  // rows of B a CTA loads
  static constexpr int A_BYTES = 128 * 128;
  static constexpr int B_BYTES = BROWS * 128;
  static constexpr int STAGE_BYTES = A_BYTES + B_BYTES;
  // fp32: the lo halves have a shorter ring of their own, so that more of the
  // shared memory holds loads in flight. A pair's is one longer, for the time that
  // word of the peer's takes (4096^3 658 to 621 us, 71680 x 128 -> 256 40.8 to 39.2).
  static constexpr int LO_STAGES = F32 ? (G == 2 ? 3 : 2) : 0;
  static constexpr int FIT = 192 * 1024 / STAGE_BYTES - LO_STAGES;
  static constexpr int STAGES = FIT < 8 ? FIT : 8;
  static constexpr int REGIONS = F32 && BN <= 128 ? 2 : 1;  // of an accumulator set: hi*hi and the cross terms, or one
  static constexpr int SET_COLS = REGIONS * BN;
  static constexpr int TMEM_COLS = 2 * SET_COLS;
  // k-blocks a set accumulates: in fp32 32 updates of hi*hi, or 24 of everything;
  // in 16 bits 256 updates, 4096 of K.
  static constexpr int CHUNK = !F32 ? 64 : (REGIONS == 2 ? 8 : 2);
  static constexpr int EPI_WARP0 = 4, EPI_WARPS = BN >= 128 ? 16 : 8;
  static constexpr int EPI_COLS = BN / (EPI_WARPS / 4);  // columns of a tile per epilogue warp
  static constexpr int SPLIT_WARP0 = EPI_WARP0 + EPI_WARPS, SPLIT_WARPS = F32 ? 4 : 0;
  static constexpr int THREADS = 32 * (SPLIT_WARP0 + SPLIT_WARPS);
  // fp32 with BN = 256: an epilogue lane's 64 sums need more registers than the
  // 80 that 768 threads launch with, the other warps less. In the six
  // warpgroups' sum: 40 + 4 x 96 + 48 = 472 of 480.
  static constexpr bool SPLIT_REGS = F32 && BN == 256;
  static constexpr int REGS_CONTROL = 40, REGS_EPI = 96, REGS_SPLIT = 48;
  static_assert(!SPLIT_REGS || (THREADS == 768 && REGS_CONTROL + 4 * REGS_EPI + REGS_SPLIT <= 480), "register split");
  static constexpr int STAGING_BYTES = EPI_WARPS * 2048;  // 32 rows x 64 bytes each
  static constexpr int SMEM_BYTES =
      1024 + (STAGES + LO_STAGES) * STAGE_BYTES + STAGING_BYTES + 8 * (2 * STAGES + 3 * LO_STAGES + 5) + 16;
  static_assert(SMEM_BYTES <= 232448 - 64, "shared memory per CTA");
  static_assert(TMEM_COLS <= 512, "TMEM columns");
};

// Output tile t: groups of 16 tile rows, column by column, so that the CTAs at
// work at one time share operand tiles in the L2 (8192 x 4096 -> 8192 bf16:
// 333 us with groups of 8, 324 with 16).
__device__ __forceinline__ void dense_tile(const DenseMm& p, int t, int& tm, int& tn) {
  const int per = 16 * p.tiles_n, g = t / per, in = t % per;
  const int rows = min(16, p.tiles_m - g * 16);
  tm = g * 16 + in % rows;
  tn = in / rows;
}

__device__ __forceinline__ float dense_residual(float v) {
  // lo = v - trunc(v), rounded to TF32 (half a TF32 ulp added; the tensor core
  // drops the low bits itself). An infinite v leaves a NaN, whose bits may be all
  // ones: the addition must not carry it past the sign.
  const float hi = __uint_as_float(__float_as_uint(v) & 0xFFFFE000u);
  return __int_as_float(min(__float_as_int(__fsub_rn(v, hi)), 0x7FFFEFFF) + 0x1000);
}

// The epilogue of a warp's 32 rows x 32 columns of sums, a row in each lane:
// bias, activation and residual there, 32 independent values a lane, then the
// block is packed into the warp's 2 KB staging buffer in the swizzle of a
// tensor map and leaves by TMA, which also clips it to the matrix. (Where K is
// short the epilogue sets the pace, by its warps' instruction latency: 71680 x
// 128 -> 256 fp32 with GELU and pre took 58-70 us with the block read back and
// stored by the lanes of 8 warps, 48 with TMA, 42 with 16 warps.) Matrices
// that a tensor map cannot take (unaligned rows) are written by the lanes, a
// column a lane.
template <class T>
struct DenseOut {
  static constexpr int V = kVec<T>;
  const DenseMm& p;
  const CUtensorMap *ty, *tpre;
  uint8_t* buf;
  int lane;

  // Columns [col0, col0 + 32) of a vector or of this lane's row; zero past n.
  __device__ __forceinline__ void row32(const T* q, bool vec, int64_t col0, float* v) const {
    if (vec && col0 + 32 <= p.n) {
#pragma unroll
      for (int i = 0; i < 32; i += V) raw_unpack<T, V>(raw_load<T, V>(q + col0 + i), v + i);
    } else {
#pragma unroll
      for (int i = 0; i < 32; ++i) v[i] = col0 + i < p.n ? to_f(q[col0 + i]) : 0.0f;
    }
  }
  __device__ __forceinline__ void bias(int64_t col0, float* v) const {
    if (p.epi.part || !p.epi.bias) {
#pragma unroll
      for (int i = 0; i < 32; ++i) v[i] = 0.0f;
    } else {
      row32(static_cast<const T*>(p.epi.bias), p.epi.vec_bias, col0, v);
    }
  }
  // 64 bytes a row of the block (32 columns, or 16 in fp32) into the buffer as U:
  // 16-byte chunk j of row r at j ^ (r / 2 % 4), which is the tensor maps'
  // 64-byte swizzle and free of bank conflicts.
  template <class U>
  __device__ __forceinline__ void stage(const float* v) {
    constexpr int W = kVec<U>;
    if (lane == 0) sm100::bulk_wait_read<0>();
    __syncwarp();
#pragma unroll
    for (int j = 0; j < 4; ++j)
      *reinterpret_cast<uint4*>(buf + lane * 64 + ((j ^ ((lane >> 1) & 3)) << 4)) = raw_pack<U, W>(v + j * W).u;
  }
  template <class U>
  __device__ __forceinline__ void emit(const CUtensorMap* map, const float* v, int64_t row0, int64_t col0, int z) {
    constexpr int COLS = 64 / int(sizeof(U));
#pragma unroll
    for (int h = 0; h < 32; h += COLS) {
      if (h > 0 && col0 + h >= p.n) break;
      stage<U>(v + h);
      sm100::fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) {
        sm100::tma_store_3d(map, buf, int(col0) + h, int(row0), z);
        sm100::bulk_commit();
      }
    }
  }
  __device__ __forceinline__ void put(T* out, int64_t stride, bool vec, const CUtensorMap* map, const float* v,
                                      int64_t row0, int64_t col0) {
    if (vec) return emit<T>(map, v, row0, col0, 0);
    const int c = lane & 15;
    const int rows = int(p.m - row0 < 32 ? p.m - row0 : 32);
#pragma unroll
    for (int h = 0; h < 32; h += 16) {
      stage<float>(v + h);
      __syncwarp();
      if (col0 + h + c < p.n) {
        T* o = out + row0 * stride + col0 + h + c;
#pragma unroll 8
        for (int r = lane >> 4; r < rows; r += 2)
          o[r * stride] = from_f<T>(
              *reinterpret_cast<const float*>(buf + r * 64 + (((c >> 2) ^ ((r >> 1) & 3)) << 4) + (c & 3) * 4));
      }
      __syncwarp();
    }
  }
  __device__ __forceinline__ void finish(float* v, int split, int64_t row0, int64_t col0) {
    const DenseEpi& e = p.epi;
    if (row0 >= p.m || col0 >= p.n) return;
    if (e.part) return emit<float>(ty, v, row0, col0, split);
    if (e.pre) put(static_cast<T*>(e.pre), e.pre_stride, e.vec_pre, tpre, v, row0, col0);
    if (e.act == MX_ACT_GELU) {
#pragma unroll
      for (int i = 0; i < 32; i += 2) gelu_f2(v[i], v[i + 1]);
    } else if (e.act == MX_ACT_LRELU) {
#pragma unroll
      for (int i = 0; i < 32; ++i) v[i] = v[i] >= 0.0f ? v[i] : e.slope * v[i];
    } else if (e.act == MX_ACT_SIGMOID) {
#pragma unroll
      for (int i = 0; i < 32; ++i) v[i] = sigmoid_f(v[i]);
    }
    if (e.residual && row0 + lane < p.m) {
      float r[32];
      row32(static_cast<const T*>(e.residual) + (row0 + lane) * e.residual_stride, e.vec_residual, col0, r);
#pragma unroll
      for (int i = 0; i < 32; ++i) v[i] += r[i];
    }
    put(static_cast<T*>(e.y), e.y_stride, e.vec_y, ty, v, row0, col0);
  }
  // Before the block's shared memory goes: the stores have read it.
  __device__ __forceinline__ void done() const {
    if (lane == 0) sm100::bulk_wait_read<0>();
    __syncwarp();
  }
};

// CHUNKED: a split may take more than CHUNK k-blocks, so a tile's sums pass
// through registers (fp32 always, 16 bits past K = 4096. An instance of its own:
// with both epilogues in one kernel the short products lose 1 to 7%, 71680 x 128
// -> 256 bf16 with GELU and pre 23.9 to 25.5 us).
template <class T, bool A_MN, bool B_MN, int BN, int G, bool CHUNKED>
__global__ void __launch_bounds__(DenseCfg<T, BN, G>::THREADS, 1)
    dense_mm_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                    const __grid_constant__ CUtensorMap tmY, const __grid_constant__ CUtensorMap tmPre, DenseMm p) {
  using C = DenseCfg<T, BN, G>;
  static_assert(CHUNKED || !C::F32, "fp32 sums always pass through registers");
  using namespace sm100;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* lo_base = base + C::STAGES * C::STAGE_BYTES;
  uint8_t* staging = lo_base + C::LO_STAGES * C::STAGE_BYTES;
  uint64_t* full = reinterpret_cast<uint64_t*>(lo_base + C::LO_STAGES * C::STAGE_BYTES + C::STAGING_BYTES);
  uint64_t* empty = full + C::STAGES;
  uint64_t* lo_ready = empty + C::STAGES;
  uint64_t* lo_empty = lo_ready + C::LO_STAGES;
  uint64_t* acc_full = lo_empty + C::LO_STAGES;
  uint64_t* acc_empty = acc_full + 2;
  uint64_t* peer_lo_ready = acc_empty + 2;  // in a pair's leader: the peer's lo_ready, passed on
  uint64_t* drained = peer_lo_ready + C::LO_STAGES;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drained + 1);
  __shared__ int abort_flag;
  __shared__ uint32_t issued;  // stages that this CTA's producer has loaded
  const volatile int* vabort = &abort_flag;
  // 16-bit pair: both CTAs' bytes count on the leader's barrier, which the MMA
  // issuer waits on. In fp32 each CTA's split warps wait on their own.
  constexpr bool SHARED = G == 2 && !C::F32;
  const int warp = __shfl_sync(0xFFFFFFFFu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int tiles = p.tiles_m * p.tiles_n;
  const int items = tiles * p.splits;
  const uint32_t rank = G == 2 ? cluster_rank() : 0;
  const int first = blockIdx.x / G, step = gridDim.x / G;

  if (threadIdx.x == 0) {
    abort_flag = 0;
    for (int s = 0; s < C::STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int s = 0; s < C::LO_STAGES; ++s) {
      mbar_init(&lo_ready[s], C::SPLIT_WARPS);
      mbar_init(&peer_lo_ready[s], 1);
      mbar_init(&lo_empty[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&acc_full[a], 1);
      mbar_init(&acc_empty[a], G * C::EPI_WARPS);
    }
    mbar_init(drained, 1);
    fence_mbar_init();
    tma_prefetch(&tmA);
    tma_prefetch(&tmB);
  }
  if (warp == 2) {
    if constexpr (G == 2) {
      tmem_alloc_pair(tmem_slot, C::TMEM_COLS);
    } else {
      tmem_alloc(tmem_slot, C::TMEM_COLS);
      tmem_relinquish();
    }
  }
  tc_fence_before();
  __syncthreads();
  if constexpr (G == 2) cluster_sync_all();  // the barriers of both exist
  tc_fence_after();
  pdl_wait();
  const uint32_t tmem = *tmem_slot;
  auto fail = [&](int code) {
    *static_cast<volatile int*>(p.status) = code;  // host memory: a plain store
    *const_cast<volatile int*>(vabort) = 1;
    if constexpr (G == 2) cluster_st_flag(map_rank(&abort_flag, rank ^ 1), 1);
  };
  auto kb_range = [&](int split, int& k0, int& k1) {
    k0 = split * p.kb_split;
    k1 = min(p.kb, k0 + p.kb_split);
  };
  // For what this CTA's threads and copies have written; for what the pair's have
  // written or read; for accumulators, whose order tcgen05's fences keep.
  auto wait = [&](uint64_t* bar, uint32_t parity) { return mbar_wait(bar, parity, vabort); };
  auto wait_pair = [&](uint64_t* bar, uint32_t parity) {
    return mbar_wait<G == 2 ? See::PAIR : See::CTA>(bar, parity, vabort);
  };
  auto wait_order = [&](uint64_t* bar, uint32_t parity) {
    return mbar_wait<G == 2 ? See::ORDER : See::CTA>(bar, parity, vabort);
  };
  auto commit = [&](uint64_t* bar) {
    if constexpr (G == 2)
      mma_commit_pair(bar);
    else
      mma_commit(bar);
  };

  if (warp < C::EPI_WARP0) {
    if constexpr (C::SPLIT_REGS) regs_dec<C::REGS_CONTROL>();
    if (warp == 0) {
      if (lane == 0) {
        uint32_t it = 0;
        for (int w = first; w < items && !*vabort; w += step) {
          int tm, tn, k0, k1;
          dense_tile(p, w % tiles, tm, tn);
          kb_range(w / tiles, k0, k1);
          const int row = (tm * G + rank) * 128, col = tn * BN + rank * C::BROWS;
          for (int kb = k0; kb < k1; ++kb, ++it) {
            const int s = it % C::STAGES;
            if (!wait_pair(&empty[s], ((it / C::STAGES) & 1) ^ 1)) {
              fail(kDenseErrProducer);
              break;
            }
            uint8_t* a = base + s * C::STAGE_BYTES;
            uint8_t* b = a + C::A_BYTES;
            if (!SHARED || rank == 0) mbar_arrive_expect_tx(&full[s], (SHARED ? 2 : 1) * (C::A_BYTES + C::B_BYTES));
            const uint32_t leader_full = SHARED ? map_rank(&full[s], 0) : 0;
            auto load = [&](uint8_t* dst, const CUtensorMap* map, int c0, int c1) {
              if constexpr (SHARED)
                tma_load_2d_pair(dst, map, leader_full, c0, c1);
              else
                tma_load_2d(dst, map, &full[s], c0, c1);
            };
            // K-major: one box of the tile's rows x 128 bytes of K. MN-major: a box
            // of BK rows of K x 128 bytes of M (N) for each 128 bytes of it.
            if (A_MN) {
#pragma unroll
              for (int c = 0; c < 128 / C::BK; ++c) load(a + c * C::BK * 128, &tmA, row + c * C::BK, kb * C::BK);
            } else {
              load(a, &tmA, kb * C::BK, row);
            }
            if (B_MN) {
#pragma unroll
              for (int c = 0; c < C::BROWS / C::BK; ++c) load(b + c * C::BK * 128, &tmB, col + c * C::BK, kb * C::BK);
            } else {
              load(b, &tmB, kb * C::BK, col);
            }
          }
        }
        issued = it;
      }
    } else if (warp == 1) {
      // The whole warp runs the loop, so that what the MMAs take is the same in
      // all lanes and stays in uniform registers; one lane issues.
      if (rank == 0) {
        constexpr uint32_t idesc =
            C::F32 ? idesc_tf32(128 * G, BN, A_MN, B_MN)
                   : idesc_f16(128 * G, BN, A_MN, B_MN, std::is_same<T, __nv_bfloat16>::value ? 1 : 0);
        // Steps of one MMA along K, in the descriptors' 16-byte units: 32 bytes
        // of a K-major row, or 16 (8 in fp32) 128-byte rows of an MN-major tile.
        constexpr uint32_t step_a = A_MN ? (C::F32 ? 64u : 128u) : 2u;
        constexpr uint32_t step_b = B_MN ? (C::F32 ? 64u : 128u) : 2u;
        auto desc = [](uint32_t addr, bool mn) {
          if (!mn) return desc_kmajor_sw128(addr);
          return C::F32 ? desc_mnmajor_sw128_32b(addr, C::BK * 128) : desc_mnmajor_sw128(addr, C::BK * 128);
        };
        auto mma = [](uint32_t d, uint64_t da, uint64_t db, uint32_t more) {
          if constexpr (C::F32) {
            if constexpr (G == 2)
              mma_tf32_pair(d, da, db, idesc, more);
            else
              mma_tf32(d, da, db, idesc, more);
          } else {
            if constexpr (G == 2)
              mma_f16_pair(d, da, db, idesc, more);
            else
              mma_f16(d, da, db, idesc, more);
          }
        };
        constexpr uint32_t CROSS = C::REGIONS == 2 ? BN : 0;  // the cross terms' columns
        const uint32_t base_u = smem_u32(base), lo_u = smem_u32(lo_base);
        uint32_t s = 0, ph = 0, l = 0, lph = 0, tc = 0;
        bool ok = true;
        for (int w = first; w < items && ok; w += step) {
          int k0, k1;
          kb_range(w / tiles, k0, k1);
          uint32_t d = 0;
          int left = 0;  // k-blocks the accumulator set still takes
          for (int kb = k0; kb < k1; ++kb) {
            const bool fresh = left == 0;
            if (fresh) {
              const uint32_t acc = tc & 1;
              ok = __all_sync(0xFFFFFFFFu, wait_order(&acc_empty[acc], ((tc >> 1) & 1) ^ 1));
              if (!ok) {
                if (lane == 0) fail(kDenseErrMmaAcc);
                break;
              }
              d = tmem + acc * C::SET_COLS;
              left = min(C::CHUNK, k1 - kb);
            }
            if constexpr (C::F32)
              ok = wait(&lo_ready[l], lph) && (G == 1 || wait_order(&peer_lo_ready[l], lph));
            else
              ok = wait_pair(&full[s], ph);
            ok = __all_sync(0xFFFFFFFFu, ok);
            if (!ok) {
              if (lane == 0) fail(kDenseErrMmaStage);
              break;
            }
            if constexpr (C::F32 && G == 2) fence_async_acquire_cluster();
            tc_fence_after();
            const uint32_t a = base_u + s * C::STAGE_BYTES, b = a + C::A_BYTES;
            const uint64_t da = desc(a, A_MN), db = desc(b, B_MN);
            --left;
            if (elect_one()) {
              if constexpr (C::F32) {
                const uint32_t alo = lo_u + l * C::STAGE_BYTES, blo = alo + C::A_BYTES;
                const uint64_t dal = desc(alo, A_MN), dbl = desc(blo, B_MN);
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                  const uint32_t more = !fresh || k > 0;
                  mma(d, da + step_a * k, db + step_b * k, more);
                  mma(d + CROSS, da + step_a * k, dbl + step_b * k, C::REGIONS == 2 ? more : 1u);
                  mma(d + CROSS, dal + step_a * k, db + step_b * k, 1u);
                }
              } else {
#pragma unroll
                for (int k = 0; k < 4; ++k) mma(d, da + step_a * k, db + step_b * k, !fresh || k > 0);
              }
              commit(&empty[s]);
              if constexpr (C::F32) commit(&lo_empty[l]);
              if (left == 0) commit(&acc_full[tc & 1]);
            }
            __syncwarp();
            if (left == 0) ++tc;
            if (++s == C::STAGES) s = 0, ph ^= 1;
            if (C::F32 && ++l == C::LO_STAGES) l = 0, lph ^= 1;
          }
        }
        // No MMA is in flight past here, whether or not an epilogue still waits for it.
        if (elect_one()) commit(drained);
        __syncwarp();
        if (!__all_sync(0xFFFFFFFFu, mbar_wait(drained, 0, nullptr)) && lane == 0) fail(kDenseErrDrain);
      } else if (C::F32 && lane == 0) {
        // The peer's lo tiles, as its split warps write them, for the leader's MMAs.
        // Here, so that the fence does not hold those warps up.
        uint32_t l = 0, lph = 0;
        bool ok = true;
        for (int w = first; w < items && ok; w += step) {
          int k0, k1;
          kb_range(w / tiles, k0, k1);
          for (int kb = k0; kb < k1; ++kb) {
            ok = wait(&lo_ready[l], lph);
            if (!ok) {
              fail(kDenseErrMmaStage);
              break;
            }
            fence_async_release_cluster();
            mbar_arrive_cluster(map_rank(&peer_lo_ready[l], 0));
            if (++l == C::LO_STAGES) l = 0, lph ^= 1;
          }
        }
      }
    }
  } else if (warp < C::SPLIT_WARP0) {
    if constexpr (C::SPLIT_REGS) regs_inc<C::REGS_EPI>();
    const int ew = warp - C::EPI_WARP0, q = warp & 3, part = ew >> 2;
    DenseOut<T> out{p, &tmY, &tmPre, staging + ew * 2048, lane};
    uint32_t tc = 0;
    bool ok = true;
    for (int w = first; w < items && ok; w += step) {
      int tm, tn, k0, k1;
      dense_tile(p, w % tiles, tm, tn);
      const int split = w / tiles;
      kb_range(split, k0, k1);
      const int64_t row0 = (int64_t(tm) * G + rank) * 128 + q * 32;
      const int64_t col0 = int64_t(tn) * BN + part * C::EPI_COLS;
      // The warp decides as one: the TMEM loads below need all its lanes.
      auto take = [&] {
        const bool got = __all_sync(0xFFFFFFFFu, wait_order(&acc_full[tc & 1], (tc >> 1) & 1));
        if (!got && lane == 0) fail(kDenseErrEpilogue);
        tc_fence_after();
        return got;
      };
      auto give = [&] {  // the set is read: the next products may have it
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          if constexpr (G == 2)
            mbar_arrive_cluster(map_rank(&acc_empty[tc & 1], 0));
          else
            mbar_arrive(&acc_empty[tc & 1]);
        }
        ++tc;
      };
      if constexpr (CHUNKED) {
        constexpr int COLS = C::EPI_COLS;
        float sum[COLS];
#pragma unroll
        for (int c = 0; c < COLS; c += 32) out.bias(col0 + c, sum + c);
        for (int kb = k0; kb < k1 && ok; kb += C::CHUNK) {
          ok = take();
          if (!ok) break;
          const uint32_t d = tmem + (uint32_t(q * 32) << 16) + (tc & 1) * C::SET_COLS + part * COLS;
#pragma unroll
          for (int c = 0; c < COLS; c += 16) {
            float hh[16], cross[16];
            if constexpr (C::REGIONS == 2) {
              tmem_ld16x2(d + c, d + BN + c, hh, cross);
#pragma unroll
              for (int i = 0; i < 16; ++i) sum[c + i] += hh[i] + cross[i];
            } else {
              tmem_ld16(d + c, hh);
#pragma unroll
              for (int i = 0; i < 16; ++i) sum[c + i] += hh[i];
            }
          }
          give();
        }
        if (!ok) break;
#pragma unroll
        for (int c = 0; c < COLS; c += 32) out.finish(sum + c, split, row0, col0 + c);
      } else {
        // One set: 32 columns at a time.
        ok = take();
        if (!ok) break;
        const uint32_t d = tmem + (uint32_t(q * 32) << 16) + (tc & 1) * C::SET_COLS + part * C::EPI_COLS;
#pragma unroll 1
        for (int c = 0; c < C::EPI_COLS; c += 32) {
          float v[32], b[32];
          out.bias(col0 + c, b);
          tmem_ld32(d + c, v);
          if (c + 32 == C::EPI_COLS) give();
#pragma unroll
          for (int i = 0; i < 32; ++i) v[i] += b[i];
          out.finish(v, split, row0, col0 + c);
        }
      }
    }
    out.done();
  } else if constexpr (C::F32) {
    if constexpr (C::SPLIT_REGS) regs_dec<C::REGS_SPLIT>();
    const int tid = threadIdx.x - 32 * C::SPLIT_WARP0;
    uint32_t s = 0, ph = 0, l = 0, lph = 0;
    bool ok = true;
    for (int w = first; w < items && ok; w += step) {
      int k0, k1;
      kb_range(w / tiles, k0, k1);
      for (int kb = k0; kb < k1; ++kb) {
        ok = __all_sync(0xFFFFFFFFu, wait(&full[s], ph) && wait_pair(&lo_empty[l], lph ^ 1));
        if (!ok) {
          if (lane == 0) fail(kDenseErrSplit);
          break;
        }
        // Elementwise, so the swizzled layouts do not matter.
        const float4* src = reinterpret_cast<const float4*>(base + s * C::STAGE_BYTES) + tid;
        float4* dst = reinterpret_cast<float4*>(lo_base + l * C::STAGE_BYTES) + tid;
        constexpr int STEP = 32 * C::SPLIT_WARPS, PER = C::STAGE_BYTES / 16 / STEP;
        constexpr int BATCH = C::SPLIT_REGS ? 4 : PER;  // loads ahead of their use
        static_assert(PER % BATCH == 0, "whole batches");
#pragma unroll
        for (int j = 0; j < PER; j += BATCH) {
          float4 v[BATCH];
#pragma unroll
          for (int i = 0; i < BATCH; ++i) v[i] = src[(j + i) * STEP];
#pragma unroll
          for (int i = 0; i < BATCH; ++i)
            dst[(j + i) * STEP] = make_float4(dense_residual(v[i].x), dense_residual(v[i].y), dense_residual(v[i].z),
                                              dense_residual(v[i].w));
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&lo_ready[l]);
        if (++s == C::STAGES) s = 0, ph ^= 1;
        if (++l == C::LO_STAGES) l = 0, lph ^= 1;
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if constexpr (G == 2) cluster_sync_all();  // neither leaves while the other's MMAs, copies or arrivals need it
  tc_fence_after();
  if (*vabort) {  // the same in both CTAs: whoever raised it did so before the barrier
    if (threadIdx.x == 0 && !(SHARED && rank != 0)) {
      uint32_t peers = issued;
      if constexpr (SHARED) peers = cluster_ld_u32(map_rank(&issued, 1));
      land_copies(
          issued, peers, C::STAGES,
          [&](uint32_t s) { mbar_arrive_expect_tx(&full[s], C::A_BYTES + C::B_BYTES); },
          [&](uint32_t s) { mbar_complete_tx(&full[s], C::A_BYTES + C::B_BYTES); },
          [&](uint32_t s, uint32_t parity) {
            return mbar_wait<SHARED ? See::PAIR : See::CTA>(&full[s], parity, nullptr);
          });
    }
    __syncthreads();
    if constexpr (G == 2) cluster_sync_all();
  }
  if (warp == 2) {
    if constexpr (G == 2)
      tmem_dealloc_pair(tmem, C::TMEM_COLS);
    else
      tmem_dealloc(tmem, C::TMEM_COLS);
  }
}

}  // namespace mx
