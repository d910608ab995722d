// Launches of the operators on a caller's device tensors, for one element type.
#pragma once

#include <algorithm>
#include <mutex>
#include <string>

#include "common.h"
#include "gpu_common.cuh"
#include "kernels_dense.cuh"
#include "kernels_norm.cuh"
#include "ops.h"

namespace mx {
namespace {

inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
inline int64_t round_up(int64_t a, int64_t b) { return ceil_div(a, b) * b; }

// Whether every row of a matrix starts on a 16-byte boundary.
template <class T>
bool aligned(const void* p, int64_t stride) {
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && stride % kVec<T> == 0;
}

// A launch in clusters of the given shape (1 x 1 x 1: a plain one). The blocks
// may be set up while the kernel before them in the stream ends (programmatic
// stream serialization): every kernel here waits for it, in pdl_wait, before
// it touches memory.
template <class... P, class... A>
void launch_clusters(void (*kernel)(P...), dim3 grid, dim3 block, int smem, dim3 cluster, cudaStream_t s, A&&... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid, cfg.blockDim = block;
  cfg.dynamicSmemBytes = size_t(smem);
  cfg.stream = s;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = cluster.x, at[1].val.clusterDim.y = cluster.y, at[1].val.clusterDim.z = cluster.z;
  cfg.attrs = at;
  cfg.numAttrs = cluster.x * cluster.y * cluster.z > 1 ? 2 : 1;
  MX_CUDA(cudaLaunchKernelEx(&cfg, kernel, std::forward<A>(args)...));
}
template <class... P, class... A>
void launch(void (*kernel)(P...), dim3 grid, unsigned threads, int smem, cudaStream_t s, A&&... args) {
  launch_clusters(kernel, grid, dim3(threads), smem, dim3(1), s, std::forward<A>(args)...);
}

// ------------------------------------------------------------- layer norm
// The lanes a row is spread over (L) and the vectors a lane holds (NV): the
// fewest lanes that hold the row in 8 values each, up to a warp (fewer lanes
// mean fewer shuffles a row: 448 x 640 rows of 64 fp32 took 32 us with 4 values
// a lane); past that a warp or a block with 16 values a thread, then 32.
// (Twice the lanes with 8 values each measured slower: 16411 x 4096 bf16
// backward 100 us against 77, the reductions cost a warp the same.)
// Two warps a row pay forward only (65536 x 1024 bf16: forward 55 to 48 us, backward
// 82 to 92).
// f(L, NV) is called with the choice as integral constants; returns false for
// rows too long.
template <int V, bool BACKWARD, class F>
bool with_norm_shape(int c, F&& f) {
  constexpr int N8 = V < 8 ? 8 / V : 1, N16 = 16 / V;
  const int64_t vecs = ceil_div(c, V);
#define MX_SHAPE(L, NV)                                                               \
  if (vecs <= int64_t(L) * (NV)) {                                                    \
    f(std::integral_constant<int, L>(), std::integral_constant<int, (NV)>());         \
    return true;                                                                      \
  }
  MX_SHAPE(1, N8)
  MX_SHAPE(2, N8)
  MX_SHAPE(4, N8)
  MX_SHAPE(8, N8)
  MX_SHAPE(16, N8)
  MX_SHAPE(32, N8)
  MX_SHAPE(32, N16)
  if constexpr (!BACKWARD && V > 1) {
    MX_SHAPE(64, N16)  // as many vectors as the next
  } else {
    MX_SHAPE(128, N8)
  }
  MX_SHAPE(128, N16)
  MX_SHAPE(256, N16)
  MX_SHAPE(512, N16)
  if constexpr (V > 1) MX_SHAPE(512, 2 * N16)
#undef MX_SHAPE
  return false;
}

// Blocks of a kernel that one SM holds at once, asked once per kernel and
// device, with the opt-in for its shared memory (`smem`, and `extra` where a launch takes more).
template <class K>
int resident_blocks(K* kernel, int threads, int smem, int extra, std::mutex& mu, int (&known)[64]) {
  int dev = 0;
  MX_CUDA(cudaGetDevice(&dev));
  std::lock_guard<std::mutex> lock(mu);
  if (!known[dev]) {
    MX_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem + extra));
    MX_CUDA(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&known[dev], kernel, threads, smem));
  }
  return std::max(1, known[dev]);
}
// A few rows' parameter gradients are summed by one cluster: up to kClusterRows
// rows for each group of lanes of each of its (at most 8) blocks, rows of up to
// kClusterCols.
constexpr int64_t kClusterRows = 10, kClusterCols = 4096;
constexpr int kClusterSmem = int(2 * kClusterCols * 4);

template <class T, int V, int L, int NV, bool BACKWARD>
int norm_resident() {
  static std::mutex mu;
  static int known[64] = {};
  if constexpr (BACKWARD)
    return resident_blocks(layer_norm_backward_kernel<T, V, L, NV>, kNormThreads<L>, kNormSmem<V, L, NV, 2>,
                           kClusterSmem, mu, known);
  else
    return resident_blocks(layer_norm_kernel<T, V, L, NV>, kNormThreads<L>, kNormSmem<V, L, NV, 1>, 0, mu, known);
}

template <class T, int V>
void norm_forward_v(const mx_layer_norm_args& a, const OpsDevice& d, cudaStream_t s) {
  NormFwd p{a.x, a.scale, a.bias, a.y, a.mean, a.rstd, a.rows, a.x_stride, a.y_stride,
            int(a.c), a.param_dtype == MX_DT_F32, a.eps};
  const bool done = with_norm_shape<V, false>(int(a.c), [&](auto l, auto nv) {
    constexpr int L = decltype(l)::value, NV = decltype(nv)::value;
    constexpr int THREADS = kNormThreads<L>, GROUPS = THREADS / L;
    const int64_t resident = norm_resident<T, V, L, NV, false>();
    const int64_t blocks = std::min<int64_t>(ceil_div(a.rows, GROUPS), d.sms * resident);
    launch(layer_norm_kernel<T, V, L, NV>, dim3(unsigned(blocks)), THREADS, kNormSmem<V, L, NV, 1>, s, p);
  });
  if (!done)
    launch(layer_norm_long_kernel<T, V>, dim3(unsigned(std::min<int64_t>(a.rows, int64_t(d.sms) * 4))), 512, 0, s, p);
}

template <class T>
void layer_norm(const mx_layer_norm_args& a, const OpsDevice& d, cudaStream_t s) {
  if (aligned<T>(a.x, a.x_stride) && aligned<T>(a.y, a.y_stride) && a.c % kVec<T> == 0)
    norm_forward_v<T, kVec<T>>(a, d, s);
  else
    norm_forward_v<T, 1>(a, d, s);
}

template <class T>
bool norm_backward_vec(const mx_layer_norm_backward_args& a) {
  return aligned<T>(a.x, a.x_stride) && aligned<T>(a.dy, a.dy_stride) && (!a.dx || aligned<T>(a.dx, a.dx_stride)) &&
         a.c % kVec<T> == 0;
}
// Blocks of the backward kernel, which is also how many partial rows of the
// parameter gradients it leaves; or those of one cluster, which leaves none.
struct NormBlocks {
  int64_t blocks;
  bool cluster;
};
template <class T, int V>
NormBlocks norm_backward_blocks(const mx_layer_norm_backward_args& a, const OpsDevice& d) {
  NormBlocks n{0, false};
  const bool done = with_norm_shape<V, true>(int(a.c), [&](auto l, auto nv) {
    constexpr int L = decltype(l)::value, NV = decltype(nv)::value, GROUPS = kNormThreads<L> / L;
    const int resident = norm_resident<T, V, L, NV, true>();
    const int64_t want = ceil_div(a.rows, GROUPS);
    n.cluster = (a.dscale || a.dbias) && want <= 8 * kClusterRows && a.c <= kClusterCols;
    n.blocks = n.cluster ? std::min<int64_t>(want, 8) : std::min<int64_t>(want, int64_t(d.sms) * resident);
  });
  if (!done) n.blocks = std::min<int64_t>(ceil_div(a.rows, 8), std::max<int64_t>(1, d.sms * 4 / ceil_div(a.c, 32 * V)));
  return n;
}

template <class T, int V>
void norm_backward_v(const mx_layer_norm_backward_args& a, const OpsDevice& d, cudaStream_t s) {
  const NormBlocks n = norm_backward_blocks<T, V>(a, d);
  float* part = (a.dscale || a.dbias) && !n.cluster ? static_cast<float*>(a.workspace) : nullptr;
  NormBwd p{a.dy, a.x, a.scale, a.mean, a.rstd, a.dx, part, n.cluster ? int(n.blocks) : 0, a.dscale, a.dbias,
            a.rows, a.dy_stride, a.x_stride, a.dx_stride, int(a.c), a.param_dtype == MX_DT_F32};
  const bool done = with_norm_shape<V, true>(int(a.c), [&](auto l, auto nv) {
    constexpr int L = decltype(l)::value, NV = decltype(nv)::value;
    const int smem = kNormSmem<V, L, NV, 2> + (n.cluster ? int(2 * a.c * 4) : 0);
    launch_clusters(layer_norm_backward_kernel<T, V, L, NV>, dim3(unsigned(n.blocks)), dim3(kNormThreads<L>), smem,
                    n.cluster ? dim3(unsigned(n.blocks)) : dim3(1), s, p);
  });
  if (!done) {
    // The sums first: dx may overwrite dy.
    if (part)
      launch(layer_norm_param_long_kernel<T, V>, dim3(unsigned(ceil_div(a.c, 32 * V)), unsigned(n.blocks)), 256, 0, s,
             p);
    if (a.dx)
      launch(layer_norm_dx_long_kernel<T, V>, dim3(unsigned(std::min<int64_t>(a.rows, int64_t(d.sms) * 4))), 512, 0, s,
             p);
  }
}

// Partial rows to out0 (columns below `split`) and out1.
template <class T>
void join_columns(const float* part, int64_t nb, int64_t cols, int64_t split, void* out0, void* out1, bool out_f32,
                  cudaStream_t s) {
  const unsigned grid = unsigned(ceil_div(cols, 32));
  if (nb <= 32)
    launch(column_join_kernel<T, 8>, dim3(grid), 256, 0, s, part, int(nb), cols, split, out0, out1, out_f32);
  else
    launch(column_join_kernel<T, 32>, dim3(grid), 1024, 0, s, part, int(nb), cols, split, out0, out1, out_f32);
}

template <class T>
NormBlocks norm_backward_plan(const mx_layer_norm_backward_args& a, const OpsDevice& d) {
  return norm_backward_vec<T>(a) ? norm_backward_blocks<T, kVec<T>>(a, d) : norm_backward_blocks<T, 1>(a, d);
}

template <class T>
int64_t layer_norm_backward_workspace(const mx_layer_norm_backward_args& a, const OpsDevice& d) {
  if ((!a.dscale && !a.dbias) || a.rows == 0) return 0;
  const NormBlocks n = norm_backward_plan<T>(a, d);
  return n.cluster ? 0 : n.blocks * 2 * a.c * 4;
}

template <class T>
void layer_norm_backward(const mx_layer_norm_backward_args& a, const OpsDevice& d, cudaStream_t s) {
  const bool out_f32 = a.param_dtype == MX_DT_F32;
  if (a.rows == 0) {
    const size_t bytes = size_t(a.c) * (out_f32 ? 4 : sizeof(T));
    if (a.dscale) MX_CUDA(cudaMemsetAsync(a.dscale, 0, bytes, s));
    if (a.dbias) MX_CUDA(cudaMemsetAsync(a.dbias, 0, bytes, s));
    return;
  }
  if (norm_backward_vec<T>(a))
    norm_backward_v<T, kVec<T>>(a, d, s);
  else
    norm_backward_v<T, 1>(a, d, s);
  const NormBlocks n = norm_backward_plan<T>(a, d);
  if ((a.dscale || a.dbias) && !n.cluster)
    join_columns<T>(static_cast<const float*>(a.workspace), n.blocks, 2 * a.c, a.c, a.dscale, a.dbias, out_f32, s);
}

// ------------------------------------------------------------------ dense
// An operand of the tensor-core product: a row-major matrix whose contiguous
// axis is the contracted one (K-major) or the other (MN-major).
struct Operand {
  const void* p;
  int64_t stride;  // elements between rows
  bool mn_major;
};

struct MmPlan {
  int bn, g;
  int splits, kb, kb_split;
  int64_t part_bytes;
};

// Tile and number of splits of K: the cheapest by a model of the kernel's
// time, in one SM's cycles, its constants fitted to sweeps of all tiles and
// splits over sizes from 64 x 512 x 512 to 20000 x 344 x 704 (the choice is within a few
// percent of the best of each). A k-block (128 bytes of K) of a tile costs
// `step` cycles, mostly its operands' way from the L2; a launch, its first
// loads and last epilogue cost 7000 (8700 for pairs); the CTAs of the slowest SM
// are what counts. Split sums cost their write and reading back (3000 bytes a
// cycle for the whole GPU) and another launch (3500).
template <class T>
MmPlan plan_mm(int64_t m, int64_t n, int64_t k, int sms) {
  constexpr bool F32 = sizeof(T) == 4;
  constexpr int BK = 128 / int(sizeof(T));
  struct Tile {
    int bn, g;
    double step;
  };
  constexpr Tile kF32[] = {{64, 1, 1050}, {128, 1, 1570}, {128, 2, 1200}, {256, 2, 1900}};
  constexpr Tile k16[] = {{64, 1, 470}, {128, 1, 540}, {256, 1, 740}, {256, 2, 640}};
  MmPlan best{};
  double best_cost = 0;
  const int kb = int(ceil_div(k, BK));
  for (int i = 0; i < 4; ++i) {
    const Tile& t = F32 ? kF32[i] : k16[i];
    // The widest fp32 tile's epilogue (64 sums a lane) pays from K = 512 on: with
    // GELU and pre, 100000 x 256 -> 512 172 us against 162, 8192 x 1024 -> 4096 291 against 372.
    if (F32 && t.bn == 256 && k < 512) continue;
    const int64_t tiles = ceil_div(m, 128 * t.g) * ceil_div(n, t.bn);
    const int workers = sms / t.g;
    auto consider = [&](int64_t want) {
      if (want < 1 || want > kb || (want > 1 && tiles * want > int64_t(workers) * 2)) return;
      const int per = int(ceil_div(kb, want)), splits = int(ceil_div(kb, per));
      const int64_t waves = ceil_div(tiles * splits, workers);
      double cost = double(waves) * (per * t.step + 1000) + (t.g == 2 ? 8700 : 7000);
      if (splits > 1) cost += 3500 + double(splits) * double(m) * double(n) * 8 / 3000;
      if (best.bn == 0 || cost < best_cost) {
        best_cost = cost;
        best = {t.bn, t.g, splits, kb, per, splits > 1 ? int64_t(splits) * m * round_up(n, 8) * 4 : 0};
      }
    };
    for (int want = 1; want <= 8; ++want) consider(want);
    for (int want = 10; want < workers; want = want * 5 / 4) consider(want);
    consider(workers / tiles);  // one full wave, or two
    consider(2 * workers / tiles);
  }
  return best;
}

template <class T>
constexpr CUtensorMapDataType map_type() {
  return sizeof(T) == 4 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                        : (std::is_same<T, __half>::value ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                          : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16);
}

template <class T>
CUtensorMap operand_map(const Operand& o, int64_t rows, int64_t cols, int box_rows) {
  constexpr int BK = 128 / int(sizeof(T));
  const cuuint64_t dims[2] = {cuuint64_t(cols), cuuint64_t(rows)};
  const cuuint64_t strides[1] = {cuuint64_t(o.stride) * sizeof(T)};
  const cuuint32_t box[2] = {cuuint32_t(BK), cuuint32_t(box_rows)};
  const cuuint32_t es[2] = {1, 1};
  // The swizzle the tensor core expects of the tile: 32-bit MN-major operands
  // have a form of their own.
  const CUtensorMapSwizzle sw =
      o.mn_major && sizeof(T) == 4 ? CU_TENSOR_MAP_SWIZZLE_128B_ATOM_32B : CU_TENSOR_MAP_SWIZZLE_128B;
  CUtensorMap m;
  CUresult r = tensor_map_encoder()(&m, map_type<T>(), 2, const_cast<void*>(o.p), dims, strides, box, es,
                                    CU_TENSOR_MAP_INTERLEAVE_NONE, sw, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                                    CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) throw Error(fmt("cuTensorMapEncodeTiled failed (%d)", int(r)), MX_E_CUDA);
  return m;
}

// A result's map: blocks of 32 rows x 64 bytes, in the swizzle the epilogue stages them in.
template <class U>
CUtensorMap result_map(void* p, int64_t stride, int64_t rows, int64_t cols, int64_t layers) {
  const cuuint64_t dims[3] = {cuuint64_t(cols), cuuint64_t(rows), cuuint64_t(layers)};
  const cuuint64_t strides[2] = {cuuint64_t(stride) * sizeof(U), cuuint64_t(stride) * sizeof(U) * cuuint64_t(rows)};
  const cuuint32_t box[3] = {64 / sizeof(U), 32, 1}, es[3] = {1, 1, 1};
  CUtensorMap m;
  CUresult r = tensor_map_encoder()(&m, map_type<U>(), 3, p, dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
                                    CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_NONE,
                                    CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) throw Error(fmt("cuTensorMapEncodeTiled failed (%d)", int(r)), MX_E_CUDA);
  return m;
}

template <class T, bool A_MN, bool B_MN, int BN, int G, bool CHUNKED = true>
void launch_mm(const Operand& a, const Operand& b, const DenseMm& p, int64_t k, const OpsDevice& d, cudaStream_t s) {
  using C = DenseCfg<T, BN, G>;
  if constexpr (sizeof(T) == 2 && CHUNKED)
    if (p.kb_split <= C::CHUNK) return launch_mm<T, A_MN, B_MN, BN, G, false>(a, b, p, k, d, s);
  constexpr int kMaxDevices = 64;
  static std::mutex mu;
  static bool opted[kMaxDevices] = {};
  auto* kernel = dense_mm_kernel<T, A_MN, B_MN, BN, G, CHUNKED>;
  {
    int dev = 0;
    MX_CUDA(cudaGetDevice(&dev));
    std::lock_guard<std::mutex> lock(mu);
    if (!opted[dev]) {
      MX_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM_BYTES));
      opted[dev] = true;
    }
  }
  const CUtensorMap ta = A_MN ? operand_map<T>(a, k, p.m, C::BK) : operand_map<T>(a, p.m, k, 128);
  const CUtensorMap tb = B_MN ? operand_map<T>(b, k, p.n, C::BK) : operand_map<T>(b, p.n, k, C::BROWS);
  // Results that no map can take have none (the kernel does not touch theirs).
  const CUtensorMap ty = p.epi.part ? result_map<float>(p.epi.part, p.epi.ldp, p.m, p.n, p.splits)
                         : p.epi.vec_y ? result_map<T>(p.epi.y, p.epi.y_stride, p.m, p.n, 1) : CUtensorMap{};
  const CUtensorMap tpre =
      !p.epi.part && p.epi.vec_pre ? result_map<T>(p.epi.pre, p.epi.pre_stride, p.m, p.n, 1) : CUtensorMap{};
  const int64_t items = int64_t(p.tiles_m) * p.tiles_n * p.splits;
  launch_clusters(kernel, dim3(unsigned(std::min<int64_t>(items, d.sms / G) * G)), dim3(C::THREADS), C::SMEM_BYTES,
                  dim3(G), s, ta, tb, ty, tpre, p);
}

// D = A B^T with the epilogue `epi`: the product, and the join of its splits.
template <class T>
void run_mm(const Operand& a, const Operand& b, int64_t m, int64_t n, int64_t k, DenseEpi epi, const MmPlan& plan,
            void* part, const OpsDevice& d, cudaStream_t s) {
  DenseMm p{};
  p.m = m, p.n = n;
  p.kb = plan.kb, p.kb_split = plan.kb_split, p.splits = plan.splits;
  p.tiles_m = int(ceil_div(m, 128 * plan.g)), p.tiles_n = int(ceil_div(n, plan.bn));
  p.epi = epi;
  p.status = d.status;
  if (plan.splits > 1) p.epi.part = static_cast<float*>(part), p.epi.ldp = round_up(n, 8);
  auto by_width = [&](auto amn, auto bmn) {
    constexpr bool A = decltype(amn)::value, B = decltype(bmn)::value;
    if constexpr (sizeof(T) == 4)
      if (plan.g == 2 && plan.bn == 128) return launch_mm<T, A, B, 128, 2>(a, b, p, k, d, s);
    if (plan.g == 2) return launch_mm<T, A, B, 256, 2>(a, b, p, k, d, s);
    if (plan.bn == 64) return launch_mm<T, A, B, 64, 1>(a, b, p, k, d, s);
    if constexpr (sizeof(T) == 2)
      if (plan.bn == 256) return launch_mm<T, A, B, 256, 1>(a, b, p, k, d, s);
    launch_mm<T, A, B, 128, 1>(a, b, p, k, d, s);
  };
  if (a.mn_major)
    by_width(std::true_type(), std::true_type());
  else if (b.mn_major)
    by_width(std::false_type(), std::true_type());
  else
    by_width(std::false_type(), std::false_type());
  if (plan.splits > 1) {
    const int64_t vecs = m * ceil_div(n, 8);
    // Eight threads an output where that still leaves the GPU short of threads.
    if (plan.splits >= 16 && vecs < int64_t(d.sms) * 512)
      launch(dense_join_kernel<T, 8>, dim3(unsigned(ceil_div(vecs, 32))), 256, 0, s, p.epi, plan.splits, m, n);
    else
      launch(dense_join_kernel<T, 1>, dim3(unsigned(std::min<int64_t>(ceil_div(vecs, 256), int64_t(d.sms) * 8))), 256,
             0, s, p.epi, plan.splits, m, n);
  }
}

// Carves the workspace into 256-byte aligned pieces; with a null base it only counts.
struct Carver {
  uint8_t* base;
  int64_t used = 0;
  void* take(int64_t bytes) {
    if (bytes == 0) return nullptr;
    void* p = base ? base + used : nullptr;
    used += round_up(bytes, 256);
    return p;
  }
};
// The workspace is 16-byte aligned only; the pieces' alignment is relative to it.

// A matrix the tensor maps can take: itself, or an aligned copy.
template <class T>
struct Staged {
  const void* src;
  int64_t src_stride, rows, cols;
  T* copy;
  int64_t stride;
  Staged(Carver& c, const void* p, int64_t st, int64_t r, int64_t n)
      : src(p), src_stride(st), rows(r), cols(n), copy(nullptr), stride(st) {
    if (!aligned<T>(p, st)) {
      stride = round_up(n, kVec<T>);
      copy = static_cast<T*>(c.take(rows * stride * int64_t(sizeof(T))));
    }
  }
  Operand operand(bool mn_major) const { return {copy ? copy : src, stride, mn_major}; }
  void add_to(DenseAlign& a, const OpsDevice& d) const {
    if (!copy) return;
    const int i = a.count++;
    a.src[i] = src, a.dst[i] = copy, a.src_stride[i] = src_stride, a.dst_stride[i] = stride;
    a.rows[i] = rows, a.cols[i] = cols;
    a.first[i + 1] =
        a.first[i] + unsigned(std::min<int64_t>(ceil_div(rows * stride / kVec<T>, 256), int64_t(d.sms) * 16));
  }
};
// The copies that staged matrices need, in one launch.
template <class T, class... S>
void align(const OpsDevice& d, cudaStream_t s, const S&... staged) {
  static_assert(sizeof...(S) <= DenseAlign::MAX, "matrices a launch copies");
  DenseAlign a{};
  (staged.add_to(a, d), ...);
  if (a.count == 0) return;
  launch(dense_align_kernel<T>, dim3(a.first[a.count]), 256, 0, s, a);
}

// Whether a product goes through the FMA kernel: one or two rows, up to four
// where the matrix of weights is small, up to eight where it is tiny. (bf16, m x k x
// n, FMA against tensor cores: 1 x 4096 x 16384 27 us against 32, 4 x 4096 x 16384 35
// against 32, 4 x 4096 x 4096 16.0 against 16.7, 4 x 8192 x 1024 10 against 14, 8 x
// 8192 x 1024 18 against 14; of GPU time alone, 8 x 1024 x 1024 4.5 against 7.6.)
inline bool few_rows(const mx_dense_args& a) {
  const int64_t weights = a.k * a.n;
  return a.m <= 2 || (a.m <= 4 && weights <= (int64_t(1) << 24)) || (a.m <= 8 && weights <= (int64_t(1) << 20));
}

template <class T>
int64_t dense_workspace(const mx_dense_args& a, const OpsDevice& d) {
  if (few_rows(a)) return 0;
  Carver c{nullptr};
  Staged<T> x(c, a.x, a.x_stride, a.m, a.k), w(c, a.w, a.w_stride, a.n, a.k);
  c.take(plan_mm<T>(a.m, a.n, a.k, d.sms).part_bytes);
  return c.used;
}

template <class T>
void dense_rows(const mx_dense_args& a, const DenseEpi& epi, const OpsDevice& d, cudaStream_t s) {
  const bool vec = aligned<T>(a.x, a.x_stride) && aligned<T>(a.w, a.w_stride) && a.k % kVec<T> == 0;
  // Four weight rows a warp where that still gives every SM a dozen warps,
  // else one; and then as many warps on one row as keep the SMs busy and
  // have a vector of K each.
  const int cpw = a.n >= int64_t(d.sms) * 48 ? 4 : 1;
  const int64_t vecs = ceil_div(a.k, (vec ? kVec<T> : 1) * 32);
  int ks = 1;
  while (ks < 8 && ks < vecs && ceil_div(a.n, cpw) * ks < int64_t(d.sms) * 16) ks *= 2;
  // Small blocks spread evenly: 16384 columns over 148 SMs are 3.46 blocks of
  // eight warps each, 6.92 of four.
  const int warps = std::max(4, ks);
  const unsigned grid = unsigned(ceil_div(ceil_div(a.n, cpw), warps / ks));
  auto go = [&](auto r, auto v, auto c) {
    launch(dense_rows_kernel<T, decltype(r)::value, decltype(v)::value, decltype(c)::value>, dim3(grid), warps * 32, 0,
           s, static_cast<const T*>(a.x), a.x_stride, static_cast<const T*>(a.w), a.w_stride, epi, int(a.m),
           int(a.n), int(a.k), ks);
  };
  auto by_cols = [&](auto r, auto v) {
    if (cpw == 4)
      go(r, v, std::integral_constant<int, 4>());
    else
      go(r, v, std::integral_constant<int, 1>());
  };
  auto by_vec = [&](auto r) {
    if (vec)
      by_cols(r, std::integral_constant<int, kVec<T>>());
    else
      by_cols(r, std::integral_constant<int, 1>());
  };
  if (a.m == 1)
    by_vec(std::integral_constant<int, 1>());
  else if (a.m == 2)
    by_vec(std::integral_constant<int, 2>());
  else if (a.m <= 4)
    by_vec(std::integral_constant<int, 4>());
  else
    by_vec(std::integral_constant<int, 8>());
}

template <class T>
void dense(const mx_dense_args& a, const OpsDevice& d, cudaStream_t s) {
  DenseEpi e{};
  e.bias = a.bias, e.residual = a.residual, e.y = a.y, e.pre = a.pre;
  e.residual_stride = a.residual_stride, e.y_stride = a.y_stride, e.pre_stride = a.pre_stride;
  e.act = a.act, e.slope = a.slope;
  e.vec_residual = a.residual && aligned<T>(a.residual, a.residual_stride);
  e.vec_y = aligned<T>(a.y, a.y_stride);
  e.vec_pre = a.pre && aligned<T>(a.pre, a.pre_stride);
  e.vec_bias = a.bias && aligned<T>(a.bias, 0);
  if (few_rows(a)) return dense_rows<T>(a, e, d, s);
  Carver c{static_cast<uint8_t*>(a.workspace)};
  Staged<T> x(c, a.x, a.x_stride, a.m, a.k), w(c, a.w, a.w_stride, a.n, a.k);
  const MmPlan plan = plan_mm<T>(a.m, a.n, a.k, d.sms);
  void* part = c.take(plan.part_bytes);
  align<T>(d, s, x, w);
  run_mm<T>(x.operand(false), w.operand(false), a.m, a.n, a.k, e, plan, part, d, s);
}

// The pieces of the backward pass and where they lie in the workspace.
template <class T>
struct DenseBackward {
  const bool act, products;
  bool vec;               // 16-byte accesses to dy, pre and d
  int lx_log2;            // the column sums' blocks: 1 << lx_log2 threads across,
  int64_t cols, chunks;   // cols x chunks of them,
  bool cluster;           // the chunks as one cluster
  T* d;                   // dy act'(pre), rounded to T
  int64_t d_stride;
  float* db_part;
  Staged<T> dy, x, w;
  MmPlan dx, dw;
  void* part;
  DenseBackward(Carver& c, const mx_dense_backward_args& a, const OpsDevice& dev)
      : act(a.act != MX_ACT_NONE), products(a.dx || a.dw), vec(false), lx_log2(5), cols(0), chunks(0), cluster(false),
        d(nullptr), d_stride(round_up(a.n, kVec<T>)), db_part(nullptr),
        // Without an activation d is dy itself.
        dy(c, act || !products ? nullptr : a.dy, act || !products ? 0 : a.dy_stride, a.m, a.n),
        x(c, a.dw ? a.x : nullptr, a.dw ? a.x_stride : 0, a.m, a.k),
        w(c, a.dx ? a.w : nullptr, a.dx ? a.w_stride : 0, a.n, a.k), dx{}, dw{}, part(nullptr) {
    vec = aligned<T>(a.dy, a.dy_stride) && (!act || aligned<T>(a.pre, a.pre_stride)) && a.n % kVec<T> == 0;
    if ((act && products) || a.db) {
      const int64_t vecs = ceil_div(a.n, vec ? kVec<T> : 1);
      while (lx_log2 > 0 && (int64_t(1) << (lx_log2 - 1)) >= vecs) --lx_log2;
      cols = ceil_div(vecs, int64_t(1) << lx_log2);
      // Up to 16 rows a thread in 8 blocks: one cluster joins the sums itself
      // (another launch would cost more).
      const int64_t subs = 256 >> lx_log2;
      cluster = a.db && a.m <= 8 * 16 * subs;
      chunks = cluster ? std::min<int64_t>(8, ceil_div(a.m, 2 * subs))
                       : std::min<int64_t>(ceil_div(a.m, 2 * subs), std::max<int64_t>(1, int64_t(dev.sms) * 6 / cols));
    }
    if (act && products) d = static_cast<T*>(c.take(a.m * d_stride * int64_t(sizeof(T))));
    if (a.db && !cluster) db_part = static_cast<float*>(c.take(chunks * a.n * 4));
    if (a.dx) dx = plan_mm<T>(a.m, a.k, a.n, dev.sms);
    if (a.dw) dw = plan_mm<T>(a.n, a.k, a.m, dev.sms);
    part = c.take(std::max(dx.part_bytes, dw.part_bytes));  // the products run one after the other
  }
};

template <class T>
int64_t dense_backward_workspace(const mx_dense_backward_args& a, const OpsDevice& dev) {
  if (a.m == 0) return 0;
  Carver c{nullptr};
  DenseBackward<T> b(c, a, dev);
  return c.used;
}

template <class T>
void dense_backward(const mx_dense_backward_args& a, const OpsDevice& dev, cudaStream_t s) {
  if (a.m == 0) {
    if (a.dw) MX_CUDA(cudaMemset2DAsync(a.dw, size_t(a.dw_stride) * sizeof(T), 0, size_t(a.k) * sizeof(T), a.n, s));
    if (a.db) MX_CUDA(cudaMemsetAsync(a.db, 0, size_t(a.n) * sizeof(T), s));
    return;
  }
  Carver c{static_cast<uint8_t*>(a.workspace)};
  DenseBackward<T> b(c, a, dev);
  if (b.chunks) {
    auto go = [&](auto v, auto store) {
      launch_clusters(dense_grad_kernel<T, decltype(v)::value, decltype(store)::value>,
                      dim3(unsigned(b.cols), unsigned(b.chunks)), dim3(256), 0,
                      b.cluster ? dim3(1, unsigned(b.chunks)) : dim3(1), s, static_cast<const T*>(a.dy), a.dy_stride,
                      static_cast<const T*>(a.pre), a.pre_stride, b.d, b.d_stride, b.db_part,
                      b.cluster ? static_cast<T*>(a.db) : nullptr, a.m, int(a.n), b.lx_log2, int(a.act), a.slope);
    };
    auto by_store = [&](auto v) {
      if (b.d)
        go(v, std::true_type());
      else
        go(v, std::false_type());
    };
    if (b.vec)
      by_store(std::integral_constant<int, kVec<T>>());
    else
      by_store(std::integral_constant<int, 1>());
    if (b.db_part) join_columns<T>(b.db_part, b.chunks, a.n, a.n, a.db, nullptr, false, s);
  }
  if (!b.products) return;
  align<T>(dev, s, b.dy, b.x, b.w);
  const Operand d = b.act ? Operand{b.d, b.d_stride, false} : b.dy.operand(false);
  DenseEpi e{};
  if (a.dx) {
    e.y = a.dx, e.y_stride = a.dx_stride, e.vec_y = aligned<T>(a.dx, a.dx_stride);
    run_mm<T>(d, b.w.operand(true), a.m, a.k, a.n, e, b.dx, b.part, dev, s);
  }
  if (a.dw) {
    e.y = a.dw, e.y_stride = a.dw_stride, e.vec_y = aligned<T>(a.dw, a.dw_stride);
    run_mm<T>({d.p, d.stride, true}, b.x.operand(true), a.n, a.k, a.m, e, b.dw, b.part, dev, s);
  }
}

template <class T>
constexpr OpsTable ops_table() {
  return {layer_norm<T>,      layer_norm_backward_workspace<T>, layer_norm_backward<T>, dense_workspace<T>, dense<T>,
          dense_backward_workspace<T>, dense_backward<T>};
}

}  // namespace
}  // namespace mx
