// SPDX-License-Identifier: Apache-2.0
// Gated feed-forward block for a few rows (single atoms, single tokens): y = (act(x Wg) * (x Wu)) Wd with up to 8 rows of x.
//
// The 128-row tiles of the tensor-core kernels would be empty, and what counts is reading the weights once: 24 MB for
// 1024 -> 4096 -> 1024 in bfloat16, 3.8 us.  So every multiplication is an fp32 FMA on CUDA cores (exact products of 16-bit
// values; float32 in float32) and the layout serves the loads: a block owns 128 bytes of columns (whole cache lines) and a part
// of the contraction axis, its threads run down the rows of the weights, 16 bytes each; the blocks of a cluster share the
// axis and their sums meet in the first one's shared memory.  All sums are added in a fixed order.  Weights whose columns are
// contiguous (transposed views) are read along the contraction axis instead, a warp per column.  Rows are taken four at a
// time; the second four find the weights in the L2.
#include "common.cuh"
#include "convert.cuh"
#include "gate.cuh"

#include <cooperative_groups.h>

namespace nva {
using at::Tensor;
namespace {

constexpr int kRowBlock = 4;   // rows of x per pass
constexpr int kMaxSmem = 96 * 1024, kLanes = 8;  // column lanes of a block

template <typename T, int VEC>
struct alignas(sizeof(T) * VEC) Vec { T v[VEC]; };

__device__ __forceinline__ float gate_of(int act, float g) {
  float a, da;
  if (act == kSilu) activate<true, kSilu>(g, a, da);
  else activate<true, kGelu>(g, a, da);
  return a;
}

// x [rows][k0, k1) to shared memory as fp32 [k][R] (one load per k for all rows)
template <typename X, int R>
__device__ __forceinline__ void stage_rows(float* xs, const X* x, int64_t ldx, int64_t sx, int rows, int k0, int k1) {
  for (int i = k0 + threadIdx.x; i < k1; i += blockDim.x)
#pragma unroll
    for (int r = 0; r < R; ++r) xs[(i - k0) * R + r] = r < rows ? widen(x[r * ldx + i * sx]) : 0.f;
  __syncthreads();
}

// MATS = 2: out = act(x W0) * (x W1); MATS = 1: out = x W0.  W [k][n], rows ld apart.  Block: kLanes lanes of VEC columns,
// blockDim / kLanes rows at a time.  grid (column blocks x cluster, passes of R rows).
template <typename T, typename X, int VEC, int MATS, int R>
__global__ void __launch_bounds__(256) rows_by_k_kernel(const X* __restrict__ x, int64_t ldx, int64_t sx, const T* __restrict__ w0,
                                                        int64_t ld0, const T* __restrict__ w1, int64_t ld1, int total_rows, int k, int n,
                                                        int act, void* __restrict__ out, int64_t ldo, int out32) {
  namespace cg = cooperative_groups;
  extern __shared__ float xs[];
  constexpr int COLS = kLanes * VEC, WARPS = 8;
  __shared__ float part[WARPS][MATS * R * COLS];
  __shared__ float sums[MATS * R * COLS];
  auto cluster = cg::this_cluster();
  const int parts = (int)cluster.num_blocks(), rank = (int)cluster.block_rank(), c0 = (int)blockIdx.x / parts * COLS;
  const int k_lo = (int)((int64_t)k * rank / parts), k_hi = (int)((int64_t)k * (rank + 1) / parts);
  const int r0 = blockIdx.y * R, rows = min(R, total_rows - r0);
  const int lc = threadIdx.x % kLanes, kr = threadIdx.x / kLanes, c = c0 + lc * VEC;
  constexpr int STEP = 256 / kLanes, U = 4;  // rows of the weights at a time, loads in flight per matrix
  float acc[MATS][R][VEC];
#pragma unroll
  for (int m = 0; m < MATS; ++m)
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int v = 0; v < VEC; ++v) acc[m][r][v] = 0.f;
  Vec<T, VEC> a[U], b[U];
  auto load = [&](int k0) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int kk = min(k0 + u * STEP, k_hi - 1);  // past the end: the last row again, not used below
      if (c < n) {
        a[u] = *reinterpret_cast<const Vec<T, VEC>*>(w0 + kk * ld0 + c);
        if constexpr (MATS == 2) b[u] = *reinterpret_cast<const Vec<T, VEC>*>(w1 + kk * ld1 + c);
      }
    }
  };
  // The first weights are on their way before x is waited for: a second launch reads what the first one writes as x alone.
  load(k_lo + kr);
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  stage_rows<X, R>(xs, x + r0 * ldx, ldx, sx, rows, k_lo, k_hi);
  for (int k0 = k_lo + kr; k0 < k_hi; k0 += U * STEP) {
    if (k0 != k_lo + kr) load(k0);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int kk = k0 + u * STEP;
      if (kk < k_hi && c < n) {
#pragma unroll
        for (int r = 0; r < R; ++r) {
          const float xv = xs[(kk - k_lo) * R + r];
#pragma unroll
          for (int v = 0; v < VEC; ++v) {
            acc[0][r][v] += xv * widen(a[u].v[v]);
            if constexpr (MATS == 2) acc[1][r][v] += xv * widen(b[u].v[v]);
          }
        }
      }
    }
  }
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
#pragma unroll
  for (int m = 0; m < MATS; ++m)
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int v = 0; v < VEC; ++v) {
        float s = acc[m][r][v];
#pragma unroll
        for (int o = 16; o >= kLanes; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        if (lane < kLanes) part[warp][(m * R + r) * COLS + lane * VEC + v] = s;
      }
  __syncthreads();
  for (int i = threadIdx.x; i < MATS * R * COLS; i += blockDim.x) {
    float s = 0.f;
#pragma unroll
    for (int q = 0; q < WARPS; ++q) s += part[q][i];
    sums[i] = s;
  }
  cluster.sync();
  if (rank == 0)
    for (int i = threadIdx.x; i < R * COLS; i += blockDim.x) {
      const int r = i / COLS, col = c0 + i % COLS;
      if (r >= rows || col >= n) continue;
      float s[MATS];
#pragma unroll
      for (int m = 0; m < MATS; ++m) {
        s[m] = 0.f;
        for (int q = 0; q < parts; ++q) s[m] += cluster.map_shared_rank(sums, q)[m * R * COLS + i];
      }
      float o = s[0];
      if constexpr (MATS == 2) o = gate_of(act, s[0]) * s[1];
      if (out32) ((float*)out)[(int64_t)(r0 + r) * ldo + col] = o;
      else ((T*)out)[(int64_t)(r0 + r) * ldo + col] = narrow<T>(o);
    }
  cluster.sync();  // the first block has read the others' sums
}

// The same for weights whose columns are contiguous: W^T [n][k], rows ld apart; a warp per column.
template <typename T, typename X, int VEC, int MATS, int R>
__global__ void __launch_bounds__(256) rows_by_n_kernel(const X* __restrict__ x, int64_t ldx, int64_t sx, const T* __restrict__ w0,
                                                        int64_t ld0, const T* __restrict__ w1, int64_t ld1, int total_rows, int k, int n,
                                                        int act, void* __restrict__ out, int64_t ldo, int out32) {
  extern __shared__ float xs[];
  const int r0 = blockIdx.y * R, rows = min(R, total_rows - r0);
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  stage_rows<X, R>(xs, x + r0 * ldx, ldx, sx, rows, 0, k);
  const int col = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (col >= n) return;
  float acc[MATS][R] = {};
#pragma unroll 2
  for (int k0 = lane * VEC; k0 < k; k0 += 32 * VEC) {
    const Vec<T, VEC> a = *reinterpret_cast<const Vec<T, VEC>*>(w0 + col * ld0 + k0);
    Vec<T, VEC> b;
    if constexpr (MATS == 2) b = *reinterpret_cast<const Vec<T, VEC>*>(w1 + col * ld1 + k0);
#pragma unroll
    for (int v = 0; v < VEC; ++v)
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const float xv = xs[(k0 + v) * R + r];
        acc[0][r] += xv * widen(a.v[v]);
        if constexpr (MATS == 2) acc[1][r] += xv * widen(b.v[v]);
      }
  }
#pragma unroll
  for (int r = 0; r < R; ++r) {
    float s[MATS];
#pragma unroll
    for (int m = 0; m < MATS; ++m) {
      s[m] = acc[m][r];
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) s[m] += __shfl_xor_sync(0xffffffffu, s[m], o);
    }
    if (lane == 0 && r < rows) {
      float o = s[0];
      if constexpr (MATS == 2) o = gate_of(act, s[0]) * s[1];
      if (out32) ((float*)out)[(int64_t)(r0 + r) * ldo + col] = o;
      else ((T*)out)[(int64_t)(r0 + r) * ldo + col] = narrow<T>(o);
    }
  }
}

struct Weight { const void* p; int64_t ld; bool by_k; };  // by_k: rows of the contraction axis are contiguous
bool as_weight(const Tensor& w, Weight& o) {
  if (w.stride(1) == 1 || w.size(1) == 1) o = {w.data_ptr(), w.stride(0), true};
  else if (w.stride(0) == 1 || w.size(0) == 1) o = {w.data_ptr(), w.stride(1), false};
  else return false;
  return true;
}

// One product; X is the type of x.  Returns after the launch.
template <typename T, typename X, int MATS, int R>
void product(const X* x, int64_t ldx, int64_t sx, const Weight& a, const Weight& b, int rows, int k, int n, int act, void* out, int64_t ldo,
             bool out32, cudaStream_t st) {
  constexpr int VEC = 16 / (int)sizeof(T);
  const int passes = (rows + R - 1) / R;
  auto aligned = [&](const Weight& w, int64_t inner) {
    return inner % VEC == 0 && w.ld % VEC == 0 && (reinterpret_cast<uintptr_t>(w.p) & 15) == 0;
  };
  const bool vec = aligned(a, a.by_k ? n : k) && (MATS == 1 || aligned(b, a.by_k ? n : k));
  auto go = [&](auto kernel, int blocks, int parts) {
    C10_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxSmem));
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)(blocks * parts), (unsigned)passes);
    cfg.blockDim = dim3(256);
    cfg.dynamicSmemBytes = (size_t)((k + parts - 1) / parts) * R * sizeof(float);
    cfg.stream = st;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = (unsigned)parts; at[0].val.clusterDim.y = 1; at[0].val.clusterDim.z = 1;
    at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = MATS == 1 ? 2 : 1;  // the first launch reads weights before it waits: it must not start early itself
    C10_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kernel, x, ldx, sx, (const T*)a.p, a.ld, (const T*)b.p, b.ld, rows, k, n, act, out, ldo, out32 ? 1 : 0));
  };
  if (!a.by_k) {
    if (vec) go(rows_by_n_kernel<T, X, VEC, MATS, R>, (n + 7) / 8, 1);
    else go(rows_by_n_kernel<T, X, 1, MATS, R>, (n + 7) / 8, 1);
    return;
  }
  // blocks of a cluster: enough for two blocks on every SM, as long as each still has 64 rows of the weights (1024 -> 4096 -> 1024,
  // one row, both launches: 50 us without clusters, 27 us in twos, 16.7 us in fours, 16.3 us in eights; with eight loads in
  // flight a thread instead of four 18.3 us; the cluster barriers are 1.8 us of a launch)
  auto split = [&](int blocks) {
    int parts = 1;
    while (parts < 8 && blocks * parts < 296 && k / (2 * parts) >= 64) parts *= 2;
    return parts;
  };
  const int cols = kLanes * (vec ? VEC : 1), blocks = (n + cols - 1) / cols;
  if (vec) go(rows_by_k_kernel<T, X, VEC, MATS, R>, blocks, split(blocks));
  else go(rows_by_k_kernel<T, X, 1, MATS, R>, blocks, split(blocks));
}

template <typename T, int R>
void block(const Tensor& x, const Weight& g, const Weight& u, const Weight& d, int H, int N, int act, Tensor& h, Tensor& y, cudaStream_t st) {
  const int M = (int)x.size(0), K = (int)x.size(1);
  product<T, T, 2, R>((const T*)x.data_ptr(), x.stride(0), x.stride(1), g, u, M, K, H, act, h.data_ptr(), H, true, st);
  product<T, float, 1, R>(h.data_ptr<float>(), H, 1, d, d, M, H, N, act, y.data_ptr(), N, false, st);
}

}  // namespace

// True when this path took the call (few rows, intermediate rows fit shared memory).  h is kept in fp32 between the launches.
bool gated_ff_rows(const Tensor& x, const Tensor& wg, const Tensor& wu, const Tensor& wd, int64_t act, Tensor& y, cudaStream_t st) {
  const int64_t M = x.size(0), K = x.size(1), H = wg.size(1), N = wd.size(1);
  const int R = M == 1 ? 1 : M == 2 ? 2 : kRowBlock;
  if (M > 2 * kRowBlock || std::max(K, H) * R * 4 > kMaxSmem || N >= (1ll << 31)) return false;
  Weight g, u, d;
  if (!as_weight(wg, g) || !as_weight(wu, u) || !as_weight(wd, d) || g.by_k != u.by_k) return false;
  Tensor h = at::empty({M, H}, x.options().dtype(at::kFloat));
  auto rows = [&](auto v) {
    using T = decltype(v);
    if (R == 1) block<T, 1>(x, g, u, d, (int)H, (int)N, (int)act, h, y, st);
    else if (R == 2) block<T, 2>(x, g, u, d, (int)H, (int)N, (int)act, h, y, st);
    else block<T, kRowBlock>(x, g, u, d, (int)H, (int)N, (int)act, h, y, st);
  };
  if (x.scalar_type() == at::kFloat) rows(float{});
  else if (x.scalar_type() == at::kHalf) rows(__half{});
  else rows(__nv_bfloat16{});
  return true;
}

}  // namespace nva
