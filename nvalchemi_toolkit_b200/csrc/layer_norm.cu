// SPDX-License-Identifier: Apache-2.0
// Layer norm over the last axis, forward and backward, with the reduction of the weight and bias gradients.
//
//   mu = mean_c x,  r = 1 / sqrt(mean_c (x - mu)^2 + eps),  xh = (x - mu) r,  y = xh w + b
//   dx = r (g w - mean_c(g w) - xh mean_c(g w xh)),  dw = sum_rows g xh,  db = sum_rows g
//
// Both directions are bound by memory: 2 (forward) and 3 (backward) row-sized arrays move once.  A row stays in the
// registers of the threads that loaded it (TPR threads, VPT vectors of VEC elements each), so the mean and the centred
// second moment are two exact passes over registers and nothing is read twice.  Statistics and all sums are fp32 (float64
// rows: float64); only the stored results are rounded to the tensors' types.
// The backward grid is persistent: a thread owns the same columns in every row it visits and keeps their dw / db sums in
// registers; the block's row groups are added in a fixed order in shared memory, one partial row per block goes to the
// workspace, and a second kernel adds the partial rows in a fixed order, so results do not change from run to run.
#include "common.cuh"

#include "convert.cuh"

namespace nva {
using at::Tensor;
namespace {

template <typename T, int VEC>
struct alignas(sizeof(T) * VEC) Pack { T v[VEC]; };

template <typename A> __device__ __forceinline__ A inv_sqrt(A x);
template <> __device__ __forceinline__ float inv_sqrt<float>(float x) { return 1.f / sqrtf(x); }
template <> __device__ __forceinline__ double inv_sqrt<double>(double x) { return 1.0 / sqrt(x); }

// Sum over the TPR threads that share a row; every one of them gets it.  TPR > 32: the whole block is one row group.
template <int TPR, typename A>
__device__ __forceinline__ A row_sum(A v, A* scratch) {
#pragma unroll
  for (int o = (TPR < 32 ? TPR : 32) / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if constexpr (TPR > 32) {
    constexpr int W = TPR / 32;
    __syncthreads();  // the previous use of scratch has been read
    if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
    __syncthreads();
    v = scratch[0];
#pragma unroll
    for (int i = 1; i < W; ++i) v += scratch[i];
  }
  return v;
}

template <int TPR> constexpr int kBlock = TPR > 32 ? TPR : 256;  // threads of a block

template <typename T, typename W, int VEC, int TPR, int VPT>
__global__ void __launch_bounds__(kBlock<TPR>)
    layer_norm_fwd_kernel(const T* __restrict__ x, int64_t ldx, const W* __restrict__ w, const W* __restrict__ b,
                          T* __restrict__ y, typename AccOf<T>::type* __restrict__ mean,
                          typename AccOf<T>::type* __restrict__ rstd, int64_t rows, int cols, double eps) {
  using A = typename AccOf<T>::type;
  __shared__ A scratch[32];
  constexpr int RPB = kBlock<TPR> / TPR;
  const int lane = threadIdx.x % TPR;
  const int64_t row = (int64_t)blockIdx.x * RPB + threadIdx.x / TPR;
  const bool live = row < rows;  // dead groups take part in the shuffles with zeros
  A v[VPT * VEC];
  A sum = 0;
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int c = (i * TPR + lane) * VEC;
    if (live && c < cols) {
      const Pack<T, VEC> p = *reinterpret_cast<const Pack<T, VEC>*>(x + row * ldx + c);
#pragma unroll
      for (int k = 0; k < VEC; ++k) { v[i * VEC + k] = widen(p.v[k]); sum += v[i * VEC + k]; }
    }
  }
  const A inv_n = (A)1 / (A)cols;
  const A mu = row_sum<TPR>(sum, scratch) * inv_n;
  A sq = 0;
#pragma unroll
  for (int i = 0; i < VPT; ++i)
    if (live && (i * TPR + lane) * VEC < cols)
#pragma unroll
      for (int k = 0; k < VEC; ++k) { const A d = v[i * VEC + k] - mu; sq += d * d; }
  const A r = inv_sqrt<A>(row_sum<TPR>(sq, scratch) * inv_n + (A)eps);
  if (!live) return;
  if (lane == 0 && mean != nullptr) { mean[row] = mu; rstd[row] = r; }
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int c = (i * TPR + lane) * VEC;
    if (c < cols) {
      Pack<W, VEC> pw, pb;
      if (w != nullptr) pw = *reinterpret_cast<const Pack<W, VEC>*>(w + c);
      if (b != nullptr) pb = *reinterpret_cast<const Pack<W, VEC>*>(b + c);
      Pack<T, VEC> o;
#pragma unroll
      for (int k = 0; k < VEC; ++k) {
        A t = (v[i * VEC + k] - mu) * r;
        if (w != nullptr) t *= widen(pw.v[k]);
        if (b != nullptr) t += widen(pb.v[k]);
        o.v[k] = narrow<T>(t);
      }
      *reinterpret_cast<Pack<T, VEC>*>(y + row * cols + c) = o;
    }
  }
}

// partial [gridDim.x][2][cols]: this block's sums of g xh and g (null when neither gradient is wanted).
template <typename T, typename W, int VEC, int TPR, int VPT>
__global__ void __launch_bounds__(kBlock<TPR>)
    layer_norm_bwd_kernel(const T* __restrict__ g, int64_t ldg, const T* __restrict__ x, int64_t ldx,
                          const typename AccOf<T>::type* __restrict__ mean, const typename AccOf<T>::type* __restrict__ rstd,
                          const W* __restrict__ w, T* __restrict__ dx, typename AccOf<T>::type* __restrict__ partial,
                          int64_t rows, int cols) {
  using A = typename AccOf<T>::type;
  constexpr int THREADS = kBlock<TPR>, RPB = THREADS / TPR, E = VPT * VEC;
  __shared__ A scratch[32];
  __shared__ A fold[RPB > 1 ? THREADS * VEC : 1];
  const int lane = threadIdx.x % TPR, group = threadIdx.x / TPR;
  A dw[E], db[E];
#pragma unroll
  for (int i = 0; i < E; ++i) { dw[i] = 0; db[i] = 0; }
  const A inv_n = (A)1 / (A)cols;
  for (int64_t row0 = (int64_t)blockIdx.x * RPB; row0 < rows; row0 += (int64_t)gridDim.x * RPB) {
    const int64_t row = row0 + group;
    const bool live = row < rows;
    Pack<T, VEC> pg[VPT], px[VPT];
    A mu = 0, r = 0;
    if (live) { mu = mean[row]; r = rstd[row]; }
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int c = (i * TPR + lane) * VEC;
      if (live && c < cols) {
        pg[i] = *reinterpret_cast<const Pack<T, VEC>*>(g + row * ldg + c);
        px[i] = *reinterpret_cast<const Pack<T, VEC>*>(x + row * ldx + c);
      }
    }
    A s1 = 0, s2 = 0;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int c = (i * TPR + lane) * VEC;
      if (live && c < cols) {
        Pack<W, VEC> pw;
        if (w != nullptr) pw = *reinterpret_cast<const Pack<W, VEC>*>(w + c);
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
          const A gv = widen(pg[i].v[k]), xh = (widen(px[i].v[k]) - mu) * r;
          dw[i * VEC + k] += gv * xh;
          db[i * VEC + k] += gv;
          const A gw = w != nullptr ? gv * widen(pw.v[k]) : gv;
          s1 += gw;
          s2 += gw * xh;
        }
      }
    }
    s1 = row_sum<TPR>(s1, scratch) * inv_n;
    s2 = row_sum<TPR>(s2, scratch) * inv_n;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int c = (i * TPR + lane) * VEC;
      if (live && c < cols) {
        Pack<W, VEC> pw;
        if (w != nullptr) pw = *reinterpret_cast<const Pack<W, VEC>*>(w + c);
        Pack<T, VEC> o;
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
          const A gv = widen(pg[i].v[k]), xh = (widen(px[i].v[k]) - mu) * r;
          const A gw = w != nullptr ? gv * widen(pw.v[k]) : gv;
          o.v[k] = narrow<T>(r * (gw - s1 - xh * s2));
        }
        *reinterpret_cast<Pack<T, VEC>*>(dx + row * cols + c) = o;
      }
    }
  }
  if (partial == nullptr) return;
  A* out = partial + (int64_t)blockIdx.x * 2 * cols;
#pragma unroll
  for (int which = 0; which < 2; ++which) {
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int c = (i * TPR + lane) * VEC;
      if constexpr (RPB > 1) {
        __syncthreads();
#pragma unroll
        for (int k = 0; k < VEC; ++k) fold[(group * VEC + k) * TPR + lane] = which ? db[i * VEC + k] : dw[i * VEC + k];
        __syncthreads();
        if (group == 0 && c < cols) {
#pragma unroll
          for (int k = 0; k < VEC; ++k) {
            A s = 0;
            for (int gr = 0; gr < RPB; ++gr) s += fold[(gr * VEC + k) * TPR + lane];
            out[which * cols + c + k] = s;
          }
        }
      } else if (c < cols) {
#pragma unroll
        for (int k = 0; k < VEC; ++k) out[which * cols + c + k] = which ? db[i * VEC + k] : dw[i * VEC + k];
      }
    }
  }
}

// Column sums of partial [blocks][2 cols]: 32 columns per block, 32 threads down each of them, added in a fixed order.
template <typename A, typename W>
__global__ void __launch_bounds__(1024) layer_norm_fold_kernel(const A* __restrict__ partial, int blocks, int cols,
                                                               W* __restrict__ dw, W* __restrict__ db) {
  __shared__ A tile[32][33];
  const int c = blockIdx.x * 32 + threadIdx.x;
  A s = 0;
  if (c < 2 * cols)
    for (int i = threadIdx.y; i < blocks; i += 32) s += partial[(int64_t)i * 2 * cols + c];
  tile[threadIdx.y][threadIdx.x] = s;
  __syncthreads();
  if (threadIdx.y == 0 && c < 2 * cols) {
    s = 0;
    for (int i = 0; i < 32; ++i) s += tile[i][threadIdx.x];
    if (c < cols) { if (dw != nullptr) dw[c] = narrow<W>(s); }
    else if (db != nullptr) db[c - cols] = narrow<W>(s);
  }
}

constexpr int64_t kMaxCols = 8192;

struct LnArgs {
  const void *g, *x, *w, *b;
  void *y, *mean, *rstd, *partial, *dw, *db;
  int64_t ldg, ldx, rows;
  int cols, blocks;
  double eps;
  bool backward;
  cudaStream_t st;
};

template <typename T, typename W, int VEC, int TPR, int VPT>
int launch(const LnArgs& a, bool count_only) {
  using A = typename AccOf<T>::type;
  constexpr int THREADS = kBlock<TPR>, RPB = THREADS / TPR;
  const int64_t need = (a.rows + RPB - 1) / RPB;
  if (!a.backward) {
    TORCH_CHECK(need < (int64_t)2147483647, "layer_norm: too many rows");
    layer_norm_fwd_kernel<T, W, VEC, TPR, VPT><<<(unsigned)need, THREADS, 0, a.st>>>(
        (const T*)a.x, a.ldx, (const W*)a.w, (const W*)a.b, (T*)a.y, (A*)a.mean, (A*)a.rstd, a.rows, a.cols, a.eps);
    return 0;
  }
  if (count_only) {  // blocks of the persistent grid: what fits on the GPU at once, less when there are fewer rows
    int per_sm = 1, dev = 0, sms = 148;
    C10_CUDA_CHECK(cudaGetDevice(&dev));
    C10_CUDA_CHECK(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev));
    C10_CUDA_CHECK(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, layer_norm_bwd_kernel<T, W, VEC, TPR, VPT>, THREADS, 0));
    return (int)std::min<int64_t>(need, (int64_t)sms * std::max(per_sm, 1));
  }
  layer_norm_bwd_kernel<T, W, VEC, TPR, VPT><<<a.blocks, THREADS, 0, a.st>>>(
      (const T*)a.g, a.ldg, (const T*)a.x, a.ldx, (const A*)a.mean, (const A*)a.rstd, (const W*)a.w, (T*)a.y, (A*)a.partial,
      a.rows, a.cols);
  return a.blocks;
}

// Threads per row: a part of a warp for short rows (no idle lanes, no shared memory), the whole warp up to four vectors a
// lane, a block of its own for longer rows.
template <typename T, typename W, int VEC>
int pick(const LnArgs& a, bool count_only) {
  const int nv = (a.cols + VEC - 1) / VEC;
  if constexpr (VEC == 1) {
    if (nv <= 128) return launch<T, W, 1, 32, 4>(a, count_only);
    if (nv <= 512) return launch<T, W, 1, 32, 16>(a, count_only);
    if (nv <= 2048) return launch<T, W, 1, 128, 16>(a, count_only);
    return launch<T, W, 1, 512, 16>(a, count_only);
  } else {
    if (nv <= 8) return launch<T, W, VEC, 8, 1>(a, count_only);
    if (nv <= 16) return launch<T, W, VEC, 16, 1>(a, count_only);
    if (nv <= 32) return launch<T, W, VEC, 32, 1>(a, count_only);
    if (nv <= 64) return launch<T, W, VEC, 32, 2>(a, count_only);
    if (nv <= 128) return launch<T, W, VEC, 32, 4>(a, count_only);
    if (nv <= 256) return launch<T, W, VEC, 128, 2>(a, count_only);
    if (nv <= 512) return launch<T, W, VEC, 256, 2>(a, count_only);
    if (nv <= 1024) return launch<T, W, VEC, 512, 2>(a, count_only);
    return launch<T, W, VEC, 512, 16 / VEC>(a, count_only);
  }
}

template <typename T, typename W>
int pick_vec(const LnArgs& a, bool count_only) {
  constexpr int VEC = 16 / (int)sizeof(T);
  // 16-byte accesses need every row of every tensor on a 16-byte boundary (weights: their own vector size)
  auto ok = [](const void* p, size_t n) { return (reinterpret_cast<uintptr_t>(p) % n) == 0; };
  constexpr size_t kW = sizeof(W) * VEC;
  const bool vec = a.cols % VEC == 0 && ok(a.x, 16) && ok(a.y, 16) && ok(a.g, 16) && a.ldx % VEC == 0 && a.ldg % VEC == 0 &&
                   ok(a.w, kW) && ok(a.b, kW);
  return vec ? pick<T, W, VEC>(a, count_only) : pick<T, W, 1>(a, count_only);
}

int dispatch(const LnArgs& a, at::ScalarType xt, at::ScalarType wt, bool count_only) {
  if (xt == at::kFloat && wt == at::kFloat) return pick_vec<float, float>(a, count_only);
  if (xt == at::kDouble && wt == at::kDouble) return pick_vec<double, double>(a, count_only);
  if (xt == at::kBFloat16 && wt == at::kBFloat16) return pick_vec<__nv_bfloat16, __nv_bfloat16>(a, count_only);
  if (xt == at::kBFloat16 && wt == at::kFloat) return pick_vec<__nv_bfloat16, float>(a, count_only);
  if (xt == at::kHalf && wt == at::kHalf) return pick_vec<__half, __half>(a, count_only);
  if (xt == at::kHalf && wt == at::kFloat) return pick_vec<__half, float>(a, count_only);
  TORCH_CHECK(false, "layer_norm: rows of type ", xt, " with weights of type ", wt, " are not supported");
}

void check_rows(const Tensor& t, const char* name) {
  TORCH_CHECK(t.is_cuda() && t.dim() == 2 && (t.size(1) == 1 || t.stride(1) == 1 || t.numel() == 0), "layer_norm: ", name,
              " must be a CUDA matrix with contiguous rows");
}
void check_vector(const c10::optional<Tensor>& t, const Tensor& x, const char* name) {
  if (!t.has_value()) return;
  TORCH_CHECK(t->device() == x.device() && t->dim() == 1 && t->is_contiguous() && t->size(0) == x.size(1), "layer_norm: ", name,
              " must be a contiguous vector of the row length on the device of x");
}
void* ptr(const c10::optional<Tensor>& t) { return t.has_value() ? t->data_ptr() : nullptr; }

}  // namespace

std::tuple<Tensor, Tensor, Tensor> layer_norm_fwd(const Tensor& x, const c10::optional<Tensor>& weight,
                                                  const c10::optional<Tensor>& bias, double eps, bool stats) {
  check_rows(x, "x");
  check_vector(weight, x, "weight");
  check_vector(bias, x, "bias");
  TORCH_CHECK(x.size(1) >= 1 && x.size(1) <= kMaxCols, "layer_norm: row length must lie in 1..", kMaxCols);
  const at::ScalarType wt = weight.has_value() ? weight->scalar_type() : bias.has_value() ? bias->scalar_type() : x.scalar_type();
  TORCH_CHECK(!bias.has_value() || bias->scalar_type() == wt, "layer_norm: weight and bias must have one type");
  c10::cuda::CUDAGuard guard(x.device());
  Tensor y = at::empty({x.size(0), x.size(1)}, x.options());
  auto so = x.options().dtype(x.scalar_type() == at::kDouble ? at::kDouble : at::kFloat);
  Tensor mean = at::empty({stats ? x.size(0) : 0}, so), rstd = at::empty({stats ? x.size(0) : 0}, so);
  if (x.size(0) == 0) return {y, mean, rstd};
  LnArgs a{};
  a.x = x.data_ptr(); a.w = ptr(weight); a.b = ptr(bias); a.y = y.data_ptr();
  a.mean = stats ? mean.data_ptr() : nullptr; a.rstd = stats ? rstd.data_ptr() : nullptr;
  a.ldx = x.stride(0); a.rows = x.size(0); a.cols = (int)x.size(1); a.eps = eps;
  a.st = at::cuda::getCurrentCUDAStream();
  dispatch(a, x.scalar_type(), wt, false);
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  return {y, mean, rstd};
}

std::tuple<Tensor, Tensor, Tensor> layer_norm_bwd(const Tensor& grad, const Tensor& x, const Tensor& mean, const Tensor& rstd,
                                                  const c10::optional<Tensor>& weight, bool want_params,
                                                  c10::optional<at::ScalarType> param_type) {
  check_rows(x, "x");
  check_rows(grad, "grad");
  check_vector(weight, x, "weight");
  TORCH_CHECK(x.size(1) >= 1 && x.size(1) <= kMaxCols, "layer_norm: row length must lie in 1..", kMaxCols);
  TORCH_CHECK(grad.sizes() == x.sizes() && grad.scalar_type() == x.scalar_type() && grad.device() == x.device(),
              "layer_norm: grad must match x");
  const at::ScalarType st = x.scalar_type() == at::kDouble ? at::kDouble : at::kFloat;
  for (const Tensor* s : {&mean, &rstd})
    TORCH_CHECK(s->device() == x.device() && s->dim() == 1 && s->is_contiguous() && s->size(0) == x.size(0) && s->scalar_type() == st,
                "layer_norm: mean and rstd must be the forward pass's statistics");
  const at::ScalarType wt = weight.has_value() ? weight->scalar_type() : param_type.value_or(x.scalar_type());
  c10::cuda::CUDAGuard guard(x.device());
  const int64_t cols = x.size(1);
  Tensor dx = at::empty({x.size(0), cols}, x.options());
  Tensor dw = at::empty({want_params ? cols : 0}, x.options().dtype(wt)), db = at::empty_like(dw);
  if (x.size(0) == 0) return {dx, dw.zero_(), db.zero_()};
  LnArgs a{};
  a.backward = true;
  a.g = grad.data_ptr(); a.x = x.data_ptr(); a.w = ptr(weight); a.y = dx.data_ptr();
  a.mean = mean.data_ptr(); a.rstd = rstd.data_ptr();
  a.ldg = grad.stride(0); a.ldx = x.stride(0); a.rows = x.size(0); a.cols = (int)cols;
  a.st = at::cuda::getCurrentCUDAStream();
  a.blocks = dispatch(a, x.scalar_type(), wt, true);
  Tensor partial;
  if (want_params) {
    partial = at::empty({a.blocks, 2, cols}, mean.options());
    a.partial = partial.data_ptr();
  }
  dispatch(a, x.scalar_type(), wt, false);
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  if (want_params) {
    const dim3 grid((unsigned)((2 * cols + 31) / 32)), block(32, 32);
    auto fold = [&](auto acc, auto wv) {
      using A = decltype(acc);
      using W = decltype(wv);
      layer_norm_fold_kernel<A, W><<<grid, block, 0, a.st>>>((const A*)a.partial, a.blocks, (int)cols, (W*)dw.data_ptr(), (W*)db.data_ptr());
    };
    if (st == at::kDouble) fold(double{}, double{});
    else if (wt == at::kFloat) fold(float{}, float{});
    else if (wt == at::kHalf) fold(float{}, __half{});
    else fold(float{}, __nv_bfloat16{});
    C10_CUDA_KERNEL_LAUNCH_CHECK();
  }
  return {dx, dw, db};
}

}  // namespace nva

TORCH_LIBRARY_FRAGMENT(nvalchemi, m) {
  m.def("layer_norm_fwd(Tensor x, Tensor? weight, Tensor? bias, float eps, bool stats) -> (Tensor, Tensor, Tensor)", &nva::layer_norm_fwd);
  m.def("layer_norm_bwd(Tensor grad, Tensor x, Tensor mean, Tensor rstd, Tensor? weight, bool want_params, ScalarType? param_type) -> (Tensor, Tensor, Tensor)", &nva::layer_norm_bwd);
}
