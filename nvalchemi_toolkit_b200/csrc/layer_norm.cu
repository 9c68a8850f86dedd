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
// What counts is bytes under way: 64 bytes a thread (R rows of a group at a time where rows are short) and many resident
// threads; loading the next rows ahead of a persistent block's reductions costs registers and with them residency, and was
// slower (16,384 x 4096 float16 backward 182 us against 112 us).  In the backward pass the grid is persistent, a thread owns the
// same columns in every row it visits and keeps their dw / db sums in registers; a block's row groups are added in a fixed
// order in shared memory, one partial row per block goes to the workspace, and a second kernel adds the partial rows in a fixed order, so results do not change from run to run.
// 131,072 x 128 bfloat16: forward 18 us (3.7 TB/s), backward 27 us (3.7 TB/s) and 4 us for the sums; 16,384 x 4096 float16: 58 us
// (4.6 TB/s), 100 us (4.0 TB/s) and 7 us.
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

// Sums over the TPR threads that share a row; every one of them gets them.  TPR > 32: the whole block is one row group, and
// two buffers take turns, so that one barrier per call is enough.
template <int TPR, int N, typename A>
__device__ __forceinline__ void row_sum(A (&v)[N], A (*scratch)[N][32], int& turn) {
#pragma unroll
  for (int n = 0; n < N; ++n)
#pragma unroll
    for (int o = (TPR < 32 ? TPR : 32) / 2; o > 0; o >>= 1) v[n] += __shfl_xor_sync(0xffffffffu, v[n], o);
  if constexpr (TPR > 32) {
    constexpr int W = TPR / 32;
    turn ^= 1;
    if ((threadIdx.x & 31) == 0)
#pragma unroll
      for (int n = 0; n < N; ++n) scratch[turn][n][threadIdx.x >> 5] = v[n];
    __syncthreads();
#pragma unroll
    for (int n = 0; n < N; ++n) {
      v[n] = scratch[turn][n][0];
#pragma unroll
      for (int i = 1; i < W; ++i) v[n] += scratch[turn][n][i];
    }
  }
}

template <int TPR> constexpr int kBlock = TPR > 32 ? TPR : 256;  // threads of a block

// threads of a block that leave room for two more blocks of 256 on the SM
template <int TPR> constexpr int kMinBlocks = kBlock<TPR> == 256 && TPR > 32 ? 3 : 1;

template <typename T, int VEC, int TPR, int VPT>
__device__ __forceinline__ void load_row(Pack<T, VEC> (&p)[VPT], const T* src, int64_t row, int64_t ld, int64_t rows, int cols, int lane) {
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int c = (i * TPR + lane) * VEC;
    if (row < rows && c < cols) p[i] = *reinterpret_cast<const Pack<T, VEC>*>(src + row * ld + c);
  }
}

template <typename T, typename W, int VEC, int TPR, int VPT, int R>
__global__ void __launch_bounds__(kBlock<TPR>)
    layer_norm_fwd_kernel(const T* __restrict__ x, int64_t ldx, const W* __restrict__ w, const W* __restrict__ b,
                          T* __restrict__ y, typename AccOf<T>::type* __restrict__ mean,
                          typename AccOf<T>::type* __restrict__ rstd, int64_t rows, int cols, double eps) {
  using A = typename AccOf<T>::type;
  __shared__ A scratch[2][R][32];
  int turn = 0;
  constexpr int RPB = kBlock<TPR> / TPR;
  const int lane = threadIdx.x % TPR;
  const int64_t row0 = (int64_t)blockIdx.x * (RPB * R) + threadIdx.x / TPR;  // rows past the end take part in the sums with zeros
  const A inv_n = (A)1 / (A)cols;
  Pack<T, VEC> p[R][VPT];
#pragma unroll
  for (int r = 0; r < R; ++r) load_row<T, VEC, TPR, VPT>(p[r], x, row0 + r * RPB, ldx, rows, cols, lane);
  A sum[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    sum[r] = 0;
#pragma unroll
    for (int i = 0; i < VPT; ++i)
      if (row0 + r * RPB < rows && (i * TPR + lane) * VEC < cols)
#pragma unroll
        for (int k = 0; k < VEC; ++k) sum[r] += widen(p[r][i].v[k]);
  }
  row_sum<TPR>(sum, scratch, turn);
  A sq[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    sum[r] *= inv_n;
    sq[r] = 0;
#pragma unroll
    for (int i = 0; i < VPT; ++i)
      if (row0 + r * RPB < rows && (i * TPR + lane) * VEC < cols)
#pragma unroll
        for (int k = 0; k < VEC; ++k) { const A d = widen(p[r][i].v[k]) - sum[r]; sq[r] += d * d; }
  }
  row_sum<TPR>(sq, scratch, turn);
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int64_t row = row0 + r * RPB;
    sq[r] = inv_sqrt<A>(sq[r] * inv_n + (A)eps);
    if (lane == 0 && row < rows && mean != nullptr) { mean[row] = sum[r]; rstd[row] = sq[r]; }
  }
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int c = (i * TPR + lane) * VEC;
    if (c >= cols) continue;
    Pack<W, VEC> pw, pb;
    if (w != nullptr) pw = *reinterpret_cast<const Pack<W, VEC>*>(w + c);
    if (b != nullptr) pb = *reinterpret_cast<const Pack<W, VEC>*>(b + c);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int64_t row = row0 + r * RPB;
      if (row >= rows) continue;
      Pack<T, VEC> o;
#pragma unroll
      for (int k = 0; k < VEC; ++k) {
        A t = (widen(p[r][i].v[k]) - sum[r]) * sq[r];
        if (w != nullptr) t *= widen(pw.v[k]);
        if (b != nullptr) t += widen(pb.v[k]);
        o.v[k] = narrow<T>(t);
      }
      *reinterpret_cast<Pack<T, VEC>*>(y + row * cols + c) = o;
    }
  }
}

// partial [gridDim.x][2][cols]: this block's sums of g xh and g (null when neither gradient is wanted).
template <typename T, typename W, int VEC, int TPR, int VPT, int R>
__global__ void __launch_bounds__(kBlock<TPR>, kMinBlocks<TPR>)
    layer_norm_bwd_kernel(const T* __restrict__ g, int64_t ldg, const T* __restrict__ x, int64_t ldx,
                          const typename AccOf<T>::type* __restrict__ mean, const typename AccOf<T>::type* __restrict__ rstd,
                          const W* __restrict__ w, T* __restrict__ dx, typename AccOf<T>::type* __restrict__ partial,
                          int64_t rows, int cols) {
  using A = typename AccOf<T>::type;
  constexpr int THREADS = kBlock<TPR>, RPB = THREADS / TPR, E = VPT * VEC;
  __shared__ A scratch[2][2 * R][32];
  int turn = 0;
  __shared__ A fold[RPB > 1 ? THREADS * VEC : 1];
  const int lane = threadIdx.x % TPR, group = threadIdx.x / TPR;
  A dw[E], db[E];
#pragma unroll
  for (int i = 0; i < E; ++i) { dw[i] = 0; db[i] = 0; }
  const A inv_n = (A)1 / (A)cols;
  for (int64_t block0 = (int64_t)blockIdx.x * (RPB * R); block0 < rows; block0 += (int64_t)gridDim.x * (RPB * R)) {
    const int64_t row0 = block0 + group;
    Pack<T, VEC> pg[R][VPT], px[R][VPT];
    A mu[R], rs[R], s[2 * R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int64_t row = row0 + r * RPB;
      load_row<T, VEC, TPR, VPT>(pg[r], g, row, ldg, rows, cols, lane);
      load_row<T, VEC, TPR, VPT>(px[r], x, row, ldx, rows, cols, lane);
      mu[r] = row < rows ? mean[row] : (A)0;
      rs[r] = row < rows ? rstd[row] : (A)0;
      s[2 * r] = 0;
      s[2 * r + 1] = 0;
    }
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int c = (i * TPR + lane) * VEC;
      if (c >= cols) continue;
      Pack<W, VEC> pw;
      if (w != nullptr) pw = *reinterpret_cast<const Pack<W, VEC>*>(w + c);
#pragma unroll
      for (int r = 0; r < R; ++r) {
        if (row0 + r * RPB >= rows) continue;
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
          const A gv = widen(pg[r][i].v[k]), xh = (widen(px[r][i].v[k]) - mu[r]) * rs[r];
          dw[i * VEC + k] += gv * xh;
          db[i * VEC + k] += gv;
          const A gw = w != nullptr ? gv * widen(pw.v[k]) : gv;
          s[2 * r] += gw;
          s[2 * r + 1] += gw * xh;
        }
      }
    }
    row_sum<TPR>(s, scratch, turn);
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int c = (i * TPR + lane) * VEC;
      if (c >= cols) continue;
      Pack<W, VEC> pw;
      if (w != nullptr) pw = *reinterpret_cast<const Pack<W, VEC>*>(w + c);
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const int64_t row = row0 + r * RPB;
        if (row >= rows) continue;
        const A s1 = s[2 * r] * inv_n, s2 = s[2 * r + 1] * inv_n;
        Pack<T, VEC> o;
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
          const A gv = widen(pg[r][i].v[k]), xh = (widen(px[r][i].v[k]) - mu[r]) * rs[r];
          const A gw = w != nullptr ? gv * widen(pw.v[k]) : gv;
          o.v[k] = narrow<T>(rs[r] * (gw - s1 - xh * s2));
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

// Column sums of partial [blocks][2 cols], added in a fixed order: COLS columns per block, 1024 / COLS threads down each of
// them.  32 columns read whole cache lines (8192 column sums of 444 rows: 5 us against 15 us), 8 columns (a 32-byte sector) give
// narrow rows four times the blocks (256 of 592: 4 us against 7 us).
template <typename A, typename W, int COLS>
__global__ void __launch_bounds__(1024) layer_norm_fold_kernel(const A* __restrict__ partial, int blocks, int cols,
                                                               W* __restrict__ dw, W* __restrict__ db) {
  constexpr int DOWN = 1024 / COLS;
  __shared__ A tile[DOWN][COLS + 1];
  const int x = threadIdx.x % COLS, y = threadIdx.x / COLS, c = blockIdx.x * COLS + x;
  A s = 0;
  if (c < 2 * cols)
#pragma unroll 4
    for (int i = y; i < blocks; i += DOWN) s += partial[(int64_t)i * 2 * cols + c];
  tile[y][x] = s;
  for (int o = DOWN / 2; o > 0; o >>= 1) {
    __syncthreads();
    if (y < o) tile[y][x] += tile[y + o][x];
  }
  if (y == 0 && c < 2 * cols) {
    if (c < cols) { if (dw != nullptr) dw[c] = narrow<W>(tile[0][x]); }
    else if (db != nullptr) db[c - cols] = narrow<W>(tile[0][x]);
  }
}

constexpr int64_t kMaxCols = 8192;  // messages name it as text: the extension links its own iostreams, which cannot format numbers

struct LnArgs {
  const void *g, *x, *w, *b;
  void *y, *mean, *rstd, *partial, *dw, *db;
  int64_t ldg, ldx, rows;
  int cols, blocks;
  double eps;
  bool backward;
  cudaStream_t st;
};

template <typename T, typename W, int VEC, int TPR, int VPT, int R>
int forward(const LnArgs& a) {
  using A = typename AccOf<T>::type;
  constexpr int THREADS = kBlock<TPR>, RPB = THREADS / TPR;
  const int64_t blocks = (a.rows + RPB * R - 1) / (RPB * R);
  TORCH_CHECK(blocks < (int64_t)2147483647, "layer_norm: too many rows");
  layer_norm_fwd_kernel<T, W, VEC, TPR, VPT, R><<<(unsigned)blocks, THREADS, 0, a.st>>>(
      (const T*)a.x, a.ldx, (const W*)a.w, (const W*)a.b, (T*)a.y, (A*)a.mean, (A*)a.rstd, a.rows, a.cols, a.eps);
  return 0;
}

template <typename T, typename W, int VEC, int TPR, int VPT, int R>
int backward(const LnArgs& a, bool count_only) {
  using A = typename AccOf<T>::type;
  constexpr int THREADS = kBlock<TPR>, RPB = THREADS / TPR;
  if (count_only) {  // blocks of the persistent grid: what fits on the GPU at once, less when there are fewer rows
    int per_sm = 1, dev = 0, sms = 148;
    C10_CUDA_CHECK(cudaGetDevice(&dev));
    C10_CUDA_CHECK(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev));
    C10_CUDA_CHECK(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, layer_norm_bwd_kernel<T, W, VEC, TPR, VPT, R>, THREADS, 0));
    return (int)std::min<int64_t>((a.rows + RPB * R - 1) / (RPB * R), (int64_t)sms * std::max(per_sm, 1));
  }
  layer_norm_bwd_kernel<T, W, VEC, TPR, VPT, R><<<a.blocks, THREADS, 0, a.st>>>(
      (const T*)a.g, a.ldg, (const T*)a.x, a.ldx, (const A*)a.mean, (const A*)a.rstd, (const W*)a.w, (T*)a.y, (A*)a.partial,
      a.rows, a.cols);
  return a.blocks;
}

// Threads per row: a part of a warp for short rows (no idle lanes), the warp with up to four vectors a lane, then a block with
// two or four (a warp with 16 vectors a lane needs no barrier, but 16,384 x 4096 float16 forward took 71 us against 57 us).
template <typename T, typename W, int VEC>
int pick(const LnArgs& a, bool count_only) {
  const int nv = (a.cols + VEC - 1) / VEC;
  if constexpr (VEC == 1) {
    if (!a.backward) {
      if (nv <= 128) return forward<T, W, 1, 32, 4, 2>(a);
      if (nv <= 512) return forward<T, W, 1, 128, 4, 1>(a);
      if (nv <= 2048) return forward<T, W, 1, 512, 4, 1>(a);
      return forward<T, W, 1, 512, 16, 1>(a);
    }
    if (nv <= 128) return backward<T, W, 1, 32, 4, 1>(a, count_only);
    if (nv <= 512) return backward<T, W, 1, 128, 4, 1>(a, count_only);
    if (nv <= 2048) return backward<T, W, 1, 512, 4, 1>(a, count_only);
    return backward<T, W, 1, 512, 16, 1>(a, count_only);
  } else {
    if (!a.backward) {
      if (nv <= 8) return forward<T, W, VEC, 8, 1, 4>(a);
      if (nv <= 16) return forward<T, W, VEC, 16, 1, 4>(a);
      if (nv <= 32) return forward<T, W, VEC, 32, 1, 4>(a);
      if (nv <= 64) return forward<T, W, VEC, 32, 2, 2>(a);
      if (nv <= 128) return forward<T, W, VEC, 32, 4, 1>(a);
      if (nv <= 256) return forward<T, W, VEC, 128, 2, 1>(a);
      if (nv <= 512) return forward<T, W, VEC, 256, 2, 1>(a);
      if (nv <= 1024) return forward<T, W, VEC, 256, 4, 1>(a);
      return forward<T, W, VEC, 512, 16 / VEC, 1>(a);
    }
    if (nv <= 8) return backward<T, W, VEC, 8, 1, 2>(a, count_only);
    if (nv <= 16) return backward<T, W, VEC, 16, 1, 2>(a, count_only);
    if (nv <= 32) return backward<T, W, VEC, 32, 1, 2>(a, count_only);
    if (nv <= 64) return backward<T, W, VEC, 32, 2, 1>(a, count_only);
    if (nv <= 128) return backward<T, W, VEC, 32, 4, 1>(a, count_only);
    if (nv <= 256) return backward<T, W, VEC, 128, 2, 1>(a, count_only);
    if (nv <= 512) return backward<T, W, VEC, 256, 2, 1>(a, count_only);
    if (nv <= 1024) return backward<T, W, VEC, 512, 2, 1>(a, count_only);
    return backward<T, W, VEC, 512, 16 / VEC, 1>(a, count_only);
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

void check_types(at::ScalarType xt, at::ScalarType wt) {
  TORCH_CHECK((xt == at::kFloat || xt == at::kDouble || xt == at::kBFloat16 || xt == at::kHalf) && (wt == xt || (wt == at::kFloat && xt != at::kDouble)),
              "layer_norm: rows of type ", xt, " with weights of type ", wt, " are not supported");
}

int dispatch(const LnArgs& a, at::ScalarType xt, at::ScalarType wt, bool count_only) {
  if (xt == at::kFloat && wt == at::kFloat) return pick_vec<float, float>(a, count_only);
  if (xt == at::kDouble && wt == at::kDouble) return pick_vec<double, double>(a, count_only);
  if (xt == at::kBFloat16 && wt == at::kBFloat16) return pick_vec<__nv_bfloat16, __nv_bfloat16>(a, count_only);
  if (xt == at::kBFloat16 && wt == at::kFloat) return pick_vec<__nv_bfloat16, float>(a, count_only);
  if (xt == at::kHalf && wt == at::kHalf) return pick_vec<__half, __half>(a, count_only);
  return pick_vec<__half, float>(a, count_only);  // check_types has passed
}

// Any tensor as a matrix with contiguous rows: a view where the strides allow one.
Tensor as_rows(const Tensor& t, const char* name) {
  TORCH_CHECK(t.is_cuda() && t.dim() >= 1, "layer_norm: ", name, " must be a CUDA tensor with at least one axis");
  const int64_t cols = t.size(-1);
  TORCH_CHECK(cols >= 1 && cols <= kMaxCols, "layer_norm: row length must lie in 1..8192");
  Tensor r = t.dim() == 2 ? t : t.reshape({t.numel() / cols, cols});
  return r.stride(1) == 1 || cols == 1 || r.numel() == 0 ? r : r.contiguous();
}
c10::optional<Tensor> as_vector(const c10::optional<Tensor>& t, const Tensor& x, const char* name) {
  if (!t.has_value()) return t;
  TORCH_CHECK(t->device() == x.device() && t->dim() == 1 && t->size(0) == x.size(-1), "layer_norm: ", name,
              " must be a vector of the row length on the device of x");
  return t->is_contiguous() ? *t : t->contiguous();
}
void* ptr(const c10::optional<Tensor>& t) { return t.has_value() ? t->data_ptr() : nullptr; }

Tensor forward_pass(const Tensor& x, const c10::optional<Tensor>& weight, const c10::optional<Tensor>& bias, double eps, Tensor* mean,
                    Tensor* rstd) {
  c10::cuda::OptionalCUDAGuard guard;
  if (x.is_cuda()) guard.set_device(x.device());
  const Tensor rows = as_rows(x, "x");
  const auto w = as_vector(weight, x, "weight"), b = as_vector(bias, x, "bias");
  const at::ScalarType wt = w.has_value() ? w->scalar_type() : b.has_value() ? b->scalar_type() : x.scalar_type();
  TORCH_CHECK(!b.has_value() || b->scalar_type() == wt, "layer_norm: weight and bias must have one type");
  Tensor y = at::empty(x.sizes(), x.options());
  if (mean != nullptr) {
    auto so = x.options().dtype(x.scalar_type() == at::kDouble ? at::kDouble : at::kFloat);
    *mean = at::empty({rows.size(0)}, so);
    *rstd = at::empty({rows.size(0)}, so);
  }
  LnArgs a{};
  a.x = rows.data_ptr(); a.w = ptr(w); a.b = ptr(b); a.y = y.data_ptr();
  a.mean = mean != nullptr ? mean->data_ptr() : nullptr; a.rstd = mean != nullptr ? rstd->data_ptr() : nullptr;
  a.ldx = rows.stride(0); a.rows = rows.size(0); a.cols = (int)rows.size(1); a.eps = eps;
  a.st = at::cuda::getCurrentCUDAStream();
  check_types(x.scalar_type(), wt);
  if (a.rows == 0) return y;
  dispatch(a, x.scalar_type(), wt, false);
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  return y;
}

}  // namespace

Tensor layer_norm_apply(const Tensor& x, const c10::optional<Tensor>& weight, const c10::optional<Tensor>& bias, double eps) {
  return forward_pass(x, weight, bias, eps, nullptr, nullptr);
}

std::tuple<Tensor, Tensor, Tensor> layer_norm_fwd(const Tensor& x, const c10::optional<Tensor>& weight,
                                                  const c10::optional<Tensor>& bias, double eps) {
  Tensor mean, rstd;
  Tensor y = forward_pass(x, weight, bias, eps, &mean, &rstd);
  return {y, mean, rstd};
}

std::tuple<Tensor, Tensor, Tensor> layer_norm_bwd(const Tensor& grad, const Tensor& x, const Tensor& mean, const Tensor& rstd,
                                                  const c10::optional<Tensor>& weight, bool want_params,
                                                  c10::optional<at::ScalarType> param_type) {
  TORCH_CHECK(grad.sizes() == x.sizes() && grad.scalar_type() == x.scalar_type() && grad.device() == x.device(),
              "layer_norm: grad must match x");
  c10::cuda::OptionalCUDAGuard guard;
  if (x.is_cuda()) guard.set_device(x.device());
  const Tensor xr = as_rows(x, "x"), gr = as_rows(grad, "grad");
  const auto w = as_vector(weight, x, "weight");
  const at::ScalarType st = x.scalar_type() == at::kDouble ? at::kDouble : at::kFloat;
  for (const Tensor* s : {&mean, &rstd})
    TORCH_CHECK(s->device() == x.device() && s->dim() == 1 && s->is_contiguous() && s->size(0) == xr.size(0) && s->scalar_type() == st,
                "layer_norm: mean and rstd must be the forward pass's statistics");
  const at::ScalarType wt = w.has_value() ? w->scalar_type() : param_type.value_or(x.scalar_type());
  check_types(x.scalar_type(), wt);
  const int64_t cols = xr.size(1);
  Tensor dx = at::empty(x.sizes(), x.options());
  Tensor dw = at::empty({want_params ? cols : 0}, x.options().dtype(wt)), db = at::empty({want_params ? cols : 0}, x.options().dtype(wt));
  if (xr.size(0) == 0) return {dx, dw.zero_(), db.zero_()};
  LnArgs a{};
  a.backward = true;
  a.g = gr.data_ptr(); a.x = xr.data_ptr(); a.w = ptr(w); a.y = dx.data_ptr();
  a.mean = mean.data_ptr(); a.rstd = rstd.data_ptr();
  a.ldg = gr.stride(0); a.ldx = xr.stride(0); a.rows = xr.size(0); a.cols = (int)cols;
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
    auto fold = [&](auto acc, auto wv) {
      using A = decltype(acc);
      using W = decltype(wv);
      if (cols >= 1024)
        layer_norm_fold_kernel<A, W, 32><<<(unsigned)((2 * cols + 31) / 32), 1024, 0, a.st>>>((const A*)a.partial, a.blocks, (int)cols,
                                                                                             (W*)dw.data_ptr(), (W*)db.data_ptr());
      else
        layer_norm_fold_kernel<A, W, 8><<<(unsigned)((2 * cols + 7) / 8), 1024, 0, a.st>>>((const A*)a.partial, a.blocks, (int)cols,
                                                                                          (W*)dw.data_ptr(), (W*)db.data_ptr());
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

// Explicit kernels: tracing must not decompose them, their C++ would launch on tensors without memory.
TORCH_LIBRARY_FRAGMENT(nvalchemi, m) {
  m.def("layer_norm_apply(Tensor x, Tensor? weight, Tensor? bias, float eps) -> Tensor", torch::dispatch(c10::DispatchKey::CompositeExplicitAutograd, &nva::layer_norm_apply));
  m.def("layer_norm_fwd(Tensor x, Tensor? weight, Tensor? bias, float eps) -> (Tensor, Tensor, Tensor)", torch::dispatch(c10::DispatchKey::CompositeExplicitAutograd, &nva::layer_norm_fwd));
  m.def("layer_norm_bwd(Tensor grad, Tensor x, Tensor mean, Tensor rstd, Tensor? weight, bool want_params, ScalarType? param_type) -> (Tensor, Tensor, Tensor)", torch::dispatch(c10::DispatchKey::CompositeExplicitAutograd, &nva::layer_norm_bwd));
}
