// SPDX-License-Identifier: Apache-2.0
// Newton-Schulz orthogonalisation of a batch of matrices: from X = G / (|G|_F + eps), `steps` times
//     A = X X^T,   B = b A + c A A,   X <- a X + B X          (tall G: A = X^T X, X <- a X + X B),
// which drives every singular value towards 1 by an odd polynomial and leaves the singular vectors.  The result is bfloat16.
//
// Every product runs on the tensor cores with float16 operands and fp32 accumulators.  The entries are bounded by the
// spectral norm (at most about 1.2), so float16 with a power-of-two scale (X and A times 2^12, B times 2^11) keeps 11 bits of
// every entry that matters, three more than bfloat16.  Two choices keep its rounding from being amplified by the iteration,
// which multiplies small singular values by up to a each step:
//   * X itself is kept as a float16 value and a float16 remainder (22 bits) and a X is added from both; the products read the
//     first alone, so its rounding only enters through B X and A, where it is multiplied by the row and column spaces of X and
//     cannot feed empty directions;
//   * the diagonals of A and B are kept in fp32 and only the rest is rounded: A = D + R, A A = D D + D R + R D + R R, and
//     B X = diag(B) X + (B - diag(B)) X with both terms taken from the same float16 X, so that directions in which they
//     cancel stay empty.
// Error of the result before its rounding: 2e-4 to 1.4e-3 of its norm over Gaussian, noisy low-rank and low-rank matrices
// from 128 x 128 to 1024 x 1024 (bfloat16 operands: 0.4 to 2.3e-2); the rounding itself is 1.7e-3.  In matrices with a side of
// 128 or less fewer roundings average out (up to 3e-3 at 8 x 8), while the products cost little: there the remainder takes part
// in A (three products) and in B X (two), which brings the error under 1e-3.
//
// A and B are symmetric: where the GPU has no tile to spare only those on and below the diagonal are computed, each written
// twice.
//
// The diagonal of A sums squares, and the tensor core loses up to 1e-7 of such a sum with every instruction: past 65,536 terms (a
// third of that where the remainders take part) A is formed in parts that are added in fp32 (max_blocks in dense16.cuh).
//
// What bounds it: 4 x 1024 x 4096 bfloat16 takes 560 us: a step is 30 us for A (540 TFLOP/s of what has to be computed; 128-wide
// tiles, 144 of them), 16 us for B (one short product and its epilogue) and 53 us for the update (600 TFLOP/s; its epilogue reads
// and writes X, 270 MB a step in all).  Small problems are bound by latency: 1537 x 515 takes 187 us, 17 launches of 3 to 12 us.
#include "dense16.cuh"

namespace nva {
using at::Tensor;
namespace {
using namespace dense;

constexpr float kXScale = 4096.f, kBScale = 2048.f;  // powers of two: exact

// 32 columns of a symmetric tile: rows as they are and, for tiles below the diagonal, transposed (a warp's 32 lanes hold 32
// consecutive rows, so each column of theirs is one 64-byte run of the transposed row).
__device__ __forceinline__ void store_symmetric(uint4* stage, const float (&v)[32], __half* out, int64_t ld, int size, int row0, int n0,
                                                bool mirror) {
  const int row = row0 + (threadIdx.x & 31);
  uint4 o[4];
  pack32<__half>(v, o);
  store_piece<__half, 4>(stage, o, out + (int64_t)row0 * ld + n0, ld, size - row0, size - n0, true);
  if (mirror && row < size) {
#pragma unroll
    for (int j = 0; j < 32; ++j)
      if (n0 + j < size) out[(int64_t)(n0 + j) * ld + row] = __float2half_rn(v[j]);
  }
}

// NaN in a warp's part of a symmetric tile, its mirror image and its rows of the diagonal.
__device__ __forceinline__ void poison_symmetric(__half* out, float* diag, int64_t ld, int size, int row0, int n0, int cols, bool mirror) {
  fill_nan(out + (int64_t)row0 * ld + n0, ld, size - row0, size - n0, cols);
  if (mirror)
    for (int c = 0; c < cols; c += 32) fill_nan(out + (int64_t)(n0 + c) * ld + row0, ld, size - n0 - c, size - row0, 32);
  fill_nan(diag + row0, 1, size - row0, 1, 1);
}

// R = A without its diagonal (times 2^12), diag(A).
template <int BN>
struct EpiGram : NoPrefetch {
  static constexpr int kAcc = 1, kStride = BN;
  static constexpr bool kLate = false;
  struct Params { __half* r; float* diag; int64_t ld, stride; };
  static __device__ __forceinline__ void poison(const Params& p, const Tiles& t, const TileAt& at, int row0, int half) {
    poison_symmetric(p.r + at.batch * p.stride, p.diag + at.batch * (int64_t)t.M, p.ld, t.M, row0, at.n * BN + half * (BN / 2), BN / 2,
                     at.n < t.lower * at.m);
  }
  static __device__ __forceinline__ void run(const Params& p, const Tiles& t, const TileAt& at, uint32_t tm, int row0, int half,
                                             uint4* stage, Pre&) {
    __half* out = p.r + at.batch * p.stride;
    const int row = row0 + (threadIdx.x & 31);
#pragma unroll 1
    for (int cb = 0; cb < BN / 64; ++cb) {
      const int c = half * (BN / 2) + cb * 32, n0 = at.n * BN + c;
      float v[32], dg = 0.f;
      tmem_ld32(tm + c, v);
#pragma unroll
      for (int j = 0; j < 32; ++j) {
        v[j] *= 1.f / kXScale;  // accumulated 2^24 A
        const bool on = row == n0 + j;
        dg = on ? v[j] : dg;
        v[j] = on ? 0.f : v[j];
      }
      if (row >= n0 && row < n0 + 32 && row < t.M) p.diag[at.batch * (int64_t)t.M + row] = dg * (1.f / kXScale);
      store_symmetric(stage, v, out, p.ld, t.M, row0, n0, at.n < t.lower * at.m);
    }
  }
};

// B = b A + c A A, split the same way.
template <int BN>
struct EpiPoly {
  static constexpr int kAcc = 1, kStride = BN;
  static constexpr bool kLate = false;
  struct Params { const __half* r; const float* diag; __half* bo; float* bdiag; int64_t ld, stride; float b, c; };
  struct Pre { uint4 raw[4]; float dl; };  // 32 columns of R (rows are padded to 8), and of the diagonal
  static __device__ __forceinline__ void poison(const Params& p, const Tiles& t, const TileAt& at, int row0, int half) {
    poison_symmetric(p.bo + at.batch * p.stride, p.bdiag + at.batch * (int64_t)t.M, p.ld, t.M, row0, at.n * BN + half * (BN / 2), BN / 2,
                     at.n < t.lower * at.m);
  }
  static __device__ __forceinline__ void fetch(const Params& p, const Tiles& t, const TileAt& at, int row0, int n0, Pre& pre) {
    const int lane = threadIdx.x & 31;
    fetch_piece<__half, 4>(pre.raw, p.r + at.batch * p.stride + (int64_t)row0 * p.ld + n0, p.ld, t.M - row0, t.M - n0);
    pre.dl = n0 + lane < t.M ? p.diag[at.batch * (int64_t)t.M + n0 + lane] : 0.f;
  }
  static __device__ __forceinline__ void prefetch(const Params& p, const Tiles& t, const TileAt& at, int row0, int half, Pre& pre) {
    fetch(p, t, at, row0, at.n * BN + half * (BN / 2), pre);
  }
  static __device__ __forceinline__ void run(const Params& p, const Tiles& t, const TileAt& at, uint32_t tm, int row0, int half,
                                             uint4* stage, Pre& pre) {
    const int row = row0 + (threadIdx.x & 31);
    const float di = row < t.M ? p.diag[at.batch * (int64_t)t.M + row] : 0.f;
#pragma unroll 1
    for (int cb = 0; cb < BN / 64; ++cb) {
      const int c = half * (BN / 2) + cb * 32, n0 = at.n * BN + c;
      turn_piece<4>(stage, pre.raw);
      uint4 raw[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) raw[q] = pre.raw[q];
      const float dl = pre.dl;
      if (cb + 1 < BN / 64) fetch(p, t, at, row0, n0 + 32, pre);
      float v[32], dg = 0.f;
      tmem_ld32(tm + c, v);
#pragma unroll
      for (int j = 0; j < 32; ++j) {
        const float aa = v[j] * (1.f / (kXScale * kXScale));
        const float rij = __half2float(reinterpret_cast<const __half*>(raw)[j]) * (1.f / kXScale);
        const float dj = __shfl_sync(0xffffffffu, dl, j);
        const bool on = row == n0 + j;
        dg = on ? aa : dg;
        v[j] = on ? 0.f : (p.b * rij + p.c * ((di + dj) * rij + aa)) * kBScale;
      }
      if (row >= n0 && row < n0 + 32 && row < t.M) p.bdiag[at.batch * (int64_t)t.M + row] = p.b * di + p.c * (di * di + dg);
      store_symmetric(stage, v, p.bo + at.batch * p.stride, p.ld, t.M, row0, n0, at.n < t.lower * at.m);
    }
  }
};

// X <- a X + diag(B) X + (B - diag(B)) X, or the bfloat16 result of the last step.
template <int BN>
struct EpiUpdate {
  static constexpr int kAcc = 1, kStride = BN;
  static constexpr bool kLate = false;
  struct Params {
    const __half* x; const float* bdiag;   // X: high parts, remainders `plane` further
    __half* x_out; __nv_bfloat16* out;     // out != null: last step
    int64_t ld, stride, plane;             // of x and x_out
    int64_t out_stride;
    int tall, short_side, two;             // two: the products read the remainders as well
    float a;
  };
  struct Pre { uint4 h[4], l[4]; float bl; };  // 32 columns of X (rows are padded to 8), diag(B)
  static __device__ __forceinline__ void poison(const Params& p, const Tiles& t, const TileAt& at, int row0, int half) {
    const int n0 = at.n * BN + half * (BN / 2);
    if (p.out != nullptr)
      fill_nan(p.out + at.batch * p.out_stride + (int64_t)row0 * t.N + n0, t.N, t.M - row0, t.N - n0, BN / 2);
    else  // the remainders need none: what reads them reads the values too
      fill_nan(p.x_out + at.batch * p.stride + (int64_t)row0 * p.ld + n0, p.ld, t.M - row0, t.N - n0, BN / 2);
  }
  static __device__ __forceinline__ void fetch(const Params& p, const Tiles& t, const TileAt& at, int row0, int n0, Pre& pre) {
    const int lane = threadIdx.x & 31;
    const int64_t off = at.batch * p.stride + (int64_t)row0 * p.ld + n0;
    fetch_piece<__half, 4>(pre.h, p.x + off, p.ld, t.M - row0, t.N - n0);
    fetch_piece<__half, 4>(pre.l, p.x + p.plane + off, p.ld, t.M - row0, t.N - n0);
    pre.bl = p.tall && n0 + lane < t.N ? p.bdiag[at.batch * (int64_t)p.short_side + n0 + lane] : 0.f;
  }
  static __device__ __forceinline__ void prefetch(const Params& p, const Tiles& t, const TileAt& at, int row0, int half, Pre& pre) {
    fetch(p, t, at, row0, at.n * BN + half * (BN / 2), pre);
  }
  static __device__ __forceinline__ void run(const Params& p, const Tiles& t, const TileAt& at, uint32_t tm, int row0, int half,
                                             uint4* stage, Pre& pre) {
    const int row = row0 + (threadIdx.x & 31);
    const float bi = !p.tall && row < t.M ? p.bdiag[at.batch * (int64_t)p.short_side + row] : 0.f;
    const float two = p.two ? 1.f : 0.f;
    const int64_t base = at.batch * p.stride;
#pragma unroll 1
    for (int cb = 0; cb < BN / 64; ++cb) {
      const int c = half * (BN / 2) + cb * 32, n0 = at.n * BN + c;
      if (n0 >= t.N) break;
      uint4 h4[4], l4[4];
      turn_piece<4>(stage, pre.h);
      turn_piece<4>(stage, pre.l);
#pragma unroll
      for (int q = 0; q < 4; ++q) { h4[q] = pre.h[q]; l4[q] = pre.l[q]; }
      const float bl = pre.bl;
      if (cb + 1 < BN / 64) fetch(p, t, at, row0, n0 + 32, pre);
      float v[32];
      tmem_ld32(tm + c, v);
#pragma unroll
      for (int j = 0; j < 32; ++j) {  // 2^12 X
        const float h = __half2float(reinterpret_cast<const __half*>(h4)[j]), l = __half2float(reinterpret_cast<const __half*>(l4)[j]);
        const float b = p.tall ? __shfl_sync(0xffffffffu, bl, j) : bi;
        v[j] = p.a * (h + l) + b * (h + two * l) + v[j] * (1.f / kBScale);  // b times the X that the product read
      }
      if (p.out != nullptr) {
#pragma unroll
        for (int j = 0; j < 32; ++j) v[j] *= 1.f / kXScale;
        uint4 o[4];
        pack32<__nv_bfloat16>(v, o);
        __nv_bfloat16* dst = p.out + at.batch * p.out_stride;
        store_piece<__nv_bfloat16, 4>(stage, o, dst + (int64_t)row0 * t.N + n0, t.N, t.M - row0, t.N - n0,
                                      t.N % 8 == 0 && (reinterpret_cast<uintptr_t>(dst) & 15) == 0);
      } else {
        uint4 o[4];
        pack32<__half>(v, o);
        __half* dst = p.x_out + base + (int64_t)row0 * p.ld + n0;
        store_piece<__half, 4>(stage, o, dst, p.ld, t.M - row0, t.N - n0, true);
#pragma unroll
        for (int j = 0; j < 32; ++j) v[j] -= __half2float(__float2half_rn(v[j]));
        pack32<__half>(v, o);
        store_piece<__half, 4>(stage, o, dst + p.plane, p.ld, t.M - row0, t.N - n0, true);
      }
    }
  }
};

// 2^12 / (|G| + eps) from the sum of squares; a zero matrix stays zero without eps too.
__device__ __forceinline__ double scale_of(double squares, double eps) {
  const double norm = sqrt(squares) + eps;
  return norm == 0.0 ? 0.0 : (double)kXScale / norm;
}

// Eight elements at a time where G's rows allow 16-byte accesses (8 | n, aligned), else one by one.
template <typename T>
__device__ __forceinline__ void load8(const T* p, bool vec, int left, double (&v)[8]) {
  if (vec) {
    uint4 raw[sizeof(T) / 2];
#pragma unroll
    for (int k = 0; k < (int)sizeof(T) / 2; ++k) raw[k] = reinterpret_cast<const uint4*>(p)[k];
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = (double)widen(reinterpret_cast<const T*>(raw)[k]);
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = k < left ? (double)widen(p[k]) : 0.0;
  }
}

// Sums of squares of G in float64 (no gradient is too small or too large for them): one partial per block.
template <typename T>
__global__ void __launch_bounds__(256) ns_norm_kernel(const T* __restrict__ g, int64_t count, bool vec, double* __restrict__ partial) {
  chain_wait();
  const T* src = g + blockIdx.y * count;
  double s = 0.0;
  for (int64_t i = (blockIdx.x * (int64_t)blockDim.x + threadIdx.x) * 8; i < count; i += (int64_t)gridDim.x * blockDim.x * 8) {
    double v[8];
    load8(src + i, vec, (int)min((int64_t)8, count - i), v);
#pragma unroll
    for (int k = 0; k < 8; ++k) s += v[k] * v[k];
  }
  __shared__ double part[8];
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < 8; ++i) s += part[i];
    partial[blockIdx.y * gridDim.x + blockIdx.x] = s;
  }
}

// X = G / (|G| + eps) as float16 values and remainders, times 2^12, rows padded to a multiple of 8.
template <typename T>
__global__ void __launch_bounds__(256) ns_init_kernel(const T* __restrict__ g, int rows, int cols, int ld, bool vec,
                                                      const double* __restrict__ partial, int parts, double eps, __half* __restrict__ x,
                                                      int64_t plane) {
  __shared__ double scale;
  chain_wait();
  if (threadIdx.x < 32) {
    double s = 0.0;
    for (int i = threadIdx.x; i < parts; i += 32) s += partial[blockIdx.y * parts + i];
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (threadIdx.x == 0) scale = scale_of(s, eps);
  }
  __syncthreads();
  const double k = scale;
  const T* src = g + blockIdx.y * (int64_t)rows * cols;
  __half* dst = x + blockIdx.y * (int64_t)rows * ld;
  const uint32_t groups = (uint32_t)ld / 8;
  for (int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; i < (int64_t)rows * groups; i += (int64_t)gridDim.x * blockDim.x) {
    const int64_t r = i / groups;
    const int c = (int)(i - r * groups) * 8;
    double v[8];
    load8(src + r * cols + c, vec, cols - c, v);
    float f[8];
    uint4 h, l;
    __half* const hp = reinterpret_cast<__half*>(&h);
    __half* const lp = reinterpret_cast<__half*>(&l);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      f[j] = (float)(v[j] * k);
      hp[j] = __float2half_rn(f[j]);
      lp[j] = __float2half_rn(f[j] - __half2float(hp[j]));
    }
    *reinterpret_cast<uint4*>(dst + r * ld + c) = h;
    *reinterpret_cast<uint4*>(dst + plane + r * ld + c) = l;
  }
}

// ---- small matrices: short side up to 128, long side up to 256 -------------------------------------------------------
// One CTA runs the whole iteration of a matrix and nothing leaves the SM: X (high and low float16 parts, [short][long] in
// chunks of 64 columns, 128 swizzled bytes a row) is the operand of both products, K-major in X X^T and MN-major in B X, so the
// same bytes serve both; A and B share one 128 x 128 buffer.  A thread holds one row and half of the columns of every
// accumulator; A stays in its registers in fp32 until B is formed.  X is kept as high + low part (22 bits), which for a
// bfloat16 result is as good as fp32.  What bounds it is the chain of 15 products with an epilogue and two block barriers
// between each; nothing of an epilogue may wait for its neighbour (conditions around shared-memory loads made B's 9400 clocks of
// 19,000 a step).  24 matrices of 128 x 128 took 183 us as 17 launches.
constexpr int kSmallThreads = 256, kSmallChunk = 128 * 128;  // bytes of 128 rows x 64 columns

__device__ __forceinline__ uint32_t small_at(int row, int col) {  // byte offset of an element in a chunked, swizzled plane
  return (uint32_t)((col >> 6) * kSmallChunk + row * 128 + ((((col >> 3) & 7) ^ (row & 7)) << 4) + (col & 7) * 2);
}

template <typename T>
__global__ void __launch_bounds__(kSmallThreads)
    ns_small_kernel(const T* __restrict__ g, int m, int n, int steps, float ca, float cb, float cc, double eps, __nv_bfloat16* __restrict__ out) {
  extern __shared__ uint8_t smem_raw[];
  __shared__ double part[8];
  __shared__ float diag[128];
  __shared__ uint64_t bar_store;
  __shared__ uint32_t tmem_slot;
  const bool tall = m > n;
  const int r = tall ? n : m, len = tall ? m : n, chunks = (len + 63) / 64, count = m * n;
  const int kr = (r + 15) / 16, kl = (len + 15) / 16;  // 16-wide blocks of the two axes
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* const sm = smem_raw + (base - smem_u32(smem_raw));
  const uint32_t plane = (uint32_t)chunks * kSmallChunk;
  uint8_t *const xh = sm, *const xl = sm + plane, *const rb = sm + 2 * plane;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, q = warp & 3, half = warp >> 2, row = q * 32 + lane;
  const uint32_t bar = smem_u32(&bar_store), cols = len <= 128 ? 256u : 512u;
  const T* src = g + blockIdx.x * (int64_t)count;
  int* const err = &error_word;

  if (threadIdx.x == 0) {
    mbar_init(bar, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)), "r"(cols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  double s = 0.0;
#pragma unroll 4
  for (int i = threadIdx.x; i < count; i += kSmallThreads) {
    const double v = (double)widen(src[i]);
    s += v * v;
  }
  for (uint32_t i = threadIdx.x; i < (2 * plane + 2 * kSmallChunk) / 16; i += kSmallThreads) reinterpret_cast<uint4*>(sm)[i] = make_uint4(0, 0, 0, 0);
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if (lane == 0) part[warp] = s;
  __syncthreads();
  s = 0.0;
  for (int i = 0; i < 8; ++i) s += part[i];
  // 2^12 / (|G| + eps) as a mantissa and two powers of two, so that no factor leaves the fp32 range
  int e;
  const float mant = (float)frexp(scale_of(s, eps), &e);
  const float p1 = scalbnf(1.f, max(-126, min(127, e / 2))), p2 = scalbnf(1.f, max(-126, min(127, e - e / 2)));
  const uint32_t magic = n > 1 ? (uint32_t)((0x100000000ull + n - 1) / n) : 0;  // i / n = umulhi(i, magic) for i < 2^16, n <= 256
  auto place = [&](uint32_t i) {
    const int gr = n > 1 ? (int)__umulhi(i, magic) : (int)i, gc = (int)i - gr * n;
    return tall ? small_at(gc, gr) : small_at(gr, gc);
  };
#pragma unroll 4
  for (int i = threadIdx.x; i < count; i += kSmallThreads) {
    const uint32_t at = place(i);
    const float v = widen(src[i]) * p1 * mant * p2;
    const __half h = __float2half_rn(v);
    *reinterpret_cast<__half*>(xh + at) = h;
    *reinterpret_cast<__half*>(xl + at) = __float2half_rn(v - __half2float(h));
  }
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = tmem_slot, t_gram = tmem, t_upd = tmem + 128, lanes = (uint32_t)(q * 32) << 16;
  const uint32_t a_xh = base, a_xl = base + plane, a_rb = base + 2 * plane;
  uint32_t phase = 0;
  bool ok = true;
  // Everyone waits for the products issued last; all leave together when the wait ran out.
  auto done = [&]() {
    ok = mbar_wait(bar, phase, err, 21);
    phase ^= 1;
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    return __syncthreads_and(ok) != 0;
  };
  // What the epilogue wrote to shared memory is visible to the next products.
  auto publish = [&]() {
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  };
  // 32 columns of this thread's row of a plane, from column c0 (a multiple of 32)
  auto put32 = [&](uint8_t* p, int c0, const float (&v)[32]) {
    uint4 o[4];
    pack32<__half>(v, o);
#pragma unroll
    for (int k = 0; k < 4; ++k) *reinterpret_cast<uint4*>(p + small_at(row, c0 + 8 * k)) = o[k];
  };
  const uint32_t id_sq = idesc16(false, false, false, 16 * kr, BM), id_up = idesc16(false, false, true, 16 * kl, BM);

  for (int step = 0; step < steps; ++step) {
    if (threadIdx.x == 0) {  // A: low . high, high . low, high . high
      for (int p = 0; p < 3; ++p)
        for (int k = 0; k < kl; ++k) {
          const uint32_t off = (uint32_t)(k >> 2) * kSmallChunk + (k & 3) * 32;
          mma16<false>(t_gram, desc16((p == 0 ? a_xl : a_xh) + off, false), desc16((p == 1 ? a_xl : a_xh) + off, false), id_sq, p + k > 0 ? 1u : 0u);
        }
      umma_commit(bar);
    }
    if (!done()) break;
    float a0[32], a1[32];  // this thread's 64 columns of A
    tmem_ld32(t_gram + lanes + half * 64, a0);
    tmem_ld32(t_gram + lanes + half * 64 + 32, a1);
    const int c0 = half * 64;
    auto strip = [&](float (&v)[32], int base_col, float k, float& d) {  // takes the diagonal out
#pragma unroll
      for (int j = 0; j < 32; ++j) {
        v[j] = (base_col + j < r && row < r) ? v[j] * k : 0.f;
        const bool on = row == base_col + j;
        d = on ? v[j] : d;
        v[j] = on ? 0.f : v[j];
      }
    };
    float dg = 0.f;
    strip(a0, c0, 1.f / kXScale, dg);  // 2^12 A
    strip(a1, c0 + 32, 1.f / kXScale, dg);
    put32(rb, c0, a0);
    put32(rb, c0 + 32, a1);
    const bool mine = row >= c0 && row < c0 + 64;
    if (mine) diag[row] = dg * (1.f / kXScale);
    publish();
    if (threadIdx.x == 0) {  // R R
      for (int k = 0; k < kr; ++k) {
        const uint32_t off = (uint32_t)(k >> 2) * kSmallChunk + (k & 3) * 32;
        mma16<false>(t_gram, desc16(a_rb + off, false), desc16(a_rb + off, false), id_sq, k > 0 ? 1u : 0u);
      }
      umma_commit(bar);
    }
    if (!done()) break;
    const float di = diag[row];
    float aad = 0.f;  // the diagonal of R R
    auto poly = [&](float (&rv)[32], int base_col) {
      float v[32];
      const float dl = diag[base_col + lane];
      tmem_ld32(t_gram + lanes + base_col, v);
#pragma unroll
      for (int j = 0; j < 32; ++j) {
        const float aa = v[j] * (1.f / (kXScale * kXScale)), rij = rv[j] * (1.f / kXScale);
        const float b = cb * rij + cc * ((di + __shfl_sync(0xffffffffu, dl, j)) * rij + aa);
        const bool on = row == base_col + j;
        aad = on ? aa : aad;
        rv[j] = on || base_col + j >= r ? 0.f : b * kBScale;  // columns past r hold nothing; rows past r are zero by themselves
      }
    };
    poly(a0, c0);
    poly(a1, c0 + 32);
    __syncthreads();  // R and the diagonal of A have been read
    put32(rb, c0, a0);
    put32(rb, c0 + 32, a1);
    if (mine) diag[row] = cb * di + cc * (di * di + aad);
    publish();
    if (threadIdx.x == 0) {  // B X: low part, high part
      for (int p = 0; p < 2; ++p)
        for (int k = 0; k < kr; ++k)
          mma16<false>(t_upd, desc16(a_rb + (uint32_t)(k >> 2) * kSmallChunk + (k & 3) * 32, false),
                       desc16((p == 0 ? a_xl : a_xh) + (uint32_t)k * 2048, true, kSmallChunk), id_up, p + k > 0 ? 1u : 0u);
      umma_commit(bar);
    }
    if (!done()) break;
    const float bi = diag[row];
    const bool last = step + 1 == steps;
    for (int c = half * 32; c < 16 * kl; c += 64) {
      float v[32];
      tmem_ld32(t_upd + lanes + c, v);  // columns past 16 * kl hold nothing and are not stored
      uint4 h4[4], l4[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        h4[k] = *reinterpret_cast<const uint4*>(xh + small_at(row, c + 8 * k));
        l4[k] = *reinterpret_cast<const uint4*>(xl + small_at(row, c + 8 * k));
      }
#pragma unroll
      for (int j = 0; j < 32; ++j) {
        const float x = __half2float(reinterpret_cast<const __half*>(h4)[j]) + __half2float(reinterpret_cast<const __half*>(l4)[j]);
        const float y = (ca + bi) * x + v[j] * (1.f / kBScale);  // 2^12 X
        v[j] = row < r && c + j < len ? y : 0.f;
      }
      if (last) {
        uint4 o[4];
#pragma unroll
        for (int j = 0; j < 32; ++j) v[j] *= 1.f / kXScale;
        pack32<__nv_bfloat16>(v, o);
#pragma unroll
        for (int k = 0; k < 4; ++k) *reinterpret_cast<uint4*>(xh + small_at(row, c + 8 * k)) = o[k];
      } else {
        put32(xh, c, v);
#pragma unroll
        for (int j = 0; j < 32; ++j) v[j] -= __half2float(__float2half_rn(v[j]));
        put32(xl, c, v);
      }
    }
    publish();
  }
  __nv_bfloat16* dst = out + blockIdx.x * (int64_t)count;
  if (__syncthreads_and(ok)) {
#pragma unroll 4
    for (int i = threadIdx.x; i < count; i += kSmallThreads) dst[i] = *reinterpret_cast<const __nv_bfloat16*>(xh + place(i));
  } else {  // a wait ran out: nothing finite that was not computed
    for (int i = threadIdx.x; i < count; i += kSmallThreads) dst[i] = __ushort_as_bfloat16(0x7fc0);
  }
  __syncthreads();
  if (warp == 0) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(cols) : "memory");
}

template <typename T>
void run_small(const Tensor& g, int64_t steps, double a, double b, double c, double eps, Tensor& out, cudaStream_t st) {
  const int m = (int)g.size(1), n = (int)g.size(2), len = std::max(m, n);
  const int smem = 1024 + (2 * ((len + 63) / 64) + 2) * kSmallChunk;
  C10_CUDA_CHECK(cudaFuncSetAttribute(ns_small_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
  ns_small_kernel<T><<<(unsigned)g.size(0), kSmallThreads, smem, st>>>((const T*)g.data_ptr(), m, n, (int)steps, (float)a, (float)b, (float)c,
                                                                       eps, (__nv_bfloat16*)out.data_ptr());
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}

// R and the diagonal of A from a [batch][r][r], the sums of 2^24 A (matrices whose long side is formed in parts).
__global__ void __launch_bounds__(256) ns_gram_kernel(const float* __restrict__ a, int64_t batch, int r, int ld, __half* __restrict__ out,
                                                      float* __restrict__ diag) {
  chain_wait();
  const int64_t total = batch * r * r;
  for (int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; i < total; i += (int64_t)gridDim.x * blockDim.x) {
    const int64_t row = i / r;  // of the batch's rows
    const int c = (int)(i - row * r);
    const float v = a[i] * (1.f / kXScale);
    const bool on = row % r == c;
    out[row * ld + c] = __float2half_rn(on ? 0.f : v);
    if (on) diag[row] = v * (1.f / kXScale);
  }
}

// Adds a segment: planes za, zb of batch-many matrices each.
void add_segment(Tiles& t, int a, bool a_mn, int b, bool b_mn, int64_t K, int n, int za = 0, int zb = 0) {
  Seg& s = t.seg[t.n_seg++];
  s = Seg{};
  s.a = (int8_t)a; s.b = s.b2 = (int8_t)b;
  s.a_mn = a_mn; s.b_mn = b_mn;
  s.spread = 1;
  s.n = (int16_t)n;
  s.za = za; s.zb = zb;
  s.za_step = s.zb_step = 1;
  s.nk = (int)((K + BK - 1) / BK);
  s.b2_off = n / 2;
  s.idesc = idesc16(false, a_mn, b_mn, n, BM);
  t.main_nk[0] = s.nk;
}

}  // namespace

// g [batch][m][n] contiguous -> bfloat16 of the same shape.
Tensor newton_schulz(const Tensor& g, int64_t steps, double a, double b, double c, double eps) {
  TORCH_CHECK(g.is_cuda() && g.dim() == 3 && g.is_contiguous(), "newton_schulz: a contiguous CUDA tensor [batch, m, n]");
  TORCH_CHECK(g.scalar_type() == at::kFloat || g.scalar_type() == at::kHalf || g.scalar_type() == at::kBFloat16,
              "newton_schulz: float32, float16 or bfloat16");
  TORCH_CHECK(steps >= 1, "newton_schulz: at least one step");
  c10::cuda::CUDAGuard guard(g.device());
  auto st = at::cuda::getCurrentCUDAStream();
  const int64_t batch = g.size(0), m = g.size(1), n = g.size(2);
  Tensor out = at::empty({batch, m, n}, g.options().dtype(at::kBFloat16));
  if (out.numel() == 0) return out;
  if (std::min(m, n) <= 128 && std::max(m, n) <= 256 && batch < (1ll << 31)) {
    if (g.scalar_type() == at::kFloat) run_small<float>(g, steps, a, b, c, eps, out, st);
    else if (g.scalar_type() == at::kHalf) run_small<__half>(g, steps, a, b, c, eps, out, st);
    else run_small<__nv_bfloat16>(g, steps, a, b, c, eps, out, st);
    return out;
  }
  TORCH_CHECK(batch <= 65535 && m < (1 << 30) && n < (1 << 30), "newton_schulz: sizes out of range");
  const bool tall = m > n;
  const int64_t r = std::min(m, n), ld = (n + 7) / 8 * 8, rld = (r + 7) / 8 * 8;
  const int parts = (int)std::max<int64_t>(1, std::min<int64_t>({(m * n + 4095) / 4096, 1024, std::max<int64_t>(1, 8 * sm_count() / batch)}));
  const bool two = r <= 128;
  const int64_t plane = batch * m * ld;
  auto opt = [&](at::ScalarType t) { return g.options().dtype(t); };
  Tensor partial = at::empty({batch, parts}, opt(at::kDouble));
  Tensor x = at::empty({2, 2, batch, m, ld}, opt(at::kHalf));  // two iterates of [high, remainder]
  Tensor ra = at::empty({2, batch, r, rld}, opt(at::kHalf)), diag = at::empty({2, batch, r}, opt(at::kFloat));
  __half *x0 = (__half*)x.data_ptr(), *rp = (__half*)ra.data_ptr(), *bp = rp + batch * r * rld;
  float *ad = diag.data_ptr<float>(), *bd = ad + batch * r;
  auto prep = [&](auto v) {
    using T = decltype(v);
    const T* p = (const T*)g.data_ptr();
    const bool vec = n % 8 == 0 && (reinterpret_cast<uintptr_t>(p) & 15) == 0;
    launch_chained(ns_norm_kernel<T>, dim3(parts, batch), 256, st, p, m * n, vec, partial.data_ptr<double>());
    launch_chained(ns_init_kernel<T>, dim3(parts, batch), 256, st, p, (int)m, (int)n, (int)ld, vec, partial.data_ptr<double>(), parts, eps, x0,
                   plane);
  };
  if (g.scalar_type() == at::kFloat) prep(float{});
  else if (g.scalar_type() == at::kHalf) prep(__half{});
  else prep(__nv_bfloat16{});
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  auto stored_x = [&](int which) { return Stored{x0 + which * 2 * plane, n, m, ld, 2 * batch, m * ld}; };
  const Stored sr{rp, r, r, rld, batch, r * rld}, sb{bp, r, r, rld, batch, r * rld};
  const TileShape gram = pick_tile(r, r, (two ? 3 : 1) * std::max(m, n), batch, true), poly = pick_tile(r, r, r, batch, true),
                  upd = pick_tile(m, n, (two ? 2 : 1) * r, batch, false);
  auto with = [](int bn, auto f) {
    if (bn == 256) f(std::integral_constant<int, 256>{});
    else if (bn == 128) f(std::integral_constant<int, 128>{});
    else f(std::integral_constant<int, 64>{});
  };
  for (int64_t i = 0; i < steps; ++i) {
    const int cur = (int)(i & 1);
    with(gram.bn, [&](auto tag) {
      constexpr int BN = decltype(tag)::value;
      Maps maps;
      Tiles t{};
      put_map(maps, 0, stored_x(cur));
      for (int k = two ? 0 : 2; k < 3; ++k)  // remainder . high, high . remainder, high . high
        add_segment(t, 0, tall, 0, tall, tall ? m : n, BN, k == 0 ? (int)batch : 0, k == 1 ? (int)batch : 0);
      const int load = t.main_nk[0] * t.n_seg, most = max_blocks(at::kBFloat16);  // of the diagonal's sums, all of one sign
      if (load > most) {
        Tensor sums = at::empty({batch, r, r}, opt(at::kFloat));
        split_product<float, BN, 1>(maps, t, r, r, batch, (load + most - 1) / most, gram.pair, sums.data_ptr<float>(), sums.options(), st);
        launch_chained(ns_gram_kernel, dim3((unsigned)std::min<int64_t>((batch * r * r + 255) / 256, 148 * 8)), 256, st, sums.data_ptr<float>(),
                       batch, (int)r, (int)rld, rp, ad);
        return;
      }
      set_tiles(t, r, r, BN, batch, 1, gram.lower, gram.pair);
      run_dense<BN, EpiGram<BN>>(maps, t, {rp, ad, rld, r * rld}, st);
    });
    with(poly.bn, [&](auto tag) {
      constexpr int BN = decltype(tag)::value;
      Maps maps;
      Tiles t{};
      put_map(maps, 0, sr);
      add_segment(t, 0, false, 0, false, r, BN);
      set_tiles(t, r, r, BN, batch, 1, poly.lower, poly.pair);
      run_dense<BN, EpiPoly<BN>>(maps, t, {rp, ad, bp, bd, rld, r * rld, (float)b, (float)c}, st);
    });
    with(upd.bn, [&](auto tag) {
      constexpr int BN = decltype(tag)::value;
      Maps maps;
      Tiles t{};
      put_map(maps, 0, tall ? stored_x(cur) : sb);
      put_map(maps, 1, tall ? sb : stored_x(cur));
      for (int k = 0; k < (two ? 2 : 1); ++k)
        add_segment(t, 0, false, 1, !tall, r, BN, tall ? k * (int)batch : 0, tall ? 0 : k * (int)batch);
      set_tiles(t, m, n, BN, batch, 1, false, upd.pair);
      run_dense<BN, EpiUpdate<BN>>(maps, t,
                                   {x0 + cur * 2 * plane, bd, x0 + (1 - cur) * 2 * plane,
                                    i + 1 == steps ? (__nv_bfloat16*)out.data_ptr() : nullptr, ld, m * ld, plane, m * n, tall ? 1 : 0, (int)r,
                                    two ? 1 : 0, (float)a},
                                   st);
    });
  }
  return out;
}

int64_t newton_schulz_error_status(const Tensor& like) { return dense::take_error(like); }

}  // namespace nva

// Explicit kernels: tracing must not decompose them, their C++ would launch on tensors without memory.
TORCH_LIBRARY_FRAGMENT(nvalchemi, m) {
  m.def("newton_schulz(Tensor g, int steps, float a, float b, float c, float eps) -> Tensor", torch::dispatch(c10::DispatchKey::CompositeExplicitAutograd, &nva::newton_schulz));
  m.def("newton_schulz_error_status(Tensor like) -> int", torch::dispatch(c10::DispatchKey::CompositeExplicitAutograd, &nva::newton_schulz_error_status));
}
