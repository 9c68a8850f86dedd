// SPDX-License-Identifier: Apache-2.0
// Newton-Schulz orthogonalisation of a batch of matrices: from X = G / (|G|_F + eps), `steps` times
//     A = X X^T,   B = b A + c A A,   X <- a X + B X          (tall G: A = X^T X, X <- a X + X B),
// which drives every singular value towards 1 by an odd polynomial and leaves the singular vectors.  The result is bfloat16.
//
// Every product runs on the tensor cores with float16 operands and fp32 accumulators.  The entries are bounded by the
// spectral norm (at most about 1.2), so float16 with a power-of-two scale (X and A times 2^12, B times 2^11) keeps 11 bits of
// every entry that matters, three more than bfloat16.  Two choices keep its rounding from being amplified by the iteration,
// which multiplies small singular values by up to a each step:
//   * X itself is kept in fp32 beside its float16 copy and a X is added from there; the rounding of the copy only enters
//     through B X and A, where it is multiplied by the row and column spaces of X and cannot feed empty directions;
//   * the diagonals of A and B are kept in fp32 and only the rest is rounded: A = D + R, A A = D D + D R + R D + R R, and
//     B X = diag(B) X + (B - diag(B)) X with both terms taken from the same float16 X, so that directions in which they
//     cancel stay empty.
// Error of the result before its rounding: 2e-4 to 1.4e-3 of its norm over Gaussian, noisy low-rank and low-rank matrices
// from 128 x 128 to 1024 x 1024 (bfloat16 operands: 0.4 to 2.3e-2); the rounding itself is 1.7e-3.  In matrices with a side of
// 128 or less fewer roundings average out (up to 3e-3 at 8 x 8), while the products cost little: there X is two float16
// values, high and low part, in A (three products) and in B X (two), which brings the error under 1e-3.
//
// A and B are symmetric: only tiles on and below the diagonal are computed, each is written twice.
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

// R = A without its diagonal (times 2^12), diag(A).
template <int BN>
struct EpiGram {
  static constexpr int kAcc = 1, kStride = BN;
  static constexpr bool kLate = false;
  struct Params { __half* r; float* diag; int64_t ld, stride; };
  static __device__ __forceinline__ void run(const Params& p, const Tiles& t, const TileAt& at, uint32_t tm, int row0, int half,
                                             uint4* stage) {
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
  static __device__ __forceinline__ void run(const Params& p, const Tiles& t, const TileAt& at, uint32_t tm, int row0, int half,
                                             uint4* stage) {
    const __half* r = p.r + at.batch * p.stride;
    const float* d = p.diag + at.batch * (int64_t)t.M;
    const int row = row0 + (threadIdx.x & 31);
    const float di = row < t.M ? d[row] : 0.f;
    // every global load of a chunk is issued before anything is done with one: inside conditions they would wait for each
    // other (15 us a launch that way)
#pragma unroll 1
    for (int cb = 0; cb < BN / 64; ++cb) {
      const int c = half * (BN / 2) + cb * 32, n0 = at.n * BN + c, lane = threadIdx.x & 31;
      uint4 raw[4];
#pragma unroll
      for (int q = 0; q < 4; ++q)  // rows are padded to 8
        raw[q] = row < t.M && n0 + 8 * q < t.M ? *reinterpret_cast<const uint4*>(r + (int64_t)row * p.ld + n0 + 8 * q) : make_uint4(0, 0, 0, 0);
      const float dl = n0 + lane < t.M ? d[n0 + lane] : 0.f;
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
    const float* x; const __half* xh; const float* bdiag;  // xh: high parts; low parts `plane` further (two != 0)
    float* x_out; __half* xh_out; __nv_bfloat16* out;  // out != null: last step
    int64_t ld, stride;                                // of x, xh, x_out, xh_out
    int64_t out_stride;
    int64_t plane;
    int tall, short_side, two;
    float a;
  };
  static __device__ __forceinline__ void run(const Params& p, const Tiles& t, const TileAt& at, uint32_t tm, int row0, int half,
                                             uint4* stage) {
    const int row = row0 + (threadIdx.x & 31);
    const float* bd = p.bdiag + at.batch * (int64_t)p.short_side;
    const float bi = !p.tall && row < t.M ? bd[row] : 0.f;
    const int64_t base = at.batch * p.stride;
#pragma unroll 1
    for (int cb = 0; cb < BN / 64; ++cb) {
      const int c = half * (BN / 2) + cb * 32, n0 = at.n * BN + c;
      if (n0 >= t.N) break;
      const int64_t off = base + (int64_t)row * p.ld + n0;
      float4 xs[8];
      uint4 raw[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) {  // rows are padded to 8
        const bool in = row < t.M && n0 + 8 * q < t.N;
        xs[2 * q] = in ? *reinterpret_cast<const float4*>(p.x + off + 8 * q) : make_float4(0.f, 0.f, 0.f, 0.f);
        xs[2 * q + 1] = in ? *reinterpret_cast<const float4*>(p.x + off + 8 * q + 4) : make_float4(0.f, 0.f, 0.f, 0.f);
        raw[q] = in && !p.two ? *reinterpret_cast<const uint4*>(p.xh + off + 8 * q) : make_uint4(0, 0, 0, 0);
      }
      const float bl = p.tall && n0 + (int)(threadIdx.x & 31) < t.N ? bd[n0 + (threadIdx.x & 31)] : 0.f;
      float v[32];
      tmem_ld32(tm + c, v);
#pragma unroll
      for (int j = 0; j < 32; ++j) {
        const float x = reinterpret_cast<const float*>(xs)[j];
        const float b = p.tall ? __shfl_sync(0xffffffffu, bl, j) : bi;
        const float xb = p.two ? x : __half2float(reinterpret_cast<const __half*>(raw)[j]) * (1.f / kXScale);  // what the product read
        v[j] = p.a * x + b * xb + v[j] * (1.f / (kXScale * kBScale));
      }
      if (p.out != nullptr) {
        uint4 o[4];
        pack32<__nv_bfloat16>(v, o);
        __nv_bfloat16* dst = p.out + at.batch * p.out_stride;
        store_piece<__nv_bfloat16, 4>(stage, o, dst + (int64_t)row0 * t.N + n0, t.N, t.M - row0, t.N - n0,
                                      t.N % 8 == 0 && (reinterpret_cast<uintptr_t>(dst) & 15) == 0);
      } else {
        uint4 o[8];
        pack32<float>(v, o);
        store_piece<float, 8>(stage, o, p.x_out + base + (int64_t)row0 * p.ld + n0, p.ld, t.M - row0, t.N - n0, true);
#pragma unroll
        for (int j = 0; j < 32; ++j) v[j] *= kXScale;
        uint4 oh[4];
        pack32<__half>(v, oh);
        __half* dst = p.xh_out + base + (int64_t)row0 * p.ld + n0;
        store_piece<__half, 4>(stage, oh, dst, p.ld, t.M - row0, t.N - n0, true);
        if (p.two) {
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] -= __half2float(__float2half_rn(v[j]));
          pack32<__half>(v, oh);
          store_piece<__half, 4>(stage, oh, dst + p.plane, p.ld, t.M - row0, t.N - n0, true);
        }
      }
    }
  }
};

// Sums of squares of G in float64 (no gradient is too small or too large for them): one partial per block.
template <typename T>
__global__ void __launch_bounds__(256) ns_norm_kernel(const T* __restrict__ g, int64_t count, double* __restrict__ partial) {
  const T* src = g + blockIdx.y * count;
  double s = 0.0;
  for (int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; i < count; i += (int64_t)gridDim.x * blockDim.x) {
    const double v = (double)widen(src[i]);
    s += v * v;
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

// X = G / (|G| + eps) in fp32 and float16, rows padded to a multiple of 8.
template <typename T>
__global__ void __launch_bounds__(256) ns_init_kernel(const T* __restrict__ g, int rows, int cols, int64_t ld, const double* __restrict__ partial,
                                                      int parts, double eps, float* __restrict__ x, __half* __restrict__ xh,
                                                      int64_t plane) {
  __shared__ double scale;
  if (threadIdx.x < 32) {
    double s = 0.0;
    for (int i = threadIdx.x; i < parts; i += 32) s += partial[blockIdx.y * parts + i];
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (threadIdx.x == 0) scale = 1.0 / (sqrt(s) + eps);
  }
  __syncthreads();
  const double k = scale;
  const T* src = g + blockIdx.y * (int64_t)rows * cols;
  const int64_t base = blockIdx.y * (int64_t)rows * ld;
  for (int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; i < (int64_t)rows * cols; i += (int64_t)gridDim.x * blockDim.x) {
    const int64_t r = i / cols, c = i - r * cols;
    const float v = (float)((double)widen(src[i]) * k);
    x[base + r * ld + c] = v;
    const __half h = __float2half_rn(v * kXScale);
    xh[base + r * ld + c] = h;
    if (plane != 0) xh[plane + base + r * ld + c] = __float2half_rn(v * kXScale - __half2float(h));
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
  TORCH_CHECK(batch <= 65535 && m < (1 << 30) && n < (1 << 30), "newton_schulz: sizes out of range");
  const bool tall = m > n;
  const int64_t r = std::min(m, n), ld = (n + 7) / 8 * 8, rld = (r + 7) / 8 * 8;
  const int planes = r <= 128 ? 2 : 1;
  const int64_t plane = batch * m * ld;
  auto opt = [&](at::ScalarType t) { return g.options().dtype(t); };
  const int parts = (int)std::max<int64_t>(1, std::min<int64_t>({(m * n + 2047) / 2048, 1024, std::max<int64_t>(1, 4 * sm_count() / batch)}));
  Tensor partial = at::empty({batch, parts}, opt(at::kDouble));
  Tensor x = at::empty({batch, m, ld}, opt(at::kFloat)), xh = at::empty({2, planes, batch, m, ld}, opt(at::kHalf));
  Tensor ra = at::empty({2, batch, r, rld}, opt(at::kHalf)), diag = at::empty({2, batch, r}, opt(at::kFloat));
  auto prep = [&](auto v) {
    using T = decltype(v);
    const T* p = (const T*)g.data_ptr();
    ns_norm_kernel<T><<<dim3(parts, batch), 256, 0, st>>>(p, m * n, partial.data_ptr<double>());
    ns_init_kernel<T><<<dim3(parts, batch), 256, 0, st>>>(p, (int)m, (int)n, ld, partial.data_ptr<double>(), parts, eps, x.data_ptr<float>(),
                                                          (__half*)xh.data_ptr(), planes == 2 ? plane : 0);
  };
  if (g.scalar_type() == at::kFloat) prep(float{});
  else if (g.scalar_type() == at::kHalf) prep(__half{});
  else prep(__nv_bfloat16{});
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  __half *xh0 = (__half*)xh.data_ptr(), *rp = (__half*)ra.data_ptr(), *bp = rp + batch * r * rld;
  float *ad = diag.data_ptr<float>(), *bd = ad + batch * r;
  auto stored_x = [&](int which) { return Stored{xh0 + which * planes * plane, n, m, ld, planes * batch, m * ld}; };
  const Stored sr{rp, r, r, rld, batch, r * rld}, sb{bp, r, r, rld, batch, r * rld};
  // columns of a tile: 256 where that still gives every pair of CTAs a tile
  auto wide = [&](int64_t rows, int64_t tiles) { return use_pair(rows) && tiles >= sm_count() / 2; };
  const int64_t rt = (r + 255) / 256;
  const int bn = wide(m, batch * ((m + 255) / 256) * ((n + 255) / 256)) ? 256 : 128, sbn = wide(r, batch * (rt * (rt + 1) / 2)) ? 256 : 128;
  for (int64_t i = 0; i < steps; ++i) {
    const int cur = (int)(i & 1);
    {
      Maps maps;
      Tiles t{};
      put_map(maps, 0, stored_x(cur));
      for (int k = planes == 2 ? 0 : 2; k < 3; ++k)  // low . high, high . low, high . high
        add_segment(t, 0, tall, 0, tall, tall ? m : n, sbn, k == 0 ? (int)batch : 0, k == 1 ? (int)batch : 0);
      set_tiles(t, r, r, sbn, batch, 1, true);
      if (sbn == 256) run_dense<256, EpiGram<256>>(maps, t, {rp, ad, rld, r * rld}, st);
      else run_dense<128, EpiGram<128>>(maps, t, {rp, ad, rld, r * rld}, st);
    }
    {
      Maps maps;
      Tiles t{};
      put_map(maps, 0, sr);
      add_segment(t, 0, false, 0, false, r, sbn);
      set_tiles(t, r, r, sbn, batch, 1, true);
      if (sbn == 256) run_dense<256, EpiPoly<256>>(maps, t, {rp, ad, bp, bd, rld, r * rld, (float)b, (float)c}, st);
      else run_dense<128, EpiPoly<128>>(maps, t, {rp, ad, bp, bd, rld, r * rld, (float)b, (float)c}, st);
    }
    Maps maps;
    Tiles t{};
    put_map(maps, 0, tall ? stored_x(cur) : sb);
    put_map(maps, 1, tall ? sb : stored_x(cur));
    for (int k = 0; k < planes; ++k) add_segment(t, 0, false, 1, !tall, r, bn, tall ? k * (int)batch : 0, tall ? 0 : k * (int)batch);
    set_tiles(t, m, n, bn, batch, 1);
    auto update = [&](auto tag) {
      constexpr int BN = decltype(tag)::value;
      typename EpiUpdate<BN>::Params ep{x.data_ptr<float>(), xh0 + cur * planes * plane, bd, x.data_ptr<float>(),
                                        xh0 + (1 - cur) * planes * plane,
                                        i + 1 == steps ? (__nv_bfloat16*)out.data_ptr() : nullptr, ld, m * ld, m * n, plane, tall ? 1 : 0, (int)r, planes - 1,
                                        (float)a};
      run_dense<BN, EpiUpdate<BN>>(maps, t, ep, st);
    };
    if (bn == 256) update(std::integral_constant<int, 256>{});
    else update(std::integral_constant<int, 128>{});
  }
  return out;
}

int64_t newton_schulz_error_status(const Tensor& like) {
  c10::cuda::CUDAGuard guard(like.device());
  int v = 0, zero = 0;
  C10_CUDA_CHECK(cudaMemcpyFromSymbol(&v, dense::error_word, sizeof(int)));
  if (v != 0) C10_CUDA_CHECK(cudaMemcpyToSymbol(dense::error_word, &zero, sizeof(int)));
  return v;
}

}  // namespace nva

TORCH_LIBRARY_FRAGMENT(nvalchemi, m) {
  m.def("newton_schulz(Tensor g, int steps, float a, float b, float c, float eps) -> Tensor", &nva::newton_schulz);
  m.def("newton_schulz_error_status(Tensor like) -> int", &nva::newton_schulz_error_status);
}
