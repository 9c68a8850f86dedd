// SPDX-License-Identifier: Apache-2.0
// Gated feed-forward block  y = (act(x Wg) * (x Wu)) Wd  and its backward pass, for 16-bit and float32 matrices.
//
// Forward: one kernel forms both projections of a tile side by side (the B tile's halves come from Wg and Wu, so one
// instruction feeds both accumulators), applies the activation and the product in its epilogue and stores h only; a second
// product gives y.  Backward: with g = x Wg, u = x Wu, dh = dy Wd^T
//     dg = dh u act'(g),  du = dh act(g),  dx = dg Wg^T + du Wu^T,  dWg = x^T dg,  dWu = x^T du,  dWd = h^T dy.
// g and u are formed again in the kernel that forms dh (three accumulators of one tile) instead of being kept: at the widths
// of per-atom networks (K <= 1024) the extra 4 M K H operations cost less than writing and reading 2 M H values in 32 bits,
// and 16-bit copies would add their rounding to every gradient.  What is rounded to 16 bits is what the next product reads:
// h, dg and du, once each (float16: values of h past 65504 become infinite).  Over many rows and columns those roundings average
// out (the error of a result is sqrt(2) times its own rounding); up to 256 rows, where the products cost next to nothing, they
// are kept as a 16-bit value and a 16-bit remainder and the next product reads both.
//
// Where the contraction axis of a projection (K, or N for dh) is too long for the accumulators of one tile (max_blocks: K past
// 8192 in float16, 65,536 in bfloat16, 2048 in float32), g, u and dh are formed as float32 matrices by split products and a
// kernel of its own applies the gate.
//
// float32 matrices run on the same tensor cores: a value is the exact sum of three bf16 values and a product the six
// partial products above 2^-24 of it; the intermediate h, dg and du are stored as three planes each, so nothing is lost to
// 16 bits.  There dh is a product of its own (its accumulators would not fit beside those of g and u).
//
// What bounds it (8192 x 1024 -> 4096 -> 1024, bfloat16): the plain products run at 1150 to 1490 TFLOP/s (51 to 58 us of 69
// GFLOP, 92 to 105 us of 137), tensor-bound up to the last, partly filled round of tiles; both projections with the gate 97 us
// (137 GFLOP), the gate's gradient 188 us (206 GFLOP), whose epilogue is only hidden behind the part of the next tile that
// forms dh.  Narrow blocks (131,072 x 128 -> 512 -> 128) are bound by the epilogue and by h going through memory: 72 us for h,
// 33 us for y.  float32 (4096 x 256 -> 1024 -> 256) does six times the products: 270 us forward and backward.
#include "dense16.cuh"
#include "gate.cuh"

namespace nva {
using at::Tensor;

// feedforward_rows.cu: up to 8 rows
bool gated_ff_rows(const Tensor& x, const Tensor& wg, const Tensor& wu, const Tensor& wd, int64_t act, Tensor& y, cudaStream_t st);

namespace {
using namespace dense;

// The branch on the activation stays outside the loop over a thread's values: inside it the values' chains of dependent
// instructions would run one after the other (131,072 x 128 x 512: 222 us that way).
template <bool EXACT, int ACT, int C>
__device__ __forceinline__ void gate(float (&g)[C], const float (&u)[C]) {
#pragma unroll
  for (int j = 0; j < C; ++j) {
    float a, da;
    activate<EXACT, ACT>(g[j], a, da);
    g[j] = a * u[j];
  }
}
// (g, u, dh) -> (dg, h, du)
template <bool EXACT, int ACT, int C>
__device__ __forceinline__ void gate_grad(float (&g)[C], float (&u)[C], float (&d)[C]) {
#pragma unroll
  for (int j = 0; j < C; ++j) {
    float a, da;
    activate<EXACT, ACT>(g[j], a, da);
    g[j] = d[j] * u[j] * da;
    d[j] *= a;
    u[j] *= a;
  }
}

// C columns of a warp's 32 rows as T (two: and the remainder as T), or as three bf16 planes of a float32 value.
template <typename T, int C>
__device__ __forceinline__ void store_cols(uint4* stage, float (&v)[C], void* dst, int64_t off, int64_t ld, int64_t plane, int rows_left,
                                           int cols_left, int two) {
  using S = typename std::conditional<sizeof(T) == 4, __nv_bfloat16, T>::type;
  auto put = [&](const uint32_t (&w)[C / 2], int64_t at) {
    uint4 o[C / 8];
#pragma unroll
    for (int j = 0; j < C / 8; ++j) o[j] = make_uint4(w[4 * j], w[4 * j + 1], w[4 * j + 2], w[4 * j + 3]);
    store_piece<S, C / 8>(stage, o, (S*)dst + at, ld, rows_left, cols_left, true);  // rows are padded to 8
  };
  if constexpr (sizeof(T) == 2) {
    uint32_t w[C / 2];
#pragma unroll
    for (int j = 0; j < C / 2; ++j) w[j] = pack2(v[2 * j], v[2 * j + 1], T{});
    put(w, off);
    if (two) {
#pragma unroll
      for (int j = 0; j < C; ++j) v[j] -= widen(narrow<T>(v[j]));
#pragma unroll
      for (int j = 0; j < C / 2; ++j) w[j] = pack2(v[2 * j], v[2 * j + 1], T{});
      put(w, off + plane);
    }
  } else {
    uint32_t w0[C / 2], w1[C / 2], w2[C / 2];
#pragma unroll
    for (int j = 0; j < C / 2; ++j) {
      uint32_t p[3];
      split3(v[2 * j], v[2 * j + 1], p);
      w0[j] = p[0]; w1[j] = p[1]; w2[j] = p[2];
    }
    put(w0, off);
    put(w1, off + plane);
    put(w2, off + 2 * plane);
  }
}

// NaN in `cols` columns of a warp's rows of an intermediate; its other planes need none, what reads them reads this one too.
template <typename T>
__device__ __forceinline__ void poison_cols(void* dst, int64_t ld, const Tiles& t, int row0, int n0, int cols) {
  using S = typename std::conditional<sizeof(T) == 4, __nv_bfloat16, T>::type;
  fill_nan((S*)dst + (int64_t)row0 * ld + n0, ld, t.M - row0, t.N - n0, cols);
}

// Columns [0, BN/2) of the accumulator: g, [BN/2, BN): u, both of the same BN/2 columns of h.
template <typename T, int BN>
struct EpiGated : NoPrefetch {
  static constexpr int kAcc = sizeof(T) == 4 ? 512 / BN : 1, kStride = BN;
  static constexpr bool kLate = false;
  struct Params { void* h; int64_t ld, plane; int act, two; };
  static __device__ __forceinline__ void poison(const Params& p, const Tiles& t, const TileAt& at, int row0, int part) {
    poison_cols<T>(p.h, p.ld, t, row0, at.n * (BN / 2) + part * (BN / 4), BN / 4);
  }
  static __device__ __forceinline__ void run(const Params& p, const Tiles& t, const TileAt& at, uint32_t tm, int row0, int part,
                                             uint4* stage, Pre&) {
    const int used = used_acc<kAcc>(t, at, 0);
#pragma unroll 1
    for (int cb = 0; cb < BN / 128; ++cb) {
      const int c = part * (BN / 4) + cb * 32, n0 = at.n * (BN / 2) + c;
      float g[32], u[32];
      acc_ld32<kAcc, kStride>(tm + c, g, used);
      acc_ld32<kAcc, kStride>(tm + BN / 2 + c, u, used);
      if (p.act == kSilu) gate<sizeof(T) == 4, kSilu>(g, u);
      else gate<sizeof(T) == 4, kGelu>(g, u);
      store_cols<T>(stage, g, p.h, (int64_t)row0 * p.ld + n0, p.ld, p.plane, t.M - row0, t.N - n0, p.two);
    }
  }
};

struct GradOut { void *dg, *du, *h; int64_t ld, plane; int act, two; };
template <typename T>
__device__ __forceinline__ void store_grads(const GradOut& p, const Tiles& t, int row0, int n0, uint4* stage, float (&g)[32], float (&u)[32],
                                            float (&d)[32]) {
  if (p.act == kSilu) gate_grad<sizeof(T) == 4, kSilu>(g, u, d);
  else gate_grad<sizeof(T) == 4, kGelu>(g, u, d);
  const int64_t off = (int64_t)row0 * p.ld + n0;
  store_cols<T>(stage, g, p.dg, off, p.ld, p.plane, t.M - row0, t.N - n0, p.two);
  store_cols<T>(stage, d, p.du, off, p.ld, p.plane, t.M - row0, t.N - n0, p.two);
  store_cols<T>(stage, u, p.h, off, p.ld, p.plane, t.M - row0, t.N - n0, p.two);
}

template <typename T>
__device__ __forceinline__ void poison_grads(const GradOut& p, const Tiles& t, int row0, int n0, int cols) {
  for (void* dst : {p.dg, p.du, p.h}) poison_cols<T>(dst, p.ld, t, row0, n0, cols);
}

// 16 bits: of 128 columns of h, g in accumulator columns [0, 128), u in [128, 256), dh after those, in turns in two places (see
// dense_kernel).
template <typename T>
struct EpiGatedGrad : NoPrefetch {
  static constexpr int kAcc = 1, kStride = 0;
  static constexpr bool kLate = true;
  using Params = GradOut;
  static __device__ __forceinline__ void poison(const Params& p, const Tiles& t, const TileAt& at, int row0, int part) {
    poison_grads<T>(p, t, row0, at.n * 128 + part * 64, 64);
  }
  static __device__ __forceinline__ void run(const Params& p, const Tiles& t, const TileAt& at, uint32_t tm, int row0, int part,
                                             uint4* stage, Pre&) {
    const uint32_t td = tm + 256 + (at.seq & 1) * 128;
#pragma unroll 1
    for (int cb = 0; cb < 2; ++cb) {
      const int c = part * 64 + cb * 32;
      float g[32], u[32], d[32];
      tmem_ld32(tm + c, g);
      tmem_ld32(tm + 128 + c, u);
      tmem_ld32(td + c, d);
      store_grads<T>(p, t, row0, at.n * 128 + c, stage, g, u, d);
    }
  }
};

// float32: g and u as in EpiGated, dh [M][ld_dh] (rows on 16-byte boundaries) from memory.
template <int BN>
struct EpiGatedGradRead {
  static constexpr int kAcc = 512 / BN, kStride = BN;
  static constexpr bool kLate = false;
  struct Params { GradOut out; const float* dh; int64_t ld_dh; };
  struct Pre { uint4 raw[8]; };  // 32 columns of dh
  static __device__ __forceinline__ void poison(const Params& p, const Tiles& t, const TileAt& at, int row0, int part) {
    poison_grads<float>(p.out, t, row0, at.n * (BN / 2) + part * (BN / 4), BN / 4);
  }
  static __device__ __forceinline__ void fetch(const Params& p, const Tiles& t, int row0, int n0, Pre& pre) {
    fetch_piece<float, 8>(pre.raw, p.dh + (int64_t)row0 * p.ld_dh + n0, p.ld_dh, t.M - row0, t.N - n0);
  }
  static __device__ __forceinline__ void prefetch(const Params& p, const Tiles& t, const TileAt& at, int row0, int part, Pre& pre) {
    fetch(p, t, row0, at.n * (BN / 2) + part * (BN / 4), pre);
  }
  static __device__ __forceinline__ void run(const Params& p, const Tiles& t, const TileAt& at, uint32_t tm, int row0, int part,
                                             uint4* stage, Pre& pre) {
    const int used = used_acc<kAcc>(t, at, 0);
#pragma unroll 1
    for (int cb = 0; cb < BN / 128; ++cb) {
      const int c = part * (BN / 4) + cb * 32, n0 = at.n * (BN / 2) + c;
      float g[32], u[32], d[32];
      turn_piece<8>(stage, pre.raw);
#pragma unroll
      for (int j = 0; j < 32; ++j) d[j] = reinterpret_cast<const float*>(pre.raw)[j];
      if (cb + 1 < BN / 128) fetch(p, t, row0, n0 + 32, pre);
      acc_ld32<kAcc, kStride>(tm + c, g, used);
      acc_ld32<kAcc, kStride>(tm + BN / 2 + c, u, used);
      store_grads<float>(p.out, t, row0, n0, stage, g, u, d);
    }
  }
};

// Copies matrices into rows on 16-byte boundaries (T 16-bit), or splits float32 into three bf16 planes: one launch for all of a
// call's operands (grid.y), two elements a thread.
constexpr int kMaxPacks = 5;
struct PackJob { const void* src; uint16_t* dst; int64_t ld, rows, cols, ldp, plane; };
struct PackJobs { PackJob j[kMaxPacks]; int n = 0; };

template <typename T, int P>
__global__ void __launch_bounds__(256) pack_kernel(const __grid_constant__ PackJobs jobs) {
  chain_wait();
  const PackJob job = jobs.j[blockIdx.y];
  const int64_t half = (job.cols + 1) / 2, total = job.rows * half;
  for (int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; i < total; i += (int64_t)gridDim.x * blockDim.x) {
    const int64_t r = total <= 0x7fffffff ? (int64_t)((uint32_t)i / (uint32_t)half) : i / half, c = (i - r * half) * 2;
    const bool two = c + 1 < job.cols;
    const T* s = (const T*)job.src + r * job.ld + c;
    uint16_t* d = job.dst + r * job.ldp + c;
    if constexpr (P == 1) {
      const uint16_t* s16 = reinterpret_cast<const uint16_t*>(s);
      *reinterpret_cast<uint32_t*>(d) = (uint32_t)s16[0] | (two ? (uint32_t)s16[1] << 16 : 0u);
    } else {
      uint32_t p[3];
      split3((float)s[0], two ? (float)s[1] : 0.f, p);
#pragma unroll
      for (int k = 0; k < 3; ++k) *reinterpret_cast<uint32_t*>(d + k * job.plane) = p[k];
    }
  }
}

void run_packs(const PackJobs& jobs, int planes, cudaStream_t st) {
  if (jobs.n == 0) return;
  int64_t most = 0;
  for (int i = 0; i < jobs.n; ++i) most = std::max(most, jobs.j[i].rows * ((jobs.j[i].cols + 1) / 2));
  const dim3 grid((unsigned)std::min<int64_t>((most + 255) / 256, 148 * 8), (unsigned)jobs.n);
  launch_chained(planes == 3 ? pack_kernel<float, 3> : pack_kernel<__half, 1>, grid, 256, st, jobs);
}

// A matrix as a product reads it.  `mn` says whether the axis that is not contracted is contiguous, when the contraction
// runs over axis `k_axis` of the logical matrix.
struct Operand {
  Stored s;
  Tensor keep, source;
  int planes = 1;  // parts of a value: 1, 2 (16-bit value and remainder) or 3 (float32)
  bool rowmajor = true;
  bool mn(int k_axis) const { return rowmajor != (k_axis == 1); }
  int64_t extent(int axis) const { return (axis == 1) == rowmajor ? s.inner : s.outer; }
};

int planes_of(const Tensor& t) { return t.scalar_type() == at::kFloat ? 3 : 1; }

// Whether a matrix is read by rows (its columns contiguous otherwise); one with neither axis contiguous is copied by rows.
bool by_rows(const Tensor& t) { return t.stride(1) == 1 || t.size(1) == 1 || !(t.stride(0) == 1 || t.size(0) == 1); }

// The operand of a tensor, read by rows or by columns; what has to be packed for it is added to `jobs` and there after run_packs.
Operand operand(Tensor t, PackJobs& jobs, bool rowmajor) {
  Operand o;
  o.rowmajor = rowmajor;
  if (!rowmajor) t = t.t();
  if (t.stride(1) != 1 && t.size(1) != 1) t = t.contiguous();
  const int64_t rows = t.size(0), cols = t.size(1), ld = rows > 1 ? t.stride(0) : cols;
  if (planes_of(t) == 1 && (rows == 1 || (ld % 8 == 0 && ld >= cols)) && (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) == 0) {
    o.keep = t;
    o.s = {t.data_ptr(), cols, rows, ld, 1, 0};
    return o;
  }
  const int P = o.planes = planes_of(t);
  const int64_t ldp = (cols + 7) / 8 * 8;
  o.source = t;
  o.keep = at::empty({P, rows, ldp}, t.options().dtype(P == 3 ? at::kBFloat16 : t.scalar_type()));
  TORCH_CHECK(jobs.n < kMaxPacks, "gated_ff: too many operands to pack");
  jobs.j[jobs.n++] = {t.data_ptr(), (uint16_t*)o.keep.data_ptr(), ld, rows, cols, ldp, rows * ldp};
  o.s = {o.keep.data_ptr(), cols, rows, ldp, P, rows * ldp};
  return o;
}
Operand operand(const Tensor& t, PackJobs& jobs) { return operand(t, jobs, by_rows(t)); }

// Intermediate [P][rows][ld] (16-bit) that epilogues write and later products read.
Operand intermediate(int64_t rows, int64_t cols, int planes, const Tensor& like, int copies = 1) {
  Operand o;
  const int64_t ld = (cols + 7) / 8 * 8;
  o.planes = planes;
  o.keep = at::empty({copies * planes, rows, ld}, like.options().dtype(like.scalar_type() == at::kFloat ? at::kBFloat16 : like.scalar_type()));
  o.s = {o.keep.data_ptr(), cols, rows, ld, copies * planes, rows * ld};
  return o;
}

struct Plan {
  Maps maps;
  Tiles t{};
  int n_maps = 0;
  bool bf16;
  explicit Plan(bool bf16_) : bf16(bf16_) {}
  int map(const Operand& o) { put_map(maps, n_maps, o.s); return n_maps++; }
  // a[.., k] . b[.., k]; ka / kb: the axis of each logical matrix that is contracted; b2 < 0: both halves from b.
  // part 0: the small partial products (added first), 1: the large one, 2: both.
  void product(int a, const Operand& oa, int ka, int b, int b2, const Operand& ob, int kb, int col, int n, int a_z = 0, int b_z = 0,
               int a_step = 0, int b_step = 0, int part = 2, int group = 0) {
    const int64_t K = oa.extent(ka);
    auto add = [&](int za, int zb) {
      const bool main = za + zb == 0;
      if (part != 2 && main != (part == 1)) return;
      TORCH_CHECK(t.n_seg < kMaxSegs, "dense: too many segments");
      Seg& s = t.seg[t.n_seg++];
      s.a = (int8_t)a; s.b = (int8_t)b; s.b2 = (int8_t)(b2 < 0 ? b : b2);
      s.a_mn = oa.mn(ka); s.b_mn = ob.mn(kb);
      s.group = (int8_t)group;
      s.spread = main;
      s.col = (int16_t)col; s.n = (int16_t)n;
      s.za = a_z + za; s.zb = b_z + zb;
      s.za_step = a_step; s.zb_step = b_step;
      s.nk = (int)((K + BK - 1) / BK);
      s.b2_off = b2 < 0 ? n / 2 : 0;
      s.idesc = idesc16(bf16, s.a_mn, s.b_mn, n, BM);
      if (main) t.main_nk[group] = s.nk;
    };
    if (oa.planes == 3 && ob.planes == 3) {  // what is left out is at most 2^-24 of a product
      add(2, 0); add(0, 2); add(1, 1); add(1, 0); add(0, 1);
    } else {
      if (oa.planes == 2) add(1, 0);
      if (ob.planes == 2) add(0, 1);
    }
    add(0, 0);
  }
};

// Plain product into `out` [batches][M][N].  The contraction axis is split over several tiles (partials added in order by a
// second kernel) when half of the GPU or more would have no tile and the axis is long, and so that no accumulator takes more
// than max_blocks.
template <typename T, int BN, int ACC>
void store_product(Plan& pl, Tensor& out, int64_t batches, int64_t M, int64_t N, cudaStream_t st) {
  set_tiles(pl.t, M, N, BN, batches, 1);
  const int tiles = pl.t.total, nk = pl.t.main_nk[0], kb = nk * pl.t.n_seg, at_once = slots(pl.t);
  int mains = 0;  // large partial products that add to the same accumulators
  for (int i = 0; i < pl.t.n_seg; ++i) mains += pl.t.seg[i].spread;
  const int limit = max_blocks(out.scalar_type()) * ACC, load = nk * (ACC > 1 ? mains : pl.t.n_seg);
  int splits = 1;
  if (2 * tiles <= at_once) splits = std::max(1, std::min({at_once / tiles, kb / 8, nk, kPartials}));
  splits = std::min(nk, std::max(splits, (load + limit - 1) / limit));
  if (splits > 1) {
    split_product<T, BN, ACC>(pl.maps, pl.t, M, N, batches, splits, true, (T*)out.data_ptr(), out.options().dtype(at::kFloat), st);
    return;
  }
  typename EpiStore<T, BN, ACC>::Params ep{(T*)out.data_ptr(), N, M * N, 0};
  run_dense<BN, EpiStore<T, BN, ACC>>(pl.maps, pl.t, ep, st);
}

// Columns of a tile of an M x N product over `kb` blocks of the contraction axis (all segments): by the number of tiles, and 256
// where splitting that axis fills at least three quarters of the GPU with wide tiles.
int store_bn(int64_t batches, int64_t M, int64_t N, int64_t kb) {
  if (!use_pair(M)) return 128;
  const int64_t rows = batches * ((M + 2 * BM - 1) / (2 * BM)), wide = rows * ((N + 255) / 256), pairs = sm_count() / 2;
  if (wide < pairs && 4 * wide * std::min(pairs / wide, kb / 8) >= 3 * pairs) return 256;
  return pick_bn(wide, rows * ((N + 127) / 128));
}
// Parts in which intermediates are kept: 16-bit ones of few rows with their remainder.
int parts_of(int P, int64_t M) { return P == 1 && M <= 256 ? 2 : P; }
// Blocks of the contraction axis of a product with an axis of K.
int64_t blocks_of(int P, int64_t K) { return (K + BK - 1) / BK * (P == 3 ? 6 : 1); }
void store_any(Plan& pl, int bn, Tensor& out, int64_t batches, int64_t M, int64_t N, cudaStream_t st) {
  auto go = [&](auto v) {
    using T = decltype(v);
    constexpr int ACC = sizeof(T) == 4 ? 2 : 1;  // float32: all of the TMEM
    if (bn == 256) store_product<T, 256, ACC>(pl, out, batches, M, N, st);
    else store_product<T, 128, 2 * ACC - (ACC == 1)>(pl, out, batches, M, N, st);
  };
  if (out.scalar_type() == at::kFloat) go(float{});
  else if (out.scalar_type() == at::kHalf) go(__half{});
  else go(__nv_bfloat16{});
}

// Whether a projection over an axis of K is too long for the accumulators of one tile (float32: four of them, at most).
bool far(const Tensor& x, int64_t K) { return (K + BK - 1) / BK > max_blocks(x.scalar_type()) * (x.scalar_type() == at::kFloat ? 4 : 1); }

// Columns (of g and u together) of the tiles that form both projections.  float32: 256 leave room for two accumulators, 128 for
// four.
int gate_bn(const Tensor& x, int64_t M, int64_t H, int64_t K) {
  const bool two = x.scalar_type() != at::kFloat || (K + BK - 1) / BK <= 2 * max_blocks(at::kFloat);
  return two ? store_bn(1, M, 2 * H, 0) : 128;
}

// out [M][N] float32 = a . b over axes 1 and `kb`.
void project(bool bf16, const Operand& a, const Operand& b, int kb, Tensor& out, cudaStream_t st) {
  Plan pl(bf16);
  const int64_t M = out.size(0), N = out.size(1);
  const int bn = store_bn(1, M, N, blocks_of(a.planes, a.extent(1)));
  const int ia = pl.map(a), ib = pl.map(b);
  pl.product(ia, a, 1, ib, -1, b, kb, 0, bn);
  store_any(pl, bn, out, 1, M, N, st);
}

// The gate on float32 matrices g, u [M][H] (and dh [M][ld_dh]): h, or dg, du and h.
template <typename T, bool GRAD>
__global__ void __launch_bounds__(256) gate_kernel(const float* __restrict__ gm, const float* __restrict__ um, const float* __restrict__ dm,
                                                   int64_t ld_dh, int64_t M, int64_t H, const __grid_constant__ GradOut out) {
  constexpr bool EXACT = sizeof(T) == 4;
  chain_wait();
  auto put = [&](void* dst, int64_t at, float v) {
    if constexpr (EXACT) {
      uint32_t p[3];
      split3(v, 0.f, p);
#pragma unroll
      for (int k = 0; k < 3; ++k) ((__nv_bfloat16*)dst)[at + k * out.plane] = __ushort_as_bfloat16((unsigned short)p[k]);
    } else {
      ((T*)dst)[at] = narrow<T>(v);
      if (out.two) ((T*)dst)[at + out.plane] = narrow<T>(v - widen(narrow<T>(v)));
    }
  };
  for (int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; i < M * H; i += (int64_t)gridDim.x * blockDim.x) {
    const int64_t r = i / H, c = i - r * H, at = r * out.ld + c;
    float g[1] = {gm[i]}, u[1] = {um[i]};
    if constexpr (GRAD) {
      float d[1] = {dm[r * ld_dh + c]};
      if (out.act == kSilu) gate_grad<EXACT, kSilu>(g, u, d);
      else gate_grad<EXACT, kGelu>(g, u, d);
      put(out.dg, at, g[0]);
      put(out.du, at, d[0]);
      put(out.h, at, u[0]);
    } else {
      if (out.act == kSilu) gate<EXACT, kSilu>(g, u);
      else gate<EXACT, kGelu>(g, u);
      put(out.h, at, g[0]);
    }
  }
}
// g = x Wg and u = x Wu through memory, then the gate (dh: float32 [M][ld_dh], or undefined for the forward pass).
void gate_through_memory(const Tensor& x, const Operand& ox, const Operand& og, const Operand& ou, const Tensor& dh, int64_t H,
                         const GradOut& out, cudaStream_t st) {
  const int64_t M = x.size(0);
  Tensor gu = at::empty({2, M, H}, x.options().dtype(at::kFloat)), g = gu.select(0, 0), u = gu.select(0, 1);
  project(x.scalar_type() != at::kHalf, ox, og, 0, g, st);
  project(x.scalar_type() != at::kHalf, ox, ou, 0, u, st);
  const dim3 grid((unsigned)std::min<int64_t>((M * H + 255) / 256, 148 * 8));
  auto go = [&](auto v) {
    using T = decltype(v);
    if (dh.defined())
      launch_chained(gate_kernel<T, true>, grid, 256, st, g.data_ptr<float>(), u.data_ptr<float>(), dh.data_ptr<float>(), dh.size(1), M, H, out);
    else
      launch_chained(gate_kernel<T, false>, grid, 256, st, g.data_ptr<float>(), u.data_ptr<float>(), (const float*)nullptr, (int64_t)0, M, H, out);
  };
  if (x.scalar_type() == at::kFloat) go(float{});
  else if (x.scalar_type() == at::kHalf) go(__half{});
  else go(__nv_bfloat16{});
}

void check_ff(const Tensor& x, const Tensor& wg, const Tensor& wu, const Tensor& wd, int64_t act) {
  for (const Tensor* t : {&x, &wg, &wu, &wd})
    TORCH_CHECK(t->is_cuda() && t->device() == x.device() && t->scalar_type() == x.scalar_type(), "gated_ff: tensors of one type on one CUDA device");
  TORCH_CHECK(x.scalar_type() == at::kFloat || x.scalar_type() == at::kHalf || x.scalar_type() == at::kBFloat16,
              "gated_ff: float32, float16 or bfloat16");
  TORCH_CHECK(x.dim() >= 1 && wg.dim() == 2 && wu.dim() == 2 && wd.dim() == 2, "gated_ff: weights must be matrices");
  TORCH_CHECK(wg.size(0) == x.size(-1) && wu.sizes() == wg.sizes() && wd.size(0) == wg.size(1), "gated_ff: shapes do not fit");
  TORCH_CHECK(act == kSilu || act == kGelu, "gated_ff: unknown activation");
  TORCH_CHECK(x.size(-1) >= 1 && wg.size(1) >= 1 && wd.size(1) >= 1, "gated_ff: sizes out of range");
  TORCH_CHECK(x.numel() / x.size(-1) < (1ll << 31) && x.size(-1) < (1ll << 31) && wg.size(1) < (1ll << 31) && wd.size(1) < (1ll << 31),
              "gated_ff: sizes out of range");
}
Tensor as_matrix(const Tensor& t) { return t.dim() == 2 ? t : t.reshape({t.numel() / t.size(-1), t.size(-1)}); }
std::vector<int64_t> out_sizes(const Tensor& x, int64_t n) {
  std::vector<int64_t> s = x.sizes().vec();
  s.back() = n;
  return s;
}

}  // namespace

Tensor gated_ff_fwd(const Tensor& x_in, const Tensor& wg, const Tensor& wu, const Tensor& wd, int64_t act) {
  check_ff(x_in, wg, wu, wd, act);
  c10::cuda::CUDAGuard guard(x_in.device());
  const Tensor x = as_matrix(x_in);
  const int64_t M = x.size(0), K = x.size(1), H = wg.size(1), N = wd.size(1);
  Tensor y = at::empty(out_sizes(x_in, N), x.options());
  if (M == 0) return y;
  auto st = at::cuda::getCurrentCUDAStream();
  if (gated_ff_rows(x, wg, wu, wd, act, y, st)) return y;
  const int P = planes_of(x);
  const bool bf16 = x.scalar_type() != at::kHalf;
  PackJobs jobs;
  Operand ox = operand(x, jobs), og = operand(wg, jobs), ou = operand(wu, jobs, og.rowmajor), od = operand(wd, jobs);
  run_packs(jobs, P, st);
  const int Pi = parts_of(P, M);
  Operand oh = intermediate(M, H, Pi, x);
  if (far(x, K)) {
    gate_through_memory(x, ox, og, ou, Tensor(), H, {nullptr, nullptr, oh.keep.data_ptr(), oh.s.ld, oh.s.plane, (int)act, Pi == 2 ? 1 : 0}, st);
  } else {
    Plan pl(bf16);
    const int a = pl.map(ox), b = pl.map(og), b2 = pl.map(ou);
    auto go = [&](auto v, auto bn_tag) {
      using T = decltype(v);
      constexpr int BN = decltype(bn_tag)::value;
      pl.product(a, ox, 1, b, b2, og, 0, 0, BN);
      set_tiles(pl.t, M, H, BN / 2, 1, 1);
      typename EpiGated<T, BN>::Params ep{oh.keep.data_ptr(), oh.s.ld, oh.s.plane, (int)act, Pi == 2 ? 1 : 0};
      run_dense<BN, EpiGated<T, BN>>(pl.maps, pl.t, ep, st);
    };
    auto wide = [&](auto v) {
      if (gate_bn(x, M, H, K) == 256) go(v, std::integral_constant<int, 256>{});
      else go(v, std::integral_constant<int, 128>{});
    };
    if (P == 3) wide(float{});
    else if (bf16) wide(__nv_bfloat16{});
    else wide(__half{});
  }
  Plan pl(bf16);
  const int bn = store_bn(1, M, N, blocks_of(P, H));
  const int a = pl.map(oh), b = pl.map(od);
  pl.product(a, oh, 1, b, -1, od, 0, 0, bn);
  store_any(pl, bn, y, 1, M, N, st);
  return y;
}

// which: bit 0 dx, bit 1 dWg and dWu, bit 2 dWd; the others come back empty.
std::tuple<Tensor, Tensor, Tensor, Tensor> gated_ff_bwd(const Tensor& dy_in, const Tensor& x_in, const Tensor& wg, const Tensor& wu,
                                                        const Tensor& wd, int64_t act, int64_t which) {
  check_ff(x_in, wg, wu, wd, act);
  TORCH_CHECK(dy_in.device() == x_in.device() && dy_in.scalar_type() == x_in.scalar_type() && dy_in.sizes().vec() == out_sizes(x_in, wd.size(1)),
              "gated_ff: dy does not fit");
  c10::cuda::CUDAGuard guard(x_in.device());
  const Tensor x = as_matrix(x_in), dy = as_matrix(dy_in);
  const int64_t M = x.size(0), K = x.size(1), H = wg.size(1), N = wd.size(1);
  auto st = at::cuda::getCurrentCUDAStream();
  Tensor dx = which & 1 ? at::empty(x_in.sizes(), x.options()) : at::empty({0}, x.options()), dgu = at::empty({2, which & 2 ? K : 0, H}, x.options()),
         dwd = at::empty({which & 4 ? H : 0, N}, x.options());
  if (M == 0 || (which & 7) == 0) {
    dgu.zero_();
    dwd.zero_();
    return {dx, dgu.select(0, 0), dgu.select(0, 1), dwd};
  }
  const int P = planes_of(x);
  const bool bf16 = x.scalar_type() != at::kHalf;
  PackJobs jobs;
  Operand ox = operand(x, jobs), og = operand(wg, jobs), ou = operand(wu, jobs, og.rowmajor), od = operand(wd, jobs), oy = operand(dy, jobs);
  run_packs(jobs, P, st);
  const int Pi = parts_of(P, M);
  Operand oe = intermediate(M, H, Pi, x, 2), oh = intermediate(M, H, Pi, x);  // dg then du; h
  uint16_t* const e = (uint16_t*)oe.keep.data_ptr();
  const GradOut out{e, e + Pi * oe.s.plane, oh.keep.data_ptr(), oh.s.ld, oh.s.plane, (int)act, Pi == 2 ? 1 : 0};
  const bool through_memory = far(x, K) || (P == 1 && far(x, N));
  if (P == 1 && !through_memory) {
    Plan pl(bf16);
    const int a = pl.map(ox), b = pl.map(og), b2 = pl.map(ou), a3 = pl.map(oy), b3 = pl.map(od);
    pl.product(a3, oy, 1, b3, -1, od, 1, 256, 128, 0, 0, 0, 0, 2, 1);
    pl.product(a, ox, 1, b, b2, og, 0, 0, 256);
    set_tiles(pl.t, M, H, 128, 1, 1);
    if (bf16) run_dense<256, EpiGatedGrad<__nv_bfloat16>>(pl.maps, pl.t, out, st);
    else run_dense<256, EpiGatedGrad<__half>>(pl.maps, pl.t, out, st);
  } else {
    const int64_t ld_dh = (H + 3) / 4 * 4;  // columns past H come out as zeros
    Tensor dh = at::empty({M, ld_dh}, x.options().dtype(at::kFloat));
    project(bf16, oy, od, 1, dh, st);
    if (through_memory) {
      gate_through_memory(x, ox, og, ou, dh, H, out, st);
    } else {
      Plan pl(bf16);
      const int a = pl.map(ox), b = pl.map(og), b2 = pl.map(ou);
      auto go = [&](auto bn_tag) {
        constexpr int BN = decltype(bn_tag)::value;
        pl.product(a, ox, 1, b, b2, og, 0, 0, BN);
        set_tiles(pl.t, M, H, BN / 2, 1, 1);
        run_dense<BN, EpiGatedGradRead<BN>>(pl.maps, pl.t, {out, dh.data_ptr<float>(), ld_dh}, st);
      };
      if (gate_bn(x, M, H, K) == 256) go(std::integral_constant<int, 256>{});
      else go(std::integral_constant<int, 128>{});
    }
  }
  if (which & 1) {
    Plan pl(bf16);
    const int bn = store_bn(1, M, K, 2 * blocks_of(P, H));
    const int a = pl.map(oe), b = pl.map(og), c = pl.map(ou);
    for (int part = 0; part < 2; ++part) {
      pl.product(a, oe, 1, b, -1, og, 1, 0, bn, 0, 0, 0, 0, part);
      pl.product(a, oe, 1, c, -1, ou, 1, 0, bn, Pi, 0, 0, 0, part);
    }
    store_any(pl, bn, dx, 1, M, K, st);
  }
  if (which & 2) {
    Plan pl(bf16);
    const int bn = store_bn(2, K, H, blocks_of(P, M));
    const int a = pl.map(ox), b = pl.map(oe);
    pl.product(a, ox, 0, b, -1, oe, 0, 0, bn, 0, 0, 0, Pi);
    store_any(pl, bn, dgu, 2, K, H, st);
  }
  if (which & 4) {
    Plan pl(bf16);
    const int bn = store_bn(1, H, N, blocks_of(P, M));
    const int a = pl.map(oh), b = pl.map(oy);
    pl.product(a, oh, 0, b, -1, oy, 0, 0, bn);
    store_any(pl, bn, dwd, 1, H, N, st);
  }
  return {dx, dgu.select(0, 0), dgu.select(0, 1), dwd};
}

int64_t gated_ff_error_status(const Tensor& like) { return dense::take_error(like); }

}  // namespace nva

// Explicit kernels: tracing must not decompose them, their C++ would launch on tensors without memory.
TORCH_LIBRARY_FRAGMENT(nvalchemi, m) {
  m.def("gated_ff_fwd(Tensor x, Tensor w_gate, Tensor w_up, Tensor w_down, int act) -> Tensor", torch::dispatch(c10::DispatchKey::CompositeExplicitAutograd, &nva::gated_ff_fwd));
  m.def("gated_ff_bwd(Tensor dy, Tensor x, Tensor w_gate, Tensor w_up, Tensor w_down, int act, int which) -> (Tensor, Tensor, Tensor, Tensor)", torch::dispatch(c10::DispatchKey::CompositeExplicitAutograd, &nva::gated_ff_bwd));
  m.def("gated_ff_error_status(Tensor like) -> int", torch::dispatch(c10::DispatchKey::CompositeExplicitAutograd, &nva::gated_ff_error_status));
}
