// SPDX-License-Identifier: Apache-2.0
// Products of 16-bit matrices on the 5th-generation tensor cores, shared by the gated feed-forward block and the
// Newton-Schulz iteration:   acc[m, n] = sum over segments of  A_s[m, :] . B_s[n, :]   (fp32 accumulators in TMEM).
//
// A segment names the tensor maps of its operands, the plane (third coordinate) of each and the accumulator columns it adds
// to; a float32 operand is three bf16 planes and its product six segments, a sum of two products is two segments.  Either
// operand may be stored with the contraction axis contiguous (K-major) or the other one (MN-major): a 64 x 64 box of 16-bit
// values is 64 rows of 128 swizzled bytes in both cases, only the coordinates and the matrix descriptors differ, so no
// operand is transposed in memory.
//
// The tensor core cuts an accumulator to 24 bits after every instruction, towards zero: after n instructions a sum has lost
// about n / 3 of half a step, always in the same direction.  That is nothing beside a 16-bit result, and 1.1e-5 of a float32
// one of 6 x 1024 terms (measured).  So a float32 product adds its five small partial products first, while the sum is small,
// and deals the large one out over up to four accumulators that the epilogue adds in fp32; longer contraction axes are split
// over several tiles.
//
// One persistent CTA per SM: warp 0 loads tiles by TMA into a ring of stages, one lane of warp 1 issues tcgen05.mma
// (M = 128, K = 16 per instruction), warps 2..9 are the epilogue.  The accumulator is double buffered (2 x 256 TMEM columns),
// so the epilogue of a tile runs beside the products of the next one; products with several accumulators use all of the TMEM
// for one tile (their six passes hide the epilogue less, but it is a tenth of them).  Every wait is bounded; on expiry the error word is
// set, the roles leave their loops, the producer waits (bounded) for its copies in flight, and the TMEM is freed.
#pragma once
#include "common.cuh"
#include "convert.cuh"

#include <cuda.h>
#include <cudaTypedefs.h>

#include "tcgen05_utils.cuh"

namespace nva {
namespace dense {

constexpr int BM = 128, BK = 64, kChunk = 64 * 64 * 2;  // a chunk: 64 x 64 16-bit values, one TMA box
constexpr int kMaxSegs = 12, kMaxMaps = 6, kEpiWarps = 8;
constexpr int kThreads = 64 + 32 * kEpiWarps;

static __device__ int error_word;

struct Seg {
  int8_t a, b, b2;       // tensor maps; the second half of the B tile comes from b2
  int8_t a_mn, b_mn;     // 1: stored with the M / N axis contiguous
  int8_t group;          // accumulator group (0 or 1) of its columns
  int8_t spread;         // 1: dealt out over the group's accumulators, 0: added to the first of them
  int16_t col, n;        // accumulator column, columns written (instruction N)
  int za, zb;            // planes, plus batch * (za_step, zb_step)
  int za_step, zb_step;
  int nk;                // 64-wide blocks of the contraction axis
  int b2_off;            // n offset of the second half
  uint32_t idesc;
};

struct Tiles {
  int M, N;              // rows and columns of one output matrix
  int mt, nt, bn;        // tiles along each, columns of a tile
  int batches, splits, total;
  int lower;             // 1: symmetric output, only tiles on and below the diagonal
  int n_seg;
  int main_nk[2];        // nk of the spread segments of each group
  Seg seg[kMaxSegs];
};

struct alignas(64) Maps { CUtensorMap m[kMaxMaps]; };

struct TileAt { int m, n, batch, split; };

// The part of a segment's blocks that one of `splits` tiles of the same output takes.
__device__ __forceinline__ int split_at(int nk, int split, int splits) { return (int)((int64_t)nk * split / splits); }
// How many of a group's ACC accumulators the tile's products have written.
template <int ACC>
__device__ __forceinline__ int used_acc(const Tiles& t, const TileAt& at, int group) {
  if constexpr (ACC == 1) return 1;
  const int nk = t.main_nk[group];
  return min(ACC, split_at(nk, at.split + 1, t.splits) - split_at(nk, at.split, t.splits));
}

// Tiles of eight row blocks run together, column by column, so that concurrent CTAs share operand tiles in the L2.
__device__ __forceinline__ TileAt tile_at(const Tiles& t, int i) {
  TileAt r;
  const int per = t.lower ? t.mt * (t.mt + 1) / 2 : t.mt * t.nt;
  const int z = i / per;
  int j = i - z * per;
  r.batch = z % t.batches;
  r.split = z / t.batches;
  if (t.lower) {  // square tiles: row m holds m + 1 of them
    int m = (int)((sqrtf(8.f * (float)j + 1.f) - 1.f) * 0.5f);
    while ((m + 1) * (m + 2) / 2 <= j) ++m;
    while (m * (m + 1) / 2 > j) --m;
    r.m = m;
    r.n = j - m * (m + 1) / 2;
    return r;
  }
  constexpr int G = 8;
  const int band = j / (G * t.nt), in = j - band * G * t.nt;
  const int rows = min(G, t.mt - band * G);
  r.n = in / rows;
  r.m = band * G + in % rows;
  return r;
}

__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
      ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar)
      : "memory");
}

// 128-byte swizzle.  K-major: 8-row groups 1024 bytes apart.  MN-major: 8 contraction rows per 1024 bytes, 64-wide chunks of
// the M / N axis one TMA box (8192 bytes) apart.
__device__ __forceinline__ uint64_t desc16(uint32_t addr, bool mn) {
  return (uint64_t)((addr & 0x3FFFFu) >> 4) | (uint64_t)((mn ? kChunk : 0) >> 4) << 16 | (uint64_t)(1024u >> 4) << 32 |
         (uint64_t)1 << 46 | (uint64_t)2 << 61;
}
inline uint32_t idesc16(bool bf16, bool a_mn, bool b_mn, int n) {
  return (1u << 4) | ((bf16 ? 1u : 0u) << 7) | ((bf16 ? 1u : 0u) << 10) | ((a_mn ? 1u : 0u) << 15) | ((b_mn ? 1u : 0u) << 16) |
         ((uint32_t)(n >> 3) << 17) | ((uint32_t)(BM >> 4) << 24);
}
__device__ __forceinline__ void mma16(uint32_t d, uint64_t da, uint64_t db, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(d), "l"(da), "l"(db), "r"(idesc), "r"(acc)
      : "memory");
}

template <int BN> constexpr int stage_bytes() { return (BM / 64 + BN / 64) * kChunk; }
// ring + per-warp staging (32 rows of 128 bytes) + barriers, and slack for 1024-byte alignment
template <int BN, int STAGES> constexpr int smem_bytes() { return 1024 + STAGES * stage_bytes<BN>() + kEpiWarps * 4096 + 256; }

// One warp's 32 rows x (SLOTS * 16) bytes from registers (lane = row) to global memory in whole row pieces: through shared
// memory, 16-byte slots swizzled by row so that neither side has bank conflicts.  `cols_left`: elements of type T that exist
// from this piece's first column on.
template <typename T, int SLOTS>
__device__ __forceinline__ void store_piece(uint4* stage, const uint4 (&v)[SLOTS], T* dst, int64_t ld, int rows_left, int cols_left,
                                            bool vec_ok) {
  const int lane = threadIdx.x & 31;
  constexpr int PER = 16 / (int)sizeof(T), RPI = 32 / SLOTS;
  if (cols_left <= 0) return;  // the same for the whole warp
#pragma unroll
  for (int j = 0; j < SLOTS; ++j) stage[lane * SLOTS + (j ^ (lane & (SLOTS - 1)))] = v[j];
  __syncwarp();
  const int slot = lane % SLOTS, r0 = lane / SLOTS;
#pragma unroll
  for (int i = 0; i < SLOTS; ++i) {
    const int r = i * RPI + r0;
    const uint4 val = stage[r * SLOTS + (slot ^ (r & (SLOTS - 1)))];
    const int left = cols_left - slot * PER;
    if (r < rows_left && left > 0) {
      T* p = dst + (int64_t)r * ld + slot * PER;
      if (vec_ok && left >= PER) {
        *reinterpret_cast<uint4*>(p) = val;
      } else {
        const T* e = reinterpret_cast<const T*>(&val);
#pragma unroll
        for (int k = 0; k < PER; ++k)
          if (k < left) p[k] = e[k];
      }
    }
  }
  __syncwarp();
}

__device__ __forceinline__ uint32_t pack2(float a, float b, __half) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pack2(float a, float b, __nv_bfloat16) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// 32 fp32 values of a row as T: 4 (16-bit) or 8 (32-bit) 16-byte slots.
template <typename T> struct Slots { static constexpr int n = (int)sizeof(T) * 2; };
template <typename T>
__device__ __forceinline__ void pack32(const float (&v)[32], uint4 (&o)[Slots<T>::n]) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      o[j] = make_uint4(__float_as_uint(v[4 * j]), __float_as_uint(v[4 * j + 1]), __float_as_uint(v[4 * j + 2]),
                        __float_as_uint(v[4 * j + 3]));
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      o[j] = make_uint4(pack2(v[8 * j], v[8 * j + 1], T{}), pack2(v[8 * j + 2], v[8 * j + 3], T{}),
                        pack2(v[8 * j + 4], v[8 * j + 5], T{}), pack2(v[8 * j + 6], v[8 * j + 7], T{}));
  }
}

// A float32 value as a sum of three bf16 values (8 + 8 + 8 bits): the remainders are exact in fp32.  Where the first would
// round up to infinity all are cut instead, so that no partial sum passes the value; infinities and NaN stay in the first
// plane alone.
__device__ __forceinline__ void split3(float v, float& p0, float& p1, float& p2) {
  p0 = __bfloat162float(__float2bfloat16_rn(v));
  p1 = __bfloat162float(__float2bfloat16_rn(v - p0));
  if (isinf(p0)) {
    p0 = __bfloat162float(__float2bfloat16_rz(v));
    p1 = __bfloat162float(__float2bfloat16_rz(v - p0));
  }
  p2 = v - p0 - p1;
  if (!isfinite(v)) { p0 = v; p1 = 0.f; p2 = 0.f; }
}

// 32 columns of the sum of a group's accumulators, STRIDE columns apart.
template <int ACC, int STRIDE>
__device__ __forceinline__ void acc_ld32(uint32_t tm, float (&v)[32], int used) {
  tmem_ld32(tm, v);
  if constexpr (ACC > 1) {
    for (int a = 1; a < used; ++a) {
      float w[32];
      tmem_ld32(tm + a * STRIDE, w);
#pragma unroll
      for (int j = 0; j < 32; ++j) v[j] += w[j];
    }
  }
}

// Epi::kAcc accumulators kStride columns apart, Epi::Params, Epi::run(params, tiles, tile, tmem (lane quarter added), first row of the warp, half, stage).
template <int BN, int STAGES, typename Epi>
__global__ void __launch_bounds__(kThreads, 1)
    dense_kernel(const __grid_constant__ Maps maps, const __grid_constant__ Tiles t, const __grid_constant__ typename Epi::Params ep) {
  extern __shared__ uint8_t smem_raw[];
  constexpr uint32_t STAGE = stage_bytes<BN>();
  constexpr int ACC = Epi::kAcc, BUFS = ACC == 1 ? 2 : 1;
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* const generic = smem_raw + (base - smem_u32(smem_raw));
  const uint32_t bar0 = base + STAGES * STAGE + kEpiWarps * 4096;
  auto full = [&](int s) { return bar0 + 8u * s; };
  auto empty = [&](int s) { return bar0 + 8u * (STAGES + s); };
  auto acc_full = [&](int s) { return bar0 + 8u * (2 * STAGES + s); };
  auto acc_empty = [&](int s) { return bar0 + 8u * (2 * STAGES + 2 + s); };
  const uint32_t slot = bar0 + 8u * (2 * STAGES + 4);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int* const err = &error_word;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) { mbar_init(full(s), 1); mbar_init(empty(s), 1); }
    for (int s = 0; s < 2; ++s) { mbar_init(acc_full(s), 1); mbar_init(acc_empty(s), kEpiWarps); }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(slot), "r"(512u) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  uint32_t tmem;
  asm volatile("ld.shared.b32 %0, [%1];" : "=r"(tmem) : "r"(slot));

  // The segment is copied out of the parameters once: the compiler may not keep what it read there over an asm statement that
  // clobbers memory, and both loops below would wait for constant loads before every instruction (43 % of the tensor pipe).
  if (warp == 0) {
    // lane c loads chunk c of a stage: the first two are A's, the others B's
    int it = 0;
    bool ok = true;
    for (int i = blockIdx.x; i < t.total && ok; i += gridDim.x) {
      const TileAt at = tile_at(t, i);
      for (int sg = 0; sg < t.n_seg && ok; ++sg) {
        const Seg s = t.seg[sg];
        const int lo = split_at(s.nk, at.split, t.splits), hi = split_at(s.nk, at.split + 1, t.splits);
        const int chunks = s.n / 64, half = (chunks + 1) / 2, c = lane - BM / 64;
        const bool mine = c < chunks, is_a = c < 0, second = c >= half;
        const CUtensorMap* const map = &maps.m[is_a ? s.a : second ? s.b2 : s.b];
        const int mn = is_a ? at.m * BM + 64 * lane : at.n * t.bn + 64 * (second ? c - half : c) + (second ? s.b2_off : 0);
        const int z = is_a ? s.za + at.batch * s.za_step : s.zb + at.batch * s.zb_step;
        const bool mn_first = is_a ? s.a_mn : s.b_mn;
        const uint32_t bytes = (uint32_t)(BM / 64 + chunks) * kChunk;
        for (int kb = lo; kb < hi; ++kb, ++it) {
          const int st = it % STAGES, k0 = kb * BK;
          if (!mbar_wait(empty(st), ((it / STAGES) & 1) ^ 1, err, 11)) ok = false;
          if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
          if (lane == 0) mbar_expect_tx(full(st), bytes);
          __syncwarp();
          if (mine) tma_load_3d(base + st * STAGE + lane * kChunk, map, mn_first ? mn : k0, mn_first ? k0 : mn, z, full(st));
        }
      }
    }
    if (!ok)  // gave up: the copies in flight must have landed before the CTA's shared memory is given back
      for (int j = it > STAGES ? it - STAGES : 0; j < it; ++j) mbar_wait(full(j % STAGES), (j / STAGES) & 1, err, 14);
  } else if (warp == 1) {
    if (lane == 0) {
      int it = 0, n_tile = 0;
      bool ok = true;
      for (int i = blockIdx.x; i < t.total && ok; i += gridDim.x, ++n_tile) {
        const TileAt at = tile_at(t, i);
        const int as = BUFS == 2 ? n_tile & 1 : 0;
        if (!mbar_wait(acc_empty(as), ((n_tile / BUFS) & 1) ^ 1, err, 12)) break;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        uint32_t started = 0;  // accumulators that hold something of this tile
        for (int sg = 0; sg < t.n_seg && ok; ++sg) {
          const Seg s = t.seg[sg];
          const int lo = split_at(s.nk, at.split, t.splits), hi = split_at(s.nk, at.split + 1, t.splits);
          const uint64_t da0 = desc16(base, s.a_mn), db0 = desc16(base + (BM / 64) * kChunk, s.b_mn);
          const uint32_t ka = (s.a_mn ? 2048 : 32) >> 4, kb_step = (s.b_mn ? 2048 : 32) >> 4;
          const uint32_t d0 = tmem + as * 256 + s.col;
          for (int kb = lo; kb < hi; ++kb, ++it) {
            const int st = it % STAGES;
            if (!mbar_wait(full(st), (it / STAGES) & 1, err, 13)) { ok = false; break; }
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const uint64_t da = da0 + (uint32_t)(st * (int)(STAGE >> 4)), db = db0 + (uint32_t)(st * (int)(STAGE >> 4));
            const int j = ACC > 1 && s.spread ? (kb - lo) % ACC : 0;
            const uint32_t d = d0 + j * Epi::kStride, bit = 1u << (s.group * ACC + j);
            const uint32_t acc = (started & bit) != 0 ? 1u : 0u;
            started |= bit;
#pragma unroll
            for (int k = 0; k < BK / 16; ++k) mma16(d, da + k * ka, db + k * kb_step, s.idesc, k == 0 ? acc : 1u);
            umma_commit(empty(st));
          }
        }
        umma_commit(acc_full(as));
      }
    }
  } else {
    const int w = warp - 2, q = warp & 3, half = w >> 2;  // q: the TMEM lanes this warp may read
    uint4* const stage = reinterpret_cast<uint4*>(generic + STAGES * STAGE + w * 4096);
    int n_tile = 0;
    for (int i = blockIdx.x; i < t.total; i += gridDim.x, ++n_tile) {
      const TileAt at = tile_at(t, i);
      const int as = BUFS == 2 ? n_tile & 1 : 0;
      if (!mbar_wait(acc_full(as), (n_tile / BUFS) & 1, err, 15)) break;
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      Epi::run(ep, t, at, tmem + as * 256 + ((uint32_t)(q * 32) << 16), at.m * BM + q * 32, half, stage);
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive(acc_empty(as));
    }
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
}

// out[batch][split][M][N] = alpha * acc, as T.
template <typename T, int BN, int ACC>
struct EpiStore {
  static constexpr int kAcc = ACC, kStride = BN;
  static_assert(ACC == 1 || ACC * BN <= 512, "dense: accumulators exceed the TMEM");
  struct Params { T* out; int64_t ld, batch_stride, split_stride; float alpha; };
  static __device__ __forceinline__ void run(const Params& p, const Tiles& t, const TileAt& at, uint32_t tm, int row0, int half,
                                             uint4* stage) {
    T* out = p.out + at.batch * p.batch_stride + at.split * p.split_stride;
    const bool vec_ok = p.ld % (16 / (int)sizeof(T)) == 0 && (reinterpret_cast<uintptr_t>(out) & 15) == 0;
    const int used = used_acc<ACC>(t, at, 0);
#pragma unroll 1
    for (int cb = 0; cb < BN / 64; ++cb) {
      const int c = half * (BN / 2) + cb * 32, n0 = at.n * BN + c;
      float v[32];
      acc_ld32<ACC, BN>(tm + c, v, used);
#pragma unroll
      for (int j = 0; j < 32; ++j) v[j] *= p.alpha;
      uint4 o[Slots<T>::n];
      pack32<T>(v, o);
      store_piece<T, Slots<T>::n>(stage, o, out + (int64_t)row0 * p.ld + n0, p.ld, t.M - row0, t.N - n0, vec_ok);
    }
  }
};

// ---- host side -------------------------------------------------------------------------------------
inline PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    C10_CUDA_CHECK(cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q));
    TORCH_CHECK(p != nullptr && q == cudaDriverEntryPointSuccess, "cuTensorMapEncodeTiled is not available");
    return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
  }();
  return fn;
}

// A stored 16-bit matrix: `outer` rows of `inner` contiguous elements, `ld` elements apart, in `planes` planes.
struct Stored {
  const void* p = nullptr;
  int64_t inner = 0, outer = 0, ld = 0, planes = 1, plane = 0;
};

inline void put_map(Maps& maps, int i, const Stored& s) {
  TORCH_CHECK(i < kMaxMaps, "dense: too many tensor maps");
  const int64_t ld = s.outer > 1 ? s.ld : (s.inner + 7) / 8 * 8;
  const int64_t plane = s.planes > 1 ? s.plane : ld * s.outer;
  TORCH_CHECK(s.inner > 0 && s.outer > 0 && ld % 8 == 0 && plane % 8 == 0 && (reinterpret_cast<uintptr_t>(s.p) & 15) == 0,
              "dense: operand rows must lie on 16-byte boundaries");
  TORCH_CHECK(s.inner < (1ll << 31) && s.outer < (1ll << 31) && s.planes < (1ll << 31) && plane < (1ll << 38), "dense: operand too large");
  cuuint64_t dims[3] = {(cuuint64_t)s.inner, (cuuint64_t)s.outer, (cuuint64_t)s.planes};
  cuuint64_t strides[2] = {(cuuint64_t)ld * 2, (cuuint64_t)plane * 2};
  cuuint32_t box[3] = {64, 64, 1}, es[3] = {1, 1, 1};
  CUresult r = encode_fn()(&maps.m[i], CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(s.p), dims, strides, box, es,
                           CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                           CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  TORCH_CHECK(r == CUDA_SUCCESS, "cuTensorMapEncodeTiled failed with code ", (int)r);
}

inline int sm_count() {
  static int n = [] {
    int dev = 0, v = 0;
    C10_CUDA_CHECK(cudaGetDevice(&dev));
    C10_CUDA_CHECK(cudaDeviceGetAttribute(&v, cudaDevAttrMultiProcessorCount, dev));
    return v;
  }();
  return n;
}

inline void set_tiles(Tiles& t, int64_t M, int64_t N, int bn, int64_t batches, int splits, bool lower = false) {
  t.M = (int)M; t.N = (int)N; t.bn = bn;
  t.mt = (int)((M + BM - 1) / BM); t.nt = (int)((N + bn - 1) / bn);
  t.batches = (int)batches; t.splits = splits; t.lower = lower ? 1 : 0;
  const int64_t per = lower ? (int64_t)t.mt * (t.mt + 1) / 2 : (int64_t)t.mt * t.nt;
  TORCH_CHECK(per * batches * splits < (1ll << 31), "dense: too many tiles");
  t.total = (int)(per * batches * splits);
}

template <int BN, int STAGES, typename Epi>
void run_dense(const Maps& maps, const Tiles& t, const typename Epi::Params& ep, cudaStream_t st) {
  constexpr int smem = smem_bytes<BN, STAGES>();
  static_assert(smem <= 227 * 1024, "dense: stages exceed shared memory");
  // set on every call: the attribute belongs to the current device's context
  C10_CUDA_CHECK(cudaFuncSetAttribute(dense_kernel<BN, STAGES, Epi>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
  dense_kernel<BN, STAGES, Epi><<<std::min(t.total, sm_count()), kThreads, smem, st>>>(maps, t, ep);
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}

}  // namespace dense
}  // namespace nva
