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
// The tensor core cuts what it adds to an accumulator towards zero: where all terms have one sign, an instruction loses up to
// 1.7 half steps of the sum so far (2^-24 of it; measured: 1.7e-3 of a sum of 16,384 instructions, 6.5e-3 of 65,536, always in the
// same direction).  So a float32 product adds its five small partial products first, while the sum is small, and deals the large
// one out over up to four accumulators that the epilogue adds in fp32.  max_blocks() below says how much one accumulator may
// take; a longer contraction axis is split over several tiles, whose partial sums are added in fp32.
//
// One persistent CTA per SM: warp 0 loads tiles by TMA into a ring of stages, one lane of warp 1 issues tcgen05.mma
// (K = 16 per instruction), warps 2..9 are the epilogue (16 warps
// leave 96 registers a thread and were slower).  The accumulator is double buffered (2 x 256 TMEM columns), so the
// epilogue of a tile runs beside the products of the next one; products with several accumulators use all of the TMEM for one
// tile (their six passes hide the epilogue less, but it is a tenth of them).
//
// Tiles of more than 128 rows are worked on by pairs of CTAs (cta_group::2): 256 rows, each CTA holds its 128 rows of A, half
// of the tile of B and 128 rows of the accumulator.  What bounds one CTA by itself is shared memory: at 128 x 256 a 64-wide
// block writes 48 KB and reads 48 KB, at the 117 bytes a clock it reaches 450 ns (1370 TFLOP/s at 18944 x 4096 x 4096), while
// the instructions need 320 ns; an instruction of 128 or 64 columns needs 195 ns whichever it is.  A pair writes 32 KB and reads
// 32 KB per CTA.
//
// Every wait is bounded; on expiry the error word is set, the products stop, the producer waits (bounded) for its copies in
// flight, the epilogue stores NaN for this tile and the CTA's remaining ones, and the TMEM is freed.
#pragma once
#include "common.cuh"
#include "convert.cuh"

#include <cuda.h>
#include <cudaTypedefs.h>

#include "tcgen05_utils.cuh"

namespace nva {
namespace dense {

constexpr int BM = 128, BK = 64, kChunk = 64 * 64 * 2;  // a chunk: 64 x 64 16-bit values, one TMA box
constexpr int kMaxSegs = 12, kMaxMaps = 6, kStaging = 32768;  // bytes of staging, shared by the epilogue's warps
constexpr int kEpiWarps = 8, kThreads = 32 * (2 + kEpiWarps);

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
  int bm;                // rows of a tile: 128, or 256 for a pair of CTAs
  int batches, splits, total;
  int split0;            // the first of the launch's splits
  int lower;             // symmetric output, only tiles that reach the diagonal or lie below it: bm / bn, else 0
  int n_seg;
  int main_nk[2];        // nk of the spread segments of each group
  Seg seg[kMaxSegs];
};

struct alignas(64) Maps { CUtensorMap m[kMaxMaps]; int n = 0; };

struct TileAt { int m, n, batch, split, seq; };  // seq: the CTA's how-manieth tile

// The part of a segment's blocks that one of `splits` tiles of the same output takes.
__device__ __forceinline__ int split_at(int nk, int split, int splits) {
  return splits == 1 ? nk * split : (int)((int64_t)nk * split / splits);
}
// How many of a group's ACC accumulators the tile's products have written.
template <int ACC>
__device__ __forceinline__ int used_acc(const Tiles& t, const TileAt& at, int group) {
  if constexpr (ACC == 1) return 1;
  const int nk = t.main_nk[group];
  return min(ACC, split_at(nk, at.split + 1, t.splits) - split_at(nk, at.split, t.splits));
}

// Tiles of eight row blocks run together, column by column, so that concurrent CTAs share operand tiles in the L2.
__device__ __forceinline__ TileAt tile_at(const Tiles& t, int i, int seq) {
  TileAt r;
  r.seq = seq;
  const int per = t.lower ? t.lower * (t.mt * (t.mt + 1) / 2) : t.mt * t.nt;
  const int z = i / per;
  const int j = i - z * per;
  r.batch = z % t.batches;
  r.split = t.split0 + z / t.batches;
  if (t.lower) {  // row m holds lower * (m + 1) tiles
    const int k = j / t.lower;
    int m = (int)((sqrtf(8.f * (float)k + 1.f) - 1.f) * 0.5f);
    while ((m + 1) * (m + 2) / 2 <= k) ++m;
    while (m * (m + 1) / 2 > k) --m;
    r.m = m;
    r.n = j - t.lower * (m * (m + 1) / 2);
    return r;
  }
  constexpr int G = 8;
  const int band = j / (G * t.nt), in = j - band * G * t.nt;
  const int rows = min(G, t.mt - band * G);
  r.n = in / rows;
  r.m = band * G + in % rows;
  return r;
}

// PAIR: the barrier may be the other CTA's (a shared::cluster address).
template <bool PAIR>
__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar) {
  if constexpr (PAIR)
    asm volatile(
        "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
        ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar)
        : "memory");
  else
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
        ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar)
        : "memory");
}

// 128-byte swizzle.  K-major: 8-row groups 1024 bytes apart.  MN-major: 8 contraction rows per 1024 bytes, 64-wide chunks of
// the M / N axis one TMA box (8192 bytes) apart.
__device__ __forceinline__ uint64_t desc16(uint32_t addr, bool mn, uint32_t chunk = kChunk) {
  return (uint64_t)((addr & 0x3FFFFu) >> 4) | (uint64_t)((mn ? chunk : 0) >> 4) << 16 | (uint64_t)(1024u >> 4) << 32 |
         (uint64_t)1 << 46 | (uint64_t)2 << 61;
}
__host__ __device__ constexpr uint32_t idesc16(bool bf16, bool a_mn, bool b_mn, int n, int m) {
  return (1u << 4) | ((bf16 ? 1u : 0u) << 7) | ((bf16 ? 1u : 0u) << 10) | ((a_mn ? 1u : 0u) << 15) | ((b_mn ? 1u : 0u) << 16) |
         ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}
template <bool PAIR>
__device__ __forceinline__ void mma16(uint32_t d, uint64_t da, uint64_t db, uint32_t idesc, uint32_t acc) {
  if constexpr (PAIR)
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(d), "l"(da), "l"(db), "r"(idesc), "r"(acc)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(d), "l"(da), "l"(db), "r"(idesc), "r"(acc)
        : "memory");
}

// A stage of one CTA: 128 rows of A and the tile of B, or half of it in a pair.
template <int BN, bool PAIR> constexpr int stage_bytes() { return (BM / 64 + BN / (PAIR ? 128 : 64)) * kChunk; }
template <int BN, bool PAIR> constexpr int stage_count() { return 196608 / stage_bytes<BN, PAIR>(); }
// ring + staging + barriers, and slack for 1024-byte alignment
template <int BN, bool PAIR> constexpr int smem_bytes() { return 1024 + stage_count<BN, PAIR>() * stage_bytes<BN, PAIR>() + kStaging + 512; }

// 16-byte slots of a staged row are turned by its number, so that eight consecutive rows' same slots lie in different banks.
template <int SLOTS>
__device__ __forceinline__ int turn_of(int row) { return (SLOTS == 8 ? row : SLOTS == 4 ? row >> 1 : row >> 2) & (SLOTS - 1); }

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
  for (int j = 0; j < SLOTS; ++j) stage[lane * SLOTS + (j ^ turn_of<SLOTS>(lane))] = v[j];
  __syncwarp();
  if (vec_ok && cols_left >= SLOTS * PER) {
    const int slot = lane % SLOTS, r0 = lane / SLOTS;
#pragma unroll
    for (int i = 0; i < SLOTS; ++i) {
      const int r = i * RPI + r0;
      if (r < rows_left)
        *reinterpret_cast<uint4*>(dst + (int64_t)r * ld + slot * PER) = stage[r * SLOTS + (slot ^ turn_of<SLOTS>(r))];
    }
  } else {  // rows off the 16-byte boundaries, or the last columns: a row at a time, an element a lane
    const T* const e = reinterpret_cast<const T*>(stage);
    constexpr int W = SLOTS * PER;  // 32 or 64 elements
#pragma unroll
    for (int c = 0; c < W; c += 32) {
      const int j = c + lane, slot = j / PER, k = j % PER;
#pragma unroll 8
      for (int r = 0; r < 32; ++r)
        if (r < rows_left && j < cols_left) dst[(int64_t)r * ld + j] = e[(r * SLOTS + (slot ^ turn_of<SLOTS>(r))) * PER + k];
    }
  }
  __syncwarp();
}

// The way back: 32 rows x (SLOTS * 16) bytes from global memory in whole row pieces (rows on 16-byte boundaries), then, through
// shared memory, a row a lane.  Row by row from global memory every lane would touch a cache line of its own: 4000 clocks for
// three pieces of eight warps.
template <typename T, int SLOTS>
__device__ __forceinline__ void fetch_piece(uint4 (&raw)[SLOTS], const T* src, int64_t ld, int rows_left, int cols_left) {
  const int lane = threadIdx.x & 31, slot = lane % SLOTS, r0 = lane / SLOTS;
  constexpr int PER = 16 / (int)sizeof(T), RPI = 32 / SLOTS;
#pragma unroll
  for (int i = 0; i < SLOTS; ++i) {
    const int r = i * RPI + r0;
    raw[i] = r < rows_left && slot * PER < cols_left ? *reinterpret_cast<const uint4*>(src + (int64_t)r * ld + slot * PER) : make_uint4(0, 0, 0, 0);
  }
}
template <int SLOTS>
__device__ __forceinline__ void turn_piece(uint4* stage, uint4 (&raw)[SLOTS]) {
  const int lane = threadIdx.x & 31, slot = lane % SLOTS, r0 = lane / SLOTS;
  constexpr int RPI = 32 / SLOTS;
#pragma unroll
  for (int i = 0; i < SLOTS; ++i) {
    const int r = i * RPI + r0;
    stage[r * SLOTS + (slot ^ turn_of<SLOTS>(r))] = raw[i];
  }
  __syncwarp();
#pragma unroll
  for (int j = 0; j < SLOTS; ++j) raw[j] = stage[lane * SLOTS + (j ^ turn_of<SLOTS>(lane))];
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

// Two float32 values as exact sums of three bf16 values each, p[i] holding the i-th parts (the first value's in the low half).
// The parts are rounded to nearest: what a product of two values leaves out (second times third parts, third times third) is then
// at most 2^-24 of it and of either sign, against 2^-21 of one sign for parts cut off towards zero.  Without branches: 16 of these
// run side by side.  First parts of values past the largest bf16 number are held at it; infinities and NaN are in the other two.
__device__ __forceinline__ void split3(float a, float b, uint32_t (&p)[3]) {
  constexpr float kTop = 3.3895313e38f;  // the largest bf16 number
  p[0] = pack2(fminf(fmaxf(a, -kTop), kTop), fminf(fmaxf(b, -kTop), kTop), __nv_bfloat16{});
#pragma unroll
  for (int i = 1; i < 3; ++i) {
    a -= __uint_as_float(p[i - 1] << 16);
    b -= __uint_as_float(p[i - 1] & 0xffff0000u);
    p[i] = pack2(a, b, __nv_bfloat16{});
  }
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

// NaN in `cols` columns of a warp's 32 rows.
template <typename T>
__device__ __forceinline__ void fill_nan(T* dst, int64_t ld, int rows_left, int cols_left, int cols) {
  const int row = threadIdx.x & 31;
  if (row >= rows_left) return;
#pragma unroll 1
  for (int c = 0; c < min(cols, cols_left); ++c) dst[row * ld + c] = narrow<T>(__int_as_float(0x7fc00000));
}

// NaN in an epilogue warp's part of the tiles from `i` on: a function of its own, so that the kernel keeps its registers.
template <int CTAS, typename Epi>
__device__ __noinline__ void poison_tiles(const Tiles& t, const typename Epi::Params& ep, int i, int step, int rank, int w) {
  for (; i < t.total; i += step) {
    const TileAt at = tile_at(t, i, 0);
    Epi::poison(ep, t, at, at.m * (BM * CTAS) + rank * BM + ((w + 2) & 3) * 32, w >> 2);
  }
}

// Epi::kAcc accumulators per column group, kStride columns apart; Epi::kLate: see below; Epi::Params; Epi::Pre: what
// Epi::prefetch(params, tiles, tile, first row of the warp, share of the columns, pre) reads before the tile's products are done;
// Epi::run(params, tiles, tile, tmem (lane quarter added), first row, share, stage, pre); Epi::poison(params, tiles, tile, first
// row, share): NaN in what `run` would store.
//
// kLate: a tile fills TMEM columns 0..383, group 0 in 0..255 and group 1 (whose segments come first) in the 128 columns after
// those, in turns with the last 128, so that the next tile's group 1 is formed while the epilogue still reads this tile.
template <int BN, bool PAIR, typename Epi>
__global__ void __launch_bounds__(kThreads, 1)
    dense_kernel(const __grid_constant__ Maps maps, const __grid_constant__ Tiles t, const __grid_constant__ typename Epi::Params ep) {
  extern __shared__ uint8_t smem_raw[];
  constexpr int STAGES = stage_count<BN, PAIR>();
  constexpr uint32_t STAGE = stage_bytes<BN, PAIR>();
  constexpr int ACC = Epi::kAcc, BUFS = ACC == 1 && !Epi::kLate ? 2 : 1, CTAS = PAIR ? 2 : 1;
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* const generic = smem_raw + (base - smem_u32(smem_raw));
  const uint32_t bar0 = base + STAGES * STAGE + kStaging;
  auto full = [&](int s) { return bar0 + 8u * s; };
  auto empty = [&](int s) { return bar0 + 8u * (STAGES + s); };
  auto acc_full = [&](int s) { return bar0 + 8u * (2 * STAGES + s); };
  auto acc_empty = [&](int s) { return bar0 + 8u * (2 * STAGES + 2 + s); };
  const uint32_t slot = bar0 + 8u * (2 * STAGES + 4);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = PAIR ? cluster_rank() : 0;
  const int first_tile = blockIdx.x / CTAS, tile_step = gridDim.x / CTAS;
  int unformed = t.total;  // an epilogue warp's first tile that was not formed
  int* const err = &error_word;

  // The next kernel of the chain may start on idle SMs and set itself up; it waits below until this one is done.
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (warp == 0 && lane < maps.n) asm volatile("prefetch.tensormap [%0];" ::"l"(&maps.m[lane]) : "memory");
  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) { mbar_init(full(s), 1); mbar_init(empty(s), 1); }
    for (int s = 0; s < 2; ++s) { mbar_init(acc_full(s), 1); mbar_init(acc_empty(s), kEpiWarps * CTAS); }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (warp == 1) {
    if constexpr (PAIR) {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(slot), "r"(512u) : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    } else {
      asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(slot), "r"(512u) : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if constexpr (PAIR) cluster_sync();  // the other CTA's barriers are ready
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  uint32_t tmem;
  asm volatile("ld.shared.b32 %0, [%1];" : "=r"(tmem) : "r"(slot));
  asm volatile("griddepcontrol.wait;" ::: "memory");  // nothing above reads or writes global memory

  // The segment is copied out of the parameters once: the compiler may not keep what it read there over an asm statement that
  // clobbers memory, and both loops below would wait for constant loads before every instruction (43 % of the tensor pipe).
  if (warp == 0) {
    if (lane == 0) {
      int st = 0, seq = 0, issued = 0;
      uint32_t phase = 1;
      bool ok = true;
      for (int i = first_tile; i < t.total && ok; i += tile_step, ++seq) {
        const TileAt at = tile_at(t, i, seq);
        for (int sg = 0; sg < t.n_seg && ok; ++sg) {
          const Seg s = t.seg[sg];
          const int lo = split_at(s.nk, at.split, t.splits), hi = split_at(s.nk, at.split + 1, t.splits);
          // chunks of B in this CTA; the tile's second half (b2) is the second CTA's, or the second half of this one's chunks
          const int chunks = s.n / (64 * CTAS), half = PAIR ? 0 : (chunks + 1) / 2;
          const CUtensorMap* const ma = &maps.m[s.a];
          const CUtensorMap* const mb = &maps.m[PAIR && rank == 1 ? s.b2 : s.b];
          const CUtensorMap* const mb2 = &maps.m[s.b2];
          const int m0 = at.m * (BM * CTAS) + (int)rank * BM, n0 = at.n * t.bn + (PAIR && rank == 1 ? s.b2_off : 0), n2 = at.n * t.bn + s.b2_off;
          const int za = s.za + at.batch * s.za_step, zb = s.zb + at.batch * s.zb_step;
          const bool a_mn = s.a_mn, b_mn = s.b_mn;
          const uint32_t bytes = (uint32_t)(BM / 64 + chunks) * kChunk * CTAS;
          for (int kb = lo; kb < hi; ++kb) {
            if (!mbar_wait(empty(st), phase, err, 11)) { ok = false; break; }
            const uint32_t bar = PAIR ? map_to_rank(full(st), 0) : full(st);
            if (rank == 0) mbar_expect_tx(full(st), bytes);
            const uint32_t dst = base + st * STAGE;
            const int k0 = kb * BK;
#pragma unroll
            for (int c = 0; c < BM / 64; ++c)
              tma_load_3d<PAIR>(dst + c * kChunk, ma, a_mn ? m0 + 64 * c : k0, a_mn ? k0 : m0 + 64 * c, za, bar);
#pragma unroll
            for (int c = 0; c < BN / (64 * CTAS); ++c)
              if (c < chunks) {
                const bool second = !PAIR && c >= half;
                const int mn = second ? n2 + 64 * (c - half) : n0 + 64 * c;
                tma_load_3d<PAIR>(dst + (BM / 64 + c) * kChunk, second ? mb2 : mb, b_mn ? mn : k0, b_mn ? k0 : mn, zb, bar);
              }
            ++issued;
            if (++st == STAGES) { st = 0; phase ^= 1; }
          }
        }
      }
      if (!ok && rank == 0)  // gave up: the copies in flight (both CTAs') must have landed before the shared memory is given back
        for (int j = issued > STAGES ? issued - STAGES : 0; j < issued; ++j) mbar_wait(full(j % STAGES), (j / STAGES) & 1, err, 14);
    }
  } else if (warp == 1) {
    if (lane == 0 && rank == 0) {
      int st = 0, seq = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int i = first_tile; i < t.total && ok; i += tile_step, ++seq) {
        const TileAt at = tile_at(t, i, seq);
        const int as = BUFS == 2 ? seq & 1 : 0;
        bool free = false;     // the epilogue has left this tile's accumulators
        uint32_t started = 0;  // accumulators that hold something of this tile
        for (int sg = 0; sg < t.n_seg && ok; ++sg) {
          const Seg s = t.seg[sg];
          if (!free && (!Epi::kLate || s.group == 0)) {
            ok = mbar_wait(acc_empty(as), ((seq / BUFS) & 1) ^ 1, err, 12);
            if (!ok) break;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            free = true;
          }
          const int lo = split_at(s.nk, at.split, t.splits), hi = split_at(s.nk, at.split + 1, t.splits);
          const uint64_t da0 = desc16(base, s.a_mn), db0 = desc16(base + (BM / 64) * kChunk, s.b_mn);
          const uint32_t ka = (s.a_mn ? 2048 : 32) >> 4, kb_step = (s.b_mn ? 2048 : 32) >> 4;
          const uint32_t d0 = tmem + as * 256 + s.col + (Epi::kLate && s.group == 1 ? (seq & 1) * 128 : 0);
          for (int kb = lo; kb < hi; ++kb) {
            if (!mbar_wait(full(st), phase, err, 13)) { ok = false; break; }
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const uint64_t da = da0 + (uint32_t)(st * (int)(STAGE >> 4)), db = db0 + (uint32_t)(st * (int)(STAGE >> 4));
            const int j = ACC > 1 && s.spread ? (kb - lo) % ACC : 0;
            const uint32_t d = d0 + j * Epi::kStride, bit = 1u << (s.group * ACC + j);
            const uint32_t acc = (started & bit) != 0 ? 1u : 0u;
            started |= bit;
#pragma unroll
            for (int k = 0; k < BK / 16; ++k) mma16<PAIR>(d, da + k * ka, db + k * kb_step, s.idesc, k == 0 ? acc : 1u);
            if constexpr (PAIR) umma_commit_pair(empty(st));
            else umma_commit(empty(st));
            if (++st == STAGES) { st = 0; phase ^= 1; }
          }
        }
        if (!ok) break;  // the tile is not complete
        if constexpr (PAIR) umma_commit_pair(acc_full(as));
        else umma_commit(acc_full(as));
      }
    }
  } else {
    const int w = warp - 2, q = warp & 3;  // q: the TMEM lanes this warp may read
    const int part = w >> 2;                        // its half of the columns
    uint4* const stage = reinterpret_cast<uint4*>(generic + STAGES * STAGE + w * (kStaging / kEpiWarps));
    int seq = 0, i = first_tile;
    for (; i < t.total; i += tile_step, ++seq) {
      const TileAt at = tile_at(t, i, seq);
      const int as = BUFS == 2 ? seq & 1 : 0, row0 = at.m * (BM * CTAS) + (int)rank * BM + q * 32;
      typename Epi::Pre pre;
      Epi::prefetch(ep, t, at, row0, part, pre);
      if (!__all_sync(0xffffffffu, mbar_wait(acc_full(as), (seq / BUFS) & 1, err, 15))) break;
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      Epi::run(ep, t, at, tmem + as * 256 + ((uint32_t)(q * 32) << 16), row0, part, stage, pre);
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      __syncwarp();
      if (lane == 0) {
        if constexpr (PAIR) mbar_arrive_cluster(map_to_rank(acc_empty(as), 0));
        else mbar_arrive(acc_empty(as));
      }
    }
    unformed = i;
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if constexpr (PAIR) cluster_sync();  // nothing of the pair is under way any more
  if (warp == 1) {
    if constexpr (PAIR) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
    else asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
  }
  if (unformed < t.total) poison_tiles<CTAS, Epi>(t, ep, unformed, tile_step, (int)rank, warp - 2);
}

// Reads and clears this file's error word in one step, so that no code is lost between the two.
static __global__ void take_error_kernel(int* out) { *out = atomicExch(&error_word, 0); }

// 0, or the code of a bounded wait that ran out since the last call.  Covers what was launched on the current stream of `like`'s
// device, or on streams that it has waited for; waits for that work.
inline int64_t take_error(const at::Tensor& like) {
  c10::cuda::CUDAGuard guard(like.device());
  at::Tensor word = at::empty({1}, like.options().dtype(at::kInt));
  take_error_kernel<<<1, 1, 0, at::cuda::getCurrentCUDAStream()>>>(word.data_ptr<int>());
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  return word.item<int>();
}

// For epilogues that read nothing.
struct NoPrefetch {
  struct Pre {};
  template <typename P>
  static __device__ __forceinline__ void prefetch(const P&, const Tiles&, const TileAt&, int, int, Pre&) {}
};

// out[batch][split][M][N] = acc, as T.
template <typename T, int BN, int ACC>
struct EpiStore : NoPrefetch {
  static constexpr int kAcc = ACC, kStride = BN;
  static constexpr bool kLate = false;
  static_assert(ACC == 1 || ACC * BN <= 512, "dense: accumulators exceed the TMEM");
  struct Params { T* out; int64_t ld, batch_stride, split_stride; };
  static __device__ __forceinline__ void poison(const Params& p, const Tiles& t, const TileAt& at, int row0, int part) {
    const int n0 = at.n * BN + part * (BN / 2);
    fill_nan(p.out + at.batch * p.batch_stride + (at.split - t.split0) * p.split_stride + (int64_t)row0 * p.ld + n0, p.ld, t.M - row0,
             t.N - n0, BN / 2);
  }
  static __device__ __forceinline__ void run(const Params& p, const Tiles& t, const TileAt& at, uint32_t tm, int row0, int part,
                                             uint4* stage, Pre&) {
    constexpr int COLS = BN / 2;  // columns of a warp
    T* out = p.out + at.batch * p.batch_stride + (at.split - t.split0) * p.split_stride;
    const bool vec_ok = p.ld % (16 / (int)sizeof(T)) == 0 && (reinterpret_cast<uintptr_t>(out) & 15) == 0;
    const int used = used_acc<ACC>(t, at, 0);
#pragma unroll 1
    for (int cb = 0; cb < COLS / 32; ++cb) {
      const int c = part * COLS + cb * 32, n0 = at.n * BN + c;
      float v[32];
      acc_ld32<ACC, BN>(tm + c, v, used);
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
  maps.n = std::max(maps.n, i + 1);
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
  TORCH_CHECK(r == CUDA_SUCCESS, "cuTensorMapEncodeTiled failed with code ", std::to_string((int)r));
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

// More than one block of 128 rows: pairs of CTAs (their tile of 256 rows costs less than two of 128).
inline bool use_pair(int64_t M) { return M > BM; }

// In a pair every CTA holds half of the tile of B, so n / 2 of each segment has to be a multiple of 64.
inline void set_tiles(Tiles& t, int64_t M, int64_t N, int bn, int64_t batches, int splits, bool lower = false, bool pair = true) {
  t.M = (int)M; t.N = (int)N; t.bn = bn;
  t.bm = pair && use_pair(M) ? 2 * BM : BM;
  t.mt = (int)((M + t.bm - 1) / t.bm); t.nt = (int)((N + bn - 1) / bn);
  t.batches = (int)batches; t.splits = splits; t.split0 = 0; t.lower = lower ? t.bm / bn : 0;
  TORCH_CHECK(!lower || (t.lower >= 1 && t.bm % bn == 0), "dense: symmetric tiles do not fit");
  const int64_t per = lower ? (int64_t)t.lower * ((int64_t)t.mt * (t.mt + 1) / 2) : (int64_t)t.mt * t.nt;
  TORCH_CHECK(per * batches * splits < (1ll << 31), "dense: too many tiles");
  t.total = (int)(per * batches * splits);
}

// The tile of a product with an epilogue of about 1 us per 64 columns (one that reads and writes several arrays), chosen by an
// estimate of its time: rounds of tiles over the GPU, each the longer of its products (0.42 us per 64-wide block of the
// contraction axis for 256 columns, 0.33 for 128, 0.30 for 64; measured) and its epilogue, and the last epilogue on top.  A
// symmetric output may compute the tiles below the diagonal alone and write them twice (an epilogue 1.6 times as long).
struct TileShape { int bn; bool pair, lower; };
inline TileShape pick_tile(int64_t M, int64_t N, int64_t K, int64_t batches, bool symmetric) {
  TileShape best{128, false, false};
  double least = 1e30;
  const double nk = (double)((K + BK - 1) / BK);
  for (int i = 0; i < 8; ++i) {
    const int bn = (i & 3) == 0 ? 256 : (i & 3) == 3 ? 64 : 128;
    const bool pair = (i & 3) < 2, lower = i >= 4;
    if ((pair && !use_pair(M)) || (lower && !symmetric)) continue;
    Tiles t{};
    set_tiles(t, M, N, bn, batches, 1, lower, pair);
    const int64_t at_once = pair ? sm_count() / 2 : sm_count();
    const double rounds = (double)((t.total + at_once - 1) / at_once), products = nk * (bn == 256 ? 0.42 : bn == 128 ? 0.33 : 0.30),
                 epilogue = (lower ? 1.6 : 1.0) * bn / 64;
    const double cost = rounds * std::max(products, epilogue) + std::min(products, epilogue) + (pair ? 1.0 : 0.4);
    if (cost < least) { least = cost; best = {bn, pair, lower}; }
  }
  return best;
}

// Columns of a pair's tile, 256 or 128, by the number of tiles of each kind: the wide one takes less shared-memory traffic per
// product (320 ns against 2 x 225 ns per 64-wide block), the narrow one may fill the last round of the GPU better.
inline int pick_bn(int64_t tiles256, int64_t tiles128) {
  const int64_t pairs = sm_count() / 2;
  const double wide = (double)((tiles256 + pairs - 1) / pairs), narrow = 0.7 * (double)((tiles128 + pairs - 1) / pairs);
  return wide <= narrow ? 256 : 128;
}

// 64-wide blocks (four instructions each) that may be added to one accumulator.  16 bits: what is lost stays under an eighth of
// half a step of the result's type, 2^-14 (float16) and 2^-11.  float32: 32 instructions, 5e-7 in sums of both signs and 3.2e-6
// at most.
inline int max_blocks(at::ScalarType t) { return t == at::kFloat ? 8 : t == at::kHalf ? 128 : 1024; }

// Tiles that run at the same time.
inline int slots(const Tiles& t) { return t.bm == BM ? sm_count() : sm_count() / 2; }

// The small kernels of a chain take part in the early launches too: they call chain_wait() before they touch memory.
__device__ __forceinline__ void chain_wait() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
}
template <typename... P, typename... A>
void launch_chained(void (*kernel)(P...), dim3 grid, int threads, cudaStream_t st, A... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  C10_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...));
}

template <int BN, bool PAIR, typename Epi>
void launch_dense(const Maps& maps, Tiles& t, const typename Epi::Params& ep, cudaStream_t st) {
  constexpr int smem = smem_bytes<BN, PAIR>();
  static_assert(smem <= 227 * 1024, "dense: stages exceed shared memory");
  for (int i = 0; i < t.n_seg; ++i) t.seg[i].idesc = (t.seg[i].idesc & 0xFFFFFFu) | (uint32_t)((PAIR ? 2 * BM : BM) >> 4) << 24;
  // set on every call: the attribute belongs to the current device's context
  C10_CUDA_CHECK(cudaFuncSetAttribute(dense_kernel<BN, PAIR, Epi>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(std::min(t.total, slots(t)) * (PAIR ? 2 : 1)));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = 2; at[1].val.clusterDim.y = 1; at[1].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = PAIR ? 2 : 1;
  C10_CUDA_CHECK(cudaLaunchKernelEx(&cfg, dense_kernel<BN, PAIR, Epi>, maps, t, ep));
}
template <int BN, typename Epi>
void run_dense(const Maps& maps, Tiles& t, const typename Epi::Params& ep, cudaStream_t st) {
  if constexpr (BN == 64) {
    launch_dense<BN, false, Epi>(maps, t, ep, st);
  } else if (t.bm == BM) {
    if constexpr (BN == 256 && !Epi::kLate) {
      TORCH_CHECK(false, "dense: 256-column tiles are for pairs");
    } else {
      launch_dense<BN, false, Epi>(maps, t, ep, st);
    }
  } else {
    for (int i = 0; i < t.n_seg; ++i) TORCH_CHECK(t.seg[i].n % 128 == 0, "dense: a segment too narrow for a pair");
    launch_dense<BN, true, Epi>(maps, t, ep, st);
  }
}

// out = base (0 if null) + the sum over splits of partial [splits][n], in order.  `base` may be `out`.
template <typename T>
__global__ void __launch_bounds__(256) split_sum_kernel(const float* __restrict__ partial, int splits, int64_t stride, int64_t n,
                                                        const float* base, T* out) {
  chain_wait();
  const int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x;
  if (i >= n) return;
  float s = base != nullptr ? base[i] : 0.f;
  for (int k = 0; k < splits; ++k) s += partial[k * stride + i];
  out[i] = narrow<T>(s);
}

// The product of t's segments into `out` [batches][M][N] with the contraction axis split over `splits` tiles of every output
// tile: partial sums in memory, added in order.  More than kPartials of them, or more than 1 GB, are formed and added in rounds.
constexpr int kPartials = 64;
constexpr int64_t kPartialFloats = 1ll << 28;
template <typename T, int BN, int ACC>
void split_product(const Maps& maps, Tiles& t, int64_t M, int64_t N, int64_t batches, int splits, bool pair, T* out,
                   const at::TensorOptions& fp32, cudaStream_t st) {
  const int64_t n = batches * M * N;
  const int round = (int)std::max<int64_t>(1, std::min<int64_t>({splits, kPartials, kPartialFloats / n}));
  at::Tensor part = at::empty({round, n}, fp32), total;
  float* sum = nullptr;
  if (splits > round) {
    if constexpr (sizeof(T) == 4) {
      sum = out;
    } else {
      total = at::empty({n}, fp32);
      sum = total.data_ptr<float>();
    }
  }
  const dim3 grid((unsigned)((n + 255) / 256));
  for (int s0 = 0; s0 < splits; s0 += round) {
    const int here = std::min(round, splits - s0);
    set_tiles(t, M, N, BN, batches, here, false, pair);
    t.splits = splits;
    t.split0 = s0;
    typename EpiStore<float, BN, ACC>::Params ep{part.data_ptr<float>(), N, M * N, n};
    run_dense<BN, EpiStore<float, BN, ACC>>(maps, t, ep, st);
    const float* const base = s0 > 0 ? sum : nullptr;
    if (s0 + here < splits) launch_chained(split_sum_kernel<float>, grid, 256, st, part.data_ptr<float>(), here, n, n, base, sum);
    else launch_chained(split_sum_kernel<T>, grid, 256, st, part.data_ptr<float>(), here, n, n, base, out);
  }
}

}  // namespace dense
}  // namespace nva
