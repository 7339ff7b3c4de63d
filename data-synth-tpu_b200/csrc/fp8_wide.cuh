// The wide FP8 product, for many rows of x.
//
// Pairs of CTAs, one per SM, work through tiles of 256 rows by 256 columns (gated: 128 of the gate and the same 128
// of up): each CTA brings 128 rows of x and 128 of the weights, and one MMA over the pair (M 256, N 128, K 32) reads
// both. A block of 128 columns of K is one row of the 128-byte swizzle and twice four MMAs, for either half of the
// columns; their sums go to one of two buffers of 128 TMEM columns for that half (in each CTA its 128 rows), and the
// half's four warps per CTA add them, times the block's two scales, to FP32 sums in their registers (a row and 128
// columns per thread) while the tensor core fills the three others. A warp issues each half's MMAs: one for both took
// about 900 cycles a block for its waits and issues, more than the products.
// Where the tiles of 256 x 256 do not fill the pairs, they are half as wide (HALF 64), with four buffers of 64 columns
// for either half: 1024 rows of 4096 x 2048 13.5 us (whole 17.3), 256 of 2048 x 9216 9.0 (11.4). A block of such a tile
// takes 0.29 us alone (whole 0.38, in a full round 0.57). The halves having every other block of 128 columns instead takes
// 0.25, but 0.7 more at the end, where they join their sums; summing a block while the next is read 0.30.
//
// Measured (B200, 1.9 GHz, in bursts / in a loop of seconds under the power cap):
//   x 16384 x 2048 of codes, 9216 columns, BF16 out   285 / 330 us, 2170 / 1870 TFLOP/s; FP32 out 334 in bursts
//   4096 x 8192, 8192 columns                         235 / 273 us, 2340 / 2010 TFLOP/s; FP32 out 240
//   gated, 8192 x 2048, 6144 columns of each          208 to 225 / 235 us, 1980 to 1830 / 1750 TFLOP/s
// What bounds it: the first takes 287 us; without the sums' loads from tensor memory and additions 237, without the output
// 255, without both 202 (2048 columns of K; of 8192 236, 196, 229 and 186), and the products alone would take 187 at
// twice the rate of BF16. So the sums come first, then the output, which runs beside the next tile's copies but not
// beside its sums, then the exchange of buffers and shared memory (x's tile is read once for either half); and the rounds:
// 2304 tiles on 74 pairs are 31.1 rounds in 32. In long loops it is the power. One buffer of 256 columns for both halves
// saves that second read, but took 317 us where this form took 303; sixteen warps for the sums took 360, five or six
// stages nothing less.
#pragma once

#include "fp8_product.cuh"

namespace qk {
namespace {

constexpr int kTileM = 256, kHalf = 128;  // rows of a pair's tile, and a CTA's of x
constexpr uint32_t kBytesA = kHalf * kFp8Block;
// What follows from HALF, the columns of either half of a tile: 128 or 64.
template <int HALF>
struct Wide {
  static constexpr int kTileN = 2 * HALF, kBuffers = 512 / kTileN, kStages = HALF == 128 ? 4 : 6;
  static constexpr uint32_t kBytesB = HALF * kFp8Block, kStageBytes = kBytesA + kBytesB;  // of one CTA
};
constexpr int kFirstSum = 4, kSumWarps = 8, kThreads = (kFirstSum + kSumWarps) * 32;
constexpr uint32_t kPiece = 4096, kStaging = 2 * kPiece;  // bytes of 32 rows of 128 on their way out, per summing warp
constexpr int kAhead = 4;            // blocks whose scales of x are on their way
// Registers per thread: 168 at launch for 3 warpgroups (504 in all).
constexpr int kSumRegs = 216, kOtherRegs = 72;
static_assert(2 * kSumRegs + kOtherRegs <= 3 * 168, "the shares fit the launch's registers");
constexpr int kGroupM = 8;  // tiles of rows that run next to one another, so that they share the weights' tiles in L2

struct WideArgs {
  int64_t M;
  int N, blocks, n_blocks;  // blocks of K, blocks of N
  int tiles_m, tiles_n;
  const float *xs, *ws, *us;  // [blocks][M], [n_blocks][blocks], and of up
  void* out;                  // [M][N], or codes [M][ld]
  int64_t ld;
  float* out_scales;          // [n_blocks][M]
  bool f32, copies;           // of out: FP32; rows that begin on 16 bytes, so that tensor copies can write them
};

struct WideControl {
  uint64_t full[6], empty[6], sum_full[4][2], sum_empty[4][2];
  uint64_t swapped[4];               // a row's two warps have left their maxima
  uint32_t tmem;
};

struct Tile {
  int m, n;
};
__device__ __forceinline__ Tile tile_of(const WideArgs& a, int t) {
  const int band = kGroupM * a.tiles_n, first = t / band * kGroupM, in = t % band;
  const int high = min(kGroupM, a.tiles_m - first);
  return Tile{first + in % high, in / high};
}

// The address of `bar` in the pair's first CTA, which issues the MMAs.
__device__ __forceinline__ uint32_t leaders(const uint64_t* bar) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(smem_addr(bar)));
  return r;
}

__device__ __forceinline__ void load_box_pair(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%2, %3}], [%4];" ::"r"(
          dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar)
      : "memory");
}

__device__ __forceinline__ void umma_e4m3_pair(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n}\n" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// Arrive once on `bar` in both CTAs when all MMAs issued so far by this thread are complete.
__device__ __forceinline__ void umma_commit_pair(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(smem_addr(bar)),
               "h"(static_cast<uint16_t>(3))
               : "memory");
}

// An arrival that orders nothing but what came before by itself: the loads from tensor memory are complete (wait::ld).
// With .release.cluster, which waits for this thread's stores to be seen in the cluster, the round trip of a buffer
// took 1.4 us and 16384 x 2048 by 9216 580 us, where this took 307.
__device__ __forceinline__ void cluster_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}

// Both CTAs: their rows of x and of the weights. The bytes count on the leader's barrier.
template <bool GATED, int HALF>
__device__ __forceinline__ bool wide_copies(const WideArgs& a, WideControl& ctl, const CUtensorMap* x, const CUtensorMap* w,
                                            const CUtensorMap* u, uint32_t smem, int rank) {
  using L = Wide<HALF>;
  uint32_t it = 0, s = 0, lap = 0;
  bool ok = true;
  const CUtensorMap* b_map = GATED && rank ? u : w;
  for (int t = blockIdx.x / 2; ok && t < a.tiles_m * a.tiles_n; t += gridDim.x / 2) {
    const Tile tile = tile_of(a, t);
    const int a_row = tile.m * kTileM + rank * kHalf, b_row = GATED ? tile.n * kFp8Block : tile.n * L::kTileN + rank * (HALF / 2);
    for (int b = 0; b < a.blocks; ++b, ++it) {
      const uint32_t at = smem + s * L::kStageBytes, bar = leaders(&ctl.full[s]);
      ok = mbar_wait_bounded(&ctl.empty[s], lap ^ 1);
      if (!ok) break;
      if (rank == 0) mbar_expect_tx(&ctl.full[s], 2 * L::kStageBytes);
      load_box_pair(at, x, b * kFp8Block, a_row, bar);
      load_box_pair(at + kBytesA, b_map, b * kFp8Block, b_row, bar);
      load_box_pair(at + kBytesA + L::kBytesB / 2, b_map, b * kFp8Block, b_row + (GATED ? 64 : HALF), bar);
      if (++s == L::kStages) s = 0, lap ^= 1;
    }
  }
  // Every copy issued must have landed before the CTA leaves: when the MMAs that read it are done.
  for (uint32_t i = it > L::kStages ? it - L::kStages : 0; i < it; ++i) mbar_wait_bounded(&ctl.empty[i % L::kStages], i / L::kStages & 1);
  return ok;
}

// The leader's MMA warps, one for each half of the columns.
template <int HALF>
__device__ __forceinline__ bool wide_products(const WideArgs& a, WideControl& ctl, uint32_t smem, const int h) {
  using L = Wide<HALF>;
  constexpr uint32_t idesc = (1u << 4) | (HALF >> 3) << 17 | (kTileM >> 4) << 24;
  const uint32_t tm = __shfl_sync(0xffffffffu, ctl.tmem, 0);
  const uint64_t ad0 = sdesc_sw128(smem, 1024u), bd0 = sdesc_sw128(smem + kBytesA + h * (L::kBytesB / 2), 1024u);
  uint32_t s = 0, full = 0, d = 0, freed = 1;
  bool ok = true;
  for (int t = blockIdx.x / 2; ok && t < a.tiles_m * a.tiles_n; t += gridDim.x / 2) {
    for (int b = 0; b < a.blocks; ++b) {
      ok = warp_wait(&ctl.sum_empty[d][h], freed) && warp_wait(&ctl.full[s], full);
      if (!ok) break;
      tc_fence_after();
      if (elect_one()) {
        const uint64_t ad = ad0 + s * (L::kStageBytes >> 4), bd = bd0 + s * (L::kStageBytes >> 4);
#pragma unroll
        for (int k = 0; k < 4; ++k) umma_e4m3_pair(tm + d * L::kTileN + h * HALF, ad + 2 * k, bd + 2 * k, idesc, k != 0);
        umma_commit_pair(&ctl.empty[s]);
        umma_commit_pair(&ctl.sum_full[d][h]);
      }
      __syncwarp();
      if (++s == L::kStages) s = 0, full ^= 1;
      if (++d == L::kBuffers) d = 0, freed ^= 1;
    }
  }
  // The last products are complete before the tensor memory is given back, also where a wait gave up (beside the warps
  // that add them, so it costs nothing). Where none were issued, this asks for the phase before the first.
  const uint32_t last = d ? d - 1 : L::kBuffers - 1;
  return warp_wait(&ctl.sum_full[last][h], (d ? freed : freed ^ 1) ^ 1) && ok;
}

// One block's sums, 64 columns at a time, times `by`, added to `acc`.
template <int COUNT>
__device__ __forceinline__ void add_block(uint32_t col, float scale, uint64_t* acc) {
  const uint64_t by = f32x2(scale, scale);
#pragma unroll
  for (int c = 0; c < COUNT; c += 64) {
    uint32_t v[64];
    tmem_get64(col + c, v);
#pragma unroll
    for (int j = 0; j < 32; ++j)
      acc[c / 2 + j] = f32x2_fma(f32x2(__uint_as_float(v[2 * j]), __uint_as_float(v[2 * j + 1])), by, acc[c / 2 + j]);
  }
}

// A piece of staged output out, by a copy that runs beside the next tile's products. (Plain stores held the warps until
// memory had taken them, all SMs' at the same time: 60 us of 350.)
__device__ __forceinline__ void store_box(const CUtensorMap* map, int x, int y, uint32_t from) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%1, %2}], [%3];" ::"l"(reinterpret_cast<uint64_t>(map)),
               "r"(x), "r"(y), "r"(from)
               : "memory");
  asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}
// Until all but the last `N` pieces that this thread sent have been read from shared memory.
template <int N>
__device__ __forceinline__ void stores_read() {
  asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(N) : "memory");
}

// 32 rows (a lane each) of HALF columns out, through shared memory, in pieces of 128 bytes a row, two of which alternate.
template <bool F32, int HALF>
__device__ __forceinline__ void wide_store(const WideArgs& a, const CUtensorMap* map, const uint64_t (&acc)[HALF / 2], uint32_t staging,
                                           int64_t row0, int col0) {
  constexpr int kSize = F32 ? 4 : 2, kColumns = 128 / kSize;
  const int lane = threadIdx.x & 31;
  const int rows = static_cast<int>(min(a.M - row0, static_cast<int64_t>(32)));
  if (rows <= 0) return;
#pragma unroll
  for (int c = 0; c < HALF; c += kColumns) {
    if (col0 + c >= a.N) break;
    const uint32_t piece = staging + (c / kColumns & 1) * kPiece;
    if (lane == 0 && c == 0) stores_read<0>();  // the last tile's
    if (lane == 0 && c >= 2 * kColumns) stores_read<1>();
    __syncwarp();
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      uint32_t w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float x, y;
        if (F32) {
          f32x2_split(acc[c / 2 + j * 2 + i / 2], x, y);
          w[i] = __float_as_uint(i & 1 ? y : x);
        } else {
          f32x2_split(acc[c / 2 + j * 4 + i], x, y);
          w[i] = pack_bf16x2(x, y);
        }
      }
      sts_v4(piece + lane * 128 + ((j ^ lane) & 7) * 16, w[0], w[1], w[2], w[3]);
    }
    if (a.copies) {
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) store_box(map, col0 + c, static_cast<int>(row0), piece);
      continue;
    }
    __syncwarp();
    uint8_t* out = static_cast<uint8_t*>(a.out) + (row0 * a.N + col0 + c) * kSize;
    for (int r = 0; r < rows; ++r) {
      const uint32_t v = lds_at(piece + r * 128 + ((lane / 4 ^ r) & 7) * 16 + (lane & 3) * 4);
      uint8_t* at = out + static_cast<int64_t>(r) * a.N * kSize + lane * 4;
      if (F32) {
        if (col0 + c + lane < a.N) *reinterpret_cast<uint32_t*>(at) = v;
      } else {
        if (col0 + c + 2 * lane < a.N) *reinterpret_cast<uint16_t*>(at) = static_cast<uint16_t>(v);
        if (col0 + c + 2 * lane + 1 < a.N) *reinterpret_cast<uint16_t*>(at + 2) = static_cast<uint16_t>(v >> 16);
      }
    }
  }
}

template <bool GATED, int HALF>
__device__ __forceinline__ bool wide_sums(const WideArgs& a, WideControl& ctl, const CUtensorMap* out_map, uint32_t staging, int rank) {
  const int warp = (threadIdx.x >> 5) - kFirstSum, quarter = warp & 3, half = warp >> 2, lane = threadIdx.x & 31;
  const uint32_t tm = ctl.tmem + (static_cast<uint32_t>(quarter * 32) << 16);
  using L = Wide<HALF>;
  const uint32_t released = leaders(&ctl.sum_empty[0][half]);
  const uint32_t scales = staging + kSumWarps * kStaging + (threadIdx.x - kFirstSum * 32) * 4;  // this thread's, kAhead slots
  const uint32_t swaps_at = scales - (threadIdx.x - kFirstSum * 32) * 4 + kAhead * kSumWarps * 128;
  staging += warp * kStaging;
  uint32_t it = 0, swaps = 0;
  for (int t = blockIdx.x / 2; t < a.tiles_m * a.tiles_n; t += gridDim.x / 2) {
    const Tile tile = tile_of(a, t);
    const int64_t row0 = static_cast<int64_t>(tile.m) * kTileM + rank * kHalf + quarter * 32, row = row0 + lane;
    // a thread's columns: half of the tile's, or 64 of the gate's and the same of up's
    const int n_block = GATED ? tile.n : HALF == 128 ? min(tile.n * 2 + half, a.n_blocks - 1) : tile.n;
    const float* ws = a.ws + static_cast<int64_t>(n_block) * a.blocks;
    const float* us = GATED ? a.us + static_cast<int64_t>(n_block) * a.blocks : nullptr;
    const float* xs = a.xs + min(row, a.M - 1);
    auto fetch = [&](int b) {  // a thread brings its row's scale of a block to its own slot, so nobody else waits for it
      if (b < a.blocks)
        asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(scales + (b % kAhead) * (kSumWarps * 128)),
                     "l"(xs + static_cast<int64_t>(b) * a.M)
                     : "memory");
      cp_async_commit();
    };
    for (int b = 0; b < kAhead; ++b) fetch(b);
    uint64_t acc[HALF / 2];
#pragma unroll
    for (int j = 0; j < HALF / 2; ++j) acc[j] = 0;
    for (int b = 0; b < a.blocks; ++b, ++it) {
      const uint32_t d = it % L::kBuffers, cols = tm + d * L::kTileN + half * HALF;
      const float w = __ldg(ws + b), u = GATED ? __ldg(us + b) : 0.f;
      cp_async_wait<kAhead - 1>();
      const float x = __uint_as_float(lds_at(scales + (b % kAhead) * (kSumWarps * 128)));
      fetch(b + kAhead);
      if (!warp_wait(&ctl.sum_full[d][half], it / L::kBuffers & 1)) return false;
      tc_fence_after();
      if constexpr (GATED) {
        add_block<64>(cols, x * w, acc);
        add_block<64>(cols + 64, x * u, acc + 32);
      } else {
        add_block<HALF>(cols, x * w, acc);
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) cluster_arrive(released + d * sizeof(ctl.sum_empty[0]));
    }
    if constexpr (!GATED) {
      if (a.f32) wide_store<true, HALF>(a, out_map, acc, staging, row0, tile.n * L::kTileN + half * HALF);
      else wide_store<false, HALF>(a, out_map, acc, staging, row0, tile.n * L::kTileN + half * HALF);
      continue;
    } else {
    // A thread has half of its row's block of 128: two threads swap their maxima. No rounding before the codes'.
    float h[64];
    uint32_t most = 0;
#pragma unroll
    for (int j = 0; j < 32; ++j) {
      float g0, g1, u0, u1;
      f32x2_split(acc[j], g0, g1);
      f32x2_split(acc[32 + j], u0, u1);
      h[2 * j] = gated(g0, u0);
      h[2 * j + 1] = gated(g1, u1);
      most = max(most, max(magnitude(h[2 * j]), magnitude(h[2 * j + 1])));
    }
    const uint32_t swap = swaps_at + (swaps & 1) * 1024 + quarter * 128 + lane * 4;
    asm volatile("st.shared.u32 [%0], %1;" ::"r"(swap + half * 512), "r"(most) : "memory");
    __syncwarp();
    if (lane == 0) mbar_arrive(&ctl.swapped[quarter]);
    if (!warp_wait(&ctl.swapped[quarter], swaps & 1)) return false;
    most = max(most, lds_at(swap + (half ^ 1) * 512));
    ++swaps;
    const Fp8Divisor by(most);
    const int col = tile.n * kFp8Block + half * 64;
    if (lane == 0) stores_read<0>();  // the last tile's
    __syncwarp();
    uint32_t codes[16];
#pragma unroll
    for (int j = 0; j < 16; ++j) codes[j] = by.codes4(h + 4 * j);
    if (col + 64 <= a.N || a.N % 16 == 0) {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        sts_v4(staging + lane * 64 + ((j ^ lane >> 1) & 3) * 16, codes[4 * j], codes[4 * j + 1], codes[4 * j + 2], codes[4 * j + 3]);
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0 && row0 < a.M && col < a.N) store_box(out_map, col, static_cast<int>(row0), staging);  // 64-byte swizzle
    } else if (row < a.M) {  // a tensor copy writes 16 bytes at a time, also past the end of a row
      uint8_t* out = static_cast<uint8_t*>(a.out) + row * a.ld + col;
#pragma unroll
      for (int j = 0; j < 64; j += 16) {
        if (col + j + 16 <= a.N) {
          *reinterpret_cast<uint4*>(out + j) = make_uint4(codes[j / 4], codes[j / 4 + 1], codes[j / 4 + 2], codes[j / 4 + 3]);
          continue;
        }
#pragma unroll
        for (int i = j; i < j + 16; ++i)
          if (col + i < a.N) out[i] = static_cast<uint8_t>(codes[i / 4] >> (8 * (i & 3)));
      }
    }
    if (half == 0 && row < a.M) a.out_scales[static_cast<int64_t>(tile.n) * a.M + row] = fp8_scale(most);
    }
  }
  return true;
}

template <bool GATED, int HALF>
__global__ void __launch_bounds__(kThreads, 1) __cluster_dims__(2, 1, 1)
    fp8_wide_kernel(const __grid_constant__ CUtensorMap x, const __grid_constant__ CUtensorMap w, const __grid_constant__ CUtensorMap u,
                    const __grid_constant__ CUtensorMap out, WideArgs a) {
  using L = Wide<HALF>;
  extern __shared__ uint8_t smem_raw[];
  __shared__ WideControl ctl;
  const uint32_t smem = (smem_addr(smem_raw) + 1023) & ~1023u;
  const int warp = threadIdx.x >> 5, rank = static_cast<int>(cluster_rank());
  if (threadIdx.x == 0) {
    for (int i = 0; i < L::kStages; ++i) {
      mbar_init(&ctl.full[i], 1);
      mbar_init(&ctl.empty[i], 2);
    }
    for (int i = 0; i < L::kBuffers; ++i) {
      for (int h = 0; h < 2; ++h) {
        mbar_init(&ctl.sum_full[i][h], 1);
        mbar_init(&ctl.sum_empty[i][h], kSumWarps);  // half of the warps of either CTA
      }
    }
    for (int i = 0; i < 4; ++i) mbar_init(&ctl.swapped[i], 2);
    fence_mbar_init();
  }
  // Both CTAs' tensor memory. They hold it while they wait for one another, but no other CTA that could wait for some
  // fits beside one of these: they have all but 1,024 of an SM's registers.
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_addr(&ctl.tmem)));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync();  // the barriers of both are there
  tc_fence_after();
  pdl_wait();
  pdl_trigger();
  bool ok = true;
  if (warp >= kFirstSum) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSumRegs));
    ok = wide_sums<GATED, HALF>(a, ctl, &out, smem + L::kStages * L::kStageBytes, rank);
    if ((threadIdx.x & 31) == 0) stores_read<0>();  // on every way out: the CTA's shared memory lives until then
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
    if (warp == 0) {
      if (threadIdx.x == 0) ok = wide_copies<GATED, HALF>(a, ctl, &x, &w, &u, smem, rank);
    } else if (warp == 1 && rank == 0) {
      ok = wide_products<HALF>(a, ctl, smem, 0);
    } else if (warp == 2 && rank == 0) {
      ok = wide_products<HALF>(a, ctl, smem, 1);
    }
  }
  if (!ok) atomicExch(&g_fp8_status, QK_ERR_TIMEOUT);
  tc_fence_before();
  __syncthreads();
  cluster_sync();  // neither reads the other's shared or tensor memory any more
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(ctl.tmem));
  }
}

template <bool GATED, int HALF>
int launch_wide(const CUtensorMap& x, const CUtensorMap& w, const CUtensorMap& u, const CUtensorMap& out, const WideArgs& a, cudaStream_t st) {
  using L = Wide<HALF>;
  const size_t smem = 1024 + L::kStages * L::kStageBytes + kSumWarps * kStaging + kAhead * kSumWarps * 128 + 2048;
  const int rc = allow_smem(reinterpret_cast<const void*>(fp8_wide_kernel<GATED, HALF>), smem);
  if (rc) return rc;
  const int tiles = a.tiles_m * a.tiles_n, pairs = sm_count() / 2;
  cudaError_t e =
      launch_dependent(fp8_wide_kernel<GATED, HALF>, dim3(2 * (tiles < pairs ? tiles : pairs)), dim3(kThreads), smem, st, x, w, u, out, a);
  if (e != cudaSuccess) return cuda_error(e, "fp8_wide_kernel");
  count_launch();
  return QK_OK;
}

}  // namespace
}  // namespace qk
