// The wide FP8 product, for many rows of x.
//
// One CTA per SM works through tiles of 128 rows by 256 columns (gated: 128 of the gate and the same 128 of up).
// A block of 128 columns of K is one row of the 128-byte swizzle and four MMAs (M 128, N 256, K 32); its sum goes to
// one of two buffers of 256 TMEM columns, and eight warps add it, times the block's two scales, to FP32 sums in
// their registers (a row and 128 columns per thread) while the tensor core fills the other buffer.
#pragma once

#include "fp8_product.cuh"

namespace qk {
namespace {

constexpr int kTileM = 128, kTileN = 256;
constexpr int kStages = 4, kBuffers = 2;
constexpr uint32_t kBytesA = kTileM * kFp8Block, kBytesB = kTileN * kFp8Block, kStageBytes = kBytesA + kBytesB;
constexpr int kFirstSum = 4, kSumWarps = 8, kThreads = (kFirstSum + kSumWarps) * 32;
constexpr uint32_t kStaging = 4096;  // bytes per summing warp
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
  bool f32, vectors;          // of out: FP32, and rows that begin on 16 bytes
};

struct WideControl {
  uint64_t full[kStages], empty[kStages], sum_full[kBuffers], sum_empty[kBuffers];
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

template <bool GATED>
__device__ __forceinline__ bool wide_copies(const WideArgs& a, WideControl& ctl, const CUtensorMap* x, const CUtensorMap* w,
                                            const CUtensorMap* u, uint32_t smem) {
  uint32_t it = 0;
  bool ok = true;
  for (int t = blockIdx.x; ok && t < a.tiles_m * a.tiles_n; t += gridDim.x) {
    const Tile tile = tile_of(a, t);
    for (int b = 0; b < a.blocks; ++b, ++it) {
      const uint32_t s = it % kStages, at = smem + s * kStageBytes;
      ok = mbar_wait_bounded(&ctl.empty[s], (it / kStages & 1) ^ 1);
      if (!ok) break;
      mbar_expect_tx(&ctl.full[s], kStageBytes);
      load_box(at, x, b * kFp8Block, tile.m * kTileM, &ctl.full[s]);
      if (GATED) {
        load_box(at + kBytesA, w, b * kFp8Block, tile.n * kFp8Block, &ctl.full[s]);
        load_box(at + kBytesA + kBytesB / 2, u, b * kFp8Block, tile.n * kFp8Block, &ctl.full[s]);
      } else {
        load_box(at + kBytesA, w, b * kFp8Block, tile.n * kTileN, &ctl.full[s]);
      }
    }
  }
  // every copy issued must have landed before the CTA leaves
  for (uint32_t i = it > kStages ? it - kStages : 0; i < it; ++i) mbar_wait_bounded(&ctl.full[i % kStages], i / kStages & 1);
  return ok;
}

__device__ __forceinline__ bool wide_products(const WideArgs& a, WideControl& ctl, uint32_t smem) {
  const uint32_t tm = __shfl_sync(0xffffffffu, ctl.tmem, 0), idesc = idesc_e4m3_m128(kTileN);
  uint32_t it = 0;
  for (int t = blockIdx.x; t < a.tiles_m * a.tiles_n; t += gridDim.x) {
    for (int b = 0; b < a.blocks; ++b, ++it) {
      const uint32_t s = it % kStages, d = it % kBuffers;
      if (!warp_wait(&ctl.full[s], it / kStages & 1)) return false;
      if (!warp_wait(&ctl.sum_empty[d], (it / kBuffers & 1) ^ 1)) return false;
      tc_fence_after();
      if (elect_one()) {
        const uint64_t ad = sdesc_sw128(smem + s * kStageBytes, 1024u), bd = sdesc_sw128(smem + s * kStageBytes + kBytesA, 1024u);
#pragma unroll
        for (int k = 0; k < 4; ++k) umma_e4m3(tm + d * kTileN, ad + 2 * k, bd + 2 * k, idesc, k != 0);
        umma_commit(&ctl.empty[s]);
        umma_commit(&ctl.sum_full[d]);
      }
      __syncwarp();
    }
  }
  return true;
}

// One block's sums, `count` columns from `col`, times `scale`, added to `acc`.
template <int COUNT>
__device__ __forceinline__ void add_block(uint32_t col, float scale, uint64_t* acc) {
  const uint64_t by = f32x2(scale, scale);
#pragma unroll
  for (int c = 0; c < COUNT; c += 32) {
    uint32_t v[32];
    tmem_ld32(col + c, v);
    tmem_wait_ld(v);
#pragma unroll
    for (int j = 0; j < 16; ++j)
      acc[c / 2 + j] = f32x2_fma(f32x2(__uint_as_float(v[2 * j]), __uint_as_float(v[2 * j + 1])), by, acc[c / 2 + j]);
  }
}

// 32 rows (a lane each) of 128 columns out, through 4 KB of shared memory, in pieces of 128 bytes a row.
template <bool F32>
__device__ __forceinline__ void wide_store(const WideArgs& a, const uint64_t (&acc)[64], uint32_t staging, int64_t row0, int col0) {
  constexpr int kSize = F32 ? 4 : 2, kColumns = 128 / kSize;
  const int lane = threadIdx.x & 31;
  const int rows = static_cast<int>(min(a.M - row0, static_cast<int64_t>(32)));
#pragma unroll
  for (int c = 0; c < 128; c += kColumns) {
    if (col0 + c >= a.N) break;
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
      sts_v4(staging + lane * 128 + ((j ^ lane) & 7) * 16, w[0], w[1], w[2], w[3]);
    }
    __syncwarp();
    uint8_t* out = static_cast<uint8_t*>(a.out) + (row0 * a.N + col0 + c) * kSize;
    if (a.vectors && col0 + c + kColumns <= a.N) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int r = i * 4 + lane / 8;
        if (r < rows)
          *reinterpret_cast<uint4*>(out + static_cast<int64_t>(r) * a.N * kSize + (lane & 7) * 16) =
              lds_v4_at(staging + r * 128 + ((lane ^ r) & 7) * 16);
      }
    } else {
      for (int r = 0; r < rows; ++r) {
        const uint32_t v = lds_at(staging + r * 128 + ((lane / 4 ^ r) & 7) * 16 + (lane & 3) * 4);
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
}

template <bool GATED>
__device__ __forceinline__ bool wide_sums(const WideArgs& a, WideControl& ctl, uint32_t staging) {
  const int warp = (threadIdx.x >> 5) - kFirstSum, quarter = warp & 3, half = warp >> 2, lane = threadIdx.x & 31;
  const uint32_t tm = ctl.tmem + (static_cast<uint32_t>(quarter * 32) << 16);
  uint32_t it = 0, swaps = 0;
  for (int t = blockIdx.x; t < a.tiles_m * a.tiles_n; t += gridDim.x) {
    const Tile tile = tile_of(a, t);
    const int64_t row0 = static_cast<int64_t>(tile.m) * kTileM + quarter * 32, row = row0 + lane;
    // a thread's columns: 128 of the tile's 256, or 64 of the gate's and the same of up's
    const int n_block = GATED ? tile.n : min(tile.n * 2 + half, a.n_blocks - 1);
    const float* ws = a.ws + static_cast<int64_t>(n_block) * a.blocks;
    const float* us = GATED ? a.us + static_cast<int64_t>(n_block) * a.blocks : nullptr;
    const float* xs = a.xs + min(row, a.M - 1);
    uint64_t acc[64];
#pragma unroll
    for (int j = 0; j < 64; ++j) acc[j] = 0;
    float x = xs[0], w = ws[0], u = GATED ? us[0] : 0.f;
    for (int b = 0; b < a.blocks; ++b, ++it) {
      const uint32_t d = it % kBuffers, cols = tm + d * kTileN;
      const float by_w = x * w, by_u = x * u;
      if (b + 1 < a.blocks) {
        x = xs[(b + 1) * a.M];
        w = ws[b + 1];
        if (GATED) u = us[b + 1];
      }
      if (!warp_wait(&ctl.sum_full[d], it / kBuffers & 1)) return false;
      tc_fence_after();
      if (GATED) {
        add_block<64>(cols + half * 64, by_w, acc);
        add_block<64>(cols + 128 + half * 64, by_u, acc + 32);
      } else {
        add_block<128>(cols + half * 128, by_w, acc);
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&ctl.sum_empty[d]);
    }
    if (!GATED) {
      if (a.f32) wide_store<true>(a, acc, staging + warp * kStaging, row0, tile.n * kTileN + half * 128);
      else wide_store<false>(a, acc, staging + warp * kStaging, row0, tile.n * kTileN + half * 128);
      continue;
    }
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
    const uint32_t swap = staging + (swaps & 1) * 1024 + quarter * 128 + lane * 4;
    asm volatile("st.shared.u32 [%0], %1;" ::"r"(swap + half * 512), "r"(most) : "memory");
    __syncwarp();
    if (lane == 0) mbar_arrive(&ctl.swapped[quarter]);
    if (!warp_wait(&ctl.swapped[quarter], swaps & 1)) return false;
    most = max(most, lds_at(swap + (half ^ 1) * 512));
    ++swaps;
    if (row < a.M) {
      const Fp8Divisor by(most);
      const int col = tile.n * kFp8Block + half * 64;
      uint8_t* out = static_cast<uint8_t*>(a.out) + row * a.ld + col;
#pragma unroll
      for (int j = 0; j < 64; j += 16)
        if (col + j < a.N)
          *reinterpret_cast<uint4*>(out + j) =
              make_uint4(by.codes4(h + j), by.codes4(h + j + 4), by.codes4(h + j + 8), by.codes4(h + j + 12));
      if (half == 0) a.out_scales[static_cast<int64_t>(tile.n) * a.M + row] = fp8_scale(most);
    }
  }
  return true;
}

template <bool GATED>
__global__ void __launch_bounds__(kThreads, 1)
    fp8_wide_kernel(const __grid_constant__ CUtensorMap x, const __grid_constant__ CUtensorMap w, const __grid_constant__ CUtensorMap u,
                    WideArgs a) {
  extern __shared__ uint8_t smem_raw[];
  __shared__ WideControl ctl;
  const uint32_t smem = (smem_addr(smem_raw) + 1023) & ~1023u;
  const int warp = threadIdx.x >> 5;
  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&ctl.full[i], 1);
      mbar_init(&ctl.empty[i], 1);
    }
    for (int i = 0; i < kBuffers; ++i) {
      mbar_init(&ctl.sum_full[i], 1);
      mbar_init(&ctl.sum_empty[i], kSumWarps);
    }
    for (int i = 0; i < 4; ++i) mbar_init(&ctl.swapped[i], 2);
    fence_mbar_init();
  }
  if (warp == 1) tmem_alloc(&ctl.tmem, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  pdl_wait();
  pdl_trigger();
  bool ok = true;
  if (warp >= kFirstSum) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSumRegs));
    ok = wide_sums<GATED>(a, ctl, smem + kStages * kStageBytes);
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
    if (warp == 0) {
      if (threadIdx.x == 0) ok = wide_copies<GATED>(a, ctl, &x, &w, &u, smem);
    } else if (warp == 1) {
      ok = wide_products(a, ctl, smem);
    }
  }
  if (!ok) atomicExch(&g_fp8_status, QK_ERR_TIMEOUT);
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(ctl.tmem, 512);
  }
}

template <bool GATED>
int launch_wide(const CUtensorMap& x, const CUtensorMap& w, const CUtensorMap& u, const WideArgs& a, cudaStream_t st) {
  const size_t smem = 1024 + kStages * kStageBytes + kSumWarps * kStaging;
  const int rc = allow_smem(reinterpret_cast<const void*>(fp8_wide_kernel<GATED>), smem);
  if (rc) return rc;
  const int tiles = a.tiles_m * a.tiles_n;
  cudaError_t e = launch_dependent(fp8_wide_kernel<GATED>, dim3(tiles < sm_count() ? tiles : sm_count()), dim3(kThreads), smem, st,
                                   x, w, u, a);
  if (e != cudaSuccess) return cuda_error(e, "fp8_wide_kernel");
  count_launch();
  return QK_OK;
}

}  // namespace
}  // namespace qk
