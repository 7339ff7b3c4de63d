// The narrow FP8 product, for few rows of x (tokens): bound by reading the weights once.
//
// The weights are the M = 128 operand and MT tokens the N operand, so a tile of 128 columns of the output is 128 rows
// of the weights. Its blocks of K are split over a cluster of CTAs, which all stream their part of the weights at
// once; each adds its blocks' sums, times their scales, in registers (a thread per weight row and half of the
// tokens) and sends every token's to the CTA that owns it, which adds them (its own, then the others' by rank) and writes.
// x comes as codes, by tensor copies beside the weights', or (ROWS) as BF16 that every CTA quantises for itself while
// its weights are on their way: that saves a launch, and the values are the same.
//
// Measured in a graph of calls over weights larger than L2 (floor: the weights' bytes at the measured HBM rate):
//   1 row of BF16, 2048 x 9216        5.4 us, floor 2.9 (18.9 MB: 3.5 TB/s);  8 rows 6.1; 32 rows of codes 5.9, 64 7.3
//   64 rows of BF16, 4096 x 2048      10.5 us, floor 1.4 (from codes 6.1);  1 row of codes 4.0, floor 1.3
//   feed-forward block, 32 rows, 2048 x 6144   17.2 to 18 us, floor 5.8, quantisation and down product included
// What bounds it is latency: the set-up, the first copy from memory (2 us), then for each block the issue of its MMAs
// (about 300 cycles), its sums and, at the end, the exchange and the output, most of it instructions that run once
// and come cold from L2.
#pragma once

#include "fp8_product.cuh"

namespace qk {
namespace {

constexpr int kNarrowStages = 8, kNarrowSumWarps = 8, kNarrowFirstSum = 2;
constexpr int kNarrowThreads = (kNarrowFirstSum + kNarrowSumWarps) * 32;
constexpr int kNarrowAhead = 4;      // blocks whose scales of x are on their way
constexpr int kMostSplits = 8;       // the portable cluster size
// Three CTAs with as much shared memory do not fit the 228 KB of an SM. Registers do not see to that: with 16 tokens a
// thread has 56, so that three fit, and they need not stay as they are from one compiler to the next.
constexpr size_t kLeastSmem = 77 * 1024;
// Rows of BF16, and blocks of them, that a CTA quantises itself, at most (gated: half, their rings are short). 32 rows of
// 4096 x 2048 (128 blocks per CTA) take 7.0 us, with a launch of its own for that 7.3; 32 of 2048 x 9216 (256) 9.7 and
// 8.5, 64 of 4096 x 2048 (256) 10.5 and 8.5, but that launch takes the host 4 us more, which is where such calls end:
// by wall clock 9.9 and 13.7, 10.8 and 13.6. So beyond 128 it is the host's time that decides, and in a captured graph a
// launch of its own is the faster way. Gated, 192 blocks (32 rows of 2048 x 6144) cost 3 us and save 1.
constexpr int kInline = 256, kInlineTokens = 256;  // kInlineTokens: of their tiles in shared memory

struct NarrowArgs {
  int64_t M;
  int N, blocks, splits, stages;
  uint32_t ring;          // bytes of the copies' ring and x's tiles
  const uint16_t* x;      // BF16 (ROWS), width a multiple of 8
  int64_t x_stride;
  int width, row_shift;   // the power of two of rows, M or more
  const float *xs, *ws, *us;
  void* out;
  int64_t ld;             // of the gated codes
  float* out_scales;
  bool f32, vectors;
};

template <int MT, bool GATED>
struct Narrow {
  static constexpr int kOperands = GATED ? 2 : 1;
  static constexpr uint32_t kBytesW = kOperands * 128 * kFp8Block, kBytesX = MT * kFp8Block, kStage = kBytesW + kBytesX;
  static constexpr int kColumns = kOperands * MT;                           // TMEM columns of a block's sums
  static constexpr int kBuffers = 256 / kColumns < 2 ? 2 : 256 / kColumns > 8 ? 8 : 256 / kColumns;
  // 256 of 512 columns at most, and two CTAs per SM at most, of whatever calls (kLeastSmem): none waits for tensor memory
  // while it holds up its cluster, whose other CTAs hold some that another cluster's may wait for
  static constexpr uint32_t kAlloc = kColumns * kBuffers < 32 ? 32 : kColumns * kBuffers;
  static constexpr int kEach = MT / 2;                                      // tokens per thread
  static constexpr bool kTwo = kColumns <= 64;                              // room for two CTAs per SM
  // shared memory: the ring (and x's tiles), then [other CTA of the cluster][owned token][operand][weight row] sums
  // (the CTA's own go where the ring was)
  static constexpr uint32_t kToken = kOperands * 512, kSums = MT * kToken;
  static uint32_t ring(int stages, int inline_blocks) {
    const uint32_t bytes = stages * (inline_blocks ? kBytesW : kStage) + inline_blocks * kBytesX;
    return bytes > kSums ? bytes : kSums;
  }
  static size_t smem(int stages, int inline_blocks, int splits, int live) {
    return 1024 + ring(stages, inline_blocks) + static_cast<size_t>(splits - 1) * ((live + splits - 1) / splits) * kToken;
  }
};

template <int MT>
struct NarrowControl {
  uint64_t full[kNarrowStages], empty[kNarrowStages], sum_full[8], sum_empty[8], stored, joined;
  int64_t began;  // clock
  uint32_t tmem;
  static constexpr int kSlot = MT > 64 ? 64 : 32;
  alignas(16) float scales[kNarrowSumWarps * kNarrowAhead * kSlot];  // of x: a warp's slots of its tokens, or (ROWS) [block][MT]
  static_assert(kInlineTokens <= kNarrowSumWarps * kNarrowAhead * kSlot, "a scale for each");
};

// The address of this CTA's `addr` in the cluster's CTA `rank`.
__device__ __forceinline__ uint32_t in_rank(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
// A copy to another CTA's shared memory that counts its bytes on that CTA's barrier: no fence, no barrier of the
// cluster. (Sums read from the others' shared memory between two cluster barriers, whose release waits for every
// store of the CTA, took 0.7 and 1 us of 10; a store per value 1.3 us for 64 tokens, most of it cold instructions.)
__device__ __forceinline__ void send(uint32_t to, uint32_t from, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.shared::cta.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(to), "r"(from),
               "r"(bytes), "r"(bar)
               : "memory");
}

template <int MT, bool GATED, bool ROWS>
__device__ __forceinline__ void narrow_copy(const NarrowArgs& a, NarrowControl<MT>& ctl, const CUtensorMap* x, const CUtensorMap* w,
                                            const CUtensorMap* u, uint32_t smem, int it, int b0, int tile, int row0) {
  using L = Narrow<MT, GATED>;
  constexpr uint32_t kStage = ROWS ? L::kBytesW : L::kStage;
  const int s = it % a.stages, b = b0 + it;
  const uint32_t at = smem + s * kStage;
  mbar_expect_tx(&ctl.full[s], kStage);
  load_box(at, w, b * kFp8Block, tile * 128, &ctl.full[s]);
  if (GATED) load_box(at + L::kBytesW / 2, u, b * kFp8Block, tile * 128, &ctl.full[s]);
  if (!ROWS) load_box(at + L::kBytesW, x, b * kFp8Block, row0, &ctl.full[s]);
}

// The copies behind the first a.stages.
template <int MT, bool GATED, bool ROWS>
__device__ __forceinline__ bool narrow_copies(const NarrowArgs& a, NarrowControl<MT>& ctl, const CUtensorMap* x, const CUtensorMap* w,
                                              const CUtensorMap* u, uint32_t smem, int b0, int count, int tile, int row0) {
  bool ok = true;
  int it = min(count, a.stages);
  for (; it < count; ++it) {
    ok = mbar_wait_bounded(&ctl.empty[it % a.stages], (it / a.stages & 1) ^ 1);
    if (!ok) break;
    narrow_copy<MT, GATED, ROWS>(a, ctl, x, w, u, smem, it, b0, tile, row0);
  }
  // every copy issued must have landed before the CTA leaves
  for (int i = max(it - a.stages, 0); i < it; ++i) mbar_wait_bounded(&ctl.full[i % a.stages], i / a.stages & 1);
  return ok;
}

template <int MT, bool GATED, bool ROWS>
__device__ __forceinline__ bool narrow_products(const NarrowArgs& a, NarrowControl<MT>& ctl, uint32_t smem, int count) {
  using L = Narrow<MT, GATED>;
  constexpr uint32_t kStage = ROWS ? L::kBytesW : L::kStage;
  const uint32_t tm = __shfl_sync(0xffffffffu, ctl.tmem, 0), idesc = idesc_e4m3_m128(MT);
  const uint64_t wd0 = sdesc_sw128(smem, 1024u), xd0 = sdesc_sw128(smem + (ROWS ? a.stages * kStage : L::kBytesW), 1024u);
  int s = 0, d = 0;
  uint32_t full = 0, freed = 1;
  bool ok = true;
  for (int it = 0; it < count; ++it) {
    ok = (it < L::kBuffers || warp_wait(&ctl.sum_empty[d], freed)) && warp_wait(&ctl.full[s], full);
    if (!ok) break;
    tc_fence_after();
    if (elect_one()) {
      const uint64_t wd = wd0 + s * (kStage >> 4), xd = xd0 + (ROWS ? it * (L::kBytesX >> 4) : s * (kStage >> 4));
#pragma unroll
      for (int o = 0; o < L::kOperands; ++o)
#pragma unroll
        for (int k = 0; k < 4; ++k)
          umma_e4m3(tm + d * L::kColumns + o * MT, wd + o * (128 * kFp8Block >> 4) + 2 * k, xd + 2 * k, idesc, k != 0);
      if (it + a.stages < count) umma_commit(&ctl.empty[s]);
      umma_commit(&ctl.sum_full[d]);
    }
    __syncwarp();
    if (++s == a.stages) s = 0, full ^= 1;
    if (++d == L::kBuffers) d = 0, freed ^= 1;
  }
  // The last products are complete before the tensor memory is given back, also where a wait gave up. Where none were
  // issued, this asks for the phase before the first.
  return warp_wait(&ctl.sum_full[d ? d - 1 : L::kBuffers - 1], (d ? freed : freed ^ 1) ^ 1) && ok;
}

// The CTA's blocks of x, quantised into the operand tiles and ctl.scales [block][MT]. Rows past M hold whatever the
// memory held: they make columns of the product that nobody reads.
template <int MT, int kAtOnce>
__device__ __forceinline__ void narrow_quantise(const NarrowArgs& a, NarrowControl<MT>& ctl, uint32_t tiles, int b0, int count) {
  const int lane = threadIdx.x & 31, in = lane & 15;
  // 16 half warps: each takes every 16th of (block, row) pairs, kAtOnce of them at a time
  const int half = (threadIdx.x - kNarrowFirstSum * 32) >> 4, units = count << a.row_shift;
  const int mask = (1 << a.row_shift) - 1;
#pragma unroll 1
  for (int first = half & ~1; first < units; first += 16 * kAtOnce) {  // as often in the whole warp
    uint4 v[kAtOnce];
    uint32_t most[kAtOnce];
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      const int unit = first + (half & 1) + 16 * i, row = unit & mask, b = unit >> a.row_shift, at = (b0 + b) * kFp8Block + in * 8;
      v[i] = row < a.M && b < count && at < a.width ? ld_guarded_v4(a.x + row * a.x_stride + at) : make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) most[i] = most8(v[i]);
    block_most(most);
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      const int unit = first + (half & 1) + 16 * i, row = unit & mask, b = unit >> a.row_shift;
      float f[8];
      unpack8(v[i], f);
      const Fp8Divisor by(most[i]);
      const uint32_t lo = by.codes4(f), hi = by.codes4(f + 4);
      if (row < a.M && b < count) {
        const uint32_t to = tiles + b * (MT * kFp8Block) + row * kFp8Block + (((in >> 1) ^ (row & 7)) << 4) + (in & 1) * 8;
        asm volatile("st.shared.v2.u32 [%0], {%1,%2};" ::"r"(to), "r"(lo), "r"(hi) : "memory");
        if (in == 0) ctl.scales[b * MT + row] = fp8_scale(most[i]);
      }
    }
  }
}

template <int MT, bool GATED, bool ROWS>
__device__ __forceinline__ bool narrow_sums(const NarrowArgs& a, NarrowControl<MT>& ctl, uint32_t smem, int b0, int count, int tile, int row0) {
  using L = Narrow<MT, GATED>;
  constexpr int kEach = L::kEach, kLoad = kEach < 32 ? kEach : 32;
  const int warp = (threadIdx.x >> 5) - kNarrowFirstSum, half = warp >> 2, lane = threadIdx.x & 31;
  const int quarter = (threadIdx.x >> 5) & 3;  // the TMEM lanes that this warp may read
  const uint32_t tm = ctl.tmem + (static_cast<uint32_t>(quarter * 32) << 16) + half * kEach;
  const float* ws = a.ws + static_cast<int64_t>(tile) * a.blocks + b0;
  const float* us = GATED ? a.us + static_cast<int64_t>(tile) * a.blocks + b0 : nullptr;
  uint64_t acc[L::kOperands][kEach / 2];
#pragma unroll
  for (int o = 0; o < L::kOperands; ++o)
#pragma unroll
    for (int j = 0; j < kEach / 2; ++j) acc[o][j] = 0;
  // codes: a warp brings its tokens' scales of a block to its own slots, kNarrowAhead blocks ahead (one ahead, each block
  // waited for its scales' way from memory: 32 rows of 2048 x 9216 7.8 us instead of 5.8)
  constexpr int kSlot = NarrowControl<MT>::kSlot;
  float* slots = ctl.scales + warp * (kNarrowAhead * kSlot);
  auto fetch = [&](int i) {
#pragma unroll
    for (int c = 0; c < kEach; c += 32) {
      const int64_t row = row0 + half * kEach + c + lane;
      if (i < count && c + lane < kEach && row < a.M)
        asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_addr(slots + i % kNarrowAhead * kSlot + c + lane)),
                     "l"(a.xs + static_cast<int64_t>(b0 + i) * a.M + row)
                     : "memory");
    }
    cp_async_commit();
  };
  if (!ROWS) {
#pragma unroll
    for (int i = 0; i < kNarrowAhead; ++i) fetch(i);
  }
  float w = ws[0], u = GATED ? us[0] : 0.f;
  for (int it = 0; it < count; ++it) {
    const int d = it % L::kBuffers;
    const float* scales = ctl.scales + it * MT + half * kEach;
    if (!ROWS) {
      cp_async_wait<kNarrowAhead - 1>();
      __syncwarp();
      scales = slots + it % kNarrowAhead * kSlot;
    }
    const float by_w = w, by_u = u;
    if (it + 1 < count) {
      w = ws[it + 1];
      if (GATED) u = us[it + 1];
    }
    if (!warp_wait(&ctl.sum_full[d], it / L::kBuffers & 1)) return false;
    tc_fence_after();
#pragma unroll
    for (int o = 0; o < L::kOperands; ++o) {
      const uint64_t by = o ? f32x2(by_u, by_u) : f32x2(by_w, by_w);
#pragma unroll
      for (int c = 0; c < kEach; c += kLoad) {
        uint32_t v[kLoad];
        tmem_get<kLoad>(tm + d * L::kColumns + o * MT + c, v);
#pragma unroll
        for (int j = 0; j < kLoad / 2; ++j) {
          const float2 s = *reinterpret_cast<const float2*>(scales + c + 2 * j);
          acc[o][c / 2 + j] = f32x2_fma(f32x2(__uint_as_float(v[2 * j]), __uint_as_float(v[2 * j + 1])),
                                        f32x2_mul(f32x2(s.x, s.y), by), acc[o][c / 2 + j]);
        }
      }
    }
    tc_fence_before();
    __syncwarp();
    if (lane == 0) mbar_arrive(&ctl.sum_empty[d]);
    if (!ROWS) fetch(it + kNarrowAhead);
  }
  // All products are done, so nothing reads or fills the ring any more: [token][operand][weight row] goes there.
  const uint32_t to = smem + half * kEach * L::kToken + (quarter * 32 + lane) * 4;
#pragma unroll
  for (int j = 0; j < kEach; ++j)
#pragma unroll
    for (int o = 0; o < L::kOperands; ++o) {
      float p, q;
      f32x2_split(acc[o][j / 2], p, q);
      asm volatile("st.shared.f32 [%0], %1;" ::"r"(to + j * L::kToken + o * 512), "f"(j & 1 ? q : p) : "memory");
    }
  fence_proxy_async_smem();
  __syncwarp();
  if (lane == 0) mbar_arrive(&ctl.stored);
  return true;
}

// A warp per other owner sends it its tokens. Who receives them waits for them, and a CTA leaves behind all the others'
// waits, so this one's memory lives while it is read. But a wait that gave up ends without them, 2^22 polls (more than
// 2^26 cycles) behind the start: sent that late, they get the time that they need before this CTA lets the others go.
template <int MT, bool GATED>
__device__ __forceinline__ bool narrow_send(const NarrowArgs& a, NarrowControl<MT>& ctl, uint32_t smem, int owned, int live, int rank) {
  using L = Narrow<MT, GATED>;
  const int owner = (threadIdx.x >> 5) - kNarrowFirstSum, tokens = min(owned, live - owner * owned);
  if (owner >= a.splits || owner == rank || tokens <= 0) return true;
  if (!warp_wait(&ctl.stored, 0)) return false;
  if (elect_one())
    send(in_rank(smem + a.ring + (rank - (rank > owner)) * owned * L::kToken, owner), smem + owner * owned * L::kToken, tokens * L::kToken,
         in_rank(smem_addr(&ctl.joined), owner));
  if (const int64_t sent = clock64(); sent - ctl.began > (1 << 25)) {
    while (clock64() - sent < (1 << 18)) {
    }
  }
  __syncwarp();
  return true;
}

// The sums of the tokens that this CTA owns, its own first and then the others' by rank, a warp per token and four
// weight rows per lane, and the output. One short loop over both operands: its instructions come cold (a loop for each
// and its unrolled form cost 0.3 us).
template <int MT, bool GATED>
__device__ __forceinline__ void narrow_join(const NarrowArgs& a, uint32_t own, uint32_t sums, int owned, int mine, int64_t first, int tile) {
  using L = Narrow<MT, GATED>;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, n = tile * 128 + lane * 4;
#pragma unroll 1
  for (int i = warp; i < mine; i += kNarrowThreads / 32) {
    float f[2][4];
    const uint32_t at = i * L::kToken + lane * 16;
#pragma unroll
    for (int o = 0; o < L::kOperands; ++o) {
      const uint4 v = lds_v4_at(own + at + o * 512);
#pragma unroll
      for (int j = 0; j < 4; ++j) f[o][j] = __uint_as_float(word(v, j));
    }
#pragma unroll 2
    for (int s = 0; s < a.splits - 1; ++s) {
#pragma unroll
      for (int o = 0; o < L::kOperands; ++o) {
        const uint4 v = lds_v4_at(sums + s * owned * L::kToken + at + o * 512);
#pragma unroll
        for (int j = 0; j < 4; ++j) f[o][j] += __uint_as_float(word(v, j));
      }
    }
    const int64_t row = first + i;
    if (GATED) {
      uint32_t most = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        f[0][j] = gated(f[0][j], f[1][j]);
        most = max(most, magnitude(f[0][j]));
      }
      most = __reduce_max_sync(0xffffffffu, most);
      const uint32_t codes = Fp8Divisor(most).codes4(f[0]);
      uint8_t* out = static_cast<uint8_t*>(a.out) + row * a.ld + n;
      if (n + 4 <= a.N) *reinterpret_cast<uint32_t*>(out) = codes;
      else
        for (int j = 0; n + j < a.N; ++j) out[j] = static_cast<uint8_t>(codes >> (8 * j));
      if (lane == 0) a.out_scales[static_cast<int64_t>(tile) * a.M + row] = fp8_scale(most);
    } else if (a.f32) {
      float* out = static_cast<float*>(a.out) + row * a.N + n;
      if (a.vectors && n < a.N) *reinterpret_cast<float4*>(out) = make_float4(f[0][0], f[0][1], f[0][2], f[0][3]);
      else
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (n + j < a.N) out[j] = f[0][j];
    } else {
      uint16_t* out = static_cast<uint16_t*>(a.out) + row * a.N + n;
      if (a.vectors && n < a.N) *reinterpret_cast<uint2*>(out) = make_uint2(pack_bf16x2(f[0][0], f[0][1]), pack_bf16x2(f[0][2], f[0][3]));
      else
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (n + j < a.N) out[j] = static_cast<uint16_t>(pack_bf16x2(f[0][j], 0.f));
    }
  }
}

// grid: (splits x tiles of 128 weight rows, tiles of MT tokens), clusters of `splits`.
template <int MT, bool GATED, bool ROWS>
__global__ void __launch_bounds__(kNarrowThreads, Narrow<MT, GATED>::kTwo ? 2 : 1)
    fp8_narrow_kernel(const __grid_constant__ CUtensorMap x, const __grid_constant__ CUtensorMap w, const __grid_constant__ CUtensorMap u,
                      NarrowArgs a) {
  using L = Narrow<MT, GATED>;
  extern __shared__ uint8_t smem_raw[];
  __shared__ NarrowControl<MT> ctl;
  const uint32_t smem = (smem_addr(smem_raw) + 1023) & ~1023u;
  const int warp = threadIdx.x >> 5, rank = static_cast<int>(cluster_rank());
  const int tile = static_cast<int>(blockIdx.x) / a.splits, row0 = static_cast<int>(blockIdx.y) * MT;
  const int b0 = static_cast<int>(static_cast<int64_t>(rank) * a.blocks / a.splits);
  const int count = static_cast<int>(static_cast<int64_t>(rank + 1) * a.blocks / a.splits) - b0;  // at least one
  const int live = static_cast<int>(min(a.M - row0, static_cast<int64_t>(MT)));
  // the tokens that a CTA owns, in their order
  const int owned = (live + a.splits - 1) / a.splits, mine = min(max(live - rank * owned, 0), owned);
  if (threadIdx.x == 0) {
    if (!ROWS) prefetch_map(&x);
    // the weights' way from memory to L2 runs beside the kernel ahead
    for (int i = 0; i < min(count, a.stages); ++i) {
      prefetch_box(&w, (b0 + i) * kFp8Block, tile * 128);
      if (GATED) prefetch_box(&u, (b0 + i) * kFp8Block, tile * 128);
    }
    for (int i = 0; i < a.stages; ++i) {
      mbar_init(&ctl.full[i], 1);
      mbar_init(&ctl.empty[i], 1);
    }
    for (int i = 0; i < L::kBuffers; ++i) {
      mbar_init(&ctl.sum_full[i], 1);
      mbar_init(&ctl.sum_empty[i], kNarrowSumWarps);
    }
    mbar_init(&ctl.stored, kNarrowSumWarps);
    mbar_init(&ctl.joined, 1);
    fence_mbar_init();
    mbar_expect_tx(&ctl.joined, (a.splits - 1) * mine * L::kToken);
    pdl_wait();
    // the first copies are on their way while the others set up
    for (int i = 0; i < min(count, a.stages); ++i) narrow_copy<MT, GATED, ROWS>(a, ctl, &x, &w, &u, smem, i, b0, tile, row0);
    ctl.began = clock64();
  }
  if (warp == 1) tmem_alloc(&ctl.tmem, L::kAlloc);
  pdl_wait();
  if (ROWS && warp >= kNarrowFirstSum) {
    if (MT > 16 && count << a.row_shift > 64) narrow_quantise<MT, 8>(a, ctl, smem + a.stages * L::kBytesW, b0, count);
    else narrow_quantise<MT, 4>(a, ctl, smem + a.stages * L::kBytesW, b0, count);
    fence_proxy_async_smem();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  cluster_arrive_relaxed();  // this CTA's barriers are there: the others may send from now on
  pdl_trigger();
  bool ok = true;
  if (warp == 0) {
    if (threadIdx.x == 0) ok = narrow_copies<MT, GATED, ROWS>(a, ctl, &x, &w, &u, smem, b0, count, tile, row0);
    __syncwarp();
    cluster_wait();
  } else if (warp == 1) {
    ok = narrow_products<MT, GATED, ROWS>(a, ctl, smem, count);
    cluster_wait();
  } else {
    ok = narrow_sums<MT, GATED, ROWS>(a, ctl, smem, b0, count, tile, row0);
    __syncwarp();
    cluster_wait();
    if (ok) ok = narrow_send<MT, GATED>(a, ctl, smem, owned, live, rank);
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(ctl.tmem, L::kAlloc);
  }
  if (!warp_wait(&ctl.joined, 0)) ok = false;
  if (!ok) atomicExch(&g_fp8_status, QK_ERR_TIMEOUT);
  cluster_arrive_relaxed();  // what the others sent has been read from their memory
  narrow_join<MT, GATED>(a, smem + rank * owned * L::kToken, smem + a.ring, owned, mine, row0 + static_cast<int64_t>(rank) * owned, tile);
  __syncwarp();
  cluster_wait();
}

// What a call does, by its sizes alone: a cluster's CTAs share a tile's blocks of K, as many as give every SM one CTA
// at most (one row of 2048 x 9216, 72 tiles: 1 / 2 / 3 / 4 CTAs take 7.4 / 5.1 / 5.9 / 7.8 us, of 4096 x 2048, 16
// tiles: 4 / 6 / 8 take 4.3 / 4.2 / 4.0). That is not always the best number: where it shortens no CTA's part, or the
// clusters fill the card, fewer are faster (192 rows of 1024 x 1000 with 6 5.3 us, with 4 or 5 4.1; 64 of 2000 x 3000
// with 6 6.2, with 5 5.2; in 7 of 99 sizes by more than a tenth). A cluster lies within a group of SMs: of 4 there is room for 33 where a CTA
// takes an SM for itself, of 8 for 15, and one cluster too many costs a second round (64 rows of 4096 x 2048 with
// eight: 6.2 us where two fit an SM, 10.0 else). So all but the largest leave room for a second, and those have four.
// Tokens per tile: all of them up to 64 (gated 32). Beyond, tiles of 64 (32) or of twice as many, which read the
// weights less often but have only one CTA per SM: the ones with the smaller cost, about the ns of a call in a graph
// (96 rows of 4096 x 2048 take 6.6 and 8.2 us, 512 of 1024 x 1000 4.8 and 6.4; but 512 of 4096 x 2048 14.4 and 12.8.
// Gated, 128 rows of 2048 x 512 11.4 and 14.4 with the down product). Of the products a block takes about 0.42 and 0.46 us beside 3.7 and 5.8 for all the rest.
struct NarrowPlan {
  int tokens, splits, rows, most;  // rows: that a CTA quantises itself, at most, and (most) blocks of them
  int64_t cost;
  NarrowPlan(int64_t M, int64_t N, int blocks, bool gated) {
    rows = gated ? 32 : 64;
    most = gated ? kInline / 2 : kInline;
    split(M <= 16 ? 16 : M <= 32 ? 32 : rows, M, N, blocks, gated);
    if (M > rows) {
      const NarrowPlan few = *this;
      split(2 * rows, M, N, blocks, gated);
      if (few.cost <= cost) *this = few;
    }
  }
  void split(int of, int64_t M, int64_t N, int blocks, bool gated) {
    tokens = of;
    const bool large = tokens * (gated ? 2 : 1) > 64;
    const int64_t tiles = (N + 127) / 128 * ((M + tokens - 1) / tokens), room = sm_count() / tiles;
    splits = static_cast<int>(room < 1 ? 1 : room > kMostSplits ? kMostSplits : room);
    if (large) splits = tiles * 4 <= sm_count() * 7 / 8 ? 4 : splits > 2 ? 2 : splits;
    if (splits > blocks) splits = blocks;
    int64_t work = each(blocks) * ((tiles * splits + sm_count() - 1) / sm_count());  // blocks that an SM goes through
    if (splits > 2 && tiles * splits * 10 > sm_count() * 9) work += work / 2;         // the last clusters share their SMs
    cost = gated ? (large ? 6500 + 560 * work : 4000 + 520 * work) : large ? 5800 + 460 * work : 3700 + 420 * work;
  }
  int each(int blocks) const { return (blocks + splits - 1) / splits; }
  // Whether the CTAs can quantise rows of x themselves.
  bool quantises(int64_t M, int blocks) const {
    int power = 1;
    while (power < M && power < rows) power *= 2;
    return M <= rows && power * each(blocks) <= most && tokens * each(blocks) <= kInlineTokens;
  }
};

template <int MT, bool GATED, bool ROWS>
int launch_narrow(const CUtensorMap& x, const CUtensorMap& w, const CUtensorMap& u, NarrowArgs a, const NarrowPlan& plan, cudaStream_t st) {
  using L = Narrow<MT, GATED>;
  const int each = plan.each(a.blocks);
  // of an SM's 228 KB, 1 KB of which each CTA reserves (and some for the alignment of what is static)
  const size_t room = (L::kTwo ? 113 : 227) * 1024 - sizeof(NarrowControl<MT>) - 256;
  const int tiles_of_x = ROWS ? each : 0, live = static_cast<int>(a.M < MT ? a.M : MT);
  a.splits = plan.splits;
  a.stages = each < kNarrowStages ? each : kNarrowStages;
  while (a.stages > 1 && L::smem(a.stages, tiles_of_x, a.splits, live) > room) --a.stages;
  a.ring = L::ring(a.stages, tiles_of_x);
  size_t smem = L::smem(a.stages, tiles_of_x, a.splits, live);
  if (smem < kLeastSmem) smem = kLeastSmem;
  const void* kernel = reinterpret_cast<const void*>(fp8_narrow_kernel<MT, GATED, ROWS>);
  const int rc = allow_smem(kernel, smem);
  if (rc) return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(plan.splits * ((a.N + 127) / 128)), static_cast<unsigned>((a.M + MT - 1) / MT));
  cfg.blockDim = dim3(kNarrowThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = static_cast<unsigned>(plan.splits);
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  cudaError_t e = cudaLaunchKernelEx(&cfg, fp8_narrow_kernel<MT, GATED, ROWS>, x, w, u, a);
  if (e != cudaSuccess) return cuda_error(e, "fp8_narrow_kernel");
  count_launch();
  return QK_OK;
}

template <bool GATED>
int launch_narrow(bool rows, const CUtensorMap& x, const CUtensorMap& w, const CUtensorMap& u, const NarrowArgs& a, const NarrowPlan& plan,
                  cudaStream_t st) {
  if (plan.tokens == 16)
    return rows ? launch_narrow<16, GATED, true>(x, w, u, a, plan, st) : launch_narrow<16, GATED, false>(x, w, u, a, plan, st);
  if (plan.tokens == 32)
    return rows ? launch_narrow<32, GATED, true>(x, w, u, a, plan, st) : launch_narrow<32, GATED, false>(x, w, u, a, plan, st);
  if constexpr (GATED) {
    return launch_narrow<64, true, false>(x, w, u, a, plan, st);  // more rows than a CTA quantises
  } else {
    if (plan.tokens == 128) return launch_narrow<128, false, false>(x, w, u, a, plan, st);
    return rows ? launch_narrow<64, false, true>(x, w, u, a, plan, st) : launch_narrow<64, false, false>(x, w, u, a, plan, st);
  }
}

}  // namespace
}  // namespace qk
