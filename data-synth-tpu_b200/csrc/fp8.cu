// Quantisation of the FP8 dense path: e4m3 codes and FP32 scales of rows (blocks of 128 columns) and of
// weights (blocks of 128 x 128), and the residual add + RMSNorm whose output leaves as codes.
//
//   most = max(max |x| of the block, 2^-100); scale = most / 448; code = e4m3(448 x / most)
//
// All are bound by HBM: one pass, a block of a row in 16 lanes of 8 values each, whose maximum is one reduction.
// Measured: 32768 x 4096 BF16 66 us (407 MB, 6.2 TB/s, 94 % of the measured copy), 8192 x 4096 FP32 28 us (6.0 TB/s),
// the norm with a residual over 16384 x 2048 40 us (236 MB, 5.8 TB/s); 64 rows of 4096 1.4 us, the norm of 8 rows 1.6.
// FP32 of odd widths (8111 x 1111: 10.8 us, 4.2 TB/s) pays for single loads, a choice of this code. Weights, which are
// packed once: 8192 x 8192 BF16 48 us (201 MB, 4.2 TB/s), FP32 50 (6.7), 9216 x 2048 BF16 16.
#include "fp8.cuh"

namespace qk {

namespace {

constexpr int kThreads = 256;

// Eight values from `at` of a row whose first `width` exist; the others are zero.
template <bool F32, bool ALIGNED>
__device__ __forceinline__ void load8(const void* row, int at, int width, float (&f)[8]) {
  if (ALIGNED) {
    if (at >= width) {
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] = 0.f;
    } else if (F32) {
      const uint4 a = ld_guarded_v4(static_cast<const float*>(row) + at);
      const uint4 b = ld_guarded_v4(static_cast<const float*>(row) + at + 4);
#pragma unroll
      for (int j = 0; j < 4; ++j) f[j] = __uint_as_float(word(a, j)), f[4 + j] = __uint_as_float(word(b, j));
    } else {
      unpack8(ld_guarded_v4(static_cast<const uint16_t*>(row) + at), f);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      f[j] = 0.f;
      if (at + j < width) f[j] = F32 ? static_cast<const float*>(row)[at + j] : bf16_to_f32(static_cast<const uint16_t*>(row)[at + j]);
    }
  }
}

// Eight codes, of which `left` belong to the row: nothing is written past its width.
__device__ __forceinline__ void store8(uint8_t* to, uint2 codes, int left) {
  if (left >= 8) {
    *reinterpret_cast<uint2*>(to) = codes;
  } else {
    for (int j = 0; j < left; ++j) to[j] = static_cast<uint8_t>((j < 4 ? codes.x : codes.y) >> (8 * (j & 3)));
  }
}

struct RowsArgs {
  const void* x;
  int64_t stride, ld;
  int64_t rows;
  int width, blocks;
  uint8_t* codes;
  float* scales;  // [blocks][rows]
};

// Half a warp per block of a row; a warp has a row and 2 U consecutive blocks, all asked for at once, a CTA eight rows,
// so that it writes whole sectors of scales. Rows that do not begin on 16 bytes (or FP32 or BF16 of odd widths) are
// read a value per lane and turned around through shared memory, which is a twelfth of the cache lookups of eight
// neighbouring values per lane.
template <bool F32, bool ALIGNED, int U>
__global__ void __launch_bounds__(kThreads) fp8_rows_kernel(RowsArgs a) {
  __shared__ __align__(16) uint8_t turned[ALIGNED ? 1 : kThreads / 16][ALIGNED ? 1 : kFp8Block];
  const int lane = threadIdx.x & 31, in = lane & 15;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * (kThreads / 32) + (threadIdx.x >> 5);
  const int block0 = blockIdx.y * (2 * U) + (lane >> 4);
  pdl_wait();
  pdl_trigger();
  if (row >= a.rows) return;
  const void* from = F32 ? static_cast<const void*>(static_cast<const float*>(a.x) + row * a.stride)
                         : static_cast<const void*>(static_cast<const uint16_t*>(a.x) + row * a.stride);
  float f[U][8];
  uint32_t most[U];
  if constexpr (ALIGNED && !F32) {
    uint4 v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int at = (block0 + 2 * u) * kFp8Block + in * 8;
      v[u] = at < a.width ? ld_guarded_v4(static_cast<const uint16_t*>(from) + at) : make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      most[u] = most8(v[u]);
      unpack8(v[u], f[u]);
    }
  } else {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int at = (block0 + 2 * u) * kFp8Block;
      if (ALIGNED) {
        load8<F32, true>(from, at + in * 8, a.width, f[u]);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int k = at + j * 16 + in;
          f[u][j] = 0.f;
          if (k < a.width) f[u][j] = F32 ? static_cast<const float*>(from)[k] : bf16_to_f32(static_cast<const uint16_t*>(from)[k]);
        }
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) most[u] = most8(f[u]);
  }
  block_most(most);
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int block = block0 + 2 * u, at = block * kFp8Block + in * 8;
    const Fp8Divisor by(most[u]);
    uint2 codes = make_uint2(by.codes4(f[u]), by.codes4(f[u] + 4));
    if (!ALIGNED) {
      uint8_t* mine = turned[threadIdx.x >> 4];
      __syncwarp();
#pragma unroll
      for (int j = 0; j < 8; ++j) mine[j * 16 + in] = static_cast<uint8_t>((j < 4 ? codes.x : codes.y) >> (8 * (j & 3)));
      __syncwarp();
      codes = *reinterpret_cast<const uint2*>(mine + in * 8);
    }
    store8(a.codes + row * a.ld + at, codes, a.width - at);
    if (block < a.blocks && in == 0) a.scales[static_cast<int64_t>(block) * a.rows + row] = fp8_scale(most[u]);
  }
}

// A CTA per block of 128 x 128 weights: 8 rows by half warps, 16 times over.
template <bool F32, bool ALIGNED>
__global__ void __launch_bounds__(kThreads) fp8_blocks_kernel(RowsArgs a) {
  __shared__ uint32_t red[kThreads / 32];
  const int lane = threadIdx.x & 31, half = threadIdx.x >> 4;
  const int at = blockIdx.x * kFp8Block + (lane & 15) * 8;
  pdl_wait();
  pdl_trigger();
  constexpr int kTimes = kFp8Block / (kThreads / 16);
  float f[kTimes][8];
  uint32_t most = 0;
#pragma unroll
  for (int i = 0; i < kTimes; ++i) {
    const int64_t row = static_cast<int64_t>(blockIdx.y) * kFp8Block + i * (kThreads / 16) + half;
    const void* from = F32 ? static_cast<const void*>(static_cast<const float*>(a.x) + row * a.stride)
                           : static_cast<const void*>(static_cast<const uint16_t*>(a.x) + row * a.stride);
    load8<F32, ALIGNED>(from, at, row < a.rows ? a.width : 0, f[i]);
    most = max(most, most8(f[i]));
  }
  most = __reduce_max_sync(0xffffffffu, most);
  if (lane == 0) red[threadIdx.x >> 5] = most;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) most = max(most, red[w]);
  const Fp8Divisor by(most);
#pragma unroll
  for (int i = 0; i < kTimes; ++i) {
    const int64_t row = static_cast<int64_t>(blockIdx.y) * kFp8Block + i * (kThreads / 16) + half;
    if (row < a.rows) store8(a.codes + row * a.ld + at, make_uint2(by.codes4(f[i]), by.codes4(f[i] + 4)), a.width - at);
  }
  if (threadIdx.x == 0) a.scales[static_cast<int64_t>(blockIdx.y) * gridDim.x + blockIdx.x] = fp8_scale(most);
}

struct NormArgs {
  const uint16_t *x, *y, *gamma;
  int64_t rows, ld;
  int width;
  float eps;
  uint16_t* sum;
  uint8_t* codes;
  float* scales;
};

// Eight values of a row's s and p = s gamma from `at`: the sum is kept, p comes out, the squares are added to `ss`.
__device__ __forceinline__ void norm8(const NormArgs& a, int64_t row, int at, uint4 x, const uint4& y, const uint4& gamma, float (&p)[8],
                                      uint64_t& ss) {
  if (a.y) {
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float u, v;
      f32x2_split(f32x2_add(f32x2_of(word(x, j)), f32x2_of(word(y, j))), u, v);
      w[j] = pack_bf16x2(u, v);
    }
    x = make_uint4(w[0], w[1], w[2], w[3]);
    if (at < a.width) *reinterpret_cast<uint4*>(a.sum + row * a.width + at) = x;
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint64_t s = f32x2_of(word(x, j));
    ss = f32x2_fma(s, s, ss);
    f32x2_split(f32x2_mul(s, f32x2_of(word(gamma, j))), p[2 * j], p[2 * j + 1]);
  }
}

__device__ __forceinline__ uint4 load16(const uint16_t* p, int at, int width) {
  return at < width ? ld_guarded_v4(p + at) : make_uint4(0, 0, 0, 0);
}
// x and y may be written as the sum: not through the read-only path.
__device__ __forceinline__ uint4 load16_rw(const uint16_t* p, int at, int width) {
  return at < width ? *reinterpret_cast<const uint4*>(p + at) : make_uint4(0, 0, 0, 0);
}

// With p = s gamma (exact in FP32) the normed row is r p, r = rsqrt(mean s^2 + eps): r moves no code, so the codes
// leave without waiting for the sum of squares and r goes into the scales. Few rows: a CTA each.
__global__ void __launch_bounds__(kRowBlock) fp8_norm_kernel(NormArgs a) {
  __shared__ float red[kRowBlock / 32];
  const int64_t row = blockIdx.x;
  const int lane = threadIdx.x & 31;
  pdl_wait();
  pdl_trigger();
  uint64_t ss = 0;
  uint32_t most[kRowChunks];
#pragma unroll
  for (int c = 0; c < kRowChunks; ++c) {
    const int at = (threadIdx.x + c * kRowBlock) * 8;
    most[c] = 0;
    if ((at & ~255) >= a.width) continue;  // the same for the warp
    const uint4 x = load16_rw(a.x + row * a.width, at, a.width), g = load16(a.gamma, at, a.width);
    const uint4 y = a.y ? load16_rw(a.y + row * a.width, at, a.width) : x;
    float p[8];
    norm8(a, row, at, x, y, g, p, ss);
    most[c] = block_most(most8(p));
    const Fp8Divisor by(most[c]);
    if (at < a.width) *reinterpret_cast<uint2*>(a.codes + row * a.ld + at) = make_uint2(by.codes4(p), by.codes4(p + 4));
  }
  float even, odd;
  f32x2_split(ss, even, odd);
  const float r = rsqrtf(__fadd_rn(__fdiv_rn(block_sum(even + odd, red), static_cast<float>(a.width)), a.eps));
  if ((lane & 15) == 0) {
#pragma unroll
    for (int c = 0; c < kRowChunks; ++c) {
      const int at = (threadIdx.x + c * kRowBlock) * 8;
      if (at < a.width) a.scales[static_cast<int64_t>(at / kFp8Block) * a.rows + row] = fp8_scale(most[c]) * r;
    }
  }
}

// Many rows: a warp each, kNormAhead loads of either addend in flight, no barrier. The sums are in another order.
// 64 registers, for four CTAs per SM: 4096 rows of 8192 take 43 us (76 registers: 51), 16384 of 2048 40 (41). Rows of 512
// and less have two loads: 16384 of 512 take 13 us, with four 17.
template <int kNormAhead>
__global__ void __launch_bounds__(kThreads, 4) fp8_norm_rows_kernel(NormArgs a) {
  __shared__ float scale[kThreads / 32][kMaxRowWidth / kFp8Block];
  const int64_t row = static_cast<int64_t>(blockIdx.x) * (kThreads / 32) + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  pdl_wait();
  pdl_trigger();
  if (row >= a.rows) return;
  float* mine = scale[threadIdx.x >> 5];
  uint64_t ss = 0;
#pragma unroll 1
  for (int at0 = 0; at0 < a.width; at0 += kNormAhead * 256) {
    uint4 x[kNormAhead], y[kNormAhead], g[kNormAhead];
#pragma unroll
    for (int c = 0; c < kNormAhead; ++c) {
      const int at = at0 + c * 256 + lane * 8;
      x[c] = load16_rw(a.x + row * a.width, at, a.width);
      y[c] = a.y ? load16_rw(a.y + row * a.width, at, a.width) : x[c];
      g[c] = load16(a.gamma, at, a.width);
    }
    float p[kNormAhead][8];
    uint32_t most[kNormAhead];
#pragma unroll
    for (int c = 0; c < kNormAhead; ++c) {
      const int at = at0 + c * 256 + lane * 8;
      norm8(a, row, at, x[c], y[c], g[c], p[c], ss);
      most[c] = most8(p[c]);
    }
    block_most(most);
#pragma unroll
    for (int c = 0; c < kNormAhead; ++c) {
      const int at = at0 + c * 256 + lane * 8;
      const Fp8Divisor by(most[c]);
      if (at < a.width) {
        *reinterpret_cast<uint2*>(a.codes + row * a.ld + at) = make_uint2(by.codes4(p[c]), by.codes4(p[c] + 4));
        if ((lane & 15) == 0) mine[at / kFp8Block] = fp8_scale(most[c]);
      }
    }
  }
  float even, odd;
  f32x2_split(ss, even, odd);
  float sum = even + odd;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  const float r = rsqrtf(__fadd_rn(__fdiv_rn(sum, static_cast<float>(a.width)), a.eps));
  __syncwarp();
  for (int b = lane; b < (a.width + kFp8Block - 1) / kFp8Block; b += 32) a.scales[static_cast<int64_t>(b) * a.rows + row] = mine[b] * r;
}

template <typename Kernel>
int launch(Kernel kernel, dim3 grid, cudaStream_t st, const RowsArgs& a, const char* name) {
  cudaError_t e = launch_dependent(kernel, grid, dim3(kThreads), 0, st, a);
  if (e != cudaSuccess) return cuda_error(e, name);
  count_launch();
  return QK_OK;
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace
}  // namespace qk

using namespace qk;

extern "C" {

int qk_fp8_quantize(const void* x, int in_dtype, int64_t x_stride, int64_t rows, int64_t width, uint8_t* codes, int64_t ld,
                    float* scales, qk_stream_t stream) {
  QK_REQUIRE(in_dtype == QK_OUT_F32 || in_dtype == QK_OUT_BF16, "x must be FP32 or BF16");
  QK_REQUIRE(rows >= 0 && rows < (1ll << 34) && width >= 1 && width < (1ll << 31) - 256 && x_stride >= width,
             "invalid rows, width or stride");
  QK_REQUIRE(ld >= width && ld % 16 == 0, "rows of codes must be a multiple of 16 bytes apart and not overlap");
  if (rows == 0) return QK_OK;
  QK_REQUIRE(x && codes && scales, "null pointer");
  QK_REQUIRE(aligned16(codes), "codes must be 16-byte aligned");
  const int f32 = in_dtype == QK_OUT_F32, size = f32 ? 4 : 2;
  QK_REQUIRE((reinterpret_cast<uintptr_t>(x) % size) == 0 && (reinterpret_cast<uintptr_t>(scales) & 3) == 0, "misaligned pointer");
  RowsArgs a{x, x_stride, ld, rows, static_cast<int>(width), static_cast<int>((width + 127) / 128), codes, scales};
  const bool aligned = aligned16(x) && x_stride * size % 16 == 0 && width % 8 == 0;
  const int64_t ctas = (rows + 7) / 8;
  QK_REQUIRE(ctas < (1ll << 31) && a.blocks <= 65535 * 8, "too many rows or columns");  // what a grid holds
  cudaStream_t st = as_stream(stream);
  // four blocks per half warp where there is work for all SMs all the same
  const bool many = ctas * a.blocks >= 64ll * sm_count() || a.blocks > 65535 * 2;
  const dim3 grid(static_cast<unsigned>(ctas), many ? (a.blocks + 7) / 8 : (a.blocks + 1) / 2);
  const char* name = "fp8_rows_kernel";
  if (f32) {
    if (aligned) return many ? launch(fp8_rows_kernel<true, true, 4>, grid, st, a, name) : launch(fp8_rows_kernel<true, true, 1>, grid, st, a, name);
    return many ? launch(fp8_rows_kernel<true, false, 4>, grid, st, a, name) : launch(fp8_rows_kernel<true, false, 1>, grid, st, a, name);
  }
  if (aligned) return many ? launch(fp8_rows_kernel<false, true, 4>, grid, st, a, name) : launch(fp8_rows_kernel<false, true, 1>, grid, st, a, name);
  return many ? launch(fp8_rows_kernel<false, false, 4>, grid, st, a, name) : launch(fp8_rows_kernel<false, false, 1>, grid, st, a, name);
}

int qk_fp8_quantize_blocks(const void* w, int in_dtype, int64_t w_stride, int64_t rows, int64_t width, uint8_t* codes, int64_t ld,
                           float* scales, qk_stream_t stream) {
  QK_REQUIRE(in_dtype == QK_OUT_F32 || in_dtype == QK_OUT_BF16, "w must be FP32 or BF16");
  QK_REQUIRE(rows >= 0 && width >= 1 && width < (1ll << 31) - 256 && w_stride >= width, "invalid rows, width or stride");
  QK_REQUIRE(ld >= width && ld % 16 == 0, "rows of codes must be a multiple of 16 bytes apart and not overlap");
  QK_REQUIRE(rows <= 65535ll * 128, "too many rows");
  if (rows == 0) return QK_OK;
  QK_REQUIRE(w && codes && scales, "null pointer");
  QK_REQUIRE(aligned16(codes), "codes must be 16-byte aligned");
  const int f32 = in_dtype == QK_OUT_F32, size = f32 ? 4 : 2;
  QK_REQUIRE((reinterpret_cast<uintptr_t>(w) % size) == 0 && (reinterpret_cast<uintptr_t>(scales) & 3) == 0, "misaligned pointer");
  RowsArgs a{w, w_stride, ld, rows, static_cast<int>(width), static_cast<int>((width + 127) / 128), codes, scales};
  const bool aligned = aligned16(w) && w_stride * size % 16 == 0 && width % 8 == 0;
  const dim3 grid(a.blocks, static_cast<unsigned>((rows + 127) / 128));
  cudaStream_t st = as_stream(stream);
  if (f32) return aligned ? launch(fp8_blocks_kernel<true, true>, grid, st, a, "fp8_blocks_kernel")
                          : launch(fp8_blocks_kernel<true, false>, grid, st, a, "fp8_blocks_kernel");
  return aligned ? launch(fp8_blocks_kernel<false, true>, grid, st, a, "fp8_blocks_kernel")
                 : launch(fp8_blocks_kernel<false, false>, grid, st, a, "fp8_blocks_kernel");
}

int qk_fp8_rms_norm(const uint16_t* x, const uint16_t* y, const uint16_t* gamma, int64_t rows, int width, float eps, uint16_t* x_out,
                    uint8_t* codes, int64_t ld, float* scales, qk_stream_t stream) {
  QK_REQUIRE(rows >= 0 && rows < (1ll << 31) && width >= 8 && width % 8 == 0 && width <= kMaxRowWidth,
             "width must be a multiple of 8, 8192 at most");
  QK_REQUIRE(ld >= width && ld % 16 == 0, "rows of codes must be a multiple of 16 bytes apart and not overlap");
  if (rows == 0) return QK_OK;
  QK_REQUIRE(x && gamma && codes && scales && (!y || x_out), "null pointer");
  QK_REQUIRE(aligned16(x) && aligned16(y) && aligned16(gamma) && aligned16(x_out) && aligned16(codes), "pointers must be 16-byte aligned");
  QK_REQUIRE((reinterpret_cast<uintptr_t>(scales) & 3) == 0, "misaligned scales");
  NormArgs a{x, y, gamma, rows, ld, width, eps, x_out, codes, scales};
  const dim3 warps(static_cast<unsigned>((rows + 7) / 8));
  cudaStream_t st = as_stream(stream);
  cudaError_t e = rows < 8ll * sm_count() ? launch_dependent(fp8_norm_kernel, dim3(static_cast<unsigned>(rows)), dim3(kRowBlock), 0, st, a)
                  : width > 512           ? launch_dependent(fp8_norm_rows_kernel<4>, warps, dim3(kThreads), 0, st, a)
                                          : launch_dependent(fp8_norm_rows_kernel<2>, warps, dim3(kThreads), 0, st, a);
  if (e != cudaSuccess) return cuda_error(e, "fp8_norm_kernel");
  count_launch();
  return QK_OK;
}

}  // extern "C"
