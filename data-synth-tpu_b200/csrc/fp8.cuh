// Shared parts of the FP8 dense path: e4m3 codes with one FP32 scale for each block of 128 values.
#pragma once

#include "umma.cuh"

namespace qk {

constexpr int kFp8Block = 128;
constexpr float kFp8Most = 448.f;  // the largest e4m3 value
// The smallest maximum of a block that counts, 2^-100: blocks of zeros have codes of zero, and no quotient overflows.
constexpr uint32_t kFp8LeastBits = 0x0d800000u;

// Pairs of FP32 in one instruction.
__device__ __forceinline__ uint64_t f32x2(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void f32x2_split(uint64_t p, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(p));
}
__device__ __forceinline__ uint64_t f32x2_fma(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t f32x2_add(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t f32x2_mul(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// The two BF16 of a word.
__device__ __forceinline__ uint64_t f32x2_of(uint32_t w) { return f32x2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)); }

// |x| as an unsigned number: in the order of magnitudes, NaN above everything, so that the maximum of a block keeps it.
__device__ __forceinline__ uint32_t magnitude(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// How a block whose largest magnitude is `most` is quantised: code = e4m3(448 x / most), scale = most / 448.
// Ties between two codes are frequent where x and most are BF16 (their quotient is a short fraction then), and a
// product with a rounded reciprocal decides them by chance, so the quotient is corrected by its remainder (Markstein):
// q = n y, q + (n - q d) y with y near 1 / d. The remainder is exact, so a quotient that has a short fraction comes
// out exactly. n and d are 7/16 x and most / 1024: no product leaves FP32's range. An infinite maximum gives codes
// 0 (finite values) and NaN, a NaN gives NaN, as the division does.
struct Fp8Divisor {
  float d, y;
  __device__ explicit Fp8Divisor(uint32_t most_bits) {
    d = __uint_as_float(max(most_bits, kFp8LeastBits)) * 0x1p-10f;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(d));
    if (y == 0.f) d = 0.f;
  }
  // Two values -> two codes, the first in the low byte.
  __device__ __forceinline__ uint16_t codes(float a, float b) const {
    const uint64_t n = f32x2_mul(f32x2(a, b), f32x2(0.4375f, 0.4375f)), yy = f32x2(y, y);
    const uint64_t q = f32x2_mul(n, yy);
    float u, v;
    f32x2_split(f32x2_fma(f32x2_fma(q, f32x2(-d, -d), n), yy, q), u, v);
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(v), "f"(u));
    return r;
  }
  __device__ __forceinline__ uint32_t codes4(const float* f) const {
    return static_cast<uint32_t>(codes(f[0], f[1])) | static_cast<uint32_t>(codes(f[2], f[3])) << 16;
  }
};

// most / 448, rounded to nearest: a quotient corrected by its remainder as above (an infinite one has none).
__device__ __forceinline__ float fp8_scale(uint32_t most_bits) {
  const float m = __uint_as_float(max(most_bits, kFp8LeastBits)), q = m * (1.f / kFp8Most);
  const float r = fmaf(fmaf(-q, kFp8Most, m), 1.f / kFp8Most, q);
  return most_bits == 0x7f800000u ? q : r;
}

// The larger magnitude of two and of three FP32, NaN above everything (its bits too), in one instruction each.
__device__ __forceinline__ float abs_max(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(fabsf(a)), "f"(fabsf(b)));
  return r;
}
__device__ __forceinline__ float abs_max(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(fabsf(a)), "f"(fabsf(b)), "f"(fabsf(c)));
  return r;
}
// The bits of the largest magnitude of eight values, as FP32 and as packed BF16 (whose magnitudes are in the order of
// their bits).
__device__ __forceinline__ uint32_t most8(const float (&f)[8]) {
  return __float_as_uint(abs_max(abs_max(f[0], f[1], f[2]), abs_max(f[3], f[4], f[5]), abs_max(f[6], f[7])));
}
__device__ __forceinline__ uint32_t most8(const uint4& v) {
  constexpr uint32_t m = 0x7fff7fffu;
  const uint32_t w = __vmaxu2(__vmaxu2(v.x & m, v.y & m), __vmaxu2(v.z & m, v.w & m));
  return max(w << 16, w & 0xffff0000u);
}

// The largest of 16 lanes' (a block's: 8 values each) magnitudes, in all of them, for N blocks per half warp at once.
template <int N>
__device__ __forceinline__ void block_most(uint32_t (&most)[N]) {
  if (threadIdx.x & 16) {
#pragma unroll
    for (int i = 0; i < N; ++i) most[i] = __reduce_max_sync(0xffff0000u, most[i]);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) most[i] = __reduce_max_sync(0x0000ffffu, most[i]);
  }
  __syncwarp();
}
__device__ __forceinline__ uint32_t block_most(uint32_t most) {
  uint32_t m[1] = {most};
  block_most(m);
  return m[0];
}

}  // namespace qk
