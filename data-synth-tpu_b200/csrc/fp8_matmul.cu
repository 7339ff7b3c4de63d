// Products of FP8 activations and weights on the tcgen05 tensor core (kind::f8f6f4):
//
//   out[m, n] = sum_b xs[b, m] ws[n / 128, b] sum_{k in block b} xc[m, k] wc[n, k]
//
// and the gated pair of them, h = silu(x Wg^T) * (x Wu^T), quantised as the next product reads it.
#include "fp8_narrow.cuh"
#include "fp8_wide.cuh"

namespace qk {
namespace {

// Sizes that a call takes: every product of two of them fits 64 bits, and a grid holds the tiles.
bool sizes_fit(int64_t M, int64_t K, int64_t N) {
  constexpr int64_t kMost = (1ll << 31) - 256;
  return M < kMost && N < kMost && K < kMost && ((M + 127) / 128) * ((N + 127) / 128) < (1ll << 28);
}

int check_weights(int64_t M, int64_t K, const uint8_t* w, int64_t w_ld, const float* ws, int64_t N, const void* out) {
  QK_REQUIRE(M >= 0 && N >= 1 && K >= 1, "invalid rows, columns or width");
  QK_REQUIRE(sizes_fit(M, K, N), "sizes must stay below 2^31 - 256 and tiles of 128 x 128 below 2^28");
  QK_REQUIRE(w_ld >= K && w_ld % 16 == 0, "rows of codes must be a multiple of 16 bytes apart");
  if (M == 0) return QK_OK;
  QK_REQUIRE(w && ws && out, "null pointer");
  QK_REQUIRE(aligned16(w) && (reinterpret_cast<uintptr_t>(ws) & 3) == 0, "codes must be 16-byte aligned, scales 4-byte");
  return QK_OK;
}

int check_operands(const uint8_t* x, int64_t x_ld, const float* xs, int64_t M, int64_t K, const uint8_t* w, int64_t w_ld, const float* ws,
                   int64_t N, const void* out) {
  const int rc = check_weights(M, K, w, w_ld, ws, N, out);
  if (rc || M == 0) return rc;
  QK_REQUIRE(x_ld >= K && x_ld % 16 == 0, "rows of codes must be a multiple of 16 bytes apart");
  QK_REQUIRE(x && xs, "null pointer");
  QK_REQUIRE(aligned16(x) && (reinterpret_cast<uintptr_t>(xs) & 3) == 0, "codes must be 16-byte aligned, scales 4-byte");
  return QK_OK;
}

int check_rows(const void* x, int in_dtype, int64_t stride, int64_t M, int64_t K) {
  QK_REQUIRE(in_dtype == QK_OUT_F32 || in_dtype == QK_OUT_BF16, "x must be FP32 or BF16");
  QK_REQUIRE(M >= 0 && K >= 1 && stride >= K, "invalid rows, width or stride");
  QK_REQUIRE(M == 0 || (x && reinterpret_cast<uintptr_t>(x) % (in_dtype == QK_OUT_F32 ? 4 : 2) == 0), "misaligned or null x");
  return QK_OK;
}

// Which form a call takes: the one with the smaller of these costs, about its ns in a graph (fitted to 65 to 4096 rows, K 256
// to 8192, N 128 to 12288); up to 64 rows (gated 32) the narrow one, whose CTAs may quantise them. The wide form has
// tiles of 256 x 256, or half as wide where that fills no more rounds of the pairs of SMs. All sides, us, narrow /
// half / whole: 128 rows of 2048 x 9216 9.3 / 8.8 / 11.2, 256 of 4096 x 2048 9.2 / 13.0 / 16.5, 512 12.8 / 13.1 / 16.6,
// 1024 of 8192 x 2048 34 / 23 / 29, 512 of 2048 x 9216 25 / 14.3 / 12.0, 2048 of 4096 x 2048 38 / 23.5 / 18.0. A gated
// pair with its down product in the same form, narrow / wide: 256 rows of 2048 x 512 11.9 / 18.6, 512 of 2048 x 1536
// 23.7 / 23.1; 128 of 2048 x 6144 28.2 / 37.6, and 26.2 with the down product narrow, which is what is taken.
// Of 110 sizes of 65 to 2048 rows the form taken is 0.1 % slower than the best in the median, 15 % at most
// (384 rows of 256 x 512), and more than 10 % in 8.
struct WidePlan {
  bool half;
  int64_t cost;
  WidePlan(int64_t M, int64_t N, int blocks, bool gated) {
    const int64_t pairs = sm_count() / 2, m = (M + 255) / 256, n = (N + 127) / 128;
    const int64_t halves = (m * n + pairs - 1) / pairs, wholes = gated ? halves : (m * ((n + 1) / 2) + pairs - 1) / pairs;
    const int64_t cost_half = 3200 + blocks * (halves == 1 ? 330 : 400 * halves);
    const int64_t cost_whole = 4000 + blocks * (wholes > 1 ? 570 * wholes : gated ? 500 : 450);
    half = !gated && cost_half < cost_whole;
    cost = half ? cost_half : cost_whole;
  }
};

// Half of a feed-forward block (u not NULL, codes out) or a product (u NULL) of codes.
struct Weights {
  const uint8_t* codes;
  int64_t ld;
  const float* scales;
};

int product(const uint8_t* x, int64_t x_ld, const float* xs, int64_t M, int64_t K, const Weights& w, const Weights* u, int64_t N, bool f32,
            void* out, int64_t ld, float* out_scales, cudaStream_t st) {
  const int blocks = static_cast<int>((K + 127) / 128), n_blocks = static_cast<int>((N + 127) / 128);
  const bool vectors = !u && aligned16(out) && N * (f32 ? 4 : 2) % 16 == 0;
  CUtensorMap xm, wm, um;
  bool ok;
  const NarrowPlan plan(M, N, blocks, u != nullptr);
  if (M <= plan.rows || plan.cost <= WidePlan(M, N, blocks, u != nullptr).cost) {
    ok = encode(&xm, x, M, K, x_ld, plan.tokens) && encode(&wm, w.codes, N, K, w.ld, 128) && (!u || encode(&um, u->codes, N, K, u->ld, 128));
    if (!ok) return set_error(QK_ERR_CUDA, "cuTensorMapEncodeTiled is unavailable or refused the codes");
    NarrowArgs a{};
    a.M = M;
    a.N = static_cast<int>(N);
    a.blocks = blocks;
    a.xs = xs;
    a.ws = w.scales;
    a.us = u ? u->scales : nullptr;
    a.out = out;
    a.ld = ld;
    a.out_scales = out_scales;
    a.f32 = f32;
    a.vectors = vectors;
    return u ? launch_narrow<true>(false, xm, wm, um, a, plan, st) : launch_narrow<false>(false, xm, wm, wm, a, plan, st);
  }
  const WidePlan wide(M, N, blocks, u != nullptr);
  ok = encode(&xm, x, M, K, x_ld, kHalf) && encode(&wm, w.codes, N, K, w.ld, wide.half ? 32 : 64) &&
       (!u || encode(&um, u->codes, N, K, u->ld, 64));
  if (!ok) return set_error(QK_ERR_CUDA, "cuTensorMapEncodeTiled is unavailable or refused the codes");
  WideArgs a{};
  a.M = M;
  a.N = static_cast<int>(N);
  a.blocks = blocks;
  a.n_blocks = n_blocks;
  a.tiles_m = static_cast<int>((M + kTileM - 1) / kTileM);
  a.tiles_n = u || wide.half ? n_blocks : static_cast<int>((N + 255) / 256);
  a.xs = xs;
  a.ws = w.scales;
  a.us = u ? u->scales : nullptr;
  a.out = out;
  a.ld = ld;
  a.out_scales = out_scales;
  a.f32 = f32;
  a.copies = vectors || u;
  CUtensorMap om = xm;
  if (u) ok = encode(&om, out, CU_TENSOR_MAP_DATA_TYPE_UINT8, M, N, ld, 32, 64, CU_TENSOR_MAP_SWIZZLE_64B);
  else if (vectors)
    ok = encode(&om, out, f32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, M, N, N * (f32 ? 4 : 2), 32, f32 ? 32 : 64,
                CU_TENSOR_MAP_SWIZZLE_128B);
  if (!ok) return set_error(QK_ERR_CUDA, "cuTensorMapEncodeTiled is unavailable or refused the output");
  if (u) return launch_wide<true, 128>(xm, wm, um, om, a, st);
  return wide.half ? launch_wide<false, 64>(xm, wm, wm, om, a, st) : launch_wide<false, 128>(xm, wm, wm, om, a, st);
}

// The same from rows of BF16 or FP32, which a narrow product of BF16 quantises itself where it can; else into `room`
// (row_bytes of it).
size_t row_bytes(int64_t M, int64_t K) {
  const size_t codes = static_cast<size_t>(M) * ((K + 15) / 16 * 16), scales = static_cast<size_t>(M) * ((K + 127) / 128) * 4;
  return (codes + 255) / 256 * 256 + (scales + 255) / 256 * 256;
}

// Whether a product of BF16 rows quantises them itself: by the sizes alone, so that the workspace's size is.
bool quantises(int in_dtype, int64_t M, int64_t K, int64_t N, bool gated) {
  const int blocks = static_cast<int>((K + 127) / 128);
  return in_dtype == QK_OUT_BF16 && K % 8 == 0 && M <= 64 && NarrowPlan(M, N, blocks, gated).quantises(M, blocks);
}
size_t room_for(int in_dtype, int64_t M, int64_t K, int64_t N, bool gated) {
  return quantises(in_dtype, M, K, N, gated) ? 0 : row_bytes(M, K);
}

int product_of_rows(const void* x, int in_dtype, int64_t x_stride, int64_t M, int64_t K, const Weights& w, const Weights* u, int64_t N,
                    bool f32, void* out, int64_t ld, float* out_scales, uint8_t* room, cudaStream_t st) {
  if (quantises(in_dtype, M, K, N, u != nullptr)) {
    QK_REQUIRE(aligned16(x) && x_stride % 8 == 0, "few rows of x must begin on 16 bytes");
    const int blocks = static_cast<int>((K + 127) / 128);
    const NarrowPlan plan(M, N, blocks, u != nullptr);
    CUtensorMap wm, um;
    if (!encode(&wm, w.codes, N, K, w.ld, 128) || (u && !encode(&um, u->codes, N, K, u->ld, 128)))
      return set_error(QK_ERR_CUDA, "cuTensorMapEncodeTiled is unavailable or refused the codes");
    NarrowArgs a{};
    a.M = M;
    a.N = static_cast<int>(N);
    a.blocks = blocks;
    a.x = static_cast<const uint16_t*>(x);
    a.x_stride = x_stride;
    a.width = static_cast<int>(K);
    while (1 << a.row_shift < M) ++a.row_shift;
    a.ws = w.scales;
    a.us = u ? u->scales : nullptr;
    a.out = out;
    a.ld = ld;
    a.out_scales = out_scales;
    a.f32 = f32;
    a.vectors = !u && aligned16(out) && N * (f32 ? 4 : 2) % 16 == 0;
    return u ? launch_narrow<true>(true, wm, wm, um, a, plan, st) : launch_narrow<false>(true, wm, wm, wm, a, plan, st);
  }
  const int64_t x_ld = (K + 15) / 16 * 16;
  float* scales = reinterpret_cast<float*>(room + (static_cast<size_t>(M) * x_ld + 255) / 256 * 256);
  const int rc = qk_fp8_quantize(x, in_dtype, x_stride, M, K, room, x_ld, scales, st);
  return rc ? rc : product(room, x_ld, scales, M, K, w, u, N, f32, out, ld, out_scales, st);
}

// A wait as the products have it, for an arrival that never comes, and its report.
__global__ void fp8_expire_kernel(int polls) {
  __shared__ uint64_t bar;
  if (threadIdx.x == 0) {
    mbar_init(&bar, 1);
    fence_mbar_init();
  }
  __syncwarp();
  if (!__all_sync(0xffffffffu, mbar_wait_bounded(&bar, 0, static_cast<uint32_t>(polls)))) atomicExch(&g_fp8_status, QK_ERR_TIMEOUT);
}

int check_room(const void* room, size_t bytes, size_t need) {
  if (need && (!room || bytes < need)) return set_error(QK_ERR_WORKSPACE, "the FP8 product needs a workspace of %zu bytes, got %zu", need, bytes);
  QK_REQUIRE((reinterpret_cast<uintptr_t>(room) & 255) == 0, "workspace must be 256-byte aligned");
  return QK_OK;
}

}  // namespace
}  // namespace qk

using namespace qk;

extern "C" {

int qk_fp8_matmul(const uint8_t* x, int64_t x_ld, const float* x_scales, int64_t M, int64_t K, const uint8_t* w, int64_t w_ld,
                  const float* w_scales, int64_t N, int out_dtype, void* out, qk_stream_t stream) {
  QK_REQUIRE(out_dtype == QK_OUT_F32 || out_dtype == QK_OUT_BF16, "out must be FP32 or BF16");
  const int rc = check_operands(x, x_ld, x_scales, M, K, w, w_ld, w_scales, N, out);
  if (rc || M == 0) return rc;
  QK_REQUIRE(reinterpret_cast<uintptr_t>(out) % (out_dtype == QK_OUT_F32 ? 4 : 2) == 0, "misaligned out");
  return product(x, x_ld, x_scales, M, K, Weights{w, w_ld, w_scales}, nullptr, N, out_dtype == QK_OUT_F32, out, 0, nullptr,
                 as_stream(stream));
}

int qk_fp8_gated(const uint8_t* x, int64_t x_ld, const float* x_scales, int64_t M, int64_t K, const uint8_t* gate, int64_t gate_ld,
                 const float* gate_scales, const uint8_t* up, int64_t up_ld, const float* up_scales, int64_t N, uint8_t* codes, int64_t ld,
                 float* scales, qk_stream_t stream) {
  int rc = check_operands(x, x_ld, x_scales, M, K, gate, gate_ld, gate_scales, N, codes);
  if (!rc) rc = check_operands(x, x_ld, x_scales, M, K, up, up_ld, up_scales, N, codes);
  if (rc || M == 0) return rc;
  QK_REQUIRE(ld >= N && ld % 16 == 0, "rows of codes must be a multiple of 16 bytes apart and not overlap");
  QK_REQUIRE(aligned16(codes) && scales && (reinterpret_cast<uintptr_t>(scales) & 3) == 0, "misaligned or null output");
  const Weights u{up, up_ld, up_scales};
  return product(x, x_ld, x_scales, M, K, Weights{gate, gate_ld, gate_scales}, &u, N, false, codes, ld, scales, as_stream(stream));
}

size_t qk_fp8_linear_workspace_bytes(int in_dtype, int64_t M, int64_t K, int64_t N) {
  return M > 0 && K > 0 && N > 0 && sizes_fit(M, K, N) ? room_for(in_dtype, M, K, N, false) : 0;
}

int qk_fp8_linear(const void* x, int in_dtype, int64_t x_stride, int64_t M, int64_t K, const uint8_t* w, int64_t w_ld,
                  const float* w_scales, int64_t N, int out_dtype, void* out, void* workspace, size_t workspace_bytes,
                  qk_stream_t stream) {
  QK_REQUIRE(out_dtype == QK_OUT_F32 || out_dtype == QK_OUT_BF16, "out must be FP32 or BF16");
  int rc = check_rows(x, in_dtype, x_stride, M, K);
  if (!rc) rc = check_weights(M, K, w, w_ld, w_scales, N, out);
  if (rc || M == 0) return rc;
  QK_REQUIRE(reinterpret_cast<uintptr_t>(out) % (out_dtype == QK_OUT_F32 ? 4 : 2) == 0, "misaligned out");
  rc = check_room(workspace, workspace_bytes, room_for(in_dtype, M, K, N, false));
  if (rc) return rc;
  return product_of_rows(x, in_dtype, x_stride, M, K, Weights{w, w_ld, w_scales}, nullptr, N, out_dtype == QK_OUT_F32, out, 0, nullptr,
                         static_cast<uint8_t*>(workspace), as_stream(stream));
}

size_t qk_fp8_ffn_workspace_bytes(int in_dtype, int64_t M, int64_t K, int64_t inner) {
  return M > 0 && K > 0 && inner > 0 && sizes_fit(M, K, inner) ? room_for(in_dtype, M, K, inner, true) + row_bytes(M, inner) : 0;
}

int qk_fp8_ffn(const void* x, int in_dtype, int64_t x_stride, int64_t M, int64_t K, const uint8_t* gate, int64_t gate_ld,
               const float* gate_scales, const uint8_t* up, int64_t up_ld, const float* up_scales, int64_t inner, const uint8_t* down,
               int64_t down_ld, const float* down_scales, int64_t N, uint16_t* out, void* workspace, size_t workspace_bytes,
               qk_stream_t stream) {
  int rc = check_rows(x, in_dtype, x_stride, M, K);
  if (!rc) rc = check_weights(M, K, gate, gate_ld, gate_scales, inner, out);
  if (!rc) rc = check_weights(M, K, up, up_ld, up_scales, inner, out);
  if (!rc) rc = check_weights(M, inner, down, down_ld, down_scales, N, out);
  if (rc || M == 0) return rc;
  QK_REQUIRE((reinterpret_cast<uintptr_t>(out) & 1) == 0, "misaligned out");
  const size_t for_x = room_for(in_dtype, M, K, inner, true);
  rc = check_room(workspace, workspace_bytes, for_x + row_bytes(M, inner));
  if (rc) return rc;
  cudaStream_t st = as_stream(stream);
  uint8_t* h = static_cast<uint8_t*>(workspace) + for_x;
  const int64_t ld = (inner + 15) / 16 * 16;
  float* h_scales = reinterpret_cast<float*>(h + (static_cast<size_t>(M) * ld + 255) / 256 * 256);
  const Weights u{up, up_ld, up_scales};
  rc = product_of_rows(x, in_dtype, x_stride, M, K, Weights{gate, gate_ld, gate_scales}, &u, inner, false, h, ld, h_scales,
                       static_cast<uint8_t*>(workspace), st);
  if (rc) return rc;
  return product(h, ld, h_scales, M, inner, Weights{down, down_ld, down_scales}, nullptr, N, false, out, 0, nullptr, st);
}

int qk_fp8_expire(int polls, qk_stream_t stream) {
  QK_REQUIRE(polls >= 1 && polls <= 1000000, "polls must be 1 to 1000000");
  fp8_expire_kernel<<<1, 32, 0, as_stream(stream)>>>(polls);
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return cuda_error(e, "fp8_expire_kernel");
  count_launch();
  return QK_OK;
}

int qk_fp8_check(qk_stream_t stream) {
  int status = 0;
  cudaStream_t st = as_stream(stream);
  void* word = nullptr;
  cudaError_t e = cudaGetSymbolAddress(&word, g_fp8_status);
  if (e == cudaSuccess) e = cudaMemcpyAsync(&status, word, sizeof(int), cudaMemcpyDeviceToHost, st);
  if (e == cudaSuccess) e = cudaStreamSynchronize(st);
  if (e == cudaSuccess && status) {
    e = cudaMemsetAsync(word, 0, sizeof(int), st);
    if (e == cudaSuccess) e = cudaStreamSynchronize(st);
  }
  if (e != cudaSuccess) return cuda_error(e, "qk_fp8_check");
  if (status) return set_error(QK_ERR_TIMEOUT, "a bounded device wait in an FP8 product gave up");
  return QK_OK;
}

}  // extern "C"
