// Attention of drafted tokens over a paged Q8 cache.
//
//   out[b, i, h] = sigmoid(gate) * sum_t p_t v_t,  p = softmax over the tokens t that node i of
//   request b sees of (q . k_t) * scale: the request's prefix t < length_b, and of the drafts
//   t = length_b + j (j < count_b) those whose bit j is set in the node's ancestor word. Keys and
//   values are code * scale of the Q8 cache, token t in slot table[b, t / P] * P + t % P. A node
//   that sees nothing and the rows i >= count_b are zero.
//
// One warp per (request, node, query head): a lane holds HD / 32 channels, dots are folded by a
// butterfly, one pass with the running maximum and sum of the softmax in FP32.
#include "common.cuh"

namespace qk {
namespace {

struct TreeArgs {
  const uint16_t* q;
  int64_t q_stride;
  const int8_t *k_codes, *v_codes;
  const uint16_t *k_scale, *v_scale;
  const int32_t *table, *lengths, *counts;
  const uint64_t* ancestors;
  const uint16_t* gate;
  float scale;
  int B, N, hq, kv, pages, pages_per_row, width, shift;
  int64_t T;
  uint16_t* out;
  int* status;
};

template <int HD>
__global__ void __launch_bounds__(256) tree_attention_kernel(TreeArgs a) {
  constexpr int C = HD / 32;  // channels per lane
  const int64_t item = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (item >= static_cast<int64_t>(a.B) * a.N * a.hq) return;
  const int h = static_cast<int>(item % a.hq);
  const int64_t bn = item / a.hq;
  const int b = static_cast<int>(bn / a.N), node = static_cast<int>(bn % a.N);
  const int kh = h / (a.hq / a.kv), D = a.kv * HD, G = D / 32;
  const int64_t room = static_cast<int64_t>(a.width) << a.shift;
  const int64_t length = min(static_cast<int64_t>(max(a.lengths[b], 0)), room);
  const int count = static_cast<int>(min(static_cast<int64_t>(a.counts ? min(max(a.counts[b], 0), a.N) : a.N), room - length));
  uint16_t* out = a.out + item * HD + lane * C;
  float q[C], acc[C];
#pragma unroll
  for (int c = 0; c < C; ++c) {
    q[c] = bf16_to_f32(a.q[bn * a.q_stride + h * HD + lane * C + c]) * a.scale;
    acc[c] = 0.f;
  }
  float m = -INFINITY, l = 0.f;
  const uint64_t path = node < count ? a.ancestors[bn] : 0;
  const int64_t end = node < count ? length + count : 0;
  for (int64_t t = 0; t < end; ++t) {
    if (t >= length && !(path >> (t - length) & 1)) continue;
    int page = a.table[static_cast<int64_t>(b) * a.width + (t >> a.shift)];
    if (page < 0 || page >= a.pages) {
      if (lane == 0) *a.status = QK_ERR_INVALID_ARGUMENT;
      continue;
    }
    const int row = page / a.pages_per_row;
    const int64_t in_row = (static_cast<int64_t>(page - row * a.pages_per_row) << a.shift) + (t & ((1 << a.shift) - 1));
    const int64_t code = (row * a.T + in_row) * D + kh * HD + lane * C;
    const int64_t plane = (static_cast<int64_t>(row) * G + kh * (HD / 32) + lane * C / 32) * a.T + in_row;
    const float ks = bf16_to_f32(a.k_scale[plane]), vs = bf16_to_f32(a.v_scale[plane]);
    float s = 0.f;
#pragma unroll
    for (int c = 0; c < C; ++c) s = fmaf(q[c], static_cast<float>(a.k_codes[code + c]) * ks, s);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    const float top = fmaxf(m, s);
    const float keep = top == -INFINITY ? 1.f : expf(m - top), p = top == -INFINITY ? 0.f : expf(s - top);
    m = top;
    l = l * keep + p;
#pragma unroll
    for (int c = 0; c < C; ++c) acc[c] = fmaf(acc[c], keep, p * (static_cast<float>(a.v_codes[code + c]) * vs));
  }
#pragma unroll
  for (int c = 0; c < C; ++c) {
    float o = l > 0.f || l != l ? acc[c] / l : 0.f;
    if (a.gate) o *= sigmoid_ref(bf16_to_f32(a.gate[item * HD + lane * C + c]));
    out[c] = node < count ? bf16_bits_rne(o) : 0;
  }
}

}  // namespace
}  // namespace qk

using namespace qk;

extern "C" {

size_t qk_tree_attention_workspace_bytes(int B, int N, int hq, int kv_heads, int head_dim) { return 256; }

int qk_tree_attention(const uint16_t* q, int64_t q_stride, const int8_t* k_codes, const int8_t* v_codes,
                      const uint16_t* k_scale, const uint16_t* v_scale, const int32_t* table, const int32_t* lengths,
                      const int32_t* counts, const uint64_t* ancestors, const uint16_t* gate, float scale, int B, int N,
                      int hq, int kv_heads, int head_dim, int rows, int64_t T, int width, int page_size, uint16_t* out,
                      void* workspace, size_t workspace_bytes, qk_stream_t stream) {
  QK_REQUIRE(head_dim == 64 || head_dim == 128 || head_dim == 256, "head_dim must be 64, 128 or 256");
  QK_REQUIRE(B >= 0 && N >= 1 && N <= 64 && kv_heads > 0 && hq > 0 && hq % kv_heads == 0,
             "invalid batch, nodes (1 to 64) or head counts");
  QK_REQUIRE(page_size >= 16 && page_size <= 1024 && (page_size & (page_size - 1)) == 0,
             "page_size must be a power of two in [16, 1024]");
  QK_REQUIRE(rows > 0 && T > 0 && T % page_size == 0 && rows * T <= 0x7fffffff && width >= 1,
             "the cache's time axis must be whole pages, its slots must fit 31 bits");
  if (B == 0) return QK_OK;
  QK_REQUIRE(q && k_codes && v_codes && k_scale && v_scale && table && lengths && ancestors && out, "null pointer");
  QK_REQUIRE(((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k_codes) | reinterpret_cast<uintptr_t>(v_codes) |
               reinterpret_cast<uintptr_t>(k_scale) | reinterpret_cast<uintptr_t>(v_scale) | reinterpret_cast<uintptr_t>(gate) |
               reinterpret_cast<uintptr_t>(out)) & 15) == 0,
             "q, gate, out and the cache must be 16-byte aligned");
  QK_REQUIRE(q_stride >= static_cast<int64_t>(hq) * head_dim && q_stride % 8 == 0,
             "tokens of q must be a multiple of 8 values apart and not overlap");
  const size_t need = qk_tree_attention_workspace_bytes(B, N, hq, kv_heads, head_dim);
  if (!workspace || workspace_bytes < need)
    return set_error(QK_ERR_WORKSPACE, "tree attention workspace needs %zu bytes, got %zu", need, workspace_bytes);
  TreeArgs a{q, q_stride, k_codes, v_codes, k_scale, v_scale, table, lengths, counts, ancestors, gate, scale, B, N, hq,
             kv_heads, static_cast<int>(rows * T / page_size), static_cast<int>(T / page_size), width, 0, T, out,
             static_cast<int*>(workspace)};
  while ((1 << a.shift) < page_size) ++a.shift;
  const int64_t warps = static_cast<int64_t>(B) * N * hq;
  const auto kernel = head_dim == 256 ? tree_attention_kernel<256> : head_dim == 128 ? tree_attention_kernel<128> : tree_attention_kernel<64>;
  kernel<<<static_cast<unsigned>((warps + 7) / 8), 256, 0, as_stream(stream)>>>(a);
  QK_LAUNCHED("tree_attention_kernel");
  return QK_OK;
}

int qk_tree_attention_check(const void* workspace, qk_stream_t stream) {
  QK_REQUIRE(workspace, "null pointer");
  int status = 0;
  cudaStream_t st = as_stream(stream);
  cudaError_t e = cudaMemcpyAsync(&status, workspace, sizeof(int), cudaMemcpyDeviceToHost, st);
  if (e == cudaSuccess) e = cudaStreamSynchronize(st);
  if (e == cudaSuccess && status) {
    e = cudaMemsetAsync(const_cast<void*>(workspace), 0, sizeof(int), st);
    if (e == cudaSuccess) e = cudaStreamSynchronize(st);
  }
  if (e != cudaSuccess) return cuda_error(e, "qk_tree_attention_check");
  if (status == QK_ERR_TIMEOUT) return set_error(status, "a bounded device wait in the tree attention gave up");
  if (status) return set_error(status, "a block table entry lies outside the cache");
  return QK_OK;
}

}  // extern "C"
