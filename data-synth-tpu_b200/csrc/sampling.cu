// Logits before the choice: penalties for repeated tokens, sparse biases, temperature and a
// grammar's bit mask, in one pass over the vocabulary.
//
//   x = logit;  in the context (history or drafted path):  x = x > 0 ? x / r : x * r
//   x -= f * count + p * [count > 0];  x += bias;  x /= temperature;  mask bit 0: x = -inf
//
// Bound by HBM: a logit in, an FP32 value out, one mask bit per entry. A block owns a tile of
// the vocabulary of one request and counts the request's history into one 32-bit word per
// entry in shared memory (the history is re-read by every tile, from L2); the words then serve
// all rows of the request, one per node of a draft tree. Entries of the word: bits 0-19 the
// count of generated tokens, then flags: in the prompt, drafted, biased. Most words are zero
// and take the short path (one multiply); drafted and biased entries, at most a few hundred per
// request, look their nodes or their bias up in short lists. Counts are integers and the last of
// several biases of one token wins by its index, so nothing depends on the order of atomics.
#include "common.cuh"

namespace qk {
namespace {

constexpr int kLogitThreads = 256;
constexpr int kMaxBias = 1024, kMaxNodes = 64;
constexpr int kMaxHistory = (1 << 20) - 1;
constexpr uint32_t kCountMask = (1u << 20) - 1, kPrompt = 1u << 20, kDraft = 1u << 21, kBias = 1u << 22;

struct LogitArgs {
  qk_logits_desc d;
  const void* logits;
  float* out;
  int B, N, V, tile, rows_per_block;
};

struct TileLists {
  int bias_n;
  int bias_id[kMaxBias];
  int bias_at[kMaxBias];
  int draft[kMaxNodes];
};

// The rare entries: in the context, drafted or biased.
__device__ __noinline__ float adjust(float x, uint32_t w, int v, const TileLists& s, const float* bias, int nodes,
                                     uint64_t path, float rep, float freq, float pres) {
  int count = w & kCountMask;
  if (w & kDraft) {
    for (int j = 0; j < nodes; ++j) count += s.draft[j] == v && (path >> j & 1);
  }
  if (count > 0 || (w & kPrompt)) x = x > 0.f ? __fdiv_rn(x, rep) : x * rep;
  if (count > 0) x -= freq * static_cast<float>(count) + pres;
  if (w & kBias) {
    int best = -1;
    for (int j = 0; j < s.bias_n; ++j)
      if (s.bias_id[j] == v && s.bias_at[j] > best) best = s.bias_at[j];
    x += bias[best];
  }
  return x;
}

// VEC entries per thread and step: 4 when every row of logits and out is 16-byte (BF16: 8-byte)
// aligned, which takes a vocabulary that is a multiple of 4, else 1.
template <bool BF16, int VEC>
__global__ void __launch_bounds__(kLogitThreads) process_logits_kernel(LogitArgs a) {
  extern __shared__ uint32_t words[];
  __shared__ TileLists s;
  const int b = blockIdx.z, tid = threadIdx.x;
  const int v0 = blockIdx.x * a.tile, n = min(a.tile, a.V - v0);
  const qk_logits_desc& d = a.d;
  for (int i = tid; i < n; i += kLogitThreads) words[i] = 0;
  if (tid == 0) s.bias_n = 0;
  __syncthreads();
  pdl_wait();
  pdl_trigger();
  const int room = d.history ? d.history_capacity : 0;
  const int length = room ? min(max(d.history_lengths[b], 0), room) : 0;
  const int prompt = room && d.prompt_lengths ? d.prompt_lengths[b] : 0;
  const int32_t* history = d.history + static_cast<int64_t>(b) * room;
  for (int i = tid; i < length; i += kLogitThreads) {
    const uint32_t v = static_cast<uint32_t>(history[i] - v0);
    if (v < static_cast<uint32_t>(n)) {
      if (i < prompt) atomicOr(&words[v], kPrompt);
      else atomicAdd(&words[v], 1u);
    }
  }
  if (d.drafts && tid < a.N) {
    const int id = d.drafts[static_cast<int64_t>(b) * a.N + tid];
    s.draft[tid] = id;
    const uint32_t v = static_cast<uint32_t>(id - v0);
    if (v < static_cast<uint32_t>(n)) atomicOr(&words[v], kDraft);
  }
  if (d.bias_ids) {
    for (int k = tid; k < d.bias_count; k += kLogitThreads) {
      const int id = d.bias_ids[static_cast<int64_t>(b) * d.bias_count + k];
      const uint32_t v = static_cast<uint32_t>(id - v0);
      if (v < static_cast<uint32_t>(n)) {
        const int at = atomicAdd(&s.bias_n, 1);
        s.bias_id[at] = id;
        s.bias_at[at] = k;
        atomicOr(&words[v], kBias);
      }
    }
  }
  const float rep = d.repetition ? d.repetition[b] : 1.f, freq = d.frequency ? d.frequency[b] : 0.f;
  const float pres = d.presence ? d.presence[b] : 0.f, inv = d.temperature ? __frcp_rn(d.temperature[b]) : 1.f;
  const float* bias = d.bias + static_cast<int64_t>(b) * d.bias_count;
  __syncthreads();

  const int mask_words = (a.V + 31) / 32;
  const int r0 = blockIdx.y * a.rows_per_block, r1 = min(r0 + a.rows_per_block, a.N);
  for (int r = r0; r < r1; ++r) {
    const int64_t row = static_cast<int64_t>(b) * a.N + r;
    const uint64_t path = d.drafts ? d.ancestors[row] : 0;
    const int64_t base = row * a.V + v0;
    const uint32_t* mask = d.mask ? reinterpret_cast<const uint32_t*>(d.mask) + row * mask_words : nullptr;
#pragma unroll 4
    for (int i = tid * VEC; i < n; i += kLogitThreads * VEC) {
      float x[VEC];
      uint32_t w[VEC];
      if (VEC == 4) {
        if (BF16) {
          const uint2 u = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(a.logits) + base + i);
          x[0] = __uint_as_float(u.x << 16);
          x[VEC > 1] = __uint_as_float(u.x & 0xffff0000u);
          x[VEC > 1 ? 2 : 0] = __uint_as_float(u.y << 16);
          x[VEC > 1 ? 3 : 0] = __uint_as_float(u.y & 0xffff0000u);
        } else {
          const float4 u = *reinterpret_cast<const float4*>(static_cast<const float*>(a.logits) + base + i);
          x[0] = u.x;
          x[VEC > 1] = u.y;
          x[VEC > 1 ? 2 : 0] = u.z;
          x[VEC > 1 ? 3 : 0] = u.w;
        }
        const uint4 u = lds_v4(words + i);
        w[0] = u.x;
        w[VEC > 1] = u.y;
        w[VEC > 1 ? 2 : 0] = u.z;
        w[VEC > 1 ? 3 : 0] = u.w;
      } else {
        x[0] = BF16 ? bf16_to_f32(static_cast<const uint16_t*>(a.logits)[base + i])
                    : static_cast<const float*>(a.logits)[base + i];
        w[0] = words[i];
      }
      const uint32_t allowed = mask ? mask[(v0 + i) >> 5] >> ((v0 + i) & 31) : 0xfu;
#pragma unroll
      for (int t = 0; t < VEC; ++t) {
        if (w[t]) x[t] = adjust(x[t], w[t], v0 + i + t, s, bias, a.N, path, rep, freq, pres);
        x[t] = allowed >> t & 1 ? x[t] * inv : -INFINITY;
      }
      if (VEC == 4) *reinterpret_cast<float4*>(a.out + base + i) = make_float4(x[0], x[VEC > 1], x[VEC > 1 ? 2 : 0], x[VEC > 1 ? 3 : 0]);
      else a.out[base + i] = x[0];
    }
  }
}

}  // namespace
}  // namespace qk

using namespace qk;

extern "C" {

int qk_process_logits(const qk_logits_desc* desc, const void* logits, int in_dtype, int B, int N, int V, float* out,
                      qk_stream_t stream) {
  QK_REQUIRE(desc, "null pointer");
  const qk_logits_desc& d = *desc;
  QK_REQUIRE(in_dtype == QK_OUT_F32 || in_dtype == QK_OUT_BF16, "logits must be F32 or BF16");
  QK_REQUIRE(B >= 0 && B <= 65535 && N >= 0 && V > 0, "invalid batch, rows or vocabulary");
  QK_REQUIRE(d.history_capacity >= 0 && d.history_capacity <= kMaxHistory, "a history holds at most %d tokens", kMaxHistory);
  QK_REQUIRE(!d.history || d.history_lengths, "a history needs its lengths");
  QK_REQUIRE(d.bias_count >= 0 && d.bias_count <= kMaxBias, "a request has at most %d biases", kMaxBias);
  QK_REQUIRE(!d.bias_ids == !d.bias, "biases need their ids");
  QK_REQUIRE(!d.drafts == !d.ancestors, "drafts and ancestors go together");
  QK_REQUIRE(!d.drafts || N <= kMaxNodes, "a draft tree has at most %d nodes", kMaxNodes);
  if (B == 0 || N == 0) return QK_OK;
  QK_REQUIRE(logits && out, "null pointer");
  LogitArgs a{d, logits, out, B, N, V, 0, 0};
  if (!a.d.bias_ids) a.d.bias_count = 0;
  // Tiles small enough that the blocks fill the SMs twice over, large enough that the history's
  // re-reads (one per tile) stay small: at most 4096 words, at least 1024.
  a.tile = 4096;
  while (a.tile > 1024 && static_cast<int64_t>(B) * N * ((V + a.tile - 1) / a.tile) < 2 * sm_count()) a.tile /= 2;
  const int tiles = (V + a.tile - 1) / a.tile;
  // a block takes all rows of its request unless that leaves SMs idle
  int parts = 1;
  while (parts < N && static_cast<int64_t>(B) * tiles * parts < 2 * sm_count()) parts *= 2;
  a.rows_per_block = (N + parts - 1) / parts;
  parts = (N + a.rows_per_block - 1) / a.rows_per_block;
  const bool bf16 = in_dtype == QK_OUT_BF16;
  const bool vec = V % 4 == 0 && (reinterpret_cast<uintptr_t>(logits) & (bf16 ? 7 : 15)) == 0 &&
                   (reinterpret_cast<uintptr_t>(out) & 15) == 0;
  const auto kernel = bf16 ? (vec ? process_logits_kernel<true, 4> : process_logits_kernel<true, 1>)
                           : (vec ? process_logits_kernel<false, 4> : process_logits_kernel<false, 1>);
  const cudaError_t e = launch_dependent(kernel, dim3(tiles, parts, B), dim3(kLogitThreads), a.tile * 4, as_stream(stream), a);
  if (e != cudaSuccess) return cuda_error(e, "process_logits_kernel");
  count_launch();
  return QK_OK;
}

}  // extern "C"
