// Logits before the choice: penalties for repeated tokens, sparse biases, temperature and a
// grammar's bit mask, in one pass over the vocabulary.
//
//   x = logit;  in the context (history or drafted path):  x = x > 0 ? x * (1 / r) : x * r
//   x -= f * count + p * [count > 0];  x += bias;  x /= temperature;  mask bit 0: x = -inf
//
// Bound by HBM: a logit in, an FP32 value out, one mask bit per entry. A block owns a tile of
// the vocabulary of one request and counts the request's history into one 32-bit word per
// entry in shared memory (the history is re-read by every tile, from L2); the words then serve
// all rows of the request, one per node of a draft tree. Word: bits 0-19 the count of generated
// tokens, then flags: in the prompt, drafted, biased. Entries without a word, nearly all, are one
// multiply; the others look up what they need. Counts are integers and the last of several
// biases of one token wins by its index, so nothing depends on the order of atomics.
#include "common.cuh"

namespace qk {
namespace {

constexpr int kLogitThreads = 256;
constexpr int kVec = 8;  // entries per access
constexpr int kMaxBias = 1024, kMaxNodes = 64, kMaxTile = 4096;
constexpr int kMaxHistory = (1 << 20) - 1;
constexpr uint32_t kCountMask = (1u << 20) - 1, kPrompt = 1u << 20, kDraft = 1u << 21, kBias = 1u << 22;

struct LogitArgs {
  qk_logits_desc d;
  const void* logits;
  float* out;
  int B, N, V, tile, rows_per_block;
  bool vector;  // logits and out start on a whole access
};

// Penalties of an entry of word w whose context also has `drafted` occurrences on the row's path. In two
// steps, the first once per entry, the second per row of it: the amount to take off, FP32, where the
// factor applies (-0 for none), +0 where nothing does.
struct Penalties {
  float rep, inv_rep, freq, pres;
  __device__ uint32_t amount(uint32_t w, int drafted) const {
    const int count = static_cast<int>(w & kCountMask) + drafted;
    const float off = count > 0 ? fmaf(freq, static_cast<float>(count), pres) : 0.f;
    return count > 0 || (w & kPrompt) ? __float_as_uint(off == 0.f ? -0.f : off) : 0;
  }
  __device__ float apply(float x, uint32_t amount) const {
    const float factor = x > 0.f ? inv_rep : rep;
    return fmaf(x, amount != 0 ? factor : 1.f, -__uint_as_float(amount));
  }
};

// A block's entries: the tile's and the kVec before it, for the rows whose accesses begin there. Entry j
// lies in column j / 8 of row j % 8: eight neighbouring entries per lane, from any first entry, are eight
// reads without a bank conflict, and so are 32 neighbours across a warp.
constexpr int kEntries = kMaxTile + kVec, kFlagWords = (kEntries + 31) / 32 + 1;
constexpr int kWordStride = kMaxTile / kVec + 4, kWords = kVec * kWordStride;
__device__ __forceinline__ int at_entry(int j) { return (j % kVec) * kWordStride + j / kVec; }

struct Tile {
  alignas(16) uint32_t words[kWords];  // of entry j at at_entry(j); then the amounts
  uint32_t flags[kFlagWords];          // a bit per drafted or biased entry
  uint64_t draft_path[kMaxNodes];      // per drafted token of the tile: the nodes that carry it
  int draft_id[kMaxNodes], draft[kMaxNodes], draft_n;
  int bias_id[kMaxBias];
  uint16_t bias_at[kMaxBias];
  int bias_n;
};

// The rare entries: drafted or biased.
__device__ __noinline__ float adjust(float x, uint32_t w, int i, int64_t row, const Tile& s, const qk_logits_desc& d,
                                     const float* bias, const Penalties& penalties) {
  int drafted = 0;
  if (w & kDraft) {
    const uint64_t path = d.ancestors[row];
    for (int j = 0; j < s.draft_n; ++j)
      if (s.draft_id[j] == i) drafted = __popcll(s.draft_path[j] & path);
  }
  x = penalties.apply(x, penalties.amount(w, drafted));
  if (w & kBias) {
    int best = -1;
    for (int j = 0; j < s.bias_n; ++j)
      if (s.bias_id[j] == i && s.bias_at[j] > best) best = s.bias_at[j];
    x += bias[best];
  }
  return x;
}

__device__ __forceinline__ void load8(const float* p, uint32_t (&x)[8]) {
  asm volatile("ld.global.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=r"(x[0]), "=r"(x[1]), "=r"(x[2]), "=r"(x[3]), "=r"(x[4]), "=r"(x[5]), "=r"(x[6]), "=r"(x[7])
               : "l"(p)
               : "memory");
}
__device__ __forceinline__ void store8(float* p, const float (&x)[8]) {
  asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "f"(x[0]), "f"(x[1]), "f"(x[2]), "f"(x[3]),
               "f"(x[4]), "f"(x[5]), "f"(x[6]), "f"(x[7])
               : "memory");
}

// One entry: the ends of rows, and rows that do not start on a whole access.
template <bool BF16>
__device__ __forceinline__ void one_entry(const LogitArgs& a, const Tile& s, const Penalties& penalties, const float* bias,
                                          float inv, int64_t row, int v, int j) {
  const int64_t at = row * a.V + v;
  float x = BF16 ? __uint_as_float(static_cast<uint32_t>(static_cast<const uint16_t*>(a.logits)[at]) << 16)
                 : static_cast<const float*>(a.logits)[at];
  const uint32_t amount = s.words[at_entry(j)];
  x = s.flags[j / 32] >> (j % 32) & 1 ? adjust(x, amount, j, row, s, a.d, bias, penalties) : penalties.apply(x, amount);
  const uint32_t* mask = reinterpret_cast<const uint32_t*>(a.d.mask);
  const bool allowed = !mask || (mask[row * ((a.V + 31) / 32) + v / 32] >> (v % 32) & 1);
  a.out[at] = allowed ? x * inv : -INFINITY;
}

// Eight entries per thread and access, on multiples of eight of the flat index row * V + v (32 bytes
// of the output, 16 or 32 of the logits) whatever the vocabulary is: a row's part of a tile begins up
// to seven entries before it, so that only the two ends of a row are not whole. kBatch accesses are in
// flight per thread.
template <bool BF16>
__global__ void __launch_bounds__(kLogitThreads, 4) process_logits_kernel(LogitArgs a) {
  __shared__ Tile s;
  constexpr int kBatch = 2;
  // the tiles of the first tokens, usually the most frequent and so the slowest, start first
  const int b = blockIdx.x, tid = threadIdx.x;
  const int v0 = blockIdx.z * a.tile - kVec;  // of entry 0; below zero in the first tile
  const uint32_t n = min(a.tile + kVec, a.V - v0);
  const qk_logits_desc& d = a.d;
  for (int i = tid * 4; i < kWords; i += kLogitThreads * 4) *reinterpret_cast<uint4*>(s.words + i) = make_uint4(0, 0, 0, 0);
  if (tid == 0) s.bias_n = s.draft_n = 0;
  __syncthreads();
  pdl_wait();
  pdl_trigger();
  const int room = d.history ? d.history_capacity : 0;
  const int length = room ? min(max(d.history_lengths[b], 0), room) : 0;
  const int prompt = room && d.prompt_lengths ? d.prompt_lengths[b] : 0;
  const int32_t* history = d.history + static_cast<int64_t>(b) * room;
  constexpr int kAhead = 16;  // tokens in flight per thread
  for (int i0 = tid; i0 < length; i0 += kAhead * kLogitThreads) {
    uint32_t v[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int i = i0 + k * kLogitThreads;
      v[k] = ~0u;
      if (i0 - tid + k * kLogitThreads >= length) break;
      v[k] = i < length ? static_cast<uint32_t>(__ldg(history + i)) - static_cast<uint32_t>(v0) : ~0u;
    }
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      if (i0 - tid + k * kLogitThreads >= length) break;
      if (v[k] >= n) continue;
      if (i0 + k * kLogitThreads >= prompt) atomicAdd(&s.words[at_entry(v[k])], 1u);
      else atomicOr(&s.words[at_entry(v[k])], kPrompt);
    }
  }
  if (d.drafts && tid < a.N) s.draft[tid] = d.drafts[static_cast<int64_t>(b) * a.N + tid];
  if (d.bias_ids) {
    for (int k = tid; k < d.bias_count; k += kLogitThreads) {
      const int id = d.bias_ids[static_cast<int64_t>(b) * d.bias_count + k];
      const uint32_t v = static_cast<uint32_t>(id) - static_cast<uint32_t>(v0);
      if (v < n) {
        const int at = atomicAdd(&s.bias_n, 1);
        s.bias_id[at] = static_cast<int>(v);
        s.bias_at[at] = static_cast<uint16_t>(k);
        atomicOr(&s.words[at_entry(v)], kBias);
      }
    }
  }
  Penalties penalties;
  penalties.rep = d.repetition ? d.repetition[b] : 1.f;
  penalties.inv_rep = __frcp_rn(penalties.rep);
  penalties.freq = d.frequency ? d.frequency[b] : 0.f;
  penalties.pres = d.presence ? d.presence[b] : 0.f;
  const float inv = d.temperature ? __frcp_rn(d.temperature[b]) : 1.f;
  const float* bias = d.bias + static_cast<int64_t>(b) * d.bias_count;
  __syncthreads();
  if (d.drafts && tid < a.N) {  // each token that is drafted once, with the nodes that carry it
    const int id = s.draft[tid];
    const uint32_t v = static_cast<uint32_t>(id) - static_cast<uint32_t>(v0);
    if (v < n) {
      uint64_t path = 0;
      for (int j = 0; j < a.N; ++j) path |= static_cast<uint64_t>(s.draft[j] == id) << j;
      if (__ffsll(path) - 1 == tid) {
        const int at = atomicAdd(&s.draft_n, 1);
        s.draft_id[at] = static_cast<int>(v);
        s.draft_path[at] = path;
        atomicOr(&s.words[at_entry(v)], kDraft);
      }
    }
  }
  __syncthreads();
  // words to amounts; drafted and biased entries keep their word and get a flag
  for (int j = tid; j < kFlagWords * 32; j += kLogitThreads) {
    const uint32_t w = j < kEntries ? s.words[at_entry(j)] : 0;
    const bool rare = w & (kDraft | kBias);
    if (w != 0 && !rare) s.words[at_entry(j)] = penalties.amount(w, 0);
    const uint32_t all = __ballot_sync(0xffffffffu, rare);
    if (tid % 32 == 0) s.flags[j / 32] = all;
  }
  __syncthreads();

  const int mask_words = (a.V + 31) / 32;
  const int r0 = blockIdx.y * a.rows_per_block, r1 = min(r0 + a.rows_per_block, a.N);
  if (!a.vector) {
    for (int r = r0; r < r1; ++r)
#pragma unroll 4
      for (int j = kVec + tid; j < static_cast<int>(n); j += kLogitThreads)
        one_entry<BF16>(a, s, penalties, bias, inv, static_cast<int64_t>(b) * a.N + r, v0 + j, j);
    return;
  }
  for (int r = r0; r < r1; ++r) {
    const int64_t row = static_cast<int64_t>(b) * a.N + r, base = row * a.V;
    const int lead = static_cast<int>(base + v0 & (kVec - 1));
    const uint32_t* mask = d.mask ? reinterpret_cast<const uint32_t*>(d.mask) + row * mask_words : nullptr;
    for (int c0 = tid; c0 < a.tile / kVec; c0 += kBatch * kLogitThreads) {
      uint32_t x[kBatch][kVec], allowed[kBatch];
#pragma unroll
      for (int k = 0; k < kBatch; ++k) {
        const int c = c0 + k * kLogitThreads, v = v0 + (c + 1) * kVec - lead;
        allowed[k] = ~0u;
        if (c >= a.tile / kVec || v < 0 || v + kVec > a.V) continue;
        if (BF16) {
          const uint4 u = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.logits) + base + v);
#pragma unroll
          for (int t = 0; t < 4; ++t) {
            x[k][2 * t] = word(u, t) << 16;
            x[k][2 * t + 1] = word(u, t) & 0xffff0000u;
          }
        } else {
          load8(static_cast<const float*>(a.logits) + base + v, x[k]);
        }
        if (mask) allowed[k] = __funnelshift_r(mask[v >> 5], mask[min((v >> 5) + 1, mask_words - 1)], v & 31);
      }
#pragma unroll
      for (int k = 0; k < kBatch; ++k) {
        const int c = c0 + k * kLogitThreads, v = v0 + (c + 1) * kVec - lead;
        if (c >= a.tile / kVec || v < 0 || v + kVec > a.V) continue;
        const int j0 = v - v0;
        const uint32_t rare = __funnelshift_r(s.flags[j0 >> 5], s.flags[(j0 >> 5) + 1], j0 & 31);
        float f[kVec];
#pragma unroll
        for (int t = 0; t < kVec; ++t) {
          const uint32_t amount = s.words[(t - lead & (kVec - 1)) * kWordStride + c + 1 - (t < lead)];
          f[t] = penalties.apply(__uint_as_float(x[k][t]), amount);
        }
        if (rare & ((1u << kVec) - 1)) {
#pragma unroll
          for (int t = 0; t < kVec; ++t)
            if (rare >> t & 1)
              f[t] = adjust(__uint_as_float(x[k][t]), s.words[at_entry(j0 + t)], j0 + t, row, s, d, bias, penalties);
        }
#pragma unroll
        for (int t = 0; t < kVec; ++t) f[t] = allowed[k] >> t & 1 ? f[t] * inv : -INFINITY;
        store8(a.out + base + v, f);
      }
    }
  }
  // The ends: up to seven entries before a row's first whole access and behind its last, a thread each.
  if (blockIdx.z != 0 && v0 + a.tile + 2 * kVec < a.V) return;
  for (int e = tid; e < (r1 - r0) * 2 * kVec; e += kLogitThreads) {
    const int64_t row = static_cast<int64_t>(b) * a.N + r0 + e / (2 * kVec), base = row * a.V;
    const int t = e % kVec, head = static_cast<int>(-base & (kVec - 1));
    const int v = e & kVec ? t : a.V - 1 - t;
    const bool end = e & kVec ? v < head : (base + a.V & (kVec - 1)) > t && v >= head;
    const int j = v - v0, lead = static_cast<int>(base + v0 & (kVec - 1));
    // the tile of the access that would hold it
    if (end && v < a.V && j >= kVec - lead && j < a.tile + kVec - lead)
      one_entry<BF16>(a, s, penalties, bias, inv, row, v, j);
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
  QK_REQUIRE(B >= 0 && N >= 0 && N <= 65535 && V > 0 && V <= 65535 * 1024, "invalid batch, rows or vocabulary");
  QK_REQUIRE(d.history_capacity >= 0 && d.history_capacity <= kMaxHistory, "a history holds at most %d tokens", kMaxHistory);
  QK_REQUIRE(!d.history || d.history_lengths, "a history needs its lengths");
  QK_REQUIRE(d.bias_count >= 0 && d.bias_count <= kMaxBias, "a request has at most %d biases", kMaxBias);
  QK_REQUIRE(!d.bias_ids == !d.bias, "biases need their ids");
  QK_REQUIRE(!d.drafts == !d.ancestors, "drafts and ancestors go together");
  QK_REQUIRE(!d.drafts || N <= kMaxNodes, "a draft tree has at most %d nodes", kMaxNodes);
  if (B == 0 || N == 0) return QK_OK;
  QK_REQUIRE(logits && out, "null pointer");
  LogitArgs a{d, logits, out, B, N, V, 0, 0, false};
  if (!a.d.bias_ids) a.d.bias_count = 0;
  // Tiles small enough that the blocks fill the SMs twice over, large enough that the history's
  // re-reads (one per tile) stay small: at most 4096 entries, at least 1024.
  a.tile = kMaxTile;
  while (a.tile > 1024 && static_cast<int64_t>(B) * N * ((V + a.tile - 1) / a.tile) < 2 * sm_count()) a.tile /= 2;
  const bool bf16 = in_dtype == QK_OUT_BF16;
  a.vector = (reinterpret_cast<uintptr_t>(logits) & (bf16 ? 15 : 31)) == 0 && (reinterpret_cast<uintptr_t>(out) & 31) == 0;
  const int lead = a.vector && V % kVec ? kVec - 1 : 0;  // by which a row's accesses may begin before a tile
  const int tiles = (V + lead + a.tile - 1) / a.tile;
  // A block takes several rows of its request (each repeats the counting), but leaves 8 blocks per SM
  // where there are as many: tiles of frequent tokens take longer than others.
  int parts = 1;
  while (parts < N && static_cast<int64_t>(B) * tiles * parts < 8 * sm_count()) parts *= 2;
  a.rows_per_block = (N + parts - 1) / parts;
  parts = (N + a.rows_per_block - 1) / a.rows_per_block;
  const auto kernel = bf16 ? process_logits_kernel<true> : process_logits_kernel<false>;
  const cudaError_t e = launch_dependent(kernel, dim3(B, parts, tiles), dim3(kLogitThreads), 0, as_stream(stream), a);
  if (e != cudaSuccess) return cuda_error(e, "process_logits_kernel");
  count_launch();
  return QK_OK;
}

}  // extern "C"
