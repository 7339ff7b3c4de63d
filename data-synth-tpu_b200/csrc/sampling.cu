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
#include <algorithm>

#include "common.cuh"

namespace qk {
namespace {

constexpr int kLogitThreads = 256, kLogitWarps = kLogitThreads / 32;
constexpr int kLogitBlocks = 3;  // per SM: shared memory
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

// A block's entries: the tile's and the kVec before it, for the rows whose accesses begin there.
constexpr int kEntries = kMaxTile + kVec, kFlagWords = (kEntries + 31) / 32;
constexpr int kSegment = kMaxTile / kLogitWarps;  // entries per warp and row, at most
constexpr int kList = kSegment + kVec, kMaskWords = kSegment / 32 + 2;
// Rows on their way to a warp, and for BF16 the row at hand in FP32.
constexpr int kStages16 = 2, kStages32 = 2;
constexpr int kRowBytes = std::max(kStages16 * 2 + 4, kStages32 * 4) * kSegment;

struct Tile {
  alignas(16) uint8_t rows[kLogitWarps][kRowBytes];
  uint32_t masks[kLogitWarps][kStages16][kMaskWords];
  uint32_t words[kFlagWords * 32];      // per entry; then the amounts
  uint32_t flags[kFlagWords];           // a bit per drafted or biased entry
  uint16_t list[kLogitWarps][kList];    // the entries that have a word; the top bit repeats the flag
  // Drafted or biased entries have a record: of a drafted token the number of its first node, of others
  // kMaxNodes + the place of the bias that holds.
  uint32_t record_word[kMaxNodes + kMaxBias];
  float record_bias[kMaxNodes + kMaxBias];
  uint64_t path[kMaxNodes], ancestors[kMaxNodes];  // the nodes that carry a record's token; per row
  int draft[kMaxNodes], draft_id[kMaxNodes];
  uint16_t bias_id[kMaxBias], bias_at[kMaxBias];
  int bias_n;
};
static_assert(kEntries < 0x8000, "an entry fits 15 bits");

// The rare entries: drafted or biased, `number` that of the record plus one; r the row of the request.
__device__ __forceinline__ float adjust(float x, uint32_t number, int r, const Tile& s, const Penalties& penalties) {
  const uint32_t i = number - 1, w = s.record_word[i];
  x = penalties.apply(x, penalties.amount(w, i < kMaxNodes ? __popcll(s.path[i] & s.ancestors[r]) : 0));
  return w & kBias ? x + s.record_bias[i] : x;
}

// The bias of an entry: the last of the request's list that names it, by its place in the tile's list, or -1.
__device__ __forceinline__ int last_bias(const Tile& s, int entry) {
  int best = -1;
  for (int k = 0; k < s.bias_n; ++k)
    if (s.bias_id[k] == entry && (best < 0 || s.bias_at[k] > s.bias_at[best])) best = k;
  return best;
}

__device__ __forceinline__ void cp_async4(void* dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_addr(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void store8(float* p, const float (&x)[8]) {
  asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "f"(x[0]), "f"(x[1]), "f"(x[2]), "f"(x[3]),
               "f"(x[4]), "f"(x[5]), "f"(x[6]), "f"(x[7])
               : "memory");
}

// One entry: the ends of rows, and rows that do not start on a whole access.
template <bool BF16>
__device__ __forceinline__ void one_entry(const LogitArgs& a, const Tile& s, const Penalties& penalties, float inv, int b,
                                          int r, int v, int j) {
  const int64_t row = static_cast<int64_t>(b) * a.N + r;
  const int64_t at = row * a.V + v;
  float x = BF16 ? __uint_as_float(static_cast<uint32_t>(static_cast<const uint16_t*>(a.logits)[at]) << 16)
                 : static_cast<const float*>(a.logits)[at];
  const uint32_t amount = s.words[j];
  x = s.flags[j / 32] >> (j % 32) & 1 ? adjust(x, amount, r, s, penalties) : penalties.apply(x, amount);
  const uint32_t* mask = reinterpret_cast<const uint32_t*>(a.d.mask);
  const bool allowed = !mask || (mask[row * ((a.V + 31) / 32) + v / 32] >> (v % 32) & 1);
  a.out[at] = allowed ? x * inv : -INFINITY;
}

// A warp's part of a row: up to kSegment entries in accesses of eight, from a multiple of eight of the
// flat index row * V + v (32 bytes of the output, 16 or 32 of the logits) whatever the vocabulary is. It
// begins up to seven entries before the warp's part of the tile, so only the ends of a row are not whole.
struct Part {
  int64_t base;  // of the row
  int v, lo, hi;  // its first entry; the accesses of it that are whole
  int word;       // of the mask, the first that is copied
  __device__ Part(const LogitArgs& a, int64_t row, int v0, int segment, int warp) : base(row * a.V) {
    v = v0 + kVec - static_cast<int>(base + v0 & (kVec - 1)) + warp * segment;
    lo = v < 0;  // an access is no longer than what lies before entry 0
    hi = min(segment, max(a.V - v, 0)) / kVec;
    word = max(v, 0) >> 5;
  }
};

// Where 16 bytes q of a row in FP32 lie, so that eight lanes that read every other 16 bytes meet all banks.
__device__ __forceinline__ int swizzled(int q) { return q ^ (q >> 3 & 1); }

template <bool BF16>
__global__ void __launch_bounds__(kLogitThreads, kLogitBlocks) process_logits_kernel(LogitArgs a) {
  extern __shared__ __align__(16) uint8_t smem[];
  Tile& s = *reinterpret_cast<Tile*>(smem);
  constexpr int kSize = BF16 ? 2 : 4, kStages = BF16 ? kStages16 : kStages32, kBatch = kSegment / (32 * kVec);
  // the tiles of the first tokens, usually the most frequent and so the slowest, start first
  const int b = blockIdx.x, tid = threadIdx.x, lane = tid % 32, warp = tid / 32;
  const int v0 = blockIdx.z * a.tile - kVec;  // of entry 0; below zero in the first tile
  const uint32_t n = min(a.tile + kVec, a.V - v0);
  const int segment = a.tile / kLogitWarps, mask_words = (a.V + 31) / 32;
  const int r0 = blockIdx.y * a.rows_per_block, r1 = min(r0 + a.rows_per_block, a.N);
  const qk_logits_desc& d = a.d;
  const uint32_t* mask = reinterpret_cast<const uint32_t*>(d.mask);
  // row r on its way to the warp, 512 bytes by all lanes at a time, and its mask, a word per lane
  const auto fetch = [&](int r) {
    if (a.vector && r < r1) {
      const int64_t row = static_cast<int64_t>(b) * a.N + r;
      const Part part(a, row, v0, segment, warp);
      const int stage = (r - r0) % kStages;
      uint8_t* to = s.rows[warp] + stage * kSegment * kSize;
      const uint8_t* from = static_cast<const uint8_t*>(a.logits) + (part.base + part.v) * kSize;
#pragma unroll
      for (int k = 0; k < kSegment * kSize / 512; ++k) {
        const int q = lane + 32 * k, c = q * 8 / kSize / 4;
        if (c >= part.lo && c < part.hi) cp_async16(to + (BF16 ? q : swizzled(q)) * 16, from + q * 16);
      }
      if (mask && lane < kMaskWords && part.lo < part.hi)
        cp_async4(&s.masks[warp][stage][lane], mask + row * mask_words + min(part.word + lane, mask_words - 1));
    }
    cp_async_commit();
  };
  for (int i = tid; i < kFlagWords * 32; i += kLogitThreads) s.words[i] = 0;
  if (tid == 0) s.bias_n = 0;
  pdl_wait();
  pdl_trigger();
#pragma unroll
  for (int k = 0; k < kStages; ++k) fetch(r0 + k);
  const int room = d.history ? d.history_capacity : 0;
  const int length = room ? min(max(d.history_lengths[b], 0), room) : 0;
  const int prompt = room && d.prompt_lengths ? d.prompt_lengths[b] : 0;
  const int32_t* history = d.history + static_cast<int64_t>(b) * room;
  if (d.drafts && tid < a.N) {
    s.draft[tid] = d.drafts[static_cast<int64_t>(b) * a.N + tid];
    s.ancestors[tid] = d.ancestors[static_cast<int64_t>(b) * a.N + tid];
  }
  Penalties penalties;
  penalties.rep = d.repetition ? d.repetition[b] : 1.f;
  penalties.inv_rep = __frcp_rn(penalties.rep);
  penalties.freq = d.frequency ? d.frequency[b] : 0.f;
  penalties.pres = d.presence ? d.presence[b] : 0.f;
  const float inv = d.temperature ? __frcp_rn(d.temperature[b]) : 1.f;
  const float* bias = d.bias + static_cast<int64_t>(b) * d.bias_count;
  __syncthreads();
  constexpr int kAhead = 16;  // tokens in flight per thread; the first of them do not wait for the length
  for (int i0 = tid, bound = room; i0 < bound; i0 += kAhead * kLogitThreads, bound = length) {
    uint32_t v[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int i = i0 + k * kLogitThreads;
      v[k] = i < bound ? static_cast<uint32_t>(__ldg(history + i)) - static_cast<uint32_t>(v0) : ~0u;
    }
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int i = i0 + k * kLogitThreads;
      if (v[k] >= n || i >= length) continue;
      if (i >= prompt) atomicAdd(&s.words[v[k]], 1u);
      else atomicOr(&s.words[v[k]], kPrompt);
    }
  }
  if (d.bias_ids) {
    for (int k = tid; k < d.bias_count; k += kLogitThreads) {
      const int id = d.bias_ids[static_cast<int64_t>(b) * d.bias_count + k];
      const uint32_t v = static_cast<uint32_t>(id) - static_cast<uint32_t>(v0);
      if (v < n) {
        const int at = atomicAdd(&s.bias_n, 1);
        s.bias_id[at] = static_cast<uint16_t>(v);
        s.bias_at[at] = static_cast<uint16_t>(k);
        atomicOr(&s.words[v], kBias);
      }
    }
  }
  __syncthreads();
  const bool records = d.drafts || s.bias_n;  // the same for the whole block
  if (d.drafts && tid < a.N) {  // each token that is drafted once, with the nodes that carry it
    const int id = s.draft[tid];
    const uint32_t v = static_cast<uint32_t>(id) - static_cast<uint32_t>(v0);
    uint64_t path = 0;
    for (int j = 0; j < a.N; ++j) path |= static_cast<uint64_t>(s.draft[j] == id) << j;
    const bool first = v < n && __ffsll(path) - 1 == tid;
    s.draft_id[tid] = first ? static_cast<int>(v) : -1;
    s.path[tid] = path;
    if (first) {
      const int k = last_bias(s, static_cast<int>(v));
      s.record_bias[tid] = k < 0 ? 0.f : bias[s.bias_at[k]];
      atomicOr(&s.words[v], kDraft);
    }
  }
  if (records) __syncthreads();
  for (int k = tid; k < s.bias_n; k += kLogitThreads) {
    const int entry = s.bias_id[k];
    const bool holds = !(s.words[entry] & kDraft) && last_bias(s, entry) == k;
    s.record_word[kMaxNodes + k] = holds;
    s.record_bias[kMaxNodes + k] = holds ? bias[s.bias_at[k]] : 0.f;
  }
  // words to amounts; drafted and biased entries get a flag
  for (int j = tid; j < kFlagWords * 32; j += kLogitThreads) {
    const uint32_t w = s.words[j];
    const bool rare = w & (kDraft | kBias);
    if (w != 0 && !rare) s.words[j] = penalties.amount(w, 0);
    const uint32_t all = __ballot_sync(0xffffffffu, rare);
    if (lane == 0) s.flags[j / 32] = all;
  }
  __syncthreads();
  if (records) {  // and the records their words
    if (d.drafts && tid < a.N && s.draft_id[tid] >= 0) {
      uint32_t& w = s.words[s.draft_id[tid]];
      s.record_word[tid] = w;
      w = 1 + tid;
    }
    for (int k = tid; k < s.bias_n; k += kLogitThreads) {
      if (!s.record_word[kMaxNodes + k]) continue;
      uint32_t& w = s.words[s.bias_id[k]];
      s.record_word[kMaxNodes + k] = w;
      w = 1 + kMaxNodes + k;
    }
    __syncthreads();
  }
  if (!a.vector) {
    for (int r = r0; r < r1; ++r)
#pragma unroll 4
      for (int j = kVec + tid; j < static_cast<int>(n); j += kLogitThreads)
        one_entry<BF16>(a, s, penalties, inv, b, r, v0 + j, j);
    return;
  }
  // what the warp's rows have to treat: the entries of its parts, which begin at one of eight places
  int listed = 0;
  for (int j0 = warp * segment; j0 < (warp + 1) * segment + kVec; j0 += 32) {
    const int j = j0 + lane;
    const bool has = j < (warp + 1) * segment + kVec && s.words[j] != 0;
    const uint32_t all = __ballot_sync(0xffffffffu, has);
    if (has) s.list[warp][listed + __popc(all & ((1u << lane) - 1))] = j | (s.flags[j / 32] >> (j % 32) & 1) << 15;
    listed += __popc(all);
  }
  __syncwarp();

  for (int r = r0; r < r1; ++r) {
    const int64_t row = static_cast<int64_t>(b) * a.N + r;
    const Part part(a, row, v0, segment, warp);
    const int stage = (r - r0) % kStages;
    uint8_t* x = s.rows[warp] + (BF16 ? kStages * kSegment * kSize : stage * kSegment * kSize);  // in FP32
    const uint32_t* allowed = s.masks[warp][stage];
    const int bit0 = part.v - part.word * 32;
    cp_async_wait<kStages - 1>();
    if (BF16) {
#pragma unroll
      for (int k = 0; k < kBatch; ++k) {  // what this lane copied
        const int q = lane + 32 * k;
        const uint4 u = lds_v4(s.rows[warp] + stage * kSegment * kSize + q * 16);
        *reinterpret_cast<uint4*>(x + swizzled(2 * q) * 16) =
            make_uint4(u.x << 16, u.x & 0xffff0000u, u.y << 16, u.y & 0xffff0000u);
        *reinterpret_cast<uint4*>(x + swizzled(2 * q + 1) * 16) =
            make_uint4(u.z << 16, u.z & 0xffff0000u, u.w << 16, u.w & 0xffff0000u);
      }
    }
    __syncwarp();
    // first the few entries that have a word, 32 at a time
    for (int i = lane; i < listed; i += 32) {
      const uint32_t e = s.list[warp][i];
      const int j = e & 0x7fff, l = j + v0 - part.v;
      if (l < part.lo * kVec || l >= part.hi * kVec) continue;
      float* at = reinterpret_cast<float*>(x + swizzled(l >> 2) * 16) + (l & 3);
      const uint32_t amount = s.words[j];
      *at = e & 0x8000 ? adjust(*at, amount, r, s, penalties) : penalties.apply(*at, amount);
    }
    __syncwarp();
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      const int c = lane + 32 * k;
      if (c < part.lo || c >= part.hi) continue;
      const int bit = bit0 + c * kVec;
      const uint32_t bits = mask ? __funnelshift_r(allowed[bit >> 5], allowed[(bit >> 5) + 1], bit & 31) : ~0u;
      float f[kVec];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint4 u = lds_v4(x + swizzled(2 * c + h) * 16);
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          const float y = __uint_as_float(word(u, t)) * inv;
          f[4 * h + t] = bits >> (4 * h + t) & 1 ? y : -INFINITY;
        }
      }
      store8(a.out + part.base + part.v + c * kVec, f);
    }
    __syncwarp();
    fetch(r + kStages);
  }
  // The ends: up to seven entries before a row's first whole access and behind its last, a thread each.
  if (blockIdx.z != 0 && v0 + a.tile + 2 * kVec < a.V) return;
  for (int e = tid; e < (r1 - r0) * 2 * kVec; e += kLogitThreads) {
    const int r = r0 + e / (2 * kVec);
    const int64_t base = (static_cast<int64_t>(b) * a.N + r) * a.V;
    const int t = e % kVec, head = static_cast<int>(-base & (kVec - 1));
    const int v = e & kVec ? t : a.V - 1 - t;
    const bool end = e & kVec ? v < head : (base + a.V & (kVec - 1)) > t && v >= head;
    const int j = v - v0, lead = static_cast<int>(base + v0 & (kVec - 1));
    // the tile of the access that would hold it
    if (end && v < a.V && j >= kVec - lead && j < a.tile + kVec - lead)
      one_entry<BF16>(a, s, penalties, inv, b, r, v, j);
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
  if (int rc = allow_smem(reinterpret_cast<const void*>(kernel), sizeof(Tile))) return rc;
  const cudaError_t e =
      launch_dependent(kernel, dim3(B, parts, tiles), dim3(kLogitThreads), sizeof(Tile), as_stream(stream), a);
  if (e != cudaSuccess) return cuda_error(e, "process_logits_kernel");
  count_launch();
  return QK_OK;
}

}  // extern "C"
