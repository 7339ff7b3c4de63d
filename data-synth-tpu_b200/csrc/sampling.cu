// Logits before the choice: penalties for repeated tokens, sparse biases, temperature and a
// grammar's bit mask, in one pass over the vocabulary.
//
//   x = logit;  in the context (history or drafted path):  x = x > 0 ? x * (1 / r) : x * r
//   x -= f * count + p * [count > 0];  x += bias;  x /= temperature;  mask bit 0: x = -inf
//
// A logit in, an FP32 value out and one mask bit per entry: 16 requests of 24 rows of 151937 FP32 logits
// have to move 475 MB, 72 us, and take 88 us (5.4 TB/s, 82% of measured HBM); in BF16 78 us. A single row
// of 151936 takes 5.3 us, the latency of its dependent reads, and 64 of them 27 (58 MB), bound by the issue
// of the counting. What made the difference (from 160 us):
//  * A block owns a tile of the vocabulary of one request and counts the request's history into a 32-bit
//    word per entry in shared memory; the words then serve all rows of the request, one per node of a draft
//    tree (each tile re-reads the history, from L2). Word: bits 0-19 the count of generated tokens, then
//    flags: in the prompt, drafted, biased.
//  * Few entries have a word. Each warp lists those of its part once, and per row treats them 32 at a time
//    in shared memory before all entries are scaled, masked and stored: a test per entry and row took
//    200 instructions per eight entries, more than the SMs issue in the time that the bytes take.
//  * Rows come by asynchronous copies a row ahead, the first ones before the history is counted.
//  * Drafted and biased entries have a record, so that no row searches lists or waits for a global read.
// Counts are integers and the last of several biases of one token holds by its index, so nothing depends on
// the order of atomics.
#include "common.cuh"

namespace qk {
namespace {

constexpr int kLogitThreads = 256, kLogitWarps = kLogitThreads / 32;
constexpr int kLogitBlocks = 3;  // per SM: shared memory
constexpr int kVec = 8;  // entries per access
constexpr int kMaxBias = 1024, kMaxNodes = 64, kMaxTile = 4096;  // tiles of 2048: 97 us for 88
constexpr int kMaxHistory = (1 << 20) - 1;
constexpr uint32_t kCountMask = (1u << 20) - 1, kPrompt = 1u << 20, kDraft = 1u << 21, kBias = 1u << 22;

struct LogitArgs {
  qk_logits_desc d;
  const void* logits;
  float* out;
  int B, N, V, tile, rows_per_block;
  bool vector;  // logits and out start on a whole access
};

// Penalties of an entry of word w whose context also has `drafted` occurrences on the row's path.
struct Penalties {
  float rep, inv_rep, freq, pres;
  __device__ float operator()(float x, uint32_t w, int drafted) const {
    const int count = static_cast<int>(w & kCountMask) + drafted;
    const float scaled = x * (x > 0.f ? inv_rep : rep);
    x = count > 0 || (w & kPrompt) ? scaled : x;
    return count > 0 ? x - fmaf(freq, static_cast<float>(count), pres) : x;
  }
};

// A block's entries: the tile's and the kVec before it, for the rows whose accesses begin there.
constexpr int kEntries = kMaxTile + kVec;
constexpr int kSegment = kMaxTile / kLogitWarps;  // entries per warp and row, at most
constexpr int kList = kSegment + kVec, kMaskWords = kSegment / 32 + 2;
// Rows on their way to a warp (a third of BF16 costs a block per SM: 78 -> 96 us); of BF16 they take half of
// the room, and the row at hand in FP32 the other half.
constexpr int kStages = 2, kRowBytes = kStages * 4 * kSegment;

struct Tile {
  alignas(16) uint8_t rows[kLogitWarps][kRowBytes];
  uint32_t masks[kLogitWarps][kStages][kMaskWords];
  alignas(16) uint32_t words[kEntries];
  uint16_t list[kLogitWarps][kList];  // the entries that have a word
  // Drafted or biased entries have a record: of a drafted token the number of its first node, of others
  // kMaxNodes + the place of the bias that holds.
  uint32_t record_word[kMaxNodes + kMaxBias];
  float record_bias[kMaxNodes + kMaxBias];
  uint64_t path[kMaxNodes], ancestors[kMaxNodes];  // the nodes that carry a record's token; per row
  int draft[kMaxNodes], draft_id[kMaxNodes];
  uint16_t bias_id[kMaxBias], bias_at[kMaxBias];
  int bias_n;
};

// An entry of word w in row r of the request. The word of a drafted or biased one has its record's number
// in place of the count.
__device__ __forceinline__ float processed(float x, uint32_t w, int r, const Tile& s, const Penalties& penalties) {
  if (!(w & (kDraft | kBias))) return penalties(x, w, 0);
  const uint32_t i = w & kCountMask, whole = s.record_word[i];
  x = penalties(x, whole, i < kMaxNodes ? __popcll(s.path[i] & s.ancestors[r]) : 0);
  return whole & kBias ? x + s.record_bias[i] : x;
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
  x = processed(x, s.words[j], r, s, penalties);
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
    lo = v < 0;  // by seven entries at most: the first access is not whole
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
  constexpr int kSize = BF16 ? 2 : 4, kBatch = kSegment / (32 * kVec);
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
  for (int i = tid * 4; i < a.tile + kVec; i += kLogitThreads * 4)
    *reinterpret_cast<uint4*>(s.words + i) = make_uint4(0, 0, 0, 0);
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
  const int32_t* bias_ids = d.bias_ids + static_cast<int64_t>(b) * d.bias_count;
  const float* bias = d.bias + static_cast<int64_t>(b) * d.bias_count;
  const int first_id = tid < d.bias_count ? bias_ids[tid] : 0;
  const float first_bias = tid < d.bias_count ? bias[tid] : 0.f;
  __syncthreads();
  // Tokens in flight per thread; the first of them do not wait for the length. 64 rows of 151936 with histories
  // of up to 2048: 27 us at 8, 30 at 16; with a branch around each of the 16 instead, 16 x 24 rows 112 for 88.
  constexpr int kAhead = 8;
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
  for (int k = tid; k < d.bias_count; k += kLogitThreads) {
    const uint32_t v = static_cast<uint32_t>(k == tid ? first_id : bias_ids[k]) - static_cast<uint32_t>(v0);
    if (v < n) {
      const int at = atomicAdd(&s.bias_n, 1);
      s.bias_id[at] = static_cast<uint16_t>(v);
      s.bias_at[at] = static_cast<uint16_t>(k);
      s.record_bias[kMaxNodes + at] = k == tid ? first_bias : bias[k];
      atomicOr(&s.words[v], kBias);
    }
  }
  __syncthreads();
  if (d.drafts) {  // a record of each token that is drafted, by its first node
    if (tid < a.N) {
      const int id = s.draft[tid];
      const uint32_t v = static_cast<uint32_t>(id) - static_cast<uint32_t>(v0);
      uint64_t path = 0;
      for (int j = 0; j < a.N; ++j) path |= static_cast<uint64_t>(s.draft[j] == id) << j;
      if (v < n && __ffsll(path) - 1 == tid) {
        const uint32_t w = s.words[v] | kDraft;
        if (w & kBias) s.record_bias[tid] = s.record_bias[kMaxNodes + last_bias(s, static_cast<int>(v))];
        s.path[tid] = path;
        s.record_word[tid] = w;
        s.words[v] = kDraft | tid;
      }
    }
    __syncthreads();
  }
  if (s.bias_n) {  // and of each other token that is biased
    for (int k = tid; k < s.bias_n; k += kLogitThreads) {
      const int entry = s.bias_id[k];
      const uint32_t w = s.words[entry];
      if (w & kDraft || last_bias(s, entry) != k) continue;
      s.record_word[kMaxNodes + k] = w;
      s.words[entry] = kBias | (kMaxNodes + k);
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
  // what the warp's rows have to treat: the entries of its parts, which begin at one of eight places. Four
  // entries per lane; an entry's place follows those of the lanes before it and its lane's own before it.
  int listed = 0;
  const uint32_t below = (1u << lane) - 1;
  for (int j0 = warp * segment, end = j0 + segment + kVec; j0 < end; j0 += 128) {
    const int j = j0 + 4 * lane;
    const uint4 u = j < end ? lds_v4(s.words + j) : make_uint4(0, 0, 0, 0);
    if (!__any_sync(0xffffffffu, (u.x | u.y | u.z | u.w) != 0)) continue;
    uint32_t all[4];
    int at = listed;
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      all[t] = __ballot_sync(0xffffffffu, word(u, t) != 0);
      at += __popc(all[t] & below);
      listed += __popc(all[t]);
    }
#pragma unroll
    for (int t = 0; t < 4; ++t)
      if (word(u, t) != 0) s.list[warp][at++] = static_cast<uint16_t>(j + t);
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
      const int j = s.list[warp][i], l = j + v0 - part.v;
      if (l < part.lo * kVec || l >= part.hi * kVec) continue;
      float* at = reinterpret_cast<float*>(x + swizzled(l >> 2) * 16) + (l & 3);
      *at = processed(*at, s.words[j], r, s, penalties);
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
  // A block takes several rows of its request (each repeats the counting), but leaves 8 blocks per SM where
  // there are as many: tiles of frequent tokens take longer than others. 16 x 24 rows of 151937: 88 us at 8,
  // 95 at 4, 96 at 12.
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
