// A verify step's bookkeeping over a pool of cache pages, and the Q8 append by slot.
//
// The pool is a Q8 cache of the library's layout (codes int8 [R, T, kv*hd], scale planes BF16
// [R*G, T]) whose R*T token slots are cut into pages of P slots; block table row b lists the
// pages of request b in order of its tokens, so token t lives in slot
// table[b, t / P] * P + t % P.
//
// Plan. With need_b = ceil((length_b + count_b) / P) pages and held_b in the table, request b
// takes want_b = max(need_b - held_b, 0) pages from the ring of free pages (in request order;
// it gets all of them or, where the ring runs out, none; nor does one that outgrows its table, without
// keeping pages from those behind it) and returns
// max(held_b - need_b, 0). Takes come from the ring's head and returns go behind its tail, so
// no block reads what another writes and every block can work alone: block (c, b) adds up the
// wants and returns of the requests before b itself (B integers from L2) and then writes the
// slots of 1024 tokens of request b. The last block row computes the new head and count.
// Ancestor words come from pointer doubling (m |= m[p], p = p[p]): six rounds for 64 nodes.
// Latency-bound, a few dependent L2 reads and one block-wide sum: 64 requests of one token take 3.4 us,
// 256 trees of 64 nodes 4.6, 61 prompt chunks of 2048 tokens 3.8, where an empty launch takes 2.
#include "common.cuh"

namespace qk {
namespace {

constexpr int kPlanThreads = 256;
constexpr int kPlanChunk = 1024;  // tokens of one request per block
constexpr int kTreeNodes = 64;    // an ancestor word has 64 bits

enum { kPlanNoPages = 1, kPlanTableFull = 2, kPlanBadLength = 4, kPlanBadParent = 8 };

struct PlanArgs {
  int32_t* table;
  const int32_t* held;
  int32_t* ring;
  const int32_t* span;
  const int32_t* lengths;
  const int32_t* counts;
  const int32_t* parents;
  int B, width, pages, shift, N;
  int32_t *slots, *positions;
  uint64_t* ancestors;
  int32_t *held_out, *span_out, *status;
};

struct Request {
  int length, count, held;
  int64_t need;
  bool bad, roomy;  // roomy: the table has a place for all its pages; one without takes none from the ring
  __device__ int64_t want() const { return roomy && need > held ? need - held : 0; }
  __device__ int64_t drop() const { return held > need ? held - need : 0; }
};

// Lengths and counts outside their ranges are brought into them (and reported): nothing below
// indexes with a value of the caller's that was not checked.
__device__ __forceinline__ Request load_request(const PlanArgs& a, int b) {
  const int n = a.lengths[b], c = a.counts[b], h = a.held[b];
  Request r;
  r.length = max(n, 0);
  r.count = min(max(c, 0), a.N);
  r.held = min(max(h, 0), a.width);
  r.bad = r.length != n || r.count != c || r.held != h;
  r.need = (static_cast<int64_t>(r.length) + r.count + (1 << a.shift) - 1) >> a.shift;
  r.roomy = r.need <= a.width;
  return r;
}

// Block-wide exclusive prefix of v over the threads, and the total.
__device__ __forceinline__ int64_t block_prefix(int64_t v, int64_t* warps, int64_t& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int64_t s = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t u = __shfl_up_sync(0xffffffffu, s, o);
    if (lane >= o) s += u;
  }
  __syncthreads();
  if (lane == 31) warps[warp] = s;
  __syncthreads();
  int64_t before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < kPlanThreads / 32; ++w) {
    if (w < warp) before += warps[w];
    total += warps[w];
  }
  return before + s - v;
}

__global__ void __launch_bounds__(kPlanThreads) paged_plan_kernel(PlanArgs a) {
  __shared__ int64_t warps[kPlanThreads / 32];
  __shared__ uint64_t word[kTreeNodes];
  __shared__ int up[kTreeNodes];
  const int b = blockIdx.y, tid = threadIdx.x;
  const int page_mask = (1 << a.shift) - 1;
  const int head = min(max(a.span[0], 0), a.pages - 1), avail = min(max(a.span[1], 0), a.pages);

  if (b == a.B) {  // the totals: which requests fit, the ring's new head and count
    if (blockIdx.x) return;
    int64_t upto = 0, taken = 0, given = 0;
    for (int b0 = 0; b0 < a.B; b0 += kPlanThreads) {
      Request r{};
      if (b0 + tid < a.B) r = load_request(a, b0 + tid);
      int64_t total, fitted, dropped;
      const int64_t w = r.want(), before = upto + block_prefix(w, warps, total);
      block_prefix(before + w <= avail ? w : 0, warps, fitted);
      block_prefix(r.drop(), warps, dropped);
      upto += total;
      taken += fitted;
      given += dropped;
    }
    if (tid == 0) {
      a.span_out[0] = static_cast<int32_t>((head + taken) % a.pages);
      a.span_out[1] = static_cast<int32_t>(avail - taken + given);
    }
    return;
  }

  int64_t want = 0, drop = 0;
  for (int j = tid; j < b; j += kPlanThreads) {
    const Request r = load_request(a, j);
    want += r.want();
    drop += r.drop();
  }
  int64_t wants, drops;
  block_prefix(want, warps, wants);
  block_prefix(drop, warps, drops);
  const Request r = load_request(a, b);
  const bool fits = r.want() == 0 || wants + r.want() <= avail;
  const int held = r.held + static_cast<int>((fits ? r.want() : 0) - r.drop());
  int32_t* row = a.table + static_cast<int64_t>(b) * a.width;
  // page p >= r.held of this request comes from the ring, in order
  auto fresh = [&](int p) { return a.ring[(head + wants + (p - r.held)) % a.pages]; };
  int status = (r.bad ? kPlanBadLength : 0) | (!r.roomy ? kPlanTableFull : fits ? 0 : kPlanNoPages);

  if (blockIdx.x == 0) {
    for (int p = r.held + tid; p < held; p += kPlanThreads) row[p] = fresh(p);
    // returned pages go behind the tail; the table keeps their (now unused) entries
    for (int p = static_cast<int>(r.need) + tid; p < r.held; p += kPlanThreads)
      a.ring[(head + avail + drops + (p - r.need)) % a.pages] = row[p];
    if (tid == 0) a.held_out[b] = held;
  }

  const int64_t out = static_cast<int64_t>(b) * a.N;
  if (a.ancestors) {  // N <= 64: one block per request
    const bool tree = a.parents != nullptr;
    bool bad = false;
    if (tid < a.N) {
      int p = tid - 1;
      if (tree) {
        p = a.parents[out + tid];
        bad = tid < r.count && (p < -1 || p >= tid);
        if (p < -1 || p >= tid) p = -1;
      }
      up[tid] = p;
      word[tid] = 1ull << tid;
    }
    status |= __syncthreads_or(bad) ? kPlanBadParent : 0;
#pragma unroll
    for (int round = 0; round < 6; ++round) {
      uint64_t m = 0;
      int p = -1;
      if (tid < a.N && up[tid] >= 0) {
        m = word[up[tid]];
        p = up[up[tid]];
      }
      __syncthreads();
      if (tid < a.N) {
        word[tid] |= m;
        up[tid] = p;
      }
      __syncthreads();
    }
  }
  if (blockIdx.x == 0 && tid == 0) a.status[b] = status;

  const int first = blockIdx.x * kPlanChunk, last = min(first + kPlanChunk, a.N);
  for (int i = first + tid; i < last; i += kPlanThreads) {
    const bool live = i < r.count;
    const int64_t t = static_cast<int64_t>(r.length) + i;
    const int64_t p = t >> a.shift;
    int slot = -1;
    if (live && p < held) {
      const int page = p < r.held ? row[p] : fresh(static_cast<int>(p));
      slot = (page << a.shift) + static_cast<int>(t & page_mask);
    }
    a.slots[out + i] = slot;
    int depth = i;
    if (a.ancestors) {
      const uint64_t m = live ? word[i] : 0;
      a.ancestors[out + i] = m;
      depth = __popcll(m) - 1;
    }
    a.positions[out + i] = live ? r.length + depth : 0;
  }
}

// rint(x / scale) of the codec, in -127 .. 127, for eight values: bytes of two words. The product with the
// reciprocal is within 2^-22 of the quotient, of about 127 at most, so it rounds to the same integer unless
// it lies that close to a half. There FP32 values, one in 4096, take the division. A quotient of two BF16
// numbers near a half is a half, as x and h * scale are multiples of 2^-8 of scale's power of two, or lies
// 2^-9 away: rounded to multiples of 2^-10 it is the half that it stands for, and rounds to even. Scales
// whose reciprocal is not normal, or not finite, take the division too.
// Adding 1.5 * 2^23 rounds and leaves the code in the sum's low byte: the conversions that this replaces
// run on a pipe an eighth as wide.
template <bool BF16>
__device__ __forceinline__ uint2 codes_of(const float (&x)[8], float scale) {
  constexpr float kRound = 12582912.f, kTenth = 12288.f;  // 1.5 * 2^23 and, to multiples of 2^-10, 1.5 * 2^13
  const float inverse = __frcp_rn(scale);
  uint32_t t[8];
  uint32_t unsure = scale > 0x1p-100f && scale < 0x1p100f ? 0u : 0xffu;  // a bit per value
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    float q = x[i] * inverse;
    if (BF16) q = (q + kTenth) - kTenth;
    const float sum = fminf(fmaxf(q, -127.f), 127.f) + kRound;
    t[i] = __float_as_uint(sum);
    if (!BF16) {
      const float off = fabsf(fabsf(q - (sum - kRound)) - 0.5f);
      unsure |= off >= 1.f / 8192 ? 0u : 1u << i;
    }
  }
  while (unsure) {
    const int i = __ffs(unsure) - 1;
    unsure &= unsure - 1;
    float n = 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k) n = k == i ? x[k] : n;
    n = fminf(fmaxf(rintf(__fdiv_rn(n, scale)), -127.f), 127.f);
    const uint32_t code = static_cast<uint32_t>(static_cast<int>(static_cast<int8_t>(n)));
#pragma unroll
    for (int k = 0; k < 8; ++k) t[k] = k == i ? code : t[k];
  }
  return make_uint2(__byte_perm(__byte_perm(t[0], t[1], 0x0040), __byte_perm(t[2], t[3], 0x0040), 0x5410),
                    __byte_perm(__byte_perm(t[4], t[5], 0x0040), __byte_perm(t[6], t[7], 0x0040), 0x5410));
}

// Codec and scatter: a thread per 8 channels (one 16-byte load of BF16, two of FP32), the
// group's maximum over its 4 lanes, 8 bytes of codes per thread and one BF16 scale per group.
// The codes and scales are the append's (scale = bf16(max|x| / 127), code = rint(x / scale) of IEEE
// quotients), so a token's bytes do not depend on the entry point that wrote it. 8111 tokens of 8 heads of
// 128: 22.0 us from FP32 (84 MB, 3.8 TB/s, 58% of measured HBM) and 22.7 from BF16, bound by the issue of
// about 150 instructions per 8 channels; 64 tokens: 2.1 us.
template <bool BF16>
__global__ void __launch_bounds__(256) write_slots_kernel(const void* __restrict__ key, const void* __restrict__ value,
                                                          int64_t key_stride, int64_t value_stride,
                                                          const int32_t* __restrict__ slots, int8_t* k_codes,
                                                          int8_t* v_codes, uint16_t* k_scale, uint16_t* v_scale,
                                                          uint32_t total, Divider by_D8, int G, int group8, int64_t T,
                                                          int64_t room) {
  pdl_wait();  // launched as a programmatic dependent: the keys' and values' producer first
  pdl_trigger();
  const uint32_t i = blockIdx.x * blockDim.x + threadIdx.x;  // below 2^31: checked by the host
  const bool in = i < total;
  const int D8 = static_cast<int>(by_D8.divisor);
  const uint32_t item = in ? by_D8(i) : 0;
  const int col = in ? static_cast<int>(i - item * D8) : 0;
  const bool is_value = item & 1;
  const int64_t token = item >> 1;
  const int64_t slot = in ? slots[token] : -1;
  float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  const bool live = in && slot >= 0 && slot < room;
  if (in) {  // also where the slot says padding: the values need not wait for it
    const int64_t at = token * (is_value ? value_stride : key_stride) + col * 8;
    if (BF16) {
      unpack8(ld_guarded_v4(static_cast<const uint16_t*>(is_value ? value : key) + at), x);
    } else {
      const float* p = static_cast<const float*>(is_value ? value : key) + at;
      const uint4 u = ld_guarded_v4(p), v = ld_guarded_v4(p + 4);
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        x[t] = __uint_as_float(word(u, t));
        x[4 + t] = __uint_as_float(word(v, t));
      }
    }
  }
  float amax = 0.f;
#pragma unroll
  for (int t = 0; t < 8; ++t) amax = fmaxf(amax, fabsf(x[t]));
  for (int o = group8 >> 1; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
  if (!live) return;
  const float scale = bf16_round(__fdiv_rn(amax, 127.f));
  const float divisor = scale == 0.f ? 1.f : scale;
  int8_t* codes = is_value ? v_codes : k_codes;
  *reinterpret_cast<uint2*>(codes + (slot * D8 + col) * 8) = codes_of<BF16>(x, divisor);
  if ((col & (group8 - 1)) == 0) {
    const int64_t row = slot < T ? 0 : slot / T, t = slot - row * T;
    (is_value ? v_scale : k_scale)[(row * G + (col >> (31 - __clz(group8)))) * T + t] = bf16_bits_rne(scale);
  }
}

}  // namespace
}  // namespace qk

using namespace qk;

extern "C" {

int qk_paged_plan(int32_t* table, const int32_t* held, int32_t* ring, const int32_t* span, const int32_t* lengths,
                  const int32_t* counts, const int32_t* parents, int B, int width, int pages, int page_size, int N,
                  int32_t* slots, int32_t* positions, uint64_t* ancestors, int32_t* held_out, int32_t* span_out,
                  int32_t* status, qk_stream_t stream) {
  QK_REQUIRE(B >= 0 && B < 65535 && N >= 1 && width >= 1 && pages >= 1, "invalid batch, nodes, table width or pages");
  QK_REQUIRE(page_size >= 16 && page_size <= 1024 && (page_size & (page_size - 1)) == 0,
             "page_size must be a power of two in [16, 1024]");
  QK_REQUIRE(static_cast<int64_t>(pages) * page_size <= 0x7fffffff, "the pool's slots must fit 31 bits");
  QK_REQUIRE(N <= kTreeNodes || (!parents && !ancestors), "a draft tree has at most %d nodes", kTreeNodes);
  QK_REQUIRE(!parents || ancestors, "parents need an ancestors output");
  QK_REQUIRE(held && ring && span && span_out && (B == 0 || (table && lengths && counts && slots && positions && held_out && status)),
             "null pointer");
  QK_REQUIRE(held_out != held && span_out != span, "held_out and span_out must be other arrays than held and span");
  PlanArgs a{table, held, ring, span, lengths, counts, parents, B, width, pages, 0, N, slots, positions, ancestors,
             held_out, span_out, status};
  while ((1 << a.shift) < page_size) ++a.shift;
  const dim3 grid((N + kPlanChunk - 1) / kPlanChunk, B + 1);
  paged_plan_kernel<<<grid, kPlanThreads, 0, as_stream(stream)>>>(a);
  QK_LAUNCHED("paged_plan_kernel");
  return QK_OK;
}

int qk_kv_q8_write_slots(const void* key, const void* value, int in_dtype, int64_t key_stride, int64_t value_stride,
                         const int32_t* slots, int8_t* k_codes, int8_t* v_codes, uint16_t* k_scale, uint16_t* v_scale,
                         int64_t tokens, int rows, int64_t T, int kv_heads, int head_dim, qk_stream_t stream) {
  QK_REQUIRE(in_dtype == QK_OUT_F32 || in_dtype == QK_OUT_BF16, "in_dtype must be F32 or BF16");
  QK_REQUIRE(tokens >= 0 && rows > 0 && T > 0 && kv_heads > 0 && head_dim > 0, "invalid cache geometry");
  const int group = head_dim < 32 ? head_dim : 32;  // config.py:91-93
  QK_REQUIRE(group >= 8 && (group & (group - 1)) == 0 && head_dim % group == 0,
             "head_dim must divide into cache quantization groups of 8, 16 or 32");
  if (tokens == 0) return QK_OK;
  QK_REQUIRE(key && value && slots && k_codes && v_codes && k_scale && v_scale, "null pointer");
  const int D = kv_heads * head_dim, per = in_dtype == QK_OUT_BF16 ? 8 : 4;
  QK_REQUIRE(key_stride >= D && value_stride >= D && key_stride % per == 0 && value_stride % per == 0 &&
                 ((reinterpret_cast<uintptr_t>(key) | reinterpret_cast<uintptr_t>(value)) & 15) == 0,
             "key and value rows must be 16-byte aligned and not overlap");
  QK_REQUIRE(((reinterpret_cast<uintptr_t>(k_codes) | reinterpret_cast<uintptr_t>(v_codes)) & 7) == 0,
             "codes must be 8-byte aligned");
  const int64_t total = tokens * 2 * (D / 8);
  const int64_t grid = (total + 255) / 256;
  QK_REQUIRE(grid * 256 < (1ll << 31), "too many tokens in one call");
  const auto kernel = in_dtype == QK_OUT_BF16 ? write_slots_kernel<true> : write_slots_kernel<false>;
  const cudaError_t e = launch_dependent(kernel, dim3(static_cast<unsigned>(grid)), dim3(256), 0, as_stream(stream),
                                         key, value, key_stride, value_stride, slots, k_codes, v_codes, k_scale, v_scale,
                                         static_cast<uint32_t>(total), Divider(D / 8), D / group, group / 8, T,
                                         static_cast<int64_t>(rows) * T);
  if (e != cudaSuccess) return cuda_error(e, "write_slots_kernel");
  count_launch();
  return QK_OK;
}

}  // extern "C"
