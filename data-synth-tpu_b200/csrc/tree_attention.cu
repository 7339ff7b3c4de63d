// Attention of drafted tokens over a paged Q8 cache, on the tcgen05 tensor core.
//
//   out[b, i, h] = sigmoid(gate) * sum_t p_t v_t,  p = softmax over the tokens t that node i of
//   request b sees of (q . k_t) * scale: the request's prefix t < length_b, and of the drafts
//   t = length_b + j (j < count_b) those whose bit j is set in the node's ancestor word. Keys and
//   values are code * scale of the Q8 cache, token t in slot table[b, t / P] * P + t % P. A node
//   that sees nothing and the rows i >= count_b are zero.
//
// The nodes and query heads that share a KV head are the rows of one matrix (row i * rep + h),
// in tiles of 128: S = Q K^T and O += P V are M = 128 products over tiles of 64 tokens, so the
// cache is read and decoded once for up to 128 rows. Work: (request, KV head, row tile) units
// times their token tiles, laid end to end and cut into one equal range per SM; a unit cut by a
// range's end leaves FP32 partials (O, maximum, sum) that a second kernel joins.
//
// One CTA per SM, three kinds of warps joined by mbarriers (every wait bounded):
//  * 4 softmax warps, a thread per row: Q to TMEM once per unit; then per tile S from TMEM, mask,
//    running maximum and sum in FP32, P as BF16 back over S's columns. O (FP32, in TMEM) is rescaled
//    only when a row's maximum grows by more than 2^8: P stays below 2^8, exact enough in FP32.
//  * 8 decode warps (4 for K, 4 for V): 16-byte loads of codes straight to registers two tiles
//    ahead, int8 -> BF16 with the group's scale (one rounding, as the cache's BF16 read has it),
//    stored as 128-byte swizzled tiles: K-major for K, and the same bytes read as an MN-major
//    operand for V (no transposition).
//  * 1 warp issues the MMAs: Q and P from TMEM, K and V from shared memory.
// TMEM: O 256 columns, Q 128, two S/P buffers of 64.
#include "umma.cuh"

namespace qk {
namespace {

constexpr int kTile = 64;   // tokens per tile
constexpr int kRows = 128;  // query rows per tile
constexpr int kStages = 2;
constexpr int kSoftmaxWarps = 4, kDecodeWarps = 8;
constexpr int kThreads = (kSoftmaxWarps + kDecodeWarps + 1) * 32;
constexpr uint32_t kColO = 0, kColQ = 256, kColS = 384;  // TMEM columns
constexpr float kLazyGrowth = 8.f;                       // in powers of two
constexpr uint32_t kHugeScale = 0x7c00;                  // BF16 bits of 2^121: times 127 leaves FP32's range
constexpr int kBadRing = 4;
constexpr int kUnitCost = 4;  // what a unit costs besides its tiles (Q, the output), in tiles

struct TreeArgs {
  const uint16_t* q;
  int64_t q_stride;
  const int8_t *k_codes, *v_codes;
  const uint16_t *k_scale, *v_scale;
  const int32_t *table, *lengths, *counts;
  const uint64_t* ancestors;
  const uint16_t* gate;
  float scale_log2;         // |scale| * log2(e), above zero
  uint32_t q_keep, q_flip;  // Q's bits & keep ^ flip: nothing for a scale of zero, the sign for a negative one
  int B, N, hq, kv, rep, pages, pages_per_row, width, shift, part_rows;
  int64_t T;
  uint16_t* out;
  int* status;
  float* part;   // [2 * CTAs][HD][part_rows] unnormalised O
  float* stats;  // [2 * CTAs][2][part_rows] maximum (log2) and sum
  struct Cut* cuts;  // [CTAs]
};

// What a range's CTA knows of the unit that its range begins inside of, where it is the first
// to do so: the unit, its parts (consecutive ranges) and which record of the first range is its.
struct Cut {
  int b, head, row_tile, count, parts, record;
};

struct Request {
  int length, count, tiles, row_tiles;
  bool cut;
  // A unit's share of the ranges: its tiles and kUnitCost steps that stand for Q and the output.
  __device__ int steps() const { return tiles + kUnitCost; }
  __device__ int64_t work(int kv) const { return tiles ? static_cast<int64_t>(kv) * row_tiles * steps() : 0; }
};

__device__ __forceinline__ Request load_request(const TreeArgs& a, int b) {
  const int64_t room = min(static_cast<int64_t>(a.width) << a.shift, int64_t(0x7fffffc0));
  const int n = a.lengths[b], c = a.counts ? a.counts[b] : a.N;
  Request r;
  r.length = static_cast<int>(min(static_cast<int64_t>(max(n, 0)), room));
  r.count = static_cast<int>(min(static_cast<int64_t>(min(max(c, 0), a.N)), room - r.length));
  r.cut = r.length != n || r.count != c;
  r.row_tiles = (r.count * a.rep + kRows - 1) / kRows;
  r.tiles = r.count ? (r.length + r.count + kTile - 1) / kTile : 0;
  return r;
}

// The CTAs' ranges of a total of `total` steps, at least one step each.
__device__ __forceinline__ int ranges(int64_t total, int ctas) {
  return static_cast<int>(total < ctas ? total : ctas);
}
__device__ __forceinline__ int64_t range_start(int64_t total, int n, int c) { return c * total / n; }
__device__ __forceinline__ int range_owner(int64_t total, int n, int64_t step) {
  return static_cast<int>(((step + 1) * n - 1) / total);
}

// Total work of all requests, and the request that holds step `want` of it with the step's
// offset in it: threads sum consecutive requests, a block scan, one thread walks its few.
struct Located {
  int64_t total, offset;
  int b;
};
template <class Want>
__device__ __forceinline__ Located locate(const TreeArgs& a, Located* shared, int64_t* warps, Want want, bool report) {
  constexpr int THREADS = kThreads;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int per = (a.B + THREADS - 1) / THREADS;
  const int b0 = min(tid * per, a.B), b1 = min(b0 + per, a.B);
  int64_t sum = 0;
  for (int b = b0; b < b1; ++b) {
    const Request r = load_request(a, b);
    if (r.cut && report) *a.status = QK_ERR_INVALID_ARGUMENT;
    sum += r.work(a.kv);
  }
  int64_t s = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t u = __shfl_up_sync(0xffffffffu, s, o);
    if (lane >= o) s += u;
  }
  if (lane == 31) warps[warp] = s;
  __syncthreads();
  int64_t before = s - sum, total = 0;
  for (int w = 0; w < THREADS / 32; ++w) {
    if (w < warp) before += warps[w];
    total += warps[w];
  }
  if (tid == 0) *shared = Located{total, 0, a.B};
  __syncthreads();
  const int64_t step = want(total);
  if (step >= before && step < before + sum) {
    int64_t off = step - before;
    for (int b = b0; b < b1; ++b) {
      const int64_t w = load_request(a, b).work(a.kv);
      if (off < w) {
        shared->offset = off;
        shared->b = b;
        break;
      }
      off -= w;
    }
  }
  __syncthreads();
  return *shared;
}

// The pieces of a CTA's range: tiles [t0, t1) of one unit each. A unit's last steps are not tiles:
// a range that holds nothing else of the unit has no piece of it.
struct Segment {
  Request r;
  int b, head, row_tile, t0, t1, index;
  bool first;  // the range begins with it
  __device__ bool whole() const { return t0 == 0 && t1 == r.tiles; }
};
struct Walk {
  int b, index;
  int64_t offset, left;
  bool first;
  __device__ bool next(const TreeArgs& a, Segment& s) {
    while (left > 0) {
      for (;; ++b) {
        s.r = load_request(a, b);
        const int64_t w = s.r.work(a.kv);
        if (offset < w) break;
        offset -= w;
      }
      const int steps = s.r.steps();
      const int unit = static_cast<int>(offset / steps);
      s.b = b;
      s.head = unit / s.r.row_tiles;
      s.row_tile = unit % s.r.row_tiles;
      s.t0 = static_cast<int>(offset % steps);
      const int end = static_cast<int>(min(static_cast<int64_t>(steps), s.t0 + left));
      left -= end - s.t0;
      offset += end - s.t0;
      s.t1 = min(end, s.r.tiles);
      s.first = first;
      first = false;
      if (s.t0 >= s.t1) continue;
      s.index = index++;
      return true;
    }
    return false;
  }
};

struct Barriers {
  uint64_t k_full[kStages], k_empty[kStages], v_full[kStages], v_empty[kStages];
  uint64_t s_full[2], p_full[2], q_full, o_full;
};

struct Control {
  Barriers bar;
  uint64_t bad[kBadRing][8];  // per unit and channel group: drafts whose value scale is not finite
  Located located;
  int64_t warps[kThreads / 32];
  uint32_t tmem;
};

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// The gate, rounded to BF16 with its product right after: the approximate exponential and
// reciprocal (2^-22 each) do, at an eighth of the instructions of the exact ones.
__device__ __forceinline__ float sigmoid_fast(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(1.f + exp2_fast(x * -1.44269504088896341f)));
  return y;
}

__device__ __forceinline__ uint4 ld_stream_v4(const void* p) {
  uint4 r;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w)
               : "l"(p));
  return r;
}

__device__ __forceinline__ void sts_v4(uint32_t addr, const uint4& v) {
  asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(addr), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}

// Four int8 codes times a BF16 scale (in both halves of `scale2`) -> two BF16 pairs. A byte c
// under the exponent of 128 is 128 + (c & 127), exact in BF16; minus 128, or 256 where the sign
// bit was set, it is the code; the product rounds once.
__device__ __forceinline__ void decode4(uint32_t codes, __nv_bfloat162 scale2, uint32_t& lo, uint32_t& hi) {
  const uint32_t t[2] = {__byte_perm(codes, 0x43434343u, 0x4140), __byte_perm(codes, 0x43434343u, 0x4342)};
  uint32_t r[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t mag = t[i] & 0xff7fff7fu, off = t[i] & 0xff80ff80u;
    const __nv_bfloat162 v = __hmul2(__hsub2(*reinterpret_cast<const __nv_bfloat162*>(&mag),
                                             *reinterpret_cast<const __nv_bfloat162*>(&off)),
                                     scale2);
    r[i] = *reinterpret_cast<const uint32_t*>(&v);
  }
  lo = r[0];
  hi = r[1];
}

// A bounded wait of a whole warp, converged behind it: false for all lanes if one gave up.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity) {
  return __all_sync(0xffffffffu, mbar_wait_bounded(bar, parity));
}

// ---- decode warps -------------------------------------------------------------------------

// A thread's share of a tile: 16 channels of SPT consecutive tokens (all in one page; codes[i] of
// token i ^ swap), and their group's scales (token i in half i % 2 of word i / 2).
template <int HD>
struct Share {
  static constexpr int SPT = HD / 32;
  uint4 codes[SPT];
  uint32_t scales[SPT / 2];
};

template <int HD>
__device__ __forceinline__ void load_share(const TreeArgs& a, const int8_t* codes, const uint16_t* scale, int head,
                                           int page, int token, int total, int chunk, int swap, Share<HD>& s) {
  constexpr int SPT = HD / 32;
  if (token >= total) {
#pragma unroll
    for (int i = 0; i < SPT; ++i) s.codes[i] = make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int i = 0; i < SPT / 2; ++i) s.scales[i] = 0;
    return;
  }
  const int row = page / a.pages_per_row;
  const int64_t in_row = (static_cast<int64_t>(page - row * a.pages_per_row) << a.shift) + (token & ((1 << a.shift) - 1));
  const int D = a.kv * HD, G = D / 32;
  const int8_t* c = codes + (row * a.T + in_row) * D + head * HD + chunk * 16;
  const uint16_t* p = scale + (static_cast<int64_t>(row) * G + head * (HD / 32) + chunk / 2) * a.T + in_row;
  const int8_t *even = c + swap * D, *odd = c - swap * D;
#pragma unroll
  for (int i = 0; i < SPT; ++i) s.codes[i] = ld_stream_v4((i & 1 ? odd : even) + i * D);
  if (SPT == 8) {
    const uint4 v = ld_nc_v4(p);
#pragma unroll
    for (int i = 0; i < SPT / 2; ++i) s.scales[i] = word(v, i);
  } else {
#pragma unroll
    for (int i = 0; i < SPT / 2; ++i) s.scales[i] = __ldg(reinterpret_cast<const uint32_t*>(p) + i);
  }
}

// Both kinds of decode warps run one copy of this code (K or V by run-time values), and the
// buffered tile moves to the front instead of the loop being unrolled over buffers: with a copy per
// kind and buffer the CTA's hot code left the instruction cache and ran at a tenth of its speed.
template <int HD>
__device__ __forceinline__ bool decode_role(const TreeArgs& a, Control& ctl, uint8_t* tiles, Walk walk) {
  constexpr int SPT = HD / 32, CHUNKS = HD / 16;
  constexpr uint32_t kStageBytes = kTile * HD * 2;
  const bool values = threadIdx.x >= (kSoftmaxWarps + 4) * 32;
  const int t = (threadIdx.x - kSoftmaxWarps * 32) & 127;
  const int chunk = t % CHUNKS, sub = (t / CHUNKS) * SPT;  // tokens sub .. sub + SPT - 1 of a tile
  // A token's 16 channels are the 16-byte pieces 2 chunk and 2 chunk + 1 of its row, in atoms of 64
  // channels, piece j at j ^ (token % 8). Half of the lanes take their tokens in the order 1, 0, 3,
  // 2, ..: then 8 lanes' stores fill the 8 different 16-byte banks.
  const int swap = HD == 64 ? (t / CHUNKS) & 1 : (chunk >> 2) & 1;
  const int8_t* codes = values ? a.v_codes : a.k_codes;
  const uint16_t* scale = values ? a.v_scale : a.k_scale;
  uint64_t* full = values ? ctl.bar.v_full : ctl.bar.k_full;
  uint64_t* empty = values ? ctl.bar.v_empty : ctl.bar.k_empty;
  const uint32_t mine = smem_addr(tiles) + (values ? kStages * kStageBytes : 0) + (chunk >> 2) * (kTile * 128) +
                        ((sub ^ swap) << 7 | (((chunk & 3) * 2) ^ ((sub ^ swap) & 7)) << 4);
  const uint32_t select[2] = {swap ? 0x3232u : 0x1010u, swap ? 0x1010u : 0x3232u};
  // the loads run two tiles ahead of the stores, page numbers one further, across units
  Walk ahead = walk;
  Segment aseg;
  int atile = 0, atotal = 0;
  bool amore = ahead.next(a, aseg);
  if (amore) {
    atile = aseg.t0;
    atotal = aseg.r.length + aseg.r.count;
  }
  auto page_of = [&]() {
    const int token = atile * kTile + sub;
    if (!amore || token >= atotal) return 0;
    const int page = __ldg(a.table + static_cast<int64_t>(aseg.b) * a.width + (token >> a.shift));
    if (page < 0 || page >= a.pages) {
      *a.status = QK_ERR_INVALID_ARGUMENT;
      return 0;
    }
    return page;
  };
  int page = page_of();
  Share<HD> cur, next;
  Segment seg;
  int tile = 0;
  seg.t1 = 0;
  uint32_t it = 0;
  bool primed = false;
  for (;;) {
    cur = next;
    if (amore) {
      load_share<HD>(a, codes, scale, aseg.head, page, atile * kTile + sub, atotal, chunk, swap, next);
      if (++atile == aseg.t1) {
        amore = ahead.next(a, aseg);
        if (amore) {
          atile = aseg.t0;
          atotal = aseg.r.length + aseg.r.count;
        }
      }
      page = page_of();
    }
    if (!primed) {
      primed = true;
      continue;
    }
    if (tile == seg.t1) {
      if (!walk.next(a, seg)) return true;
      tile = seg.t0;
    }
    const int token0 = tile * kTile + sub;
    if (tile * kTile + kTile > seg.r.length) {  // drafts, or past the end
      const int total = seg.r.length + seg.r.count;
#pragma unroll
      for (int i = 0; i < SPT; ++i) {
        const int token = token0 + i;
        const uint32_t mask = i & 1 ? 0xffff0000u : 0xffffu;
        const uint32_t bits = cur.scales[i / 2] >> (16 * (i & 1)) & 0x7fffu;
        if (token >= total) {
          cur.scales[i / 2] &= ~mask;
        } else if (values && token >= seg.r.length && bits >= kHugeScale) {
          // a draft's value that is not finite must not reach the rows that do not see it (0 * inf):
          // zero here, NaN at the end for those that do
          atomicOr(reinterpret_cast<unsigned long long*>(&ctl.bad[seg.index % kBadRing][chunk / 2]),
                   1ull << (token - seg.r.length));
          cur.scales[i / 2] &= ~mask;
        }
      }
    }
    const uint32_t stage = it % kStages;
    if (!warp_wait(&empty[stage], ((it / kStages) & 1) ^ 1)) return false;
    const uint32_t base = mine + stage * kStageBytes;
#pragma unroll
    for (int i = 0; i < SPT; ++i) {
      const uint32_t two = __byte_perm(cur.scales[i / 2], 0, select[i & 1]);
      const __nv_bfloat162 scale2 = *reinterpret_cast<const __nv_bfloat162*>(&two);
      uint4 piece[2];
      decode4(cur.codes[i].x, scale2, piece[0].x, piece[0].y);
      decode4(cur.codes[i].y, scale2, piece[0].z, piece[0].w);
      decode4(cur.codes[i].z, scale2, piece[1].x, piece[1].y);
      decode4(cur.codes[i].w, scale2, piece[1].z, piece[1].w);
      const uint32_t to = base ^ (i << 7 | i << 4);
      sts_v4(to, piece[0]);
      sts_v4(to ^ 16, piece[1]);
    }
    fence_proxy_async_smem();
    mbar_arrive(&full[stage]);
    ++it;
    ++tile;
  }
}

// ---- MMA warp -----------------------------------------------------------------------------

template <int HD>
__device__ __forceinline__ bool mma_role(const TreeArgs& a, Control& ctl, uint8_t* ktiles, uint8_t* vtiles, Walk walk) {
  constexpr uint32_t kStageBytes = kTile * HD * 2;
  const uint32_t tm = ctl.tmem;
  const uint32_t idesc_s = idesc_bf16_m128(kTile), idesc_o = idesc_bf16_m128_bmn(HD);
  Segment seg;
  uint32_t it = 0;
  auto scores = [&](uint32_t i) {
    const uint32_t stage = i % kStages;
    if (!mbar_wait_bounded(&ctl.bar.k_full[stage], (i / kStages) & 1)) return false;
    tc_fence_after();
    const uint32_t base = smem_addr(ktiles + stage * kStageBytes);
#pragma unroll
    for (int k = 0; k < HD / 16; ++k) {
      const uint64_t desc = sdesc_sw128(base + (k / 4) * (kTile * 128) + (k % 4) * 32, 1024u);
      umma_ts(tm + kColS + (i & 1) * kTile, tm + kColQ + k * 8, desc, idesc_s, k != 0);
    }
    umma_commit(&ctl.bar.k_empty[stage]);
    umma_commit(&ctl.bar.s_full[i & 1]);
    return true;
  };
  auto values = [&](uint32_t i, bool first) {
    const uint32_t stage = i % kStages;
    if (!mbar_wait_bounded(&ctl.bar.v_full[stage], (i / kStages) & 1)) return false;
    if (!mbar_wait_bounded(&ctl.bar.p_full[i & 1], (i / 2) & 1)) return false;
    tc_fence_after();
    const uint32_t base = smem_addr(vtiles + stage * kStageBytes);
#pragma unroll
    for (int k = 0; k < kTile / 16; ++k) {
      const uint64_t desc = sdesc_sw128_mn(base + k * 2048, kTile * 128, 1024u);
      umma_ts(tm + kColO, tm + kColS + (i & 1) * kTile + k * 8, desc, idesc_o, !first || k != 0);
    }
    umma_commit(&ctl.bar.v_empty[stage]);
    return true;
  };
  while (walk.next(a, seg)) {
    if (!mbar_wait_bounded(&ctl.bar.q_full, seg.index & 1)) return false;
    tc_fence_after();
    const int n = seg.t1 - seg.t0;
    for (int j = 0; j <= n; ++j) {
      if (j < n && !scores(it + j)) return false;
      if (j > 0 && !values(it + j - 1, j == 1)) return false;
    }
    umma_commit(&ctl.bar.o_full);
    it += n;
  }
  return true;
}

// ---- softmax warps ------------------------------------------------------------------------

template <int HD>
__device__ __forceinline__ bool softmax_role(const TreeArgs& a, Control& ctl, Walk walk) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t tm = ctl.tmem + (static_cast<uint32_t>(warp * 32) << 16);
  Segment seg;
  uint32_t it = 0;
  while (walk.next(a, seg)) {
    const int row = seg.row_tile * kRows + warp * 32 + lane;
    const int node = row / a.rep, h = seg.head * a.rep + row % a.rep;
    const bool live = node < seg.r.count;
    const bool busy = seg.row_tile * kRows + warp * 32 < seg.r.count * a.rep;  // the same for the warp
    const int64_t bn = static_cast<int64_t>(seg.b) * a.N + node;
    uint64_t path = 0;
    if (live) {
      path = a.ancestors[bn];
      if (seg.r.count < 64) path &= (1ull << seg.r.count) - 1;
    }
    if (busy) {
      const uint4* q = reinterpret_cast<const uint4*>(a.q + bn * a.q_stride + static_cast<int64_t>(h) * HD);
#pragma unroll
      for (int c = 0; c < HD / 64; ++c) {
        uint32_t r[32];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const uint4 v = live ? ld_nc_v4(q + c * 8 + j) : make_uint4(0, 0, 0, 0);
#pragma unroll
          for (int w = 0; w < 4; ++w) r[j * 4 + w] = (word(v, w) & a.q_keep) ^ a.q_flip;
        }
        tmem_st32(tm + kColQ + c * 32, r);
      }
      tmem_wait_st();
    }
    tc_fence_before();
    __syncwarp();
    if (lane == 0) mbar_arrive(&ctl.bar.q_full);

    float m = -INFINITY, l = 0.f;
    for (int tile = seg.t0; tile < seg.t1; ++tile, ++it) {
      if (!warp_wait(&ctl.bar.s_full[it & 1], (it / 2) & 1)) return false;
      if (busy) {
        tc_fence_after();
        uint32_t s[2][32];
        const uint32_t cols = tm + kColS + (it & 1) * kTile;
        tmem_ld32(cols, s[0]);
        tmem_ld32(cols + 32, s[1]);
        tmem_wait_ld();
        const int first = tile * kTile;
        if (first + kTile > seg.r.length) {  // drafts, or past the end: the row's 64 bits
          const int cut = seg.r.length - first;
          uint64_t see = 0;
          if (cut > 0) see = cut < 64 ? (path << cut) | ((1ull << cut) - 1) : ~0ull;
          else if (cut > -64) see = path >> -cut;
          if (!live) see = 0;
#pragma unroll
          for (int j = 0; j < 64; ++j)
            if (!(see >> j & 1)) s[j / 32][j % 32] = 0xff800000u;
        }
        float top = __uint_as_float(s[0][0]);
#pragma unroll
        for (int j = 1; j < 64; ++j) top = fmaxf(top, __uint_as_float(s[j / 32][j % 32]));
        top *= a.scale_log2;
        const bool grow = top > m + kLazyGrowth;
        if (__any_sync(0xffffffffu, grow)) {
          const float next = fmaxf(m, top);
          const float keep = m == -INFINITY ? 0.f : exp2_fast(m - next);
          m = next;
          l *= keep;
          if (tile > seg.t0) {
            // every product so far has left O: the commit of the tile before
            const uint32_t last = it - 1;
            if (!warp_wait(&ctl.bar.v_empty[last % kStages], (last / kStages) & 1)) return false;
            tc_fence_after();
#pragma unroll 1
            for (int c = 0; c < HD / 32; ++c) {
              uint32_t o[32];
              tmem_ld32(tm + kColO + c * 32, o);
              tmem_wait_ld();
#pragma unroll
              for (int j = 0; j < 32; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * keep);
              tmem_st32(tm + kColO + c * 32, o);
            }
          }
        }
        const float shift = m == -INFINITY ? 0.f : m;
        float sum[4] = {0.f, 0.f, 0.f, 0.f};
        uint32_t p[32];
#pragma unroll
        for (int j = 0; j < 32; ++j) {
          const float x = exp2_fast(fmaf(__uint_as_float(s[j / 16][(2 * j) % 32]), a.scale_log2, -shift));
          const float y = exp2_fast(fmaf(__uint_as_float(s[j / 16][(2 * j + 1) % 32]), a.scale_log2, -shift));
          sum[j & 1] += x;
          sum[2 + (j & 1)] += y;
          p[j] = pack_bf16x2(x, y);
        }
        l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
        tmem_st32(cols, p);
        tmem_wait_st();
        tc_fence_before();
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&ctl.bar.p_full[it & 1]);
    }

    if (!warp_wait(&ctl.bar.o_full, seg.index & 1)) return false;
    if (!busy) continue;
    tc_fence_after();
    const uint64_t* bad = ctl.bad[seg.index % kBadRing];
    if (seg.whole()) {
      const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
      const int64_t at = (bn * a.hq + h) * HD;
#pragma unroll 1
      for (int c = 0; c < HD / 32; ++c) {
        uint32_t o[32];
        uint4 gate[4];
        if (a.gate && live) {
#pragma unroll
          for (int j = 0; j < 4; ++j) gate[j] = ld_nc_v4(a.gate + at + c * 32 + j * 8);
        }
        __syncwarp();
        tmem_ld32(tm + kColO + c * 32, o);
        tmem_wait_ld();
        const bool poisoned = bad[c] & path;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (!live) break;
          float f[8];
#pragma unroll
          for (int k = 0; k < 8; ++k) f[k] = poisoned ? __uint_as_float(0x7fc00000u) : __uint_as_float(o[j * 8 + k]) * inv;
          if (a.gate) {
            float z[8];
            unpack8(gate[j], z);
#pragma unroll
            for (int k = 0; k < 8; ++k) f[k] *= sigmoid_fast(z[k]);
          }
          uint32_t w[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) w[k] = pack_bf16x2(f[2 * k], f[2 * k + 1]);
          *reinterpret_cast<uint4*>(a.out + at + c * 32 + j * 8) = make_uint4(w[0], w[1], w[2], w[3]);
        }
        __syncwarp();
      }
    } else {
      const int64_t slot = 2 * static_cast<int64_t>(blockIdx.x) + (seg.first ? 0 : 1);
      float* part = a.part + slot * HD * a.part_rows + warp * 32 + lane;
#pragma unroll 1
      for (int c = 0; c < HD / 32; ++c) {
        uint32_t o[32];
        tmem_ld32(tm + kColO + c * 32, o);
        tmem_wait_ld();
        const bool poisoned = bad[c] & path;
#pragma unroll
        for (int j = 0; j < 32; ++j)
          part[(c * 32 + j) * a.part_rows] = poisoned ? __uint_as_float(0x7fc00000u) : __uint_as_float(o[j]);
      }
      float* stats = a.stats + slot * 2 * a.part_rows + warp * 32 + lane;
      stats[0] = m;
      stats[a.part_rows] = l;
    }
    tc_fence_before();
    if (seg.r.length < seg.t1 * kTile) {  // the unit saw drafts: its record of bad values is read, clear it
      asm volatile("bar.sync 1, %0;" ::"r"(32 * min(kSoftmaxWarps, (seg.r.count * a.rep - seg.row_tile * kRows + 31) / 32)) : "memory");
      if (warp == 0 && lane < 8) ctl.bad[seg.index % kBadRing][lane] = 0;
    }
  }
  return true;
}

template <int HD>
__global__ void __launch_bounds__(kThreads, 1) tree_attention_kernel(TreeArgs a) {
  extern __shared__ uint8_t smem_raw[];
  __shared__ Control ctl;
  uint8_t* tiles = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  constexpr uint32_t kStageBytes = kTile * HD * 2;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&ctl.bar.k_full[i], 128);
      mbar_init(&ctl.bar.k_empty[i], 1);
      mbar_init(&ctl.bar.v_full[i], 128);
      mbar_init(&ctl.bar.v_empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&ctl.bar.s_full[i], 1);
      mbar_init(&ctl.bar.p_full[i], kSoftmaxWarps);
    }
    mbar_init(&ctl.bar.q_full, kSoftmaxWarps);
    mbar_init(&ctl.bar.o_full, 1);
    fence_mbar_init();
  }
  if (threadIdx.x < kBadRing * 8) ctl.bad[threadIdx.x / 8][threadIdx.x % 8] = 0;
  constexpr int kMmaWarp = kSoftmaxWarps + kDecodeWarps;
  if (warp == kMmaWarp) tmem_alloc(&ctl.tmem, 512);
  tc_fence_before();
  pdl_wait();
  pdl_trigger();
  const int me = blockIdx.x;
  const Located at = locate(
      a, &ctl.located, ctl.warps,
      [&](int64_t total) {
        const int n = ranges(total, gridDim.x);
        return me < n ? range_start(total, n, me) : total;
      },
      me == 0);
  tc_fence_after();
  const int n = ranges(at.total, gridDim.x);
  Walk walk{at.b, 0, at.offset, 0, true};
  if (me < n) walk.left = range_start(at.total, n, me + 1) - range_start(at.total, n, me);

  if (threadIdx.x == 0) {
    Cut cut{0, 0, 0, 0, 0, 0};
    if (me > 0 && me < n) {
      const Request r = load_request(a, at.b);
      const int unit = static_cast<int>(at.offset / r.steps()), t = static_cast<int>(at.offset % r.steps());
      const int64_t unit0 = range_start(at.total, n, me) - t;
      const int c0 = range_owner(at.total, n, unit0), c1 = range_owner(at.total, n, unit0 + r.tiles - 1);
      if (t > 0 && t < r.tiles && c0 == me - 1)
        cut = Cut{at.b, unit / r.row_tiles, unit % r.row_tiles, r.count, c1 - c0 + 1,
                  2 * c0 + (range_start(at.total, n, c0) == unit0 ? 0 : 1)};
    }
    a.cuts[me] = cut;
  }

  // rows of nodes that are not there
  if (a.counts) {
    const int64_t row16 = static_cast<int64_t>(a.hq) * HD / 8;
    for (int64_t i = me; i < static_cast<int64_t>(a.B) * a.N; i += gridDim.x) {
      if (static_cast<int>(i % a.N) < load_request(a, static_cast<int>(i / a.N)).count) continue;
      for (int64_t j = threadIdx.x; j < row16; j += kThreads)
        reinterpret_cast<uint4*>(a.out)[i * row16 + j] = make_uint4(0, 0, 0, 0);
    }
  }

  bool ok = true;
  if (warp < kSoftmaxWarps) ok = softmax_role<HD>(a, ctl, walk);
  else if (warp < kMmaWarp) ok = decode_role<HD>(a, ctl, tiles, walk);
  else if (lane == 0) ok = mma_role<HD>(a, ctl, tiles, tiles + kStages * kStageBytes, walk);
  if (!ok) *a.status = QK_ERR_TIMEOUT;
  tc_fence_before();
  __syncthreads();
  if (warp == kMmaWarp) {
    tc_fence_after();
    tmem_dealloc(ctl.tmem, 512);
  }
}

// ---- joining the partials of a cut unit ------------------------------------------------------

// Pieces of the cut units (32 rows x 16 channels each) in turn over the blocks. A unit can have as
// many parts as there are ranges, so nothing walks them one by one: 8 warps each take every eighth
// part's statistics (a lane per row) for the common maximum and the weights, then 4 pairs of warps
// add every fourth part's channels (8 per thread) and shared memory adds the groups in a fixed order.
constexpr int kJoinThreads = 256, kJoinCols = 16, kMaxRanges = 256;

template <int HD>
__global__ void __launch_bounds__(kJoinThreads) tree_join_kernel(TreeArgs a, int ctas) {
  __shared__ int used[kMaxRanges], warps[kJoinThreads / 32];
  __shared__ float weight[kMaxRanges][32];
  __shared__ float red[2][8][32];
  __shared__ float acc[4][kJoinCols][33];
  static_assert(kMaxRanges == kJoinThreads, "a thread per range");
  pdl_wait();
  pdl_trigger();
  Cut mine{0, 0, 0, 0, 0, 0};
  if (threadIdx.x < ctas) mine = a.cuts[threadIdx.x];
  // the cut units in the order of their ranges, the same in every block
  const uint32_t ballot = __ballot_sync(0xffffffffu, mine.parts > 0);
  if ((threadIdx.x & 31) == 0) warps[threadIdx.x >> 5] = __popc(ballot);
  __syncthreads();
  int found = 0, at = __popc(ballot & ((1u << (threadIdx.x & 31)) - 1));
  for (int w = 0; w < kJoinThreads / 32; ++w) {
    if (w < threadIdx.x >> 5) at += warps[w];
    found += warps[w];
  }
  if (mine.parts) used[at] = threadIdx.x;
  __syncthreads();
  const int groups = a.part_rows / 32, pieces = groups * (HD / kJoinCols);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, half = warp & 1, quarter = warp >> 1;
  const int pr = a.part_rows;
  for (int p = blockIdx.x; p < found * pieces; p += gridDim.x) {
    const Cut cut = a.cuts[used[p / pieces]];
    const int group = p % pieces % groups, col0 = p % pieces / groups * kJoinCols;
    const int in_tile = group * 32 + lane, row = cut.row_tile * kRows + in_tile;
    if (row - lane >= cut.count * a.rep) continue;
    // the first part may be the second record of its range, the others are the first of theirs
    auto slot = [&](int i) { return static_cast<int64_t>(i ? (cut.record & ~1) + 2 * i : cut.record); };
    float m = -INFINITY;
#pragma unroll 4
    for (int i = warp; i < cut.parts; i += 8) {
      const float x = a.stats[slot(i) * 2 * pr + in_tile];
      weight[i][lane] = x;
      m = fmaxf(m, x);
    }
    red[0][warp][lane] = m;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 8; ++w) m = fmaxf(m, red[0][w][lane]);
    const float shift = m == -INFINITY ? 0.f : m;
    float l = 0.f;
#pragma unroll 4
    for (int i = warp; i < cut.parts; i += 8) {
      const float w = exp2_fast(weight[i][lane] - shift);
      weight[i][lane] = w;
      l = fmaf(a.stats[slot(i) * 2 * pr + pr + in_tile], w, l);
    }
    red[1][warp][lane] = l;
    __syncthreads();
    l = 0.f;
#pragma unroll
    for (int w = 0; w < 8; ++w) l += red[1][w][lane];
    float o[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int i = quarter; i < cut.parts; i += 4) {
      const float w = weight[i][lane];
      const float* part = a.part + (slot(i) * HD + col0 + half * 8) * pr + in_tile;
#pragma unroll
      for (int j = 0; j < 8; ++j) o[j] = fmaf(part[j * pr], w, o[j]);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) acc[quarter][half * 8 + j][lane] = o[j];
    __syncthreads();
    const int node = row / a.rep;
    if (quarter == 0 && node < cut.count) {
      const int64_t to =
          ((static_cast<int64_t>(cut.b) * a.N + node) * a.hq + cut.head * a.rep + row % a.rep) * HD + col0 + half * 8;
      const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
      float f[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int k = half * 8 + j;
        f[j] = ((acc[0][k][lane] + acc[1][k][lane]) + (acc[2][k][lane] + acc[3][k][lane])) * inv;
      }
      if (a.gate) {
        float z[8];
        unpack8(ld_nc_v4(a.gate + to), z);
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] *= sigmoid_fast(z[j]);
      }
      uint32_t w[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) w[j] = pack_bf16x2(f[2 * j], f[2 * j + 1]);
      *reinterpret_cast<uint4*>(a.out + to) = make_uint4(w[0], w[1], w[2], w[3]);
    }
    __syncthreads();  // weight, red and acc are free again
  }
}

constexpr size_t kHeader = 256 + kMaxRanges * sizeof(Cut);
static_assert(kHeader % 256 == 0, "the partials begin aligned");

// One CTA per SM: each holds all of its SM's tensor memory.
int tree_ctas() { return sm_count() < kMaxRanges ? sm_count() : kMaxRanges; }

int part_rows(int N, int rep) {
  const int rows = (N * rep + 31) / 32 * 32;
  return rows < kRows ? rows : kRows;
}

template <int HD>
int launch(const TreeArgs& a, cudaStream_t st) {
  const size_t smem = 1024 + 2 * kStages * static_cast<size_t>(kTile) * HD * 2;
  const int rc = allow_smem(reinterpret_cast<const void*>(tree_attention_kernel<HD>), smem);
  if (rc) return rc;
  const int ctas = tree_ctas();
  cudaError_t e = launch_dependent(tree_attention_kernel<HD>, dim3(ctas), dim3(kThreads), smem, st, a);
  if (e != cudaSuccess) return cuda_error(e, "tree_attention_kernel");
  if (ctas > 1) {
    e = launch_dependent(tree_join_kernel<HD>, dim3(4 * ctas), dim3(kJoinThreads), 0, st, a, ctas);
    if (e != cudaSuccess) return cuda_error(e, "tree_join_kernel");
  }
  count_launch(2);
  return QK_OK;
}

}  // namespace
}  // namespace qk

using namespace qk;

extern "C" {

size_t qk_tree_attention_workspace_bytes(int B, int N, int hq, int kv_heads, int head_dim) {
  if (B <= 0 || N <= 0 || N > 64 || kv_heads <= 0 || hq <= 0 || hq % kv_heads || head_dim <= 0) return kHeader;
  return kHeader + 2 * static_cast<size_t>(tree_ctas()) * part_rows(N, hq / kv_heads) * (head_dim + 2) * sizeof(float);
}

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
  QK_REQUIRE(scale == scale && scale - scale == 0.f, "scale must be finite");
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
  QK_REQUIRE((reinterpret_cast<uintptr_t>(workspace) & 255) == 0, "workspace must be 256-byte aligned");
  TreeArgs a{};
  a.q = q;
  a.q_stride = q_stride;
  a.k_codes = k_codes;
  a.v_codes = v_codes;
  a.k_scale = k_scale;
  a.v_scale = v_scale;
  a.table = table;
  a.lengths = lengths;
  a.counts = counts;
  a.ancestors = ancestors;
  a.gate = gate;
  a.scale_log2 = scale == 0.f ? 1.f : fabsf(scale) * 1.44269504088896341f;
  a.q_keep = scale == 0.f ? 0u : ~0u;
  a.q_flip = scale < 0.f ? 0x80008000u : 0u;
  a.B = B;
  a.N = N;
  a.hq = hq;
  a.kv = kv_heads;
  a.rep = hq / kv_heads;
  a.pages = static_cast<int>(rows * T / page_size);
  a.pages_per_row = static_cast<int>(T / page_size);
  a.width = width;
  while ((1 << a.shift) < page_size) ++a.shift;
  a.part_rows = part_rows(N, a.rep);
  a.T = T;
  a.out = out;
  a.status = static_cast<int*>(workspace);
  a.cuts = reinterpret_cast<Cut*>(static_cast<uint8_t*>(workspace) + 256);
  a.part = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + kHeader);
  a.stats = a.part + 2 * static_cast<size_t>(tree_ctas()) * a.part_rows * head_dim;
  return head_dim == 256   ? launch<256>(a, as_stream(stream))
         : head_dim == 128 ? launch<128>(a, as_stream(stream))
                           : launch<64>(a, as_stream(stream));
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
  if (status) return set_error(status, "a block table entry lies outside the cache, or a length outside the table");
  return QK_OK;
}

}  // extern "C"
