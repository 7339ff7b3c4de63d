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
// range's end has several parts. Each part leaves O, maximum and sum in FP32, and a second kernel
// joins them, divides, gates and rounds.
//
// One CTA per SM, three kinds of warps joined by mbarriers (every wait bounded):
//  * 8 softmax warps, two threads per row: Q to TMEM once per unit; then per tile S from TMEM, mask,
//    running maximum and sum in FP32, P as FP16 back over S's columns. O (FP32, in TMEM) is rescaled
//    only when a row's maximum grows by more than 2^8: P, 2^7 at the maximum, stays below 2^15.
//  * 8 decode warps (4 for K, 4 for V): codes and scales from shared memory, where a copy warp each
//    brings them by tensor copies two tiles ahead; int8 -> FP16 with the group's scale (rounded once, to
//    11 bits where BF16 has 8; the join computes what does not fit FP16 again, from the cache), stored as
//    128-byte swizzled tiles: K-major for K, and the same bytes read as an MN-major operand for V.
//  * 2 warps issue the MMAs, Q K^T and P V: Q and P from TMEM, K and V from shared memory.
// TMEM: O 256 columns, Q 128, two S/P buffers of 64.
//
// Measured with 16 query and 2 KV heads of 256 (join included; the floor is the cache's bytes at the measured
// HBM rate, from 64 nodes on the products' flop at the measured BF16 rate):
//   32 requests, 8 nodes, 8192 tokens    52 us, floor 23 (154 MB: 3.0 TB/s)
//   16 requests, 64 nodes, 16384 tokens 137 us, floor 68 (112 GFLOP: 820 TFLOP/s; 159 us in a loop of seconds,
//                                       under the power cap)
//   1 request, 16 nodes, 32768 tokens    29 us, floor 5.5;  1 request, 1 node, 4096 tokens  18 us, floor 0.7
// What bounds it: at 64 nodes a tile's chain of barriers (copy, decode, S, softmax, P, O; the copies and
// barriers alone, nothing computed, took 106 us of 140) and the decode, which each of a KV head's four
// row tiles repeats; at few rows the fixed 9 to 14 thousand cycles before the first tile (cold
// instructions, four dependent reads to the first copy) and the 5 thousand of the last output and the join.
#include <cuda.h>  // CUtensorMap and its enums; the encoder is looked up at run time

#include "umma.cuh"

namespace qk {
namespace {

constexpr int kTile = 64;   // tokens per tile
constexpr int kRows = 128;  // query rows per tile
constexpr int kStages = 2;
constexpr int kRaw = 2;     // raw tiles (codes and scales) in flight
constexpr int kSoftmaxWarps = 8, kDecodeWarps = 8, kSide = kDecodeWarps / 2;  // half decode K, half V
constexpr int kScoreWarp = kSoftmaxWarps + kDecodeWarps, kCopyWarp = kScoreWarp + 1;  // K, then V; then the values' warp
constexpr int kThreads = (kSoftmaxWarps + kDecodeWarps + 4) * 32;                 // whole warpgroups
// Registers per thread: 96 at launch for 5 warpgroups (480 in all).
constexpr int kSoftmaxRegs = 128, kOtherRegs = 72;
static_assert(2 * kSoftmaxRegs + 3 * kOtherRegs <= 5 * 96, "the shares fit the launch's registers");
constexpr uint32_t kColO = 0, kColQ = 256, kColS = 384;  // TMEM columns
constexpr float kLazyGrowth = 8.f;                       // in powers of two
constexpr uint32_t kHugeScale = 0x7c00;                  // BF16 bits of 2^121: times 127 it leaves FP32's range
// Units whose records of bad values are alive at once. The value warps write tile n's when tile n - 3's product
// is done, so all softmax warps have left the unit of tile n - 4 and its record is cleared.
constexpr int kBadRing = 4;
// Queries and keys are multiplied by these for FP16: up to 2^22 and 2^20 fit it, and it leaves errors of
// 2^-19 and 2^-21 to small ones, a few 2^-16 of a score.
constexpr float kQueryPower = 1.f / 64, kKeyPower = 1.f / 16;
// Values are divided by a power of two that a part finds for each 32 channels from the prefix in its first tile:
// the largest scale there becomes 1 to 2. Scales up to 256 times as large still fit FP16 with their codes, those
// down to 2^-14 keep all 11 bits, smaller ones leave errors of 127 * 2^-25. Drafts are not asked, for one must not
// decide for the others: in a tile without prefix the values are divided by 2^-6, which takes those between 2^-13
// and 2^10. (To ask the prefix's end then instead took code that cost 4 us of 135 where it was not run.)
constexpr uint32_t kValueSpan = 64;  // of the exponents
constexpr float kOnlyDrafts = 1.f / 64;
constexpr float kDraftLimit = 512.f;  // a draft's scale by that power: 127 times this is no longer sure to fit
// Weights go out as 2^(score - m + kWeightRoom), 2^15 at most: FP16 then keeps weights down to 2^-31 of the largest.
constexpr float kWeightRoom = 7.f, kMostWeight = 32768.f;
// Values below 2^-9 of their power may have lost bits to FP16's range: their scales lie below 2^-14, where a half
// step is 2^-10 of them. They show as outputs smaller than that: an average over n tokens of equal weight is
// smaller by sqrt(n), and n is at least the sum of the weights by the largest that there can be.
constexpr float kSmall = 1.f / 512;
constexpr uint32_t kQStage = 2048;  // bytes per softmax warp
// What a unit costs besides its tiles (Q in, the output out), in tiles of the ranges, at 2 / 4 / 6 / 8: 16 requests of
// 64 nodes over 16384 tokens take 154 / 141 / 137 / 138 us, 32 of 8 nodes over 8192 60 / 54 / 53 / 53, with 32 / 8
// heads of 64 16 requests of 64 nodes over 8192 116 / 101 / 102 / 105, of 128 with 16 nodes 73 / 63 / 63 / 64.
constexpr int kUnitCost = 6;

// What calls on the device reported last, besides the word in their workspaces: a workspace can be gone, or belong
// to a graph, when somebody asks.
__device__ int g_tree_status;

struct TreeArgs {
  const uint16_t* q;
  int64_t q_stride;
  const int8_t *k_codes, *v_codes;
  const uint16_t *k_scale, *v_scale;
  const int32_t *table, *lengths, *counts;
  const uint64_t* ancestors;
  const uint16_t* gate;
  float scale_log2;         // |scale| * log2(e) / (kQueryPower * kKeyPower), above zero
  uint32_t q_keep, q_flip;  // Q's bits & keep ^ flip: nothing for a scale of zero, the sign for a negative one
  int B, N, hq, kv, rep, pages, pages_per_row, width, room, shift, row_tiles, part_rows, ctas;  // room: tokens of a table row
  int64_t T;
  uint16_t* out;
  int* status;
  float* part;          // [units + CTAs][HD][part_rows] unnormalised O
  float* stats;         // [units + CTAs][3][part_rows] maximum (log2) and two sums
  float* powers;        // [units + CTAs][HD / 32] what the part's values were divided by
  struct Parts* parts;  // [units]
};

// A unit's parts: the ranges first .. first + count - 1. The part of unit u in range c is record
// u + c, which no two parts share: units and ranges both go up along the work.
struct Parts {
  int first, count;
};

struct Request {
  int length, count, tiles, row_tiles;
  bool cut;
  // A unit's share of the ranges: its tiles and kUnitCost steps that stand for Q and the output.
  __device__ int steps() const { return tiles + kUnitCost; }
  __device__ int work(int kv) const { return tiles ? kv * row_tiles * steps() : 0; }
};

__device__ __forceinline__ Request load_request(const TreeArgs& a, int b) {
  const int n = a.lengths[b], c = a.counts ? a.counts[b] : a.N;
  Request r;
  r.length = min(max(n, 0), a.room);
  r.count = min(min(max(c, 0), a.N), a.room - r.length);
  r.cut = r.length != n || r.count != c;
  r.row_tiles = (r.count * a.rep + kRows - 1) / kRows;
  r.tiles = r.count ? (r.length + r.count + kTile - 1) / kTile : 0;
  return r;
}

__device__ __forceinline__ void report(const TreeArgs& a, int status) {
  *a.status = status;
  atomicExch(&g_tree_status, status);
}

// The CTAs' ranges of a total of `total` steps: n of them, the first total % n one step longer. All
// counts of steps fit 31 bits (the host checks): 64-bit divisions alone cost as much as two tiles.
struct Ranges {
  int n, each, longer;
  __device__ Ranges(int total, int ctas)
      : n(min(total, ctas)), each(n ? total / n : 0), longer(n ? total - each * n : 0) {}
  __device__ int start(int c) const { return c * each + min(c, longer); }
  __device__ int owner(int step) const {
    const int head = longer * (each + 1);
    return step < head ? step / (each + 1) : longer + (step - head) / each;
  }
};

// The pieces of a CTA's range: tiles [t0, t1) of one unit each. A unit's last steps are not tiles:
// a range that holds nothing else of the unit has no piece of it.
struct Segment {
  Request r;
  int b, head, row_tile, t0, t1, index;
  int start;  // the unit's first step in the whole work
};
struct Walk {
  Request r;
  int b, index;
  int offset, left, at;  // in request b's work; of the range; the next step in the whole work
  __device__ bool next(const TreeArgs& a, Segment& s) {
    while (left > 0) {
      for (int w = r.work(a.kv); offset >= w; w = r.work(a.kv)) {
        offset -= w;
        r = load_request(a, ++b);
      }
      const int steps = r.steps(), unit = offset / steps;
      s.r = r;
      s.b = b;
      s.head = unit / r.row_tiles;
      s.row_tile = unit - s.head * r.row_tiles;
      s.t0 = offset - unit * steps;
      const int end = min(steps, s.t0 + left), did = end - s.t0;
      s.start = at - s.t0;
      left -= did;
      offset += did;
      at += did;
      s.t1 = min(end, r.tiles);
      if (s.t0 >= s.t1) continue;
      s.index = index++;
      return true;
    }
    return false;
  }
};

// A piece's unit among all, present or not.
__device__ __forceinline__ int unit_of(const TreeArgs& a, const Segment& s) {
  return (s.b * a.kv + s.head) * a.row_tiles + s.row_tile;
}

// The whole work and where range `me` of it begins; every warp finds out for itself (a lane per
// request, no barrier).
__device__ __forceinline__ Walk locate(const TreeArgs& a, int me, int& total, bool tell) {
  const int lane = threadIdx.x & 31;
  total = 0;
  for (int b0 = 0; b0 < a.B; b0 += 32) {
    int w = 0;
    if (b0 + lane < a.B) {
      const Request r = load_request(a, b0 + lane);
      w = r.work(a.kv);
      if (r.cut && tell) report(a, QK_ERR_INVALID_ARGUMENT);
    }
    total += __reduce_add_sync(0xffffffffu, w);
  }
  const Ranges ranges(total, gridDim.x);
  Walk walk{};
  if (me >= ranges.n) return walk;
  walk.at = ranges.start(me);
  walk.left = ranges.start(me + 1) - walk.at;
  int before = 0;
  for (int b0 = 0; b0 < a.B; b0 += 32) {
    const int w = b0 + lane < a.B ? load_request(a, b0 + lane).work(a.kv) : 0;
    int upto = before + w;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, upto - before, o);
      if (lane >= o) upto += u;
    }
    const uint32_t past = __ballot_sync(0xffffffffu, upto > walk.at);
    if (past) {
      const int which = __ffs(past) - 1;
      walk.b = b0 + which;
      walk.offset = walk.at - __shfl_sync(0xffffffffu, upto - w, which);
      break;
    }
    before = __shfl_sync(0xffffffffu, upto, 31);
  }
  walk.r = load_request(a, walk.b);
  return walk;
}

struct Barriers {
  uint64_t k_full[kStages], k_empty[kStages], v_full[kStages], v_empty[kStages];
  uint64_t s_full[kStages], p_full[kStages], q_full, o_full;
  uint64_t swapped[4], bad_read;  // a row's two warps have left their maxima; a unit's record of bad values is read
  uint64_t raw_full[2][kRaw], raw_empty[2][kRaw];  // K, V
};

struct Control {
  Barriers bar;
  float top[2][2][kRows];     // by tile parity: the row maxima that a row's two warps swap
  uint64_t bad[kBadRing][8];  // per unit and channel group: drafts whose values do not fit FP16 there
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

// Pairs of FP32 in one instruction, and a three-way maximum.
__device__ __forceinline__ uint64_t pair(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void unpair(uint64_t p, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(p));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

__device__ __forceinline__ void sts_v4(uint32_t addr, const uint4& v) {
  asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(addr), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}

__device__ __forceinline__ uint4 lds_v4_at(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ uint32_t lds_at(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}

// Four int8 codes times an FP16 scale -> two FP16 pairs, each code * scale rounded once. With the sign
// bit flipped a code c is the byte c + 128, under the exponent of 1024 it reads 1152 + c; minus 1152 it
// is the code, exactly. Three and a half instructions per pair, of which one and a half on the integer
// pipe, which is half as wide: with a sign extension there (and one fused multiply-add) it was slower.
__device__ __forceinline__ void decode4(uint32_t codes, __half2 scale, uint32_t& lo, uint32_t& hi) {
  const uint32_t u = codes ^ 0x80808080u;
  const uint32_t t[2] = {__byte_perm(u, 0x64646464u, 0x4140), __byte_perm(u, 0x64646464u, 0x4342)};
  uint32_t r[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const __half2 v = __hmul2(__hadd2(*reinterpret_cast<const __half2*>(&t[i]), __half2{-1152.f, -1152.f}), scale);
    r[i] = *reinterpret_cast<const uint32_t*>(&v);
  }
  lo = r[0];
  hi = r[1];
}

__device__ __forceinline__ uint32_t pack_f16x2(float a, float b) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
  return r;
}

// A power of two by its exponent, biased as FP32 has it, and the inverse of one.
__device__ __forceinline__ float power_of(uint32_t biased) { return __uint_as_float(biased << 23); }
__device__ __forceinline__ float inverse_power(float power) {
  return __uint_as_float((254u - (__float_as_uint(power) >> 23)) << 23);
}

// A bounded wait of a whole warp, converged behind it: false for all lanes if one gave up.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity) {
  return __all_sync(0xffffffffu, mbar_wait_bounded(bar, parity));
}

// ---- decode warps -------------------------------------------------------------------------

// A raw tile as the copies leave it: K codes, V codes [token][HD], then per box of a page's tokens
// the K scales and the V scales [group][token].
template <int HD>
struct Raw {
  static constexpr uint32_t kCodes = kTile * HD, kGroups = HD / 32;
  static constexpr uint32_t kScales = kTile / 16 * 128 > kTile * kGroups * 2 ? kTile / 16 * 128 : kTile * kGroups * 2;
  static constexpr uint32_t kBytes = 2 * (kCodes + kScales);
  // bytes from one box's scales to the next's: copies land on 128-byte boundaries
  static __device__ uint32_t box_stride(uint32_t box) { return box * kGroups * 2 < 128 ? 128 : box * kGroups * 2; }
};

struct Maps {
  CUtensorMap k_codes, v_codes, k_scale, v_scale;
};

__device__ __forceinline__ void tma_load_2d(uint32_t dst, const CUtensorMap* map, int x, int y, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(smem_addr(bar))
      : "memory");
}

// A copy warp for K and one for V: per tile a box of min(page, 64) tokens per lane, two tensor copies
// each (codes and scales), kRaw tiles ahead; page numbers one tile further. One warp for both was the
// slowest of all: a tile's worth of its instructions took as long as two tiles of the others'.
template <int HD>
__device__ __forceinline__ bool copy_role(const TreeArgs& a, Control& ctl, const Maps& maps, uint32_t raw, int v,
                                          Walk walk) {
  const int lane = threadIdx.x & 31;
  const int box = min(1 << a.shift, kTile), boxes = kTile / box, mine = lane * box;
  const uint32_t codes = raw + v * Raw<HD>::kCodes + mine * HD;
  const uint32_t scales = raw + 2 * Raw<HD>::kCodes + v * Raw<HD>::kScales + lane * Raw<HD>::box_stride(box);
  const CUtensorMap* code_map = v ? &maps.v_codes : &maps.k_codes;
  const CUtensorMap* scale_map = v ? &maps.v_scale : &maps.k_scale;
  uint64_t *full = ctl.bar.raw_full[v], *empty = ctl.bar.raw_empty[v];
  Segment seg;
  uint32_t it = 0;
  bool ok = true;
  while (ok && walk.next(a, seg)) {
    const int total = seg.r.length + seg.r.count;
    const int32_t* table = a.table + static_cast<int64_t>(seg.b) * a.width;
    auto page_of = [&](int tile) {
      const int token = tile * kTile + mine;
      return tile < seg.t1 && lane < boxes && token < total ? __ldg(table + (token >> a.shift)) : 0;
    };
    int page = page_of(seg.t0);
    for (int tile = seg.t0; tile < seg.t1; ++tile, ++it) {
      const uint32_t slot = it % kRaw;
      if (static_cast<uint32_t>(page) >= static_cast<uint32_t>(a.pages)) {  // reported, and read as page 0
        report(a, QK_ERR_INVALID_ARGUMENT);
        page = 0;
      }
      const int y = (page << a.shift) + ((tile * kTile + mine) & ((1 << a.shift) - 1));  // the slot
      int x = y, plane = seg.head * (HD / 32);
      if (a.pages != a.pages_per_row) {  // a cache of several rows: the slot's row and time
        const int row = page / a.pages_per_row;
        x -= (row * a.pages_per_row) << a.shift;
        plane += row * a.kv * (HD / 32);
      }
      const int live = min((total - tile * kTile + box - 1) / box, boxes);
      ok = warp_wait(&empty[slot], ((it / kRaw) & 1) ^ 1);
      if (!ok) break;
      if (lane == 0) mbar_expect_tx(&full[slot], live * box * (HD + 2 * (HD / 32)));
      __syncwarp();
      if (lane < live) {
        tma_load_2d(codes + slot * Raw<HD>::kBytes, code_map, seg.head * HD, y, &full[slot]);
        tma_load_2d(scales + slot * Raw<HD>::kBytes, scale_map, x, plane, &full[slot]);
      }
      page = page_of(tile + 1);
    }
  }
  // every copy issued must have landed before the CTA leaves (bounded, should a reader have given up)
  for (uint32_t i = it > kRaw ? it - kRaw : 0; i < it; ++i) warp_wait(&full[i % kRaw], (i / kRaw) & 1);
  return ok;
}

// For the power of two of a part's values: the largest scale, in 32 channels, of the prefix tokens in its first tile,
// of which `scales` is the first.
__device__ __forceinline__ uint32_t top_scale(uint32_t scales, int box, uint32_t box_stride, int known) {
  uint32_t top = 0;
  const int box_shift = 31 - __clz(box);
#pragma unroll 1
  for (int t = 0; t < known; t += 8) {
    const uint4 u = lds_v4_at(scales + (t >> box_shift) * box_stride + (t & (box - 1)) * 2);
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const int left = known - t - 2 * w;
      top = __vmaxu2(top, left > 1 ? word(u, w) & 0x7fff7fffu : left > 0 ? word(u, w) & 0x7fffu : 0u);
    }
  }
  return max(top & 0xffffu, top >> 16);
}

// 4 decode warps for K and 4 for V, all in one copy of this code: with a copy each the CTA's hot code
// left the instruction cache. FP16 has the bits but not the range of the cache's BF16 scales. Keys (and
// queries) go in with a fixed power of two: what matters of them is a score's absolute error. Values
// count relatively, so a part has a power of its own per 32 channels, by which the join multiplies.
template <int HD>
__device__ __forceinline__ bool decode_role(const TreeArgs& a, Control& ctl, uint32_t tiles, uint32_t raw, Walk walk) {
  constexpr int SPT = HD / 32, CHUNKS = HD / 16;  // a thread's share of a tile: 16 channels of SPT tokens
  constexpr uint32_t kStageBytes = kTile * HD * 2;
  const bool values = threadIdx.x >= (kSoftmaxWarps + kSide) * 32;
  const int t = threadIdx.x & (kSide * 32 - 1), lane = threadIdx.x & 31;
  const int chunk = t % CHUNKS, sub = (t / CHUNKS) * SPT;
  // A token's 16 channels are the 16-byte pieces 2 chunk and 2 chunk + 1 of its row, in atoms of 64
  // channels, piece j at j ^ (token % 8). Half of the lanes take their tokens in the order 1, 0, 3,
  // 2, ..: then 8 lanes' stores fill the 8 different 16-byte banks.
  const int swap = HD == 64 ? (t / CHUNKS) & 1 : (chunk >> 2) & 1;
  uint64_t* full = (values ? ctl.bar.v_full : ctl.bar.k_full);
  uint64_t* empty = (values ? ctl.bar.v_empty : ctl.bar.k_empty);
  uint64_t *raw_full = ctl.bar.raw_full[values], *raw_empty = ctl.bar.raw_empty[values];
  const uint32_t to0 = tiles + (values ? kStages : 0) * kStageBytes + (chunk >> 2) * (kTile * 128) +
                       ((sub ^ swap) << 7 | (((chunk & 3) * 2) ^ ((sub ^ swap) & 7)) << 4);
  const uint32_t select[2] = {swap ? 0x3232u : 0x1010u, swap ? 0x1010u : 0x3232u};
  const uint32_t from = raw + (values ? Raw<HD>::kCodes : 0) + sub * HD + chunk * 16;
  const uint32_t from_even = from + swap * HD, from_odd = from - swap * HD;
  const int box = min(1 << a.shift, kTile);
  const uint32_t scales_at = raw + 2 * Raw<HD>::kCodes + (values ? Raw<HD>::kScales : 0) +
                             sub / box * Raw<HD>::box_stride(box) + (chunk / 2 * box + (sub & (box - 1))) * 2;
  const uint32_t group_scales = raw + 2 * Raw<HD>::kCodes + Raw<HD>::kScales + chunk / 2 * box * 2;
  float inverse = kKeyPower;
  Segment seg;
  uint32_t it = 0;
  while (walk.next(a, seg)) {
    if (values) {  // outside the loop over tiles, whose code has to stay in the instruction cache
      if (!warp_wait(&raw_full[it & 1], it >> 1 & 1)) return false;
      const int known = seg.r.length - seg.t0 * kTile;
      const uint32_t top = top_scale(group_scales + (it & 1) * Raw<HD>::kBytes, box, Raw<HD>::box_stride(box), min(known, kTile));
      const float power = top ? power_of(min(max(top >> 7, 127u - kValueSpan), 127u + kValueSpan)) : kOnlyDrafts;
      inverse = inverse_power(power);
      if (t < CHUNKS && !(chunk & 1))
        a.powers[static_cast<int64_t>(unit_of(a, seg) + static_cast<int>(blockIdx.x)) * (HD / 32) + chunk / 2] = power;
    }
#pragma unroll 1
    for (int tile = seg.t0; tile < seg.t1; ++tile, ++it) {
      const uint32_t stage = it & 1, phase = it >> 1 & 1, slot = stage * Raw<HD>::kBytes;
      if (!warp_wait(&raw_full[stage], phase)) return false;
      uint32_t scales[SPT / 2];
#pragma unroll
      for (int i = 0; i < SPT / 2; ++i) scales[i] = lds_at(scales_at + slot + 4 * i);
      uint4 code[SPT];
#pragma unroll
      for (int i = 0; i < SPT; ++i) code[i] = lds_v4_at((i & 1 ? from_odd : from_even) + slot + i * HD);
      if (tile * kTile + kTile > seg.r.length) {  // drafts, or past the end
        const int total = seg.r.length + seg.r.count;
#pragma unroll
        for (int i = 0; i < SPT; ++i) {
          const int token = tile * kTile + sub + i;
          const uint32_t mask = i & 1 ? 0xffff0000u : 0xffffu;
          const uint32_t bits = scales[i / 2] >> (16 * (i & 1)) & 0x7fffu;
          if (token >= total) {
            scales[i / 2] &= ~mask;
          } else if (token < seg.r.length) {
            // a prefix value past FP16's range is infinite in the products, which the join finds
          } else if (!values) {
            // the scores of a draft's key that is not finite are NaN, which the mask keeps from rows that do not see it
            if (bits >= kHugeScale) scales[i / 2] |= mask & 0x7fff7fffu;
          } else if (!(__uint_as_float(bits << 16) * inverse < kDraftLimit)) {
            // a draft's value that does not fit must not reach the rows that do not see it as 0 * inf: zero here,
            // and NaN for the rows that do
            atomicOr(reinterpret_cast<unsigned long long*>(&ctl.bad[seg.index % kBadRing][chunk / 2]),
                     1ull << (token - seg.r.length));
            scales[i / 2] &= ~mask;
          }
        }
      }
#pragma unroll
      for (int i = 0; i < SPT / 2; ++i)
        scales[i] = pack_f16x2(__uint_as_float(scales[i] << 16) * inverse, __uint_as_float(scales[i] & 0xffff0000u) * inverse);
      if (!warp_wait(&empty[stage], phase ^ 1)) return false;
#pragma unroll
      for (int i = 0; i < SPT; ++i) {
        const uint32_t two = __byte_perm(scales[i / 2], 0, select[i & 1]);
        const __half2 h = *reinterpret_cast<const __half2*>(&two);
        uint4 piece[2];
        decode4(code[i].x, h, piece[0].x, piece[0].y);
        decode4(code[i].y, h, piece[0].z, piece[0].w);
        decode4(code[i].z, h, piece[1].x, piece[1].y);
        decode4(code[i].w, h, piece[1].z, piece[1].w);
        const uint32_t to = (to0 + stage * kStageBytes) ^ (i << 7 | i << 4);
        sts_v4(to, piece[0]);
        sts_v4(to ^ 16, piece[1]);
      }
      fence_proxy_async_smem();
      __syncwarp();
      // The raw slot goes back only here, where the stores above have used every code. An arrival right behind
      // the loads does not hold them: the compiler may let them sink below it and the wait for the stage, and
      // where that wait was long (a unit's first tiles) a warp decoded the tile that had come into the slot
      // meanwhile: in a pass of four over 16 trees of 64 nodes. It costs no time (139.5 us, loads that are volatile
      // instead 143.7).
      if (lane == 0) {
        mbar_arrive(&full[stage]);
        mbar_arrive(&raw_empty[stage]);
      }
    }
  }
  return true;
}

// ---- MMA warp -----------------------------------------------------------------------------

// One lane of the (converged) warp, the same each time. The whole warp runs the role and only the
// instructions themselves are one lane's: their operands are then known to be uniform; issued from
// a lane's own branch each took about 80 cycles.
__device__ __forceinline__ bool elect_one() {
  uint32_t one;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(one));
  return one != 0;
}

// One warp issues the score products, another the value products: the tensor core takes an
// instruction only shortly before it can run it, so a single issuer stands idle in all its waits.
template <int HD>
__device__ __forceinline__ bool score_role(const TreeArgs& a, Control& ctl, uint32_t ktiles, Walk walk) {
  constexpr uint32_t kStageBytes = kTile * HD * 2;
  const uint32_t tm = __shfl_sync(0xffffffffu, ctl.tmem, 0);
  const uint32_t idesc = idesc_f16_m128(kTile);
  const uint64_t kdesc = sdesc_sw128(ktiles, 1024u);
  Segment seg;
  uint32_t it = 0;
  while (walk.next(a, seg)) {
    if (!warp_wait(&ctl.bar.q_full, seg.index & 1)) return false;
    for (int tile = seg.t0; tile < seg.t1; ++tile, ++it) {
      const uint32_t stage = it % kStages, phase = (it / kStages) & 1;
      if (!warp_wait(&ctl.bar.k_full[stage], phase)) return false;
      // the weights of the tile before last lie where these scores go: until its product is done
      if (!warp_wait(&ctl.bar.v_empty[stage], phase ^ 1)) return false;
      tc_fence_after();
      if (elect_one()) {
        const uint64_t desc = kdesc + stage * (kStageBytes >> 4);
        const uint32_t d = tm + kColS + stage * kTile;
#pragma unroll
        for (int k = 0; k < HD / 16; ++k)
          umma_ts(d, tm + kColQ + k * 8, desc + ((k / 4) * (kTile * 128) + (k % 4) * 32 >> 4), idesc, k != 0);
        umma_commit(&ctl.bar.k_empty[stage]);
        umma_commit(&ctl.bar.s_full[stage]);
      }
      __syncwarp();
    }
  }
  return true;
}

template <int HD>
__device__ __forceinline__ bool value_role(const TreeArgs& a, Control& ctl, uint32_t vtiles, Walk walk) {
  constexpr uint32_t kStageBytes = kTile * HD * 2;
  const uint32_t tm = __shfl_sync(0xffffffffu, ctl.tmem, 0);
  const uint32_t idesc = idesc_f16_m128_bmn(HD);
  const uint64_t vdesc = sdesc_sw128_mn(vtiles, kTile * 128, 1024u);
  Segment seg;
  uint32_t it = 0;
  while (walk.next(a, seg)) {
    for (int tile = seg.t0; tile < seg.t1; ++tile, ++it) {
      const uint32_t stage = it % kStages, phase = (it / kStages) & 1;
      if (!warp_wait(&ctl.bar.v_full[stage], phase)) return false;
      if (!warp_wait(&ctl.bar.p_full[stage], phase)) return false;
      tc_fence_after();
      if (elect_one()) {
        const uint64_t desc = vdesc + stage * (kStageBytes >> 4);
        const uint32_t p = tm + kColS + stage * kTile;
#pragma unroll
        for (int k = 0; k < kTile / 16; ++k)
          umma_ts(tm + kColO, p + k * 8, desc + k * (2048 >> 4), idesc, tile != seg.t0 || k != 0);
        umma_commit(&ctl.bar.v_empty[stage]);
        if (tile + 1 == seg.t1) umma_commit(&ctl.bar.o_full);
      }
      __syncwarp();
    }
  }
  return true;
}

// ---- softmax warps ------------------------------------------------------------------------

// Q of a unit to TMEM. Rows pass through 2 KB of shared memory per warp (32 rows x 64 B, row r's
// 16-byte piece j at j ^ (r / 2 % 4)): a thread owns a row in TMEM, but 4 threads read 64 B of a row
// from global memory, which takes a quarter of the cache-line lookups of a thread per row.
// The two warps of a row take half of the channels each.
template <int HD>
__device__ __forceinline__ void load_q(const TreeArgs& a, const Segment& seg, uint32_t tm, uint32_t stage) {
  const int quarter = threadIdx.x >> 5 & 3, half = threadIdx.x >> 7, lane = threadIdx.x & 31;
  const int row = seg.row_tile * kRows + quarter * 32 + lane, node = row / a.rep;
  const uint16_t* q = a.q + static_cast<int64_t>(seg.b) * a.N * a.q_stride + static_cast<int64_t>(seg.head) * a.rep * HD +
                      half * (HD / 2);
  const int mine = node < seg.r.count ? node * static_cast<int>(a.q_stride) + (row - node * a.rep) * HD : -1;
  int at[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) at[i] = __shfl_sync(0xffffffffu, mine, 8 * i + lane / 4);
  constexpr int kAtOnce = HD >= 128 ? 2 : 1;  // pieces of 32 channels in flight
#pragma unroll
  for (int c0 = 0; c0 < HD / 64; c0 += kAtOnce) {
    uint4 v[kAtOnce][4];
#pragma unroll
    for (int c = 0; c < kAtOnce; ++c)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        v[c][i] = at[i] >= 0 ? ld_guarded_v4(q + at[i] + (c0 + c) * 32 + lane % 4 * 8) : make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int c = 0; c < kAtOnce; ++c) {
      __syncwarp();
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = 8 * i + lane / 4;
        sts_v4(stage + r * 64 + ((lane ^ r / 2) & 3) * 16, v[c][i]);
      }
      __syncwarp();
      uint32_t u[16];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint4 x = lds_v4_at(stage + lane * 64 + ((i ^ lane / 2) & 3) * 16);
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const uint32_t y = (word(x, w) & a.q_keep) ^ a.q_flip;
          u[i * 4 + w] = pack_f16x2(__uint_as_float(y << 16) * kQueryPower, __uint_as_float(y & 0xffff0000u) * kQueryPower);
        }
      }
      tmem_st16(tm + kColQ + half * (HD / 4) + (c0 + c) * 16, u);
    }
  }
  tmem_wait_st();
}

// Two warps per 32 rows, each with half of a tile's tokens: with one, its scores-to-weights chain was
// the longest of all. They swap their rows' maxima through shared memory, decide alike, and keep a
// sum each; O's rescaling and Q and O themselves are shared by channels.
template <int HD>
__device__ __forceinline__ bool softmax_role(const TreeArgs& a, Control& ctl, uint32_t stage, Walk walk, int total) {
  constexpr int kHalf = kTile / 2;
  const int warp = threadIdx.x >> 5, quarter = warp & 3, half = warp >> 2, lane = threadIdx.x & 31;
  const uint32_t tm = ctl.tmem + (static_cast<uint32_t>(quarter * 32) << 16);
  const uint32_t o_cols = tm + kColO + half * (HD / 2);
  Segment seg, next;
  uint32_t it = 0, swaps = 0, reads = 0;
  bool more = walk.next(a, next);
  auto busy_of = [&](const Segment& s) { return s.row_tile * kRows + quarter * 32 < s.r.count * a.rep; };
  auto give_q = [&](const Segment& s) {
    if (busy_of(s)) load_q<HD>(a, s, tm, stage);
    tc_fence_before();
    __syncwarp();
    if (lane == 0) mbar_arrive(&ctl.bar.q_full);
  };
  if (more) give_q(next);
  while (more) {
    seg = next;
    const int node = (seg.row_tile * kRows + quarter * 32 + lane) / a.rep;
    const bool live = node < seg.r.count;
    const bool busy = busy_of(seg);  // the same for the warp
    uint64_t path = 0;
    if (live) {
      path = a.ancestors[static_cast<int64_t>(seg.b) * a.N + node];
      if (seg.r.count < 64) path &= (1ull << seg.r.count) - 1;
    }
    float m = -INFINITY, l = 0.f;
    for (int tile = seg.t0; tile < seg.t1; ++tile, ++it) {
      if (!warp_wait(&ctl.bar.s_full[it & 1], (it / 2) & 1)) return false;
      tc_fence_after();  // also where no row is busy: the next unit's Q goes where these products read theirs
      if (busy) {
        uint32_t s[kHalf];
        const uint32_t cols = tm + kColS + (it & 1) * kTile;
        tmem_ld32(cols + half * kHalf, s);
        tmem_wait_ld(s);
        const int first = tile * kTile + half * kHalf;
        if (first + kHalf > seg.r.length) {  // drafts, or past the end: the row's 32 bits
          const int cut = seg.r.length - first;
          uint32_t see = 0;
          if (cut > 0) see = static_cast<uint32_t>(path << cut) | ((1u << cut) - 1);
          else if (cut > -64) see = static_cast<uint32_t>(path >> -cut);
          if (!live) see = 0;
#pragma unroll
          for (int j = 0; j < kHalf; ++j)
            if (!(see >> j & 1)) s[j] = 0xff800000u;
        }
        float most = -INFINITY, most2 = -INFINITY;
#pragma unroll
        for (int j = 0; j < kHalf; j += 4) {
          most = max3(most, __uint_as_float(s[j]), __uint_as_float(s[j + 1]));
          most2 = max3(most2, __uint_as_float(s[j + 2]), __uint_as_float(s[j + 3]));
        }
        float top = fmaxf(most, most2) * a.scale_log2;
        float(*tops)[kRows] = ctl.top[it & 1];
        tops[half][quarter * 32 + lane] = top;
        // the pair's scores are both read by then: P may go over either's columns
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&ctl.bar.swapped[quarter]);
        if (!warp_wait(&ctl.bar.swapped[quarter], swaps++ & 1)) return false;
        tc_fence_after();
        top = fmaxf(top, tops[half ^ 1][quarter * 32 + lane]);
        const bool grow = top > m + kLazyGrowth;
        if (__any_sync(0xffffffffu, grow)) {
          const float now = fmaxf(m, top);
          const float keep = m == -INFINITY ? 0.f : exp2_fast(m - now);
          m = now;
          l *= keep;
          if (tile > seg.t0) {
            // every product so far has left O: the commit of the tile before
            const uint32_t last = it - 1;
            if (!warp_wait(&ctl.bar.v_empty[last % kStages], (last / kStages) & 1)) return false;
            tc_fence_after();
#pragma unroll 1
            for (int c = 0; c < HD / 64; ++c) {
              uint32_t o[32];
              tmem_ld32(o_cols + c * 32, o);
              tmem_wait_ld(o);
#pragma unroll
              for (int j = 0; j < 32; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * keep);
              tmem_st32(o_cols + c * 32, o);
            }
          }
        }
        const float shift = (m == -INFINITY ? 0.f : m) - kWeightRoom;
        uint32_t p[kHalf / 2];
        const uint64_t mul2 = pair(a.scale_log2, a.scale_log2), add2m = pair(-shift, -shift);
        uint64_t sum[2] = {0, 0};
#pragma unroll
        for (int j = 0; j < kHalf / 2; ++j) {
          float x, y;
          unpair(fma2(pair(__uint_as_float(s[2 * j]), __uint_as_float(s[2 * j + 1])), mul2, add2m), x, y);
          x = exp2_fast(x);
          y = exp2_fast(y);
          sum[j & 1] = add2(sum[j & 1], pair(x, y));
          p[j] = pack_f16x2(x, y);
        }
        float even, odd;
        unpair(add2(sum[0], sum[1]), even, odd);
        l += even + odd;
        tmem_st16(cols + half * (kHalf / 2), p);
        tmem_wait_st();
        tc_fence_before();
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&ctl.bar.p_full[it & 1]);
    }
    // every product with this Q is done: the next unit's Q goes in and its first scores are on their
    // way while this unit's O leaves
    more = walk.next(a, next);
    if (more) give_q(next);
    if (!warp_wait(&ctl.bar.o_full, seg.index & 1)) return false;
    if (busy) {
      tc_fence_after();
      // The unit's part of O as it is, FP32, channel by channel (32 rows are 128 B): the join divides,
      // gates and rounds. A quarter of the instructions of doing that here, where nothing hides them.
      const uint64_t* bad = ctl.bad[seg.index % kBadRing] + half * (HD / 64);
      const int unit = unit_of(a, seg);
      const int64_t record = static_cast<int64_t>(unit) + blockIdx.x;
      float* part = a.part + (record * HD + half * (HD / 2)) * a.part_rows + quarter * 32 + lane;
  #pragma unroll 1
      for (int c = 0; c < HD / 64; ++c) {
        uint32_t o[32];
        tmem_ld32(o_cols + c * 32, o);
        tmem_wait_ld(o);
        if (bad[c] & path) {
  #pragma unroll
          for (int j = 0; j < 32; ++j) o[j] = 0x7fc00000u;
        }
  #pragma unroll
        for (int j = 0; j < 32; ++j) part[(c * 32 + j) * a.part_rows] = __uint_as_float(o[j]);
        __syncwarp();
      }
      float* stats = a.stats + record * 3 * a.part_rows + quarter * 32 + lane;
      if (half == 0) stats[0] = m;
      stats[(1 + half) * a.part_rows] = l;
      if (seg.t0 == 0 && threadIdx.x == 0)
        a.parts[unit] = Parts{static_cast<int>(blockIdx.x),
                              Ranges(total, gridDim.x).owner(seg.start + seg.r.tiles - 1) - static_cast<int>(blockIdx.x) + 1};
      tc_fence_before();
    }
    if (seg.r.length < seg.t1 * kTile) {  // the unit saw drafts: when all have read its bad values, clear them
      __syncwarp();
      if (lane == 0) mbar_arrive(&ctl.bar.bad_read);
      if (warp == 0) {
        if (!warp_wait(&ctl.bar.bad_read, reads++ & 1)) return false;
        if (lane < 8) ctl.bad[seg.index % kBadRing][lane] = 0;
      }
    }
  }
  return true;
}

template <int HD>
__global__ void __launch_bounds__(kThreads, 1) tree_attention_kernel(const __grid_constant__ Maps maps, TreeArgs a) {
  extern __shared__ uint8_t smem_raw[];
  __shared__ Control ctl;
  uint8_t* tiles = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  constexpr uint32_t kStageBytes = kTile * HD * 2;
  const int warp = threadIdx.x >> 5;
  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&ctl.bar.k_full[i], kSide);
      mbar_init(&ctl.bar.k_empty[i], 1);
      mbar_init(&ctl.bar.v_full[i], kSide);
      mbar_init(&ctl.bar.v_empty[i], 1);
    }
    for (int i = 0; i < kRaw; ++i) {
      for (int v = 0; v < 2; ++v) {
        mbar_init(&ctl.bar.raw_full[v][i], 1);
        mbar_init(&ctl.bar.raw_empty[v][i], kSide);
      }
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&ctl.bar.s_full[i], 1);
      mbar_init(&ctl.bar.p_full[i], kSoftmaxWarps);
    }
    mbar_init(&ctl.bar.q_full, kSoftmaxWarps);
    mbar_init(&ctl.bar.o_full, 1);
    mbar_init(&ctl.bar.bad_read, kSoftmaxWarps);
    for (int i = 0; i < 4; ++i) mbar_init(&ctl.bar.swapped[i], 2);
    fence_mbar_init();
  }
  if (threadIdx.x < kBadRing * 8) ctl.bad[threadIdx.x / 8][threadIdx.x % 8] = 0;
  // All of the SM's tensor memory, asked for before earlier kernels end: this CTA's 61,440 registers leave
  // room for no other that could be waiting for some at the same time.
  if (warp == kScoreWarp) tmem_alloc(&ctl.tmem, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  pdl_wait();
  pdl_trigger();
  int total;
  const Walk walk = locate(a, blockIdx.x, total, threadIdx.x < 32 && blockIdx.x == 0);

  const uint32_t ktiles = smem_addr(tiles), vtiles = ktiles + kStages * kStageBytes, raw = vtiles + kStages * kStageBytes;
  const uint32_t rows = raw + kRaw * Raw<HD>::kBytes;
  bool ok = true;
  if (warp < kSoftmaxWarps) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
    ok = softmax_role<HD>(a, ctl, rows + warp * kQStage, walk, total);
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
    if (warp < kScoreWarp) ok = decode_role<HD>(a, ctl, ktiles, raw, walk);
    else if (warp == kCopyWarp || warp == kCopyWarp + 1) ok = copy_role<HD>(a, ctl, maps, raw, warp - kCopyWarp, walk);
    else if (warp == kScoreWarp) ok = score_role<HD>(a, ctl, ktiles, walk);
    else ok = value_role<HD>(a, ctl, vtiles, walk);
  }
  if (!ok) report(a, QK_ERR_TIMEOUT);
  tc_fence_before();
  __syncthreads();
  if (warp == kScoreWarp) {
    tc_fence_after();
    tmem_dealloc(ctl.tmem, 512);
  }
}

// ---- joining a unit's parts ------------------------------------------------------------------

// Every row of the output, also those of nodes that are not there, in pieces of 32 rows (a lane
// each) x 16 channels. WARPS warps share a piece: 1 where there are enough pieces to fill the GPU, 8
// where few units have many parts (a unit can have as many as there are ranges): each takes every
// WARPS-th part, and shared memory adds them in a fixed order. Bound by latency: two rounds of loads,
// what the piece is and then its parts, so everything that can is asked for in the first.
constexpr int kJoinWarps = 8, kJoinCols = 16;

// Rows whose products may have left FP16's range, over 16 channels (of one group of 32), straight from the cache
// in FP32: values past the range or far below their part's power, and what is not finite at all. `rows` are lanes,
// row row0 + lane of a KV head; `zeros` those that came out zero. A warp per row, a lane per token: slow (a row of
// 16384 tokens takes 1.5 ms), and no cache of ordinary values comes here.
template <int HD>
__device__ __forceinline__ void exact_rows(const TreeArgs& a, int b, int head, int row0, int col0, uint32_t rows,
                                                uint32_t zeros) {
  constexpr int G = HD / 32;
  const int lane = threadIdx.x & 31;
  const Request r = load_request(a, b);
  const int total = r.length + r.count, page_mask = (1 << a.shift) - 1;
  const int32_t* table = a.table + static_cast<int64_t>(b) * a.width;
  const float scale_log2 = a.scale_log2 * (kQueryPower * kKeyPower);
  // the slot of a token and its first scale among the head's
  const auto find = [&](int t, int64_t& slot, int64_t& plane) {
    int page = table[t >> a.shift];
    if (static_cast<uint32_t>(page) >= static_cast<uint32_t>(a.pages)) page = 0;  // reported by the first kernel
    slot = (static_cast<int64_t>(page) << a.shift) + (t & page_mask);
    const int cache_row = page / a.pages_per_row;
    plane = (static_cast<int64_t>(cache_row) * a.kv + head) * G * a.T + slot - cache_row * a.T;
  };
  // the largest scale that a row sees, by whose power of two its sums stay in FP32's range: first of the prefix
  uint32_t prefix = 0;
#pragma unroll 4
  for (int t = lane; t < r.length; t += 32) {
    int64_t slot, plane;
    find(t, slot, plane);
    prefix = max(prefix, a.v_scale[plane + col0 / 32 * a.T] & 0x7fffu);
  }
  prefix = __reduce_max_sync(0xffffffffu, prefix);
  for (; rows; rows &= rows - 1) {
    const int i = __ffs(rows) - 1, row = row0 + i, node = row / a.rep, query = head * a.rep + row - node * a.rep;
    const uint64_t path = a.ancestors[static_cast<int64_t>(b) * a.N + node];
    const uint16_t* q = a.q + (static_cast<int64_t>(b) * a.N + node) * a.q_stride + static_cast<int64_t>(query) * HD;
    uint32_t top = prefix;
    bool broken = false;  // by a draft that is not finite
    for (int t = r.length + lane; t < total; t += 32) {
      if (!(path >> (t - r.length) & 1)) continue;
      int64_t slot, plane;
      find(t, slot, plane);
      const uint32_t bits = a.v_scale[plane + col0 / 32 * a.T] & 0x7fffu;
      top = max(top, bits);
      broken = broken || bits >= kHugeScale;
      for (int g = 0; g < G; ++g) broken = broken || (a.k_scale[plane + g * a.T] & 0x7fffu) >= kHugeScale;
    }
    top = __reduce_max_sync(0xffffffffu, top);
    broken = __any_sync(0xffffffffu, broken);
    const float power = power_of(min(max(top >> 7, 1u), 253u)), inverse = inverse_power(power);
    float m = -INFINITY, l = 0.f, o[kJoinCols];
#pragma unroll
    for (int j = 0; j < kJoinCols; ++j) o[j] = 0.f;
    const bool done = broken || (top == 0 && (zeros >> i & 1));  // values that are all zero: so is what was found
    for (int t = done ? total : lane; t < total; t += 32) {
      if (t >= r.length && !(path >> (t - r.length) & 1)) continue;
      int64_t slot, plane;
      find(t, slot, plane);
      const int64_t code = (slot * a.kv + head) * HD;
      const uint4 v = *reinterpret_cast<const uint4*>(a.v_codes + code + col0);
      const float scale = bf16_to_f32(a.v_scale[plane + col0 / 32 * a.T]) * inverse;
      float x = 0.f;
#pragma unroll 1
      for (int c = 0; c < HD; c += 64) {
        uint4 k[4];
        float by[2];
#pragma unroll
        for (int h = 0; h < 4; ++h) k[h] = *reinterpret_cast<const uint4*>(a.k_codes + code + c + 16 * h);
#pragma unroll
        for (int h = 0; h < 2; ++h) by[h] = bf16_to_f32(a.k_scale[plane + (c / 32 + h) * a.T]);
#pragma unroll
        for (int g = 0; g < 2; ++g) {
          float part = 0.f;
#pragma unroll
          for (int h = 0; h < 4; ++h) {
            uint4 u = *reinterpret_cast<const uint4*>(q + c + 32 * g + 8 * h);
            u = make_uint4((u.x & a.q_keep) ^ a.q_flip, (u.y & a.q_keep) ^ a.q_flip, (u.z & a.q_keep) ^ a.q_flip,
                           (u.w & a.q_keep) ^ a.q_flip);
            float f[8];
            unpack8(u, f);
#pragma unroll
            for (int j = 0; j < 8; ++j)
              part = fmaf(f[j], static_cast<float>(static_cast<int8_t>(word(k[2 * g + h / 2], 2 * (h % 2) + j / 4) >> 8 * (j % 4))),
                          part);
          }
          x = fmaf(part, by[g], x);
        }
      }
      x *= scale_log2;
      const float now = fmaxf(m, x), shift = now == -INFINITY ? 0.f : now;
      const float keep = exp2f(m - shift), p = exp2f(x - shift);
      m = now;
      l = fmaf(l, keep, p);
#pragma unroll
      for (int j = 0; j < kJoinCols; ++j)
        o[j] = fmaf(o[j], keep, p * (static_cast<float>(static_cast<int8_t>(word(v, j / 4) >> 8 * (j % 4))) * scale));
    }
    float most = m;
#pragma unroll
    for (int s = 16; s; s >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, s));
    const float share = exp2f(m - (most == -INFINITY ? 0.f : most));
    l *= share;
#pragma unroll
    for (int s = 16; s; s >>= 1) l += __shfl_xor_sync(0xffffffffu, l, s);
    const int64_t to = ((static_cast<int64_t>(b) * a.N + node) * a.hq + query) * HD + col0;
#pragma unroll
    for (int j = 0; j < kJoinCols; ++j) {
      float sum = o[j] * share;
#pragma unroll
      for (int s = 16; s; s >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, s);
      if (lane != j) continue;
      float f = broken ? __uint_as_float(0x7fc00000u) : l == 0.f ? 0.f : sum / l * power;
      if (a.gate) f *= sigmoid_fast(bf16_to_f32(a.gate[to + j]));
      a.out[to + j] = bf16_bits_rne(f);
    }
    __syncwarp();
  }
}

template <int HD, int WARPS>
__global__ void __launch_bounds__(kJoinWarps * 32, 2) tree_join_kernel(const __grid_constant__ TreeArgs a, int pieces) {
  __shared__ float red[WARPS > 1 ? WARPS : 1][3][32];
  __shared__ float acc[WARPS > 1 ? WARPS : 1][kJoinCols][33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int p = WARPS > 1 ? blockIdx.x : blockIdx.x * kJoinWarps + warp;
  if (p >= pieces) return;
  const int groups = a.part_rows / 32, pr = a.part_rows;
  const int group = p % groups, col0 = p / groups % (HD / kJoinCols) * kJoinCols;
  const int unit = p / groups / (HD / kJoinCols);
  const int b = unit / (a.kv * a.row_tiles), head = unit / a.row_tiles % a.kv, row_tile = unit % a.row_tiles;
  const int in_tile = group * 32 + lane, row = row_tile * kRows + in_tile, node = row / a.rep;
  const int64_t to =
      ((static_cast<int64_t>(b) * a.N + node) * a.hq + head * a.rep + (row - node * a.rep)) * HD + col0;
  const int first = WARPS > 1 ? warp : 0;
  pdl_wait();
  pdl_trigger();
  uint4 gate[2];
  if (a.gate && first == 0 && node < a.N) {
    gate[0] = ld_guarded_v4(a.gate + to);
    gate[1] = ld_guarded_v4(a.gate + to + 8);
  }
  Parts parts = a.parts[unit];
  // a first kernel that gave up may have left them unwritten: what is read stays in the workspace
  parts.first = min(max(parts.first, 0), a.ctas - 1);
  parts.count = min(parts.count, a.ctas - parts.first);
  const int count = load_request(a, b).count;
  uint4* out = reinterpret_cast<uint4*>(a.out + to);
  if (row - lane >= count * a.rep) {  // nobody in these rows
    if (first == 0 && node < a.N) out[0] = out[1] = make_uint4(0, 0, 0, 0);
    return;
  }
  const int64_t record = static_cast<int64_t>(unit) + parts.first;
  // one pass with a running maximum, as over tiles; `power`: the parts' powers by their weight
  const float* powers = a.powers + record * (HD / 32) + col0 / 32;
  float m = -INFINITY, l = 0.f, power = 0.f, o[kJoinCols];
#pragma unroll
  for (int j = 0; j < kJoinCols; ++j) o[j] = 0.f;
#pragma unroll 2
  for (int i = first; i < parts.count; i += WARPS) {
    const float* st = a.stats + (record + i) * 3 * pr + in_tile;
    const float* part = a.part + ((record + i) * HD + col0) * pr + in_tile;
    const float x = st[0], y = st[pr] + st[2 * pr];
    const float by = powers[i * (HD / 32)];
    float v[kJoinCols];
#pragma unroll
    for (int j = 0; j < kJoinCols; ++j) v[j] = part[j * pr];
    const float top = fmaxf(m, x), shift = top == -INFINITY ? 0.f : top;
    const float keep = exp2_fast(m - shift), w = exp2_fast(x - shift);
    m = top;
    l = fmaf(l, keep, y * w);
    power = fmaf(power, keep, y * w * by);
#pragma unroll
    for (int j = 0; j < kJoinCols; ++j) o[j] = fmaf(o[j], keep, v[j] * (w * by));
  }
  if (WARPS > 1) {
    red[warp][0][lane] = m;
    red[warp][1][lane] = l;
    red[warp][2][lane] = power;
#pragma unroll
    for (int j = 0; j < kJoinCols; ++j) acc[warp][j][lane] = o[j];
    __syncthreads();
    if (warp) return;
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) top = fmaxf(top, red[w][0][lane]);
    const float shift = top == -INFINITY ? 0.f : top;
    l = power = 0.f;
#pragma unroll
    for (int j = 0; j < kJoinCols; ++j) o[j] = 0.f;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      const float f = exp2_fast(red[w][0][lane] - shift);
      l = fmaf(red[w][1][lane], f, l);
      power = fmaf(red[w][2][lane], f, power);
#pragma unroll
      for (int j = 0; j < kJoinCols; ++j) o[j] = fmaf(acc[w][j][lane], f, o[j]);
    }
  }
  const bool sees = node < count && (l > 0.f || l != l);
  float size = 0.f;
#pragma unroll
  for (int j = 0; j < kJoinCols; ++j) size += fabsf(o[j]);
  const float least = power * (kSmall * kJoinCols) * rsqrtf(fmaxf(l * (1.f / kMostWeight), 1.f));
  const bool lost = sees && !(size >= least && size < INFINITY);  // also where something is NaN
  if (node < a.N && !lost) {
    const float inv = sees ? 1.f / l : 0.f;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float f[8], z[8];
      if (a.gate) unpack8(gate[h], z);
      uint32_t w[4];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        f[j] = inv == 0.f ? 0.f : o[h * 8 + j] * inv;
        if (a.gate && inv != 0.f) f[j] *= sigmoid_fast(z[j]);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) w[j] = pack_bf16x2(f[2 * j], f[2 * j + 1]);
      out[h] = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
  // Last, where nothing has to be kept. Inlined: as a function it made the compiler spill, 20.6 -> 21.6 us for one node.
  const uint32_t rows = __ballot_sync(0xffffffffu, lost), zeros = __ballot_sync(0xffffffffu, size == 0.f && l == l);
  if (__builtin_expect(rows != 0, 0)) exact_rows<HD>(a, b, head, row - lane, col0, rows, zeros);
}

constexpr size_t kHeader = 256;

int part_rows(int N, int rep) {
  const int rows = (N * rep + 31) / 32 * 32;
  return rows < kRows ? rows : kRows;
}

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                  const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// A row-major matrix [rows, width] with rows `pitch` bytes apart, in boxes of box_rows x box_width.
bool encode(CUtensorMap* map, const void* base, CUtensorMapDataType type, uint64_t width, uint64_t rows, uint64_t pitch,
            uint32_t box_width, uint32_t box_rows) {
  EncodeTiledFn fn = reinterpret_cast<EncodeTiledFn>(tensor_map_encoder());
  if (!fn) return false;
  const cuuint64_t dims[2] = {width, rows};
  const cuuint64_t strides[1] = {pitch};
  const cuuint32_t box[2] = {box_width, box_rows};
  const cuuint32_t estr[2] = {1, 1};
  return fn(map, type, 2, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

struct Layout {
  int row_tiles, part_rows;
  int64_t units, records;
  size_t parts, part, stats, powers, bytes;
};
Layout layout_of(int B, int N, int hq, int kv, int hd) {
  Layout w;
  const int rep = hq / kv;
  w.row_tiles = (N * rep + kRows - 1) / kRows;
  w.part_rows = part_rows(N, rep);
  w.units = static_cast<int64_t>(B) * kv * w.row_tiles;
  w.records = w.units + sm_count();
  w.parts = kHeader;
  w.stats = w.parts + (w.units * sizeof(Parts) + 255) / 256 * 256;
  w.powers = w.stats + static_cast<size_t>(w.records) * 3 * w.part_rows * sizeof(float);
  w.part = w.powers + (static_cast<size_t>(w.records) * (hd / 32) * sizeof(float) + 255) / 256 * 256;
  w.bytes = w.part + static_cast<size_t>(w.records) * hd * w.part_rows * sizeof(float);
  return w;
}

template <int HD>
int launch(const Maps& maps, const TreeArgs& a, const Layout& w, cudaStream_t st) {
  const size_t smem = 1024 + 2 * kStages * static_cast<size_t>(kTile) * HD * 2 + kRaw * Raw<HD>::kBytes + kSoftmaxWarps * kQStage;
  const int rc = allow_smem(reinterpret_cast<const void*>(tree_attention_kernel<HD>), smem);
  if (rc) return rc;
  // one CTA per SM: each holds all of its SM's tensor memory
  cudaError_t e = launch_dependent(tree_attention_kernel<HD>, dim3(sm_count()), dim3(kThreads), smem, st, maps, a);
  if (e != cudaSuccess) return cuda_error(e, "tree_attention_kernel");
  const int pieces = static_cast<int>(w.units * (w.part_rows / 32) * (HD / kJoinCols));
  if (pieces >= 4 * sm_count()) {
    e = launch_dependent(tree_join_kernel<HD, 1>, dim3((pieces + kJoinWarps - 1) / kJoinWarps), dim3(kJoinWarps * 32), 0, st,
                         a, pieces);
  } else {
    e = launch_dependent(tree_join_kernel<HD, kJoinWarps>, dim3(pieces), dim3(kJoinWarps * 32), 0, st, a, pieces);
  }
  if (e != cudaSuccess) return cuda_error(e, "tree_join_kernel");
  count_launch(2);
  return QK_OK;
}

}  // namespace
}  // namespace qk

using namespace qk;

extern "C" {

size_t qk_tree_attention_workspace_bytes(int B, int N, int hq, int kv_heads, int head_dim) {
  if (B <= 0 || N <= 0 || N > 64 || kv_heads <= 0 || hq <= 0 || hq % kv_heads || head_dim <= 0) return kHeader;
  return layout_of(B, N, hq, kv_heads, head_dim).bytes;
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
  QK_REQUIRE(static_cast<int64_t>(N) * q_stride < (1ll << 31), "a request's queries must span fewer than 2^31 values");
  const Layout w = layout_of(B, N, hq, kv_heads, head_dim);
  QK_REQUIRE(w.units * (w.part_rows / 32) * (head_dim / kJoinCols) < (1ll << 31), "too many rows in one call");
  QK_REQUIRE(static_cast<int64_t>(width) * page_size < (1ll << 31) - kTile, "a table row must span fewer than 2^31 - 64 tokens");
  QK_REQUIRE(w.units * (static_cast<int64_t>(width) * page_size / kTile + kUnitCost + 1) < (1ll << 31),
             "too many requests of such a length in one call");
  const size_t need = w.bytes;
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
  a.scale_log2 = scale == 0.f ? 1.f : fabsf(scale) * (1.44269504088896341f / (kQueryPower * kKeyPower));
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
  a.room = static_cast<int>(static_cast<int64_t>(width) * page_size);
  while ((1 << a.shift) < page_size) ++a.shift;
  a.row_tiles = w.row_tiles;
  a.part_rows = w.part_rows;
  a.ctas = sm_count();
  a.T = T;
  a.out = out;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  a.status = reinterpret_cast<int*>(ws);
  a.parts = reinterpret_cast<Parts*>(ws + w.parts);
  a.part = reinterpret_cast<float*>(ws + w.part);
  a.stats = reinterpret_cast<float*>(ws + w.stats);
  a.powers = reinterpret_cast<float*>(ws + w.powers);
  Maps maps;
  const uint64_t D = static_cast<uint64_t>(kv_heads) * head_dim, slots = static_cast<uint64_t>(rows) * T;
  const uint32_t box = page_size < kTile ? page_size : kTile;
  if (!encode(&maps.k_codes, k_codes, CU_TENSOR_MAP_DATA_TYPE_UINT8, D, slots, D, head_dim, box) ||
      !encode(&maps.v_codes, v_codes, CU_TENSOR_MAP_DATA_TYPE_UINT8, D, slots, D, head_dim, box) ||
      !encode(&maps.k_scale, k_scale, CU_TENSOR_MAP_DATA_TYPE_UINT16, T, rows * (D / 32), 2 * T, box, head_dim / 32) ||
      !encode(&maps.v_scale, v_scale, CU_TENSOR_MAP_DATA_TYPE_UINT16, T, rows * (D / 32), 2 * T, box, head_dim / 32))
    return set_error(QK_ERR_CUDA, "cuTensorMapEncodeTiled is unavailable or refused the cache");
  return head_dim == 256   ? launch<256>(maps, a, w, as_stream(stream))
         : head_dim == 128 ? launch<128>(maps, a, w, as_stream(stream))
                           : launch<64>(maps, a, w, as_stream(stream));
}

int qk_tree_attention_check(const void* workspace, qk_stream_t stream) {
  int status = 0;
  cudaStream_t st = as_stream(stream);
  void* word = const_cast<void*>(workspace);
  cudaError_t e = word ? cudaSuccess : cudaGetSymbolAddress(&word, g_tree_status);
  if (e == cudaSuccess) e = cudaMemcpyAsync(&status, word, sizeof(int), cudaMemcpyDeviceToHost, st);
  if (e == cudaSuccess) e = cudaStreamSynchronize(st);
  if (e == cudaSuccess && status) {
    e = cudaMemsetAsync(word, 0, sizeof(int), st);
    if (e == cudaSuccess) e = cudaStreamSynchronize(st);
  }
  if (e != cudaSuccess) return cuda_error(e, "qk_tree_attention_check");
  if (status == QK_ERR_TIMEOUT) return set_error(status, "a bounded device wait in the tree attention gave up");
  if (status) return set_error(status, "a block table entry lies outside the cache, or a length outside the table");
  return QK_OK;
}

}  // extern "C"
