// Attention of new tokens over the paged cache: the kernels, with and without rules.
//
//   s_t = scale * q . k_t  for the tokens t the row sees: those up to its own
//         position, the last `window` of them if there is one
//   out = sum_t softmax(s)_t v_t;  a row that sees nothing is zeros
//
// Rows are (new token, query head of the group): the query heads that share a
// key/value head are rows of one tile, so a cached row is read once for all of
// them. A wave takes 32 cached tokens a step, in registers from end to end:
//   S' = K q'   16 tokens x 16 rows per v_mfma_f32_16x16x32_f16: lane (n, g) =
//               (lane % 16, lane / 16) gets row n's scores of tokens 4 g .. 4 g + 3
//   P           the running maximum and sum of row n live in its 4 lanes
//   O' += V' P' the same lanes hold what the second operand needs: 8 of the 32
//               tokens of row n, and V's operand is 8 rows of V, 2 E bytes each,
//               turned in the lane with v_perm (E = D / 16 columns of a lane)
// so neither scores nor weights ever leave the lane.
//
// Precision. q (scaled by a power of two to a row maximum of 2^13) and p (scaled
// by 2^14) are split in two fp16 parts, 22 bits, each its own matrix step; the
// cached fp16 or int8 values are exact operands; sums are f32. An int8 row's scale
// (of either sign) multiplies its scores, and its weights: the fp16 parts are of the
// products, in units of 2^-14 of the largest one the row has met, which shrinks with
// the weights as the maximum grows. (Not of the largest scale: a token of no weight
// and a large scale would take the others' bits.)
//
// Rules (RULES; else none of what follows is compiled in). A score s = scale q . k becomes
//   cap tanh(s / cap)                 where there is a cap
//   less slope |p - p_t|              p, p_t the positions of the row's token and of t
// and a row sees t where its range, or for the drafts of a tree its row of the tree,
// says so.
#pragma once

#include <algorithm>

#include "eff_device.h"
#include "eff_kv.h"

namespace eff {

typedef float float4v __attribute__((ext_vector_type(4)));
typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef short short2v __attribute__((ext_vector_type(2)));

__device__ __forceinline__ float4v mfma(half8 a, half8 b, float4v c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

// int8 quants (with the sign bit flipped: 0 .. 255) in the low bytes of fp16
// 1024 + u, less 1152: exact.
__device__ __forceinline__ uint32_t i8_half2(uint32_t bits) {
  const half2v c = {(_Float16)1152.f, (_Float16)1152.f};
  return __builtin_bit_cast(uint32_t, __builtin_bit_cast(half2v, bits) - c);
}

__device__ __forceinline__ half8 i8_half8(uint32_t a, uint32_t b) {
  a ^= 0x80808080u, b ^= 0x80808080u;
  const uint32_t k = 0x64646464u;
  const u32x4 v = {i8_half2(__builtin_amdgcn_perm(k, a, 0x04010400u)), i8_half2(__builtin_amdgcn_perm(k, a, 0x04030402u)),
                   i8_half2(__builtin_amdgcn_perm(k, b, 0x04010400u)), i8_half2(__builtin_amdgcn_perm(k, b, 0x04030402u))};
  return __builtin_bit_cast(half8, v);
}

__device__ __forceinline__ half8 join8(const half2v v[4]) {
  return half8{v[0][0], v[0][1], v[1][0], v[1][1], v[2][0], v[2][1], v[3][0], v[3][1]};
}

// 16 bytes of LDS.
__device__ __forceinline__ void ld_lds(uint32_t *o, const uint8_t *p) {
  const u32x4 v = *(const u32x4 *)p;
#pragma unroll
  for (int i = 0; i < 4; ++i) o[i] = v[i];
}

// 4 N bytes of the cache. An address made of two words may be LDS for all the compiler
// knows: without its space named the loads would be counted with LDS's, and a wait for
// one of them would wait for all that are under way.
template <typename T>
using cached = const __attribute__((address_space(1))) T *;
template <int N>
__device__ __forceinline__ void ld_cache(uint32_t *o, const uint8_t *p) {
  typedef uint32_t words __attribute__((ext_vector_type(N == 1 ? 2 : N)));
  if constexpr (N == 1) {
    *o = *(cached<uint32_t>)p;
  } else {
    const words v = *(cached<words>)p;
#pragma unroll
    for (int i = 0; i < N; ++i) o[i] = v[i];
  }
}

// A constant that the compiler does not see, so that it keeps the instruction
// around it.
__device__ __forceinline__ float unseen(float v) {
  __asm__("" : "=s"(v) : "0"(v));
  return v;
}

// The larger of two numbers. (fmaxf first quiets each operand that may be a
// signalling NaN, an instruction each; a NaN here makes the row's sum NaN anyway.)
__device__ __forceinline__ float max2(float a, float b) { return __builtin_amdgcn_fmed3f(a, b, unseen(INFINITY)); }

// Of 8 numbers, NaN if one is: three operands an instruction.
__device__ __forceinline__ float max8(const float s[2][4]) {
  float m = s[0][0];
#pragma unroll
  for (int k = 1; k < 8; ++k) m = __builtin_elementwise_maximum(m, s[k / 4][k % 4]);
  return m;
}

__device__ __forceinline__ float min8(const float s[2][4]) {
  float m = s[0][0];
#pragma unroll
  for (int k = 1; k < 8; ++k) m = __builtin_elementwise_minimum(m, s[k / 4][k % 4]);
  return m;
}

// Maximum and sum over the 4 lanes that hold a row (lane % 16). The swaps leave
// the two halves (two 16-lane rows) of v side by side in two registers.
__device__ __forceinline__ float row_max(float v) {
  auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = max2(__uint_as_float(a[0]), __uint_as_float(a[1]));
  auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return max2(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

__device__ __forceinline__ float row_add(float v) {
  auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// Two values in two fp16 parts: v = hi + lo to 22 bits. (hi * -1 + v in one
// instruction each, with the conversions.)
__device__ __forceinline__ void split2(float a, float b, half2v &hi, half2v &lo) {
  uint32_t h = __builtin_bit_cast(uint32_t, half2v{(_Float16)a, (_Float16)b});
  __asm__("" : "+v"(h));   // one packed conversion, not two more for the halves
  hi = __builtin_bit_cast(half2v, h);
  const float m = unseen(-1.f);
  lo = half2v{(_Float16)fmaf((float)hi[0], m, a), (_Float16)fmaf((float)hi[1], m, b)};
}

constexpr uint32_t kLeast = 2, kShort = 8;   // units of a share
constexpr uint32_t kUnit = 128;   // tokens: a step of each of four waves
constexpr float kLeastUnit = 0x1p-100f;   // of weights times scales

// The rows of a tile, their tokens and what they see.
struct AttnTile {
  uint32_t seq, token0;   // the sequence's first new token
  uint32_t r0, rows;      // rows r0 .. r0 + rows - 1 of the sequence's n * group
  int first, last;        // positions of the first and last row
  int begin, end;         // the cached tokens that any row sees
};

// The same under rules.
struct AttnTileRules : AttnTile {
  int base, len;          // position of the sequence's first new token, and of the one behind its last
  int all_from, all_to;   // the cached tokens that every row sees
};
template <bool RULES>
struct AttnTileOf {
  typedef AttnTile type;
};
template <>
struct AttnTileOf<true> {
  typedef AttnTileRules type;
};

// Of a group of L lanes, that of lane `of` (16: DPP, 64: then swaps), the largest number, and the smallest.
template <uint32_t L>
__device__ __forceinline__ int lanes_max(int v, uint32_t of = 0) {
  v = max(v, __builtin_amdgcn_update_dpp(0, v, 0xB1, 0xF, 0xF, false));
  v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x4E, 0xF, 0xF, false));
  v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x141, 0xF, 0xF, false));
  v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x140, 0xF, 0xF, false));
  if constexpr (L == 64u) {
    auto a = __builtin_amdgcn_permlane32_swap((uint32_t)v, (uint32_t)v, false, false);
    v = max((int)a[0], (int)a[1]);
    auto b = __builtin_amdgcn_permlane16_swap((uint32_t)v, (uint32_t)v, false, false);
    v = max((int)b[0], (int)b[1]);
  }
  return __builtin_amdgcn_readlane(v, of);
}
template <uint32_t L>
__device__ __forceinline__ int lanes_min(int v, uint32_t of = 0) { return -lanes_max<L>(-v, of); }

// The cached tokens that a row's range names, of `len`.
__device__ __forceinline__ void range_of(const KvRulesView &r, uint32_t token, int len, int &from, int &to) {
  const uint2 v = *(const uint2 *)(r.ranges + 2ull * token);
  from = (int)min(v.x, (uint32_t)len), to = (int)min(v.y, (uint32_t)len);
}

// The range of row i of a tile; empty for a token without a position, and where there are
// no ranges.
__device__ __forceinline__ void attn_range(const AttnTileRules &t, const KvRulesView &r, uint32_t group, uint32_t i, int &from, int &to) {
  from = 0, to = 0;
  if (!r.ranges || i >= t.rows) return;
  const uint32_t tok = (t.r0 + i) / group;
  range_of(r, t.token0 + tok, max(t.len, 0), from, to);
  if (t.base + (int)tok < 0) to = 0;
}

// What a tile's rows see under rules (without rules it stands): R rows at most, whose
// ranges lie in the R lanes from lane `of` on.
template <uint32_t R>
__device__ __forceinline__ void attn_seen(AttnTile &, NoRules, int, int, int, uint32_t = 0) {}
template <uint32_t R>
__device__ __forceinline__ void attn_seen(AttnTileRules &t, const KvRulesView &r, int window, int from, int to, uint32_t of = 0) {
  t.all_from = window ? max(0, t.last - window + 1) : 0;
  t.all_to = t.first + 1;
  if (r.tree) {
    // a row's position is not known before its tree row is read: base - 1 to the last's
    t.begin = window ? max(0, t.base - window) : 0;
    t.end = max(t.len, 0);
    t.all_from = window ? max(0, t.len - window) : 0;
    t.all_to = max(t.base, 0);
  } else if (r.ranges) {
    const bool on = (threadIdx.x & 63u) - of < t.rows, some = on && from < to;
    t.begin = lanes_min<R>(some ? from : 0x7FFFFFFF, of);
    t.end = lanes_max<R>(some ? to : 0, of);
    if (t.end == 0) t.begin = 0;
    t.all_from = lanes_max<R>(on ? from : 0, of);
    t.all_to = lanes_min<R>(on ? to : 0x7FFFFFFF, of);
  }
}

// Tile `sub` of a sequence of n new tokens from s0 on, `len` with them.
template <uint32_t R, typename TILE>
__device__ __forceinline__ void attn_rows_of(TILE &t, uint32_t sub, uint32_t s0, uint32_t n, int len, uint32_t group, uint32_t window) {
  t.token0 = s0;
  t.r0 = sub * R;
  t.rows = min(R, n * group - t.r0);
  t.first = len - (int)n + (int)(t.r0 / group);
  t.last = len - (int)n + (int)((t.r0 + t.rows - 1u) / group);
  t.end = max(t.last + 1, 0);
  t.begin = window ? max(0, t.first - (int)min(window, 0x40000000u) + 1) : 0;
  if constexpr (__is_same(TILE, AttnTileRules)) t.base = len - (int)n, t.len = len;
}

// The tile of a workgroup, of the sequences that have min_rows .. max_rows rows:
// `per_seq` tiles of each sequence, or (per_seq = 0) their tiles one after the other.
template <uint32_t R, typename TILE>
__device__ __forceinline__ bool attn_tile(const KvBatchView &b, uint32_t group, uint32_t window, uint32_t tile,
                                          uint32_t per_seq, uint32_t min_rows, uint32_t max_rows, TILE &t) {
  const uint32_t lane = threadIdx.x & 63u;
  uint32_t sub;
  if (per_seq) {
    t.seq = tile / per_seq, sub = tile % per_seq;
  } else {
    uint32_t base = 0;
    t.seq = b.seqs;
    sub = 0;
    for (uint32_t at = 0; at < b.seqs; at += 64u) {
      const uint32_t i = at + lane;
      uint32_t n = 0;
      if (i < b.seqs) {
        const uint32_t s0 = b.starts[i], s1 = b.starts[i + 1];
        n = s1 > s0 ? min(s1 - s0, b.max_new) * group : 0u;
        n = n >= min_rows && n <= max_rows ? (n + R - 1u) / R : 0u;
      }
      uint32_t sum = n;
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const uint32_t u = __shfl_up(sum, o);
        if ((int)lane >= o) sum += u;
      }
      const uint64_t past = __ballot(base + sum > tile);
      if (past) {
        const int l = __ffsll((unsigned long long)past) - 1;
        t.seq = at + l;
        sub = tile - (base + __shfl(sum - n, l));
        break;
      }
      base += __shfl(sum, 63);
    }
  }
  if (t.seq >= b.seqs) return false;
  t.seq = __builtin_amdgcn_readfirstlane(t.seq);
  sub = __builtin_amdgcn_readfirstlane(sub);
  const uint32_t s0 = __builtin_amdgcn_readfirstlane(b.starts[t.seq]);
  const uint32_t s1 = min((uint32_t)__builtin_amdgcn_readfirstlane(b.starts[t.seq + 1]), b.tokens);
  const uint32_t n = s1 > s0 ? min(s1 - s0, b.max_new) : 0u;
  if (sub * R >= n * group || n * group < min_rows || n * group > max_rows) return false;
  attn_rows_of<R>(t, sub, s0, n, __builtin_amdgcn_readfirstlane((int)kv_len(b, t.seq)), group, window);
  return true;
}

// A workgroup's share of the cached tokens that all tiles see, in units of 128 tokens,
// the tiles' one after the other: the next tile of it.
struct AttnShare {
  uint32_t each, left;    // units of a workgroup; units that this one has left
  uint32_t sub, of;       // the tile within its sequence, and units of each of the sequence's tiles
  uint32_t start, at;     // the tile's first unit of all, and the share's first within the tile
};

// Units of each tile of a sequence of `len` tokens at most; under a window the tokens of
// its rows (of a tree all new ones, `tree` of them at most) and the window before them.
template <uint32_t R>
__device__ __forceinline__ uint32_t attn_units(uint32_t len, uint32_t group, uint32_t window, uint32_t tree) {
  const uint32_t span = window ? min(len, min(window, 0x40000000u) + max(R / group, tree) + 33u) : len;
  return max((span + kUnit - 1u) / kUnit, 1u);
}

// The share of workgroup `item` of `items`, kLeast units at least: every one has the
// same work, whatever the lengths are. Each wave adds the sequences up for itself, 64
// at a time. A share that goes on into the next tile starts anew there, with its
// loads' latency: short shares end with a tile instead (ENDS: all; there are more
// items than tiles).
template <uint32_t R, bool ENDS, typename TILE>
__device__ __forceinline__ bool attn_share(const KvBatchView &b, uint32_t group, uint32_t window, uint32_t tree, uint32_t item,
                                           uint32_t items, uint32_t max_rows, TILE &t, AttnShare &c) {
  const uint32_t lane = threadIdx.x & 63u;
  uint32_t s0 = 0, n = 0, len = 0, tiles = 0, of = 0;
  const auto load = [&](uint32_t at) {
    const uint32_t i = at + lane;
    n = len = 0;
    if (i < b.seqs) {
      s0 = b.starts[i];
      const uint32_t s1 = min(b.starts[i + 1], b.tokens);
      len = kv_len(b, i);
      n = s1 > s0 ? min(s1 - s0, b.max_new) : 0u;
    }
    tiles = n * group <= max_rows ? (n * group + R - 1u) / R : 0u;
    of = attn_units<R>(len, group, window, tree);
  };
  if (ENDS && b.seqs == 1u) {   // scalar all the way
    const uint32_t from = __builtin_amdgcn_readfirstlane(b.starts[0]), to = min((uint32_t)__builtin_amdgcn_readfirstlane(b.starts[1]), b.tokens);
    const uint32_t l = __builtin_amdgcn_readfirstlane(kv_len(b, 0)), m = to > from ? min(to - from, b.max_new) : 0u;
    const uint32_t units = attn_units<R>(l, group, window, tree), many = (m * group + R - 1u) / R;
    if (m * group > max_rows || many >= items) return false;
    c.each = max((many * units + items - many - 1u) / (items - many), kLeast);
    c.of = (units + c.each - 1u) / c.each * c.each;
    c.sub = item * c.each / c.of;
    if (c.sub >= many) return false;
    c.start = c.sub * c.of, c.at = item * c.each - c.start, c.left = c.each;
    t.seq = 0;
    attn_rows_of<R>(t, c.sub, from, m, (int)l, group, window);
    return true;
  }
  load(0);
  uint32_t total = 0, count = 0;
  for (uint32_t at = 0;;) {
    total += tiles * of;
    count += tiles;
    if ((at += 64u) >= b.seqs) break;
    load(at);
  }
  if (b.seqs > 1u) {
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) total += __shfl_xor(total, o), count += __shfl_xor(count, o);
  }
  total = __builtin_amdgcn_readfirstlane(total);
  count = __builtin_amdgcn_readfirstlane(count);
  uint32_t each = (total + items - 1u) / items, whole = 1;
  if (ENDS && count >= items) return false;
  if (ENDS || (each < kShort && count < items)) whole = each = max((total + items - count - 1u) / (items - count), kLeast);
  if (ENDS && __is_same(TILE, AttnTileRules) && b.seqs <= 64u) {
    // that holds for any lengths; the smallest share that these need, which may be half of
    // it (16 trees of up to 32 over up to 16384: 189 -> 174 us; 40 of up to 6 over int8
    // pages 256 wide, 4096 of up to 9001 seen: 73 -> 64)
    for (uint32_t least = max((total + items - 1u) / items, kLeast); least < each;) {
      const uint32_t mid = (least + each) / 2u;
      if ((uint32_t)wave_sum((float)(tiles * ((of + mid - 1u) / mid))) <= items) each = mid;
      else least = mid + 1u;
    }
    whole = each;
  }
  each = max(each, kLeast);
  c.each = __builtin_amdgcn_readfirstlane(each);
  whole = __builtin_amdgcn_readfirstlane(whole);
  const uint32_t first = item * c.each;
  uint32_t base = 0;
  for (uint32_t at = 0; at < b.seqs; at += 64u) {
    if (b.seqs > 64u) load(at);
    if (whole > 1u) of = (of + whole - 1u) / whole * whole;
    const uint32_t mine = tiles * of;
    uint32_t sum = mine;
    if (b.seqs > 1u) {
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const uint32_t u = __shfl_up(sum, o);
        if ((int)lane >= o) sum += u;
      }
    }
    const uint64_t past = __ballot(base + sum > first);
    if (past) {
      const int l = __ffsll((unsigned long long)past) - 1;
      c.of = __builtin_amdgcn_readlane(of, l);
      const uint32_t before = base + __builtin_amdgcn_readlane(sum - mine, l), i = first - before;
      c.sub = __builtin_amdgcn_readfirstlane(i / c.of);
      c.at = i - c.sub * c.of;
      c.start = first - c.at;
      c.left = c.each;
      t.seq = at + l;
      attn_rows_of<R>(t, c.sub, __builtin_amdgcn_readlane(s0, l), __builtin_amdgcn_readlane(n, l), (int)__builtin_amdgcn_readlane(len, l),
                      group, window);
      return true;
    }
    base += __builtin_amdgcn_readlane(sum, 63);
  }
  return false;
}

// To the share's next tile; false: it ends.
template <uint32_t R, typename TILE>
__device__ __forceinline__ bool attn_next(const KvBatchView &b, uint32_t group, uint32_t window, uint32_t tree, uint32_t max_rows,
                                          TILE &t, AttnShare &c) {
  const uint32_t took = min(c.left, c.of - c.at);
  c.left -= took;
  if (c.left == 0u) return false;
  c.start += c.of;
  c.at = 0;
  ++c.sub;
  for (;;) {
    const uint32_t s0 = __builtin_amdgcn_readfirstlane(b.starts[t.seq]);
    const uint32_t s1 = min((uint32_t)__builtin_amdgcn_readfirstlane(b.starts[t.seq + 1]), b.tokens);
    const uint32_t len = __builtin_amdgcn_readfirstlane(kv_len(b, t.seq));
    const uint32_t n = s1 > s0 ? min(s1 - s0, b.max_new) : 0u;
    if (n * group <= max_rows && c.sub * R < n * group) {
      c.of = attn_units<R>(len, group, window, tree);
      attn_rows_of<R>(t, c.sub, s0, n, (int)len, group, window);
      return true;
    }
    if (++t.seq >= b.seqs) return false;
    c.sub = 0;
  }
}

// The walk over a tile's cached tokens: steps of 32 tokens at lo, lo + stride, ... up
// to hi, each two runs of 16 tokens of one page. The places of the next 32 steps'
// runs are computed at once, one in each lane; a step takes its two out of them.
struct AttnWalk {
  const uint32_t *table;   // the sequence's
  const uint8_t *heads;    // the first page's K of the head
  int lo, hi, stride;
  uint32_t low, high, slots;   // a lane's: address of its run's first row of K, and slot in the page
  uint64_t none;               // lanes whose run has no page
  const uint8_t *at[2];
  uint32_t slot[2];
  bool gone[2];

  template <int ROW>
  __device__ __forceinline__ void look(const KvView &kv, int t0) {
    const uint32_t lane = threadIdx.x & 63u;
    const int t = t0 + (int)(lane >> 1) * stride + 16 * (int)(lane & 1u);
    const uint32_t page = t < hi ? table[(uint32_t)t >> kv.page_log2] : ~0u;
    const bool there = page < kv.pages;
    none = __ballot(!there);
    slots = (uint32_t)t & ((1u << kv.page_log2) - 1u);
    // a run without a page reads the first page's rows, which are masked
    const uint64_t a = (uint64_t)(uintptr_t)heads + (there ? (uint64_t)page * kv.page_bytes : 0ull) + slots * (uint32_t)ROW;
    low = (uint32_t)a, high = (uint32_t)(a >> 32);
  }

  // To step i (in order).
  template <int ROW>
  __device__ __forceinline__ void go(const KvView &kv, int i) {
    if ((i & 31) == 0) look<ROW>(kv, lo + i * stride);
    const uint32_t l = 2u * (i & 31);
#pragma unroll
    for (uint32_t u = 0; u < 2u; ++u) {
      at[u] = (const uint8_t *)((uint64_t)__builtin_amdgcn_readlane(high, l + u) << 32 | (uint32_t)__builtin_amdgcn_readlane(low, l + u));
      slot[u] = __builtin_amdgcn_readlane(slots, l + u);
    }
    const uint32_t two = (uint32_t)(none >> l) & 3u;
    gone[0] = two & 1u, gone[1] = two >> 1;
  }

  // int8 pages: the scales of run u's rows of K.
  __device__ __forceinline__ const uint8_t *scales(int u, const KvView &kv, uint32_t dim) const {
    return at[u] + (dim << kv.page_log2) + 4u * slot[u] - dim * slot[u];
  }
};

// One wave's share of a tile of 16 rows: 16, because that is the matrix instruction's
// side, and a group of query heads seldom has more.
//   SCALED  rows of the cache have scales
//   I8      K and V arrive as int8 (else fp16, also where int8 was converted on the way)
//   QL      the parts of q are in LDS, shared by the waves of the tile, and read for
//           each step
//   VIN     V arrives as rows, as the operands that it is (turned by the LDS read), or
//           is read by the caller as it is used (for want of registers)
enum { kVRows, kVTurned, kVLater };

// tanh(z) / z in z^2 up to z = kTanhFew: within 4e-9 there (a least-maximum fit), 5.3e-8 in
// f32. Scores below 0.625 of the cap, the ordinary ones, cost 8 instructions each.
constexpr float kTanhFew = 0.625f;
constexpr float kTanh[6] = {1.f, -0.3333326f, 0.13331127f, -0.053721067f, 0.020590989f, -0.0056599886f};

// What a row sees and where it is, in LDS: a step reads it where it needs it, so that it
// takes no registers from step to step (fp16 256 wide would not have them).
struct AttnRule {
  int from, to;   // the cached tokens that it sees, but for the tree's
  int pos;        // its position
  float slope;    // times log2 e
};

// The rules as a wave has them; nothing without rules.
template <bool RULES>
struct AttnRulesOf {
  typedef NoRules type;
};
struct AttnRules {
  const KvRulesView &all;
  AttnRule *row;   // of the wave's first row; lane n has row n
  uint32_t group;
};
template <>
struct AttnRulesOf<true> {
  typedef AttnRules type;
};
__device__ __forceinline__ NoRules attn_rules(NoRules, AttnRule *, uint32_t) { return {}; }
__device__ __forceinline__ AttnRules attn_rules(const KvRulesView &r, AttnRule *row, uint32_t group) { return {r, row, group}; }

template <int D, bool SCALED, bool I8, bool QL, int VIN, bool RULES = false>
struct AttnWave {
  typedef typename AttnTileOf<RULES>::type Tile;
  typedef typename AttnRulesOf<RULES>::type Rules;
  static constexpr int E = D / 16;                     // columns of a lane
  static constexpr int KS = D / 32;                    // matrix steps of a score
  static constexpr int KW = I8 ? 2 : 4;                // words of a lane's part of a step of K
  static constexpr int VW = I8 ? (E + 3) / 4 : E / 2;  // words of a lane's part of a row of V
  static constexpr int ROW = I8 ? D : 2 * D;           // bytes of a row as it arrives
  // fp16 weights are scaled by 2^14, in the exponent itself where instruction issue
  // bounds the kernel (V not in rows: prompts of 64-wide heads 123 us, else 130). Next
  // to 14 the exponent has 4 bits less than next to 0, where it is computed elsewhere:
  // 9.2e-8 -> 6.2e-8 of 3 tokens' output, 2.4e-7 -> 2.0e-7 of 150's (f32 throughout
  // 5.0e-8 and 3.8e-7); of prompts' 2.6e-7 -> 2.3e-7 (3.4e-7).
  static constexpr bool RAISED = !SCALED && VIN != kVRows;

  half8 qh[QL ? 1 : KS], ql[QL ? 1 : KS];
  const uint8_t *qs;    // QL: [step][part][lane] of 16 bytes
  float sc;             // > 0: what a raw score of row n is multiplied by (log2 e included)
  int pos;              // the row's position, -1 for none
  float m, l;           // running maximum (of raw scores), and this lane's share of the sum
  float unit, inv;      // SCALED: what 1 in acc stands for, and its reciprocal
  float4v acc[E];

  uint32_t kw[2][KS * KW];
  uint32_t ks[2][4];                          // SCALED: the scales of the lane's tokens (f32 bits)
  static constexpr int VN = VIN == kVRows ? 8 : VIN == kVTurned ? E : 1, VM = VIN == kVRows ? VW : VIN == kVTurned ? 4 : 1;
  uint32_t vw[VN][VM];                        // V: 8 rows, or the operands of E columns
  uint32_t vs[2][4];

  // column of acc[i][j] of lane group g: turned, and at D = 96, side by side with the
  // group's 4 rows; else E side by side
  static __device__ __forceinline__ uint32_t column(uint32_t g, int i, int j) {
    if constexpr (VIN != kVRows) return 16u * i + 4u * g + j;
    if constexpr (D == 96) return i < 4 ? 4u * (4u * g + j) + i : 64u + 2u * (4u * g + j) + (i - 4);
    return (uint32_t)E * (4u * g + j) + i;
  }

  // The rows' q as it is in memory; rows that are none read the tile's first.
  __device__ __forceinline__ void load_q(float q[KS][8], const KvAttnArgs &a, const AttnTile &t, uint32_t group, uint32_t kvh,
                                         uint32_t n, uint32_t g) {
    const bool on = n < t.rows;
    const uint32_t r = t.r0 + (on ? n : 0u), tok = r / group, h = r % group;
    const float *src = a.q + (uint64_t)(t.token0 + tok) * a.q_stride + (kvh * group + h) * D;
#pragma unroll
    for (int c = 0; c < KS; ++c) {
      uint32_t d;
      if constexpr (I8) d = 2 * (c / 2) + 1 < KS ? 64u * (c / 2) + 16u * g + 8u * (c & 1) : 32u * c + 8u * g;
      else d = 32u * c + 8u * g;
      const float4 u = *(const float4 *)(src + d), w = *(const float4 *)(src + d + 4);
      q[c][0] = u.x, q[c][1] = u.y, q[c][2] = u.z, q[c][3] = u.w;
      q[c][4] = w.x, q[c][5] = w.y, q[c][6] = w.z, q[c][7] = w.w;
    }
    pos = on ? t.first + (int)(tok - t.r0 / group) : -1;
  }

  // What row n sees and how it scores, for the steps to read.
  static __device__ __forceinline__ void put_rule(const Rules &r, const Tile &t, uint32_t kvh, uint32_t n, uint32_t g, int window, int from, int to) {
    if constexpr (RULES) {
      const bool on = n < t.rows;
      const uint32_t i = t.r0 + (on ? n : 0u), tok = i / r.group;
      const int place = t.base + (int)tok;
      AttnRule x = {0, 0, place, 0.f};
      if (on && r.all.tree && (window || r.all.slopes)) x.pos = key_position(r, t, t.token0 + tok);
      if (r.all.ranges) x.from = from, x.to = to;
      else if (on) x.from = window ? max(0, x.pos - window + 1) : 0, x.to = r.all.tree ? t.len : place + 1;
      if (place < 0) x.to = 0;   // without a position it sees nothing
      // far from all that it sees, a row's distances are counted from the nearest of it: the
      // same weights, and small numbers
      if (r.all.ranges) x.pos = max(min(x.pos, x.to - 1), x.from);
      if (r.all.slopes) x.slope = r.all.slopes[kvh * r.group + i % r.group] * 1.44269504088896341f;
      if (g == 0u) r.row[n] = x;
    }
  }
  // Row n's, read here and not kept from step to step.
  static __device__ __forceinline__ AttnRule get_rule(const Rules &r, uint32_t n) {
    uint32_t nothing = 0;
    __asm__ volatile("" : "+v"(nothing));
    return r.row[n + nothing];
  }

  // The position of a new token of a tree: it sees itself and its ancestors.
  static __device__ __forceinline__ int key_position(const Rules &r, const Tile &t, uint32_t token) {
    const uint32_t n = (uint32_t)(t.len - t.base);
    const uint32_t *row = r.all.tree + (uint64_t)token * r.all.tree_words;
    uint32_t sees = 0;
    for (uint32_t w = 0; 32u * w < n; ++w) sees += __popc(row[w] & (n - 32u * w < 32u ? (1u << (n - 32u * w)) - 1u : ~0u));
    return t.base + (int)sees - 1;
  }

  // What the rows' scores and maxima are multiplied by: rules on the scores leave them in
  // units of log2.
  __device__ __forceinline__ float of_scores(const Rules &r) const {
    if constexpr (RULES) return r.all.cap > 0.f || r.all.slopes ? 1.f : sc;
    else return sc;
  }

  // The scores of a step under the rules, from the raw ones.
  __device__ __forceinline__ void rule(const Rules &r, const Tile &t, int t0, uint32_t n, uint32_t g, float s[2][4]) const {
    if constexpr (RULES) {
      if (r.all.cap > 0.f) {
        // finite, so that a raw score of 0 stays 0, and not less than that: int8 keys may have raw
        // scores of 1e-32 that are far past the cap
        const float to_z = fminf(sc * r.all.per_cap, 0x1.fffffep127f), most = r.all.cap;
        float top = 0.f;
#pragma unroll
        for (int k = 0; k < 8; ++k) top = fmaxf(top, fabsf(s[k / 4][k % 4]));
        if (__any(top * to_z >= kTanhFew)) {
          // 1 - 2 / (1 + e^2z), and the odd polynomial below kTanhFew, where that loses bits
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            float &y = s[k / 4][k % 4];
            const float z = y * to_z, e = __builtin_amdgcn_exp2f(fabsf(z) * 2.88539008177792681f);
            const float far = copysignf(fmaf(-2.f, __builtin_amdgcn_rcpf(1.f + e), 1.f), z);
            // a raw score that is not finite stays so; a small one has the same bits whatever the
            // others are, which its row may not see
            y = fabsf(z) < kTanhFew ? y * sc * tanh_few(z * z) : fmaf(y, 0.f, far * most);
          }
        } else {
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            float &y = s[k / 4][k % 4];
            const float z = y * to_z;
            y = y * sc * tanh_few(z * z);
          }
        }
      } else if (r.all.slopes) {
#pragma unroll
        for (int k = 0; k < 8; ++k) s[k / 4][k % 4] *= sc;
      }
      if (r.all.slopes) {
        const AttnRule row = get_rule(r, n);
        if (r.all.tree && t0 + 32 > t.base) {
#pragma unroll 1
          for (int k = 0; k < 8; ++k) {
            const int at = t0 + 16 * (k / 4) + 4 * (int)g + k % 4;
            const int key = at >= max(t.base, 0) && at < t.len ? key_position(r, t, t.token0 + (uint32_t)(at - t.base)) : at;
            const float bias = -row.slope * fabsf((float)(row.pos - key));
#pragma unroll
            for (int i = 0; i < 8; ++i) s[i / 4][i % 4] += i == k ? bias : 0.f;
          }
        } else {
          const float far = (float)(row.pos - t0 - 4 * (int)g);
#pragma unroll
          for (int k = 0; k < 8; ++k) s[k / 4][k % 4] = fmaf(-row.slope, fabsf(far - (float)(16 * (k / 4) + k % 4)), s[k / 4][k % 4]);
        }
      }
    }
  }
  static __device__ __forceinline__ float tanh_few(float u) {
    float p = kTanh[5];
#pragma unroll
    for (int i = 4; i >= 0; --i) p = fmaf(p, u, kTanh[i]);
    return p;
  }

  // Of the 32 tokens of a step those that row n sees, a bit each; none without a page.
  static __device__ __forceinline__ uint32_t seen_bits(const Rules &r, const Tile &t, int t0, uint32_t n, const bool gone[2]) {
    const AttnRule row = get_rule(r, n);
    const int lo = min(max(row.from - t0, 0), 32), hi = min(max(row.to - t0, 0), 32);
    uint32_t m = (uint32_t)((1ull << hi) - 1ull) & ~(uint32_t)((1ull << lo) - 1ull);
    if (r.all.tree && t0 + 32 > t.base && n < t.rows) {
      // the bits of the tree begin at token base
      const uint32_t *bits = r.all.tree + (uint64_t)(t.token0 + (t.r0 + n) / r.group) * r.all.tree_words;
      const int j = t0 - t.base;
      const auto word = [&](uint32_t w) { return w < r.all.tree_words ? bits[w] : 0u; };
      m &= j >= 0 ? (uint32_t)(((uint64_t)word((uint32_t)j / 32u + 1u) << 32 | word((uint32_t)j / 32u)) >> (j & 31))
                  : word(0u) << -j | ((1u << -j) - 1u);
    }
    if (gone[0]) m &= 0xFFFF0000u;
    if (gone[1]) m &= 0x0000FFFFu;
    return m;
  }

  // q in its two fp16 parts, and empty sums. Rows that are none see nothing
  // (pos -1), so what q they have does not matter.
  __device__ __forceinline__ void init(const float q[KS][8], float scale, uint8_t *lds, uint32_t wave, uint32_t waves) {
    qs = lds + 16u * (threadIdx.x & 63u);
    float top = 0.f;
#pragma unroll
    for (int c = 0; c < KS; ++c)
#pragma unroll
      for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(q[c][i]));
    top = row_max(top);
    const int e = min(max((int)(__float_as_uint(top) >> 23) - 127, -100), 127);
    // the scale's sign goes to q; a scale of zero makes every score zero
    const float up = scale == 0.f ? 0.f : copysignf(ldexpf(1.f, 13 - e), scale);
    sc = fmaxf(fabsf(scale) * 1.44269504088896341f * ldexpf(1.f, e - 13), 1e-37f);
#pragma unroll
    for (int c = 0; c < KS; ++c) {
      half2v hi[4], lo[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) split2(q[c][2 * i] * up, q[c][2 * i + 1] * up, hi[i], lo[i]);
      const half8 h = join8(hi), r = join8(lo);
      if constexpr (!QL) {
        qh[c] = h, ql[c] = r;
      } else if (c % waves == wave) {
        *(half8 *)(const_cast<uint8_t *>(qs) + c * 2048) = h;
        *(half8 *)(const_cast<uint8_t *>(qs) + c * 2048 + 1024) = r;
      }
    }
    m = -INFINITY, l = 0.f, unit = 0.f, inv = 0.f;
#pragma unroll
    for (int i = 0; i < E; ++i) acc[i] = float4v{0.f, 0.f, 0.f, 0.f};
  }

  // K of the 16 tokens from p on, into half u of the step.
  __device__ __forceinline__ void load_k(int u, const uint8_t *p, const uint8_t *scales, uint32_t n, uint32_t g) {
    if constexpr (!I8) {
#pragma unroll
      for (int c = 0; c < KS; ++c) ld_cache<4>(kw[u] + 4 * c, p + (n * ROW + 16u * g) + 64u * c);
    } else {
#pragma unroll
      for (int c = 0; c + 1 < KS; c += 2) ld_cache<4>(kw[u] + 2 * c, p + (n * ROW + 16u * g) + 32u * c);
      if constexpr (KS & 1) ld_cache<2>(kw[u] + 2 * (KS - 1), p + (n * ROW + 8u * g) + 32u * (KS - 1));
      ld_cache<4>(ks[u], scales + 16u * g);
    }
  }

  // V of the same tokens: the lane's columns of the rows 4 g .. 4 g + 3.
  __device__ __forceinline__ void load_v(int u, const uint8_t *p, const uint8_t *scales, uint32_t n, uint32_t g) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint8_t *r = p + 4u * g * ROW + j * ROW;
      uint32_t *o = vw[4 * u + j];
      if constexpr (D == 96 && I8) {
        o[0] = *(cached<uint32_t>)(r + 4u * n);
        o[1] = *(cached<uint16_t>)(r + 64 + 2u * n);
      } else if constexpr (D == 96) {
        ld_cache<2>(o, r + 8u * n);
        o[2] = *(cached<uint32_t>)(r + 128 + 4u * n);
      } else if constexpr (VW == 8) {
        ld_cache<4>(o, r + 32u * n);
        ld_cache<4>(o + 4, r + 32u * n + 16);
      } else {
        ld_cache<VW>(o, r + 4u * VW * n);
      }
    }
    if constexpr (I8) ld_cache<4>(vs[u], scales + 16u * g);
  }

  // Column i of the 8 tokens of the lane as the first operand.
  __device__ __forceinline__ u32x4 v_operand(int i) const {
    u32x4 o;
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      if constexpr (VIN == kVTurned) {
        o[x] = vw[i][x];
      } else if constexpr (I8) {
        const uint32_t w = i / 4, k = i % 4;
        const uint32_t sel = 0x0C000C00u | k | ((4u + k) << 16);
        o[x] = i8_half2(__builtin_amdgcn_perm(vw[2 * x + 1][w] ^ 0x80808080u, vw[2 * x][w] ^ 0x80808080u, sel) | 0x64006400u);
      } else {
        o[x] = __builtin_amdgcn_perm(vw[2 * x + 1][i / 2], vw[2 * x][i / 2], i & 1 ? 0x07060302u : 0x05040100u);
      }
    }
    return o;
  }

  // Takes out of V what is not finite.
  __device__ __forceinline__ void clean_v() {
#pragma unroll
    for (int k = 0; k < VN; ++k)
#pragma unroll
      for (int w = 0; w < VM; ++w) vw[k][w] &= ~not_finite_halves(vw[k][w]);
  }

  // Takes the tokens out of V whose halves of `keep` are 0.
  __device__ __forceinline__ void keep_v(u32x4 keep) {
    if constexpr (VIN == kVTurned) {
#pragma unroll
      for (int i = 0; i < E; ++i)
#pragma unroll
        for (int x = 0; x < 4; ++x) vw[i][x] &= keep[x];
    } else if constexpr (VIN == kVRows) {
#pragma unroll
      for (int k = 0; k < 8; ++k)
#pragma unroll
        for (int w = 0; w < VW; ++w) vw[k][w] = (keep[k / 2] >> 16 * (k & 1) & 1u) ? vw[k][w] : 0u;
    }
  }

  // Matrix step k's operand of the 16 tokens of half u.
  __device__ __forceinline__ half8 k_operand(int u, int k) const {
    if constexpr (I8) return i8_half8(kw[u][2 * k], kw[u][2 * k + 1]);
    else return __builtin_bit_cast(half8, u32x4{kw[u][4 * k], kw[u][4 * k + 1], kw[u][4 * k + 2], kw[u][4 * k + 3]});
  }

  // The step's raw scores: s[u][j] of token 16 u + 4 g + j. The two halves in turn,
  // so that a matrix step does not wait for the one before it.
  __device__ __forceinline__ void scores(float s[2][4]) const {
    float4v c[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
    uint32_t nothing = 0;
    if constexpr (QL) __asm__ volatile("" : "+v"(nothing));   // q is read here, not kept from step to step
    const uint8_t *parts = qs + nothing;
#pragma unroll
    for (int k = 0; k < KS; ++k) {
      half8 a[2];
#pragma unroll
      for (int u = 0; u < 2; ++u) a[u] = k_operand(u, k);
      half8 h, r;
      if constexpr (QL) h = *(const half8 *)(parts + k * 2048), r = *(const half8 *)(parts + k * 2048 + 1024);
      else h = qh[k], r = ql[k];
#pragma unroll
      for (int u = 0; u < 2; ++u) c[u] = mfma(a[u], h, c[u]);
#pragma unroll
      for (int u = 0; u < 2; ++u) c[u] = mfma(a[u], r, c[u]);
    }
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int j = 0; j < 4; ++j) s[u][j] = SCALED ? c[u][j] * __uint_as_float(ks[u][j]) : c[u][j];
  }

  static __device__ __forceinline__ bool sees(int pos, int window, int t) { return t <= pos && (window == 0 || t > pos - window); }

  // The weights of the step at token t0, and the weighted sum; v(i) is V's operand of
  // column i, scales(u) the lane's value scales of half u. `masked`: some row does not
  // see every one of its 32 tokens (wave-uniform); a half without a page is `gone`.
  // A score of -inf says that a row does not see the token. That of a token it sees is
  // -inf where the key is not finite (or the score passes f32): the row's sum becomes
  // NaN, as it does with +inf.
  template <typename V, typename S>
  __device__ __forceinline__ void step(int t0, bool masked, const bool gone[2], const Tile &t, int window, const Rules &r, uint32_t n, uint32_t g, float s[2][4], V v, S scales) {
    u32x4 keep = {~0u, ~0u, ~0u, ~0u};   // the halves of an operand whose token some row sees
    bool dirty = false;                  // and whether some of them are not finite
    half8 ph, pl;
    weights(t0, masked, gone, t, window, r, n, g, s, v, scales, keep, dirty, ph, pl);
    if (VIN == kVLater && !SCALED && masked) {
#pragma unroll
      for (int i = 0; i < E; ++i) {
        u32x4 o = v(i) & keep;
        if (dirty) {
#pragma unroll
          for (int x = 0; x < 4; ++x) o[x] &= ~not_finite_halves(o[x]);
        }
        acc[i] = mfma(__builtin_bit_cast(half8, o), ph, acc[i]);
        acc[i] = mfma(__builtin_bit_cast(half8, o), pl, acc[i]);
        __builtin_amdgcn_sched_barrier(0);
      }
      return;
    }
#pragma unroll
    for (int i = 0; i < E; ++i) {
      const half8 o = __builtin_bit_cast(half8, v(i));
      acc[i] = mfma(o, ph, acc[i]);
      acc[i] = mfma(o, pl, acc[i]);
    }
  }

  // The step's weights, in their two parts; what no row sees of V is taken out (by the
  // product itself where V is read as it is used).
  template <typename V, typename S>
  __device__ __forceinline__ void weights(int t0, bool masked, const bool gone[2], const Tile &t, int window, const Rules &r, uint32_t n, uint32_t g,
                                          float s[2][4], V v, S scales, u32x4 &keep, bool &dirty, half8 &ph, half8 &pl) {
    rule(r, t, t0, n, g, s);
    const float sc = of_scores(r);
    uint32_t bits = 0;
    float low = 0.f;                     // the smallest score that the row sees (a NaN hides it: no matter)
    if (masked) {
      if constexpr (RULES) bits = seen_bits(r, t, t0, n, gone) >> (4u * g);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int at = t0 + 16 * (k / 4) + 4 * (int)g + k % 4;
        float &y = s[k / 4][k % 4];
        const bool seen = RULES ? bits >> (16 * (k / 4) + k % 4) & 1u : !gone[k / 4] && sees(pos, window, at);
        low = seen ? __builtin_elementwise_minimum(low, y) : low;
        y = seen ? y : -INFINITY;
        // what no row sees may be any bits (int8 are numbers whatever they are)
        if (!SCALED && (gone[k / 4] || at < t.begin || at >= t.end)) keep[k / 2] &= k & 1 ? 0x0000FFFFu : 0xFFFF0000u;
      }
      // A value that only some rows see and that is not finite: 0 * inf would
      // reach the others. (int8 values are finite, and their scales go with the weights.)
      if constexpr (!SCALED) {
        keep_v(keep);
        if (unlike(t, r)) {
          uint32_t most = 0;
          short2v both = {0, 0};   // under rules two at a time: no number's magnitude is negative
#pragma unroll
          for (int i = 0; i < (VIN == kVLater ? E : VN * VM / 4); ++i) {
            u32x4 o;
            if constexpr (VIN == kVLater) o = v(i) & keep;
            else
#pragma unroll
              for (int x = 0; x < 4; ++x) o[x] = vw[(4 * i + x) / VM][(4 * i + x) % VM];
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              if constexpr (RULES) both = __builtin_elementwise_max(both, __builtin_bit_cast(short2v, o[x] & 0x7FFF7FFFu));
              else most = max(most, max(o[x] & 0x7FFFu, o[x] >> 16 & 0x7FFFu));
            }
            __builtin_amdgcn_sched_barrier(0);   // one column's registers at a time
          }
          if constexpr (RULES) most = (uint32_t)max(both[0], both[1]);
          dirty = __any(most >= 0x7C00u);
          if constexpr (RULES) {
            if (dirty) spoil(bad_tokens(keep, v), bits);
            if (dirty && VIN != kVLater) clean_v();
          } else {
            if (dirty) poison(t0, gone, window, g, keep, v);
          }
        }
      }
    } else {
      low = min8(s);
    }
    const float mx = row_max(max8(s));
    if (__any(mx > m)) {
      const float mn = fmaxf(m, mx);
      const float f = m == mn ? 1.f : __builtin_amdgcn_exp2f((m - mn) * sc);
      m = mn;
      l *= f;
      if constexpr (SCALED) {
        unit *= f;
        inv = 1.f / unit;
      } else {
#pragma unroll
        for (int i = 0; i < E; ++i) acc[i] *= f;
      }
    }
    const float up = m == -INFINITY ? 0.f : RAISED ? 14.f - m * sc : -(m * sc);
    float sum = low == -INFINITY ? NAN : 0.f;
    float p[8];
    u32x4 scale = {};
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      if (SCALED && k % 4 == 0) scale = scales(k / 4);
      const float y = s[k / 4][k % 4];
      p[k] = __builtin_amdgcn_exp2f(fmaf(y, sc, up));
      if constexpr (!SCALED && !RAISED) p[k] *= 0x1p14f;
      sum += p[k];
      // a weight of nothing takes nothing of a scale that is not finite
      if constexpr (SCALED) p[k] = masked && y == -INFINITY ? 0.f : p[k] * __uint_as_float(scale[k % 4]);
    }
    l += sum;
    if constexpr (SCALED) {
      // the weights with their scales, in units that leave fp16 a factor of 2 to grow
      float top = 0.f;
#pragma unroll
      for (int k = 0; k < 8; ++k) top = fmaxf(top, fabsf(p[k]));
      if (__any(top * inv > 0x1p15f || unit < kLeastUnit)) {
        top = row_max(top);
        const float un = fmaxf(top * inv > 0x1p15f ? top * 0x1p-14f : unit, kLeastUnit), f = unit / un;
        unit = un;
        inv = 1.f / un;
#pragma unroll
        for (int i = 0; i < E; ++i) acc[i] *= f;
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) p[k] *= inv;
    }
    half2v hi[4], lo[4];
#pragma unroll
    for (int k = 0; k < 8; k += 2) split2(p[k], p[k + 1], hi[k / 2], lo[k / 2]);
    ph = join8(hi), pl = join8(lo);
  }

  // fp16 1 where a half is not finite, else 0.
  static __device__ __forceinline__ uint32_t not_finite(uint32_t w) {
    return ((w & 0x7C00u) == 0x7C00u ? 0x3C00u : 0u) | ((w & 0x7C000000u) == 0x7C000000u ? 0x3C000000u : 0u);
  }

  // All bits of such a half.
  static __device__ __forceinline__ uint32_t not_finite_halves(uint32_t w) { return not_finite(w) / 0x3C00u * 0xFFFFu; }

  // The columns of the rows that see a value that is not finite become NaN (the
  // product of the two indicators says which), and such values are taken out of the
  // step (by the product itself where V is read as it is used).
  template <typename V>
  __device__ __forceinline__ void poison(int t0, const bool gone[2], int window, uint32_t g, u32x4 keep, V v) {
    half8 seen;
#pragma unroll
    for (int k = 0; k < 8; ++k) seen[k] = (_Float16)(!gone[k / 4] && sees(pos, window, t0 + 16 * (k / 4) + 4 * (int)g + k % 4) ? 1.f : 0.f);
#pragma unroll
    for (int i = 0; i < E; ++i) {
      const u32x4 o = v(i) & keep;
      const u32x4 bad = {not_finite(o[0]), not_finite(o[1]), not_finite(o[2]), not_finite(o[3])};
      const float4v c = mfma(__builtin_bit_cast(half8, bad), seen, float4v{0.f, 0.f, 0.f, 0.f});
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[i][j] = c[j] > 0.f ? NAN : acc[i][j];
      __builtin_amdgcn_sched_barrier(0);   // one column's registers at a time
    }
    if constexpr (VIN != kVLater) clean_v();
  }

  // Under rules the whole row becomes NaN (its sum does: no second set of the columns'
  // registers is needed for that). Of the lane's 8 tokens those that have a value which
  // is not finite, a bit each:
  template <typename V>
  __device__ __forceinline__ uint32_t bad_tokens(u32x4 keep, V v) const {
    uint32_t bad = 0;
#pragma unroll
    for (int i = 0; i < E; ++i) {
      const u32x4 o = v(i) & keep;
#pragma unroll
      for (int k = 0; k < 8; ++k) bad |= (o[k / 2] >> 16 * (k & 1) & 0x7C00u) == 0x7C00u ? 1u << k : 0u;
      __builtin_amdgcn_sched_barrier(0);   // one column's registers at a time
    }
    bad |= (uint32_t)__builtin_amdgcn_update_dpp(0, (int)bad, 0xB1, 0xF, 0xF, false);
    bad |= (uint32_t)__builtin_amdgcn_update_dpp(0, (int)bad, 0x4E, 0xF, 0xF, false);
    bad |= (uint32_t)__builtin_amdgcn_update_dpp(0, (int)bad, 0x141, 0xF, 0xF, false);
    bad |= (uint32_t)__builtin_amdgcn_update_dpp(0, (int)bad, 0x140, 0xF, 0xF, false);
    return bad;
  }
  // bits: of the tokens 4 g .. of the two halves those that the row sees.
  __device__ __forceinline__ void spoil(uint32_t bad, uint32_t bits) {
    if (bad & ((bits & 0xFu) | (bits >> 12 & 0xF0u))) l = NAN;
  }

  // Whether a token that some row of the tile sees may be one that another does not: not
  // where they are one token's, but for the drafts of a tree that it does not see.
  static __device__ __forceinline__ bool unlike(const Tile &t, const Rules &r) {
    if constexpr (RULES) return t.first != t.last || r.all.tree;
    else return t.first != t.last;
  }
  static __device__ __forceinline__ int full_of(const Tile &t) {
    if constexpr (RULES) return t.all_to - 32;
    else return t.first - 31;
  }
  static __device__ __forceinline__ int from_of(const Tile &t, int window) {
    if constexpr (RULES) return t.all_from;
    else return window ? t.last - window + 1 : 0;
  }

  // The steps of `k`, whose first keys are on their way (fetch_k). The last one is on
  // its own: behind a branch that may or may not ask for the next keys, a wait for V
  // would be one for whatever is under way.
  __device__ __forceinline__ void run(AttnWalk &k, const KvView &kv, const Tile &t, int window, const Rules &r, uint32_t n, uint32_t g) {
    int t0 = k.lo, i = 0;
    if (t0 >= k.hi) return;
#pragma unroll 1
    for (; t0 + k.stride < k.hi; t0 += k.stride, ++i) one<false>(k, kv, t, window, r, n, g, t0, i);
    one<true>(k, kv, t, window, r, n, g, t0, i);
  }

  template <bool LAST>
  __device__ __forceinline__ void one(AttnWalk &k, const KvView &kv, const Tile &t, int window, const Rules &r, uint32_t n, uint32_t g, int t0, int i) {
    const uint32_t to_v = kv.heads * kv.block_bytes;
    const int full = full_of(t), from = from_of(t, window);   // steps from .. full need no mask
#pragma unroll
    for (int u = 0; u < 2; ++u) load_v(u, k.at[u] + to_v, k.scales(u, kv, D) + to_v, n, g);
    __builtin_amdgcn_sched_barrier(0);   // requested before the scores
    float s[2][4];
    scores(s);
    const bool gone[2] = {k.gone[0], k.gone[1]};
    const bool masked = gone[0] || gone[1] || t0 > full || t0 < from;
    if constexpr (!LAST) {
      fetch_k(k, kv, i + 1, n, g);
      __builtin_amdgcn_sched_barrier(0);
    }
    step(t0, masked, gone, t, window, r, n, g, s, [&](int c) { return v_operand(c); },
         [&](int u) { return u32x4{vs[u][0], vs[u][1], vs[u][2], vs[u][3]}; });
  }

  __device__ __forceinline__ void fetch_k(AttnWalk &k, const KvView &kv, int i, uint32_t n, uint32_t g) {
    k.go<ROW>(kv, i);
#pragma unroll
    for (int u = 0; u < 2; ++u) load_k(u, k.at[u], k.scales(u, kv, D), n, g);
  }
};

struct AttnPlan {
  uint32_t tiles, per_seq;    // row tiles; tiles of each sequence (0: packed)
  uint32_t items;             // workgroups of a head that share the cached tokens (0: one a tile)
  bool on;                    // a share may go on into the next tile
  uint32_t rows;              // rows of a tile at most
  uint32_t waves;             // of a workgroup
  uint32_t max_rows;          // of the sequences taken; those with more go to k_attn_rows:
  uint32_t many_tiles, many_per_seq;   // its tiles (0: none go), shared by `items` workgroups where there are no others
};

// The sums of a tile that several workgroups share: each has two slots for a head, for
// the tile that it begins in and for the one that it ends in, of `rows` rows'
// weighted sums and their maxima and sums.
__host__ __device__ constexpr uint32_t attn_part_floats(const AttnPlan &p, uint32_t dim) { return p.rows * (dim + 2u); }

constexpr uint32_t kFewRows = 64;
// Values that one join reads: of more than these it takes longer than the second round
// trip of two (32 workgroups x 8 rows x 128: 14.7 us, in two 15.3; 64 x 8 x 128 22.3 and
// 20.3; 128 x 8 x 128 40.9 and 26.9).
constexpr uint32_t kJoin = 32768;
// Of tiles of 64 rows: round trips of one join, and workgroups of a head, of which either
// step of two joins then has at most 32 (the LDS of 64 wide).
constexpr uint32_t kJoinRows = 5, kItemsRows = 1024, kJoinSide = 32;
constexpr int kSc1 = 16;   // cache policy bit 4: sc1, past the XCD's own L2

enum { kAttnWhole, kAttnEnds, kAttnOn };   // a workgroup has a tile; a part of one; a share that may go on into the next

// A wave's copy of what a workgroup has in LDS, in scalar registers.
template <typename T>
__device__ __forceinline__ void from_lds(T &to, const T &from) {
  uint32_t w[sizeof(T) / 4];
  __builtin_memcpy(w, &from, sizeof(T));
#pragma unroll
  for (uint32_t i = 0; i < sizeof(T) / 4; ++i) w[i] = __builtin_amdgcn_readfirstlane(w[i]);
  __builtin_memcpy(&to, w, sizeof(T));
}

// Joins the sums of a tile that several workgroups share, `chunks` of them from workgroup
// `first` on: the last of them to arrive adds all up, of more than kJoin values in two
// steps, groups first. Every wave's own sums lie in its slot, stored past the XCD's L2.
// LDS: wt as many floats as one step has workgroups times rows, half 4 T, sm and sl a
// float a row.
template <int D, uint32_t T, typename TILE>
__device__ __forceinline__ void attn_join(const AttnPlan &p, rsrc_t prs, uint32_t *cnt, const KvAttnArgs &a, const TILE &t, uint32_t group,
                                          uint32_t kvh, uint32_t item, uint32_t first, uint32_t chunks, float *wt, float *half, float *sm,
                                          float *sl, uint32_t &arrived, uint32_t slot_floats, uint32_t ml, uint32_t tid, uint32_t lane, uint32_t wave) {
  const auto place = [&](uint32_t z) { return 2u * (first + z) + (z == 0u ? 1u : 0u); };   // the slot of the tile's workgroup z
  // one join, or where there is much to read, one of each group of about sqrt(chunks)
  // workgroups, whose sums take its first one's slot, and one of the groups
  const uint32_t side = chunks * p.rows * D <= kJoin ? chunks : __builtin_amdgcn_readfirstlane((uint32_t)ceilf(sqrtf((float)chunks)));
  const uint32_t groups = (chunks + side - 1u) / side;
  uint32_t z0 = (item - first) / side * side, step = 1u, count = min(side, chunks - z0);
  for (bool last = groups == 1u;; last = true) {
    __asm__ volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    uint32_t *counter = cnt + (step == 1u ? 0u : kAttnCounters / 2u) + (uint64_t)kvh * p.items * 2u + place(z0);
    if (tid == 0u) arrived = __hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();
    if (arrived != count - 1u) break;
    if (tid == 0u) __hip_atomic_store(counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    // each thread a part of the workgroups' 4 columns of a row, U of them under way,
    // the first before the weights are known
    constexpr uint32_t U = 8;
    const uint32_t pieces = t.rows * (D / 4u), parts = max(1u, T / pieces);
    const uint32_t part_i = parts > 1u ? tid / pieces : 0u, p0 = parts > 1u ? tid % pieces : tid;
    float4v x[U] = {};   // (else live from tile to tile)
    const auto request = [&](uint32_t i, uint32_t z) {
#pragma unroll
      for (uint32_t k = 0; k < U; ++k) {
        const uint32_t at = place(z0 + step * min(z + k * parts, count - 1u)) * slot_floats + i / (D / 4u) * D + 4u * (i % (D / 4u));
        x[k] = __builtin_bit_cast(float4v, __builtin_amdgcn_raw_buffer_load_b128(prs, (int)(at * 4u), 0, kSc1));
      }
    };
    if (p0 < pieces && part_i < parts) request(p0, part_i);
    // the workgroups' weights relative to the largest maximum, [workgroup][row],
    // and the rows' sums: a wave per row, its lanes over the workgroups
    for (uint32_t r = wave; r < t.rows; r += T / 64u) {
      const auto both = [&](uint32_t z, float &mz, float &lz) {
        const int at = (int)((place(z0 + step * z) * slot_floats + ml + 2u * r) * 4u);
        mz = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(prs, at, 0, kSc1));
        lz = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(prs, at + 4, 0, kSc1));
      };
      float m0 = -INFINITY, l0 = 0.f, mz, lz;
      if (lane < count) both(lane, m0, l0);
      float mx = m0, l = 0.f;
      for (uint32_t z = lane + 64u; z < count; z += 64u) both(z, mz, lz), mx = fmaxf(mx, mz);
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) mx = fmaxf(mx, __shfl_xor(mx, o));
      for (uint32_t z = lane; z < count; z += 64u) {
        if (z < 64u) mz = m0, lz = l0;
        else both(z, mz, lz);
        const float f = mz == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mz - mx);
        wt[z * p.rows + r] = f;
        l += f * lz;
      }
      l = wave_sum(l);
      if (lane == 0u) sl[r] = l, sm[r] = mx;
    }
    __syncthreads();
    for (uint32_t i = p0; i < (parts > 1u ? p0 + 1u : (pieces + T - 1u) / T * T); i += T) {
      const bool here = i < pieces && part_i < parts;
      const uint32_t r = here ? i / (D / 4u) : 0u, d = 4u * (i % (D / 4u));
      float4v o = {0.f, 0.f, 0.f, 0.f};
      if (here) {
        for (uint32_t z = part_i; z < count; z += U * parts) {
          if (i != p0 || z != part_i) request(i, z);
#pragma unroll
          for (uint32_t k = 0; k < U; ++k)
            if (z + k * parts < count) o += x[k] * wt[(z + k * parts) * p.rows + r];
        }
      }
      if (parts > 1u) {
        *(float4v *)(half + 4u * tid) = o;
        __syncthreads();
        if (here && part_i == 0u)
          for (uint32_t k = 1; k < parts; ++k) o += *(const float4v *)(half + 4u * (tid + k * pieces));
      }
      if (!here || part_i != 0u) continue;
      const float l = sl[r];
      if (last) {
        const uint32_t tok = (t.r0 + r) / group, h = (t.r0 + r) % group;
        float *dst = a.out + ((uint64_t)(t.token0 + tok) * a.q_heads + kvh * group + h) * D + d;
        *(float4v *)dst = l == 0.f ? float4v{0.f, 0.f, 0.f, 0.f} : o / l;
      } else {
        const uint32_t at = place(z0) * slot_floats;
        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, o), prs, (int)((at + r * D + d) * 4u), 0, kSc1);
        if (d == 0u) {
          // a sum that is not a number is not nothing
          const float mx = sm[r] == -INFINITY && l != 0.f ? 0.f : sm[r];
          __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(mx), prs, (int)((at + ml + 2u * r) * 4u), 0, kSc1);
          __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(l), prs, (int)((at + ml + 2u * r + 1u) * 4u), 0, kSc1);
        }
      }
    }
    if (last) break;
    z0 = 0u, step = side, count = groups;
  }
}

// Few rows: NW waves take the 32-token steps of a tile in turn; their sums meet in
// LDS. Where a tile has several workgroups, the last of them to arrive joins their
// sums, in the tokens' order, so that the bits do not depend on who was last (many in
// two steps, groups first); stores and loads of these go past the XCD's L2 (sc1), every
// wave waits for its stores before the barrier ahead of the counter's increment, and
// the counters are left at zero for the next launch.
//
// The cache's bytes bound a batch: K and V go from memory to the registers that the
// matrix unit reads, a step of V and the next step of K under way in each wave, 16 KB
// of fp16 rows of 128, 64 KB a CU and more (64 sequences up to 16384 long, 32 heads of
// 128 on 8: 358 us, 5.9 TB/s; one of 130001: 95 us, 5.6 TB/s). The matrix unit is busy
// 8 % of the time there, so the second parts of q and p are free. int8 rows are half
// the bytes with as many instructions, which shows where the shares are short (40 up
// to 9001, 16 heads of 256 on 2: 43 to 46 us, 3.6 to 3.9 TB/s). A single short sequence
// is round trips: lengths, page table, K, V, the join (517 tokens: 6.3 to 6.8 us, an
// empty launch 3.4). Under rules: 48 up to 8192, 16 heads of 256 on 8, capped, 319 us, 5.7
// TB/s; one of 20001, 32 heads of 128 with slopes, 60 us, 5.5 TB/s; int8 trees of up to 6
// drafts (48 rows, three tiles) over 4096 of up to 9001, 16 heads of 256 on 2, 65 us: each
// tile reads and converts the keys and values for itself, and what another has read is
// seldom left in its L2, so that 297 MB come where the caches have 142, at 4.6 TB/s, 88 % of
// a large copy's rate; the VALU is busy 53 % of the time with 1.6 waves a SIMD. Shares that
// go on keep 32 to 52 scalar registers in vector ones (under rules 71 to 85; fp16 256 wide
// has 3 vector ones in scratch for that, under rules 5), outside the steps.
template <int TYPE, int D, int NW, int MODE, typename RULES>
__global__ __launch_bounds__(64 * NW, NW == 8 ? 1 : 2) void k_attn(KvView kv, KvBatchView b, KvAttnArgs a, AttnPlan p, uint32_t *cnt, float *part, RULES rules) {
  constexpr bool I8 = TYPE == EFF_KV_I8, QL = D == 256;   // 256 wide, q's parts would take a quarter of the registers
  constexpr bool RULED = !__is_same(RULES, NoRules);
  using W = AttnWave<D, I8, I8, QL, kVRows, RULED>;
  constexpr uint32_t R = 16u, LD = D + 4u, T = 64u * NW;
  static_assert(!QL || W::KS * 2048u <= NW * R * LD * 4u, "q's parts share the sums' space");
  static_assert(MODE == kAttnWhole || kUnit == 32u * NW, "a unit is a step of each wave");
  __shared__ float so[NW][R][LD];
  __shared__ float sm[NW][R], sl[NW][R], sv[NW][R];
  __shared__ AttnRule rule_rows[RULED ? NW : 1u][RULED ? R : 1u];
  __shared__ uint32_t arrived;
  __shared__ typename W::Tile kept_t;
  __shared__ AttnShare kept_c;
  const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = __builtin_amdgcn_readfirstlane(tid >> 6), n = lane & 15u, g = lane >> 4;
  const uint32_t group = a.q_heads / kv.heads;
  const uint32_t kvh = blockIdx.x % kv.heads, item = blockIdx.x / kv.heads;
  const int window = (int)min(a.window, 0x40000000u);
  constexpr bool shared = MODE != kAttnWhole, on = MODE == kAttnOn;
  uint32_t tree = 0;   // new tokens of a tree at most
  if constexpr (RULED) tree = rules.tree ? min(b.max_new, b.tokens) : 0u;
  typename W::Tile t;
  AttnShare c = {1u, 1u, 0u, 1u, 0u, 0u};
  if constexpr (shared) {
    if (!attn_share<R, !on>(b, group, a.window, tree, item, p.items, p.max_rows, t, c)) return;
  } else {
    if (!attn_tile<R>(b, group, a.window, item, p.per_seq, 1u, p.max_rows, t)) return;
  }
  for (;;) {
    int from = 0, to = 0;   // lane n: row n's range
    if constexpr (RULED) attn_range(t, rules, group, n, from, to);
    attn_seen<R>(t, rules, window, from, to);
    const int base = t.begin & ~31;
    int lo = base, hi = t.end;
    if (shared) {
      lo = base + (int)(c.at * kUnit);
      hi = min(base + (int)(min(c.at + c.left, c.of) * kUnit), t.end);
      // the steps take all scalar registers: the rest waits in LDS
      if (on && tid == 0u) kept_t = t, kept_c = c;
    }
    const bool mine = lo < hi || lo == base;   // past the end the tile's other workgroups have it all
    if (mine) {
      W w;
      const auto wr = attn_rules(rules, rule_rows[RULED ? wave : 0u], group);
      {
        AttnWalk k;
        k.table = b.table + (uint64_t)t.seq * b.table_pages;
        k.heads = kv.base + (uint64_t)kvh * kv.block_bytes;
        k.lo = lo + 32 * (int)wave, k.hi = hi, k.stride = 32 * NW;
        float q[W::KS][8];
        w.load_q(q, a, t, group, kvh, n, g);
        w.fetch_k(k, kv, 0, n, g);   // of the first page, where the wave has no step
        w.init(q, a.scale, (uint8_t *)so, wave, NW);
        W::put_rule(wr, t, kvh, n, g, window, from, to);
        if constexpr (QL) __syncthreads();
        w.run(k, kv, t, window, wr, n, g);
        if constexpr (QL) __syncthreads();   // the sums take q's place
      }
      const float wl = row_add(w.l);
      if (g == 0u) sm[wave][n] = w.m * w.of_scores(wr), sl[wave][n] = wl, sv[wave][n] = w.unit;
#pragma unroll
      for (int i = 0; i < W::E; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) so[wave][n][W::column(g, i, j)] = w.acc[i][j];
    }
    __syncthreads();
    uint32_t first = 0, chunks = 1;   // the tile's workgroups
    if (shared) {
      if constexpr (on) {
        from_lds(t, kept_t);
        from_lds(c, kept_c);
      }
      const int tokens = t.end - (t.begin & ~31);
      const uint32_t units = tokens > 0 ? ((uint32_t)tokens + kUnit - 1u) / kUnit : 1u;
      first = __builtin_amdgcn_readfirstlane(c.start / c.each);
      chunks = __builtin_amdgcn_readfirstlane((c.start + units - 1u) / c.each) - first + 1u;
    }
    // the head's slots: of a workgroup, the one of the tile that it begins in, then of
    // the tile that it ends in
    const uint32_t slot_floats = attn_part_floats(p, D), ml = p.rows * D;   // ml: where a slot's maxima and sums begin
    const rsrc_t prs = make_rsrc(part + (uint64_t)kvh * p.items * 2u * slot_floats, (uint64_t)p.items * 2u * slot_floats * 4u);
    const uint32_t slot = (2u * item + (item == first ? 1u : 0u)) * slot_floats;
    if (mine) {
      for (uint32_t i = tid; i < t.rows * (D / 4u); i += T) {
        const uint32_t r = i / (D / 4u), d = 4u * (i % (D / 4u));
        float mx = -INFINITY, l = 0.f;
#pragma unroll
        for (int v = 0; v < NW; ++v) mx = fmaxf(mx, sm[v][r]);
        float4v o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int v = 0; v < NW; ++v) {
          const float f = sm[v][r] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(sm[v][r] - mx);
          l += f * sl[v][r];
          const float4v x = *(const float4v *)&so[v][r][d];
          o += x * (I8 ? f * sv[v][r] : f);
        }
        if (!shared || chunks == 1u) {
          const uint32_t tok = (t.r0 + r) / group, h = (t.r0 + r) % group;
          float *dst = a.out + ((uint64_t)(t.token0 + tok) * a.q_heads + kvh * group + h) * D + d;
          *(float4v *)dst = l == 0.f ? float4v{0.f, 0.f, 0.f, 0.f} : o / l;
        } else {
          __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, o), prs, (int)((slot + r * D + d) * 4u), 0, kSc1);
          if (d == 0u) {
            __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(mx), prs, (int)((slot + ml + 2u * r) * 4u), 0, kSc1);
            __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(l), prs, (int)((slot + ml + 2u * r + 1u) * 4u), 0, kSc1);
          }
        }
      }
    }
    if (shared && mine && chunks > 1u) {
      float *wt = &so[0][0][0];
      attn_join<D, T>(p, prs, cnt, a, t, group, kvh, item, first, chunks, wt, wt + NW * R * LD - 4u * T, sm[0], sl[0], arrived, slot_floats, ml, tid, lane, wave);
    }
    if (!on || !attn_next<R>(b, group, a.window, tree, p.max_rows, t, c)) return;
    __syncthreads();   // the next tile's sums take these ones' place
  }
}

// Many rows: four waves of 16 rows each walk the same cached tokens, 32 a step,
// which come through LDS as fp16: two buffers, one filled while the other is read. A
// wave that has waited for its loads (or LDS writes) and passed the barrier knows that
// the step's tokens are there, and that every wave is done with the buffer it fills
// next. fp16 pages go straight to LDS; int8 ones are requested before the step and
// converted after it, once for the four waves.
// K's 16-byte pieces are turned within their row, and V's 32-byte ones, so that the
// rows of an operand lie in different banks (V's 16 all do; K's, turned by 8 places, two
// to a bank from 128 wide on, a third of the LDS's active cycles: with 16 places there
// were no conflicts, and 186 -> 185 us of the prompts below, 237 -> 232 of int8); V's
// operand comes out of LDS turned (ds_read_b64_tr_b16: of 16 lanes, lane 4 j + q reads 4
// values of row j, and lane c gets column c of the 4 rows).
//
// Under rules a tile may be shared by workgroups (kAttnEnds), each with its tokens, whose
// sums attn_join_rows adds up; q is read and split while the first step's tokens are on
// their way. Trees: 16 of up to 32 drafts over up to 16384, 32 heads of 128 on 8, 167 to 173
// us, 300 TFLOP/s of the product itself (600 with the second parts), where the cache's bytes
// alone take 109: the second tile of a long sequence reads a quarter again (702 MB of 557, 4.1
// TB/s), the VALU is busy 49 % and the matrix unit 37 % of the time with 2.45 waves a SIMD,
// and a wave does its matrix steps and its softmax in turn; none of these is a limit by
// itself. Prompts into which documents were packed, 2 x 2500 tokens: 63 us; a tile
// sees some ten steps there, a third of them masked, and the rest is its beginning (ranges,
// table, first tokens, q) and end. Three buffers were no faster with shared tiles either
// (105 us of 32 x 8 drafts over up to 8000: 118).
//
// Instruction issue bounds it: per step of 32 tokens x 16 rows x 128 a wave has 32
// matrix instructions of 16 cycles and 106 of the softmax, the operands and the walk of
// 4 and more, and three waves a SIMD overlap them to 44 and 37 % of the busy time (3 x
// 1000 new tokens at lengths up to 3001, 32 heads of 128 on 8: 181 to 190 us, 440
// TFLOP/s of the product itself, 880 with q's and p's second parts, where a large fp16
// product reaches 1090; of int8 239, where the conversions are VALU work too). Three
// buffers, two steps ahead, were no faster (185 us): the loads are not waited for. Vector
// registers in scratch: 9 of int8 256 wide, fp16 none; under rules 10 and, shared, 13 of
// fp16 256 wide, 20 of int8, 2 of fp16 128 wide shared, 4 of int8.
template <int D>
struct AttnStage {
  static constexpr uint32_t ROW = 2 * D, PIECES = ROW / 16u;
  static constexpr uint32_t FILLS = ROW / 64u;                // loads of 64 x 16 bytes for 16 rows
  static constexpr uint32_t HALF = 16u * ROW;
  static constexpr uint32_t V = 2u * HALF, SCALES = 2u * V, BYTES = 2u * V + 256u;

  // where piece c of K's row r lies in the row, and what lies there
  static __device__ __forceinline__ uint32_t place(uint32_t r, uint32_t c) {
    return PIECES % 8u == 0u ? c ^ (r & 7u) : (c + (r >> 1 & 3u)) % PIECES;
  }
  static __device__ __forceinline__ uint32_t piece(uint32_t r, uint32_t at) {
    return PIECES % 8u == 0u ? at ^ (r & 7u) : (at + PIECES - (r >> 1 & 3u)) % PIECES;
  }
  // the same of the 16 columns c of V's row r
  static __device__ __forceinline__ uint32_t v_place(uint32_t r, uint32_t c) {
    return PIECES >= 16u ? c ^ (r & 7u) : PIECES == 8u ? c ^ (r >> 1 & 3u) : (c + (r >> 2 & 3u)) % (PIECES / 2u);
  }
  static __device__ __forceinline__ uint32_t v_piece(uint32_t r, uint32_t at) {
    const uint32_t c = at / 2u;
    return (PIECES >= 16u ? c ^ (r & 7u) : PIECES == 8u ? c ^ (r >> 1 & 3u) : (c + PIECES / 2u - (r >> 2 & 3u)) % (PIECES / 2u)) * 2u + (at & 1u);
  }
};

// Waits for the wave's loads and LDS operations, then for the other waves.
__device__ __forceinline__ void wait_step() { __asm__ volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" : : : "memory"); }

typedef short short4v __attribute__((ext_vector_type(4)));
__device__ __forceinline__ uint2 ld_turned(const uint8_t *p) {
  typedef __attribute__((address_space(3))) short4v *lds_ptr;
  return __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(__attribute__((address_space(3))) void *)p));
}

// The join of a tile of 64 rows, as attn_join: workgroup by workgroup, a thread's PIECES
// parts of 4 columns of a row at once, U workgroups under way, and a lane a row for the
// maxima and sums, since the way to what the others stored is all that it waits for (8
// trees of 20 drafts over up to 8192 tokens, 32 heads of 128 on 8: 82 -> 56 us against
// attn_join's rows and columns one after the other). LDS: 128 floats for each workgroup
// of one step.
template <int D, typename TILE>
__device__ __forceinline__ void attn_join_rows(const AttnPlan &p, rsrc_t prs, uint32_t *cnt, const KvAttnArgs &a, const TILE &t, uint32_t group,
                                               uint32_t kvh, uint32_t item, uint32_t first, uint32_t chunks, float *wt, float *sm, float *sl,
                                               uint32_t &arrived) {
  constexpr uint32_t T = 256u, R = 64u, PIECES = R * D / 4u / T, U = PIECES < 16u ? 16u / PIECES : 1u;   // U workgroups under way
  const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint32_t slot_floats = attn_part_floats(p, D), ml = p.rows * D, pieces = t.rows * (D / 4u);
  const auto place = [&](uint32_t z) { return 2u * (first + z) + (z == 0u ? 1u : 0u); };   // the slot of the tile's workgroup z
  const uint32_t side = chunks <= kJoinRows * U ? chunks : __builtin_amdgcn_readfirstlane((uint32_t)ceilf(sqrtf((float)chunks)));
  const uint32_t groups = (chunks + side - 1u) / side;
  uint32_t z0 = (item - first) / side * side, step = 1u, count = min(side, chunks - z0);
  for (bool last = groups == 1u;; last = true) {
    __asm__ volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    uint32_t *counter = cnt + (step == 1u ? 0u : kAttnCounters / 2u) + (uint64_t)kvh * p.items * 2u + place(z0);
    if (tid == 0u) arrived = __hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();
    if (arrived != count - 1u) break;
    if (tid == 0u) __hip_atomic_store(counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    float4v x[U][PIECES], o[PIECES] = {};
    const auto request = [&](uint32_t z) {
#pragma unroll
      for (uint32_t u = 0; u < U; ++u)
#pragma unroll
        for (uint32_t k = 0; k < PIECES; ++k) {
          const uint32_t i = min(tid + T * k, pieces - 1u);
          x[u][k] = __builtin_bit_cast(float4v, __builtin_amdgcn_raw_buffer_load_b128(prs, (int)((place(z0 + step * min(z + u, count - 1u)) * slot_floats + 4u * i) * 4u), 0, kSc1));
        }
    };
    request(0);
    // the rows' maxima and sums: a lane has a row, a wave every fourth workgroup; then the
    // weights relative to the largest maximum
    float *ls = wt + count * R;
    if (lane < t.rows)
      for (uint32_t z = wave; z < count; z += 4u) {
        const int at = (int)((place(z0 + step * z) * slot_floats + ml + 2u * lane) * 4u);
        wt[z * R + lane] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(prs, at, 0, kSc1));
        ls[z * R + lane] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(prs, at + 4, 0, kSc1));
      }
    __syncthreads();
    if (tid < t.rows) {
      float mx = -INFINITY, l = 0.f;
      for (uint32_t z = 0; z < count; ++z) mx = fmaxf(mx, wt[z * R + tid]);
      for (uint32_t z = 0; z < count; ++z) {
        const float m = wt[z * R + tid], f = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - mx);
        wt[z * R + tid] = f;
        l += f * ls[z * R + tid];
      }
      sl[tid] = l, sm[tid] = mx;
    }
    __syncthreads();
    for (uint32_t z = 0; z < count; z += U) {
      if (z) request(z);
#pragma unroll
      for (uint32_t u = 0; u < U; ++u)
#pragma unroll
        for (uint32_t k = 0; k < PIECES; ++k)
          if (z + u < count) o[k] += x[u][k] * wt[(z + u) * R + min(tid + T * k, pieces - 1u) / (D / 4u)];
    }
#pragma unroll
    for (uint32_t k = 0; k < PIECES; ++k) {
      const uint32_t i = tid + T * k, r = i / (D / 4u), d = 4u * (i % (D / 4u));
      if (i >= pieces) break;
      const float l = sl[r];
      if (last) {
        const uint32_t tok = (t.r0 + r) / group, h = (t.r0 + r) % group;
        float *dst = a.out + ((uint64_t)(t.token0 + tok) * a.q_heads + kvh * group + h) * D + d;
        *(float4v *)dst = l == 0.f ? float4v{0.f, 0.f, 0.f, 0.f} : o[k] / l;
      } else {
        const uint32_t at = place(z0) * slot_floats;
        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, o[k]), prs, (int)((at + 4u * i) * 4u), 0, kSc1);
        if (d == 0u) {
          // a sum that is not a number is not nothing
          const float mx = sm[r] == -INFINITY && l != 0.f ? 0.f : sm[r];
          __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(mx), prs, (int)((at + ml + 2u * r) * 4u), 0, kSc1);
          __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(l), prs, (int)((at + ml + 2u * r + 1u) * 4u), 0, kSc1);
        }
      }
    }
    if (last) break;
    z0 = 0u, step = side, count = groups;
  }
}

template <int TYPE, int D, int MODE, typename RULES>
__global__ __launch_bounds__(256, D <= 128 ? 3 : 2) void k_attn_rows(KvView kv, KvBatchView b, KvAttnArgs a, uint32_t tiles,
                                                                      uint32_t per_seq, uint32_t min_rows, RULES rules, AttnPlan p,
                                                                      uint32_t *cnt, float *part) {
  constexpr bool I8 = TYPE == EFF_KV_I8, RULED = !__is_same(RULES, NoRules);
  using W = AttnWave<D, I8, false, false, D <= 128 ? kVTurned : kVLater, RULED>;
  using S = AttnStage<D>;
  constexpr uint32_t NW = 4u, R = 16u * NW;
  __shared__ __align__(1024) uint8_t buf[2][S::BYTES];
  const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = __builtin_amdgcn_readfirstlane(tid >> 6), n = lane & 15u, g = lane >> 4;
  const uint32_t group = a.q_heads / kv.heads;
  // The last tiles of a sequence see the most: first; sequence after sequence, and a
  // head to an XCD where there are 8, so that tiles which run together read the same
  // rows out of its L2 (the sequences in turn, longest tiles of all first: 199 us
  // for the above, 371 -> 453 for 4 x 500 over up to 8000)
  constexpr bool shared = MODE == kAttnEnds;
  const uint32_t kvh = blockIdx.x % kv.heads, item = blockIdx.x / kv.heads, tile = tiles - 1u - item;
  typename W::Tile t;
  AttnShare c = {1u, 1u, 0u, 1u, 0u, 0u};
  if constexpr (shared) {
    uint32_t tree = 0;   // new tokens of a tree at most
    if constexpr (RULED) tree = rules.tree ? min(b.max_new, b.tokens) : 0u;
    if (!attn_share<R, true>(b, group, a.window, tree, item, p.items, ~0u, t, c)) return;
  } else {
    if (!attn_tile<R>(b, group, a.window, tile, per_seq, min_rows, ~0u, t)) return;
  }
  const int window = (int)min(a.window, 0x40000000u);
  typename W::Tile m = t;   // the wave's own rows
  int row_from = 0, row_to = 0;   // lane r: the range of the tile's row r
  if constexpr (RULED) attn_range(t, rules, group, lane, row_from, row_to);
  attn_seen<R>(t, rules, window, row_from, row_to);
  const int tile_base = t.begin & ~31;
  int base = tile_base, hi = t.end;
  uint32_t first = 0, chunks = 1;   // the tile's workgroups
  if constexpr (shared) {
    base += (int)(c.at * kUnit);
    hi = min(tile_base + (int)(min(c.at + c.left, c.of) * kUnit), t.end);
    if (base >= hi && base != tile_base) return;   // the tile's other workgroups have it all
    const uint32_t units = t.end > tile_base ? ((uint32_t)(t.end - tile_base) + kUnit - 1u) / kUnit : 1u;
    first = __builtin_amdgcn_readfirstlane(c.start / c.each);
    chunks = __builtin_amdgcn_readfirstlane((c.start + units - 1u) / c.each) - first + 1u;
  }
  const uint32_t row0 = 16u * wave;
  m.rows = t.rows > row0 ? min(t.rows - row0, 16u) : 0u;
  if (m.rows) {
    m.r0 = t.r0 + row0;
    m.first = t.first + (int)(m.r0 / group - t.r0 / group);
    m.last = t.first + (int)((m.r0 + m.rows - 1u) / group - t.r0 / group);
    m.end = max(m.last + 1, 0);
    m.begin = window ? max(0, m.first - window + 1) : 0;
    attn_seen<16>(m, rules, window, row_from, row_to, row0);
  } else {
    m.r0 = t.r0, m.end = 0;
  }
  W w;
  const auto begin_rows = [&] {
    float q[W::KS][8];
    w.load_q(q, a, m, group, kvh, n, g);
    w.init(q, a.scale, nullptr, wave, NW);
  };
  if constexpr (!RULED) begin_rows();
  __shared__ AttnRule rule_rows[RULED ? NW : 1u][RULED ? 16u : 1u];
  const auto wr = attn_rules(rules, rule_rows[RULED ? wave : 0u], group);
  if constexpr (RULED) W::put_rule(wr, m, kvh, n, g, window, __shfl(row_from, row0 + n), __shfl(row_to, row0 + n));

  const uint32_t to_v = kv.heads * kv.block_bytes;
  AttnWalk k;
  k.table = b.table + (uint64_t)t.seq * b.table_pages;
  k.heads = kv.base + (uint64_t)kvh * kv.block_bytes;
  k.lo = base, k.hi = hi, k.stride = 32;
  // fp16: a step's fills, K's 16 rows of each half, then V's; the wave's are NW apart.
  // int8: a step's 16-byte pieces, K's, then V's; the thread's are 256 apart
  constexpr uint32_t MINE = I8 ? (4u * D + 255u) / 256u : 4u * S::FILLS / NW;
  // which of K's halves and V's a fill or piece is of, and its place there: known
  // when a wave's are whole
  constexpr bool EVEN = I8 ? D % 256u == 0u : S::FILLS % NW == 0u;
  constexpr uint32_t PER = EVEN ? (I8 ? D / 256u : S::FILLS / NW) : 1u;
  uint32_t off[MINE], which[MINE];   // bytes within the 16 rows
#pragma unroll
  for (uint32_t j = 0; j < MINE; ++j) {
    if constexpr (I8) {
      const uint32_t x = 256u * j + tid;
      which[j] = EVEN ? j / PER : D % 64u ? x / D : __builtin_amdgcn_readfirstlane(x / D);
      off[j] = 16u * (x % D);
    } else {
      const uint32_t l = NW * j + wave, x = l % S::FILLS * 64u + lane, r = x / S::PIECES, c = x % S::PIECES;
      which[j] = EVEN ? j / PER : l / S::FILLS;
      off[j] = r * S::ROW + 16u * (which[j] < 2u ? S::piece(r, c) : S::v_piece(r, c));
    }
  }
  // where the lane's parts of the operands lie in a buffer. From 128 wide the places
  // are those of piece 0 with bits turned, one instruction instead of a register
  constexpr bool TURN = S::PIECES >= 16u;
  const uint32_t vr = 4u * g + n / 4u;
  uint32_t ka[TURN ? 1 : W::KS], va[TURN ? 1 : W::E];
#pragma unroll
  for (int c = 0; c < (TURN ? 1 : W::KS); ++c) ka[c] = n * S::ROW + 16u * S::place(n, 4u * c + g);
#pragma unroll
  for (int i = 0; i < (TURN ? 1 : W::E); ++i) va[i] = S::V + vr * S::ROW + 32u * S::v_place(vr, i) + 8u * (n & 3u);

  const int steps = hi > base ? (hi - base + 31) / 32 : 0;
  u32x4 raw[I8 ? MINE : 1];
  uint32_t raw_scale = 0;
  // Requests step i: into buffer `lds`, or (int8) into registers.
  const auto issue = [&](int i, const uint8_t *lds) {
    k.go<I8 ? D : 2 * D>(kv, i);
    rsrc_t run[2];
#pragma unroll
    for (int u = 0; u < 2; ++u)
      run[u] = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t *>(k.at[u]), (short)0, (int)(to_v + kv.block_bytes), kRsrcFlags);
    if constexpr (I8) {
#pragma unroll
      for (uint32_t j = 0; j < MINE; ++j) {
        if (MINE * 256u > 4u * D && 256u * j + tid >= 4u * D) break;
        const uint32_t o = off[j] + (which[j] >> 1 ? to_v : 0u);
        if (D % 64u) {   // a wave's 64 pieces may lie in two halves
          if (which[j] & 1u) raw[j] = __builtin_amdgcn_raw_buffer_load_b128(run[1], (int)o, 0, 0);
          else raw[j] = __builtin_amdgcn_raw_buffer_load_b128(run[0], (int)o, 0, 0);
        } else {
          raw[j] = __builtin_amdgcn_raw_buffer_load_b128(which[j] & 1u ? run[1] : run[0], (int)o, 0, 0);
        }
      }
      if (wave == 3u) {   // the scales: K's of the 32 tokens, then V's
        const uint8_t *p = lane & 16u ? k.scales(1, kv, D) : k.scales(0, kv, D);
        raw_scale = *(cached<uint32_t>)(p + 4u * (lane & 15u) + (lane < 32u ? 0u : to_v));
      }
    } else {
#pragma unroll
      for (uint32_t j = 0; j < MINE; ++j)
        dma16(which[j] & 1u ? run[1] : run[0], lds + 1024u * (NW * j + wave), off[j], which[j] >> 1 ? to_v : 0u);
    }
  };
  // int8: what step i's issue() asked for, as fp16 into buffer `lds`.
  const auto convert = [&](uint8_t *lds) {
    if constexpr (I8) {
#pragma unroll
      for (uint32_t j = 0; j < MINE; ++j) {
        const uint32_t x = 256u * j + tid, r = x % D / (D / 16u), c = x % D % (D / 16u);
        if (MINE * 256u > 4u * D && x >= 4u * D) break;
        uint8_t *row = lds + which[j] * S::HALF + r * S::ROW;
        const uint32_t first = which[j] >> 1 ? 2u * S::v_place(r, c) : S::place(r, 2u * c);
        const uint32_t second = which[j] >> 1 ? first + 1u : S::place(r, 2u * c + 1u);
        *(half8 *)(row + 16u * first) = i8_half8(raw[j][0], raw[j][1]);
        *(half8 *)(row + 16u * second) = i8_half8(raw[j][2], raw[j][3]);
      }
      if (wave == 3u) *(uint32_t *)(lds + S::SCALES + 4u * lane) = raw_scale;
    }
  };
  const int full = W::full_of(m), from = W::from_of(m, window);   // steps from .. full need no mask
  if (steps) {
    issue(0, buf[0]);
    convert(buf[0]);
  }
  if constexpr (RULED) begin_rows();   // on the first steps' way
#pragma unroll 1
  for (int i0 = 0; i0 < steps; i0 += 2) {
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const int i = i0 + half;
      if (i >= steps) break;
      const bool was[2] = {k.gone[0], k.gone[1]};
      wait_step();
      if (i + 1 < steps) issue(i + 1, buf[1 - half]);
      const int t0 = base + 32 * i;
      if (t0 < m.end && t0 + 32 > m.begin) {
        const uint8_t *lds = buf[half];
        if constexpr (TURN) __asm__("" : "+v"(ka[0]), "+v"(va[0]));   // computed here, not kept
#pragma unroll
        for (int u = 0; u < 2; ++u) {
#pragma unroll
          for (int c = 0; c < W::KS; ++c) ld_lds(w.kw[u] + 4 * c, lds + (TURN ? ka[0] ^ (64u * c) : ka[TURN ? 0 : c]) + u * S::HALF);
          if constexpr (I8) ld_lds(w.ks[u], lds + S::SCALES + 64u * u + 16u * g);
        }
        __builtin_amdgcn_sched_barrier(0);
        float s[2][4];
        w.scores(s);
        __builtin_amdgcn_sched_barrier(0);
        const auto turned = [&](int c) {
          const uint8_t *p = lds + (TURN ? va[0] ^ (32u * c) : va[TURN ? 0 : c]);
          const uint2 x = ld_turned(p), y = ld_turned(p + S::HALF);
          return u32x4{x.x, x.y, y.x, y.y};
        };
        if constexpr (D <= 128) {
#pragma unroll
          for (int c = 0; c < W::E; ++c) __builtin_memcpy(w.vw[c], &(const u32x4 &)turned(c), 16);
        }
        w.step(t0, was[0] || was[1] || t0 > full || t0 < from, was, m, window, wr, n, g, s, [&](int c) { return D <= 128 ? w.v_operand(c) : turned(c); },
               [&](int u) { return *(const u32x4 *)(lds + S::SCALES + 128u + 64u * u + 16u * g); });   // late: no register waits for it
      }
      if (i + 1 < steps) convert(buf[1 - half]);
    }
  }
  const float l = row_add(w.l);
  if constexpr (shared) if (chunks > 1u) {
    const uint32_t slot_floats = attn_part_floats(p, D), slot = (2u * item + (item == first ? 1u : 0u)) * slot_floats;
    const rsrc_t prs = make_rsrc(part + (uint64_t)kvh * p.items * 2u * slot_floats, (uint64_t)p.items * 2u * slot_floats * 4u);
    if (n < m.rows) {
      const uint32_t r = row0 + n;
#pragma unroll
      for (int i = 0; i < W::E; ++i)
        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, I8 ? w.acc[i] * w.unit : w.acc[i]), prs,
                                               (int)((slot + r * D + W::column(g, i, 0)) * 4u), 0, kSc1);
      if (g == 0u) {
        __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(w.m * w.of_scores(wr)), prs, (int)((slot + p.rows * D + 2u * r) * 4u), 0, kSc1);
        __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(l), prs, (int)((slot + p.rows * D + 2u * r + 1u) * 4u), 0, kSc1);
      }
    }
    // the waves have passed the last step's barrier, but may still read its buffer
    static_assert(kJoinSide * kJoinSide >= kItemsRows && sizeof(buf) >= 2u * kJoinSide * R * 4u && 4u * kJoinRows <= kJoinSide, "a join's LDS");
    __shared__ float sm[R], sl[R];
    __shared__ uint32_t arrived;
    attn_join_rows<D>(p, prs, cnt, a, t, group, kvh, item, first, chunks, (float *)buf, sm, sl, arrived);
    return;
  }
  if (n >= m.rows) return;
  // no weight: nothing seen, or the largest score past f32
  const float f = l == 0.f ? (w.m == -INFINITY ? 0.f : NAN) : (I8 ? w.unit : 1.f) / l;
  const uint32_t tok = (m.r0 + n) / group, h = (m.r0 + n) % group;
  float *dst = a.out + ((uint64_t)(t.token0 + tok) * a.q_heads + kvh * group + h) * D;
#pragma unroll
  for (int i = 0; i < W::E; ++i) *(float4v *)(dst + W::column(g, i, 0)) = w.acc[i] * f;
}

// Tiles of R rows for sequences of at most `most` rows, `rows` of them in all.
inline void attn_tiles(uint64_t most, uint64_t rows, uint32_t seqs, uint32_t r, uint32_t *tiles, uint32_t *per_seq) {
  const uint64_t each = (most + r - 1u) / r, direct = each * seqs, packed = rows / r + seqs;
  *per_seq = direct <= packed ? (uint32_t)each : 0u;
  *tiles = (uint32_t)std::min(direct, packed);
}

// Tiles of 16 rows of the sequences, which have `most` rows at most and `rows` in all, and
// see `seen` tokens at most.
inline void attn_plan_few(AttnPlan &p, const KvView &kv, const KvBatchView &b, uint64_t most, uint64_t rows, uint64_t seen) {
  constexpr uint32_t R = 16u;
  attn_tiles(most, rows, b.seqs, R, &p.tiles, &p.per_seq);
  p.rows = (uint32_t)std::min<uint64_t>(most, R);
  const uint64_t span = seen + 31u, wgs = (uint64_t)p.tiles * kv.heads;
  // Where the tiles alone fill two thirds of the CUs and are short, or there are many, a
  // workgroup has a tile, as where there are 5 units or fewer (4 at 256 wide): a join
  // takes time (1 x 8 heads of 64 over 517 tokens: 6.8 us, shared 7.6, over 1000 9.3
  // and 8.0; 24 x 8 heads of drafts that see 1024 tokens 14.7, shared 22.0; heads of one
  // token up to 2000: 16 x 8 22.6, shared 18.3, 32 x 8 35.5 and 45.5; 24 x 8 up to 1500
  // 19.4, shared 22.5, up to 3000 44.6 and 42.3, in between either way; 480 x 8 heads of
  // 64 up to 3000 287, shared 288, 1000 x 8 552 and 567).
  const uint64_t units = (span + kUnit - 1u) / kUnit, each = (most + R - 1u) / R;
  if ((wgs < 171u || span > 2176u) && wgs < 4096u && units > (kv.dim < 256u ? 5u : 4u) && each * b.seqs * units < 1u << 31) {
    // Two workgroups to a CU, or one where its waves have enough bytes under way: 256
    // wide (24 x 2 heads up to 8000 48.9 us, two 54.1; of int8 33.6 and 35.0), or fp16
    // rows of 128 and long shares (1 x 8 up to 130001 96.7, two 99.4; 24 x 8 up to 6000
    // 69.2 and 71.1; 8 x 8 drafts up to 5000, short ones, 30.6 and 28.1; next to the
    // limit, 16 x 8 up to 8000, 68.8 and 63.5). Less wide they take two (16 x 8 of int8
    // up to 30000 102, two 99).
    // Shares that may go on into the next tile pay where they are long (64 x 8 up to
    // 16384 357 us, ending with a tile 411; 24 x 8 up to 6000 70, 93, up to 3000 42.1,
    // 41.5; below the limit from shares of 12 on they would too, up to 4000 55, 77); 256
    // wide, where the scalar registers of that take vector ones, only with many tiles
    // (100 x 2 of int8 up to 9000 115, 156; 24 x 2 up to 30000 76, 73).
    uint64_t slots = 512u;
    const uint64_t share = wgs * units / slots;
    const bool wide = kv.dim >= 256u;
    if (wide || (kv.dim == 128u && kv.type == EFF_KV_F16 && share >= 12u)) slots = 256u;
    p.on = share >= 16u && (!wide || wgs * 4u > slots);
    p.items = (uint32_t)std::max<uint64_t>(slots / kv.heads, p.on ? 1u : 2u * p.tiles);
  }
  // 8 waves where a CU has one workgroup and the steps to share (the drafts above:
  // 14.7 us, 4 waves 15.5; 128 of up to 2000 of int8, 256 wide, 32.3 and 35.6; fp16 of
  // that width 46.8 and 45.7; 1024 workgroups of up to 300 tokens 20.5 and 20.2)
  p.waves = !p.items && wgs <= 256u && span >= 512u && (kv.dim < 256u || kv.type == EFF_KV_I8) ? 8u : 4u;
}

inline AttnPlan attn_plan(const KvView &kv, const KvBatchView &b, const KvAttnArgs &a) {
  const uint32_t group = a.q_heads / kv.heads;
  constexpr uint32_t R = 16u;
  AttnPlan p{};
  uint64_t most = std::min<uint64_t>(b.max_new, b.tokens) * group;
  const uint64_t rows = (uint64_t)b.tokens * group;
  p.max_rows = ~0u;
  const uint64_t seen = a.window ? std::min<uint64_t>(b.max_len, (uint64_t)a.window + R / group + 2u) : b.max_len;
  // Sequences with more than 64 rows go to k_attn_rows where there are enough tiles of
  // that (1 x 32 heads of 128 on 8 over 4000 tokens: 300 new tokens 108 us, k_attn 104,
  // 400 108 and 131; int8 pages cost a conversion more for the same tile: 600 174 and
  // 160, 800 175 and 201). The others go with them where lengths and new tokens are
  // alike, since a second launch waits for the first (32 of up to 24 new tokens: 71 us,
  // two launches 97); a long one's tile there is not shared.
  if (most > kFewRows && rows / 64u * kv.heads >= (kv.type == EFF_KV_F16 ? 176u : 400u)) {
    attn_tiles(most, rows, b.seqs, 64u, &p.many_tiles, &p.many_per_seq);
    if (b.seqs == 1u || (most * b.seqs <= 3u * rows && seen <= 4096u)) return p;
    p.max_rows = kFewRows;
    most = kFewRows;
  }
  attn_plan_few(p, kv, b, most, rows, seen);
  return p;
}

// Under rules all sequences go to one kernel.
inline AttnPlan attn_plan(const KvView &kv, const KvBatchView &b, const KvAttnArgs &a, const KvRulesView &r) {
  const uint32_t group = a.q_heads / kv.heads;
  AttnPlan p{};
  const uint32_t new_most = std::min(b.max_new, b.tokens);
  const uint64_t most = (uint64_t)new_most * group, rows = (uint64_t)b.tokens * group;
  p.max_rows = ~0u;
  const uint64_t reach = (uint64_t)a.window + std::max(64u / group, r.tree ? new_most : 0u) + 2u;   // under a window
  const uint64_t seen = a.window ? std::min<uint64_t>(b.max_len, reach) : b.max_len, units = (seen + 31u + kUnit - 1u) / kUnit;
  uint32_t tiles, per_seq;
  attn_tiles(most, rows, b.seqs, 64u, &tiles, &per_seq);
  const uint64_t wgs = (uint64_t)tiles * kv.heads, work = (rows / 16u + b.seqs) * kv.heads * units;
  // Tiles of 64 rows from 176 of them on, or where there is much to read (32 heads of 128 on
  // 8: 1 x 200 new tokens 11.8 us, tiles of 16 10.0, 1 x 400 19.5 and 20.9; trees: 2 x 10
  // over up to 3000 21.7 and 19.0, 8 x 20 over up to 8192 54 and 82). int8 pages cost
  // them a conversion more (16 x 60 rows over up to 8000 76 and 74, 3 x 600 new tokens of 4
  // heads 54 and 49, 2 x 900 of 8 88 and 112).
  const bool f16 = kv.type == EFF_KV_F16;
  if (most <= 16u || (f16 ? wgs < 176u && work < 8192u : wgs < 400u)) {
    attn_plan_few(p, kv, b, most, rows, seen);
    return p;
  }
  p.many_tiles = tiles, p.many_per_seq = per_seq;
  p.rows = (uint32_t)std::min<uint64_t>(most, 64u);
  // Shared where they do not fill the card, or not evenly: few new tokens, long contexts of
  // any length (three workgroups a CU, two 256 wide: 16 trees of up to 32 over up to 16384
  // 174 us, two 195, four 183; a chunk of 300 tokens over 4000 70, not shared 128, of 600
  // over 2000 87 and 73).
  const uint32_t slots = kv.dim <= 128u ? 768u : 512u;
  const uint64_t items = std::max<uint64_t>(slots / kv.heads, 2u * tiles), each = (most + 63u) / 64u;
  if (f16 && units > 2u && (wgs < 200u || (wgs < slots && units >= 8u && seen >= 16ull * new_most)) && items <= kItemsRows && items * kv.heads <= kAttnCounters / 4u &&
      each * b.seqs * units < 1u << 31)
    p.items = (uint32_t)items;
  return p;
}

inline AttnPlan attn_plan(const KvView &kv, const KvBatchView &b, const KvAttnArgs &a, NoRules) { return attn_plan(kv, b, a); }

inline size_t attn_scratch(const AttnPlan &p, const KvView &kv) {
  return p.items ? kAttnCounters * 4u + (uint64_t)p.items * kv.heads * 2u * attn_part_floats(p, kv.dim) * 4u : 0u;
}

template <int TYPE, int D, typename RULES>
hipError_t attn_go(const KvView &kv, const KvBatchView &b, const KvAttnArgs &a, const RULES &rules, void *scratch, hipStream_t s) {
  const AttnPlan p = attn_plan(kv, b, a, rules);
  const bool shared = p.items && !p.tiles;   // the tiles of 64
  const uint64_t many = (uint64_t)(shared ? p.items : p.many_tiles) * kv.heads, grid = (uint64_t)(p.items ? p.items : p.tiles) * kv.heads;
  if (!fits(many, 256u) || !fits(grid, 512u)) return hipErrorInvalidConfiguration;
  if (p.items && (grid > kAttnCounters / 4u || !scratch)) return hipErrorInvalidValue;
  uint32_t *cnt = (uint32_t *)scratch;
  float *part = (float *)((uint8_t *)scratch + kAttnCounters * 4u);
  if (many) {
    const uint32_t min_rows = p.tiles ? kFewRows + 1u : 1u;
    const auto rows = [&](auto kernel) {
      hipLaunchKernelGGL(kernel, dim3((uint32_t)many), dim3(256), 0, s, kv, b, a, p.many_tiles, p.many_per_seq, min_rows, rules, p, cnt, part);
    };
    // Tiles of 64 are shared under rules only: the plain plan has not been measured with it (a
    // chunk of 300 tokens over 4000, 32 heads of 128 on 8: capped 71 us, plain, in shared tiles
    // of 16, 103; 400 tokens over 400 and 1000 over 1000, not shared: 19 and 40, plain 17 and 35).
    constexpr bool may = !__is_same(RULES, NoRules) && TYPE == EFF_KV_F16;
    if (may && shared) rows(k_attn_rows<TYPE, D, may ? kAttnEnds : kAttnWhole, RULES>);
    else rows(k_attn_rows<TYPE, D, kAttnWhole, RULES>);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || !p.tiles) return e;
  }
  const auto go = [&](auto kernel, uint32_t threads) {
    hipLaunchKernelGGL(kernel, dim3((uint32_t)grid), dim3(threads), 0, s, kv, b, a, p, cnt, part, rules);
  };
  constexpr int E = D < 256 || TYPE == EFF_KV_I8 ? D : 64;   // no fp16 tiles 256 wide of eight waves
  if (p.on) go(k_attn<TYPE, D, 4, kAttnOn, RULES>, 256u);
  else if (p.items) go(k_attn<TYPE, D, 4, kAttnEnds, RULES>, 256u);
  else if (p.waves == 8u) go(k_attn<TYPE, E, 8, kAttnWhole, RULES>, 512u);
  else go(k_attn<TYPE, D, 4, kAttnWhole, RULES>, 256u);
  return hipGetLastError();
}

template <int TYPE, typename RULES>
hipError_t attn_dim(const KvView &kv, const KvBatchView &b, const KvAttnArgs &a, const RULES &rules, void *scratch, hipStream_t s) {
  switch (kv.dim) {
    case 64: return attn_go<TYPE, 64>(kv, b, a, rules, scratch, s);
    case 96: return attn_go<TYPE, 96>(kv, b, a, rules, scratch, s);
    case 128: return attn_go<TYPE, 128>(kv, b, a, rules, scratch, s);
    case 256: return attn_go<TYPE, 256>(kv, b, a, rules, scratch, s);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace eff
