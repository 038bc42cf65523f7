// The paged key/value cache: its layout, and the views that the entry points
// give the append and attention kernels.
//
// Page p of a cache is [K, V][head][block]; a block holds the `page_tokens` rows
// of one head: fp16 rows of head_dim values (EFF_KV_F16), or int8 rows followed
// by the rows' f32 scales (EFF_KV_I8: value = int8 * scale). A head's rows lie
// side by side, so that a wave reads 16 rows of a page as one run.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/elffuss_amd.h"

namespace eff {

constexpr uint32_t kKvPageMin = 16, kKvPageMax = 1024;   // tokens of a page, a power of two

inline bool kv_type_known(int t) { return t == EFF_KV_F16 || t == EFF_KV_I8; }
inline bool kv_dim_known(uint32_t d) { return d == 64u || d == 96u || d == 128u || d == 256u; }

// Bytes of one head's rows of a page, K or V.
constexpr uint32_t kv_block_bytes(int type, uint32_t dim, uint32_t page) {
  return page * (type == EFF_KV_F16 ? 2u * dim : dim + 4u);
}

// A grid's threads are counted in 32 bits.
inline bool fits(uint64_t wgs, uint32_t threads) { return wgs * threads <= 0xFFFFFFFFull; }

struct KvView {
  uint8_t *base;
  int type;
  uint32_t heads, dim, page_log2, pages;
  uint32_t block_bytes;   // kv_block_bytes
  uint64_t page_bytes;    // 2 * heads * block_bytes
};

struct KvBatchView {
  const uint32_t *table;    // [seqs][table_pages]
  const uint32_t *starts;   // [seqs + 1]
  const uint32_t *lens;     // [seqs]
  uint32_t seqs, tokens, table_pages, max_new, max_len;
};

// The rows of one append: f32, `stride` floats from token to token.
struct KvAppendArgs {
  const float *q, *k, *v;            // q null: none
  uint32_t q_stride, k_stride, v_stride;
  float *q_out;                      // [tokens][q_heads * dim]
  uint32_t q_heads;
  const float *rope;                 // [positions][2][rope_dim / 2]
  uint32_t rope_dim;                 // 0: no rotation
  int halves;                        // pairs (i, i + rope_dim / 2), else (2 i, 2 i + 1)
  const float *q_norm, *k_norm;      // null: none
  float eps;
};

// Positions to turn by, of the new tokens on each axis, and the axis of each pair.
struct KvTurnsView {
  const uint32_t *at;                // [axes][tokens]
  uint32_t tokens, positions;        // of the rope table
  uint8_t axis[128];
};

struct KvAttnArgs {
  const float *q;
  uint32_t q_stride;
  float *out;                        // [tokens][q_heads * dim]
  uint32_t q_heads;
  float scale;
  uint32_t window;                   // 0: none
};

// Rules on the scores of attention, and what the new tokens see.
struct KvRulesView {
  float cap, per_cap;                // times log2 e, and 1 over that (0: none)
  const float *slopes;               // [q_heads], null: none
  const uint32_t *ranges;            // [tokens][2], null: none
  const uint32_t *tree;              // [tokens][tree_words], null: none
  uint32_t tree_words;
};
struct NoRules {};
constexpr uint32_t kRopeMaxPairs = 256;
struct RopeFreqs {
  double f[kRopeMaxPairs];
};
hipError_t launch_rope_table(const RopeFreqs &f, uint32_t pairs, uint32_t positions, float scale, float *out,
                             hipStream_t stream);
hipError_t launch_kv_append(const KvView &kv, const KvBatchView &b, const KvAppendArgs &a, const KvTurnsView *turns,
                            hipStream_t stream);   // turns null: by the place in the cache

// The caches of a group of layers, alike but for their memory (`kv.base` is not used).
constexpr uint32_t kKvLayers = 64;
struct KvLayers {
  uint8_t *base[kKvLayers];
};
hipError_t launch_kv_copy(const KvView &kv, const KvLayers &l, uint32_t layers, const uint32_t *copies, uint32_t count,
                          hipStream_t stream);
hipError_t launch_kv_keep(const KvView &kv, const KvLayers &l, uint32_t layers, const KvBatchView &b, const uint32_t *kept,
                          const uint32_t *counts, uint32_t *new_lens, hipStream_t stream);
// The scratch of tiles that several workgroups share (0: none): counters, zero before
// the first launch and left zero by each, then the workgroups' sums.
constexpr uint32_t kAttnCounters = 65536;
size_t kv_attn_scratch(const KvView &kv, const KvBatchView &b, const KvAttnArgs &a);
hipError_t launch_kv_attn(const KvView &kv, const KvBatchView &b, const KvAttnArgs &a, void *scratch,
                          hipStream_t stream);
size_t kv_attn_rules_scratch(const KvView &kv, const KvBatchView &b, const KvAttnArgs &a, const KvRulesView &r);
hipError_t launch_kv_attn_rules(const KvView &kv, const KvBatchView &b, const KvAttnArgs &a, const KvRulesView &r, void *scratch,
                                hipStream_t stream);

struct LogitsArgs {
  const float *in;
  float *out;
  uint32_t rows, vocab, stride;
  const uint32_t *history, *history_starts;   // null: none
  uint32_t history_count;
  const double *penalties;                    // [rows][3]: repeat, frequency, presence
  const uint32_t *bias_ids, *bias_starts;     // null: none
  const float *bias_values;
  uint32_t bias_count;
  const uint32_t *mask, *mask_of;             // null: none
  uint32_t mask_count;
};
hipError_t launch_logits(const LogitsArgs &a, hipStream_t stream);

#ifdef __HIP__
// The sequence of new token t (the whole wave asks for one t): the last whose
// first token is at most t, its first token, the next one's, and its length; one
// round trip up to 63 sequences. False for a token of no sequence.
struct KvSeq {
  uint32_t seq, first, next, len;
};
__device__ __forceinline__ bool kv_seq_of(const KvBatchView &b, uint32_t t, KvSeq &s) {
  const uint32_t lane = threadIdx.x & 63u;
  for (uint32_t at = 0;; at += 63u) {   // a block's last start is the next one's first
    const uint32_t i = at + lane;
    const uint32_t start = i <= b.seqs ? b.starts[i] : ~0u, len = i < b.seqs ? b.lens[i] : 0u;
    const uint64_t past = __ballot(start > t);
    const uint32_t n = past ? (uint32_t)__ffsll((unsigned long long)past) - 1u : 64u;   // starts[at .. at + n) <= t
    if (n == 64u && at + 64u <= b.seqs) continue;
    if (n == 0u || at + n > b.seqs) return false;
    s.seq = at + n - 1u;
    s.first = __builtin_amdgcn_readlane(start, n - 1u);
    s.next = n < 64u ? __builtin_amdgcn_readlane(start, n) : ~0u;
    s.len = min((uint32_t)__builtin_amdgcn_readlane(len, n - 1u), b.max_len);
    return true;
  }
}

// Tokens of sequence s, the new ones included, as far as the call reaches.
__device__ __forceinline__ uint32_t kv_len(const KvBatchView &b, uint32_t s) { return min(b.lens[s], b.max_len); }
#endif

}  // namespace eff
