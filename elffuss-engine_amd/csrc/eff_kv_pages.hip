// Copies within the paged cache: pages of a forked request, and the drafts that stay
// after a batch of them was verified, which move up behind the tokens before them. Both
// go over the caches of all layers in one launch; nothing is computed, the bytes bound
// them, or for a few rows the round trips from the lists to the rows.
#include <algorithm>

#include "eff_device.h"
#include "eff_kv.h"

namespace eff {

// Bytes of a row, without its scale.
template <int TYPE>
__device__ __forceinline__ uint32_t row_bytes(uint32_t dim) {
  return TYPE == EFF_KV_F16 ? 2u * dim : dim;
}

constexpr uint32_t kCopyUnder = 2;   // pieces of a thread under way

// A workgroup takes 512 pieces of 16 bytes of the tokens that one copy has in one layer,
// over the page's heads, K and V; int8 pages then have the rows' scales, 4 bytes each. The
// copied rows go past the L2, which the copy would only sweep. HBM bounds it (30 pages of
// 32 tokens, three quarters filled, 8 heads of 128, 32 layers, 169 MB: 30.9 us, 5.5 TB/s,
// stored through the L2 38.2; four pieces a thread 34.1 and 40.4, one 31.6), the launch a
// few of them (8 pages 4.9 us).
template <int TYPE>
__global__ __launch_bounds__(256) void k_kv_copy(KvView kv, KvLayers layers, const uint32_t *__restrict__ copies, uint32_t count, uint32_t parts) {
  const uint32_t part = blockIdx.x % parts, of = blockIdx.x / parts, i = of % count;
  uint8_t *const base = layers.base[of / count];
  const uint32_t from = copies[3u * i], to = copies[3u * i + 1u], n = min(copies[3u * i + 2u], 1u << kv.page_log2);
  if (from >= kv.pages || to >= kv.pages || from == to) return;
  const uint8_t *src = base + (uint64_t)from * kv.page_bytes;
  uint8_t *dst = base + (uint64_t)to * kv.page_bytes;
  const uint32_t runs = 2u * kv.heads, per = n * row_bytes<TYPE>(kv.dim) / 16u, all = runs * per;   // a run's pieces
  u32x4 x[kCopyUnder];
  uint32_t at[kCopyUnder];
#pragma unroll
  for (uint32_t u = 0; u < kCopyUnder; ++u) {
    const uint32_t p = (part * kCopyUnder + u) * 256u + threadIdx.x;
    at[u] = p < all ? p / per * kv.block_bytes + p % per * 16u : ~0u;
    if (p < all) x[u] = *(const u32x4 *)(src + at[u]);
  }
#pragma unroll
  for (uint32_t u = 0; u < kCopyUnder; ++u)
    if (at[u] != ~0u) __builtin_nontemporal_store(x[u], (u32x4 *)(dst + at[u]));
  if constexpr (TYPE == EFF_KV_I8) {
    const uint32_t rows = kv.dim << kv.page_log2;   // bytes of the rows, before the scales
    for (uint32_t p = part * 256u + threadIdx.x; p < runs * n; p += parts * 256u) {
      const uint32_t o = p / n * kv.block_bytes + rows + p % n * 4u;
      *(uint32_t *)(dst + o) = *(const uint32_t *)(src + o);
    }
  }
}

// The drafts that stay, of one sequence in one layer: a wave moves their rows in some of
// its runs (a head's K or V), 64 entries of the list at a time, whose places are looked up
// at once, one in each lane. An entry is not below its place, so that a row is read before
// its place is written if the rows are taken in order: a step's loads have all arrived
// before its first store, and no two waves have a run in common. Round trips bound it
// (lists, table, rows: 24 sequences that keep up to 7, 8 heads of 128, 32 layers 5.0 us,
// of which a launch alone is 3.4; 64 that keep up to 16 13.5 us). Runs one after the other
// in fewer waves: 16 heads of 64, 40 sequences, 7.3 us, a wave for each run 11.7.
constexpr uint32_t kKeepUnder = 4;   // pieces of a lane under way

template <int TYPE, int D>
__global__ __launch_bounds__(256) void k_kv_keep(KvView kv, KvLayers layers, KvBatchView b, const uint32_t *__restrict__ kept,
                                                 const uint32_t *__restrict__ counts, uint32_t *__restrict__ new_lens, uint32_t per,
                                                 uint32_t parts, uint32_t waves) {
  constexpr uint32_t ROW = TYPE == EFF_KV_F16 ? 2u * D : D, P = ROW / 16u;
  const uint32_t lane = threadIdx.x & 63u, w = blockIdx.x * 4u + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (w >= waves) return;
  const uint32_t part = w % parts, s = w / parts % b.seqs, layer = w / parts / b.seqs;
  const uint32_t s0 = b.starts[s], s1 = min(b.starts[s + 1u], b.tokens), len = kv_len(b, s);
  const uint32_t n = s1 > s0 ? min(s1 - s0, b.max_new) : 0u, stay = min(counts[s], n);
  const int first = (int)len - (int)n;   // the first new token's position; below 0 it has none
  if (new_lens && layer == 0u && part == 0u && lane == 0u) new_lens[s] = (uint32_t)max(first + (int)stay, 0);
  uint8_t *const base = layers.base[layer];
  const uint32_t *table = b.table + (uint64_t)s * b.table_pages;
  const uint32_t r0 = part * per, runs = min(per, 2u * kv.heads - r0);
  for (uint32_t i0 = 0; i0 < stay; i0 += 64u) {
    const uint32_t i = i0 + lane, k = i < stay ? kept[s0 + i] : 0u;
    uint32_t from = ~0u, to = ~0u, from_slot = 0, to_slot = 0;
    if (i < stay && k > i && k < n && first + (int)i >= 0) {
      const uint32_t a = (uint32_t)(first + (int)k), c = (uint32_t)(first + (int)i), mask = (1u << kv.page_log2) - 1u;
      from = table[a >> kv.page_log2], to = table[c >> kv.page_log2];
      from_slot = a & mask, to_slot = c & mask;
    }
    const uint32_t here = min(64u, stay - i0), items = runs * here * P;
    for (uint32_t at = 0; at < items; at += 64u * kKeepUnder) {
      u32x4 v[kKeepUnder];
      uint32_t scale[kKeepUnder];
      uint8_t *to_row[kKeepUnder];
      uint32_t *to_scale[kKeepUnder] = {};
#pragma unroll
      for (uint32_t u = 0; u < kKeepUnder; ++u) {
        const uint32_t y = at + 64u * u + lane, x = min(y, items - 1u), p = x % P, j = x / P % here, run = r0 + x / P / here;
        const uint32_t fp = __shfl(from, j), tp = __shfl(to, j), fs = __shfl(from_slot, j), ts = __shfl(to_slot, j);
        const uint64_t block = (uint64_t)run * kv.block_bytes;
        const uint8_t *src = base + (uint64_t)fp * kv.page_bytes + block;
        to_row[u] = nullptr;
        if (y >= items || fp >= kv.pages || tp >= kv.pages) continue;
        v[u] = *(const u32x4 *)(src + fs * ROW + 16u * p);
        if (TYPE == EFF_KV_I8 && p == 0u) scale[u] = *(const uint32_t *)(src + (D << kv.page_log2) + 4u * fs);
        to_row[u] = base + (uint64_t)tp * kv.page_bytes + block + ts * ROW + 16u * p;
        if (TYPE == EFF_KV_I8 && p == 0u) to_scale[u] = (uint32_t *)(base + (uint64_t)tp * kv.page_bytes + block + (D << kv.page_log2) + 4u * ts);
      }
      __asm__ volatile("s_waitcnt vmcnt(0)" : : : "memory");
#pragma unroll
      for (uint32_t u = 0; u < kKeepUnder; ++u) {
        if (!to_row[u]) continue;
        *(u32x4 *)to_row[u] = v[u];
        if (TYPE == EFF_KV_I8 && to_scale[u]) *to_scale[u] = scale[u];
      }
    }
  }
}

hipError_t launch_kv_copy(const KvView &kv, const KvLayers &l, uint32_t layers, const uint32_t *copies, uint32_t count, hipStream_t stream) {
  const uint64_t pieces = 2ull * kv.heads * (kv.dim * (kv.type == EFF_KV_F16 ? 2u : 1u) << kv.page_log2) / 16u;
  const uint64_t parts = (pieces + 256u * kCopyUnder - 1u) / (256u * kCopyUnder);
  if (!fits((uint64_t)layers * count * parts, 256u)) return hipErrorInvalidConfiguration;
  const dim3 grid((uint32_t)(layers * count * parts));
  if (kv.type == EFF_KV_F16) hipLaunchKernelGGL(k_kv_copy<EFF_KV_F16>, grid, dim3(256), 0, stream, kv, l, copies, count, (uint32_t)parts);
  else hipLaunchKernelGGL(k_kv_copy<EFF_KV_I8>, grid, dim3(256), 0, stream, kv, l, copies, count, (uint32_t)parts);
  return hipGetLastError();
}

template <int TYPE, int D>
static hipError_t keep_go(const KvView &kv, const KvLayers &l, uint32_t layers, const KvBatchView &b, const uint32_t *kept,
                          const uint32_t *counts, uint32_t *new_lens, hipStream_t s) {
  // enough waves to fill the card twice, if there are so many runs
  const uint32_t runs = 2u * kv.heads;
  const uint32_t per = (uint32_t)std::min<uint64_t>(runs, ((uint64_t)layers * b.seqs * runs + 8191u) / 8192u), parts = (runs + per - 1u) / per;
  const uint64_t waves = (uint64_t)layers * b.seqs * parts;
  if (!fits((waves + 3u) / 4u, 256u)) return hipErrorInvalidConfiguration;
  hipLaunchKernelGGL((k_kv_keep<TYPE, D>), dim3((uint32_t)((waves + 3u) / 4u)), dim3(256), 0, s, kv, l, b, kept, counts, new_lens, per, parts,
                     (uint32_t)waves);
  return hipGetLastError();
}

template <int TYPE>
static hipError_t keep_dim(const KvView &kv, const KvLayers &l, uint32_t layers, const KvBatchView &b, const uint32_t *kept,
                           const uint32_t *counts, uint32_t *new_lens, hipStream_t s) {
  switch (kv.dim) {
    case 64: return keep_go<TYPE, 64>(kv, l, layers, b, kept, counts, new_lens, s);
    case 96: return keep_go<TYPE, 96>(kv, l, layers, b, kept, counts, new_lens, s);
    case 128: return keep_go<TYPE, 128>(kv, l, layers, b, kept, counts, new_lens, s);
    case 256: return keep_go<TYPE, 256>(kv, l, layers, b, kept, counts, new_lens, s);
    default: return hipErrorInvalidValue;
  }
}

hipError_t launch_kv_keep(const KvView &kv, const KvLayers &l, uint32_t layers, const KvBatchView &b, const uint32_t *kept,
                          const uint32_t *counts, uint32_t *new_lens, hipStream_t stream) {
  return kv.type == EFF_KV_F16 ? keep_dim<EFF_KV_F16>(kv, l, layers, b, kept, counts, new_lens, stream)
                               : keep_dim<EFF_KV_I8>(kv, l, layers, b, kept, counts, new_lens, stream);
}

}  // namespace eff
