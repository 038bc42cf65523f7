// Appending new keys and values to the paged cache, with the norm and the
// position rotation of q and k on the way, and the table the rotation reads.
//
// A row x of a head (q, k):
//   norm      x_i <- x_i * (1 / sqrt(sum x^2 / D + eps)) * w_i            (optional)
//   rotation  the pair (a, b) at position p and frequency i becomes
//             (a cos - b sin, a sin + b cos), cos and sin from the table  (the first rope_dim values)
//             p is the token's place in the cache, or of each pair the token's position
//             on the pair's axis (TURNS)
// k and v rows are then stored as fp16 (round to nearest even), or as int8:
//   scale = max|x| / 127,  n = round(x * (127 / max|x|)), 0 where max|x| < 2^-119.
// Every operation is a separate f32 rounding (no contraction).
#include "eff_device.h"
#include "eff_kv.h"

namespace eff {

// The angle is computed and reduced in 64 bits: at position 10^5 a 32-bit
// product would be off by 10^-3 rad. Made once for a model: the 64-bit sine and cosine
// bound it (131072 positions of 64 pairs 33 us, 2 TB/s written).
__global__ __launch_bounds__(256) void k_rope_table(RopeFreqs f, uint32_t pairs, uint32_t positions, float scale,
                                                    float *__restrict__ out) {
  const uint64_t i = (uint64_t)blockIdx.x * 256u + threadIdx.x;
  if (i >= (uint64_t)pairs * positions) return;
  const uint32_t p = (uint32_t)(i / pairs), j = (uint32_t)(i % pairs);
  double s, c;
  sincos((double)p * f.f[j], &s, &c);
  out[(uint64_t)p * 2u * pairs + j] = (float)(c * (double)scale);
  out[(uint64_t)p * 2u * pairs + pairs + j] = (float)(s * (double)scale);
}

// Sum and maximum over groups of L lanes: DPP within 16, then swaps of 16-lane
// rows and of the wave's halves.
template <int L>
__device__ __forceinline__ float group_sum(float v) {
  v = dpp_row_sum(v);
  if constexpr (L >= 32) {
    auto p = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(p[0]) + __uint_as_float(p[1]);
  }
  if constexpr (L == 64) {
    auto p = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(p[0]) + __uint_as_float(p[1]);
  }
  return v;
}

template <int L>
__device__ __forceinline__ uint32_t group_max(uint32_t v) {
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xF, 0xF, false));
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xF, 0xF, false));
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x141, 0xF, 0xF, false));
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x140, 0xF, 0xF, false));
  if constexpr (L >= 32) {
    auto p = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    v = max((uint32_t)p[0], (uint32_t)p[1]);
  }
  if constexpr (L == 64) {
    auto p = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    v = max((uint32_t)p[0], (uint32_t)p[1]);
  }
  return v;
}

// The lane's 4 values of a row, as its pairs: (0, 1) and (2, 3). `apart`: 2 l and
// 2 l + 1 of each half of the rotated part, else 4 side by side.
__device__ __forceinline__ void load4(float x[4], const float *p, bool apart, uint32_t half, uint32_t l) {
  if (apart) {
    const float2 c = *(const float2 *)(p + 2u * l), d = *(const float2 *)(p + half + 2u * l);
    x[0] = c.x, x[1] = d.x, x[2] = c.y, x[3] = d.y;
  } else {
    const float4 c = *(const float4 *)(p + 4u * l);
    x[0] = c.x, x[1] = c.y, x[2] = c.z, x[3] = c.w;
  }
}

// Where the rotation goes by the token's place in the cache.
struct ByPlace {};

// cos and sin of the lane's pairs 2 l and 2 l + 1, each by its own axis: they do not
// wait for the token's place. A position that the table does not have is not read.
template <typename TURNS>
__device__ __forceinline__ void turn_at(const TURNS &turned, const KvAppendArgs &a, uint32_t t, uint32_t half, uint32_t l, float2 &c, float2 &d) {
  float *cs[2] = {&c.x, &c.y}, *ds[2] = {&d.x, &d.y};
#pragma unroll
  for (uint32_t i = 0; i < 2u; ++i) {
    const uint32_t pair = 2u * l + i, p = turned.at[(uint64_t)turned.axis[pair] * turned.tokens + t];
    const float *row = a.rope + (uint64_t)min(p, turned.positions - 1u) * a.rope_dim + pair;
    const float x = row[0], y = row[half];
    *cs[i] = p < turned.positions ? x : NAN, *ds[i] = p < turned.positions ? y : NAN;
  }
}

// A workgroup takes rows of one token and of one kind (q, k or v: what differs
// between them is then scalar); L lanes take a row, 4 values each: the pairs 2 l
// and 2 l + 1 of the row's D / 2 pairs. Its bytes bound a long append, round trips a
// short one: the token's sequence and then its page are two dependent ones, and a
// thread's U rows are requested before them, so that many tokens keep enough bytes
// under way (us, U = 1 / 4: 4780 tokens of 24 heads of 256 with norms 72.2 / 56.9, 3.9
// TB/s; 4780 of 48 heads of 128 54.4 / 48.8, 4.6 TB/s; 1340 tokens 14.9 / 16.1, 270
// 6.8 / 7.1).
typedef float float2v __attribute__((ext_vector_type(2)));
typedef float float4v __attribute__((ext_vector_type(4)));
template <bool PAST, typename T>
__device__ __forceinline__ void put(T *o, T v) {
  if constexpr (PAST) __builtin_nontemporal_store(v, o);
  else *o = v;
}

// With positions of their own (TURNED) a wave has a team's part instead of a workgroup, so
// that few key heads do not leave the threads of whole workgroups without a row (5 prompts
// of 1531 tokens and fewer, 16 heads of 128 on 2, q/k norm, 100 MB: 37 -> 26 us; with q stored
// past the L2 18.7 us, 5.4 TB/s). Where there are 4 rows a thread q goes past it whatever its
// size: the attention that reads it next gives a part of that back or, from 20 MB of q on, a
// little more. Append and attention of 32 heads of 128 on 8, q past the L2 and through it: 8 x
// 24 drafts over 1000 (3 MB of q) 29.5 and 29.7 us, a prompt of 1000 (16 MB) 48.8 and 49.3, 48
// x 25 drafts over 2000 (20 MB) 134 and 134, over 500 53.6 and 52.4, a prompt of 4000 (66 MB)
// 331 and 328; the append alone 4.9 and 5.6, 8.6 and 9.8, 10.4 and 11.4, 10.0 and 11.1, 27.7
// and 36.8.
template <int TYPE, int D, int U, typename TURNS>
__global__ __launch_bounds__(256) void k_kv_append(KvView kv, KvBatchView b, KvAppendArgs a, uint32_t q_wgs, uint32_t k_wgs, TURNS turned) {
#pragma clang fp contract(off)
  constexpr bool TURNED = !__is_same(TURNS, ByPlace), PAST = TURNED && U == 4;   // q goes past the L2
  constexpr uint32_t L = D == 96 ? 32u : D / 4u, TEAM = TURNED ? 64u : 256u, ROWS = TEAM / L;
  const uint32_t id = TURNED ? __builtin_amdgcn_readfirstlane(blockIdx.x * 4u + (threadIdx.x >> 6)) : blockIdx.x;
  const uint32_t wgs = q_wgs + 2u * k_wgs, t = id / wgs, w = id % wgs, l = (threadIdx.x & 63u) % L;
  if (TURNED && t >= b.tokens) return;
  const bool is_q = w < q_wgs, is_v = w >= q_wgs + k_wgs;
  const uint32_t heads = is_q ? a.q_heads : kv.heads, h0 = (is_q ? w : is_v ? w - q_wgs - k_wgs : w - q_wgs) * ROWS * U + threadIdx.x % TEAM / L;
  const float *src = is_q ? a.q + (uint64_t)t * a.q_stride : is_v ? a.v + (uint64_t)t * a.v_stride : a.k + (uint64_t)t * a.k_stride;
  const float *norm = is_q ? a.q_norm : is_v ? nullptr : a.k_norm;
  const uint32_t half = is_v ? 0u : a.rope_dim / 2u;
  const bool in = D != 96 || l < D / 4u, turns = 2u * l < half, apart = turns && a.halves;
  float x[U][4];
#pragma unroll
  for (uint32_t u = 0; u < U; ++u) {
    x[u][0] = x[u][1] = x[u][2] = x[u][3] = 0.f;
    if (in && h0 + ROWS * u < heads) load4(x[u], src + (h0 + ROWS * u) * D, apart, half, l);
  }
  float weight[4] = {};
  if (norm && in) load4(weight, norm, apart, half, l);
  float2 c = make_float2(1.f, 1.f), d = make_float2(0.f, 0.f);
  if constexpr (TURNED) {
    if (turns) turn_at(turned, a, t, half, l, c, d);
  }
  KvSeq s;
  if (!kv_seq_of(b, t, s)) return;
  const uint32_t back = s.next - t;   // positions from the sequence's end
  const bool placed = back <= s.len;
  const uint32_t pos = placed ? s.len - back : 0u;
  // a page number past the cache holds nothing
  uint32_t page = ~0u;
  if (placed && !is_q) page = b.table[(uint64_t)s.seq * b.table_pages + (pos >> kv.page_log2)];
  if (!TURNED && turns) {
    const float *p = a.rope + (uint64_t)pos * a.rope_dim + 2u * l;
    c = *(const float2 *)p, d = *(const float2 *)(p + half);
  }
  const bool store = is_q || page < kv.pages;
  uint8_t *block = kv.base + (is_q || !store ? 0u : (uint64_t)page * kv.page_bytes + (is_v ? (uint64_t)kv.heads * kv.block_bytes : 0u));
  const uint32_t slot = pos & ((1u << kv.page_log2) - 1u);
#pragma unroll
  for (uint32_t u = 0; u < U; ++u) {
    const uint32_t h = h0 + ROWS * u;
    float *y = x[u];
    if (norm) {
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) sum += y[i] * y[i];
      const float inv = __builtin_amdgcn_rsqf(group_sum<L>(sum) * (1.f / D) + a.eps);   // to one unit in the last place
#pragma unroll
      for (int i = 0; i < 4; ++i) y[i] = y[i] * inv * weight[i];
    }
    if (turns) {
      const float y0 = y[0] * c.x - y[1] * d.x, y1 = y[0] * d.x + y[1] * c.x;
      const float y2 = y[2] * c.y - y[3] * d.y, y3 = y[2] * d.y + y[3] * c.y;
      y[0] = y0, y[1] = y1, y[2] = y2, y[3] = y3;
    }
    const bool on = in && h < heads;
    if (is_q) {
      if (!on) continue;
      float *o = a.q_out + ((uint64_t)t * a.q_heads + h) * D;
      if (!placed) y[0] = y[1] = y[2] = y[3] = 0.f;
      if (apart) {
        put<PAST>((float2v *)(o + 2u * l), float2v{y[0], y[2]}), put<PAST>((float2v *)(o + half + 2u * l), float2v{y[1], y[3]});
      } else {
        put<PAST>((float4v *)(o + 4u * l), float4v{y[0], y[1], y[2], y[3]});
      }
      continue;
    }
    uint8_t *blk = block + (uint64_t)h * kv.block_bytes;
    if constexpr (TYPE == EFF_KV_F16) {
      if (!on || !store) continue;
      typedef _Float16 half2v __attribute__((ext_vector_type(2)));
      _Float16 *o = (_Float16 *)blk + slot * D;
      if (apart) {
        *(half2v *)(o + 2u * l) = half2v{(_Float16)y[0], (_Float16)y[2]};
        *(half2v *)(o + half + 2u * l) = half2v{(_Float16)y[1], (_Float16)y[3]};
      } else {
        *(half4 *)(o + 4u * l) = half4{(_Float16)y[0], (_Float16)y[1], (_Float16)y[2], (_Float16)y[3]};
      }
    } else {
      // the largest magnitude by its bits: a NaN is larger than any number, and
      // makes the row's scale, and so every value of the row, NaN
      uint32_t top = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) top = max(top, __float_as_uint(y[i]) & 0x7FFFFFFFu);
      const float m = __uint_as_float(group_max<L>(top));
      if (!on || !store) continue;
      // the smallest rows' 127 / m would pass the largest number: they become zeros
      const float inv = m >= 0x1p-119f ? 127.f / m : 0.f;
      int8_t *o = (int8_t *)blk + slot * D;
      uint32_t q[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) q[i] = (uint32_t)(int)__builtin_amdgcn_fmed3f(rintf(y[i] * inv), -127.f, 127.f) & 0xFFu;   // a NaN too
      if (apart) {
        *(uint16_t *)(o + 2u * l) = (uint16_t)(q[0] | q[2] << 8), *(uint16_t *)(o + half + 2u * l) = (uint16_t)(q[1] | q[3] << 8);
      } else {
        *(uint32_t *)(o + 4u * l) = q[0] | q[1] << 8 | q[2] << 16 | q[3] << 24;
      }
      if (l == 0u) ((float *)(blk + ((uint64_t)D << kv.page_log2)))[slot] = m * (1.f / 127.f);
    }
  }
}

hipError_t launch_rope_table(const RopeFreqs &f, uint32_t pairs, uint32_t positions, float scale, float *out,
                             hipStream_t stream) {
  const uint64_t n = (uint64_t)pairs * positions;
  if (!fits((n + 255u) / 256u, 256u)) return hipErrorInvalidConfiguration;
  hipLaunchKernelGGL(k_rope_table, dim3((uint32_t)((n + 255u) / 256u)), dim3(256), 0, stream, f, pairs, positions,
                     scale, out);
  return hipGetLastError();
}

template <int TYPE, int D, int U, typename TURNS>
static hipError_t append_launch(const KvView &kv, const KvBatchView &b, const KvAppendArgs &a, const TURNS &turned, hipStream_t s) {
  constexpr uint32_t teams = __is_same(TURNS, ByPlace) ? 1u : 4u;         // of a workgroup
  constexpr uint32_t rows = (D == 96 ? 8u : 1024u / D) * U / teams;   // of a team
  const uint32_t q = (a.q_heads + rows - 1u) / rows, k = (kv.heads + rows - 1u) / rows;
  const uint64_t wgs = ((uint64_t)b.tokens * (q + 2u * k) + teams - 1u) / teams;
  if (!fits(wgs, 256u)) return hipErrorInvalidConfiguration;
  hipLaunchKernelGGL((k_kv_append<TYPE, D, U, TURNS>), dim3((uint32_t)wgs), dim3(256), 0, s, kv, b, a, q, k, turned);
  return hipGetLastError();
}

template <int TYPE, int D, typename TURNS>
static hipError_t append_dim(const KvView &kv, const KvBatchView &b, const KvAppendArgs &a, const TURNS &turned, hipStream_t s) {
  // 4 rows a thread where a CU still has 8 workgroups to take; of waves by themselves, from
  // two workgroups on (32 heads of 128 on 8: 250 tokens 5.3 us, one row a thread 5.6, 500
  // 6.9 and 8.7, 100 5.0 and 4.9)
  const uint64_t from = __is_same(TURNS, ByPlace) ? 2048ull * 4096u : 2048ull * 512u;
  if ((uint64_t)b.tokens * (a.q_heads + 2u * kv.heads) * D >= from) return append_launch<TYPE, D, 4>(kv, b, a, turned, s);
  return append_launch<TYPE, D, 1>(kv, b, a, turned, s);
}

template <int TYPE, typename TURNS>
static hipError_t append_go(const KvView &kv, const KvBatchView &b, const KvAppendArgs &a, const TURNS &turned, hipStream_t s) {
  switch (kv.dim) {
    case 64: return append_dim<TYPE, 64>(kv, b, a, turned, s);
    case 96: return append_dim<TYPE, 96>(kv, b, a, turned, s);
    case 128: return append_dim<TYPE, 128>(kv, b, a, turned, s);
    case 256: return append_dim<TYPE, 256>(kv, b, a, turned, s);
    default: return hipErrorInvalidValue;
  }
}

hipError_t launch_kv_append(const KvView &kv, const KvBatchView &b, const KvAppendArgs &a, const KvTurnsView *turns, hipStream_t stream) {
  if (turns) return kv.type == EFF_KV_F16 ? append_go<EFF_KV_F16>(kv, b, a, *turns, stream) : append_go<EFF_KV_I8>(kv, b, a, *turns, stream);
  return kv.type == EFF_KV_F16 ? append_go<EFF_KV_F16>(kv, b, a, ByPlace{}, stream) : append_go<EFF_KV_I8>(kv, b, a, ByPlace{}, stream);
}

}  // namespace eff
