// Appending new keys and values to the paged cache, with the norm and the
// position rotation of q and k on the way, and the table the rotation reads.
//
// A row x of a head (q, k):
//   norm      x_i <- x_i * (1 / sqrt(sum x^2 / D + eps)) * w_i            (optional)
//   rotation  the pair (a, b) at position p and frequency i becomes
//             (a cos - b sin, a sin + b cos), cos and sin from the table  (the first rope_dim values)
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

// A workgroup takes rows of one token and of one kind (q, k or v: what differs
// between them is then scalar); L lanes take a row, 4 values each: the pairs 2 l
// and 2 l + 1 of the row's D / 2 pairs. Its bytes bound a long append, round trips a
// short one: the token's sequence and then its page are two dependent ones, and a
// thread's U rows are requested before them, so that many tokens keep enough bytes
// under way (us, U = 1 / 4: 4780 tokens of 24 heads of 256 with norms 72.2 / 56.9, 3.9
// TB/s; 4780 of 48 heads of 128 54.4 / 48.8, 4.6 TB/s; 1340 tokens 14.9 / 16.1, 270
// 6.8 / 7.1).
template <int TYPE, int D, int U>
__global__ __launch_bounds__(256) void k_kv_append(KvView kv, KvBatchView b, KvAppendArgs a, uint32_t q_wgs, uint32_t k_wgs) {
#pragma clang fp contract(off)
  constexpr uint32_t L = D == 96 ? 32u : D / 4u, ROWS = 256u / L;
  const uint32_t wgs = q_wgs + 2u * k_wgs, t = blockIdx.x / wgs, w = blockIdx.x % wgs, l = (threadIdx.x & 63u) % L;
  const bool is_q = w < q_wgs, is_v = w >= q_wgs + k_wgs;
  const uint32_t heads = is_q ? a.q_heads : kv.heads, h0 = (is_q ? w : is_v ? w - q_wgs - k_wgs : w - q_wgs) * ROWS * U + threadIdx.x / L;
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
  KvSeq s;
  if (!kv_seq_of(b, t, s)) return;
  const uint32_t back = s.next - t;   // positions from the sequence's end
  const bool placed = back <= s.len;
  const uint32_t pos = placed ? s.len - back : 0u;
  // a page number past the cache holds nothing
  uint32_t page = ~0u;
  if (placed && !is_q) page = b.table[(uint64_t)s.seq * b.table_pages + (pos >> kv.page_log2)];
  float2 c = make_float2(1.f, 1.f), d = make_float2(0.f, 0.f);
  if (turns) {
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
        *(float2 *)(o + 2u * l) = make_float2(y[0], y[2]), *(float2 *)(o + half + 2u * l) = make_float2(y[1], y[3]);
      } else {
        *(float4 *)(o + 4u * l) = make_float4(y[0], y[1], y[2], y[3]);
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

template <int TYPE, int D, int U>
static hipError_t append_launch(const KvView &kv, const KvBatchView &b, const KvAppendArgs &a, hipStream_t s) {
  constexpr uint32_t rows = (D == 96 ? 8u : 1024u / D) * U;   // of a workgroup
  const uint32_t q = (a.q_heads + rows - 1u) / rows, k = (kv.heads + rows - 1u) / rows;
  if (!fits((uint64_t)b.tokens * (q + 2u * k), 256u)) return hipErrorInvalidConfiguration;
  hipLaunchKernelGGL((k_kv_append<TYPE, D, U>), dim3(b.tokens * (q + 2u * k)), dim3(256), 0, s, kv, b, a, q, k);
  return hipGetLastError();
}

template <int TYPE, int D>
static hipError_t append_dim(const KvView &kv, const KvBatchView &b, const KvAppendArgs &a, hipStream_t s) {
  // 4 rows a thread where a CU still has 8 workgroups to take
  if ((uint64_t)b.tokens * (a.q_heads + 2u * kv.heads) * D >= 2048ull * 4096u) return append_launch<TYPE, D, 4>(kv, b, a, s);
  return append_launch<TYPE, D, 1>(kv, b, a, s);
}

template <int TYPE>
static hipError_t append_go(const KvView &kv, const KvBatchView &b, const KvAppendArgs &a, hipStream_t s) {
  switch (kv.dim) {
    case 64: return append_dim<TYPE, 64>(kv, b, a, s);
    case 96: return append_dim<TYPE, 96>(kv, b, a, s);
    case 128: return append_dim<TYPE, 128>(kv, b, a, s);
    case 256: return append_dim<TYPE, 256>(kv, b, a, s);
    default: return hipErrorInvalidValue;
  }
}

hipError_t launch_kv_append(const KvView &kv, const KvBatchView &b, const KvAppendArgs &a, hipStream_t stream) {
  return kv.type == EFF_KV_F16 ? append_go<EFF_KV_F16>(kv, b, a, stream) : append_go<EFF_KV_I8>(kv, b, a, stream);
}

}  // namespace eff
