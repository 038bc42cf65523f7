// Appending new keys and values to the paged cache, with the norm and the
// position rotation of q and k on the way, and the table the rotation reads.
//
// A row x of a head (q, k):
//   norm      x_i <- x_i * (1 / sqrt(sum x^2 / D + eps)) * w_i            (optional)
//   rotation  the pair (a, b) at position p and frequency i becomes
//             (a cos - b sin, a sin + b cos), cos and sin from the table  (the first rope_dim values)
// k and v rows are then stored as fp16 (round to nearest even), or as int8:
//   scale = max|x| / 127,  n = round(x * (127 / max|x|)).
// Every operation is a separate f32 rounding (no contraction).
#include "eff_device.h"
#include "eff_kv.h"

namespace eff {

// The angle is computed and reduced in 64 bits: at position 10^5 a 32-bit
// product would be off by 10^-3 rad.
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

template <int L>
__device__ __forceinline__ float group_sum(float v) {
#pragma unroll
  for (int o = 1; o < L; o <<= 1) v += __shfl_xor(v, o);
  return v;
}

template <int L>
__device__ __forceinline__ uint32_t group_max(uint32_t v) {
#pragma unroll
  for (int o = 1; o < L; o <<= 1) v = max(v, (uint32_t)__shfl_xor((int)v, o));
  return v;
}

// A workgroup takes rows of one token; L lanes take a row, 4 values each: the
// pairs 2 l and 2 l + 1 of the row's D / 2 pairs. The token's sequence and page are
// two dependent round trips; a thread's U rows are requested before them, so that
// many tokens keep enough bytes under way (7 prompts of up to 1021 tokens of 24
// heads of 256: U = 1 77 us, 4 WAIT_FOR_MEASUREMENT).
template <int TYPE, int D, int U>
__global__ __launch_bounds__(256) void k_kv_append(KvView kv, KvBatchView b, KvAppendArgs a, uint32_t wgs) {
#pragma clang fp contract(off)
  constexpr uint32_t L = D == 96 ? 32u : D / 4u, ROWS = 256u / L;
  const uint32_t t = blockIdx.x / wgs, l = (threadIdx.x & 63u) % L;
  const uint32_t heads = a.q_heads + 2u * kv.heads, r0 = (blockIdx.x % wgs) * ROWS * U + threadIdx.x / L;
  const uint32_t half = a.rope_dim / 2u;
  // the places of the lane's pairs: (i0, j0) and (i0 + step, j0 + step); v rows
  // take the unsplit ones
  const bool turns = 2u * l < half, apart = turns && a.halves;
  float x[U][4];
#pragma unroll
  for (uint32_t u = 0; u < U; ++u) {
    const uint32_t r = r0 + ROWS * u;
    const bool is_q = r < a.q_heads, is_v = r >= a.q_heads + kv.heads;
    const uint32_t h = is_q ? r : is_v ? r - a.q_heads - kv.heads : r - a.q_heads;
    const float *src = (is_q ? a.q + (uint64_t)t * a.q_stride : is_v ? a.v + (uint64_t)t * a.v_stride : a.k + (uint64_t)t * a.k_stride) + h * D;
    x[u][0] = x[u][1] = x[u][2] = x[u][3] = 0.f;
    if (r < heads && l < D / 4u) {
      if (apart && !is_v) {
        const float2 c = *(const float2 *)(src + 2u * l), d = *(const float2 *)(src + half + 2u * l);
        x[u][0] = c.x, x[u][1] = d.x, x[u][2] = c.y, x[u][3] = d.y;
      } else {
        const float4 c = *(const float4 *)(src + 4u * l);
        x[u][0] = c.x, x[u][1] = c.y, x[u][2] = c.z, x[u][3] = c.w;
      }
    }
  }
  KvSeq s;
  if (!kv_seq_of(b, t, s)) return;
  const uint32_t back = s.next - t;   // positions from the sequence's end
  const bool placed = back <= s.len;
  const uint32_t pos = placed ? s.len - back : 0u;
  // a page number past the cache holds nothing
  const uint32_t page = placed ? b.table[(uint64_t)s.seq * b.table_pages + (pos >> kv.page_log2)] : ~0u;
  const uint32_t slot = pos & ((1u << kv.page_log2) - 1u);
  float2 cs = make_float2(1.f, 1.f), sn = make_float2(0.f, 0.f);
  if (turns) {
    const float *p = a.rope + (uint64_t)pos * a.rope_dim + 2u * l;
    cs = *(const float2 *)p, sn = *(const float2 *)(p + half);
  }
#pragma unroll
  for (uint32_t u = 0; u < U; ++u) {
    const uint32_t r = r0 + ROWS * u;
    const bool on = r < heads && l < D / 4u, is_q = r < a.q_heads, is_v = r >= a.q_heads + kv.heads;
    const uint32_t h = is_q ? r : is_v ? r - a.q_heads - kv.heads : r - a.q_heads;
    const bool split = apart && !is_v;
    const uint32_t i0 = split ? 2u * l : 4u * l, j0 = split ? half + 2u * l : 4u * l + 1u, step = split ? 1u : 2u;
    const float *w = is_q ? a.q_norm : is_v ? nullptr : a.k_norm;
    if (w != nullptr) {
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) sum += x[u][i] * x[u][i];
      sum = group_sum<L>(sum);
      const float inv = 1.f / sqrtf(sum / (float)D + a.eps);
      if (on) {
        x[u][0] = x[u][0] * inv * w[i0], x[u][1] = x[u][1] * inv * w[j0];
        x[u][2] = x[u][2] * inv * w[i0 + step], x[u][3] = x[u][3] * inv * w[j0 + step];
      }
    }
    if (!is_v && turns) {
      const float y0 = x[u][0] * cs.x - x[u][1] * sn.x, y1 = x[u][0] * sn.x + x[u][1] * cs.x;
      const float y2 = x[u][2] * cs.y - x[u][3] * sn.y, y3 = x[u][2] * sn.y + x[u][3] * cs.y;
      x[u][0] = y0, x[u][1] = y1, x[u][2] = y2, x[u][3] = y3;
    }
    if (is_q) {
      if (!on) continue;
      float *o = a.q_out + ((uint64_t)t * a.q_heads + h) * D;
      if (!placed) x[u][0] = x[u][1] = x[u][2] = x[u][3] = 0.f;
      if (split) {
        *(float2 *)(o + i0) = make_float2(x[u][0], x[u][2]);
        *(float2 *)(o + j0) = make_float2(x[u][1], x[u][3]);
      } else {
        *(float4 *)(o + i0) = make_float4(x[u][0], x[u][1], x[u][2], x[u][3]);
      }
      continue;
    }
    const bool store = on && page < kv.pages;
    uint8_t *blk = kv.base + (store ? (uint64_t)page * kv.page_bytes + (uint64_t)((is_v ? kv.heads : 0u) + h) * kv.block_bytes : 0u);
    if constexpr (TYPE == EFF_KV_F16) {
      if (!store) continue;
      typedef _Float16 half2v __attribute__((ext_vector_type(2)));
      _Float16 *o = (_Float16 *)blk + slot * D;
      if (split) {
        *(half2v *)(o + i0) = half2v{(_Float16)x[u][0], (_Float16)x[u][2]};
        *(half2v *)(o + j0) = half2v{(_Float16)x[u][1], (_Float16)x[u][3]};
      } else {
        *(half4 *)(o + i0) = half4{(_Float16)x[u][0], (_Float16)x[u][1], (_Float16)x[u][2], (_Float16)x[u][3]};
      }
    } else {
      // the largest magnitude by its bits: a NaN is larger than any number, and
      // makes the row's scale, and so every value of the row, NaN
      uint32_t top = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) top = max(top, __float_as_uint(x[u][i]) & 0x7FFFFFFFu);
      const float m = __uint_as_float(group_max<L>(top));
      if (!store) continue;
      const float inv = m > 0.f ? 127.f / m : 0.f;
      int8_t *o = (int8_t *)blk + slot * D;
      uint32_t q[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float y = rintf(x[u][i] * inv);
        q[i] = (uint32_t)(int)(y >= -127.f && y <= 127.f ? y : 0.f) & 0xFFu;
      }
      if (split) {
        *(uint16_t *)(o + i0) = (uint16_t)(q[0] | q[2] << 8), *(uint16_t *)(o + j0) = (uint16_t)(q[1] | q[3] << 8);
      } else {
        *(uint32_t *)(o + i0) = q[0] | q[1] << 8 | q[2] << 16 | q[3] << 24;
      }
      if (l == 0u) ((float *)(blk + ((uint64_t)D << kv.page_log2)))[slot] = m * (1.f / 127.f);
    }
  }
}

hipError_t launch_rope_table(const RopeFreqs &f, uint32_t pairs, uint32_t positions, float scale, float *out,
                             hipStream_t stream) {
  const uint64_t n = (uint64_t)pairs * positions;
  hipLaunchKernelGGL(k_rope_table, dim3((uint32_t)((n + 255u) / 256u)), dim3(256), 0, stream, f, pairs, positions,
                     scale, out);
  return hipGetLastError();
}

template <int TYPE, int D>
static hipError_t append_dim(const KvView &kv, const KvBatchView &b, const KvAppendArgs &a, hipStream_t s) {
  constexpr uint32_t rows = D == 96 ? 8u : 1024u / D;   // of a workgroup, U = 1
  const uint32_t heads = a.q_heads + 2u * kv.heads;
  // 4 rows a thread where that still gives a CU 8 workgroups
  const uint32_t one = (heads + rows - 1u) / rows, four = (heads + 4u * rows - 1u) / (4u * rows);
  if ((uint64_t)b.tokens * four >= 2048u)
    hipLaunchKernelGGL((k_kv_append<TYPE, D, 4>), dim3(b.tokens * four), dim3(256), 0, s, kv, b, a, four);
  else
    hipLaunchKernelGGL((k_kv_append<TYPE, D, 1>), dim3(b.tokens * one), dim3(256), 0, s, kv, b, a, one);
  return hipGetLastError();
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
