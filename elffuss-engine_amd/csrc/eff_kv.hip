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
// pairs 2 l and 2 l + 1 of the row's D / 2 pairs.
template <int TYPE, int D>
__global__ __launch_bounds__(256) void k_kv_append(KvView kv, KvBatchView b, KvAppendArgs a, uint32_t wgs) {
#pragma clang fp contract(off)
  constexpr uint32_t L = D == 96 ? 32u : D / 4u, ROWS = 256u / L;
  const uint32_t t = blockIdx.x / wgs, lane = threadIdx.x & 63u, l = lane % L;
  const uint32_t heads = a.q_heads + 2u * kv.heads;
  const uint32_t r = (blockIdx.x % wgs) * ROWS + threadIdx.x / L;
  const uint32_t s = kv_seq_of(b, t);
  if (s >= b.seqs) return;
  const uint32_t n = b.starts[s + 1] - b.starts[s], len = kv_len(b, s), back = n - (t - b.starts[s]);
  const bool on = r < heads && l < D / 4u, placed = back <= len;
  const uint32_t pos = placed ? len - back : 0u;
  const bool is_q = r < a.q_heads, is_v = r >= a.q_heads + kv.heads;
  const uint32_t h = is_q ? r : is_v ? r - a.q_heads - kv.heads : r - a.q_heads;
  const float *src = is_q ? a.q + (uint64_t)t * a.q_stride : is_v ? a.v + (uint64_t)t * a.v_stride
                                                                  : a.k + (uint64_t)t * a.k_stride;
  // the places of the lane's pairs: (i0, j0) and (i0 + step, j0 + step)
  const uint32_t half = a.rope_dim / 2u;
  const bool split = !is_v && a.halves && 2u * l < half;
  const uint32_t i0 = split ? 2u * l : 4u * l, j0 = split ? half + 2u * l : 4u * l + 1u;
  float x[4] = {};   // pair 0, pair 1
  if (on) {
    if (split) {
      const float2 u = *(const float2 *)(src + h * D + i0), w = *(const float2 *)(src + h * D + j0);
      x[0] = u.x, x[1] = w.x, x[2] = u.y, x[3] = w.y;
    } else {
      const float4 u = *(const float4 *)(src + h * D + i0);
      x[0] = u.x, x[1] = u.y, x[2] = u.z, x[3] = u.w;
    }
  }
  const uint32_t step = split ? 1u : 2u;
  const float *w = is_q ? a.q_norm : is_v ? nullptr : a.k_norm;
  if (w != nullptr) {
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) sum += x[i] * x[i];
    sum = group_sum<L>(sum);
    const float inv = 1.f / sqrtf(sum / (float)D + a.eps);
    if (on) {
      x[0] = x[0] * inv * w[i0], x[1] = x[1] * inv * w[j0];
      x[2] = x[2] * inv * w[i0 + step], x[3] = x[3] * inv * w[j0 + step];
    }
  }
  if (!is_v && on && 2u * l < half) {
    const float *cs = a.rope + (uint64_t)pos * a.rope_dim + 2u * l;
    const float2 c = *(const float2 *)cs, sn = *(const float2 *)(cs + half);
    const float y0 = x[0] * c.x - x[1] * sn.x, y1 = x[0] * sn.x + x[1] * c.x;
    const float y2 = x[2] * c.y - x[3] * sn.y, y3 = x[2] * sn.y + x[3] * c.y;
    x[0] = y0, x[1] = y1, x[2] = y2, x[3] = y3;
  }
  if (is_q) {
    if (!on) return;
    float *o = a.q_out + ((uint64_t)t * a.q_heads + h) * D;
    if (!placed) x[0] = x[1] = x[2] = x[3] = 0.f;
    if (split) {
      *(float2 *)(o + i0) = make_float2(x[0], x[2]);
      *(float2 *)(o + j0) = make_float2(x[1], x[3]);
    } else {
      *(float4 *)(o + i0) = make_float4(x[0], x[1], x[2], x[3]);
    }
    return;
  }
  // a page number past the cache holds nothing
  const uint32_t page = placed ? b.table[(uint64_t)s * b.table_pages + (pos >> kv.page_log2)] : ~0u;
  const uint32_t slot = pos & ((1u << kv.page_log2) - 1u);
  const bool store = on && page < kv.pages;
  uint8_t *blk = kv.base + (store ? (uint64_t)page * kv.page_bytes + (uint64_t)((is_v ? kv.heads : 0u) + h) * kv.block_bytes : 0u);
  if constexpr (TYPE == EFF_KV_F16) {
    if (!store) return;
    _Float16 *o = (_Float16 *)blk + slot * D;
    if (split) {
      o[i0] = (_Float16)x[0], o[i0 + 1] = (_Float16)x[2], o[j0] = (_Float16)x[1], o[j0 + 1] = (_Float16)x[3];
    } else {
#pragma unroll
      for (uint32_t i = 0; i < 4u; ++i) o[i0 + i] = (_Float16)x[i];
    }
  } else {
    // the largest magnitude by its bits: a NaN is larger than any number, and
    // makes the row's scale, and so every value of the row, NaN
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) top = max(top, __float_as_uint(x[i]) & 0x7FFFFFFFu);
    const float m = __uint_as_float(group_max<L>(top));
    if (!store) return;
    const float inv = m > 0.f ? 127.f / m : 0.f;
    int8_t *o = (int8_t *)blk + slot * D;
    int8_t q[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float y = rintf(x[i] * inv);
      q[i] = (int8_t)(int)(y >= -127.f && y <= 127.f ? y : 0.f);
    }
    o[i0] = q[0], o[j0] = q[1], o[i0 + step] = q[2], o[j0 + step] = q[3];
    if (l == 0u) ((float *)(blk + ((uint64_t)D << kv.page_log2)))[slot] = m * (1.f / 127.f);
  }
}

hipError_t launch_rope_table(const RopeFreqs &f, uint32_t pairs, uint32_t positions, float scale, float *out,
                             hipStream_t stream) {
  const uint64_t n = (uint64_t)pairs * positions;
  hipLaunchKernelGGL(k_rope_table, dim3((uint32_t)((n + 255u) / 256u)), dim3(256), 0, stream, f, pairs, positions,
                     scale, out);
  return hipGetLastError();
}

template <int TYPE>
static hipError_t append_go(const KvView &kv, const KvBatchView &b, const KvAppendArgs &a, hipStream_t s) {
  const uint32_t rows = kv.dim == 96u ? 8u : 1024u / kv.dim;   // of a workgroup
  const uint32_t wgs = (a.q_heads + 2u * kv.heads + rows - 1u) / rows;
  const dim3 grid(b.tokens * wgs);
  switch (kv.dim) {
    case 64: hipLaunchKernelGGL((k_kv_append<TYPE, 64>), grid, dim3(256), 0, s, kv, b, a, wgs); break;
    case 96: hipLaunchKernelGGL((k_kv_append<TYPE, 96>), grid, dim3(256), 0, s, kv, b, a, wgs); break;
    case 128: hipLaunchKernelGGL((k_kv_append<TYPE, 128>), grid, dim3(256), 0, s, kv, b, a, wgs); break;
    case 256: hipLaunchKernelGGL((k_kv_append<TYPE, 256>), grid, dim3(256), 0, s, kv, b, a, wgs); break;
    default: return hipErrorInvalidValue;
  }
  return hipGetLastError();
}

hipError_t launch_kv_append(const KvView &kv, const KvBatchView &b, const KvAppendArgs &a, hipStream_t stream) {
  return kv.type == EFF_KV_F16 ? append_go<EFF_KV_F16>(kv, b, a, stream) : append_go<EFF_KV_I8>(kv, b, a, stream);
}

}  // namespace eff
