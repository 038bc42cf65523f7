// Attention of new tokens over the paged cache.
//
//   s_t = scale * q . k_t  for the tokens t the row sees: those up to its own
//         position, the last `window` of them if there is one
//   out = sum_t softmax(s)_t v_t;  a row that sees nothing is zeros
// The softmax is taken in one pass with the running maximum and sum.
#include "eff_device.h"
#include "eff_kv.h"

namespace eff {

// One workgroup per row (new token and query head): a wave per cached token,
// the lanes over the head's values.
template <int TYPE, int D>
__global__ __launch_bounds__(256) void k_attn(KvView kv, KvBatchView b, KvAttnArgs a) {
  constexpr int N = (D + 63) / 64;
  __shared__ float sm[4], sl[4], so[4][D];
  const uint32_t t = blockIdx.y, h = blockIdx.x, lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
  const uint32_t kvh = h / (a.q_heads / kv.heads);
  const uint32_t s = kv_seq_of(b, t);
  if (s >= b.seqs) return;
  const uint32_t n = b.starts[s + 1] - b.starts[s], len = kv_len(b, s), back = n - (t - b.starts[s]);
  const uint32_t end = back <= len ? len - back + 1u : 0u;   // the row sees [first, end)
  const uint32_t first = a.window && end > a.window ? end - a.window : 0u;
  float q[N], o[N], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const uint32_t d = lane + 64u * i;
    q[i] = d < (uint32_t)D ? a.q[(uint64_t)t * a.q_stride + h * D + d] * a.scale : 0.f;
    o[i] = 0.f;
  }
  for (uint32_t p = first + wave; p < end; p += 4u) {
    const uint32_t page = b.table[(uint64_t)s * b.table_pages + (p >> kv.page_log2)];
    if (page >= kv.pages) continue;
    const uint32_t slot = p & ((1u << kv.page_log2) - 1u);
    const uint8_t *kb = kv.base + (uint64_t)page * kv.page_bytes + (uint64_t)kvh * kv.block_bytes;
    const uint8_t *vb = kb + (uint64_t)kv.heads * kv.block_bytes;
    float k[N], v[N], dot = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const uint32_t d = lane + 64u * i, at = slot * D + (d < (uint32_t)D ? d : 0u);
      if constexpr (TYPE == EFF_KV_F16) {
        k[i] = (float)((const _Float16 *)kb)[at];
        v[i] = (float)((const _Float16 *)vb)[at];
      } else {
        const uint64_t so = (uint64_t)D << kv.page_log2;
        k[i] = (float)((const int8_t *)kb)[at] * ((const float *)(kb + so))[slot];
        v[i] = (float)((const int8_t *)vb)[at] * ((const float *)(vb + so))[slot];
      }
      if (d < (uint32_t)D) dot += q[i] * k[i];
    }
    dot = wave_sum(dot);
    const float mn = fmaxf(m, dot), al = m == mn ? 1.f : expf(m - mn), w = mn == -INFINITY ? 0.f : expf(dot - mn);
    l = l * al + w;
#pragma unroll
    for (int i = 0; i < N; ++i) o[i] = o[i] * al + w * v[i];
    m = mn;
  }
  if (lane == 0u) sm[wave] = m, sl[wave] = l;
#pragma unroll
  for (int i = 0; i < N; ++i)
    if (lane + 64u * i < (uint32_t)D) so[wave][lane + 64u * i] = o[i];
  __syncthreads();
  float mm = -INFINITY;
  for (int w = 0; w < 4; ++w) mm = fmaxf(mm, sm[w]);
  for (uint32_t d = threadIdx.x; d < (uint32_t)D; d += 256u) {
    float sum = 0.f, tot = 0.f;
    for (int w = 0; w < 4; ++w) {
      const float f = sm[w] == -INFINITY ? 0.f : expf(sm[w] - mm);
      tot += f * sl[w];
      sum += f * so[w][d];
    }
    a.out[((uint64_t)t * a.q_heads + h) * D + d] = tot == 0.f ? 0.f : sum / tot;
  }
}

template <int TYPE>
static hipError_t attn_go(const KvView &kv, const KvBatchView &b, const KvAttnArgs &a, hipStream_t s) {
  const dim3 grid(a.q_heads, b.tokens);
  switch (kv.dim) {
    case 64: hipLaunchKernelGGL((k_attn<TYPE, 64>), grid, dim3(256), 0, s, kv, b, a); break;
    case 96: hipLaunchKernelGGL((k_attn<TYPE, 96>), grid, dim3(256), 0, s, kv, b, a); break;
    case 128: hipLaunchKernelGGL((k_attn<TYPE, 128>), grid, dim3(256), 0, s, kv, b, a); break;
    case 256: hipLaunchKernelGGL((k_attn<TYPE, 256>), grid, dim3(256), 0, s, kv, b, a); break;
    default: return hipErrorInvalidValue;
  }
  return hipGetLastError();
}

hipError_t launch_kv_attn(const KvView &kv, const KvBatchView &b, const KvAttnArgs &a, hipStream_t stream) {
  return kv.type == EFF_KV_F16 ? attn_go<EFF_KV_F16>(kv, b, a, stream) : attn_go<EFF_KV_I8>(kv, b, a, stream);
}

}  // namespace eff
