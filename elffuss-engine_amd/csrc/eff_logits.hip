// Rules on the logits of a batch, before its sampler: for a token v that is
// c > 0 times in the row's history
//   z <- z > 0 ? z / repeat : z * repeat,  z <- z - (frequency * c + presence),
// then z <- z + bias(v), then -inf where the row's mask has no bit for v. The
// first two steps are computed in 64 bits and rounded to 32 after each, as the
// host's sampler does (a Float32Array of logits, 64-bit numbers).
#include "eff_device.h"
#include "eff_kv.h"

namespace eff {

constexpr uint32_t kTile = 4096;   // tokens of the vocabulary that a workgroup takes

__global__ __launch_bounds__(256) void k_logits(LogitsArgs a) {
#pragma clang fp contract(off)
  __shared__ uint32_t count[kTile], bias[kTile];
  const uint32_t tiles = (a.vocab + kTile - 1u) / kTile;
  const uint32_t row = blockIdx.x / tiles, v0 = (blockIdx.x % tiles) * kTile, n = min(kTile, a.vocab - v0);
  for (uint32_t i = threadIdx.x; i < kTile; i += 256u) count[i] = bias[i] = 0u;
  __syncthreads();
  if (a.history) {
    const uint32_t e = min(a.history_starts[row + 1], a.history_count);
    for (uint32_t i = a.history_starts[row] + threadIdx.x; i < e; i += 256u) {
      const uint32_t v = a.history[i] - v0;
      if (v < n) atomicAdd(&count[v], 1u);
    }
  }
  if (a.bias_ids) {
    // of several pairs of one id the last counts: the largest place in the list
    const uint32_t e = min(a.bias_starts[row + 1], a.bias_count);
    for (uint32_t i = a.bias_starts[row] + threadIdx.x; i < e; i += 256u) {
      const uint32_t v = a.bias_ids[i] - v0;
      if (v < n) atomicMax(&bias[v], i + 1u);
    }
  }
  __syncthreads();
  const uint32_t m = a.mask ? a.mask_of[row] : ~0u;
  const uint32_t *bits = m < a.mask_count ? a.mask + (uint64_t)m * ((a.vocab + 31u) / 32u) : nullptr;
  const float *in = a.in + (uint64_t)row * a.stride + v0;
  float *out = a.out + (uint64_t)row * a.stride + v0;
  for (uint32_t i = threadIdx.x; i < n; i += 256u) {
    float z = in[i];
    if (count[i]) {
      const double *p = a.penalties + 3u * (uint64_t)row;
      if (p[0] != 1.0) z = (float)(z > 0.f ? (double)z / p[0] : (double)z * p[0]);
      z = (float)((double)z - (p[1] * (double)count[i] + p[2]));
    }
    if (bias[i]) z += a.bias_values[bias[i] - 1u];
    if (bits && !((bits[(v0 + i) >> 5] >> ((v0 + i) & 31u)) & 1u)) z = -INFINITY;
    out[i] = z;
  }
}

hipError_t launch_logits(const LogitsArgs &a, hipStream_t stream) {
  hipLaunchKernelGGL(k_logits, dim3((a.vocab + kTile - 1u) / kTile * a.rows), dim3(256), 0, stream, a);
  return hipGetLastError();
}

}  // namespace eff
