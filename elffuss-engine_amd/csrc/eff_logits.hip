// Rules on the logits of a batch, before its sampler: for a token v that is
// c > 0 times in the row's history
//   z <- z > 0 ? z / repeat : z * repeat,  z <- z - (frequency * c + presence),
// then z <- z + bias(v), then -inf where the row's mask has no bit for v. The
// first two steps are computed in 64 bits and rounded to 32 after each, as the
// host's sampler does (a Float32Array of logits, 64-bit numbers).
//
// A workgroup takes a tile of a row into LDS, requested before the history, the
// biases and the mask so that the round trips overlap (32 rows of 131072: 12.4 -> 10.9
// us, 48 of 50021 with masks 13.3 -> 11.9); it reads the whole history, counts the ids
// of its tile in LDS (whole numbers: any order gives the same counts), and then changes
// the logits that have one. The tile passes through once: the bytes of the logits bound
// a batch (200 x 150001: 47 us, 5.1 TB/s), the round trips a single row (5 us, a launch
// alone 3.4), the reading of a long history by every tile of the row the rest.
#include "eff_device.h"
#include "eff_kv.h"

namespace eff {

constexpr uint32_t kThreads = 1024, kItems = 2;   // of a workgroup; groups of 4 logits of a thread

// Rows start wherever the stride puts them: 4-byte aligned.
typedef float float4u __attribute__((ext_vector_type(4), aligned(4)));

// The ids from `a` to `e` of a list, 4 of a thread under way at a time: the first are
// requested by start(). f(i, id); past the end the id is ~0, past every vocabulary.
struct Ids {
  static constexpr uint32_t U = 4;
  const uint32_t *list;
  uint32_t a, e, id[U];

  __device__ __forceinline__ void load(uint32_t *o, uint32_t i) const {
#pragma unroll
    for (uint32_t k = 0; k < U; ++k) o[k] = i + kThreads * k < e ? list[i + kThreads * k] : ~0u;
  }
  __device__ __forceinline__ void start(const uint32_t *from, uint32_t first, uint32_t end) {
    list = from, a = first, e = end;
    load(id, a + threadIdx.x);
  }
  template <typename F>
  __device__ __forceinline__ void each(F f) {
    uint32_t i = a + threadIdx.x;
    for (uint32_t at = a; at < e; at += kThreads * U, i += kThreads * U) {
      uint32_t next[U];
      load(next, i + kThreads * U);
#pragma unroll
      for (uint32_t k = 0; k < U; ++k) f(i + kThreads * k, id[k]), id[k] = next[k];
    }
  }
};

__global__ __launch_bounds__(kThreads) void k_logits(LogitsArgs a, uint32_t tiles) {
#pragma clang fp contract(off)
  constexpr uint32_t T = 4u * kThreads * kItems;
  __shared__ __align__(16) float z[T];
  __shared__ __align__(16) uint32_t count[T];
  const uint32_t row = blockIdx.x / tiles, v0 = (blockIdx.x % tiles) * T, n = min(T, a.vocab - v0), tid = threadIdx.x;
  const float *in = a.in + (uint64_t)row * a.stride + v0;
  float *out = a.out + (uint64_t)row * a.stride + v0;
  float4u x[kItems];
#pragma unroll
  for (uint32_t k = 0; k < kItems; ++k) {
    const uint32_t v = 4u * (kThreads * k + tid);
    if (v + 4u <= n) x[k] = *(const float4u *)(in + v);
  }
  // where the row's lists and mask begin, asked for together
  uint32_t h0 = 0, h1 = 0, b0 = 0, b1 = 0, m = ~0u;
  if (a.history) h0 = a.history_starts[row], h1 = min(a.history_starts[row + 1], a.history_count);
  if (a.bias_ids) b0 = a.bias_starts[row], b1 = min(a.bias_starts[row + 1], a.bias_count);
  if (a.mask) m = a.mask_of[row];
  const bool touched = a.history || a.bias_ids;
  Ids h;
  h.start(a.history, h0, h1);
  // the thread's first bias; the rest of a long list is read when it is needed
  uint32_t bias_id = ~0u;
  float bias = 0.f;
  if (b0 + tid < b1) bias_id = a.bias_ids[b0 + tid], bias = a.bias_values[b0 + tid];
  const bool masked = m < a.mask_count;
  uint32_t bits[kItems];
  if (masked) {
    const uint32_t *words = a.mask + (uint64_t)m * ((a.vocab + 31u) / 32u);
#pragma unroll
    for (uint32_t k = 0; k < kItems; ++k) {
      const uint32_t v = v0 + 4u * (kThreads * k + tid);   // 4 logits lie in one word: v0 and v are multiples of 4
      bits[k] = words[min(v, a.vocab - 1u) >> 5] >> (v & 31u);
    }
  }
  if (touched) {
#pragma unroll
    for (uint32_t k = 0; k < kItems; ++k) *(u32x4 *)(count + 4u * (kThreads * k + tid)) = u32x4{0u, 0u, 0u, 0u};
    __syncthreads();
  }
  if (a.history)
    h.each([&](uint32_t, uint32_t id) {
      if (id - v0 < n) atomicAdd(&count[id - v0], 1u);
    });
#pragma unroll
  for (uint32_t k = 0; k < kItems; ++k) {
    const uint32_t v = 4u * (kThreads * k + tid);
    if (v + 4u <= n) {
      *(float4u *)(z + v) = x[k];
    } else {
      for (uint32_t i = v; i < n; ++i) z[i] = in[i];
    }
  }
  __syncthreads();
  if (touched) {
    if (a.history) {
      const double *p = a.penalties + 3u * (uint64_t)row;
      const double repeat = p[0], frequency = p[1], presence = p[2];
      // y / repeat as y * (1 / repeat), which is off by less than 4 of its last bits: the
      // same f32 except within 16 of the middle between two, where the quotient itself
      // is taken, as it is below the smallest normal and for repeats out of the ordinary
      const bool plain = repeat > 1e-100 && repeat < 1e100;
      double inverse = __builtin_amdgcn_rcp(repeat);
      inverse = fma(fma(-repeat, inverse, 1.0), inverse, inverse);
      inverse = fma(fma(-repeat, inverse, 1.0), inverse, inverse);
#pragma unroll 1
      for (uint32_t v = tid; v < n; v += kThreads) {
        const uint32_t c = count[v];
        if (c == 0u) continue;
        if (a.bias_ids) count[v] = 0u;
        const float y = z[v];
        const bool up = y > 0.f;
        const double q = (double)y * (up ? inverse : repeat);
        float w = (float)q;
        const uint32_t middle = ((uint32_t)__double_as_longlong(q) & 0x1FFFFFFFu) - 0x0FFFFFF0u;
        if (up && (middle < 32u || !plain || fabs(q) < 0x1p-126)) w = (float)((double)y / repeat);
        w = repeat != 1.0 ? w : y;
        z[v] = (float)((double)w - (frequency * (double)c + presence));
      }
      __syncthreads();
    }
    if (a.bias_ids) {
      // of several pairs of one id the last counts: the largest place in the list
      if (bias_id - v0 < n) atomicMax(&count[bias_id - v0], b0 + tid + 1u);
      for (uint32_t i = b0 + kThreads + tid; i < b1; i += kThreads) {
        const uint32_t at = a.bias_ids[i] - v0;
        if (at < n) atomicMax(&count[at], i + 1u);
      }
      __syncthreads();
      if (bias_id - v0 < n && count[bias_id - v0] == b0 + tid + 1u) z[bias_id - v0] += bias;
      for (uint32_t i = b0 + kThreads + tid; i < b1; i += kThreads) {
        const uint32_t at = a.bias_ids[i] - v0;
        if (at < n && count[at] == i + 1u) z[at] += a.bias_values[i];
      }
      __syncthreads();
    }
  }
#pragma unroll
  for (uint32_t k = 0; k < kItems; ++k) {
    const uint32_t v = 4u * (kThreads * k + tid);
    if (v >= n) break;
    float4u y = *(const float4u *)(z + v);
    if (masked) {
#pragma unroll
      for (uint32_t j = 0; j < 4u; ++j) y[j] = bits[k] >> j & 1u ? y[j] : -INFINITY;
    }
    if (v + 4u <= n) {
      *(float4u *)(out + v) = y;
    } else {
      for (uint32_t i = 0; v + i < n; ++i) out[v + i] = i == 0u ? y[0] : i == 1u ? y[1] : y[2];
    }
  }
}

hipError_t launch_logits(const LogitsArgs &a, hipStream_t stream) {
  // Tiles of 8192 logits: two workgroups fill a CU, and a history is read once for each
  // (48 x 50021, histories of 16000: 11.9 us, tiles of 2048 14.1; a single row of 131072
  // 5.9 and 6.0).
  constexpr uint32_t T = 4u * kThreads * kItems;
  const uint32_t tiles = (a.vocab + T - 1u) / T;
  if (!fits((uint64_t)tiles * a.rows, kThreads)) return hipErrorInvalidConfiguration;
  hipLaunchKernelGGL(k_logits, dim3(tiles * a.rows), dim3(kThreads), 0, stream, a, tiles);
  return hipGetLastError();
}

}  // namespace eff
