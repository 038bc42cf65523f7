// Rules on the logits of a batch, before its sampler: for a token v that is
// c > 0 times in the row's history
//   z <- z > 0 ? z / repeat : z * repeat,  z <- z - (frequency * c + presence),
// then z <- z + bias(v), then -inf where the row's mask has no bit for v. The
// first two steps are computed in 64 bits and rounded to 32 after each, as the
// host's sampler does (a Float32Array of logits, 64-bit numbers).
//
// A workgroup takes a tile of a row into LDS, requested before the history so that
// the two round trips overlap; it reads the whole history, counts the ids of its
// tile in LDS (whole numbers: any order gives the same counts), and then changes the
// logits that have one. The tile passes through once: the bytes of the logits bound a
// batch, the round trips a single row, the reading of a long history by every tile the
// rest.
#include "eff_device.h"
#include "eff_kv.h"

namespace eff {

// Rows start wherever the stride puts them: 4-byte aligned.
typedef float float4u __attribute__((ext_vector_type(4), aligned(4)));

// The ids from `a` to `e` of a list, 4 of a thread under way at a time: the first are
// requested by start(). f(i, id); past the end the id is ~0, past every vocabulary.
template <uint32_t THREADS>
struct Ids {
  static constexpr uint32_t U = 4;
  const uint32_t *list;
  uint32_t a, e, id[U];

  __device__ __forceinline__ void load(uint32_t *o, uint32_t i) const {
#pragma unroll
    for (uint32_t k = 0; k < U; ++k) o[k] = i + THREADS * k < e ? list[i + THREADS * k] : ~0u;
  }
  __device__ __forceinline__ void start(const uint32_t *from, uint32_t first, uint32_t end) {
    list = from, a = first, e = end;
    load(id, a + threadIdx.x);
  }
  template <typename F>
  __device__ __forceinline__ void each(F f) {
    uint32_t i = a + threadIdx.x;
    for (uint32_t at = a; at < e; at += THREADS * U, i += THREADS * U) {
      uint32_t next[U];
      load(next, i + THREADS * U);
#pragma unroll
      for (uint32_t k = 0; k < U; ++k) f(i + THREADS * k, id[k]), id[k] = next[k];
    }
  }
};

// ITEMS: groups of 4 logits of a thread.
template <uint32_t THREADS, uint32_t ITEMS>
__global__ __launch_bounds__(THREADS) void k_logits(LogitsArgs a, uint32_t tiles) {
#pragma clang fp contract(off)
  constexpr uint32_t T = 4u * THREADS * ITEMS;
  __shared__ __align__(16) float z[T];
  __shared__ __align__(16) uint32_t count[T];
  const uint32_t row = blockIdx.x / tiles, v0 = (blockIdx.x % tiles) * T, n = min(T, a.vocab - v0), tid = threadIdx.x;
  const float *in = a.in + (uint64_t)row * a.stride + v0;
  float *out = a.out + (uint64_t)row * a.stride + v0;
  float4u x[ITEMS];
#pragma unroll
  for (uint32_t k = 0; k < ITEMS; ++k) {
    const uint32_t v = 4u * (THREADS * k + tid);
    if (v + 4u <= n) x[k] = *(const float4u *)(in + v);
  }
  const uint32_t m = a.mask ? a.mask_of[row] : ~0u;
  const bool masked = m < a.mask_count;
  uint32_t bits[ITEMS];
  if (masked) {
    const uint32_t *words = a.mask + (uint64_t)m * ((a.vocab + 31u) / 32u);
#pragma unroll
    for (uint32_t k = 0; k < ITEMS; ++k) {
      const uint32_t v = v0 + 4u * (THREADS * k + tid);   // 4 logits lie in one word: v0 and v are multiples of 4
      bits[k] = words[min(v, a.vocab - 1u) >> 5] >> (v & 31u);
    }
  }
  const bool touched = a.history || a.bias_ids;
  Ids<THREADS> h;
  if (a.history) h.start(a.history, a.history_starts[row], min(a.history_starts[row + 1], a.history_count));
  if (touched) {
#pragma unroll
    for (uint32_t k = 0; k < ITEMS; ++k) *(u32x4 *)(count + 4u * (THREADS * k + tid)) = u32x4{0u, 0u, 0u, 0u};
    __syncthreads();
  }
  if (a.history)
    h.each([&](uint32_t, uint32_t id) {
      if (id - v0 < n) atomicAdd(&count[id - v0], 1u);
    });
  // the biases take the history's place once it is read
  if (a.bias_ids) h.start(a.bias_ids, a.bias_starts[row], min(a.bias_starts[row + 1], a.bias_count));
#pragma unroll
  for (uint32_t k = 0; k < ITEMS; ++k) {
    const uint32_t v = 4u * (THREADS * k + tid);
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
#pragma unroll 1
      for (uint32_t v = tid; v < n; v += THREADS) {
        const uint32_t c = count[v];
        if (c == 0u) continue;
        if (a.bias_ids) count[v] = 0u;
        float y = z[v];
        if (repeat != 1.0) y = (float)(y > 0.f ? (double)y / repeat : (double)y * repeat);
        z[v] = (float)((double)y - (frequency * (double)c + presence));
      }
      __syncthreads();
    }
    if (a.bias_ids) {
      // of several pairs of one id the last counts: the largest place in the list
      Ids<THREADS> again = h;
      h.each([&](uint32_t i, uint32_t id) {
        if (id - v0 < n) atomicMax(&count[id - v0], i + 1u);
      });
      __syncthreads();
      again.each([&](uint32_t i, uint32_t id) {
        if (id - v0 < n && count[id - v0] == i + 1u) z[id - v0] += a.bias_values[i];
      });
      __syncthreads();
    }
  }
#pragma unroll
  for (uint32_t k = 0; k < ITEMS; ++k) {
    const uint32_t v = 4u * (THREADS * k + tid);
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
  // tiles of 8192 logits where they give every CU a workgroup, else of 2048
  const uint32_t t4 = (a.vocab + 8191u) / 8192u, t1 = (a.vocab + 2047u) / 2048u;
  const bool big = (uint64_t)a.rows * t4 >= 256u;
  if (big) hipLaunchKernelGGL((k_logits<1024, 2>), dim3(t4 * a.rows), dim3(1024), 0, stream, a, t4);
  else hipLaunchKernelGGL((k_logits<512, 1>), dim3(t1 * a.rows), dim3(512), 0, stream, a, t1);
  return hipGetLastError();
}

}  // namespace eff
