// Device helpers of the signal operators: element types, rows of channels, and the
// elementwise functions of the scan and the convolution.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "ns_error.h"
#include "ns_host.h"
#include "neurosim_hip_signal.h"

namespace ns {

constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kLn2 = 0.69314718055994530942f;

// A [T, B, N] operand with unit channel stride.
template <class T>
struct Signal {
  T* data;
  int64_t st, sb;
  __device__ __forceinline__ T* row(int64_t t, int64_t b) const { return data + t * st + b * sb; }
};

template <class T>
inline Signal<T> signal(const ns_signal& s) {
  return Signal<T>{static_cast<T*>(s.data), s.stride_t, s.stride_b};
}

// V channels at any element alignment: one wide load where V * sizeof(T) allows
// (gfx950 reads unaligned addresses).
template <class T, int V>
struct Pack {
  T v[V];
};

template <class T, int V>
__device__ __forceinline__ Pack<T, V> load_pack(const T* p) {
  Pack<T, V> out;
  __builtin_memcpy(&out, p, sizeof(out));
  return out;
}

template <class T, int V>
__device__ __forceinline__ void store_pack(T* p, const Pack<T, V>& x) {
  __builtin_memcpy(p, &x, sizeof(x));
}

// The same in 16-byte words, kStream: past the caches (non-temporal), for what is not read
// again soon.
template <class T, int V, bool kStream = true>
__device__ __forceinline__ void stream_pack(T* p, const Pack<T, V>& x) {
  static_assert(sizeof(x) % 16 == 0, "whole 16-byte words");
  typedef uint32_t word __attribute__((ext_vector_type(4), aligned(2)));
  word w[sizeof(x) / 16];
  __builtin_memcpy(w, &x, sizeof(x));
#pragma unroll
  for (unsigned i = 0; i < sizeof(x) / 16; ++i)
    if constexpr (kStream)
      __builtin_nontemporal_store(w[i], reinterpret_cast<word*>(p) + i);
    else
      reinterpret_cast<word*>(p)[i] = w[i];
}

// 1 / (1 + exp(-x)); exp overflows to infinity for very negative x, whose reciprocal is 0.
__device__ __forceinline__ float sigmoid(float x) {
  return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-kLog2e * x));
}

// log(1 + exp(x)) = max(x, 0) + log1p(e), e = exp(-|x|) in (0, 1].  log1p(e) =
// log(u) e / (u - 1) with u = 1 + e rounded, which keeps its relative accuracy for
// small e (Goldberg 1991, theorem 4); u = 1 gives e itself.  fmaxf drops a NaN, the
// second term keeps it.
__device__ __forceinline__ float softplus(float x) {
  const float e = __builtin_amdgcn_exp2f(-kLog2e * fabsf(x));
  const float u = 1.0f + e;
  const float wide = kLn2 * __builtin_amdgcn_logf(u) * (e * __builtin_amdgcn_rcpf(u - 1.0f));
  return fmaxf(x, 0.0f) + (u == 1.0f ? e : wide);
}

// Column length: [0, ticks].
__device__ __forceinline__ int64_t column_ticks(const int32_t* lengths, int64_t b, int64_t ticks) {
  if (!lengths) return ticks;
  const int64_t own = lengths[b];
  return own < 0 ? 0 : (own < ticks ? own : ticks);
}

// out[m] = sum over p of partials[p*m_total + m], in a fixed order.
int sum_partials(const float* partials, int64_t parts, int64_t m_total, float* out, void* stream);

}  // namespace ns
