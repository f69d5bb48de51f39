// Eight elements at a time of a bf16, fp16 or float32 row, at any element alignment.
#pragma once

#include "common.h"

namespace flk {

// What one lane loads and keeps of a row: eight elements as they are in memory.
template <typename T>
struct Raw8 {
  T v[8];
};

// A whole chunk is read and written as 16-byte words (two for float32) that assume no more than a 16-bit
// element's alignment: the target's unaligned access mode takes them as they are.
typedef uint32_t word __attribute__((ext_vector_type(4), aligned(2), may_alias));
template <typename T>
constexpr int kWords = sizeof(Raw8<T>) / 16;

// Eight elements at p, of which the first `count` exist (the rest read as zero).  kStream: the access leaves
// the caches to others (nontemporal).
template <bool kStream = false, typename T>
__device__ __forceinline__ Raw8<T> load8(const T* p, int count) {
  Raw8<T> r;
  if (count >= 8) {
    word w[kWords<T>];
#pragma unroll
    for (int i = 0; i < kWords<T>; ++i) {
      const word* at = reinterpret_cast<const word*>(p) + i;
      w[i] = kStream ? __builtin_nontemporal_load(at) : *at;
    }
    __builtin_memcpy(&r, &w, sizeof(r));
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) r.v[i] = i < count ? p[i] : (T)0.0f;
  }
  return r;
}

template <bool kStream = false, typename T>
__device__ __forceinline__ void store8(T* p, int count, const float (&x)[8]) {
  Raw8<T> r;
#pragma unroll
  for (int i = 0; i < 8; ++i) r.v[i] = (T)x[i];
  if (count >= 8) {
    word w[kWords<T>];
    __builtin_memcpy(&w, &r, sizeof(r));
#pragma unroll
    for (int i = 0; i < kWords<T>; ++i) {
      word* at = reinterpret_cast<word*>(p) + i;
      if constexpr (kStream)
        __builtin_nontemporal_store(w[i], at);
      else
        *at = w[i];
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < count) p[i] = r.v[i];
  }
}

// s = 1 / (1 + exp(-g)) and 1 - s, both from exp(-|g|): no overflow, and neither is a difference of
// nearly equal numbers, so each is right to a few units in the last place for every g.
struct Sigmoid {
  float s, rest;
  __device__ __forceinline__ explicit Sigmoid(float g) {
    const float e = __expf(-fabsf(g)), r = __builtin_amdgcn_rcpf(1.0f + e), er = e * r;
    s = g >= 0.0f ? r : er;
    rest = g >= 0.0f ? er : r;
  }
};

// silu(g) u, and its gradients for an incoming d: of g and of u.
__device__ __forceinline__ float gate(float g, float u) { return g * Sigmoid(g).s * u; }
__device__ __forceinline__ void gate_backward(float d, float g, float u, float& dg, float& du) {
  const Sigmoid z(g);
  dg = d * u * (z.s * (1.0f + g * z.rest));
  du = d * (g * z.s);
}

}  // namespace flk
