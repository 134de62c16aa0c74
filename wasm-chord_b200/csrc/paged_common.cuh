// Device helpers shared by the paged operators: element types and their
// 16-byte vectors, the batch's checked rows, page lookup.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cfloat>
#include <cmath>
#include <cstdint>

#include "paged.h"

namespace wcb {
namespace paged {
namespace {

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
// round to nearest: at most half a step of the type
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// N consecutive elements (a multiple of 16 bytes) at a 16-byte aligned address
template <typename T, int N>
__device__ __forceinline__ void load_vec(const T* p, float (&x)[N]) {
  constexpr int V = 16 / sizeof(T);
  static_assert(N % V == 0, "whole 16-byte words");
#pragma unroll
  for (int i = 0; i < N / V; ++i) {
    const uint4 w = *reinterpret_cast<const uint4*>(p + V * i);
    T e[V];
    *reinterpret_cast<uint4*>(e) = w;
#pragma unroll
    for (int j = 0; j < V; ++j) x[V * i + j] = to_f32(e[j]);
  }
}
template <typename T, int N>
__device__ __forceinline__ void store_vec(T* p, const float (&x)[N]) {
  constexpr int V = 16 / sizeof(T);
  static_assert(N % V == 0, "whole 16-byte words");
#pragma unroll
  for (int i = 0; i < N / V; ++i) {
    alignas(16) T e[V];
#pragma unroll
    for (int j = 0; j < V; ++j) e[j] = from_f32<T>(x[V * i + j]);
    *reinterpret_cast<uint4*>(p + V * i) = *reinterpret_cast<const uint4*>(e);
  }
}

// The new tokens of sequence s: rows r0 .. r0 + n - 1 (n = 0 where q_start is
// not sound), and the tokens in its cache.
struct Seq {
  int r0, n, kv;
  bool sound;
};
__device__ __forceinline__ Seq read_seq(const Batch& b, int s) {
  Seq q;
  const int lo = __ldg(b.q_start + s), hi = __ldg(b.q_start + s + 1);
  q.kv = max(0, __ldg(b.kv_len + s));
  q.r0 = lo;
  q.sound = lo >= 0 && hi >= lo && hi <= b.n_tokens;
  q.n = q.sound ? hi - lo : 0;
  return q;
}
// tokens that the page table's row can name (and 32 bits count, with room for the tile after the last)
__device__ __forceinline__ int table_tokens(const Pool& p, const Batch& b) {
  const long long n = static_cast<long long>(b.max_pages) * p.page_size;
  return n > 0x7ffff000 ? 0x7ffff000 : int(n);
}
__device__ __forceinline__ void report(const Batch& b, uint32_t bits) {
  if (b.status && bits) atomicOr(b.status, bits);
}

}  // namespace
}  // namespace paged
}  // namespace wcb
