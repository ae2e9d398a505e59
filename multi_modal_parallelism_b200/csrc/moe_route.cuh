// Top-k routing of one token by one warp, shared by the routing kernel, the plan and the few-token kernels.
#pragma once
#include "moe.cuh"

namespace mmp {
namespace {

// Floats as unsigned integers of the same order; 0 stands for "not to be chosen" (-inf, NaN, already taken): every
// other float maps above it. +inf is the largest float: in fp32 the two tie; no bf16 is equal to it, there only the value
// is clamped.
constexpr float LARGEST = 3.402823466e38f;
template <bool F32>
__device__ __forceinline__ uint32_t order_key(float v) {
  if (!(v > -INFINITY)) return 0u;
  if (F32) v = fminf(v, LARGEST);
  const uint32_t u = __float_as_uint(v + 0.f);  // + 0: the two zeros are one value
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t k) {
  return fminf(__uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k), LARGEST);
}

template <bool F32>
__device__ __forceinline__ float load_logit(const void* p, int64_t i) {
  if constexpr (F32) return static_cast<const float*>(p)[i];
  else return bf2f(static_cast<const bf16*>(p)[i]);
}

// One token by one warp; lane j ends with place j's expert and weight (j < top_k + shared). V values a lane. A bf16 key has
// 16 bits: with the index below it one maximum finds the largest key and, among equals, the lowest index.
template <int V, bool F32>
__device__ __forceinline__ void route_token(const RouteParams& P, int t, int lane, int& id, float& w) {
  const int64_t row = static_cast<int64_t>(t) * P.l_t;
  uint32_t key[V];
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const int e = lane + 32 * j;
    key[j] = e < P.E ? order_key<F32>(load_logit<F32>(P.logits, row + e)) : 0u;
  }
  float gate = 0.f;
  if (P.shared) gate = load_logit<F32>(P.logits, row + P.E);
  auto largest = [&]() {
    uint32_t m = key[0];
#pragma unroll
    for (int j = 1; j < V; ++j) m = max(m, key[j]);
    return __reduce_max_sync(0xffffffffu, m);
  };
  float z = 0.f;
  const uint32_t top = largest();
  const float vmax = key_value(top);
  if (!P.renorm) {
#pragma unroll
    for (int j = 0; j < V; ++j) z += key[j] ? expf(key_value(key[j]) - vmax) : 0.f;
    z = warp_sum(z);
  }
  id = -1;
  uint32_t mine = 0;
  if constexpr (F32) {
    uint32_t m = top;
    for (int k = 0; k < P.top_k && m; ++k) {  // m == 0: nothing left to choose
      int at = 1 << 30;
#pragma unroll
      for (int j = V - 1; j >= 0; --j) at = key[j] == m ? lane + 32 * j : at;
      at = __reduce_min_sync(0xffffffffu, at);
      if (lane == k) {
        id = at;
        mine = m;
      }
#pragma unroll
      for (int j = 0; j < V; ++j) key[j] = lane + 32 * j == at ? 0u : key[j];
      m = largest();
    }
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) key[j] = key[j] ? (key[j] & 0xffff0000u) | (0xffffu - (lane + 32 * j)) : 0u;
    for (int k = 0; k < P.top_k; ++k) {
      const uint32_t m = largest();
      if (m == 0) break;
      if (lane == k) {
        id = 0xffff - static_cast<int>(m & 0xffffu);
        // the low half of a bf16's key: 0, or all ones below zero
        mine = (m & 0xffff0000u) | ((m & 0x80000000u) ? 0u : 0xffffu);
      }
#pragma unroll
      for (int j = 0; j < V; ++j) key[j] = key[j] == m ? 0u : key[j];
    }
  }
  w = id >= 0 ? expf(key_value(mine) - vmax) : 0.f;
  if (P.renorm) z = warp_sum(w);
  if (id >= 0) w /= z;
  if (P.shared && lane == P.top_k) {
    id = P.E;
    w = 1.f / (1.f + expf(-gate));
  }
}

}  // namespace
}  // namespace mmp
