// Reading of logit rows shared by the top-logit records, the distillation loss
// and the beam selection. Rows are fp32 or bf16 with a pitch in elements; all
// arithmetic on them is fp32 or wider.
#pragma once
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <cfloat>
#include <cstdint>

namespace rnet_logits {

__device__ __forceinline__ float to_f(float x) { return x; }
__device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ void from_f(float* p, float v) { *p = v; }
// one rounding to the logits' own type, on the way out
__device__ __forceinline__ void from_f(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

// Selection sees NaN as -inf (never chosen, no probability), +inf as the
// largest finite number and one zero, so that every row has a total order.
__device__ __forceinline__ float canon(float x) {
  if (x != x) return -INFINITY;
  return fminf(x, FLT_MAX) + 0.0f;
}

// Unsigned order of floats: a < b <=> order(a) < order(b). No NaN.
__device__ __forceinline__ uint32_t order(float x) {
  const uint32_t u = __float_as_uint(x);
  return u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u);
}
__device__ __forceinline__ float unorder(uint32_t o) {
  return __uint_as_float(o ^ ((o & 0x80000000u) ? 0x80000000u : 0xFFFFFFFFu));
}
// Larger key = larger value, then lower index. Keys of one row are distinct.
__device__ __forceinline__ uint64_t make_key(float x, uint32_t idx) {
  return ((uint64_t)order(x) << 32) | (uint32_t)~idx;
}
__device__ __forceinline__ float key_value(uint64_t k) { return unorder((uint32_t)(k >> 32)); }
__device__ __forceinline__ int key_index(uint64_t k) { return (int)~(uint32_t)k; }

}  // namespace rnet_logits
