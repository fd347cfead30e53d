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

// 2^x, relative error below 2^-22 (the unit's own); 2^-inf = 0, NaN stays NaN.
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
constexpr float LOG2E = 1.4426950408889634f;
constexpr float LN2 = 0.6931471805599453f;

__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v = fmaxf(v, __shfl_xor_sync(~0u, v, o));
  return v;
}
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
  return v;
}

// One 16-byte piece of a row: 4 fp32 or 8 bf16 values.
template <class T>
struct Piece {
  static constexpr int N = 16 / sizeof(T);
  uint32_t w[4];
  __device__ __forceinline__ float get(int i) const {
    if constexpr (sizeof(T) == 4) return __uint_as_float(w[i]);
    else return __uint_as_float(i & 1 ? w[i >> 1] & 0xFFFF0000u : w[i >> 1] << 16);
  }
  // Elements [first, first + N) of a row of V elements at z; elements outside
  // the row read as -inf. z + first is 16-byte aligned.
  __device__ __forceinline__ void load(const T* z, int first, int V) {
    if (first >= 0 && first + N <= V) {
      const uint4 v = *reinterpret_cast<const uint4*>(z + first);
      w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
      return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = sizeof(T) == 4 ? 0xFF800000u : 0xFF80FF80u;  // -inf
    if (first >= V) return;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int e = first + i;
      if (e < 0 || e >= V) continue;
      if constexpr (sizeof(T) == 4) {
        w[i] = __float_as_uint(z[e]);
      } else {
        const uint32_t b = *reinterpret_cast<const unsigned short*>(z + e);
        w[i >> 1] = i & 1 ? (w[i >> 1] & 0xFFFFu) | (b << 16) : (w[i >> 1] & 0xFFFF0000u) | b;
      }
    }
  }
  // Store v[0..N) to elements [first, first + N) of the row d of V elements, as
  // one 16-byte store where `wide` says that d + first is 16-byte aligned.
  static __device__ __forceinline__ void store(T* d, int first, int V, const float* v, bool wide) {
    if (wide && first >= 0 && first + N <= V) {
      uint4 o;
      if constexpr (sizeof(T) == 4) {
        o = make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]),
                       __float_as_uint(v[3]));
      } else {
        __nv_bfloat162 h[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) h[i] = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
        o = *reinterpret_cast<const uint4*>(h);
      }
      *reinterpret_cast<uint4*>(d + first) = o;
      return;
    }
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (first + i >= 0 && first + i < V) from_f(d + first + i, v[i]);
  }
};

// Elements of z that lie before its first 16-byte boundary, counted from the
// boundary below: element e of the row sits at place e + phase(z) of a 16-byte
// grid.
template <class T>
__device__ __forceinline__ int phase(const T* z) {
  return (int)(((uintptr_t)z & 15) / sizeof(T));
}

}  // namespace rnet_logits
