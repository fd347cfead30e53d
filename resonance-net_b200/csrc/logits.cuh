// Reading of logit rows shared by the top-logit records, the distillation loss
// and the beam selection. Rows are fp32 or bf16 with a pitch in elements; all
// arithmetic on them is fp32 or wider.
#pragma once
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <atomic>
#include <cfloat>
#include <cstdint>

#include "common.cuh"

namespace rnet_logits {

// Lets a kernel use `bytes` of dynamic shared memory on the current device, once per
// device: `ready` is the kernel's own record of devices.
inline cudaError_t allow_smem(const void* kernel, int bytes, std::atomic<uint64_t>& ready) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 64 && (ready.load(std::memory_order_relaxed) >> dev & 1)) return cudaSuccess;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess && dev < 64) ready.fetch_or(1ull << dev, std::memory_order_relaxed);
  return e;
}

// Launch of `grid` CTAs in clusters of grid.y.
struct ClusterLaunch {
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute at[1];
  ClusterLaunch(dim3 grid, int threads, size_t smem, cudaStream_t s) {
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.y = grid.y;
    at[0].val.clusterDim.x = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = grid.y > 1;
  }
};

// How many CTAs of a kernel may form a cluster: `wanted` (above 8, which every device
// places) where the current device, or the part of it that the process has, can place
// them, else 8. Asked once per device: `known` holds the answers.
inline cudaError_t cluster_ctas(const void* kernel, int wanted, int threads, size_t smem,
                                std::atomic<int> (&known)[64], int& ctas) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 64 && (ctas = known[dev].load(std::memory_order_relaxed))) return cudaSuccess;
  ctas = 8;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  if (e != cudaSuccess) return e;
  int fit = 0;
  ClusterLaunch one(dim3(1, wanted), threads, smem, nullptr);
  if (cudaOccupancyMaxActiveClusters(&fit, kernel, &one.cfg) != cudaSuccess)
    cudaGetLastError();  // not placed: no error of this call
  else if (fit > 0)
    ctas = wanted;
  if (dev < 64) known[dev].store(ctas, std::memory_order_relaxed);
  return cudaSuccess;
}

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

// The largest value of a warp; NaN loses against any number.
__device__ __forceinline__ float warp_max(float v) {
  float y;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(y) : "f"(v));
  return y;
}
// The same as warp_max for groups of G neighbouring lanes.
template <int G>
__device__ __forceinline__ float group_max(float v) {
  if (G == 32) return warp_max(v);
#pragma unroll
  for (int o = G / 2; o; o >>= 1) v = fmaxf(v, __shfl_xor_sync(~0u, v, o));
  return v;
}
template <int G>
__device__ __forceinline__ float group_sum(float v) {
#pragma unroll
  for (int o = G / 2; o; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
  return v;
}
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
  return v;
}

// log2 of a softmax term: (x - m) c, c = log2(e) / tau, with the product and
// the difference in one rounding: the shift is the rounded m c, the same in
// every term and in the sum, so its rounding cancels. Where that rounding could
// exceed 1, and 2 to its power leave fp32 (logits far from 0, rows whose every logit
// is masked with a large number), the difference is taken first: from |m| = limit
// on, which is 2^24 over the largest c in use.
__device__ __forceinline__ bool far(float m, float limit) { return !(fabsf(m) < limit); }
__device__ __forceinline__ float term(float x, float m, float c, float limit) {
  return far(m, limit) ? (x - m) * c : fmaf(x, c, -__fmul_rn(m, c));
}
// What a sum relative to `from` is multiplied with to be relative to `to`, both
// the largest logits of parts of a row, from <= to. A part without a logit above
// -inf has the lowest number as its largest: its sum is 0 (or NaN) and stays so.
__device__ __forceinline__ float rebase(float from, float to, float c, float limit) {
  const float f = __fmul_rn(from, c), t = __fmul_rn(to, c);
  const float both = (from - to) * c, one = fmaf(from, c, -t), other = -fmaf(to, c, -f);
  const bool ff = far(from, limit), ft = far(to, limit);
  const float d = ff ? (ft ? both : one) : (ft ? other : f - t);
  return exp2_fast(d);
}

// One 16-byte piece of a row: 4 fp32 or 8 bf16 values.
template <class T>
struct Piece {
  static constexpr int N = 16 / sizeof(T);
  uint4 w;
  __device__ __forceinline__ void load(const T* p) { w = *reinterpret_cast<const uint4*>(p); }
  __device__ __forceinline__ void none() {  // -inf everywhere
    const uint32_t v = sizeof(T) == 4 ? 0xFF800000u : 0xFF80FF80u;
    w = make_uint4(v, v, v, v);
  }
  __device__ __forceinline__ float get(int i) const {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
    if constexpr (sizeof(T) == 4) return __uint_as_float(u[i]);
    else return __uint_as_float(i & 1 ? u[i >> 1] & 0xFFFF0000u : u[i >> 1] << 16);
  }
  static __device__ __forceinline__ void store(T* p, const float* v, bool wide) {
    if (wide) {
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
      *reinterpret_cast<uint4*>(p) = o;
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) from_f(p + i, v[i]);
    }
  }
};

// The largest value of a thread's pieces, at least the lowest number (bf16: two
// at a time; NaN is ignored, the sum of exponentials finds it).
template <int NP>
__device__ __forceinline__ float piece_max(const Piece<float>* x) {
  float m = -FLT_MAX;
#pragma unroll
  for (int j = 0; j < NP; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) m = fmaxf(m, x[j].get(i));
  return m;
}
template <int NP>
__device__ __forceinline__ float piece_max(const Piece<__nv_bfloat16>* x) {
  auto h = [](uint32_t u) { return *reinterpret_cast<const __nv_bfloat162*>(&u); };
  __nv_bfloat162 m = h(0xFF80FF80u);
#pragma unroll
  for (int j = 0; j < NP; ++j)
    m = __hmax2(m, __hmax2(__hmax2(h(x[j].w.x), h(x[j].w.y)), __hmax2(h(x[j].w.z), h(x[j].w.w))));
  return fmaxf(fmaxf(__low2float(m), __high2float(m)), -FLT_MAX);
}

// How a row of V elements at z lies on the 16-byte grid: `head` elements before
// the first boundary, `pieces` whole pieces, then the rest. The at most
// 2 (N - 1) elements outside the pieces are edge elements, one a thread.
template <class T>
struct Grid {
  int head, pieces, V;
  __device__ __forceinline__ Grid(const T* z, int v) : V(v) {
    constexpr int N = Piece<T>::N;
    head = min((N - (int)(((uintptr_t)z & 15) / sizeof(T))) & (N - 1), v);
    pieces = (v - head) / N;
  }
  __device__ __forceinline__ int at(int piece) const { return head + piece * Piece<T>::N; }
  // edge element i, or -1
  __device__ __forceinline__ int edge(int i) const {
    const int e = i < head ? i : at(pieces) + i - head;
    return e < V ? e : -1;
  }
};

// Copy of `bytes` (a multiple of 16, both ends 16-byte aligned) to shared
// memory; its arrival counts on the barrier.
__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes,
                                          uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::
          "r"(rnet_dev::smem_u32(dst)),
      "l"(src), "r"(bytes), "r"(rnet_dev::smem_u32(bar))
      : "memory");
}

}  // namespace rnet_logits
