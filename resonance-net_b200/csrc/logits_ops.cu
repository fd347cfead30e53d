// Records of a row's largest logits, and the distillation loss against such
// records with its gradient.
#include "common.cuh"
#include "kernels.cuh"
#include "logits.cuh"

namespace rnet_k {
namespace {

using namespace rnet_logits;

constexpr int LT = 256;  // threads per row

__device__ __forceinline__ float block_max(float v, float* sh) {
  for (int o = 16; o; o >>= 1) v = fmaxf(v, __shfl_xor_sync(~0u, v, o));
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
  __syncthreads();
  v = sh[0];
  for (int i = 1; i < LT / 32; ++i) v = fmaxf(v, sh[i]);
  __syncthreads();
  return v;
}
__device__ __forceinline__ float block_sum(float v, float* sh) {
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0.f;
  for (int i = 0; i < LT / 32; ++i) v += sh[i];
  __syncthreads();
  return v;
}

// One CTA per row; K rounds, each finds the largest key below the last one.
template <class T>
__global__ void __launch_bounds__(LT) topk_kernel(const T* __restrict__ logits, long long ld,
                                                  float inv_tau, float* __restrict__ top,
                                                  int* __restrict__ idx, float* __restrict__ lse,
                                                  int V, int K) {
  rnet_dev::pdl_trigger();
  __shared__ float sh[LT / 32];
  __shared__ uint64_t shk[LT / 32];
  const T* z = logits + (size_t)blockIdx.x * ld;
  float m = -INFINITY;
  for (int i = threadIdx.x; i < V; i += LT) m = fmaxf(m, canon(to_f(z[i])));
  m = block_max(m, sh);
  if (lse) {
    float s = 0.f;
    if (m > -INFINITY)
      for (int i = threadIdx.x; i < V; i += LT) s += expf((canon(to_f(z[i])) - m) * inv_tau);
    s = block_sum(s, sh);
    if (threadIdx.x == 0) lse[blockIdx.x] = m > -INFINITY ? m * inv_tau + logf(s) : -INFINITY;
  }
  uint64_t below = ~0ull;
  for (int k = 0; k < K; ++k) {
    uint64_t best = 0;
    for (int i = threadIdx.x; i < V; i += LT) {
      const float x = canon(to_f(z[i]));
      const uint64_t key = make_key(x, i);
      if (x > -INFINITY && key < below && key > best) best = key;
    }
    for (int o = 16; o; o >>= 1) {
      const uint64_t b = __shfl_xor_sync(~0u, best, o);
      best = b > best ? b : best;
    }
    if ((threadIdx.x & 31) == 0) shk[threadIdx.x >> 5] = best;
    __syncthreads();
    for (int i = 0; i < LT / 32; ++i) best = shk[i] > best ? shk[i] : best;
    __syncthreads();
    if (threadIdx.x == 0) {
      top[(size_t)blockIdx.x * K + k] = best ? key_value(best) : -INFINITY;
      idx[(size_t)blockIdx.x * K + k] = best ? key_index(best) : -1;
    }
    below = best;
  }
}

struct DistillArgs {
  const int* t_idx;
  const float* t_val;
  const float* t_lse;
  const int* targets;
  const float* weight;
  float inv_tau, tau, soft, hard, scale;
  float* row_loss;
  unsigned* err;
  int V, K;
};

// One CTA per row, three passes over it.
template <class T>
__global__ void __launch_bounds__(LT) distill_kernel(const T* logits, long long ld, T* dlogits,
                                                     long long ldd, DistillArgs a) {
  rnet_dev::pdl_trigger();
  __shared__ float sh[LT / 32];
  __shared__ int s_idx[RNET_TOPK_MAX];
  __shared__ float s_p[RNET_TOPK_MAX];
  const size_t row = blockIdx.x;
  const T* z = logits + row * ld;
  T* d = dlogits ? dlogits + row * ldd : nullptr;
  const float w = a.weight ? a.weight[row] : 1.0f;
  const int V = a.V;
  float m = -INFINITY;
  for (int i = threadIdx.x; i < V; i += LT) m = fmaxf(m, to_f(z[i]));
  m = block_max(m, sh);
  if (w == 0.0f || m == -INFINITY) {
    // no weight, or no distribution (every logit -inf): no loss, no gradient
    bool nan = false;
    if (w != 0.0f)
      for (int i = threadIdx.x; i < V; i += LT) nan |= to_f(z[i]) != to_f(z[i]);
    nan = __syncthreads_or(nan);
    const float v = nan ? NAN : 0.0f;
    if (d)
      for (int i = threadIdx.x; i < V; i += LT) from_f(d + i, v);
    if (threadIdx.x == 0) a.row_loss[row] = v;
    return;
  }
  float s = 0.f, s1 = 0.f;
  for (int i = threadIdx.x; i < V; i += LT) {
    const float x = to_f(z[i]) - m;
    s += expf(x * a.inv_tau);
    if (a.hard != 0.f) s1 += expf(x);
  }
  s = block_sum(s, sh);
  s1 = block_sum(s1, sh);
  int target = -1;
  float z_target = 0.f;
  if (a.targets && a.hard != 0.f) {
    target = a.targets[row];
    if (target >= V) {
      if (a.err && threadIdx.x == 0) atomicOr(a.err, rnet_dev::ERR_BAD_INDEX);
      target = -1;
    }
    if (target >= 0) z_target = to_f(z[target]);
  }
  // teacher: thread k holds entry k
  float t = -INFINITY, zk = 0.f;
  int ti = -1;
  if (threadIdx.x < a.K) {
    ti = a.t_idx[row * a.K + threadIdx.x];
    if (ti >= V) {
      if (a.err) atomicOr(a.err, rnet_dev::ERR_BAD_INDEX);
      ti = -1;
    }
    if (ti >= 0) {
      t = a.t_val[row * a.K + threadIdx.x] * a.inv_tau;
      zk = to_f(z[ti]);
    }
  }
  const float tm = block_max(t, sh);
  float lt;
  if (a.t_lse) {
    lt = a.t_lse[row];
  } else {
    const float e = ti >= 0 && t > -INFINITY ? expf(t - tm) : (t != t ? t : 0.f);
    lt = tm + logf(block_sum(e, sh));
  }
  const float p = ti >= 0 && !(t == -INFINITY) ? expf(t - lt) : 0.f;
  const float P = block_sum(p, sh);
  const float ls = logf(s);
  const float kl = block_sum(p != 0.f ? p * ((t - lt) - ((zk - m) * a.inv_tau - ls)) : 0.f, sh);
  if (threadIdx.x == 0) {
    float loss = a.soft != 0.f ? a.soft * a.tau * a.tau * kl : 0.f;
    if (target >= 0) loss += a.hard * (m - z_target + logf(s1));
    a.row_loss[row] = w * loss;
  }
  if (!d) return;
  if (threadIdx.x < a.K) {
    s_idx[threadIdx.x] = ti;
    s_p[threadIdx.x] = p;
  }
  const float g = w * a.scale;
  const float cs = a.soft * a.tau, ch = target >= 0 ? a.hard : 0.f;
  const float is = 1.0f / s, is1 = target >= 0 ? 1.0f / s1 : 0.f;
  auto grad = [&](float x, float pk, bool hot) {
    float v = cs * (P * (expf((x - m) * a.inv_tau) * is) - pk);
    if (ch != 0.f) v += ch * (expf(x - m) * is1 - (hot ? 1.0f : 0.0f));
    return g * v;
  };
  __syncthreads();
  for (int i = threadIdx.x; i < V; i += LT) {
    float pk = 0.f;
    for (int k = 0; k < a.K; ++k)
      if (s_idx[k] == i) pk += s_p[k];
    from_f(d + i, grad(to_f(z[i]), pk, i == target));
  }
}

__global__ void __launch_bounds__(1024) sum_rows_kernel(const float* __restrict__ x, int n,
                                                        float* __restrict__ out) {
  rnet_dev::pdl_trigger();
  __shared__ double sh[1024];
  double a = 0.0;
  for (int i = threadIdx.x; i < n; i += 1024) a += x[i];
  sh[threadIdx.x] = a;
  __syncthreads();
  for (int o = 512; o > 0; o >>= 1) {
    if (threadIdx.x < o) sh[threadIdx.x] += sh[threadIdx.x + o];
    __syncthreads();
  }
  if (threadIdx.x == 0) *out = (float)sh[0];
}

}  // namespace

cudaError_t topk_logits(const void* logits, bool bf16, long long ld, float tau, float* top,
                        int* idx, float* lse, int rows, int V, int K, cudaStream_t s) {
  if (rows <= 0) return cudaSuccess;
  if (bf16)
    topk_kernel<<<rows, LT, 0, s>>>((const __nv_bfloat16*)logits, ld, 1.0f / tau, top, idx, lse, V,
                                    K);
  else
    topk_kernel<<<rows, LT, 0, s>>>((const float*)logits, ld, 1.0f / tau, top, idx, lse, V, K);
  return launched();
}

cudaError_t distill_topk(const void* logits, bool bf16, long long ld, const int* t_idx,
                         const float* t_val, const float* t_lse, const int* targets,
                         const float* weight, float tau, float soft, float hard, float scale,
                         float* row_loss, float* loss, void* dlogits, long long ldd, int rows,
                         int V, int K, unsigned* err, cudaStream_t s) {
  DistillArgs a{t_idx, t_val, t_lse, targets, weight, 1.0f / tau, tau, soft, hard, scale, row_loss,
                err, V, K};
  unsigned n = 0;
  if (rows > 0) {
    if (bf16)
      distill_kernel<<<rows, LT, 0, s>>>((const __nv_bfloat16*)logits, ld, (__nv_bfloat16*)dlogits,
                                         ldd, a);
    else
      distill_kernel<<<rows, LT, 0, s>>>((const float*)logits, ld, (float*)dlogits, ldd, a);
    cudaError_t e = launched();
    if (e != cudaSuccess) return e;
  }
  if (loss) {
    sum_rows_kernel<<<1, 1024, 0, s>>>(row_loss, rows, loss);
    ++n;
  }
  return launched(n);
}

}  // namespace rnet_k
