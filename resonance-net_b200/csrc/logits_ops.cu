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

// ---------------------------------------------------------------- distillation
// L = w [ soft tau^2 sum_k p_k (log p_k - log q_ik) + hard (lse_1 - z_y) ],
// q = softmax(z / tau), and dL/dz = w [ soft tau (P q - p) + hard (softmax(z) -
// 1_y) ] with P = sum p. A row is read once and held in registers: its maximum
// and sum of exponentials, then the gradient of every element without the
// record, then the at most K + 1 elements that a record or label touches once
// more. What bounds it is HBM: one read and one write of the logits.
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

// What a row's gradient needs beside its elements.
struct RowGrad {
  float m;        // largest logit
  float c;        // log2(e) / tau
  float a, a1;    // factors of 2^((x - m) c) and of 2^((x - m) log2(e))
  float pf, hf;   // what a unit of teacher probability and the label take off
  template <bool HARD>
  __device__ __forceinline__ float at(float x) const {
    const float d = x - m;
    float v = a * exp2_fast(d * c);
    if (HARD) v += a1 * exp2_fast(d * LOG2E);
    return v;
  }
};

// The record of one row in shared memory, filled by one warp.
struct Record {
  int idx[RNET_TOPK_MAX];
  float p[RNET_TOPK_MAX];
  float lp[RNET_TOPK_MAX];  // log p
  float z[RNET_TOPK_MAX];
  int target;
  float z_target;
  float P;         // sum p
  int has_target;  // the label is one of the entries
  int twice;       // an index may come more than once
};

// Reads a row's record and label (one warp). Probabilities relative to the
// record's own maximum, or to the teacher's normaliser if it is given.
template <class T>
__device__ __forceinline__ void read_record(Record& r, const T* z, size_t row,
                                            const DistillArgs& a, bool report) {
  constexpr int J = RNET_TOPK_MAX / 32;
  const int lane = threadIdx.x & 31;
  int y = -1;
  if (a.hard != 0.f) y = a.targets[row];
  bool bad = y >= a.V;
  if (bad) y = -1;
  float t[J];
  float tm = -INFINITY;
  bool hot = false, twice = a.K > 32;
#pragma unroll
  for (int j = 0; j < J; ++j) {
    const int k = lane + 32 * j;
    t[j] = -INFINITY;
    if (32 * j >= a.K) break;
    int i = -1;
    if (k < a.K && a.soft != 0.f) i = a.t_idx[row * a.K + k];
    if (i >= a.V) bad = true, i = -1;
    if (i >= 0) {
      t[j] = a.t_val[row * a.K + k] * a.inv_tau;
      r.z[k] = to_f(z[i]);
      hot |= i == y;
    }
    if (k < a.K) r.idx[k] = i;
    tm = fmaxf(tm, t[j]);
    if (j == 0 && !twice)
      twice = __any_sync(~0u, (__match_any_sync(~0u, i < 0 ? ~lane : i) & ~(1u << lane)) != 0);
  }
  const float shift = a.t_lse ? a.t_lse[row] : warp_max(tm);
  float S = 0.f;
  float d[J];
#pragma unroll
  for (int j = 0; j < J; ++j) {
    // an entry at -inf (padding reads as one) has no probability
    d[j] = t[j] - shift;
    t[j] = t[j] == -INFINITY ? 0.f : expf(d[j]);
    S += t[j];
  }
  S = warp_sum(S);
  const bool given = a.t_lse != nullptr;
  const float norm = given || S == 0.f ? 1.0f : 1.0f / S;
  const float ln = given || S == 0.f ? 0.f : logf(S);
#pragma unroll
  for (int j = 0; j < J; ++j)
    if (lane + 32 * j < a.K) {
      r.p[lane + 32 * j] = t[j] * norm;
      r.lp[lane + 32 * j] = d[j] - ln;
    }
  hot = __any_sync(~0u, hot);
  if (lane == 0) {
    r.target = y;
    r.z_target = y >= 0 ? to_f(z[y]) : 0.f;
    r.P = S * norm;
    r.has_target = hot;
    r.twice = twice;
  }
  if (bad && report && a.err) atomicOr(a.err, rnet_dev::ERR_BAD_INDEX);
}

// Gradient factors from the row's maximum m and its sums s (at tau) and s1 (at
// 1) of 2^((x - m) ...).
__device__ __forceinline__ RowGrad row_factors(const Record& r, const DistillArgs& a, float w,
                                               float m, float s, float s1) {
  RowGrad g;
  const bool none = m == -INFINITY && s == 0.f;  // every logit -inf: no distribution
  const bool label = r.target >= 0;
  const float gw = none ? 0.f : w * a.scale;
  g.m = none ? 0.f : m;
  g.c = a.inv_tau * LOG2E;
  g.pf = a.soft != 0.f ? gw * a.soft * a.tau : 0.f;
  g.hf = label ? gw * a.hard : 0.f;
  g.a = none || a.soft == 0.f ? 0.f : g.pf * r.P / s;
  g.a1 = none || !label ? 0.f : g.hf / s1;
  return g;
}

// The row's loss (one warp; the result in every lane).
__device__ __forceinline__ float row_loss(const Record& r, const DistillArgs& a, float w, float m,
                                          float s, float s1) {
  if (m == -INFINITY && s == 0.f) return 0.f;
  float loss = 0.f;
  if (a.soft != 0.f) {
    float kl = 0.f;
    for (int k = threadIdx.x & 31; k < a.K; k += 32)
      if (r.p[k] != 0.f) kl += r.p[k] * (r.lp[k] - (r.z[k] - m) * a.inv_tau);
    kl = warp_sum(kl);
    if (r.P != 0.f) kl += r.P * logf(s);
    loss = a.soft * a.tau * a.tau * kl;
  }
  if (r.target >= 0) loss += a.hard * ((m - r.z_target) + logf(s1));
  return w * loss;
}

// Element i of the record (i == K: the label) once more, with its own terms.
template <class T, bool HARD>
__device__ __forceinline__ void fix_entry(T* d, int i, const Record& r, const RowGrad& g, int K,
                                          int lo, int hi) {
  if (i == K && r.has_target) return;
  const int e = i < K ? r.idx[i] : r.target;
  if (e < lo || e >= hi) return;
  float p = i < K ? r.p[i] : 0.f;
  if (r.twice) {
    p = 0.f;
    for (int k = 0; k < K; ++k)
      if (r.idx[k] == e) p += r.p[k];
  }
  float v = g.at<HARD>(i < K ? r.z[i] : r.z_target) - g.pf * p;
  if (HARD && e == r.target) v -= g.hf;
  from_f(d + e, v);
}

constexpr int WARPS = 8;  // rows of a CTA of the warp-per-row kernel

// Up to 32 * NP pieces of 16 bytes: a warp per row, the row in registers.
template <class T, int NP, bool HARD>
__global__ void __launch_bounds__(32 * WARPS) distill_warp_kernel(
    const T* logits, long long ld, T* dlogits, long long ldd, DistillArgs a, int rows) {
  rnet_dev::pdl_trigger();
  constexpr int N = Piece<T>::N;
  __shared__ Record rec[WARPS];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const size_t row = (size_t)blockIdx.x * WARPS + warp;
  if (row >= rows) return;
  const T* z = logits + row * ld;
  T* d = dlogits ? dlogits + row * ldd : nullptr;
  const int V = a.V, ph = phase(z);
  const bool wide = d && phase(d) == ph;
  const float w = a.weight ? a.weight[row] : 1.0f;
  if (w == 0.f) {  // whatever the row holds
    const float zero[N] = {};
    if (d)
      for (int j = 0; j < NP; ++j) Piece<T>::store(d, (lane + 32 * j) * N - ph, V, zero, wide);
    if (lane == 0) a.row_loss[row] = 0.f;
    return;
  }
  Piece<T> x[NP];
#pragma unroll
  for (int j = 0; j < NP; ++j) x[j].load(z, (lane + 32 * j) * N - ph, V);
  Record& r = rec[warp];
  read_record(r, z, row, a, true);
  float m = -INFINITY;
#pragma unroll
  for (int j = 0; j < NP; ++j)
#pragma unroll
    for (int i = 0; i < N; ++i) m = fmaxf(m, x[j].get(i));
  m = warp_max(m);
  const float ms = m == -INFINITY ? 0.f : m, c = a.inv_tau * LOG2E;
  float s = 0.f, s1 = 0.f;
#pragma unroll
  for (int j = 0; j < NP; ++j)
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float e = x[j].get(i) - ms;
      s += exp2_fast(e * c);
      if (HARD) s1 += exp2_fast(e * LOG2E);
    }
  s = warp_sum(s);
  if (HARD) s1 = warp_sum(s1);
  __syncwarp();
  const float loss = row_loss(r, a, w, m, s, s1);
  if (lane == 0) a.row_loss[row] = loss;
  if (!d) return;
  const RowGrad g = row_factors(r, a, w, m, s, s1);
#pragma unroll
  for (int j = 0; j < NP; ++j) {
    float v[N];
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = g.at<HARD>(x[j].get(i));
    Piece<T>::store(d, (lane + 32 * j) * N - ph, V, v, wide);
  }
  __syncwarp();  // orders the stores above before those below
  for (int i = lane; i <= a.K; i += 32) fix_entry<T, HARD>(d, i, r, g, a.K, 0, V);
}

__device__ __forceinline__ void store_remote(float* p, uint32_t rank, float v) {
  asm volatile(
      "{\n\t.reg .b32 ra;\n\t"
      "mapa.shared::cluster.u32 ra, %0, %1;\n\t"
      "st.shared::cluster.f32 [ra], %2;\n\t}" ::"r"(rnet_dev::smem_u32(p)),
      "r"(rank), "f"(v)
      : "memory");
}

// Longer rows: a cluster of C = 1, 2, 4 or 8 CTAs per row, each with up to
// THREADS * NP pieces in registers. The CTAs' maxima and sums meet through
// distributed shared memory and are joined in rank order, so every CTA uses the
// same bits.
template <class T, int THREADS, int NP, bool HARD>
__global__ void __launch_bounds__(THREADS) distill_cta_kernel(const T* logits, long long ld,
                                                              T* dlogits, long long ldd,
                                                              DistillArgs a, int C) {
  rnet_dev::pdl_trigger();
  constexpr int N = Piece<T>::N, NW = THREADS / 32;
  __shared__ Record r;
  __shared__ float part[NW][3];
  __shared__ float joint[8][3];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const size_t row = blockIdx.x / C;
  const int rank = blockIdx.x % C;
  const T* z = logits + row * ld;
  T* d = dlogits ? dlogits + row * ldd : nullptr;
  const int V = a.V, ph = phase(z);
  const bool wide = d && phase(d) == ph;
  const int pieces = (V + ph + N - 1) / N, per = (pieces + C - 1) / C;
  const int begin = rank * per, end = min(begin + per, pieces);
  auto first = [&](int j) {  // V: no element
    const int q = begin + tid + j * THREADS;
    return q < end ? q * N - ph : V;
  };
  const float w = a.weight ? a.weight[row] : 1.0f;
  if (w == 0.f) {  // whatever the row holds; the whole cluster leaves
    const float zero[N] = {};
    if (d)
      for (int j = 0; j < NP; ++j) Piece<T>::store(d, first(j), V, zero, wide);
    if (rank == 0 && tid == 0) a.row_loss[row] = 0.f;
    return;
  }
  // the peers' shared memory may be written once all of them run
  if (C > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
  Piece<T> x[NP];
#pragma unroll
  for (int j = 0; j < NP; ++j) x[j].load(z, first(j), V);
  if (warp == 0) read_record(r, z, row, a, rank == 0);
  const float c = a.inv_tau * LOG2E;
  float m = -INFINITY;
#pragma unroll
  for (int j = 0; j < NP; ++j)
#pragma unroll
    for (int i = 0; i < N; ++i) m = fmaxf(m, x[j].get(i));
  const float m0 = m == -INFINITY ? 0.f : m;
  float s = 0.f, s1 = 0.f;
#pragma unroll
  for (int j = 0; j < NP; ++j)
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float e = x[j].get(i) - m0;
      s += exp2_fast(e * c);
      if (HARD) s1 += exp2_fast(e * LOG2E);
    }
  // relative to the warp's maximum, the CTA's, the row's (a part without a
  // logit above -inf has sums of 0, or of NaN, and keeps them)
  auto rebase = [&](float to, float from, float& v, float& v1) {
    const float e = from == -INFINITY ? 0.f : from - to;
    v *= exp2_fast(e * c);
    if (HARD) v1 *= exp2_fast(e * LOG2E);
  };
  const float mw = warp_max(m);
  rebase(mw, m, s, s1);
  s = warp_sum(s);
  if (HARD) s1 = warp_sum(s1);
  if (lane == 0) part[warp][0] = mw, part[warp][1] = s, part[warp][2] = s1;
  __syncthreads();
  m = -INFINITY;
  for (int i = 0; i < NW; ++i) m = fmaxf(m, part[i][0]);
  s = s1 = 0.f;
  for (int i = 0; i < NW; ++i) {
    float v = part[i][1], v1 = part[i][2];
    rebase(m, part[i][0], v, v1);
    s += v, s1 += v1;
  }
  if (C > 1) {
    asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
    if (tid < C) {
      store_remote(&joint[rank][0], tid, m);
      store_remote(&joint[rank][1], tid, s);
      store_remote(&joint[rank][2], tid, s1);
    }
    rnet_dev::cluster_sync();
    m = -INFINITY;
    for (int i = 0; i < C; ++i) m = fmaxf(m, joint[i][0]);
    s = s1 = 0.f;
    for (int i = 0; i < C; ++i) {
      float v = joint[i][1], v1 = joint[i][2];
      rebase(m, joint[i][0], v, v1);
      s += v, s1 += v1;
    }
  }
  if (rank == 0 && warp == 0) {
    const float loss = row_loss(r, a, w, m, s, s1);
    if (lane == 0) a.row_loss[row] = loss;
  }
  if (!d) return;
  const RowGrad g = row_factors(r, a, w, m, s, s1);
#pragma unroll
  for (int j = 0; j < NP; ++j) {
    float v[N];
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = g.at<HARD>(x[j].get(i));
    Piece<T>::store(d, first(j), V, v, wide);
  }
  __syncthreads();  // orders the stores above before those below
  const int lo = max(begin * N - ph, 0), hi = min(end * N - ph, V);
  for (int i = tid; i <= a.K; i += THREADS) fix_entry<T, HARD>(d, i, r, g, a.K, lo, hi);
}

template <class T, int THREADS, int NP, bool HARD>
cudaError_t distill_cta(const T* z, long long ld, T* d, long long ldd, const DistillArgs& a,
                        int rows, int C, cudaStream_t s) {
  if ((long long)rows * C > 0x7fffffffLL) return cudaErrorInvalidValue;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(rows * C);
  cfg.blockDim = dim3(THREADS);
  cfg.stream = s;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = C;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = C > 1;
  return cudaLaunchKernelEx(&cfg, distill_cta_kernel<T, THREADS, NP, HARD>, z, ld, d, ldd, a, C);
}

template <class T, bool HARD>
cudaError_t distill_launch(const T* z, long long ld, T* d, long long ldd, const DistillArgs& a,
                           int rows, cudaStream_t s) {
  constexpr int N = Piece<T>::N;
  // places before a row's first element, at most
  const int ph = ((size_t)z | (size_t)ld * sizeof(T)) % 16 ? N - 1 : 0;
  const int pieces = (a.V + ph + N - 1) / N;
  const int grid = (rows + WARPS - 1) / WARPS, block = 32 * WARPS;
  if (pieces <= 32)
    distill_warp_kernel<T, 1, HARD><<<grid, block, 0, s>>>(z, ld, d, ldd, a, rows);
  else if (pieces <= 64)
    distill_warp_kernel<T, 2, HARD><<<grid, block, 0, s>>>(z, ld, d, ldd, a, rows);
  else if (pieces <= 128)
    distill_warp_kernel<T, 4, HARD><<<grid, block, 0, s>>>(z, ld, d, ldd, a, rows);
  else {
    // the fewest CTAs of 256 threads that hold the row, 8 pieces a thread;
    // more of them while they leave SMs idle
    int C = 1;
    while (C < 8 && 256 * 8 * C < pieces) C *= 2;
    while (C < 8 && rows * C < 148 && 256 * C < pieces) C *= 2;
    const int per = (pieces + C - 1) / C;
    if (per <= 256) return distill_cta<T, 256, 1, HARD>(z, ld, d, ldd, a, rows, C, s);
    if (per <= 512) return distill_cta<T, 256, 2, HARD>(z, ld, d, ldd, a, rows, C, s);
    if (per <= 1024) return distill_cta<T, 256, 4, HARD>(z, ld, d, ldd, a, rows, C, s);
    if (per <= 2048) return distill_cta<T, 256, 8, HARD>(z, ld, d, ldd, a, rows, C, s);
    if (per <= 4096) return distill_cta<T, 512, 8, HARD>(z, ld, d, ldd, a, rows, C, s);
    // the limit of the vocabulary, in an unaligned row
    constexpr int LAST = RNET_DISTILL_VOCAB_MAX / 8 / 1024 / N + 1;
    if (per <= 1024 * LAST) return distill_cta<T, 1024, LAST, HARD>(z, ld, d, ldd, a, rows, C, s);
    return cudaErrorInvalidValue;
  }
  return cudaGetLastError();
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
  if (rows > 0) {
    cudaError_t e;
    if (bf16) {
      const __nv_bfloat16* z = (const __nv_bfloat16*)logits;
      __nv_bfloat16* d = (__nv_bfloat16*)dlogits;
      e = hard != 0.f ? distill_launch<__nv_bfloat16, true>(z, ld, d, ldd, a, rows, s)
                      : distill_launch<__nv_bfloat16, false>(z, ld, d, ldd, a, rows, s);
    } else {
      const float* z = (const float*)logits;
      float* d = (float*)dlogits;
      e = hard != 0.f ? distill_launch<float, true>(z, ld, d, ldd, a, rows, s)
                      : distill_launch<float, false>(z, ld, d, ldd, a, rows, s);
    }
    if (e != cudaSuccess) return e;
    launched();
  }
  if (!loss) return cudaSuccess;
  sum_rows_kernel<<<1, 1024, 0, s>>>(row_loss, rows, loss);
  return launched();
}

}  // namespace rnet_k
