// Beam search: selection over beams and vocabulary, reordering of the streams'
// states by the chosen parents, and the sequences behind the last beams.
#include "common.cuh"
#include "kernels.cuh"
#include "logits.cuh"

namespace rnet_k {
namespace {

using namespace rnet_logits;

constexpr int BT = 256;

struct Cand {
  double total;
  unsigned long long flat;  // beam * vocab + token
};
__device__ __forceinline__ bool better(const Cand& a, const Cand& b) {
  return a.total > b.total || (a.total == b.total && a.flat < b.flat);
}

// One CTA per sequence: the log-normaliser of each beam's row, then `beams`
// rounds, each finding the best candidate after the last one.
template <class T>
__global__ void __launch_bounds__(BT) beam_select_kernel(
    const T* __restrict__ logits, long long ld, const float* scores_in, const int* finished_in,
    int eos, float* scores, int* tokens, int* parents, int* finished, int W, int V) {
  rnet_dev::pdl_trigger();
  __shared__ double s_lse[RNET_BEAMS_MAX], s_score[RNET_BEAMS_MAX];
  __shared__ int s_done[RNET_BEAMS_MAX];
  __shared__ double shd[BT / 32];
  __shared__ float shf[BT / 32];
  __shared__ Cand shc[BT / 32];
  const size_t m0 = (size_t)blockIdx.x * W;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (threadIdx.x < W) {
    s_score[threadIdx.x] = canon(scores_in[m0 + threadIdx.x]);
    s_done[threadIdx.x] = finished_in ? finished_in[m0 + threadIdx.x] != 0 : 0;
  }
  for (int b = 0; b < W; ++b) {
    const T* z = logits + (m0 + b) * ld;
    float m = -INFINITY;
    for (int i = threadIdx.x; i < V; i += BT) m = fmaxf(m, canon(to_f(z[i])));
    for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, o));
    if (lane == 0) shf[warp] = m;
    __syncthreads();
    for (int i = 0; i < BT / 32; ++i) m = fmaxf(m, shf[i]);
    double s = 0.0;
    if (m > -INFINITY)
      for (int i = threadIdx.x; i < V; i += BT) s += expf(canon(to_f(z[i])) - m);
    for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(~0u, s, o);
    if (lane == 0) shd[warp] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
      s = 0.0;
      for (int i = 0; i < BT / 32; ++i) s += shd[i];
      s_lse[b] = m + log(s);
    }
    __syncthreads();
  }
  Cand last{INFINITY, 0};
  for (int j = 0; j < W; ++j) {
    Cand best{-INFINITY, ~0ull};
    for (int b = 0; b < W; ++b) {
      const T* z = logits + (m0 + b) * ld;
      const unsigned long long f0 = (unsigned long long)b * V;
      if (s_done[b]) {
        const Cand c{s_score[b], f0 + eos};
        if (threadIdx.x == 0 && better(last, c) && better(c, best)) best = c;
        continue;
      }
      for (int i = threadIdx.x; i < V; i += BT) {
        const float x = canon(to_f(z[i]));
        if (x == -INFINITY) continue;
        const Cand c{s_score[b] + ((double)x - s_lse[b]), f0 + i};
        if (better(last, c) && better(c, best)) best = c;
      }
    }
    for (int o = 16; o; o >>= 1) {
      const Cand c{__shfl_xor_sync(~0u, best.total, o), __shfl_xor_sync(~0u, best.flat, o)};
      if (better(c, best)) best = c;
    }
    if (lane == 0) shc[warp] = best;
    __syncthreads();
    for (int i = 0; i < BT / 32; ++i)
      if (better(shc[i], best)) best = shc[i];
    __syncthreads();
    last = best;
    if (threadIdx.x == 0) {
      const bool live = best.total > -INFINITY;
      const int parent = live ? (int)(best.flat / V) : j;
      const int token = live ? (int)(best.flat % V) : (eos >= 0 ? eos : 0);
      scores[m0 + j] = live ? (float)best.total : -INFINITY;
      parents[m0 + j] = parent;
      tokens[m0 + j] = token;
      if (finished) finished[m0 + j] = s_done[parent] || token == eos;
    }
  }
}

// Rows [outer][batch][beams] of `row` vectors: dst row j of a group is src row
// parents[j]. A thread owns one vector column of a group: it reads the parents'
// values of every beam before it writes any, so dst may be src.
template <class Vec, int W>
__global__ void __launch_bounds__(256) beam_reorder_kernel(
    const char* src, char* dst, size_t row, size_t pitch, size_t outer_pitch,
    const int* __restrict__ parents, int beams, unsigned* err) {
  rnet_dev::pdl_trigger();
  __shared__ int s_par[W];
  const size_t g = blockIdx.y;
  if (threadIdx.x < beams) {
    int p = parents[g * beams + threadIdx.x];
    if (p < 0 || p >= beams) {
      if (err && blockIdx.x == 0 && blockIdx.z == 0) atomicOr(err, rnet_dev::ERR_BAD_INDEX);
      p = threadIdx.x;
    }
    s_par[threadIdx.x] = p;
  }
  __syncthreads();
  const size_t c = blockIdx.x * (size_t)blockDim.x + threadIdx.x;
  if (c >= row) return;
  const size_t base = blockIdx.z * outer_pitch + g * beams * pitch + c * sizeof(Vec);
  const bool in_place = src == dst;
  Vec v[W];
#pragma unroll
  for (int j = 0; j < W; ++j)
    if (j < beams && !(in_place && s_par[j] == j))
      v[j] = *reinterpret_cast<const Vec*>(src + base + s_par[j] * pitch);
#pragma unroll
  for (int j = 0; j < W; ++j)
    if (j < beams && !(in_place && s_par[j] == j))
      *reinterpret_cast<Vec*>(dst + base + j * pitch) = v[j];
}

// One CTA per sequence; thread j walks the parents of last beam j backwards.
__global__ void __launch_bounds__(32) beam_backtrack_kernel(
    const int* __restrict__ tokens, const int* __restrict__ parents,
    const float* __restrict__ scores, int eos, float alpha, int* __restrict__ seq,
    int* __restrict__ lengths, float* __restrict__ ranked, int T, int M, int W, unsigned* err) {
  rnet_dev::pdl_trigger();
  const int j = threadIdx.x;
  const size_t m0 = (size_t)blockIdx.x * W;
  int len = T;
  bool bad = false;
  if (j < W) {
    int a = j;
    for (int t = T - 1; t >= 0; --t) {
      const size_t at = (size_t)t * M + m0 + a;
      if (eos >= 0 && tokens[at] == eos) len = t + 1;
      const int p = parents[at];
      bad |= p < 0 || p >= W;
      a = p < 0 || p >= W ? a : p;
    }
  }
  if (bad && err) atomicOr(err, rnet_dev::ERR_BAD_INDEX);
  double r = -INFINITY;
  if (j < W) r = (double)canon(scores[m0 + j]) / pow((double)(len > 0 ? len : 1), (double)alpha);
  int rank = 0;
  for (int i = 0; i < W; ++i) {
    const double o = __shfl_sync(~0u, r, i);
    rank += o > r || (o == r && i < j);
  }
  if (j >= W) return;
  lengths[m0 + rank] = len;
  ranked[m0 + rank] = (float)r;
  int a = j;
  for (int t = T - 1; t >= 0; --t) {
    const size_t at = (size_t)t * M + m0 + a;
    seq[(m0 + rank) * T + t] = t >= len ? eos : tokens[at];
    const int p = parents[at];
    a = p < 0 || p >= W ? a : p;
  }
}

template <class Vec>
cudaError_t reorder_as(const char* src, char* dst, size_t row_bytes, size_t pitch, size_t outer,
                       size_t outer_pitch, const int* parents, int batch, int beams, unsigned* err,
                       cudaStream_t s) {
  const size_t row = row_bytes / sizeof(Vec);
  const dim3 grid((unsigned)((row + 255) / 256), batch, (unsigned)outer);
  if (beams <= 8)
    beam_reorder_kernel<Vec, 8><<<grid, 256, 0, s>>>(src, dst, row, pitch, outer_pitch, parents,
                                                     beams, err);
  else
    beam_reorder_kernel<Vec, 32><<<grid, 256, 0, s>>>(src, dst, row, pitch, outer_pitch, parents,
                                                      beams, err);
  return launched();
}

}  // namespace

cudaError_t beam_select(const void* logits, bool bf16, long long ld, const float* scores_in,
                        const int* finished_in, int eos, float* scores, int* tokens, int* parents,
                        int* finished, int batch, int beams, int V, cudaStream_t s) {
  if (batch <= 0) return cudaSuccess;
  if (bf16)
    beam_select_kernel<<<batch, BT, 0, s>>>((const __nv_bfloat16*)logits, ld, scores_in,
                                            finished_in, eos, scores, tokens, parents, finished,
                                            beams, V);
  else
    beam_select_kernel<<<batch, BT, 0, s>>>((const float*)logits, ld, scores_in, finished_in, eos,
                                            scores, tokens, parents, finished, beams, V);
  return launched();
}

cudaError_t beam_reorder(const void* src, void* dst, size_t row_bytes, size_t pitch, size_t outer,
                         size_t outer_pitch, const int* parents, int batch, int beams,
                         unsigned* err, cudaStream_t s) {
  if (!row_bytes || !outer || batch <= 0) return cudaSuccess;
  const char* a = (const char*)src;
  char* b = (char*)dst;
  const size_t bits = (size_t)a | (size_t)b | row_bytes | pitch | outer_pitch;
  if (bits % 16 == 0)
    return reorder_as<uint4>(a, b, row_bytes, pitch, outer, outer_pitch, parents, batch, beams,
                             err, s);
  return reorder_as<uint32_t>(a, b, row_bytes, pitch, outer, outer_pitch, parents, batch, beams,
                              err, s);
}

cudaError_t beam_backtrack(const int* tokens, const int* parents, const float* scores, int eos,
                           float alpha, int* sequences, int* lengths, float* ranked, int steps,
                           int batch, int beams, unsigned* err, cudaStream_t s) {
  if (batch <= 0) return cudaSuccess;
  beam_backtrack_kernel<<<batch, 32, 0, s>>>(tokens, parents, scores, eos, alpha, sequences,
                                             lengths, ranked, steps, batch * beams, beams, err);
  return launched();
}

}  // namespace rnet_k
