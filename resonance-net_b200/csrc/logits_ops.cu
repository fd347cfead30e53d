// Records of a row's largest logits, and the distillation loss against such
// records with its gradient.
#include "common.cuh"
#include "gemm.cuh"
#include "kernels.cuh"
#include "logits.cuh"
#include "select.cuh"

namespace rnet_k {
namespace {

using namespace rnet_logits;

// ---------------------------------------------------------------- records
// One pass over the row for its K largest logits and its sum of exponentials.
// What bounds it is HBM for long rows, and the instructions of the selection for
// short ones.
struct TopkArgs {
  float c, inv_tau;
  float* top;
  int* idx;
  float* lse;
  int V, K;
  unsigned* err;
};

__device__ __forceinline__ void write_place(const TopkArgs& a, size_t row, int k, bool in,
                                            uint64_t key) {
  a.top[row * a.K + k] = in ? key_value(key) : -INFINITY;
  a.idx[row * a.K + k] = in ? key_index(key) : -1;
}

constexpr int TOPK_WARPS = 4;

// Rows of up to 32 * R words: a warp per row. 64 values a lane take up to 255 registers
// and are still the faster way (4096 rows of 2000 fp32, top 16: 18 us, 29.5 with a CTA a
// row; bf16, top 64: 33 and 38).
template <class T, int R>
__global__ void __launch_bounds__(32 * TOPK_WARPS) topk_warp_kernel(const T* __restrict__ logits,
                                                                    long long ld, TopkArgs a,
                                                                    int rows) {
  rnet_dev::pdl_trigger();
  __shared__ uint64_t keys[TOPK_WARPS][WARP_CAP];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const size_t row = (size_t)blockIdx.x * TOPK_WARPS + warp;
  if (row >= rows) return;
  const T* z = logits + row * ld;
  const bool even = even_start(z);
  uint32_t w[R];
#pragma unroll
  for (int j = 0; j < R; ++j) w[j] = load_word(z, lane + 32 * j, a.V, even);
  float m, s;
  const int n = warp_select<T, R>(w, a.K, a.c, keys[warp], m, s);
  for (int k = lane; k < a.K; k += 32) write_place(a, row, k, k < n, keys[warp][k]);
  if (lane == 0 && a.lse) a.lse[row] = log_sum(m, s, a.inv_tau);
}

// Longer rows: a CTA of NT threads per row.
template <class T, int NT>
__global__ void __launch_bounds__(NT, NT > 128 ? 1 : sizeof(T) == 2 ? 7 : 4)
    topk_cta_kernel(const T* __restrict__ logits, long long ld, TopkArgs a) {
  rnet_dev::pdl_trigger();
  extern __shared__ uint4 sel_buf[];
  auto& sel = *reinterpret_cast<Selection<T, NT, 32>*>(sel_buf);
  const size_t row = blockIdx.x;
  float m;
  double s;
  uint32_t parity;
  select_setup(sel, parity);
  const int n = cta_select(sel, logits + row * ld, 0, a.V, a.K, a.c, m, s, parity, a.err);
  if (threadIdx.x < a.K)
    write_place(a, row, threadIdx.x, threadIdx.x < n, sel.key[threadIdx.x]);
  if (threadIdx.x == 0 && a.lse) a.lse[row] = log_sum(m, (float)s, a.inv_tau);
}

template <class T, int NT>
cudaError_t topk_cta(const T* z, long long ld, const TopkArgs& a, int rows, cudaStream_t s) {
  auto kernel = topk_cta_kernel<T, NT>;
  constexpr int smem = sizeof(Selection<T, NT, 32>);
  static std::atomic<uint64_t> ready{0};
  const cudaError_t e = allow_smem((const void*)kernel, smem, ready);
  if (e != cudaSuccess) return e;
  kernel<<<rows, NT, smem, s>>>(z, ld, a);
  return cudaGetLastError();
}

template <class T>
cudaError_t topk_launch(const T* z, long long ld, const TopkArgs& a, int rows, cudaStream_t s) {
  constexpr int N = Words<T>::N;
  const int grid = (rows - 1) / TOPK_WARPS + 1, block = 32 * TOPK_WARPS;
  if (a.V <= 256)
    topk_warp_kernel<T, 8 / N><<<grid, block, 0, s>>>(z, ld, a, rows);
  else if (a.V <= 1024)
    topk_warp_kernel<T, 32 / N><<<grid, block, 0, s>>>(z, ld, a, rows);
  else if (a.V <= 2048)
    topk_warp_kernel<T, 64 / N><<<grid, block, 0, s>>>(z, ld, a, rows);
  else
    // while every row has an SM of its own, more threads for it (148 rows of 50001
    // fp32, top 64: 16.0 us with 512 threads, 26.9 with 128; 592 rows: 35.7 with 128;
    // 256 threads lie between)
    return rows <= rnet_gemm::num_sms() ? topk_cta<T, 512>(z, ld, a, rows, s)
                                        : topk_cta<T, 128>(z, ld, a, rows, s);
  return cudaGetLastError();
}

// ---------------------------------------------------------------- distillation
// L = w [ soft tau^2 sum_k p_k (log p_k - log q_ik) + hard (lse_1 - z_y) ],
// q = softmax(z / tau), and dL/dz = w [ soft tau (P q - p) + hard (softmax(z) -
// 1_y) ] with P = sum p. A row is read once; its exponentials, relative to the
// thread's own maximum, stay in registers until the row's sum is known and then
// only need a factor. The at most K + 1 elements that a record or label touches
// are written a second time. What bounds it is HBM: one read and one write of
// the logits.
struct DistillArgs {
  const int* t_idx;
  const float* t_val;
  const float* t_lse;
  const int* targets;
  const float* weight;
  float inv_tau, tau, soft, hard, scale;
  float limit;  // of a largest logit that is not far
  float* row_loss;
  unsigned* err;
  int V, K;
};

// What a row's gradient needs beside its elements.
struct RowGrad {
  float m;      // largest logit
  float c;      // log2(e) / tau
  float limit;
  float a, a1;  // factors of 2^term(x, m, c) and of 2^term(x, m, log2(e))
  float pf, hf; // what a unit of teacher probability and the label take off
  template <bool HARD>
  __device__ __forceinline__ float at(float x) const {
    float v = a * exp2_fast(term(x, m, c, limit));
    if (HARD) v += a1 * exp2_fast(term(x, m, LOG2E, limit));
    return v;
  }
};

// The record and label of one row, held by G lanes: entry k in lane k % G.
template <int J, int G>
struct Record {
  int idx[J];  // -1: no entry
  float z[J], p[J], lp[J];  // student's logit, teacher's probability, log2 p + ln / ln 2
  float ln;    // log of the record's own normaliser
  int y;       // label, -1: none
  float zy;
  float P;     // sum p
  bool bad;    // this lane saw an index beyond the vocabulary

  // First the loads that depend on nothing, then the student's logits at the
  // indices.
  __device__ __forceinline__ void read(size_t row, const DistillArgs& a) {
    const int lane = threadIdx.x & (G - 1);
    y = a.hard != 0.f ? a.targets[row] : -1;
#pragma unroll
    for (int j = 0; j < J; ++j) {
      const int k = lane + G * j;
      const bool in = k < a.K && a.soft != 0.f;
      idx[j] = in ? a.t_idx[row * a.K + k] : -1;
      lp[j] = in ? a.t_val[row * a.K + k] : -INFINITY;
    }
  }
  // No entry, no label.
  __device__ __forceinline__ void clear() {
    y = -1;
#pragma unroll
    for (int j = 0; j < J; ++j) idx[j] = -1;
  }
  template <class T>
  __device__ __forceinline__ void gather(const T* row, int V) {
    bad = y >= V;
    if (bad) y = -1;
    zy = y >= 0 ? to_f(row[y]) : 0.f;
#pragma unroll
    for (int j = 0; j < J; ++j) {
      if (idx[j] >= V) bad = true, idx[j] = -1;
      z[j] = idx[j] >= 0 ? to_f(row[idx[j]]) : 0.f;
    }
  }
  // Probabilities relative to the record's own maximum, or to the teacher's
  // normaliser if it is given. An entry at -inf has none. They are taken to base 2
  // with the same constant c as the student's terms, so that its rounding does not
  // show in the difference of the two, which may be small (a student near its
  // teacher); what is done once a row or entry here and in loss() is done with
  // the accurate functions for the same reason.
  __device__ __forceinline__ void weigh(size_t row, const DistillArgs& a, float c) {
    float tm = -INFINITY;
#pragma unroll
    for (int j = 0; j < J; ++j) {
      if (idx[j] < 0) lp[j] = -INFINITY;
      tm = fmaxf(tm, lp[j]);
    }
    const bool given = a.t_lse != nullptr;
    const float lse = given ? a.t_lse[row] : 0.f;
    if (!given) tm = group_max<G>(tm);
    float S = 0.f;
#pragma unroll
    for (int j = 0; j < J; ++j) {
      const float t = lp[j], d = t - tm;
      lp[j] = given ? fmaf(t, c, -__fmul_rn(lse, LOG2E)) : d * c;
      p[j] = t == -INFINITY ? 0.f : exp2f(lp[j]);
      S += p[j];
    }
    P = group_sum<G>(S);
    ln = 0.f;
    if (given || P == 0.f) return;
    ln = logf(P);
    const float inv = 1.0f / P;
#pragma unroll
    for (int j = 0; j < J; ++j) p[j] *= inv;
    P *= inv;
  }
  // tau ln(2) term(x, m, c), in the logits' own unit: where the term itself leaves
  // fp32 (a logit masked with the type's lowest value) it is the difference.
  static __device__ __forceinline__ float unit(float x, float m, float c, float tau,
                                               float limit) {
    const float t = term(x, m, c, limit);
    return t == -INFINITY && x > -INFINITY ? x - m : tau * (LN2 * t);
  }
  // This lane's part of tau sum p (ln(2) lp - ln(2) term).
  __device__ __forceinline__ float kl(float m, float c, float tau, float limit) const {
    float v = 0.f;
#pragma unroll
    for (int j = 0; j < J; ++j)
      if (p[j] != 0.f) {
        const float t = term(z[j], m, c, limit);
        v += p[j] * (t > -INFINITY ? tau * (LN2 * (lp[j] - t))
                                   : tau * (LN2 * lp[j]) - unit(z[j], m, c, tau, limit));
      }
    return v;
  }
  // The row's loss from that sum and the sums of 2^term.
  __device__ __forceinline__ float loss(const DistillArgs& a, float w, float kl, float m, float s,
                                        float s1) const {
    if (s == 0.f) return 0.f;  // every logit -inf: no distribution
    float l = 0.f;
    if (a.soft != 0.f) {
      if (P != 0.f) kl += a.tau * (P * (logf(s) - ln));
      l = a.soft * a.tau * kl;
    }
    if (y >= 0) l += a.hard * (logf(s1) - unit(zy, m, LOG2E, 1.0f, a.limit));
    return w * l;
  }
  // The record's and the label's elements, those that are `in` this CTA's share,
  // once more with their own terms, after the stores of the whole share.
  template <bool HARD, class T, class In>
  __device__ __forceinline__ void fix(T* d, const RowGrad& g, int K, In in) const {
    const int lane = threadIdx.x & 31, base = lane & ~(G - 1);
    bool hot = false, twice = J > 1;
#pragma unroll
    for (int j = 0; j < J; ++j) hot |= y >= 0 && idx[j] == y;
    if (J == 1) {
      // the same index in two lanes of a group (groups told apart by their first lane)
      const int tag = idx[0] < 0 ? ~lane : idx[0] | base << 20;
      twice = __any_sync(~0u, (__match_any_sync(~0u, tag) & ~(1u << lane)) != 0);
    }
    float sum[J];
#pragma unroll
    for (int j = 0; j < J; ++j) sum[j] = p[j];
    if (twice) {  // the same index may come more than once: all its parts, in order
#pragma unroll
      for (int j = 0; j < J; ++j) sum[j] = 0.f;
#pragma unroll
      for (int h = 0; h < J; ++h)
        for (int k = 0; k < G && k + G * h < K; ++k) {
          const int i = __shfl_sync(~0u, idx[h], base + k);
          const float v = __shfl_sync(~0u, p[h], base + k);
#pragma unroll
          for (int j = 0; j < J; ++j)
            if (idx[j] == i) sum[j] += v;
        }
    }
#pragma unroll
    for (int j = 0; j < J; ++j)
      if (idx[j] >= 0 && in(idx[j])) {
        float v = g.at<HARD>(z[j]) - g.pf * sum[j];
        if (HARD && idx[j] == y) v -= g.hf;
        from_f(d + idx[j], v);
      }
    if (HARD) {
      const uint32_t any = __ballot_sync(~0u, hot) >> base & (G == 32 ? ~0u : (1u << (G & 31)) - 1);
      if (!any && lane == base && y >= 0 && in(y)) from_f(d + y, g.at<HARD>(zy) - g.hf);
    }
  }
};

// Gradient factors from the row's maximum m and its sums s (at tau) and s1 (at
// 1) of 2^term. The quotients are within 2 ulp.
__device__ __forceinline__ RowGrad row_factors(float P, bool label, const DistillArgs& a, float w,
                                               float m, float s, float s1) {
  RowGrad g;
  const bool none = s == 0.f;  // every logit -inf: no distribution
  const float gw = none ? 0.f : w * a.scale;
  g.m = m;
  g.c = a.inv_tau * LOG2E;
  g.limit = a.limit;
  g.pf = a.soft != 0.f ? gw * a.soft * a.tau : 0.f;
  g.hf = label ? gw * a.hard : 0.f;
  g.a = none || a.soft == 0.f ? 0.f : g.pf * __fdividef(P, s);
  g.a1 = none || !label ? 0.f : g.hf * __fdividef(1.0f, s1);
  return g;
}

// A thread's share of a row: E elements in pieces, and one edge element. The
// exponentials are kept (KEEP) and only need a factor later. With labels there are
// two of each: a CTA per row computes them again instead, which leaves room for more
// CTAs (4096 rows of 8000 fp32: 45 us, 58 with both kept); a warp per row keeps them
// (16384 rows of 1000: 35.6 us, 39.5 computed again).
template <class T, int E, bool HARD, bool KEEP>
struct Share {
  static constexpr int N = Piece<T>::N, NP = E / N;
  float e[KEEP ? E + 1 : 1], e1[KEEP && HARD ? E + 1 : 1];
  float m, s, s1;  // largest logit and sums, relative to it

  __device__ __forceinline__ void take(const Piece<T>* x, float edge, float c,
                                       float limit) {
    m = fmaxf(piece_max<NP>(x), edge);
    s = s1 = 0.f;
    const float mc = __fmul_rn(m, c), m1 = __fmul_rn(m, LOG2E);
    if (far(m, limit)) {
      fill(x, edge, [&](float v) { return (v - m) * c; }, [&](float v) { return (v - m) * LOG2E; });
    } else {
      fill(x, edge, [&](float v) { return fmaf(v, c, -mc); },
           [&](float v) { return fmaf(v, LOG2E, -m1); });
    }
  }
  template <class F, class F1>
  __device__ __forceinline__ void fill(const Piece<T>* x, float edge, F t, F1 t1) {
#pragma unroll
    for (int i = 0; i <= E; ++i) {
      const float v = i < E ? x[i / N].get(i % N) : edge;
      const float w = exp2_fast(t(v));
      s += w;
      if (KEEP) e[i] = w;
      if (HARD) {
        const float w1 = exp2_fast(t1(v));
        s1 += w1;
        if (KEEP) e1[i] = w1;
      }
    }
  }
  // The gradient of every element, to the pieces q0 + j * step below q1 and to the
  // edge element. f, f1: what this thread's kept exponentials are multiplied with.
  __device__ __forceinline__ void write(T* d, const Grid<T>& grid, const Piece<T>* x, float xe,
                                        int q0, int step, int q1, int edge, const RowGrad& g,
                                        float f, float f1) const {
    T* p = d + grid.at(q0);
    auto all = [&](bool wide, auto grad) {
#pragma unroll
      for (int j = 0; j < NP; ++j) {
        float v[N];
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = grad(j * N + i);
        if (q0 + j * step < q1) Piece<T>::store(p + j * step * N, v, wide);
      }
      if (edge >= 0) from_f(d + edge, grad(E));
    };
    const bool wide = ((uintptr_t)p & 15) == 0;
    if constexpr (!KEEP) {
      auto at = [&](int i) { return i < E ? x[i / N].get(i % N) : xe; };
      const float mc = __fmul_rn(g.m, g.c), m1 = __fmul_rn(g.m, LOG2E);
      if (wide && !far(g.m, g.limit))
        all(true, [&](int i) {
          return fmaf(g.a1, exp2_fast(fmaf(at(i), LOG2E, -m1)),
                      g.a * exp2_fast(fmaf(at(i), g.c, -mc)));
        });
      else
        all(wide, [&](int i) { return g.template at<true>(at(i)); });
    } else {
      auto grad = [&](int i) { return HARD ? fmaf(f1, e1[i], f * e[i]) : f * e[i]; };
      if (wide) all(true, grad);
      else all(false, grad);  // the logits and their gradient lie differently on the grid
    }
  }
};

// The pieces q0 + j * step below q1 of a row.
template <class T, int NP>
__device__ __forceinline__ void load_pieces(Piece<T>* x, const T* z, const Grid<T>& grid, int q0,
                                            int step, int q1) {
  const T* p = z + grid.at(q0);
#pragma unroll
  for (int j = 0; j < NP; ++j) {
    x[j].none();
    if (q0 + j * step < q1) x[j].load(p + j * step * Piece<T>::N);
  }
}
template <class T>
__device__ __forceinline__ void zero_pieces(T* d, const Grid<T>& grid, int q0, int step, int q1,
                                            int edge) {
  const float zero[Piece<T>::N] = {};
  for (int q = q0; q < q1; q += step)
    Piece<T>::store(d + grid.at(q), zero, ((uintptr_t)(d + grid.head) & 15) == 0);
  if (edge >= 0) from_f(d + edge, 0.f);
}

constexpr int WARPS = 8;  // rows of a CTA of the warp-per-row kernel

// Rows of up to G * E elements in pieces: G lanes per row. With 16 lanes a warp
// has two rows and what a row costs beside its elements is paid once for both. Six CTAs
// to an SM make 8 elements with labels spill 44 to 140 bytes; four, which need no spill,
// are neither slower nor faster (16384 rows of 256, top 32: 16.5 us, 16.9 with four).
template <class T, int E, int G, int J, bool HARD>
__global__ void __launch_bounds__(32 * WARPS, E <= 8 ? 6 : E <= 16 ? 3 : 2) distill_warp_kernel(
    const T* logits, long long ld, T* dlogits, long long ldd, DistillArgs a, int rows) {
  rnet_dev::pdl_trigger();
  constexpr int N = Piece<T>::N, NP = E / N, PER = 32 / G;
  const int lane = threadIdx.x & (G - 1);
  const size_t first = ((size_t)blockIdx.x * WARPS + (threadIdx.x >> 5)) * PER;
  if (first >= rows) return;
  // a group without a row of its own works on the last one, and keeps it to itself
  const size_t own = first + (threadIdx.x & 31) / G;
  const bool on = own < rows;
  const size_t row = on ? own : rows - 1;
  const float w = a.weight ? a.weight[row] : 1.0f;
  Record<J, G> r;
  r.read(row, a);
  const T* z = logits + row * ld;
  const Grid<T> grid(z, a.V);
  const int edge = grid.edge(lane);
  Piece<T> x[NP];
  load_pieces<T, NP>(x, z, grid, lane, G, grid.pieces);
  float xe = edge >= 0 ? to_f(z[edge]) : -INFINITY;
  if (w == 0.f) {
    // whatever the row holds: as one without a distribution, a record and a label
#pragma unroll
    for (int j = 0; j < NP; ++j) x[j].none();
    xe = -INFINITY;
    r.clear();
  }
  r.gather(z, a.V);
  const float c = a.inv_tau * LOG2E;
  Share<T, E, HARD, true> h;
  h.take(x, xe, c, a.limit);
  r.weigh(row, a, c);
  const float m = group_max<G>(h.m);
  const float f = rebase(h.m, m, c, a.limit), f1 = HARD ? rebase(h.m, m, LOG2E, a.limit) : 0.f;
  const float s = group_sum<G>(h.s * f), s1 = HARD ? group_sum<G>(h.s1 * f1) : 0.f;
  const float kl = group_sum<G>(r.kl(m, c, a.tau, a.limit));
  if (lane == 0 && on) a.row_loss[row] = r.loss(a, w, kl, m, s, s1);
  if (r.bad && a.err) atomicOr(a.err, rnet_dev::ERR_BAD_INDEX);
  if (!dlogits) return;
  T* d = dlogits + row * ldd;
  const RowGrad g = row_factors(r.P, r.y >= 0, a, w, m, s, s1);
  __syncwarp();  // the reads of the row come before the stores, where dlogits are the logits
  if (on) h.write(d, grid, x, xe, lane, G, grid.pieces, edge, g, g.a * f, g.a1 * f1);
  __syncwarp();  // orders the stores above before those below
  r.template fix<HARD>(d, g, a.K, [&](int) { return on; });
}

// A row's maximum and sums from the parts (m, s, s1) of n warps, joined in the
// same order by every warp.
template <int MOST, bool HARD>
__device__ __forceinline__ void join_parts(const float4* part, int n, float c, float limit,
                                           float& m, float& s, float& s1) {
  const int lane = threadIdx.x & 31;
  float4 got[MOST];
  m = -FLT_MAX;
#pragma unroll
  for (int i = 0; i < MOST; ++i) {
    got[i] = make_float4(-FLT_MAX, 0.f, 0.f, 0.f);
    if (lane + 32 * i < n) got[i] = part[lane + 32 * i];
    m = fmaxf(m, got[i].x);
  }
  m = warp_max(m);
  s = s1 = 0.f;
#pragma unroll
  for (int i = 0; i < MOST; ++i) {
    if (32 * i >= n) break;
    s += got[i].y * rebase(got[i].x, m, c, limit);
    if (HARD) s1 += got[i].z * rebase(got[i].x, m, LOG2E, limit);
  }
  s = warp_sum(s);
  if (HARD) s1 = warp_sum(s1);
}

// Rows of up to 256 * E elements in pieces: a CTA per row, the row in
// registers. Warp 0 holds the record. As many CTAs to an SM as need no spills, but for 8
// bytes of 8 fp32 elements with labels and a long record (4096 rows of 8000 fp32 with
// labels: 45 us with four, 49.6 with three).
template <class T, int E, int J, bool HARD>
constexpr int CTAS = E <= 8 ? 6 : E <= 16 ? 5 : (sizeof(T) == 2 && HARD ? 6 : 5) - J;
template <class T, int E, int J, bool HARD>
__global__ void __launch_bounds__(256, CTAS<T, E, J, HARD>)
    distill_cta_kernel(const T* logits, long long ld, T* dlogits, long long ldd, DistillArgs a) {
  rnet_dev::pdl_trigger();
  constexpr int N = Piece<T>::N, NP = E / N;
  __shared__ float4 part[8];
  __shared__ float s_P;
  __shared__ int s_label;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const size_t row = blockIdx.x;
  const float w = a.weight ? a.weight[row] : 1.0f;
  Record<J, 32> r;
  if (warp == 0) r.read(row, a);
  const T* z = logits + row * ld;
  const Grid<T> grid(z, a.V);
  const int edge = tid < 2 * N ? grid.edge(tid) : -1;
  Piece<T> x[NP];
  load_pieces<T, NP>(x, z, grid, tid, 256, grid.pieces);
  const float xe = edge >= 0 ? to_f(z[edge]) : -INFINITY;
  T* d = dlogits ? dlogits + row * ldd : nullptr;
  if (w == 0.f) {  // whatever the row holds
    if (d) zero_pieces(d, grid, tid, 256, grid.pieces, edge);
    if (tid == 0) a.row_loss[row] = 0.f;
    return;
  }
  if (warp == 0) r.gather(z, a.V);
  const float c = a.inv_tau * LOG2E;
  Share<T, E, HARD, !HARD> h;
  h.take(x, xe, c, a.limit);
  if (warp == 0) {
    r.weigh(row, a, c);
    if (lane == 0) s_P = r.P, s_label = r.y >= 0;
    if (r.bad && a.err) atomicOr(a.err, rnet_dev::ERR_BAD_INDEX);
  }
  float m = warp_max(h.m);
  float s = warp_sum(h.s * rebase(h.m, m, c, a.limit));
  float s1 = HARD ? warp_sum(h.s1 * rebase(h.m, m, LOG2E, a.limit)) : 0.f;
  if (lane == 0) part[warp] = make_float4(m, s, s1, 0.f);
  __syncthreads();
  join_parts<1, HARD>(part, 8, c, a.limit, m, s, s1);
  if (warp == 0) {
    const float kl = warp_sum(r.kl(m, c, a.tau, a.limit));
    if (lane == 0) a.row_loss[row] = r.loss(a, w, kl, m, s, s1);
  }
  if (!d) return;
  const RowGrad g = row_factors(s_P, s_label, a, w, m, s, s1);
  h.write(d, grid, x, xe, tid, 256, grid.pieces, edge, g,
          HARD ? 0.f : g.a * rebase(h.m, m, c, a.limit), 0.f);
  __syncthreads();  // orders the stores above before those below
  if (warp == 0) r.template fix<HARD>(d, g, a.K, [](int) { return true; });
}

__device__ __forceinline__ void store_remote(float4* p, uint32_t rank, float4 v) {
  asm volatile(
      "{\n\t.reg .b32 ra;\n\t"
      "mapa.shared::cluster.u32 ra, %0, %1;\n\t"
      "st.shared::cluster.v4.f32 [ra], {%2, %3, %4, %5};\n\t}" ::"r"(rnet_dev::smem_u32(p)),
      "r"(rank), "f"(v.x), "f"(v.y), "f"(v.z), "f"(v.w)
      : "memory");
}

constexpr int CLUSTER = 8;  // CTAs of one row at most
constexpr int CHUNKS = 5;
// Pieces of a row in one CTA's shared memory, so that two CTAs of 512 threads share
// an SM and one reads while the other computes and writes; with 256 threads, four
// (4096 rows of 10000 fp32: 56.4 us, 79.1 with 512 threads).
constexpr int SHARE = 108 * 1024 / 16, SHARE_256 = 54 * 1024 / 16;
// Pieces that arrive together, 64 bytes a thread.
template <int NT>
constexpr int CHUNK = 4 * NT;
static_assert(RNET_DISTILL_VOCAB_MAX * 4 / 16 <= CLUSTER * CHUNK<512> * CHUNKS, "vocab limit");
static_assert(SHARE_256 <= CHUNK<256> * CHUNKS, "share limit");

// Longer rows: a cluster of C CTAs per row, each with `per` pieces in shared
// memory. Chunks of the row arrive by bulk copies, and their maxima and sums are
// taken as they do. Every warp leaves its own in the shared memory of all CTAs of
// the cluster: one exchange, and the same bits everywhere. The gradient is then
// computed from shared memory. Warp 0 of each CTA holds the record.
template <class T, int NT, int J, bool HARD>
__global__ void __launch_bounds__(NT, 1024 / NT)
    distill_long_kernel(const T* logits, long long ld, T* dlogits, long long ldd, DistillArgs a,
                        int per) {
  rnet_dev::pdl_trigger();
  constexpr int N = Piece<T>::N, NW = NT / 32, CH = CHUNK<NT>;
  extern __shared__ uint4 long_buf[];
  Piece<T>* const buf = reinterpret_cast<Piece<T>*>(long_buf);
  __shared__ float4 part[CLUSTER * NW];  // m, s, s1
  __shared__ __align__(8) uint64_t bar[CHUNKS];
  __shared__ float s_P;
  __shared__ int s_label, s_abort[2];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const size_t row = blockIdx.x;
  const int rank = blockIdx.y, C = gridDim.y;
  const T* z = logits + row * ld;
  const Grid<T> grid(z, a.V);
  const int begin = min(rank * per, grid.pieces), n = min(per, grid.pieces - begin);
  if (tid == 0) {
    s_abort[0] = s_abort[1] = 0;
    for (int i = 0; i < CHUNKS; ++i) rnet_dev::mbar_init(&bar[i], 1);
    rnet_dev::fence_barrier_init();
    for (int i = 0; i * CH < n; ++i) {
      const uint32_t bytes = 16u * min(CH, n - i * CH);
      rnet_dev::mbar_arrive_expect_tx(&bar[i], bytes);
      bulk_load(buf + i * CH, z + grid.at(begin + i * CH), bytes, &bar[i]);
    }
  }
  // the peers' shared memory may be written once all of them run
  if (C > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
  const float w = a.weight ? a.weight[row] : 1.0f;
  Record<J, 32> r;
  if (warp == 0) r.read(row, a);
  const int edge = rank == 0 && tid < 2 * N ? grid.edge(tid) : -1;  // the first CTA's
  const float xe = edge >= 0 ? to_f(z[edge]) : -INFINITY;
  T* d = dlogits ? dlogits + row * ldd : nullptr;
  const float c = a.inv_tau * LOG2E;
  if (warp == 0) {
    r.gather(z, a.V);
    r.weigh(row, a, c);
    if (lane == 0) s_P = r.P, s_label = r.y >= 0;
    if (r.bad && rank == 0 && w != 0.f && a.err) atomicOr(a.err, rnet_dev::ERR_BAD_INDEX);
  }
  __syncthreads();  // the barriers are set up
  float m = -FLT_MAX, s = 0.f, s1 = 0.f;
  bool again = false;  // a largest logit on the way was far
  auto add = [&](float mx, bool first, auto each) {
    const float mc = __fmul_rn(mx, c), m1 = __fmul_rn(mx, LOG2E);
    again |= far(mx, a.limit);
    if (!first) {
      s *= exp2_fast(__fmul_rn(m, c) - mc);
      if (HARD) s1 *= exp2_fast(__fmul_rn(m, LOG2E) - m1);
    }
    m = mx;
    each([&](float v) {
      s += exp2_fast(fmaf(v, c, -mc));
      if (HARD) s1 += exp2_fast(fmaf(v, LOG2E, -m1));
    });
  };
  for (int i = 0; i * CH < n; ++i) {
    // a copy that does not come is reported and given the same time once more:
    // none may land in memory that the CTA has left
    if (!rnet_dev::mbar_wait(&bar[i], 0, a.err, &s_abort[0]))
      rnet_dev::mbar_wait(&bar[i], 0, a.err, &s_abort[1]);
    Piece<T> x[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int q = i * CH + j * NT + tid;
      x[j].none();
      if (q < n) x[j] = buf[q];
    }
    add(fmaxf(m, piece_max<4>(x)), i == 0, [&](auto f) {
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int k = 0; k < N; ++k) f(x[j].get(k));
    });
  }
  if (edge >= 0) add(fmaxf(m, xe), false, [&](auto f) { f(xe); });
  if (again) {  // the sums once more, relative to the largest of all
    s = s1 = 0.f;
    auto take = [&](float v) {
      s += exp2_fast(term(v, m, c, a.limit));
      if (HARD) s1 += exp2_fast(term(v, m, LOG2E, a.limit));
    };
    for (int q = tid; q < n; q += NT) {
      const Piece<T> x = buf[q];
#pragma unroll
      for (int k = 0; k < N; ++k) take(x.get(k));
    }
    if (edge >= 0) take(xe);
  }
  {
    const float mw = warp_max(m);
    s = warp_sum(s * rebase(m, mw, c, a.limit));
    if (HARD) s1 = warp_sum(s1 * rebase(m, mw, LOG2E, a.limit));
    m = mw;
  }
  const float4 mine = make_float4(m, s, s1, 0.f);
  if (C > 1) {
    asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
    if (lane < C) store_remote(&part[rank * NW + warp], lane, mine);
    rnet_dev::cluster_sync();
  } else {
    if (lane == 0) part[warp] = mine;
    __syncthreads();
  }
  if (w == 0.f) {  // whatever the row holds
    if (d) zero_pieces(d, grid, begin + tid, NT, begin + n, edge);
    if (rank == 0 && tid == 0) a.row_loss[row] = 0.f;
    return;
  }
  join_parts<CLUSTER * NW / 32, HARD>(part, C * NW, c, a.limit, m, s, s1);
  if (rank == 0 && warp == 0) {
    const float kl = warp_sum(r.kl(m, c, a.tau, a.limit));
    if (lane == 0) a.row_loss[row] = r.loss(a, w, kl, m, s, s1);
  }
  if (!d) return;
  const RowGrad g = row_factors(s_P, s_label, a, w, m, s, s1);
  T* p = d + grid.at(begin);
  auto write = [&](bool wide, auto value) {
#pragma unroll 2
    for (int q = tid; q < n; q += NT) {
      const Piece<T> x = buf[q];
      float v[N];
#pragma unroll
      for (int k = 0; k < N; ++k) v[k] = value(x.get(k));
      Piece<T>::store(p + (size_t)q * N, v, wide);
    }
  };
  const float mc = __fmul_rn(m, c), m1 = __fmul_rn(m, LOG2E);
  auto near_value = [&](float v) {
    const float e = g.a * exp2_fast(fmaf(v, c, -mc));
    return HARD ? fmaf(g.a1, exp2_fast(fmaf(v, LOG2E, -m1)), e) : e;
  };
  if (far(m, a.limit) || ((uintptr_t)p & 15))
    // also where logits and gradient lie differently on the 16-byte grid
    write(((uintptr_t)p & 15) == 0, [&](float v) { return g.template at<HARD>(v); });
  else
    write(true, near_value);
  if (edge >= 0) from_f(d + edge, g.template at<HARD>(xe));
  __syncthreads();  // orders the stores above before those below
  if (warp == 0) {
    const int lo = grid.at(begin), hi = grid.at(begin + n);
    const int head = grid.head, tail = grid.at(grid.pieces);
    r.template fix<HARD>(d, g, a.K, [&](int e) {
      return (e >= lo && e < hi) || (rank == 0 && (e < head || e >= tail));
    });
  }
}

template <class T, int NT, int J, bool HARD>
cudaError_t distill_long_as(const T* z, long long ld, T* d, long long ldd, const DistillArgs& a,
                            int rows, int C, cudaStream_t s) {
  auto kernel = distill_long_kernel<T, NT, J, HARD>;
  const int per = (a.V / Piece<T>::N + C - 1) / C;
  if (per > CHUNK<NT> * CHUNKS) return cudaErrorInvalidValue;
  static std::atomic<uint64_t> ready{0};
  cudaError_t e = allow_smem((const void*)kernel, 16 * CHUNK<NT> * CHUNKS, ready);
  if (e != cudaSuccess) return e;
  const ClusterLaunch l(dim3(rows, C), NT, (size_t)per * 16, s);
  return cudaLaunchKernelEx(&l.cfg, kernel, z, ld, d, ldd, a, per);
}

template <class T, int J, bool HARD>
cudaError_t distill_long(const T* z, long long ld, T* d, long long ldd, const DistillArgs& a,
                         int rows, cudaStream_t s) {
  const int pieces = a.V / Piece<T>::N, sms = rnet_gemm::num_sms();
  // one CTA while the row fits one, else shares of the smaller size (2048 rows of
  // 30000 fp32: 90.5 us in three CTAs, 106 in two)
  int C = pieces <= SHARE ? 1 : (pieces + SHARE_256 - 1) / SHARE_256;
  if (C > CLUSTER) C = (pieces + SHARE - 1) / SHARE;
  // more CTAs while they would leave SMs idle and have two chunks each
  while (C < CLUSTER && (long long)rows * (C + 1) <= sms && pieces / (C + 1) >= 1024) ++C;
  if (C > CLUSTER) C = CLUSTER;
  return (pieces + C - 1) / C <= SHARE_256 && rows > sms
             ? distill_long_as<T, 256, J, HARD>(z, ld, d, ldd, a, rows, C, s)
             : distill_long_as<T, 512, J, HARD>(z, ld, d, ldd, a, rows, C, s);
}

template <class T, int E, int G, int J, bool HARD>
void distill_warp(const T* z, long long ld, T* d, long long ldd, const DistillArgs& a, int rows,
                  cudaStream_t s) {
  constexpr int PER = WARPS * (32 / G);  // rows of a CTA
  distill_warp_kernel<T, E, G, J, HARD>
      <<<(rows - 1) / PER + 1, 32 * WARPS, 0, s>>>(z, ld, d, ldd, a, rows);
}

template <class T, int J, bool HARD>
cudaError_t distill_launch(const T* z, long long ld, T* d, long long ldd, const DistillArgs& a,
                           int rows, cudaStream_t s) {
  const int V = a.V;  // at least the elements in pieces
  if constexpr (J == 1) {
    // two rows a warp (16384 rows of 256, top 16: 10.7 us, 13.3 with a row each; with
    // labels 13.4 and 15.9; 1024 rows 4.8 and 4.5). A longer record would take two
    // entries a lane, and the search for repeated indices more than it saves.
    if (V <= 32 * 8 && a.K <= 16 && rows >= 2048) {
      distill_warp<T, 16, 16, J, HARD>(z, ld, d, ldd, a, rows, s);
      return cudaGetLastError();
    }
  }
  if (V <= 32 * 8)
    distill_warp<T, 8, 32, J, HARD>(z, ld, d, ldd, a, rows, s);
  else if (V <= 32 * 16)
    distill_warp<T, 16, 32, J, HARD>(z, ld, d, ldd, a, rows, s);
  else if (V <= 32 * 32)
    distill_warp<T, 32, 32, J, HARD>(z, ld, d, ldd, a, rows, s);
  else if (V <= 256 * 8)
    distill_cta_kernel<T, 8, J, HARD><<<rows, 256, 0, s>>>(z, ld, d, ldd, a);
  else if (V <= 256 * 16)
    distill_cta_kernel<T, 16, J, HARD><<<rows, 256, 0, s>>>(z, ld, d, ldd, a);
  else if (V <= 256 * 32)
    distill_cta_kernel<T, 32, J, HARD><<<rows, 256, 0, s>>>(z, ld, d, ldd, a);
  else
    return distill_long<T, J, HARD>(z, ld, d, ldd, a, rows, s);
  return cudaGetLastError();
}

// Sum of the rows' losses in 64 bits, in a fixed order. Launched so that it may
// start while the last rows are still at work, and then waits for all of them.
__global__ void __launch_bounds__(1024) sum_rows_kernel(const float* __restrict__ x,
                                                        unsigned n,
                                                        float* __restrict__ out) {
  __shared__ double sh[32];
  rnet_dev::pdl_wait();
  rnet_dev::pdl_trigger();
  double a = 0.0;
  unsigned i = threadIdx.x;  // steps past the last of up to 2^31 - 1 rows
  for (; i + 7 * 1024 < n; i += 8 * 1024) {
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = x[i + j * 1024];
#pragma unroll
    for (int j = 0; j < 8; ++j) a += v[j];
  }
  for (; i < n; i += 1024) a += x[i];
#pragma unroll
  for (int o = 16; o; o >>= 1) a += __shfl_xor_sync(~0u, a, o);
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = a;
  __syncthreads();
  if (threadIdx.x >= 32) return;
  a = sh[threadIdx.x];
#pragma unroll
  for (int o = 16; o; o >>= 1) a += __shfl_xor_sync(~0u, a, o);
  if (threadIdx.x == 0) *out = (float)a;
}

cudaError_t sum_rows(const float* x, int n, float* out, cudaStream_t s) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(1);
  cfg.blockDim = dim3(1024);
  cfg.stream = s;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, sum_rows_kernel, x, n, out);
}

}  // namespace

cudaError_t topk_logits(const void* logits, bool bf16, long long ld, float tau, float* top,
                        int* idx, float* lse, int rows, int V, int K, unsigned* err,
                        cudaStream_t s) {
  if (rows <= 0) return cudaSuccess;
  const TopkArgs a{LOG2E / tau, 1.0f / tau, top, idx, lse, V, K, err};
  const cudaError_t e = bf16 ? topk_launch((const __nv_bfloat16*)logits, ld, a, rows, s)
                             : topk_launch((const float*)logits, ld, a, rows, s);
  return e != cudaSuccess ? e : launched();
}

cudaError_t distill_topk(const void* logits, bool bf16, long long ld, const int* t_idx,
                         const float* t_val, const float* t_lse, const int* targets,
                         const float* weight, float tau, float soft, float hard, float scale,
                         float* row_loss, float* loss, void* dlogits, long long ldd, int rows,
                         int V, int K, unsigned* err, cudaStream_t s) {
  const float c = LOG2E / tau, most = hard != 0.f && c < LOG2E ? LOG2E : c;
  DistillArgs a{t_idx, t_val, t_lse, targets, weight,        1.0f / tau, tau, soft,
                hard,  scale, 0x1p24f / most, row_loss, err, V,          K};
  if (rows > 0) {
    auto run = [&](auto type) {
      using T = decltype(type);
      const T* z = (const T*)logits;
      T* d = (T*)dlogits;
      if (hard != 0.f)
        return K > 32 ? distill_launch<T, 2, true>(z, ld, d, ldd, a, rows, s)
                      : distill_launch<T, 1, true>(z, ld, d, ldd, a, rows, s);
      return K > 32 ? distill_launch<T, 2, false>(z, ld, d, ldd, a, rows, s)
                    : distill_launch<T, 1, false>(z, ld, d, ldd, a, rows, s);
    };
    const cudaError_t e = bf16 ? run(__nv_bfloat16()) : run(0.0f);
    if (e != cudaSuccess) return e;
    launched();
  }
  if (!loss) return cudaSuccess;
  const cudaError_t e = sum_rows(row_loss, rows, loss, s);
  return e != cudaSuccess ? e : launched();
}

}  // namespace rnet_k
