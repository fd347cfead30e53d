// Beam search: selection over beams and vocabulary, reordering of the streams'
// states by the chosen parents, and the sequences behind the last beams.
#include "common.cuh"
#include "gemm.cuh"
#include "kernels.cuh"
#include "logits.cuh"
#include "select.cuh"

namespace rnet_k {
namespace {

using namespace rnet_logits;

// ---------------------------------------------------------------- selection
// The best `beams` of score[b] + z[b][v] - lse[b] over (b, v): within a row the
// order of the totals is that of the logits, so each row (or slice of a row)
// gives its W largest logits and its sum of exponentials, and one CTA merges the
// lists. Totals are formed and compared in 64 bits, score and logit first: beams
// with the same row tie where their sums are equal.
// What bounds it is HBM for long rows, latency for short ones.
struct SelectArgs {
  const float* scores_in;
  const int* finished_in;
  int eos;
  float* scores;
  int *tokens, *parents, *finished;
  int W, V;
  unsigned* err;
};

constexpr int SELECT_CTAS = 16;  // of one sequence's cluster, where the device places them

// A list per (beam, slice), in that order, largest first.
struct Lists {
  uint64_t key[RNET_BEAMS_MAX][RNET_BEAMS_MAX];
  double s[RNET_BEAMS_MAX];
  float m[RNET_BEAMS_MAX];
  int n[RNET_BEAMS_MAX];
  // the merge's own
  uint64_t total[RNET_BEAMS_MAX * RNET_BEAMS_MAX];
  int which[RNET_BEAMS_MAX * RNET_BEAMS_MAX];  // 32 list + place
  double score[RNET_BEAMS_MAX], lse[RNET_BEAMS_MAX];
  uint32_t done, bound;
  int totals;
};

__device__ __forceinline__ uint64_t order(double x) {
  const int64_t b = __double_as_longlong(x);
  return (uint64_t)b ^ ((uint64_t)(b >> 63) | 0x8000000000000000ull);
}

__device__ __forceinline__ double unorder(uint64_t o) {
  return __longlong_as_double((int64_t)(o >> 63 ? o ^ 0x8000000000000000ull : ~o));
}

// What lane l of the first warp knows of list l's beam. Loaded ahead of the lists, so
// that the merge does not wait for it.
struct Standing {
  float score = 0.f;
  bool done = false;
  __device__ __forceinline__ void load(const SelectArgs& a, size_t m0, int S) {
    const int lane = threadIdx.x & 31;
    if (lane >= a.W * S) return;
    score = a.scores_in[m0 + lane / S];
    done = a.finished_in && a.finished_in[m0 + lane / S];
  }
};

// Candidates that are ranked by counting. Beyond, a warp takes the best head W times over
// (8 x 32 x 256 of equal logits: 18 us, 129 by counting).
constexpr int MERGE_COUNT = 128;
static_assert(SELECT_CTAS * (SELECT_CTAS / 2) <= MERGE_COUNT, "more only from whole rows");

// The W best of the W * S lists, by a whole CTA. W candidates reach the W-th largest of
// the lists' first ones (of their distinct upper halves), and what reaches it is ranked
// by counting (32 x 8 x 256: 4.2 us, 5.3 with a warp that takes the best head W times
// over). With many lists, all of them whole rows, that bound is the worst list's and lets
// most of the W * W through: d * r >= W candidates also reach the r-th largest of the
// lists' d-th ones, and a warp for each d = 2, 4, .. finds one more bound.
__device__ __forceinline__ void merge(Lists& in, const SelectArgs& a, size_t m0, int S,
                                      const Standing& now) {
  const int tid = threadIdx.x, W = a.W, lists = W * S;
  const uint64_t none = order(-(double)INFINITY);
  if (tid < 32) {
    const bool on = tid < lists;
    const double score = canon(now.score);
    double lse = 0.0;
    uint64_t head = none;
    if (on) {
      if (now.done) {
        in.n[tid] = tid % S == 0;  // (beam, eos) at its own score
        if (tid % S == 0) head = order(score);
      } else {
        const int first = tid - tid % S;
        float m = in.m[tid];
        double s = in.s[tid];
        if (S > 1) {
#pragma unroll 4
          for (int i = 0; i < S; ++i) m = fmaxf(m, in.m[first + i]);
          s = 0.0;
#pragma unroll 4
          for (int i = 0; i < S; ++i)
            s += in.s[first + i] * (double)exp2_fast((in.m[first + i] - m) * LOG2E);
        }
        lse = log_sum(m, s);
        if (in.n[tid]) head = order((score + (double)key_value(in.key[tid][0])) - lse);
      }
      in.score[tid] = score;
      in.lse[tid] = lse;
    }
    const uint32_t done = __ballot_sync(~0u, now.done);
    uint32_t high = (uint32_t)(head >> 32), bound;
    if (S == 1) {
      bound = __reduce_min_sync(~0u, on ? high : ~0u);
    } else {
      high = on ? high : 0;
      bound = __reduce_max_sync(~0u, high);
      for (int j = 1; j < W; ++j) {
        high = high == bound ? 0 : high;
        bound = __reduce_max_sync(~0u, high);
      }
    }
    if (tid == 0) in.done = done, in.bound = bound, in.totals = 0;
  }
  __syncthreads();
  if (W > 8 && S == 1) {
    const int lane = tid & 31, d = 2 << (tid >> 5);
    if (d <= W) {
      uint32_t high = 0;
      if (lane < W && in.n[lane] >= d)
        high = order((in.score[lane] + (double)key_value(in.key[lane][d - 1])) - in.lse[lane]) >>
               32;
      uint32_t bound = __reduce_max_sync(~0u, high);
      for (int j = d; j < W; j += d) {
        high = high == bound ? 0 : high;
        bound = __reduce_max_sync(~0u, high);
      }
      if (lane == 0) atomicMax(&in.bound, bound);
    }
    __syncthreads();
  }
  for (int c = tid; c < lists * W; c += blockDim.x) {
    const int list = c / W, i = c % W;
    if (i >= in.n[list]) continue;
    // the sum of two fp32 is exact, or near it
    double t = in.score[list];
    if (!(in.done >> list & 1)) t = (t + (double)key_value(in.key[list][i])) - in.lse[list];
    const uint64_t o = order(t);
    if (o <= none || (uint32_t)(o >> 32) < in.bound) continue;
    const int at = atomicAdd(&in.totals, 1);
    in.total[at] = o;
    in.which[at] = list * 32 + i;
  }
  __syncthreads();
  const int n = in.totals, end = a.eos >= 0 ? a.eos : 0;
  auto put = [&](int j, float score, int parent, int token, bool done) {
    a.scores[m0 + j] = score;
    a.parents[m0 + j] = parent;
    a.tokens[m0 + j] = token;
    if (a.finished) a.finished[m0 + j] = done || token == a.eos;
  };
  auto choose = [&](int place, int which, uint64_t total) {
    const int list = which >> 5;
    const bool done = in.done >> list & 1;
    put(place, (float)unorder(total), list / S,
        done ? end : key_index(in.key[list][which & 31]), done);
  };
  // Equal totals go to the lower beam, then the larger logit or lower token: a row's
  // slices do not show.
  if (n <= MERGE_COUNT) {
    for (int c = tid; c < n; c += blockDim.x) {
      const uint64_t own = in.total[c];
      const int which = in.which[c], list = which >> 5;
      int place = 0, equal = 0;
#pragma unroll 4
      for (int k = 0; k < n; ++k) {
        const uint64_t t = in.total[k];
        place += t > own;
        equal += t == own;
      }
      if (equal > 1 && S == 1) {
        for (int k = 0; k < n; ++k) place += in.total[k] == own && in.which[k] < which;
      } else if (equal > 1) {
        const uint64_t key = in.key[list][which & 31];
        const int first = list - list % S;  // of the beam's lists
        for (int k = 0; k < n; ++k) {
          const int other = in.which[k] >> 5;
          place += in.total[k] == own &&
                   (other < first ||
                    (other < first + S && in.key[other][in.which[k] & 31] > key));
        }
      }
      if (place < W) choose(place, which, own);
    }
  } else if (tid < 32) {
    // ties let many through (of more than 8 beams, so S is 1): a lane to a list, and the
    // best head W times over, the lowest lane's of equal ones
    int at = 0;
    auto next = [&]() -> uint64_t {
      if (tid >= W || at >= in.n[tid]) return 0;
      double t = in.score[tid];
      if (!(in.done >> tid & 1)) t = (t + (double)key_value(in.key[tid][at])) - in.lse[tid];
      const uint64_t o = order(t);
      return o > none ? o : 0;
    };
    uint64_t head = next();
    for (int j = 0; j < W; ++j) {
      const uint32_t high = __reduce_max_sync(~0u, (uint32_t)(head >> 32));
      const uint32_t low =
          __reduce_max_sync(~0u, (uint32_t)(head >> 32) == high ? (uint32_t)head : 0u);
      const uint64_t best = (uint64_t)high << 32 | low;
      const int from = __ffs(__ballot_sync(~0u, head == best)) - 1;
      if (tid == from) {
        choose(j, tid * 32 + at, head);
        ++at;
        head = next();
      }
    }
  }
  // beams that no candidate is left for
  for (int j = n + tid; j < W; j += blockDim.x) put(j, -INFINITY, j, end, in.done >> (j * S) & 1);
}

__device__ __forceinline__ uint32_t in_first_cta(const void* p) {
  uint32_t ra;
  asm("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(ra) : "r"(rnet_dev::smem_u32(p)));
  return ra;
}
__device__ __forceinline__ void store_u64(uint32_t ra, uint64_t v) {
  asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(ra), "l"(v) : "memory");
}
__device__ __forceinline__ void store_u32(uint32_t ra, uint32_t v) {
  asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(ra), "r"(v) : "memory");
}

// A part's list and sum, into the first CTA's shared memory: lane (or thread) t
// brings key t.
__device__ __forceinline__ void deliver(Lists& lists, int u, int t, int n, uint64_t key, float m,
                                        double s) {
  if (t < n) store_u64(in_first_cta(&lists.key[u][t]), key);
  if (t == 0) {
    store_u32(in_first_cta(&lists.n[u]), n);
    store_u32(in_first_cta(&lists.m[u]), __float_as_uint(m));
    store_u64(in_first_cta(&lists.s[u]), (uint64_t)__double_as_longlong(s));
  }
}

constexpr int ROWS = 8;  // beams of a CTA of the warp-per-beam kernel

// Rows of up to 32 * R words: a warp per beam, eight beams to a CTA, a cluster of
// CTAs per sequence.
template <class T, int R>
__global__ void __launch_bounds__(32 * ROWS) beam_select_warps_kernel(
    const T* __restrict__ logits, long long ld, SelectArgs a) {
  rnet_dev::pdl_trigger();
  __shared__ Lists lists;
  __shared__ uint64_t keys[ROWS][WARP_CAP];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int beam = blockIdx.y * ROWS + warp;
  const size_t m0 = (size_t)blockIdx.x * a.W;
  // the first CTA's shared memory may be written once it runs
  const bool many = gridDim.y > 1;
  if (many) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
  Standing now;
  if (blockIdx.y == 0 && warp == 0) now.load(a, m0, 1);
  float m = 0.f;
  double s = 0.0;
  int n = 0;
  if (beam < a.W) {
    const T* z = logits + (m0 + beam) * ld;
    const bool even = even_start(z);
    uint32_t w[R];
#pragma unroll
    for (int j = 0; j < R; ++j) w[j] = load_word(z, lane + 32 * j, a.V, even);
    n = warp_select<T, R>(w, a.W, LOG2E, keys[warp], m, s);
  }
  if (many) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
  if (beam < a.W) deliver(lists, beam, lane, n, keys[warp][lane], m, s);
  if (many) rnet_dev::cluster_sync();
  else __syncthreads();
  if (blockIdx.y == 0) merge(lists, a, m0, 1, now);
}

// Two CTAs of 512 threads to an SM hide each other's latency better than more
// values to a thread (32 x 8 rows of 50001 fp32 in L2: 21.1 us with 256 threads of
// 32 values, 18.1 us so; 21.3 us from HBM).
template <class T>
using BeamSelection = Selection<T, 512, 16>;

// Longer rows: a cluster per sequence. The W * S (beam, slice) parts go round the
// CTAs of the cluster; their lists meet in the first CTA's shared memory.
template <class T>
__global__ void __launch_bounds__(BeamSelection<T>::NT, 2) beam_select_cluster_kernel(
    const T* __restrict__ logits, long long ld, SelectArgs a, int S, int slice) {
  rnet_dev::pdl_trigger();
  __shared__ Lists lists;
  extern __shared__ uint4 cluster_buf[];
  auto& sel = *reinterpret_cast<BeamSelection<T>*>(cluster_buf);
  const int tid = threadIdx.x, rank = blockIdx.y, C = gridDim.y;
  const size_t m0 = (size_t)blockIdx.x * a.W;
  // the first CTA's shared memory may be written once it runs
  if (C > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
  bool waited = C == 1;
  Standing now;
  if (rank == 0 && tid < 32) now.load(a, m0, S);
  uint32_t parity;
  select_setup(sel, parity);
  for (int u = rank; u < a.W * S; u += C) {
    const int beam = u / S, begin = (u % S) * slice, end = min(begin + slice, a.V);
    float m = 0.f;
    double s = 0.0;
    int n = 0;
    if (!(a.finished_in && a.finished_in[m0 + beam]))
      n = cta_select(sel, logits + (m0 + beam) * ld, min(begin, a.V), end, a.W, LOG2E, m, s,
                     parity, a.err);
    if (!waited) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
    waited = true;
    deliver(lists, u, tid, n, tid < n ? sel.key[tid] : 0, m, s);
    __syncthreads();  // sel is free again
  }
  if (C > 1) rnet_dev::cluster_sync();
  if (rank == 0) merge(lists, a, m0, S, now);
}

template <class Kernel, class... Args>
cudaError_t launch_cluster(Kernel kernel, int batch, int C, int threads, size_t smem,
                           cudaStream_t s, Args... args) {
  const ClusterLaunch l(dim3(batch, C), threads, smem, s);
  return cudaLaunchKernelEx(&l.cfg, kernel, args...);
}

template <class T>
cudaError_t select_launch(const T* z, long long ld, const SelectArgs& a, int batch,
                          cudaStream_t s) {
  constexpr int N = Words<T>::N;
  if (a.V <= 2048) {
    const int C = (a.W + ROWS - 1) / ROWS, threads = 32 * (a.W < ROWS ? a.W : ROWS);
    auto kernel = a.V <= 256    ? beam_select_warps_kernel<T, 8 / N>
                  : a.V <= 1024 ? beam_select_warps_kernel<T, 32 / N>
                                : beam_select_warps_kernel<T, 64 / N>;
    return launch_cluster(kernel, batch, C, threads, 0, s, z, ld, a);
  }
  auto kernel = beam_select_cluster_kernel<T>;
  constexpr int smem = sizeof(BeamSelection<T>);
  static std::atomic<uint64_t> ready{0};
  cudaError_t e = allow_smem((const void*)kernel, smem, ready);
  if (e != cudaSuccess) return e;
  static std::atomic<int> known[64];
  int most;
  e = cluster_ctas((const void*)kernel, SELECT_CTAS, BeamSelection<T>::NT, smem, known, most);
  if (e != cudaSuccess) return e;
  // slices of a row where the rows alone leave SMs idle, a chunk or more each
  const int sms = rnet_gemm::num_sms();
  int S = 1;
  while (a.W * (S + 1) <= most && (long long)batch * a.W * (S + 1) <= sms &&
         S * BeamSelection<T>::CHUNK * N < a.V)
    ++S;
  const int slice = (((a.V + S - 1) / S) + 15) & ~15;  // whole 16-byte places
  const int C = a.W * S < most ? a.W * S : most;
  return launch_cluster(kernel, batch, C, BeamSelection<T>::NT, smem, s, z, ld, a, S, slice);
}

// ---------------------------------------------------------------- states
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

// ---------------------------------------------------------------- sequences
// The way back from the last step is a chain of dependent looks at the parents.
// It is cut into segments of steps, and a lane walks a segment for a beam: 32 / P
// segments in a warp (P = beams, rounded up to a power of two), so that a look is
// a shuffle inside P lanes and the loads do not wait for it. Each segment first
// finds where every beam at its end comes from; these maps are chained over the
// segments of a warp, then over the warps, and the segments are walked again from
// the right beams, first for the first eos, then to write. What bounds it is the
// latency of one segment's loads and shuffles, three times.
constexpr int BACK_WARPS = 32;
constexpr int BACK_CTAS = 8;
constexpr int BACK = 8;  // steps whose loads are under way together

struct Segment {
  const int *parents, *tokens;  // of this lane's beam
  size_t M;
  int begin, end;  // steps
  int first;       // lane of the segment's beam 0
  int W;
  bool on;         // this lane has a beam

  // From beam a at step end - 1 to the first step; f(t, tokens) sees the tokens of
  // steps t - 1, .. t - BACK on the way (those below `begin` are not the segment's).
  // Returns the beam before the segment. `steps` is the same in all lanes.
  template <bool TOKENS, class F>
  __device__ __forceinline__ int walk(int steps, int a, bool& bad, F f) const {
    const int own = (threadIdx.x & 31) - first;
    for (int k = 0; k < steps; k += BACK) {
      int p[BACK], v[BACK];
#pragma unroll
      for (int i = 0; i < BACK; ++i) {
        const int t = end - 1 - k - i;
        const bool in = on && t >= begin;
        p[i] = in ? parents[(size_t)t * M] : own;
        if (TOKENS) v[i] = in ? tokens[(size_t)t * M] : 0;
      }
#pragma unroll
      for (int i = 0; i < BACK; ++i) {
        if (on && (p[i] < 0 || p[i] >= W)) p[i] = own, bad = true;
        if (TOKENS) v[i] = __shfl_sync(~0u, v[i], first + a);
        a = __shfl_sync(~0u, p[i], first + a);
      }
      if (TOKENS) f(end - k, v);
    }
    return a;
  }
};

__device__ __forceinline__ void store_int_in(int* p, int rank, int v) {
  asm volatile(
      "{\n\t.reg .b32 ra;\n\t"
      "mapa.shared::cluster.u32 ra, %0, %1;\n\t"
      "st.shared::cluster.u32 [ra], %2;\n\t}" ::"r"(rnet_dev::smem_u32(p)),
      "r"(rank), "r"(v)
      : "memory");
}

// A cluster of CTAs per sequence (one where they have enough segments).
__global__ void __launch_bounds__(32 * BACK_WARPS) beam_backtrack_kernel(
    const int* __restrict__ tokens, const int* __restrict__ parents, const float* scores, int eos,
    float alpha, int* __restrict__ seq, int* __restrict__ lengths, float* ranked, int T, size_t M,
    int W, int P, int steps, unsigned* err) {
  rnet_dev::pdl_trigger();
  __shared__ int map[BACK_WARPS][32], from[BACK_WARPS][32], ends[BACK_WARPS][32];
  __shared__ int cta_map[BACK_CTAS][32], cta_len[BACK_CTAS][32];
  __shared__ int s_start[32], s_len[32], s_rank[32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  const int cta = blockIdx.y, ctas = gridDim.y;
  const int G = 32 / P, beam = lane & (P - 1), part = lane / P;
  const size_t m0 = (size_t)blockIdx.x * W;
  // the peers' shared memory may be written once all of them run
  if (ctas > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
  Segment sg;
  sg.M = M;
  sg.W = W;
  sg.first = lane - beam;
  sg.on = beam < W;
  sg.begin = (int)min((long long)((cta * warps + warp) * G + part) * steps, (long long)T);
  sg.end = min(sg.begin + steps, T);
  sg.parents = parents + m0 + beam;
  sg.tokens = tokens + m0 + beam;
  // read before the first exchange: the ranked scores may take its place
  const float score = sg.on ? scores[m0 + beam] : 0.f;
  bool bad = false;
  const int before = sg.walk<false>(steps, beam, bad, [](int, int*) {});
  if (bad && err) atomicOr(err, rnet_dev::ERR_BAD_INDEX);
  // this segment's start for every beam at the end of the warp's last segment
  int a = beam, start = beam;
  for (int g = G - 1; g >= 0; --g) {
    if (part == g) start = a;
    a = __shfl_sync(~0u, before, g * P + a);
  }
  map[warp][lane] = a;  // the same in all parts
  __syncthreads();
  if (ctas > 1) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
  if (warp == 0) {  // the same over the CTA's warps, for every beam at its end
    int b = beam;
    for (int k = warps - 1; k >= 0; --k) {
      from[k][lane] = b;
      b = map[k][b];
    }
    if (ctas > 1)
      for (int r = 0; r < ctas; ++r) store_int_in(&cta_map[cta][lane], r, b);
  }
  if (ctas > 1) rnet_dev::cluster_sync();
  if (warp == 0) {  // and over the CTAs behind this one
    int b = beam;
    for (int r = ctas - 1; r > cta; --r) b = cta_map[r][b];
    s_start[lane] = b;
  }
  __syncthreads();
  start = __shfl_sync(~0u, start, sg.first + from[warp][s_start[beam]]);
  int len = T;
  if (eos >= 0) {
    sg.walk<true>(steps, start, bad, [&](int t, const int* token) {
#pragma unroll
      for (int i = 0; i < BACK; ++i)
        if (t - 1 - i >= sg.begin && token[i] == eos) len = t - i;
    });
    for (int o = P; o < 32; o <<= 1) len = min(len, __shfl_xor_sync(~0u, len, o));
    ends[warp][lane] = len;
    __syncthreads();
    if (warp == 0) {
      for (int k = 0; k < warps; ++k) len = min(len, ends[k][lane]);
      if (ctas > 1)
        for (int r = 0; r < ctas; ++r) store_int_in(&cta_len[cta][lane], r, len);
    }
    if (ctas > 1) {
      rnet_dev::cluster_sync();
      for (int r = 0; r < ctas; ++r) len = min(len, cta_len[r][lane]);
    }
  }
  if (warp == 0) {
    // 0 and -inf stay what they are: the power may leave 64 bits, and 0 / 0 or inf / inf
    // would be a rank that is neither above nor below the others
    double r = sg.on ? (double)canon(score) : -(double)INFINITY;
    if (r != 0.0 && r != -(double)INFINITY) r /= pow((double)len, (double)alpha);
    int rank = 0;
    for (int i = 0; i < W; ++i) {
      const double o = __shfl_sync(~0u, r, i);
      rank += o > r || (o == r && i < beam);
    }
    s_len[lane] = len;
    s_rank[lane] = rank;
    if (lane < W && cta == 0) {
      lengths[m0 + rank] = len;
      ranked[m0 + rank] = (float)r;
    }
  }
  __syncthreads();
  len = s_len[beam];
  int* out = seq + (m0 + (sg.on ? s_rank[beam] : 0)) * T;
  sg.walk<true>(steps, start, bad, [&](int t, int* token) {
    if (!sg.on) return;
#pragma unroll
    for (int i = 0; i < BACK; ++i)
      if (t - 1 - i >= len) token[i] = eos;
    int* to = out + t - BACK;
    if (t - BACK >= sg.begin && ((uintptr_t)to & 15) == 0) {
      // 32 bytes of one sequence at a time: a sector is written once
#pragma unroll
      for (int i = BACK - 4; i >= 0; i -= 4)
        *reinterpret_cast<int4*>(to + BACK - 4 - i) =
            make_int4(token[i + 3], token[i + 2], token[i + 1], token[i]);
    } else {
#pragma unroll
      for (int i = 0; i < BACK; ++i)
        if (t - 1 - i >= sg.begin) out[t - 1 - i] = token[i];
    }
  });
}

// ---------------------------------------------------------------- a search's records
__global__ void beam_begin_kernel(float* scores, int* finished, int* step, int M, int W) {
  rnet_dev::pdl_trigger();
  const int i = blockIdx.x * blockDim.x + threadIdx.x;
  if (i == 0) *step = 0;
  if (i >= M) return;
  scores[i] = i % W ? -INFINITY : 0.f;
  finished[i] = 0;
}

// One CTA: the row is known to all threads before the first one moves it on.
__global__ void __launch_bounds__(1024) beam_record_kernel(const int* tokens, const int* parents,
                                                           int* hist_tokens, int* hist_parents,
                                                           int M, int* step, int* pos) {
  rnet_dev::pdl_trigger();
  const int row = *step;
  __syncthreads();
  if (threadIdx.x == 0) {
    *step = row + 1;
    if (row) *pos += 1;
  }
  for (int i = threadIdx.x; i < M; i += 1024) {
    hist_tokens[(size_t)row * M + i] = tokens[i];
    hist_parents[(size_t)row * M + i] = parents[i];
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
                        int* finished, int batch, int beams, int V, unsigned* err, cudaStream_t s) {
  if (batch <= 0) return cudaSuccess;
  const SelectArgs a{scores_in, finished_in, eos, scores, tokens, parents, finished, beams, V,
                     err};
  const cudaError_t e = bf16 ? select_launch((const __nv_bfloat16*)logits, ld, a, batch, s)
                             : select_launch((const float*)logits, ld, a, batch, s);
  return e != cudaSuccess ? e : launched();
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

cudaError_t beam_begin(float* scores, int* finished, int* step, int batch, int beams,
                       cudaStream_t s) {
  const int M = batch * beams;
  beam_begin_kernel<<<(M + 255) / 256, 256, 0, s>>>(scores, finished, step, M, beams);
  return launched();
}

cudaError_t beam_record(const int* tokens, const int* parents, int* hist_tokens,
                        int* hist_parents, int M, int* step, int* pos, cudaStream_t s) {
  beam_record_kernel<<<1, 1024, 0, s>>>(tokens, parents, hist_tokens, hist_parents, M, step, pos);
  return launched();
}

cudaError_t beam_backtrack(const int* tokens, const int* parents, const float* scores, int eos,
                           float alpha, int* sequences, int* lengths, float* ranked, int steps,
                           int batch, int beams, unsigned* err, cudaStream_t s) {
  if (batch <= 0) return cudaSuccess;
  int P = 1;
  while (P < beams) P *= 2;
  // segments of at least BACK steps; eight warps of them to a CTA while a cluster of
  // CTAs finds idle SMs (4 sequences of 4096 steps: 7.3 us, 19.4 in one CTA each)
  const int per_warp = 32 / P;
  int warps = (steps + BACK * per_warp - 1) / (BACK * per_warp);
  int ctas = 1;
  while (ctas < BACK_CTAS && warps > 8 * ctas &&
         (long long)batch * 2 * ctas <= rnet_gemm::num_sms())
    ctas *= 2;
  warps = (warps + ctas - 1) / ctas;
  if (warps > BACK_WARPS) warps = BACK_WARPS;
  const int segments = ctas * warps * per_warp;
  int per = (steps + segments - 1) / segments;
  per = (per + BACK - 1) / BACK * BACK;  // whole batches, which start on a multiple of BACK
  const cudaError_t e = launch_cluster(beam_backtrack_kernel, batch, ctas, 32 * warps, 0, s, tokens,
                                       parents, scores, eos, alpha, sequences, lengths, ranked,
                                       steps, (size_t)batch * beams, beams, P, per, err);
  return e != cudaSuccess ? e : launched();
}

}  // namespace rnet_k
