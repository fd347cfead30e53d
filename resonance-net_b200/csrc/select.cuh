// The K largest logits of a row with its sum of exponentials, in one pass over
// the row: by a warp (short rows, held in registers) or by a CTA (streamed).
//
// Both work from a bound T that at least K logits are known to reach: with the
// largest logit of every thread at hand, the r-th largest of a warp's 32 is
// reached by r logits of that warp. The few logits that reach T are kept as
// distinct 64-bit keys (value, then lower index) in shared memory and ranked by
// counting, so the result does not depend on the order in which they came. Where
// more reach T than there is room for (ties, sorted rows), the exact K-th key is
// found bit by bit and becomes the bound.
//
// Element e of a row goes to the same thread whatever the row's alignment: equal
// rows give the same bits, so that equal candidates of a beam search tie.
#pragma once
#include "logits.cuh"

namespace rnet_logits {

// 32-bit words of logits: one fp32 value, or two neighbouring bf16 values.
template <class T>
struct Words {
  static constexpr int N = 4 / sizeof(T);
};

// Word w (elements N w, N w + 1) of the row z of elements below end; -inf beyond.
// NaN reads as -inf.
__device__ __forceinline__ uint32_t load_word(const float* z, int w, int end, bool) {
  return __float_as_uint(fmaxf(w < end ? z[w] : -INFINITY, -INFINITY));
}
__device__ __forceinline__ uint32_t load_word(const __nv_bfloat16* z, int w, int end, bool even) {
  const int e = 2 * w;
  uint32_t u = 0xFF80FF80u;
  if (even && e + 1 < end) {  // the row starts on a 4-byte boundary
    u = *reinterpret_cast<const uint32_t*>(z + e);
  } else {
    const unsigned short* p = reinterpret_cast<const unsigned short*>(z);
    if (e < end) u = 0xFF800000u | p[e];
    if (e + 1 < end) u = (u & 0xFFFFu) | (uint32_t)p[e + 1] << 16;
  }
  const uint32_t none = 0xFF80FF80u;
  const __nv_bfloat162 h = __hmax2(*reinterpret_cast<const __nv_bfloat162*>(&u),
                                   *reinterpret_cast<const __nv_bfloat162*>(&none));
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <class T>
__device__ __forceinline__ bool even_start(const T* z) {
  return ((uintptr_t)z & 3) == 0;
}
// Value i of a word; +inf as the largest number.
template <class T>
__device__ __forceinline__ float word_value(uint32_t w, int i) {
  if constexpr (sizeof(T) == 4) return fminf(__uint_as_float(w), FLT_MAX);
  else return fminf(__uint_as_float(i ? w & 0xFFFF0000u : w << 16), FLT_MAX);
}
// The largest value of R words.
template <class T, int R>
__device__ __forceinline__ float words_max(const uint32_t* w) {
  if constexpr (sizeof(T) == 4) {
    float m = __uint_as_float(w[0]);
#pragma unroll
    for (int j = 1; j < R; ++j) m = fmaxf(m, __uint_as_float(w[j]));
    return fminf(m, FLT_MAX);
  } else {
    auto h = [&](int j) { return *reinterpret_cast<const __nv_bfloat162*>(&w[j]); };
    __nv_bfloat162 m = h(0);
#pragma unroll
    for (int j = 1; j < R; ++j) m = __hmax2(m, h(j));
    return fminf(fmaxf(__low2float(m), __high2float(m)), FLT_MAX);
  }
}

// The r-th largest (r = 1..32) of a warp's 32 values.
__device__ __forceinline__ float warp_nth(float v, int r) {
  const int lane = threadIdx.x & 31;
  // bitonic sort, largest first
#pragma unroll
  for (int k = 2; k <= 32; k <<= 1)
#pragma unroll
    for (int j = k >> 1; j; j >>= 1) {
      const float o = __shfl_xor_sync(~0u, v, j);
      const bool first = (lane & j) == 0, down = (lane & k) == 0;
      v = first == down ? fmaxf(v, o) : fminf(v, o);
    }
  return __shfl_sync(~0u, v, r - 1);
}

__device__ __forceinline__ double warp_sum_d(double v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
  return v;
}

// log of the sum of exponentials at c = log2(e) / tau from the largest logit m
// and the sum s of 2^((x - m) c); -inf for a row without a logit above -inf.
__device__ __forceinline__ double log_sum(float m, double s, float inv_tau) {
  return s > 0.0 ? (double)m * (double)inv_tau + log(s) : -(double)INFINITY;
}

// ---------------------------------------------------------------- a warp
constexpr int WARP_CAP = 128;  // keys kept at most

// The K <= 64 largest of the words of a row of V elements, word lane + 32 j in
// w[j]. key[0 .. return value) are sorted; key has WARP_CAP places. m and s as
// for log_sum.
template <class T, int R>
__device__ __forceinline__ int warp_select(const uint32_t* w, int K, float c, uint64_t* key,
                                           float& m, double& s) {
  constexpr int N = Words<T>::N;
  const int lane = threadIdx.x & 31;
  auto each = [&](auto f) {
#pragma unroll
    for (int j = 0; j < R; ++j)
#pragma unroll
      for (int i = 0; i < N; ++i) f(word_value<T>(w[j], i), (lane + 32 * j) * N + i);
  };
  const float mine = words_max<T, R>(w);
  m = fmaxf(warp_max(mine), -FLT_MAX);
  float sum = 0.f;
  each([&](float x, int) { sum += exp2_fast((x - m) * c); });
  s = warp_sum_d(sum);
  // K logits reach T: from K lanes, or two each from K / 2 lanes
  float T_;
  if (K <= 32 || R == 1) {
    T_ = K <= 32 ? warp_nth(mine, K) : -INFINITY;
  } else {
    constexpr int H = (R + 1) / 2;
    T_ = warp_nth(fminf(words_max<T, H>(w), words_max<T, R - H ? R - H : 1>(w + H % R)),
                  (K + 1) / 2);
  }
  int count = 0;
  each([&](float x, int) { count += x >= T_ && x > -INFINITY; });
  uint32_t last = ~0u;  // of the logits equal to T, those up to this index
  if (__reduce_add_sync(~0u, count) > WARP_CAP) {
    // the exact K-th largest value, bit by bit, and how many of its equals count
    auto reach = [&](auto f) {
      int n = 0;
      each([&](float x, int e) { n += x > -INFINITY && f(order(x + 0.0f), (uint32_t)e); });
      return __reduce_add_sync(~0u, n);
    };
    uint32_t o = 0;
    for (uint32_t b = 1u << 31; b; b >>= 1)
      if (reach([&](uint32_t x, uint32_t) { return x >= (o | b); }) >= K) o |= b;
    const int above = reach([&](uint32_t x, uint32_t) { return x > o; });
    last = 0;
    for (uint32_t b = 1u << 10; b; b >>= 1)
      if (reach([&](uint32_t x, uint32_t e) { return x == o && e < (last | b); }) < K - above)
        last |= b;
    T_ = unorder(o);
  }
  // keys of the logits that reach the bound
  int n = 0;
  each([&](float x, int e) {
    const bool in = x > -INFINITY && (x > T_ || (x == T_ && (uint32_t)e <= last));
    const uint32_t mask = __ballot_sync(~0u, in);
    if (mask) {
      if (in) key[n + __popc(mask & ((1u << lane) - 1))] = make_key(x + 0.0f, e);
      n += __popc(mask);
    }
  });
  __syncwarp();
  // each key's place is the number of larger ones
  uint64_t own[WARP_CAP / 32];
  int place[WARP_CAP / 32];
#pragma unroll
  for (int j = 0; j < WARP_CAP / 32; ++j) {
    place[j] = 0;
    own[j] = 0;
    if (32 * j >= n) break;
    own[j] = lane + 32 * j < n ? key[lane + 32 * j] : 0;
    for (int k = 0; k < n; ++k) place[j] += key[k] > own[j];
  }
  __syncwarp();
#pragma unroll
  for (int j = 0; j < WARP_CAP / 32; ++j)
    if (lane + 32 * j < n && place[j] < K) key[place[j]] = own[j];
  __syncwarp();
  return min(n, K);
}

// ---------------------------------------------------------------- a CTA
constexpr int SEL_THREADS = 256;
constexpr int SEL_WARPS = SEL_THREADS / 32;
constexpr int SEL_R = 16;     // words of a thread at a time
constexpr int SEL_CAP = 1024; // keys kept at most

struct Selection {
  uint64_t key[SEL_CAP];
  float bound[SEL_WARPS], m[SEL_WARPS];
  double s[SEL_WARPS];
  int count;
};

// Leaves the K largest of the n <= SEL_CAP keys that `keep` accepts, in any
// order, and returns a bound that exactly they reach (0 if there are no more
// than K). All threads.
template <class Keep>
__device__ __forceinline__ uint64_t shrink(Selection& sel, int n, int K, Keep keep) {
  constexpr int J = SEL_CAP / SEL_THREADS;
  uint64_t k[J];
#pragma unroll
  for (int j = 0; j < J; ++j) {
    const int i = threadIdx.x + j * SEL_THREADS;
    k[j] = i < n ? sel.key[i] : 0;
  }
  uint64_t t = 0;
  if (n > K)
    for (int b = 63; b >= 0; --b) {
      const uint64_t u = t | 1ull << b;
      int reach = 0;
#pragma unroll
      for (int j = 0; j < J; ++j)
        if (j * SEL_THREADS < n) reach += __syncthreads_count(k[j] >= u);
      if (reach >= K) t = u;
      if (reach == K) break;
    }
  __syncthreads();
  if (threadIdx.x == 0) sel.count = 0;
  __syncthreads();
#pragma unroll
  for (int j = 0; j < J; ++j)
    if (k[j] && k[j] >= t && keep(k[j])) sel.key[atomicAdd(&sel.count, 1)] = k[j];
  __syncthreads();
  return t;
}

// The K <= 64 largest of the elements [begin, end) of the row z (begin even).
// sel.key[0 .. return value) are sorted. m and s as for log_sum. All
// SEL_THREADS threads.
template <class T>
__device__ __forceinline__ int cta_select(Selection& sel, const T* z, int begin, int end, int K,
                                          float c, float& m, double& s) {
  constexpr int N = Words<T>::N, STEP = SEL_THREADS * SEL_R;  // words a pass
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const bool even = even_start(z);
  if (tid == 0) sel.count = 0;
  uint64_t bound = 0;
  float lowest = -INFINITY;  // its value
  float sum = 0.f;
  m = -FLT_MAX;
  uint32_t w[SEL_R];
  auto load = [&](int w0) {
#pragma unroll
    for (int j = 0; j < SEL_R; ++j)
      w[j] = load_word(z, w0 + j * SEL_THREADS + tid, end, even);
  };
  const int w1 = begin < end ? (end + N - 1) / N : 0;
  for (int w0 = begin / N; w0 < w1; w0 += STEP) {
    load(w0);
    const float mine = words_max<T, SEL_R>(w), mx = fmaxf(m, mine);
    sum *= exp2_fast((m - mx) * c);
    m = mx;
#pragma unroll
    for (int j = 0; j < SEL_R; ++j)
#pragma unroll
      for (int i = 0; i < N; ++i) sum += exp2_fast((word_value<T>(w[j], i) - m) * c);
    if (w0 == begin / N) {
      // K logits reach the least of the warps' r-th largest thread maxima
      const float v = warp_nth(mine, (K + SEL_WARPS - 1) / SEL_WARPS);
      if (lane == 0) sel.bound[warp] = v;
      __syncthreads();
      lowest = sel.bound[0];
#pragma unroll
      for (int i = 1; i < SEL_WARPS; ++i) lowest = fminf(lowest, sel.bound[i]);
      bound = (uint64_t)order(lowest + 0.0f) << 32;
    }
    for (bool again = true; again;) {
      bool full = false;
      if (mine >= lowest && mine > -INFINITY) {
#pragma unroll
        for (int j = 0; j < SEL_R; ++j)
#pragma unroll
          for (int i = 0; i < N; ++i) {
            const float x = word_value<T>(w[j], i);
            if (x < lowest || x == -INFINITY) continue;
            const uint64_t k = make_key(x + 0.0f, (w0 + j * SEL_THREADS + tid) * N + i);
            if (k < bound) continue;
            const int at = atomicAdd(&sel.count, 1);
            if (at < SEL_CAP) sel.key[at] = k;
            full |= at >= SEL_CAP / 2;
          }
      }
      again = false;
      if (__syncthreads_or(full)) {
        const int n = sel.count;
        __syncthreads();
        // beyond the room: this pass's keys are dropped and come again
        again = n > SEL_CAP;
        const uint32_t first = w0 * N;
        bound = shrink(sel, min(n, SEL_CAP), K, [&](uint64_t k) {
          return !again || (uint32_t)key_index(k) < first;
        });
        if (bound) lowest = key_value(bound);
      }
    }
  }
  __syncthreads();
  int n = sel.count;
  if (n > SEL_THREADS) {
    shrink(sel, n, K, [](uint64_t) { return true; });
    n = sel.count;
  }
  const uint64_t own = tid < n ? sel.key[tid] : 0;
  int place = 0;
  for (int k = 0; k < n; ++k) place += sel.key[k] > own;
  const float mw = warp_max(m);
  if (lane == 0) sel.m[warp] = mw;
  __syncthreads();
  if (tid < n && place < K) sel.key[place] = own;
  const float mine = m;
  m = sel.m[0];
#pragma unroll
  for (int i = 1; i < SEL_WARPS; ++i) m = fmaxf(m, sel.m[i]);
  const double part = warp_sum_d((double)(sum * exp2_fast((mine - m) * c)));
  if (lane == 0) sel.s[warp] = part;
  __syncthreads();
  s = 0.0;
#pragma unroll
  for (int i = 0; i < SEL_WARPS; ++i) s += sel.s[i];
  return min(n, K);
}

}  // namespace rnet_logits
