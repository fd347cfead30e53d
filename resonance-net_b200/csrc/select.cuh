// The K largest logits of a row with its sum of exponentials, in one pass over
// the row: by a warp (short rows, held in registers) or by a CTA (streamed
// through shared memory).
//
// Both work from a bound T that at least K logits are known to reach: with the
// largest logit of every thread at hand, the r-th largest of a warp's 32 is
// reached by r logits of that warp. The few logits that reach T are kept as
// distinct 64-bit keys (value, then lower index) and ranked by counting, so the
// result does not depend on the order in which they came. Where more reach T than
// there is room for (ties, sorted rows), the exact K-th key is found bit by bit
// and becomes the bound.
//
// NaN and +inf are not looked for: either makes the sum of exponentials NaN, and
// only then the row is gone through again with every value made finite.
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

// Word w (elements N w, N w + 1) of a row z of `end` elements, -inf beyond.
__device__ __forceinline__ uint32_t load_word(const float* z, int w, int end, bool) {
  return w < end ? __float_as_uint(z[w]) : 0xFF800000u;
}
__device__ __forceinline__ uint32_t load_word(const __nv_bfloat16* z, int w, int end, bool even) {
  const int e = 2 * w;
  if (even && e + 1 < end)  // the row starts on a 4-byte boundary
    return *reinterpret_cast<const uint32_t*>(z + e);
  const unsigned short* p = reinterpret_cast<const unsigned short*>(z);
  const uint32_t lo = e < end ? p[e] : 0xFF80u, hi = e + 1 < end ? p[e + 1] : 0xFF80u;
  return lo | hi << 16;
}
template <class T>
__device__ __forceinline__ bool even_start(const T* z) {
  return ((uintptr_t)z & 3) == 0;
}
// Value i of a word; CLEAN: NaN as -inf, +inf as the largest number.
template <class T, bool CLEAN>
__device__ __forceinline__ float word_value(uint32_t w, int i) {
  float x;
  if constexpr (sizeof(T) == 4) x = __uint_as_float(w);
  else x = __uint_as_float(i ? w & 0xFFFF0000u : w << 16);
  return CLEAN ? fminf(fmaxf(x, -INFINITY), FLT_MAX) : x;
}
// The largest value of R words.
template <class T, int R, bool CLEAN>
__device__ __forceinline__ float words_max(const uint32_t* w) {
  float m;
  if constexpr (sizeof(T) == 4) {
    m = fmaxf(__uint_as_float(w[0]), -INFINITY);
#pragma unroll
    for (int j = 1; j < R; ++j) m = fmaxf(m, __uint_as_float(w[j]));
  } else {
    auto h = [&](int j) { return *reinterpret_cast<const __nv_bfloat162*>(&w[j]); };
    __nv_bfloat162 a = h(0);
#pragma unroll
    for (int j = 1; j < R; ++j) a = __hmax2(a, h(j));
    m = fmaxf(fmaxf(__low2float(a), __high2float(a)), -INFINITY);
  }
  return CLEAN ? fminf(m, FLT_MAX) : m;
}
// Sum of 2^((x - m) c) over R words. m + 0 > -inf.
template <class T, int R, bool CLEAN>
__device__ __forceinline__ float words_sum(const uint32_t* w, float m, float c) {
  float s = 0.f;
#pragma unroll
  for (int j = 0; j < R; ++j)
#pragma unroll
    for (int i = 0; i < Words<T>::N; ++i)
      s += exp2_fast((word_value<T, CLEAN>(w[j], i) - m) * c);
  return s;
}

// A bound that at least r of a warp's values of type T reach, or all that are above
// -FLT_MAX, by r rounds: the r-th largest, in fp32, where equal values are rare, of
// the distinct values.
template <class T>
__device__ __forceinline__ float warp_nth_few(float v, int r) {
  const int lane = threadIdx.x & 31;
  float t = warp_max(v);
  for (int i = 1; i < r; ++i) {
    if (sizeof(T) == 4 ? v == t : lane == __ffs(__ballot_sync(~0u, v == t)) - 1) v = -FLT_MAX;
    t = warp_max(v);
  }
  return t;
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

__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
  return v;
}

// log of the sum of exponentials at tau from the largest logit m and the sum s of
// 2^((x - m) log2(e) / tau); -inf for a row without a logit above -inf.
__device__ __forceinline__ float log_sum(float m, float s, float inv_tau) {
  return s > 0.f ? m * inv_tau + logf(s) : -INFINITY;
}
__device__ __forceinline__ double log_sum(float m, double s) {
  return s > 0.0 ? (double)m + log(s) : -(double)INFINITY;
}

// ---------------------------------------------------------------- a warp
constexpr int WARP_CAP = 128;  // keys kept at most

// The K <= 64 largest of the words of a row, word lane + 32 j in w[j]. key[0 ..
// return value) are sorted; key has WARP_CAP places. m is the row's largest
// logit, s the sum as Sum.
template <class T, int R, bool CLEAN, class Sum>
__device__ __forceinline__ int warp_select_as(const uint32_t* w, int K, float c, uint64_t* key,
                                              float& m, Sum& s) {
  constexpr int N = Words<T>::N;
  const int lane = threadIdx.x & 31;
  auto each = [&](auto f) {
#pragma unroll
    for (int j = 0; j < R; ++j)
#pragma unroll
      for (int i = 0; i < N; ++i) f(word_value<T, CLEAN>(w[j], i), (lane + 32 * j) * N + i);
  };
  const float mine = words_max<T, R, CLEAN>(w);
  m = fmaxf(warp_max(mine), -FLT_MAX);
  s = warp_sum((Sum)words_sum<T, R, CLEAN>(w, m, c));
  if (!CLEAN && s != s) return 0;
  // K logits reach T: the K-th largest of the lanes' maxima, or, where that would be
  // a small one, about the K-th largest of the maxima of the lanes' quarters
  float T_;
  if (K <= 16) {
    T_ = K <= (N == 1 ? 8 : 4) ? warp_nth_few<T>(mine, K) : warp_nth(mine, K);
  } else {
    constexpr int Q = R / 4;
    uint32_t g[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) g[i] = order(words_max<T, Q, CLEAN>(w + i * Q) + 0.0f);
    uint32_t o = 0;
    for (uint32_t b = 1u << 31; b > 1u << 12; b >>= 1) {
      int k = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) k += g[i] >= (o | b);
      k = __reduce_add_sync(~0u, k);
      if (k >= K) o |= b;
      if (k >= K && k <= K + K / 8) break;
    }
    T_ = o > order(-FLT_MAX) ? unorder(o) : -FLT_MAX;
  }
  T_ = fmaxf(T_, -FLT_MAX);  // -inf is no candidate
  int mine_in = 0;
  each([&](float x, int) { mine_in += x >= T_; });
  int at = mine_in;  // keys of the lanes up to this one
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(~0u, at, o);
    if (lane >= o) at += v;
  }
  int n = __shfl_sync(~0u, at, 31);
  at -= mine_in;
  if (n <= WARP_CAP) {
    each([&](float x, int e) {
      if (x >= T_) key[at++] = make_key(x + 0.0f, e);
    });
  } else {
    // the exact K-th largest value, bit by bit, and how many of its equals count
    auto reach = [&](auto f) {
      int k = 0;
      each([&](float x, int e) { k += x > -INFINITY && f(order(x + 0.0f), (uint32_t)e); });
      return __reduce_add_sync(~0u, k);
    };
    uint32_t o = 0, last = ~0u;
    int got = 0;
    for (uint32_t b = 1u << 31; b && got != K; b >>= 1) {
      const int k = reach([&](uint32_t x, uint32_t) { return x >= (o | b); });
      if (k >= K) o |= b, got = k;
    }
    if (got != K) {
      const int above = reach([&](uint32_t x, uint32_t) { return x > o; });
      last = 0;
      for (uint32_t b = 1u << 11; b; b >>= 1)
        if (reach([&](uint32_t x, uint32_t e) { return x == o && e < (last | b); }) < K - above)
          last |= b;
    }
    n = 0;
    each([&](float x, int e) {
      const uint32_t v = order(x + 0.0f);
      const bool in = x > -INFINITY && (v > o || (v == o && (uint32_t)e <= last));
      const uint32_t mask = __ballot_sync(~0u, in);
      if (in) key[n + __popc(mask & ((1u << lane) - 1))] = make_key(x + 0.0f, e);
      n += __popc(mask);
    });
  }
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
template <class T, int R, class Sum>
__device__ __forceinline__ int warp_select(const uint32_t* w, int K, float c, uint64_t* key,
                                           float& m, Sum& s) {
  const int n = warp_select_as<T, R, false>(w, K, c, key, m, s);
  return s == s ? n : warp_select_as<T, R, true>(w, K, c, key, m, s);
}

// ---------------------------------------------------------------- a CTA
constexpr int SEL_GROUP = 4;    // words that are kept together
constexpr int SEL_STAGES = 2;   // chunks in shared memory
constexpr int SEL_QUEUE = 512;  // groups kept at most
constexpr int SEL_CAP = 512;    // keys kept at most

// The shared memory of a CTA of NT threads that take VALUES values each of one
// chunk.
template <class T, int NT_, int VALUES>
struct alignas(16) Selection {
  using Type = T;
  static constexpr int NT = NT_, WARPS = NT / 32;
  static constexpr int N = Words<T>::N;
  static constexpr int R = VALUES / N;   // words of a thread in one chunk
  static constexpr int CHUNK = NT * R;   // words
  uint32_t ring[SEL_STAGES][CHUNK + 4];
  uint32_t group[SEL_GROUP][SEL_QUEUE];
  int group_word[SEL_QUEUE];  // the group's first word
  uint64_t key[SEL_CAP];
  double s[WARPS];
  float bound[2][WARPS], m[WARPS];
  uint64_t bar[SEL_STAGES];
  int keys, groups, abort[2];
};

// Once per CTA, before the first selection; parity belongs to the barriers.
template <class Sel>
__device__ __forceinline__ void select_setup(Sel& sel, uint32_t& parity) {
  parity = 0;
  if (threadIdx.x == 0) {
    sel.abort[0] = sel.abort[1] = 0;
    for (int i = 0; i < SEL_STAGES; ++i) rnet_dev::mbar_init(&sel.bar[i], 1);
    rnet_dev::fence_barrier_init();
  }
}

// Leaves the K largest of the n <= SEL_CAP keys, or those of them that `keep`
// accepts, in any order, and returns a bound that exactly K of all n reach (0 if
// there are no more than K). All threads; a barrier lies between the last key and the
// call.
template <class Sel, class Keep>
__device__ __forceinline__ uint64_t shrink(Sel& sel, int n, int K, Keep keep) {
  constexpr int NT = Sel::NT, J = (SEL_CAP + NT - 1) / NT;
  uint64_t k[J];
#pragma unroll
  for (int j = 0; j < J; ++j) {
    const int i = threadIdx.x + j * NT;
    k[j] = i < n ? sel.key[i] : 0;
  }
  uint64_t t = 0;
  if (n > K)
    for (int b = 63; b >= 0; --b) {
      const uint64_t u = t | 1ull << b;
      int reach = 0;
#pragma unroll
      for (int j = 0; j < J; ++j)
        if (j * NT < n) reach += __syncthreads_count(k[j] >= u);
      if (reach >= K) t = u;
      if (reach == K) break;
    }
  __syncthreads();
  if (threadIdx.x == 0) sel.keys = 0;
  __syncthreads();
#pragma unroll
  for (int j = 0; j < J; ++j)
    if (k[j] && k[j] >= t && keep(k[j])) sel.key[atomicAdd(&sel.keys, 1)] = k[j];
  __syncthreads();
  return t;
}

// Turns the n queued groups into keys that reach the bound. All threads; a barrier
// lies between the last group or key and the call. Where they are more than there is
// room for, the bound is raised to the K-th of those at hand and the groups are gone
// through again; the keys of earlier groups (elements before `first`) stay. They are at
// most K, so that SEL_CAP - K > K keys of these groups are at hand and the bound rises.
template <bool CLEAN, class Sel>
__device__ __forceinline__ void drain(Sel& sel, int n, int K, int first, uint64_t& bound,
                                      unsigned* err) {
  using T = typename Sel::Type;
  constexpr int N = Sel::N, NT = Sel::NT;
  constexpr int EACH = NT < 512 ? SEL_GROUP : 1;  // words of a thread: few threads take a group
  for (bool again = true; again;) {
    for (int i = threadIdx.x; i < n * (SEL_GROUP / EACH); i += NT) {
      const int g = i / (SEL_GROUP / EACH), part = i % (SEL_GROUP / EACH) * EACH;
      const int word = sel.group_word[g];
#pragma unroll
      for (int j = part; j < part + EACH; ++j)
#pragma unroll
        for (int h = 0; h < N; ++h) {
          const float x = word_value<T, CLEAN>(sel.group[j][g], h);
          if (!(x > -INFINITY)) continue;
          const uint64_t k = make_key(x + 0.0f, (word + j * NT) * N + h);
          if (k < bound) continue;
          const int at = atomicAdd(&sel.keys, 1);
          if (at < SEL_CAP) sel.key[at] = k;
        }
    }
    __syncthreads();
    const int got = sel.keys;
    again = got > SEL_CAP;
    if (again) {
      const uint64_t t = shrink(sel, SEL_CAP, K, [&](uint64_t k) {
        return key_index(k) < first;
      });
      if (t <= bound) {  // no round may follow that finds the same keys
        again = false;
        if (threadIdx.x == 0 && err) atomicOr(err, rnet_dev::ERR_NO_PROGRESS);
      } else {
        bound = t;
      }
    }
  }
}

// The K <= 64 largest of the elements [begin, end) of the row z (begin on a
// 16-byte place of the row, and a multiple of 2). sel.key[0 .. return value) are
// sorted. m is the slice's largest logit, s the sum. All threads; sel
// is set up and not in use.
template <bool CLEAN, class Sel, class T>
__device__ __forceinline__ int cta_select_as(Sel& sel, const T* z, int begin, int end, int K,
                                             float c, float& m, double& s, uint32_t& parity,
                                             unsigned* err) {
  constexpr int N = Sel::N, R = Sel::R, CHUNK = Sel::CHUNK, NT = Sel::NT, WARPS = Sel::WARPS;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const bool even = even_start(z);
  const int total = begin < end ? (end - begin + N - 1) / N : 0;  // words
  const int chunks = (total + CHUNK - 1) / CHUNK;
  const T* zb = z + begin;
  const uint32_t skew = (uint32_t)((uintptr_t)zb & 15);  // of every chunk's first byte
  // A chunk comes through shared memory if the 16-byte pieces that cover it lie
  // inside the slice; the first one of an unaligned row and the last do not.
  auto staged = [&](int i) {
    return (i > 0 || skew == 0) && (i + 1) * CHUNK * N + (skew ? 16 / (int)sizeof(T) : 0) <=
                                       end - begin;
  };
  auto fetch = [&](int i) {  // one thread
    const uint32_t bytes = CHUNK * 4 + (skew ? 16 : 0);
    uint64_t* bar = &sel.bar[i % SEL_STAGES];
    rnet_dev::mbar_arrive_expect_tx(bar, bytes);
    bulk_load(sel.ring[i % SEL_STAGES],
              reinterpret_cast<const char*>(zb + (size_t)i * CHUNK * N) - skew, bytes, bar);
  };
  if (tid == 0) {
    sel.keys = sel.groups = 0;
    for (int i = 0; i < SEL_STAGES && i < chunks; ++i)
      if (staged(i)) fetch(i);
  }
  __syncthreads();
  uint64_t bound = 0;
  float lowest = -FLT_MAX;  // its value
  bool exact = false;       // the bound is a key of the row, not a value alone
  float sum = 0.f;
  int epoch = begin;        // the queue's elements lie behind this one
  m = -FLT_MAX;
  for (int i = 0; i < chunks; ++i) {
    const int w0 = begin / N + i * CHUNK;  // the row's first word of the chunk
    uint32_t w[R];
    if (staged(i)) {
      const int b = i % SEL_STAGES;
      // a copy that does not come is reported and given the same time once more:
      // none may land in memory that the CTA has left
      if (!rnet_dev::mbar_wait(&sel.bar[b], parity >> b & 1, err, &sel.abort[0]))
        rnet_dev::mbar_wait(&sel.bar[b], parity >> b & 1, err, &sel.abort[1]);
      parity ^= 1u << b;
      const char* p = reinterpret_cast<const char*>(sel.ring[b]) + skew + 4 * tid;
      if (even) {
#pragma unroll
        for (int j = 0; j < R; ++j)
          w[j] = *reinterpret_cast<const uint32_t*>(p + 4 * NT * j);
      } else {
#pragma unroll
        for (int j = 0; j < R; ++j) {
          const unsigned short* q =
              reinterpret_cast<const unsigned short*>(p + 4 * NT * j);
          w[j] = q[0] | (uint32_t)q[1] << 16;
        }
      }
    } else {
#pragma unroll
      for (int j = 0; j < R; ++j)
        w[j] = load_word(z, w0 + j * NT + tid, end, even);
    }
    float top[R / SEL_GROUP];
    float mine = -INFINITY;
#pragma unroll
    for (int g = 0; g < R / SEL_GROUP; ++g) {
      top[g] = words_max<T, SEL_GROUP, CLEAN>(w + g * SEL_GROUP);
      mine = fmaxf(mine, top[g]);
    }
    const float mx = fmaxf(m, mine);
    sum = sum * exp2_fast((m - mx) * c) + words_sum<T, R, CLEAN>(w, mx, c);
    m = mx;
    if (i < 2 || (i & (i - 1)) == 0) {
      // K logits reach the K-th largest of the warps' maxima so far, or the least of
      // their r-th largest thread maxima
      const float v = K <= WARPS ? warp_max(m) : warp_nth(m, (K + WARPS - 1) / WARPS);
      if (lane == 0) sel.bound[i & 1][warp] = v;
      __syncthreads();
      float least;
      if (WARPS >= 8 && K <= 8) {
        least = warp_nth_few<T>(lane < WARPS ? sel.bound[i & 1][lane] : -FLT_MAX, K);
      } else {
        least = sel.bound[i & 1][0];
#pragma unroll
        for (int j = 1; j < WARPS; ++j) least = fminf(least, sel.bound[i & 1][j]);
      }
      const uint64_t t = (uint64_t)order(least + 0.0f) << 32;
      if (t > bound) {
        bound = t;
        lowest = least;
        exact = false;
      }
    }
    // where the bound is a key, a group whose largest logit equals its value
    // is looked at key by key (the volatile move keeps the compiler from forming all
    // the keys ahead of time)
    auto reaches = [&](int g) {
      bool in = false;
#pragma unroll
      for (int j = 0; j < SEL_GROUP; ++j) {
        uint32_t v;
        asm volatile("mov.b32 %0, %1;" : "=r"(v) : "r"(w[g * SEL_GROUP + j]));
#pragma unroll
        for (int h = 0; h < N; ++h) {
          const float x = word_value<T, CLEAN>(v, h);
          // a NaN gives no key, here as in drain(): it must not bring its group back
          in |= x > -INFINITY &&
                make_key(x + 0.0f, (w0 + (g * SEL_GROUP + j) * NT + tid) * N + h) >= bound;
        }
      }
      return in;
    };
    bool full;
    auto queue = [&](auto wanted) {
#pragma unroll
      for (int g = 0; g < R / SEL_GROUP; ++g)
        if (top[g] >= lowest && wanted(g)) {
          const int at = atomicAdd(&sel.groups, 1);
          full |= at >= SEL_QUEUE - SEL_QUEUE / 4;
          if (at < SEL_QUEUE) {
            sel.group_word[at] = w0 + g * SEL_GROUP * NT + tid;
#pragma unroll
            for (int j = 0; j < SEL_GROUP; ++j) sel.group[j][at] = w[g * SEL_GROUP + j];
          }
        }
    };
    // Ends: a group is queued for a key that reaches the bound, so where more are
    // queued than there is room for, SEL_QUEUE > K keys are at hand, the bound rises to the
    // K-th, and at most K of those groups come again.
    for (bool again = true; again;) {
      full = false;
      if (!exact) queue([](int) { return true; });
      else queue([&](int g) { return top[g] > lowest || reaches(g); });
      again = false;
      if (__syncthreads_or(full)) {
        const int n = sel.groups;
        const uint64_t before = bound;
        __syncthreads();
        again = n > SEL_QUEUE;  // then this chunk's groups come again
        drain<CLEAN>(sel, min(n, SEL_QUEUE), K, epoch, bound, err);
        const int got = sel.keys, here = w0 * N;
        const uint64_t t = shrink(sel, got, K, [&](uint64_t k) {
          return !again || key_index(k) < here;
        });
        bound = t > bound ? t : bound;
        if (again && bound <= before) {
          again = false;
          if (tid == 0 && err) atomicOr(err, rnet_dev::ERR_NO_PROGRESS);
        }
        lowest = key_value(bound);
        exact = true;
        if (tid == 0) sel.groups = 0;
        epoch = again ? here : here + CHUNK * N;
        __syncthreads();
      }
    }
    // the chunk's place is free
    if (tid == 0 && i + SEL_STAGES < chunks && staged(i + SEL_STAGES)) fetch(i + SEL_STAGES);
  }
  drain<CLEAN>(sel, sel.groups, K, epoch, bound, err);  // complete since the loop's last barrier
  int n = sel.keys;
  if (n > NT) {
    shrink(sel, n, K, [](uint64_t) { return true; });
    n = sel.keys;
  }
  const uint64_t own = tid < n ? sel.key[tid] : 0;
  int place = 0;
  if (tid < ((n + 31) & ~31))
    for (int k = 0; k < n; ++k) place += sel.key[k] > own;
  const float mw = warp_max(m);
  if (lane == 0) sel.m[warp] = mw;
  __syncthreads();
  if (tid < n && place < K) sel.key[place] = own;
  const float mine = m;
  m = sel.m[0];
#pragma unroll
  for (int i = 1; i < WARPS; ++i) m = fmaxf(m, sel.m[i]);
  const double part = warp_sum((double)(sum * exp2_fast((mine - m) * c)));
  if (lane == 0) sel.s[warp] = part;
  __syncthreads();
  s = 0.0;
#pragma unroll
  for (int i = 0; i < WARPS; ++i) s += sel.s[i];
  return min(n, K);
}
template <class Sel, class T>
__device__ __forceinline__ int cta_select(Sel& sel, const T* z, int begin, int end, int K,
                                          float c, float& m, double& s, uint32_t& parity,
                                          unsigned* err) {
  int n = cta_select_as<false>(sel, z, begin, end, K, c, m, s, parity, err);
  if (s != s) {
    __syncthreads();
    n = cta_select_as<true>(sel, z, begin, end, K, c, m, s, parity, err);
  }
  return n;
}

}  // namespace rnet_logits
