// The next token of each row of logits, from given Gumbel noise g:
//   t = x / temperature;  order: t descending, equal values by index
//   kept: the first top_k of the order; of those the shortest prefix whose mass
//         (softmax over them) reaches top_p; of those exp(t - max) >= min_p;
//         the first token always, a logit of -inf never
//   token = argmax over the kept of t + g (equal scores: the lowest index),
//   logprob = t[token] - logsumexp(t) over the whole row.
// temperature <= 0 (or below the smallest normal number) is greedy: the first token
// of the order, logprob at temperature 1; above the largest number it counts as that.
// A t below the smallest normal number is 0. NaN logits count as -inf; a row without a
// finite or +inf logit (or whose t are all -inf) gives token -1 and logprob -inf.
//
// Drawing by the maximum of t + g needs no sorted order: whether a token is kept
// is a question about the tokens before it, answered by one sum. So the winner
// among all candidates is taken first and then checked; a token that is not kept
// rules out everything after it too, and the next winner is looked for among what
// is left. With top_p = 0.9 nine of ten first winners stand. The candidates are
// narrowed first by bounds that cost little: min_p; top_p by the mass a token must
// have if V of its like are to count; top_k by a histogram of each thread's own
// largest logits, whose k-th is a lower bound of the row's k-th. What top_k leaves
// is a list; up to 256 entries are ranked against each other at once, which answers
// everything in one round. Only candidates' noise is read.
//
// One CTA per row; the row is read once and stays in shared memory as fp32 (longer
// rows are read again from L2 in each pass). t is divided out only for candidates;
// the passes over the whole row work on x, of which t is a monotone function. Bound
// by one SM's load rate, its passes over shared memory and the barriers between
// them, not by HBM. Masses are summed as integers of 2^-31 of the largest, so every
// sum and with it every choice is independent of the order of the additions;
// logsumexp is an fp32 sum in a fixed order.
//
// One row of 50257 in bf16, top-k 40 and top-p: 14 us, of which about 3 the load, 2
// the exponentials of the row, 3 the list, 1.5 its ranking and the rest some 20
// barriers of 1024 threads; 128 fp32 rows with settings of their own 53 us, the time
// of the slowest row (top-p alone over a flat distribution).
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include "common.h"

namespace dst {
namespace sampling {

constexpr int kThreads = 1024;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxCached = 52224;  // a row in shared memory (204 KB)
constexpr int kList = 2048;        // candidates kept as a list
constexpr int kRanked = 256;       // of a list ranked pair by pair
constexpr int kBins = 256;

struct Args {
  const void* logits;
  int64_t row_stride;
  const float* gumbel;
  int64_t gumbel_stride;
  int64_t* token;
  float* logprob;
  int V;
  // one value for all rows, or one per row where the pointer is set
  float temperature, top_p, min_p;
  int64_t top_k;
  const float *temperature_rows, *top_p_rows, *min_p_rows;
  const int64_t* top_k_rows;
};

// Keys in the order of the floats they come from.
__device__ __forceinline__ uint32_t key_of(float t) {
  const uint32_t u = __float_as_uint(t);
  return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}

constexpr float kMost = 3.402823466e38f;    // the largest finite number
constexpr float kLeast = 1.175494351e-38f;  // the smallest normal number

constexpr uint32_t kLowestKey = 0x007fffffu;  // of -inf; below it are the keys of NaN

struct Best {  // larger score first, then lower index
  float score;
  int index;
};

__device__ __forceinline__ Best better(Best a, Best b) {
  return (b.score > a.score || (b.score == a.score && b.index < a.index)) ? b : a;
}

struct Scratch {
  Best best[kWarps];
  float f[kWarps];
  unsigned long long u[kWarps];
  uint32_t hist[kBins];
  uint32_t pick[4];
  uint32_t weights[kRanked];
  int list_n;
  int list[kList];
  float list_t[kList];
};

__device__ __forceinline__ Best block_best(Best v, Scratch& s) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    Best w;
    w.score = __shfl_xor_sync(0xffffffff, v.score, o);
    w.index = __shfl_xor_sync(0xffffffff, v.index, o);
    v = better(v, w);
  }
  __syncthreads();
  if ((threadIdx.x & 31) == 0) s.best[threadIdx.x >> 5] = v;
  __syncthreads();
  v = s.best[threadIdx.x & 31];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    Best w;
    w.score = __shfl_xor_sync(0xffffffff, v.score, o);
    w.index = __shfl_xor_sync(0xffffffff, v.index, o);
    v = better(v, w);
  }
  return v;
}

__device__ __forceinline__ float block_max(float v, Scratch& s) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffff, v, o));
  __syncthreads();
  if ((threadIdx.x & 31) == 0) s.f[threadIdx.x >> 5] = v;
  __syncthreads();
  v = s.f[threadIdx.x & 31];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffff, v, o));
  return v;
}

__device__ __forceinline__ float block_min(float v, Scratch& s) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fminf(v, __shfl_xor_sync(0xffffffff, v, o));
  __syncthreads();
  if ((threadIdx.x & 31) == 0) s.f[threadIdx.x >> 5] = v;
  __syncthreads();
  v = s.f[threadIdx.x & 31];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fminf(v, __shfl_xor_sync(0xffffffff, v, o));
  return v;
}

__device__ __forceinline__ float block_sum(float v, Scratch& s) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffff, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) s.f[threadIdx.x >> 5] = v;
  __syncthreads();
  v = s.f[threadIdx.x & 31];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffff, v, o);
  return v;
}

__device__ __forceinline__ unsigned long long block_sum(unsigned long long v, Scratch& s) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffff, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) s.u[threadIdx.x >> 5] = v;
  __syncthreads();
  v = s.u[threadIdx.x & 31];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffff, v, o);
  return v;
}

// exp(t - max) with max itself (also +inf) giving 1.
__device__ __forceinline__ float mass_of(float t, float max) {
  return t == max ? 1.f : exp2f((t - max) * 1.4426950408889634f);
}

__device__ __forceinline__ unsigned long long weight(float mass) {
  return __float2uint_rn(mass * 2147483648.f);
}

template <typename T>
__device__ __forceinline__ float to_float(T x);
template <>
__device__ __forceinline__ float to_float(float x) {
  return x;
}
template <>
__device__ __forceinline__ float to_float(__nv_bfloat16 x) {
  return __bfloat162float(x);
}

// The row: x by index (NaN as -inf, one zero: keys order -0 below +0), and t. In
// shared memory x starts `pad` floats in, so that the global row's 16-byte vectors
// land on 16-byte boundaries; what is left of the first and last four is -inf.
template <typename T, bool CACHED>
struct Row {
  const T* x;
  float* cache;
  float temperature;
  int V, head, pad;
  __device__ __forceinline__ Row(const T* x_, float* cache_, float temperature_, int V_)
      : x(x_), cache(cache_), temperature(temperature_), V(V_) {
    head = min(V, static_cast<int>((16 - (reinterpret_cast<uintptr_t>(x) & 15)) % 16 / sizeof(T)));
    pad = (4 - head % 4) % 4;
  }
  static __device__ __forceinline__ float clean(T v) {
    return __fadd_rn(fmaxf(to_float(v), -INFINITY), 0.f);
  }
  __device__ __forceinline__ float t_of(float f) const {
    if (temperature == 1.f) return f;
    const float t = __fdiv_rn(f, temperature);
    return t == 0.f ? 0.f : t;
  }
  __device__ __forceinline__ float operator()(int i) const { return CACHED ? cache[i + pad] : clean(x[i]); }

  // The first pass: the row into shared memory, f(i, x) for each element of this
  // thread, reading global memory in 16-byte vectors, several in flight.
  template <typename F>
  __device__ __forceinline__ void load(F&& f) const {
    constexpr int N = 16 / sizeof(T), U = 6;
    const int vectors = (V - head) / N;
    const uint4* p = reinterpret_cast<const uint4*>(x + head);
    auto one = [&](int i) {
      const float v = clean(x[i]);
      if (CACHED) cache[i + pad] = v;
      f(i, v);
    };
    if (threadIdx.x < head) one(threadIdx.x);
    for (int v0 = threadIdx.x; v0 < vectors; v0 += U * kThreads) {
      uint4 w[U];
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (v0 + u * kThreads < vectors) w[u] = __ldg(p + v0 + u * kThreads);
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (v0 + u * kThreads < vectors) {
          const T* e = reinterpret_cast<const T*>(&w[u]);
          const int i = head + (v0 + u * kThreads) * N;
#pragma unroll
          for (int j = 0; j < N; j += 4) {
            const float4 v = make_float4(clean(e[j]), clean(e[j + 1]), clean(e[j + 2]), clean(e[j + 3]));
            if (CACHED) *reinterpret_cast<float4*>(cache + i + pad + j) = v;
            f(i + j, v.x), f(i + j + 1, v.y), f(i + j + 2, v.z), f(i + j + 3, v.w);
          }
        }
    }
    const int tail = head + vectors * N + threadIdx.x;
    if (tail < V) one(tail);
    if (CACHED && threadIdx.x < 4) {
      if (threadIdx.x < pad) cache[threadIdx.x] = -INFINITY;
      if ((V + pad + threadIdx.x) / 4 == (V + pad) / 4) cache[V + pad + threadIdx.x] = -INFINITY;
    }
  }

  // A later pass: f(i, x) for each element of this thread. Also called with x = -inf
  // for up to 3 indices on either side of the row.
  template <typename F>
  __device__ __forceinline__ void sweep(F&& f) const {
    if (CACHED) {
      const int groups = (V + pad + 3) >> 2;
#pragma unroll 2
      for (int g = threadIdx.x; g < groups; g += kThreads) {
        const float4 v = reinterpret_cast<const float4*>(cache)[g];
        const int i = g * 4 - pad;
        f(i, v.x), f(i + 1, v.y), f(i + 2, v.z), f(i + 3, v.w);
      }
    } else {
#pragma unroll 4
      for (int i = threadIdx.x; i < V; i += kThreads) f(i, clean(x[i]));
    }
  }
};

// What is still in question: tokens before (bound, bound_index) in the order, if
// their t is at least `least`.
struct Candidates {
  float bound;
  int bound_index;
  float least;
  __device__ __forceinline__ bool has(float t, int i) const {
    return t >= least && (t > bound || (t == bound && i < bound_index));
  }
};

// f(i, t) over the listed candidates, or over the row's elements from x = `from` on.
template <typename R, typename F>
__device__ __forceinline__ void each(const R& row, const Scratch& s, bool listed, float from, F&& f) {
  if (listed) {
    for (int i = threadIdx.x; i < s.list_n; i += kThreads) f(s.list[i], s.list_t[i]);
  } else {
    row.sweep([&](int i, float x) {
      if (x >= from && static_cast<unsigned>(i) < static_cast<unsigned>(row.V)) f(i, row.t_of(x));
    });
  }
}

// The elements that `take(i, x)` accepts (none of -inf) as a list; false if they
// are too many.
template <typename R, typename F>
__device__ __forceinline__ bool make_list(const R& row, Scratch& s, F&& take) {
  __syncthreads();
  if (threadIdx.x == 0) s.list_n = 0;
  __syncthreads();
  row.sweep([&](int i, float x) {
    if (take(i, x)) {  // one addition for the lanes that take together
      const unsigned lanes = __activemask();
      const int lane = threadIdx.x & 31, leader = __ffs(lanes) - 1;
      int at = 0;
      if (lane == leader) at = atomicAdd(&s.list_n, __popc(lanes));
      at = __shfl_sync(lanes, at, leader) + __popc(lanes & ((1u << lane) - 1));
      if (at < kList) {
        s.list[at] = i;
        s.list_t[at] = row.t_of(x);
      }
    }
  });
  __syncthreads();
  return s.list_n <= kList;
}

// The k-th largest (k >= 1) of the keys in [lo, hi] that `each` and `key` give,
// at least k of them: 256 bins of the range at a time, until a bin is one key or
// is taken whole. Returns the least key taken; *taken is how many of the last
// bin's keys were asked for, 0 where all keys >= the result are taken.
template <typename Each, typename Key>
__device__ uint32_t select_key(Scratch& s, uint32_t lo, uint32_t hi, uint32_t k, uint32_t* taken, Each&& each_of,
                               Key&& key) {
  while (true) {
    const uint32_t range = hi - lo;
    const int shift = range < kBins ? 0 : 24 - __clz(range);
    __syncthreads();
    if (threadIdx.x < kBins) s.hist[threadIdx.x] = 0;
    __syncthreads();
    each_of([&](int i, float t) {
      uint32_t u;
      if (key(i, t, u) && u >= lo && u <= hi) atomicAdd(&s.hist[(hi - u) >> shift], 1u);
    });
    __syncthreads();
    if (threadIdx.x < 32) {  // 8 bins a lane, running sums over the warp
      uint32_t c[8], sum = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) sum += c[j] = s.hist[threadIdx.x * 8 + j];
      uint32_t incl = sum;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t up = __shfl_up_sync(0xffffffff, incl, o);
        if (threadIdx.x >= o) incl += up;
      }
      uint32_t before = incl - sum;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (before < k && before + c[j] >= k) {
          s.pick[0] = threadIdx.x * 8 + j;
          s.pick[1] = k - before;  // asked of this bin
          s.pick[2] = c[j];
        }
        before += c[j];
      }
    }
    __syncthreads();
    const uint32_t bin = s.pick[0], count = s.pick[2];
    k = s.pick[1];
    const uint32_t top = hi - (bin << shift);
    const uint32_t width = (1u << shift) - 1;
    lo = top - lo > width ? top - width : lo;
    hi = top;
    if (k == count || lo == hi) {
      *taken = k == count ? 0 : k;
      return lo;
    }
  }
}

template <typename T, bool CACHED>
__global__ void __launch_bounds__(kThreads, 1) sample_kernel(const Args a) {
  extern __shared__ __align__(16) float cache[];
  __shared__ Scratch s;
  const int b = blockIdx.x, tid = threadIdx.x, V = a.V;
  // An infinite temperature would make NaN of infinite logits, which no histogram of keys
  // from the lowest to the largest counts: a search for the k-th would not end.
  const float asked = a.temperature_rows ? a.temperature_rows[b] : a.temperature, temperature = fminf(asked, kMost);
  const bool greedy = !(asked > 0.f);
  const int64_t k64 = a.top_k_rows ? a.top_k_rows[b] : a.top_k;
  const uint32_t top_k = (k64 <= 0 || k64 >= V) ? 0u : static_cast<uint32_t>(k64);
  const float top_p = a.top_p_rows ? a.top_p_rows[b] : a.top_p;
  const float min_p = a.min_p_rows ? a.min_p_rows[b] : a.min_p;
  const Row<T, CACHED> row(static_cast<const T*>(a.logits) + b * a.row_stride, cache, greedy ? 1.f : temperature, V);
  const float* gumbel = a.gumbel + b * a.gumbel_stride;

  // the row, its largest logit, and each thread's own
  float own_max = -INFINITY;
  row.load([&](int, float x) { own_max = fmaxf(own_max, x); });
  const float x_max = block_max(own_max, s);  // also orders the cache's writes before the reads below
  const float max = row.t_of(x_max);
  if (max == -INFINITY) {  // also where every quotient overflows
    if (tid == 0) {
      a.token[b] = -1;
      a.logprob[b] = -INFINITY;
    }
    return;
  }
  // not 0 (a quotient by more than 2^126 is, in fast division): -inf times it is -inf
  const float per_x = fmaxf(1.4426950408889634f / row.temperature, kLeast);
  const bool by_mass = !greedy && !(top_p >= 1.f);  // with NaN only the first token is kept, as with a min_p of NaN
  // The largest t is +inf, of every x that overflows (or is +inf): they share the mass,
  // and x orders nothing and bounds nothing among them.
  const bool flat = max == INFINITY;
  float sum = 0.f;
  unsigned long long total = 0;
  if (flat)
    row.sweep([&](int, float x) {
      const float e = row.t_of(x) == max ? 1.f : 0.f;
      sum += e;
      if (by_mass && !top_k) total += weight(e);
    });
  else if (by_mass && !top_k)
    row.sweep([&](int, float x) {
      const float e = x == x_max ? 1.f : exp2f((x - x_max) * per_x);
      sum += e;
      total += weight(e);
    });
  else
    row.sweep([&](int, float x) { sum += x == x_max ? 1.f : exp2f((x - x_max) * per_x); });
  sum = block_sum(sum, s);

  Best winner = {-INFINITY, V};  // of the kept
  if (!greedy) {
    // no token below this x is kept (with room for the rounding of t and exp)
    float from = -kMost;  // a logit of -inf never is
    const float room = flat ? INFINITY : 1e-3f * row.temperature + 1e-5f * fabsf(x_max);
    const float zeros = 2.f * kLeast * row.temperature;  // as wide as the x whose t is 0
    if (min_p > 0.f) from = fmaxf(from, x_max + logf(min_p) * row.temperature - room);
    Candidates c = {-INFINITY, V, -kMost};
    bool listed = false, done = false;
    if (top_k) {
      // Bins of x, from the largest down, holding each thread's `m` largest: where
      // k of those are reached, so are k of the row. One bin more than that, as
      // different x may share a t.
      const int m = top_k <= 256 ? 1 : 4;
      float own[4] = {own_max, -INFINITY, -INFINITY, -INFINITY};
      if (m > 1) {
        own[0] = -INFINITY;
        row.sweep([&](int, float x) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float up = fmaxf(own[j], x);
            x = fminf(own[j], x);
            own[j] = up;
          }
        });
      }
      float least = own[0];
#pragma unroll
      for (int j = 1; j < 4; ++j)
        if (j < m && own[j] > -INFINITY) least = own[j];
      const float x_min = block_min(least > -INFINITY ? least : x_max, s);
      const float bins = (kBins - 1) / (x_max - x_min);
      if (x_max > x_min && bins < 3e38f && !flat && top_k <= 1024) {
        auto bin = [&](float x) { return static_cast<int>(fminf((x_max - x) * bins, kBins - 1.f)); };
        if (tid < kBins) s.hist[tid] = 0;
        if (tid == 0) s.pick[0] = kBins;
        __syncthreads();
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (j < m && own[j] > -INFINITY) atomicAdd(&s.hist[bin(own[j])], 1u);
        __syncthreads();
        if (tid < 32) {
          uint32_t h[8], n = 0;
#pragma unroll
          for (int j = 0; j < 8; ++j) n += h[j] = s.hist[tid * 8 + j];
          uint32_t upto = n;
#pragma unroll
          for (int o = 1; o < 32; o <<= 1) {
            const uint32_t up = __shfl_up_sync(0xffffffff, upto, o);
            if (tid >= o) upto += up;
          }
          uint32_t before = upto - n;
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            if (before < top_k && before + h[j] >= top_k) s.pick[0] = tid * 8 + j;
            before += h[j];
          }
        }
        __syncthreads();
        const int last = static_cast<int>(s.pick[0]) + 1;
        // the last bin holds everything below x_min too
        // (top_p needs the mass of all k, so min_p does not thin them here)
        if (last < kBins - 1) {
          // everything with bin(x) <= last, and what rounding adds
          const float end = x_max - static_cast<float>(last + 1) / bins * 1.00001f - 1e-6f * fabsf(x_max) - zeros;
          const float low = by_mass ? fmaxf(end, -kMost) : fmaxf(end, from);
          listed = make_list(row, s, [&](int, float x) { return x >= low; });
        }
      }
      const int n = s.list_n;
      if (listed && n <= kRanked) {
        // few: each against all
        if (tid < n) s.weights[tid] = static_cast<uint32_t>(weight(mass_of(s.list_t[tid], max)));
        __syncthreads();
        // four neighbouring threads a candidate, a quarter of the others each
        const int mine = tid >> 2;
        const bool on = mine < n;
        const int i = on ? s.list[mine] : V;
        const float t = on ? s.list_t[mine] : INFINITY;
        uint32_t rank = 0;
        unsigned long long before = 0;
#pragma unroll 4
        for (int j = tid & 3; j < n; j += 4) {
          const float u = s.list_t[j];
          const bool is = u > t || (u == t && s.list[j] < i);
          const uint32_t w = s.weights[j];
          rank += is;
          before += is ? w : 0u;
        }
#pragma unroll
        for (int o = 1; o < 4; o <<= 1) {
          rank += __shfl_xor_sync(0xffffffff, rank, o);
          before += __shfl_xor_sync(0xffffffff, before, o);
        }
        const bool owner = on && (tid & 3) == 0 && rank < top_k && t >= -kMost;
        if (by_mass) total = block_sum(owner ? static_cast<unsigned long long>(s.weights[mine]) : 0ull, s);
        if (owner && mass_of(t, max) >= min_p &&
            (!by_mass || before == 0 || static_cast<float>(before) < top_p * static_cast<float>(total))) {
          const float g = t + __ldg(gumbel + i);
          winner = Best{g == g ? g : -INFINITY, i};
        }
        winner = block_best(winner, s);
        done = true;
      } else {
        const float all = -INFINITY;
        uint32_t taken;
        auto among = [&](auto&& f) { each(row, s, listed, all, f); };
        const uint32_t key_k = select_key(s, kLowestKey, key_of(max), min(top_k, static_cast<uint32_t>(listed ? n : V)),
                                          &taken, among, [&](int, float t, uint32_t& u) { u = key_of(t); return true; });
        int last_index = V;
        if (taken) {  // some of the equal values at the end, lowest index first
          uint32_t rest;
          const uint32_t u = select_key(s, 0u, static_cast<uint32_t>(V - 1), taken, &rest, among,
                                        [&](int i, float t, uint32_t& v) {
                                          v = static_cast<uint32_t>(V - 1 - i);
                                          return key_of(t) == key_k;
                                        });
          last_index = V - static_cast<int>(u);
        }
        // the order's prefix ends at key_k, last_index
        const uint32_t bits = (key_k & 0x80000000u) ? key_k & 0x7fffffffu : ~key_k;
        c.bound = __uint_as_float(bits);
        c.bound_index = last_index;
        if (by_mass) {
          total = 0;
          among([&](int i, float t) {
            if (c.has(t, i)) total += weight(mass_of(t, max));
          });
        }
      }
    }
    if (by_mass && !done) {
      total = block_sum(total, s);
      // V tokens of less than this cannot add up to the mass that top_p leaves out
      const float tiny = (1.f - top_p) * (static_cast<float>(total) * 4.656612873e-10f) / static_cast<float>(V);
      if (tiny > 0.f) from = fmaxf(from, x_max + logf(tiny) * row.temperature - room);
      const float bins = (kBins - 1) / (x_max - from);
      if (!top_k && !flat && bins > 0.f && bins < 3e38f) {
        // Masses by bins of x from the largest down, rounded down: where they reach
        // what is wanted the kept tokens end, or before. One bin more, as different x
        // may share a t.
        const float unit = 2147483648.f / static_cast<float>(V);  // no bin overflows
        if (tid < kBins) s.hist[tid] = 0;
        if (tid == 0) s.pick[0] = kBins;
        __syncthreads();
        row.sweep([&](int, float x) {
          if (x >= from) {
            const uint32_t w = __float2uint_rz((x == x_max ? 1.f : exp2f((x - x_max) * per_x)) * unit);
            if (w) atomicAdd(&s.hist[static_cast<int>(fminf((x_max - x) * bins, kBins - 1.f))], w);
          }
        });
        __syncthreads();
        if (tid < 32) {
          unsigned long long sum = 0;
#pragma unroll
          for (int j = 0; j < 8; ++j) sum += s.hist[tid * 8 + j];
          unsigned long long upto = sum;
#pragma unroll
          for (int o = 1; o < 32; o <<= 1) {
            const unsigned long long up = __shfl_up_sync(0xffffffff, upto, o);
            if (tid >= o) upto += up;
          }
          unsigned long long before = upto - sum;
          const float enough = top_p * static_cast<float>(total) * 1.00001f / static_cast<float>(V);
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const unsigned long long after = before + s.hist[tid * 8 + j];
            if (static_cast<float>(before) < enough && static_cast<float>(after) >= enough) s.pick[0] = tid * 8 + j;
            before = after;
          }
        }
        __syncthreads();
        const int last = static_cast<int>(s.pick[0]) + 1;
        if (last < kBins)
          from = fmaxf(from, x_max - static_cast<float>(last + 1) / bins * 1.00001f - 1e-6f * fabsf(x_max) - zeros);
        listed = make_list(row, s, [&](int, float x) { return x >= from; });
      }
    }
    const float wanted = by_mass ? top_p * static_cast<float>(total) : 0.f;
    while (!done) {
      Best w = {-INFINITY, V};
      auto consider = [&](int i, float t, float g) {
        if (c.has(t, i) && (min_p <= 0.f || mass_of(t, max) >= min_p)) {
          const float score = t + g;
          w = better(w, Best{score == score ? score : -INFINITY, i});
        }
      };
      if (listed) {
        for (int j = tid; j < s.list_n; j += kThreads) consider(s.list[j], s.list_t[j], __ldg(gumbel + s.list[j]));
      } else {
        constexpr int U = 8;  // noise of so many candidates in flight
        for (int i0 = tid; i0 < V; i0 += U * kThreads) {
          float x[U], g[U];
#pragma unroll
          for (int u = 0; u < U; ++u) {
            const int i = i0 + u * kThreads;
            x[u] = i < V ? row(i) : -INFINITY;
            g[u] = x[u] >= from ? __ldg(gumbel + i) : 0.f;
          }
#pragma unroll
          for (int u = 0; u < U; ++u)
            if (x[u] >= from) consider(i0 + u * kThreads, row.t_of(x[u]), g[u]);
        }
      }
      w = block_best(w, s);
      if (w.index >= V) break;  // nothing but the first token
      winner = w;
      if (!by_mass) break;
      const float t_w = row.t_of(row(w.index));
      unsigned long long before = 0, count = 0;
      each(row, s, listed, from, [&](int i, float t) {
        if (t > t_w || (t == t_w && i < w.index)) {
          before += weight(mass_of(t, max));
          ++count;
        }
      });
      before = block_sum(before, s);
      if (before == 0 || static_cast<float>(before) < wanted) break;
      winner = Best{-INFINITY, V};
      c.bound = t_w;  // out, and with it everything after it
      c.bound_index = w.index;
      if (!listed) {
        count = block_sum(count, s);
        if (count <= kList)
          listed = make_list(row, s, [&](int i, float x) { return x >= from && c.has(row.t_of(x), i); });
      }
    }
  }
  if (winner.index >= V) {  // greedy, or nothing else is kept: the first token of the order
    row.sweep([&](int i, float x) {
      // different x may share the largest t, near one another or around 0
      const float near = flat ? -kMost : x_max - 1e-5f * fabsf(x_max) - 2.f * kLeast * row.temperature;
      if (x == x_max || (x >= near && row.t_of(x) == max)) winner = better(winner, Best{0.f, i});
    });
    winner = block_best(winner, s);
  }
  if (tid == 0) {
    const float t = row.t_of(row(winner.index));
    a.token[b] = winner.index;
    a.logprob[b] = (t == max ? 0.f : t - max) - static_cast<float>(log(static_cast<double>(sum)));
  }
}

template <typename T>
void launch(const Args& a, int B) {
  auto st = at::cuda::getCurrentCUDAStream();
  if (a.V <= kMaxCached) {
    const int smem = (a.V + 8) * 4;
    C10_CUDA_CHECK(cudaFuncSetAttribute(sample_kernel<T, true>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                        (kMaxCached + 8) * 4));
    sample_kernel<T, true><<<B, kThreads, smem, st>>>(a);
  } else {
    sample_kernel<T, false><<<B, kThreads, 0, st>>>(a);
  }
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}

}  // namespace sampling
}  // namespace dst

using namespace dst;

// logits [B, V] (bf16 or fp32, rows may be strided), gumbel fp32 [B, V]. Each
// setting is a number or, where the tensor is given, one value per row.
std::vector<at::Tensor> sample_tokens(const at::Tensor& logits, const at::Tensor& gumbel, double temperature,
                                      int64_t top_k, double top_p, double min_p,
                                      const c10::optional<at::Tensor>& temperature_rows,
                                      const c10::optional<at::Tensor>& top_k_rows,
                                      const c10::optional<at::Tensor>& top_p_rows,
                                      const c10::optional<at::Tensor>& min_p_rows) {
  TORCH_CHECK(logits.is_cuda() && logits.dim() == 2 && logits.stride(1) == 1 &&
                  (logits.scalar_type() == at::kBFloat16 || logits.scalar_type() == at::kFloat),
              "sampling: CUDA logits [B, V], bf16 or fp32, with unit inner stride required");
  TORCH_CHECK(gumbel.is_cuda() && gumbel.device() == logits.device() && gumbel.scalar_type() == at::kFloat &&
                  gumbel.sizes() == logits.sizes() && gumbel.stride(1) == 1,
              "sampling: fp32 noise shaped like the logits, with unit inner stride, required");
  const int64_t B = logits.size(0), V = logits.size(1);
  TORCH_CHECK(B >= 1 && V >= 1 && B < (int64_t(1) << 31) && V < (int64_t(1) << 30), "sampling: empty or oversized logits");
  auto rows = [&](const c10::optional<at::Tensor>& x, at::ScalarType type, const char* name) -> const void* {
    if (!x) return nullptr;
    TORCH_CHECK(x->is_cuda() && x->device() == logits.device() && x->scalar_type() == type && x->dim() == 1 &&
                    x->size(0) == B && x->is_contiguous(),
                "sampling: ", name, " per row must be a contiguous CUDA tensor [B] of ", type);
    return x->data_ptr();
  };
  sampling::Args a;
  a.logits = logits.data_ptr();
  a.row_stride = logits.stride(0);
  a.gumbel = gumbel.data_ptr<float>();
  a.gumbel_stride = gumbel.stride(0);
  a.V = static_cast<int>(V);
  a.temperature = static_cast<float>(temperature);
  a.top_k = top_k;
  a.top_p = static_cast<float>(top_p);
  a.min_p = static_cast<float>(min_p);
  a.temperature_rows = static_cast<const float*>(rows(temperature_rows, at::kFloat, "temperature"));
  a.top_k_rows = static_cast<const int64_t*>(rows(top_k_rows, at::kLong, "top_k"));
  a.top_p_rows = static_cast<const float*>(rows(top_p_rows, at::kFloat, "top_p"));
  a.min_p_rows = static_cast<const float*>(rows(min_p_rows, at::kFloat, "min_p"));
  c10::cuda::CUDAGuard guard(logits.device());
  at::Tensor token = at::empty({B}, logits.options().dtype(at::kLong));
  at::Tensor logprob = at::empty({B}, logits.options().dtype(at::kFloat));
  a.token = token.data_ptr<int64_t>();
  a.logprob = logprob.data_ptr<float>();
  if (logits.scalar_type() == at::kBFloat16)
    sampling::launch<__nv_bfloat16>(a, static_cast<int>(B));
  else
    sampling::launch<float>(a, static_cast<int>(B));
  return {token, logprob};
}

void register_sampling(pybind11::module& m) {
  namespace py = pybind11;
  m.def("sample_tokens", &sample_tokens, "token and logprob of each row of logits", py::arg("logits"),
        py::arg("gumbel"), py::arg("temperature"), py::arg("top_k"), py::arg("top_p"), py::arg("min_p"),
        py::arg("temperature_rows"), py::arg("top_k_rows"), py::arg("top_p_rows"), py::arg("min_p_rows"));
}
