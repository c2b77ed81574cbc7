// The next token of each row of logits, from given Gumbel noise g:
//   t = x / temperature;  order: t descending, equal values by index
//   kept: the first top_k of the order; of those the shortest prefix whose mass
//         (softmax over them) reaches top_p; of those exp(t - max) >= min_p;
//         the first token always, a logit of -inf never
//   token = argmax over the kept of t + g (equal scores: the lowest index),
//   logprob = t[token] - logsumexp(t) over the whole row.
// temperature <= 0 is greedy: the first token of the order, logprob at
// temperature 1. NaN logits count as -inf; a row without a finite or +inf logit
// gives token -1 and logprob -inf.
//
// Drawing by the maximum of t + g needs no sorted order: whether a token is kept
// is a question about the tokens before it, answered by one sum over the row. So
// the winner among all candidates is taken first and then checked; a token that
// is not kept rules out everything after it too, and the next winner is looked
// for among what is left. With top_p = 0.9 nine of ten first winners stand. The
// candidates are narrowed first by bounds that cost nothing: min_p; top_k by the
// k-th largest of the threads' own maxima (a lower bound of the k-th largest
// logit); top_p by the mass a token must have if V of its like are to count.
// Only candidates' noise is read.
//
// One CTA per row; the row is read once and stays in shared memory as fp32 t
// (longer rows are read again from L2 in each pass). Bound by one SM's load rate
// and by the passes over shared memory, not by HBM. Masses are summed as integers
// of 2^-31 of the largest, so every sum and with it every choice is independent
// of the order of the additions; logsumexp is an fp32 sum in a fixed order.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include "common.h"

namespace dst {
namespace sampling {

constexpr int kThreads = 1024;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxCached = 55296;  // t of a row in shared memory (216 KB)
constexpr int kList = 1024;        // candidates kept as a list
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
  int list_n;
  int list[kList];
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

// The row: t by index.
template <typename T, bool CACHED>
struct Row {
  const T* x;
  float* cache;
  float temperature;
  int V;
  __device__ __forceinline__ float scaled(T v) const {
    const float f = to_float(v);
    const float t = temperature == 1.f ? f : __fdiv_rn(f, temperature);
    return t != t ? -INFINITY : (t == 0.f ? 0.f : t);  // one zero: keys order -0 below +0
  }
  __device__ __forceinline__ float operator()(int i) const { return CACHED ? cache[i] : scaled(x[i]); }

  // Calls f(i, t) for each element of this thread, in the order of a fixed
  // assignment of elements to threads, reading global memory in 16-byte vectors.
  template <typename F>
  __device__ __forceinline__ void load(F&& f) const {
    constexpr int N = 16 / sizeof(T), U = 4;
    const int head = min(V, static_cast<int>((16 - (reinterpret_cast<uintptr_t>(x) & 15)) % 16 / sizeof(T)));
    const int vectors = (V - head) / N;
    const uint4* p = reinterpret_cast<const uint4*>(x + head);
    if (threadIdx.x < head) f(threadIdx.x, scaled(x[threadIdx.x]));
    for (int v0 = threadIdx.x; v0 < vectors; v0 += U * kThreads) {
      uint4 w[U];
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (v0 + u * kThreads < vectors) w[u] = __ldg(p + v0 + u * kThreads);
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (v0 + u * kThreads < vectors) {
          const T* e = reinterpret_cast<const T*>(&w[u]);
#pragma unroll
          for (int j = 0; j < N; ++j) f(head + (v0 + u * kThreads) * N + j, scaled(e[j]));
        }
    }
    const int tail = head + vectors * N + threadIdx.x;
    if (tail < V) f(tail, scaled(x[tail]));
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

// f(i, t) over the row or over the listed candidates.
template <typename R, typename F>
__device__ __forceinline__ void each(const R& row, const Scratch& s, bool listed, F&& f) {
  if (listed) {
    if (threadIdx.x < s.list_n) {
      const int i = s.list[threadIdx.x];
      f(i, row(i));
    }
  } else {
#pragma unroll 4
    for (int i = threadIdx.x; i < row.V; i += kThreads) f(i, row(i));
  }
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
  const float temperature = a.temperature_rows ? a.temperature_rows[b] : a.temperature;
  const bool greedy = !(temperature > 0.f);
  const int64_t k64 = a.top_k_rows ? a.top_k_rows[b] : a.top_k;
  const uint32_t top_k = (k64 <= 0 || k64 >= V) ? 0u : static_cast<uint32_t>(k64);
  const float top_p = a.top_p_rows ? a.top_p_rows[b] : a.top_p;
  const float min_p = a.min_p_rows ? a.min_p_rows[b] : a.min_p;
  const Row<T, CACHED> row{static_cast<const T*>(a.logits) + b * a.row_stride, cache, greedy ? 1.f : temperature, V};
  const float* gumbel = a.gumbel + b * a.gumbel_stride;

  // the row, its first token, and each thread's largest t
  Best first = {-INFINITY, V};
  row.load([&](int i, float t) {
    if (CACHED) cache[i] = t;
    first = better(first, Best{t, i});
  });
  const float own_max = first.score;
  first = block_best(first, s);  // also orders the cache's writes before the reads below
  const float max = first.score;
  if (max == -INFINITY) {
    if (tid == 0) {
      a.token[b] = -1;
      a.logprob[b] = -INFINITY;
    }
    return;
  }
  float sum = 0.f;
  unsigned long long total = 0;
  const bool by_mass = !greedy && top_p < 1.f;
#pragma unroll 4
  for (int i = tid; i < V; i += kThreads) {
    const float e = mass_of(row(i), max);
    sum += e;
    if (by_mass) total += weight(e);
  }
  sum = block_sum(sum, s);
  if (by_mass) total = block_sum(total, s);

  Best winner = first;
  if (!greedy) {
    Candidates c = {-INFINITY, V, -3.402823466e38f};  // a logit of -inf is never drawn
    bool listed = false;
    auto among = [&](auto&& f) { each(row, s, listed, f); };
    if (top_k) {
      // at least k threads have a maximum >= the k-th largest maximum
      uint32_t low_key = kLowestKey, taken;
      if (top_k <= kThreads) {
        const uint32_t mine = key_of(own_max);
        low_key = select_key(s, kLowestKey, key_of(max), top_k, &taken, [&](auto&& f) { f(tid, own_max); },
                             [&](int, float, uint32_t& u) { u = mine; return true; });
      }
      __syncthreads();
      if (tid == 0) s.list_n = 0;
      __syncthreads();
      if (top_k <= kThreads) {
#pragma unroll 4
        for (int i = tid; i < V; i += kThreads)
          if (key_of(row(i)) >= low_key) {
            const int at = atomicAdd(&s.list_n, 1);
            if (at < kList) s.list[at] = i;
          }
        __syncthreads();
        listed = s.list_n <= kList;
      }
      const uint32_t key_k = select_key(s, low_key, key_of(max), top_k, &taken, among,
                                        [&](int, float t, uint32_t& u) { u = key_of(t); return true; });
      int last_index = V;
      if (taken) {  // some of the equal values at the end, lowest index first
        uint32_t rest;
        const uint32_t u = select_key(s, 0u, static_cast<uint32_t>(V - 1), taken, &rest, among,
                                      [&](int i, float t, uint32_t& v) {
                                        v = static_cast<uint32_t>(V - 1 - i);
                                        return key_of(t) == key_k;
                                      });
        last_index = V - 1 - static_cast<int>(u) + 1;
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
        total = block_sum(total, s);
      }
    }
    const float wanted = by_mass ? top_p * static_cast<float>(total) : 0.f;
    if (by_mass) {
      // V tokens of less than this cannot add up to the mass that top_p leaves out
      const float tiny = (1.f - top_p) * (static_cast<float>(total) * 4.656612873e-10f) / static_cast<float>(V);
      if (tiny > 0.f) c.least = fmaxf(c.least, max + logf(tiny) - 1e-3f);
    }
    for (int tries = 0;; ++tries) {
      Best w = {-INFINITY, V};
      among([&](int i, float t) {
        if (c.has(t, i) && mass_of(t, max) >= min_p) {
          const float g = t + __ldg(gumbel + i);
          w = better(w, Best{g == g ? g : -INFINITY, i});
        }
      });
      w = block_best(w, s);
      if (w.index >= V) break;  // nothing but the first token
      winner = w;
      if (!by_mass || w.index == first.index) break;
      const float t_w = row(w.index);
      unsigned long long before = 0;
      among([&](int i, float t) {
        if (t > t_w || (t == t_w && i < w.index)) before += weight(mass_of(t, max));
      });
      before = block_sum(before, s);
      if (static_cast<float>(before) < wanted) break;
      winner = first;
      c.bound = t_w;  // out, and with it everything after it
      c.bound_index = w.index;
    }
  }
  if (tid == 0) {
    const float t = row(winner.index);
    a.token[b] = winner.index;
    a.logprob[b] = (t == max ? 0.f : t - max) - static_cast<float>(log(static_cast<double>(sum)));
  }
}

template <typename T>
void launch(const Args& a, int B) {
  auto st = at::cuda::getCurrentCUDAStream();
  if (a.V <= kMaxCached) {
    const int smem = a.V * 4;
    C10_CUDA_CHECK(cudaFuncSetAttribute(sample_kernel<T, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxCached * 4));
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
