// Log probabilities of given tokens with entropy and top alternatives, and their gradient (gfx950).
//
// Row x[0 .. n), m = max x, S = sum exp(x - m), T = sum (x - m) exp(x - m):
//   logprob(t) = (x_t - m) - log S,   entropy = log S - T / S,   top: the k largest (value, lowest index first)
//   d x_v = g_lp ([v = t] - p_v) + sum_j g_top_j ([v = i_j] - p_v) - g_H p_v (log p_v + entropy)
// Both directions are bound by HBM: a value is read once and costs a handful of vector instructions.
#include "ops.hpp"

#include <hip/hip_fp16.h>

namespace ed {
namespace {

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.69314718055994531f;
constexpr float NEG_INF = -__builtin_huge_valf();

template <int DT>
struct Elem;
template <>
struct Elem<DT_FP32> {
  typedef float T;
  static __device__ __forceinline__ float get(T v) { return v; }
  static __device__ __forceinline__ T put(float v) { return v; }
};
template <>
struct Elem<DT_BF16> {
  typedef __bf16 T;
  static __device__ __forceinline__ float get(T v) { return (float)v; }
  static __device__ __forceinline__ T put(float v) { return (__bf16)v; }
};
template <>
struct Elem<DT_FP16> {
  typedef _Float16 T;
  static __device__ __forceinline__ float get(T v) { return (float)v; }
  static __device__ __forceinline__ T put(float v) { return (_Float16)v; }
};

template <typename T>
__device__ __forceinline__ const T* row_of(const LogitsView& x, long r) {
  return (const T*)x.p + (r / x.inner) * x.outer_stride + (r % x.inner) * x.inner_stride;
}

// Running softmax sums of a set of values: m the largest, s = sum exp(x - m), t = sum (x - m) exp(x - m).  Values of
// -inf add nothing; a set without a larger value stays (-inf, 0, 0).
struct Sums {
  float m, s, t;
  __device__ __forceinline__ void clear() {
    m = NEG_INF;
    s = t = 0.f;
  }
  // Differences are kept at -1e30 or above where they multiply a sum: with the lowest finite values in a row they would
  // pass the type's range and make nothing times infinity.
  __device__ __forceinline__ void add(float x) {
    if (x == NEG_INF) return;
    if (x > m) {
      const float d = fmaxf(m - x, -1.0e30f), f = exp2f(d * LOG2E);
      t = f * fmaf(d, s, t);
      s *= f;
      m = x;
    }
    const float d = x - m, e = exp2f(d * LOG2E);  // (NaN where x is NaN or +inf: it shows in s)
    s += e;
    t = fmaf(fmaxf(d, -1.0e30f), e, t);
  }
  __device__ __forceinline__ void join(const Sums& o) {
    const float mm = fmaxf(m, o.m);
    const float da = fmaxf(m - mm, -1.0e30f), db = fmaxf(o.m - mm, -1.0e30f);
    const float fa = exp2f(da * LOG2E), fb = exp2f(db * LOG2E);
    t = fa * fmaf(da, s, t) + fb * fmaf(db, o.s, o.t);
    s = s * fa + o.s * fb;
    m = mm;
  }
};

// One whole number in the order of (value, then lower index first); -0 and 0 are one value, a NaN is largest.
__device__ __forceinline__ unsigned long long key_of(float x, int idx) {
  const unsigned b = __float_as_uint(x + 0.0f);
  const unsigned o = x != x ? 0xffffffffu : b ^ ((unsigned)((int)b >> 31) | 0x80000000u);
  return ((unsigned long long)o << 32) | (0xffffffffu - (unsigned)idx);
}
__device__ __forceinline__ float key_value(unsigned long long k) {
  const unsigned o = (unsigned)(k >> 32);
  return __uint_as_float(o & 0x80000000u ? o ^ 0x80000000u : ~o);
}
__device__ __forceinline__ int key_index(unsigned long long k) { return (int)(0xffffffffu - (unsigned)k); }

__device__ __forceinline__ unsigned long long max_key(unsigned long long a, unsigned long long b) { return a > b ? a : b; }

// What a row's results are once its sums are known.
struct RowResult {
  float m, log_s, entropy;
  bool empty, bad;  // every class is -inf; a NaN or +inf is in the row
  __device__ __forceinline__ RowResult(const Sums& a) {
    empty = a.m == NEG_INF && a.s == 0.f;
    bad = !empty && !(a.s >= 1.0f && a.s < __builtin_huge_valf() && a.m < __builtin_huge_valf());
    m = empty ? 0.f : a.m;
    log_s = empty ? 0.f : bad ? __builtin_nanf("") : log2f(a.s) * LN2;
    entropy = empty ? 0.f : bad ? __builtin_nanf("") : log_s - a.t / a.s;
  }
  // the maximum as the gradient reads it: -inf marks a row without a class
  __device__ __forceinline__ float mark() const { return empty ? NEG_INF : bad ? __builtin_nanf("") : m; }
  __device__ __forceinline__ float logprob(float x) const { return bad ? __builtin_nanf("") : (x - m) - log_s; }
};

__device__ __forceinline__ void skip_row(const LogprobsOut& out, long r, int top_k, int tid, int threads) {
  if (tid == 0) {
    if (out.logprob) out.logprob[r] = 0.f;
    out.entropy[r] = 0.f;
    if (out.stats) out.stats[2 * r] = out.stats[2 * r + 1] = 0.f;
  }
  for (int j = tid; j < top_k; j += threads) {
    out.top_logprob[r * top_k + j] = 0.f;
    out.top_token[r * top_k + j] = -1;
  }
}

template <int DT>
__global__ __launch_bounds__(256) void logprobs_row_kernel(LogitsView x, const int64_t* __restrict__ targets,
                                                           const uint8_t* __restrict__ select, int top_k,
                                                           LogprobsOut out) {
  typedef typename Elem<DT>::T T;
  __shared__ Sums sums[256];
  __shared__ unsigned long long keys[256];
  const int tid = threadIdx.x;
  for (long r = blockIdx.x; r < x.rows; r += gridDim.x) {
  __syncthreads();
  if (select && !select[r]) {
    skip_row(out, r, top_k, tid, 256);
    continue;
  }
  const T* row = row_of<T>(x, r);
  Sums a;
  a.clear();
  for (int v = tid; v < x.n; v += 256) a.add(Elem<DT>::get(row[v]));
  sums[tid] = a;
  __syncthreads();
  for (int o = 128; o > 0; o >>= 1) {
    if (tid < o) sums[tid].join(sums[tid + o]);
    __syncthreads();
  }
  const RowResult res(sums[0]);
  if (tid == 0) {
    if (targets) {
      const int64_t t = targets[r];
      out.logprob[r] = t < 0 || t >= x.n ? __builtin_nanf("") : res.logprob(Elem<DT>::get(row[t]));
    }
    out.entropy[r] = res.entropy;
    if (out.stats) {
      out.stats[2 * r] = res.mark();
      out.stats[2 * r + 1] = res.log_s;
    }
  }
  unsigned long long last = ~0ull;
  for (int j = 0; j < top_k; ++j) {
    unsigned long long best = 0;
    for (int v = tid; v < x.n; v += 256) {
      const unsigned long long k = key_of(Elem<DT>::get(row[v]), v);
      if (k < last) best = max_key(best, k);
    }
    keys[tid] = best;
    __syncthreads();
    for (int o = 128; o > 0; o >>= 1) {
      if (tid < o) keys[tid] = max_key(keys[tid], keys[tid + o]);
      __syncthreads();
    }
    last = keys[0];
    __syncthreads();
    if (tid == 0) {
      out.top_logprob[r * top_k + j] = res.logprob(key_value(last));
      out.top_token[r * top_k + j] = key_index(last);
    }
  }
  }
}

template <int DT>
__global__ __launch_bounds__(256) void logprobs_grad_kernel(LogitsView x, const int64_t* __restrict__ targets,
                                                            const uint8_t* __restrict__ select, int top_k,
                                                            LogprobsGrad g) {
  typedef typename Elem<DT>::T T;
  const int tid = threadIdx.x;
  for (long r = blockIdx.x; r < x.rows; r += gridDim.x) {
  const T* row = row_of<T>(x, r);
  T* dst = (T*)g.dlogits + r * g.columns;
  const bool skip = (select && !select[r]) || g.stats[2 * r] == NEG_INF;
  const float m = g.stats[2 * r], log_s = g.stats[2 * r + 1], h = g.entropy[r];
  const float g_lp = g.g_logprob ? g.g_logprob[r] : 0.f, g_h = g.g_entropy ? g.g_entropy[r] : 0.f;
  const int64_t t = targets ? targets[r] : 0;
  float weight = g_lp;
  if (g.g_top)
    for (int j = 0; j < top_k; ++j) weight += g.g_top[r * top_k + j];
  if (t < 0 || t >= x.n) weight = __builtin_nanf("");
  for (int v = tid; v < g.columns; v += 256) {
    float d = 0.f;
    if (!skip && v < x.n) {
      const float lp = (Elem<DT>::get(row[v]) - m) - log_s;
      const float p = exp2f(lp * LOG2E);
      d = p == 0.f ? 0.f * weight : -p * (weight + g_h * (lp + h));
      if (v == t) d += g_lp;
      if (g.g_top)
        for (int j = 0; j < top_k; ++j)
          if (g.top_token[r * top_k + j] == v) d += g.g_top[r * top_k + j];
    }
    dst[v] = Elem<DT>::put(d);
  }
  }
}

}  // namespace

int64_t token_logprobs_workspace(int64_t rows, int64_t n, int top_k) { return 0; }

hipError_t launch_token_logprobs(const LogitsView& x, const int64_t* targets, const uint8_t* select, int top_k,
                                 const LogprobsOut& out, void* workspace, hipStream_t stream) {
  const dim3 grid((unsigned)(x.rows < (1 << 20) ? x.rows : 1 << 20));
  if (x.dt == DT_FP32) hipLaunchKernelGGL((logprobs_row_kernel<DT_FP32>), grid, dim3(256), 0, stream, x, targets, select, top_k, out);
  else if (x.dt == DT_BF16) hipLaunchKernelGGL((logprobs_row_kernel<DT_BF16>), grid, dim3(256), 0, stream, x, targets, select, top_k, out);
  else hipLaunchKernelGGL((logprobs_row_kernel<DT_FP16>), grid, dim3(256), 0, stream, x, targets, select, top_k, out);
  return hipGetLastError();
}

hipError_t launch_token_logprobs_backward(const LogitsView& x, const int64_t* targets, const uint8_t* select, int top_k,
                                          const LogprobsGrad& g, hipStream_t stream) {
  const dim3 grid((unsigned)(x.rows < (1 << 20) ? x.rows : 1 << 20));
  if (x.dt == DT_FP32) hipLaunchKernelGGL((logprobs_grad_kernel<DT_FP32>), grid, dim3(256), 0, stream, x, targets, select, top_k, g);
  else if (x.dt == DT_BF16) hipLaunchKernelGGL((logprobs_grad_kernel<DT_BF16>), grid, dim3(256), 0, stream, x, targets, select, top_k, g);
  else hipLaunchKernelGGL((logprobs_grad_kernel<DT_FP16>), grid, dim3(256), 0, stream, x, targets, select, top_k, g);
  return hipGetLastError();
}

}  // namespace ed
