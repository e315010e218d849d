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
constexpr int TOP_MAX = 32;  // = ED_TOP_K_MAX

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
  __device__ __forceinline__ RowResult(const Sums& a) : RowResult(a, log2f(a.s) * LN2) {}
  __device__ __forceinline__ RowResult(const Sums& a, float log_sum) {  // log_sum: log a.s
    empty = a.m == NEG_INF && a.s == 0.f;
    bad = !empty && !(a.s >= 1.0f && a.s < __builtin_huge_valf() && a.m < __builtin_huge_valf());
    m = empty ? 0.f : a.m;
    log_s = empty ? 0.f : bad ? __builtin_nanf("") : log_sum;
    entropy = empty ? 0.f : bad ? __builtin_nanf("") : log_s - a.t / a.s;
  }
  // the maximum as the gradient reads it: -inf marks a row without a class
  __device__ __forceinline__ float mark() const { return empty ? NEG_INF : bad ? __builtin_nanf("") : m; }
  __device__ __forceinline__ float logprob(float x) const { return bad ? __builtin_nanf("") : (x - m) - log_s; }
};

__device__ __forceinline__ void put_stats(float* to, float m, float log_s) {
  to[0] = m;
  to[1] = log_s;
}
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

// ---------------------------------------------------------------------------------------------------
// Few classes (n <= G * E <= 512): G lanes own a row and keep it in registers, lane j the classes j, j + G, ...  The alternatives are
// taken one after the other, a largest key of the group each.  64 x 31 fp32 top 5 4.5 us on the GPU, 16384 x 31
// without alternatives 3.5, most of it the launch: bound by the host's call (9.0 us).
// ---------------------------------------------------------------------------------------------------
template <int G>
__device__ __forceinline__ float group_sum(float v) {
#pragma unroll
  for (int o = 1; o < G; o <<= 1) v += __shfl_xor(v, o);
  return v;
}
template <int G>
__device__ __forceinline__ float group_max(float v) {
#pragma unroll
  for (int o = 1; o < G; o <<= 1) v = fmaxf(v, __shfl_xor(v, o));
  return v;
}

template <int DT, int G, int E>
__global__ __launch_bounds__(256) void logprobs_group_kernel(LogitsView x, const int64_t* __restrict__ targets,
                                                             const uint8_t* __restrict__ select, int top_k,
                                                             LogprobsOut out) {
  typedef typename Elem<DT>::T T;
  const int lane = threadIdx.x & (G - 1);
  for (long r = (long)blockIdx.x * (256 / G) + threadIdx.x / G; r < x.rows; r += (long)gridDim.x * (256 / G)) {
    if (select && !select[r]) {
      skip_row(out, r, top_k, lane, G);
      continue;
    }
    const T* row = row_of<T>(x, r);
    const int64_t target = targets ? targets[r] : -1;
    float v[E];
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] = e * G + lane < x.n ? Elem<DT>::get(row[e * G + lane]) : NEG_INF;
    const float xt = target >= 0 && target < x.n ? Elem<DT>::get(row[target]) : __builtin_nanf("");
    Sums a;
    a.m = v[0];
#pragma unroll
    for (int e = 1; e < E; ++e) a.m = fmaxf(a.m, v[e]);
    a.m = group_max<G>(a.m);
    a.t = 0.f;
    const float m = a.m == NEG_INF ? 0.f : a.m;
    // The term of a largest class is 1.  One of them is left out, so that the others keep their bits where they are small: log S =
    // log1p(S - 1), and the log probability of a class that is all but certain is as exact as another (12 classes, p = 0.99998: off
    // by 1e-6 of it, 2e-2 with the 1 in the sum).  (None is found where the largest is infinite: the sum is 0 or NaN.)
    float rest = 0.f;
    int largest = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const float d = v[e] - m, p = exp2f(d * LOG2E);
      const bool one = d == 0.f;
      largest += one;
      rest += one ? 0.f : p;
      a.t = fmaf(fmaxf(d, -1.0e30f), p, a.t);
    }
    const unsigned long long held = __ballot(largest > 0) >> (threadIdx.x & 63 & ~(G - 1)) & (~0ull >> (64 - G));
    if (held && lane == (int)__builtin_ctzll(held)) --largest;
    rest = group_sum<G>(rest + (float)largest);
    a.s = held ? 1.0f + rest : rest;
    a.t = group_sum<G>(a.t);
    // log1p by Kahan's quotient: log(u) / (u - 1) varies so slowly that the rounding of u = 1 + rest does not matter
    const float over = a.s - 1.0f;
    const RowResult res(a, over == 0.f ? rest : log2f(a.s) * LN2 * (rest / over));
    if (lane == 0) {
      if (targets) out.logprob[r] = res.logprob(xt);
      out.entropy[r] = res.entropy;
      if (out.stats) put_stats(out.stats + 2 * r, res.mark(), res.log_s);
    }
    if (top_k == 0) continue;
    unsigned key[E];  // order of the values; 0: taken, or no class
#pragma unroll
    for (int e = 0; e < E; ++e) key[e] = e * G + lane < x.n ? (unsigned)(key_of(v[e], 0) >> 32) : 0u;
    for (int j = 0; j < top_k; ++j) {
      unsigned best = key[0];
      int at = 0;
#pragma unroll
      for (int e = 1; e < E; ++e)
        if (key[e] > best) {
          best = key[e];
          at = e;
        }
      int idx = at * G + lane;
#pragma unroll
      for (int o = 1; o < G; o <<= 1) {
        const unsigned b = (unsigned)__shfl_xor((int)best, o);
        const int i = __shfl_xor(idx, o);
        const bool take = b > best || (b == best && i < idx);
        best = take ? b : best;
        idx = take ? i : idx;
      }
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (e * G + lane == idx) key[e] = 0u;
      if (lane == 0) {
        out.top_logprob[r * top_k + j] = res.logprob(key_value((unsigned long long)best << 32));
        out.top_token[r * top_k + j] = idx;
      }
    }
  }
}

// ---------------------------------------------------------------------------------------------------
// Many classes: one pass of 16-byte loads by a workgroup per row, or per piece of a row where there are few rows (the
// pieces are joined by a second kernel).
//
// Sums.  In base 2: y = x * log2(e) - R with one fused operation, R = M * log2(e) for M the wave's largest value so far, S = sum
// 2^y, T = sum y 2^y.  (log2(e) is off by 1.3e-8 relative in fp32, as if every logit were scaled by that: under one rounding of
// a log probability.)  y is kept at -200 or above, so that a forbidden class adds nothing and not a NaN.  Values of 2^20 and
// more leave the products too coarse: a row with such a maximum is summed once more, plainly.
//
// Top alternatives.  A group is the contiguous classes of one load; the k largest values lie in the k groups with the largest
// maxima, and as groups are ordered as their classes are, ties go the same way.  Every thread keeps its best group; the k-th
// of them (joined over the four waves: 64) is a bound tau that at least k groups reach, renewed after 1, 2, 4, ... tiles.
// Groups that reach it go to a list, about 1.2 k for each doubling; in the end the first k of the list are found by
// counting, read again class by class, and ranked the same way.  A list that overflows (rows in rising order) takes k
// plain passes: 4096 x 50257 top 20 7.8 ms.
//
// Bound by HBM where there is much to read: 4096 x 50257 bf16 80 us without alternatives (5.1 TB/s), 105 us with 20 of them;
// 4096 x 32000 54 and 60 (8).  8 x 131072 bf16 top 20 is two launches of 9.0 and 5.9 us: a chain of latencies.
// ---------------------------------------------------------------------------------------------------
constexpr float Y_MIN = -200.0f, R_MIN = -2097152.0f, PLAIN_FROM = 1048576.0f;
constexpr int LIST = 512;
typedef unsigned long long u64;

__device__ __forceinline__ float max_nan(float a, float b) { return __builtin_elementwise_maximum(a, b); }  // a NaN stays one

// Sums of a wave, workgroup or row in base 2.
struct Sums2 {
  float m, r, s, t;  // largest value, reference, sum 2^y, sum y 2^y
  __device__ __forceinline__ void rebase(float to) {
    const float d = r - to, f = __builtin_amdgcn_exp2f(d);
    t = f * fmaf(d, s, t);
    s *= f;
    r = to;
  }
  __device__ __forceinline__ void join(Sums2 o) {
    const float to = fmaxf(r, o.r);
    rebase(to);
    o.rebase(to);
    s += o.s;
    t += o.t;
    m = fmaxf(m, o.m);
  }
};

struct RowEnd {  // what follows from the sums of a whole row
  float m, log_s, entropy;
  bool empty, bad;
  __device__ __forceinline__ RowEnd(const Sums2& a) {
    empty = a.m == NEG_INF && a.s == 0.f;
    bad = !empty && !(a.s > 0.f && a.s < __builtin_huge_valf());
    const float l2 = __builtin_amdgcn_logf(a.s);
    m = empty ? 0.f : a.m;
    log_s = empty ? 0.f : bad ? __builtin_nanf("") : (l2 - fmaf(a.m, LOG2E, -a.r)) * LN2;
    entropy = empty ? 0.f : bad ? __builtin_nanf("") : (l2 - a.t / a.s) * LN2;
  }
  __device__ __forceinline__ RowEnd(const RowResult& a) : m(a.m), log_s(a.log_s), entropy(a.entropy), empty(a.empty), bad(a.bad) {}
  __device__ __forceinline__ float mark() const { return empty ? NEG_INF : bad ? __builtin_nanf("") : m; }
  __device__ __forceinline__ float logprob(float x) const { return bad ? __builtin_nanf("") : (x - m) - log_s; }
};

// The 16-byte loads of a row: classes [0, head) and [n - tail, n) stand alone, the rest are vectors of EPV.
template <int DT>
struct Vectors {
  typedef typename Elem<DT>::T T;
  static constexpr int EPV = 16 / sizeof(T);
  const T* row;
  int n, head, count;  // vectors
  __device__ __forceinline__ Vectors(const T* p, int classes) : row(p), n(classes) {
    head = (int)((16 - (reinterpret_cast<uintptr_t>(p) & 15)) & 15) / (int)sizeof(T);
    head = head < n ? head : n;
    count = (n - head) / EPV;
  }
  __device__ __forceinline__ int tail() const { return n - head - count * EPV; }
  __device__ __forceinline__ int first(int v) const { return head + v * EPV; }  // class of vector v
  __device__ __forceinline__ bool single(int e) const { return e < head || e >= head + count * EPV; }
};

template <int DT>
__device__ __forceinline__ void unpack(const uint4& raw, float (&v)[16 / sizeof(typename Elem<DT>::T)]) {
  if constexpr (DT == DT_FP32) {
    v[0] = __uint_as_float(raw.x); v[1] = __uint_as_float(raw.y); v[2] = __uint_as_float(raw.z); v[3] = __uint_as_float(raw.w);
  } else {
    const unsigned w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (DT == DT_BF16) {
        v[2 * i] = __uint_as_float(w[i] << 16);
        v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
      } else {
        v[2 * i] = (float)__builtin_bit_cast(_Float16, (unsigned short)w[i]);
        v[2 * i + 1] = (float)__builtin_bit_cast(_Float16, (unsigned short)(w[i] >> 16));
      }
    }
  }
}

// The threads of a row: a workgroup (TR = 256), or one wave of it (64), which needs no barrier.
template <int TR>
__device__ __forceinline__ void row_sync() {
  if constexpr (TR > 64) {
    __syncthreads();
  } else {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  }
}

template <int TR>
struct TopSpace {
  alignas(16) u64 best[TR];               // a thread's best group
  alignas(16) u64 list[LIST + 8];         // groups that reached tau, zeros up to a multiple of eight
  alignas(16) u64 found[TOP_MAX * 8 + 8];  // classes that may be among the k, likewise
  int group[TOP_MAX];
  u64 tau;
  int listed, n_found;
};

// tau = the k-th of the 64 best groups (as it was, where there are fewer)
template <int TR>
__device__ __forceinline__ void renew_tau(TopSpace<TR>& sp, u64 mine, int top_k, int tid) {
  sp.best[tid] = mine;
  row_sync<TR>();
  if (tid < 64) {
    u64 k = mine;
    if constexpr (TR == 256) {
      k = max_key(max_key(sp.best[tid], sp.best[tid + 64]), max_key(sp.best[tid + 128], sp.best[tid + 192]));
      sp.best[tid] = k;
      row_sync<64>();
    }
    int rank = 0;
#pragma unroll 8
    for (int j = 0; j < 64; j += 2) {
      const ulonglong2 two = *(const ulonglong2*)(sp.best + j);
      rank += (two.x > k) + (two.y > k);
    }
    if (rank == top_k - 1 && k) sp.tau = k;
  }
  row_sync<TR>();
}

// put(rank, key) for the k largest of found[0 .. n), by counting; found holds eight more (16-byte aligned).  A barrier is inside.
template <int TR, typename Put>
__device__ __forceinline__ void rank_found(u64* found, int n, int top_k, int tid, Put put) {
  if (tid < 8) found[n + tid] = 0;
  row_sync<TR>();
  for (int i = tid; i < n; i += TR) {
    const u64 k = found[i];
    int rank = 0;
    for (int j = 0; j < n; j += 8) {
#pragma unroll
      for (int e = 0; e < 8; e += 2) {
        const ulonglong2 two = *(const ulonglong2*)(found + j + e);
        rank += (two.x > k) + (two.y > k);
      }
    }
    if (rank < top_k) put(rank, k);
  }
}

// k plain passes over classes [from, to) (and [from2, to2)), each for the largest below the one before
template <int DT, int TR, typename Put>
__device__ void plain_top(const typename Elem<DT>::T* row, int from, int to, int from2, int to2, int top_k, u64* keys, int tid, Put put) {
  u64 last = ~0ull;
  for (int j = 0; j < top_k; ++j) {
    u64 best = 0;
    for (int v = from + tid; v < to; v += TR) {
      const u64 k = key_of(Elem<DT>::get(row[v]), v);
      if (k < last) best = max_key(best, k);
    }
    for (int v = from2 + tid; v < to2; v += TR) {
      const u64 k = key_of(Elem<DT>::get(row[v]), v);
      if (k < last) best = max_key(best, k);
    }
    row_sync<TR>();
    keys[tid] = best;
    row_sync<TR>();
    for (int o = TR / 2; o > 0; o >>= 1) {
      if (tid < o) keys[tid] = max_key(keys[tid], keys[tid + o]);
      row_sync<TR>();
    }
    last = keys[0];
    if (tid == 0) put(j, last);
  }
  row_sync<TR>();
}

// a row's sums without base 2 and vectors, for maxima of any size; space: 3 TR floats
template <int DT, int TR>
__device__ RowResult plain_sums(const typename Elem<DT>::T* row, int n, float* space, int tid) {
  Sums a;
  a.clear();
  for (int v = tid; v < n; v += TR) a.add(Elem<DT>::get(row[v]));
  row_sync<TR>();
  space[tid] = a.m; space[TR + tid] = a.s; space[2 * TR + tid] = a.t;
  row_sync<TR>();
  for (int o = TR / 2; o > 0; o >>= 1) {
    if (tid < o) {
      Sums b;
      a.m = space[tid]; a.s = space[TR + tid]; a.t = space[2 * TR + tid];
      b.m = space[tid + o]; b.s = space[TR + tid + o]; b.t = space[2 * TR + tid + o];
      a.join(b);
      space[tid] = a.m; space[TR + tid] = a.s; space[2 * TR + tid] = a.t;
    }
    row_sync<TR>();
  }
  a.m = space[0]; a.s = space[TR]; a.t = space[2 * TR];
  row_sync<TR>();
  return RowResult(a);
}

struct Piece {  // of a row: its sums, followed in memory by top_k keys
  Sums2 sums;
};
__host__ __device__ inline long piece_bytes(int top_k) { return (long)sizeof(Piece) + 8L * top_k; }

template <int DT, bool TOP, int TR>
__global__ __launch_bounds__(256, 4) void logprobs_stream_kernel(LogitsView x, const int64_t* __restrict__ targets,
                                                              const uint8_t* __restrict__ select, int top_k,
                                                              LogprobsOut out, char* __restrict__ pieces, int splits) {
  typedef typename Elem<DT>::T T;
  constexpr int EPV = Vectors<DT>::EPV, U = 4;
  constexpr int ROWS = 256 / TR;  // a workgroup works on
  __shared__ TopSpace<TR> spaces[TOP ? ROWS : 1];
  __shared__ Sums2 wave_sums[4];
  __shared__ float plain_spaces[ROWS][3 * TR];
  const int in = threadIdx.x / TR, tid = threadIdx.x % TR, lane = tid & 63, wid = tid >> 6;
  TopSpace<TR>& sp = spaces[TOP ? in : 0];
  const long items = x.rows * splits;
  for (long item = (long)blockIdx.x * ROWS + in; item < items; item += (long)gridDim.x * ROWS) {
    const long r = item / splits;
    const int piece = (int)(item - r * splits);
    if (select && !select[r]) {
      if (piece == 0 && splits == 1) skip_row(out, r, top_k, tid, TR);
      continue;
    }
    const Vectors<DT> vec(row_of<T>(x, r), x.n);
    const int chunk = (vec.count + splits - 1) / splits;
    const int v0 = piece * chunk < vec.count ? piece * chunk : vec.count;
    const int v1 = v0 + chunk < vec.count ? v0 + chunk : vec.count;
    const uint4* src = (const uint4*)(vec.row + vec.head);
    const unsigned none = DT == DT_FP32 ? 0xff800000u : DT == DT_BF16 ? 0xff80ff80u : 0xfc00fc00u;

    row_sync<TR>();  // the row before is done with the shared memory
    if (TOP && tid == 0) {
      sp.tau = 0;
      sp.listed = sp.n_found = 0;
    }
    Sums2 a{NEG_INF, R_MIN, 0.f, 0.f};
    auto raise = [&](float v) {  // a larger value somewhere in the wave: new reference
      a.m = fmaxf(a.m, v);
#pragma unroll
      for (int o = 32; o > 0; o >>= 1) a.m = fmaxf(a.m, __shfl_xor(a.m, o));
      a.rebase(fmaxf(a.m * LOG2E, R_MIN));
    };
    auto add = [&](float v) {
      const float y = max_nan(fmaf(v, LOG2E, -a.r), Y_MIN), e = __builtin_amdgcn_exp2f(y);
      a.s += e;
      a.t = fmaf(y, e, a.t);
    };
    // classes in front of and behind the vectors
    float alone = NEG_INF;
    int alone_at = -1;
    if (piece == 0) {
      if (tid < vec.head) alone_at = tid;
      else if (tid >= 32 && tid - 32 < vec.tail()) alone_at = vec.n - vec.tail() + tid - 32;
      if (alone_at >= 0) alone = Elem<DT>::get(vec.row[alone_at]);
      if (__any(alone > a.m)) raise(alone);
      add(alone);
      if (TOP) {
        row_sync<TR>();
        if (alone_at >= 0) sp.list[atomicAdd(&sp.listed, 1)] = key_of(alone, alone_at);
      }
    }

    uint4 raw[U], next[U];
    auto load = [&](uint4 (&to)[U], int at) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int v = at + u * TR + tid;
        to[u] = v < v1 ? src[v] : make_uint4(none, none, none, none);
      }
    };
    float best = NEG_INF, tau_value = NEG_INF;  // this thread's best group
    int best_at = -1, tiles = 0, renew_at = 1;
    u64 tau = 0;
    load(next, v0);
    for (int at = v0; at < v1; at += TR * U) {
#pragma unroll
      for (int u = 0; u < U; ++u) raw[u] = next[u];
      load(next, at + TR * U);
      float high[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        float v[EPV];
        unpack<DT>(raw[u], v);
        high[u] = v[0];
#pragma unroll
        for (int i = 1; i < EPV; ++i) high[u] = fmaxf(high[u], v[i]);
        if (__any(high[u] > a.m)) raise(high[u]);
#pragma unroll
        for (int i = 0; i < EPV; ++i) add(v[i]);
      }
      if constexpr (TOP) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int g = at + u * TR + tid;
          if (g < v1 && (high[u] > best || best_at < 0)) {
            best = high[u];
            best_at = vec.first(g);
          }
        }
        if (++tiles == renew_at && at + TR * U < v1 || tiles == 1) {
          renew_tau<TR>(sp, best_at < 0 ? 0 : key_of(best, best_at), top_k, tid);
          tau = sp.tau;
          tau_value = tau ? key_value(tau) : NEG_INF;
          renew_at *= TR == 64 ? 2 : 4;
        }
        if (__any(fmaxf(fmaxf(high[0], high[1]), fmaxf(high[2], high[3])) >= tau_value)) {
#pragma unroll
          for (int u = 0; u < U; ++u) {
            const int g = at + u * TR + tid;
            const u64 k = key_of(high[u], vec.first(g));
            const bool take = g < v1 && k >= tau;
            const u64 mask = __ballot(take);
            if (mask) {
              int base = 0;
              if (lane == (int)__builtin_ctzll(mask)) base = atomicAdd(&sp.listed, (int)__popcll(mask));
              base = __shfl(base, (int)__builtin_ctzll(mask));
              const int pos = base + (int)__popcll(mask & ((1ull << lane) - 1));
              if (take && pos < LIST) sp.list[pos] = k;
            }
          }
        }
      }
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
      a.s += __shfl_xor(a.s, o);
      a.t += __shfl_xor(a.t, o);
    }
    if constexpr (TR > 64) {
      if (lane == 0) wave_sums[wid] = a;
      __syncthreads();
      a = wave_sums[0];
#pragma unroll
      for (int w = 1; w < TR / 64; ++w) a.join(wave_sums[w]);
    } else {
      row_sync<TR>();
    }

    char* const mine = pieces + item * piece_bytes(top_k);
    if (splits > 1) {
      if (tid == 0) ((Piece*)mine)->sums = a;
    }
    const bool plain = splits == 1 && (a.m > PLAIN_FROM || a.m < -PLAIN_FROM) && a.m != NEG_INF;
    const RowEnd res = plain ? RowEnd(plain_sums<DT, TR>(vec.row, vec.n, plain_spaces[in], tid)) : RowEnd(a);
    if (splits == 1 && tid == 0) {
      if (targets) {
        const int64_t t = targets[r];
        out.logprob[r] = t < 0 || t >= x.n ? __builtin_nanf("") : res.logprob(Elem<DT>::get(vec.row[t]));
      }
      out.entropy[r] = res.entropy;
      if (out.stats) put_stats(out.stats + 2 * r, res.mark(), res.log_s);
    }
    if constexpr (TOP) {
      auto put = [&](int rank, u64 k) {
        if (splits > 1) {
          ((u64*)(mine + sizeof(Piece)))[rank] = k;
        } else {
          out.top_logprob[r * top_k + rank] = res.logprob(key_value(k));
          out.top_token[r * top_k + rank] = key_index(k);
        }
      };
      const int listed = sp.listed;  // at least k groups (all there are, if fewer)
      const bool fits = listed <= LIST;
      if (fits) {
        // the k groups of the list that come first, the last of them as the bound; then their classes that reach it
        rank_found<TR>(sp.list, listed, top_k, tid, [&](int rank, u64 k) {
          sp.group[rank] = key_index(k);
          if (rank == top_k - 1) sp.tau = k;
        });
        if (tid == 0 && listed < top_k) sp.tau = 0;
        row_sync<TR>();
        const u64 floor = sp.tau ? sp.tau - (EPV - 1) : 0;  // (its value, the last class of its group)
        const int groups = listed < top_k ? listed : top_k;
        for (int i = tid; i < groups * EPV; i += TR) {
          const int e0 = sp.group[i / EPV], e = e0 + i % EPV;
          if (vec.single(e0) && e != e0) continue;
          const u64 k = key_of(Elem<DT>::get(vec.row[e]), e);
          if (k >= floor) sp.found[atomicAdd(&sp.n_found, 1)] = k;
        }
        row_sync<TR>();
        const int n = sp.n_found;
        rank_found<TR>(sp.found, n, top_k, tid, put);
        // a piece may hold fewer classes than k (or a NaN may have hidden some)
        for (int j = n + tid; j < top_k; j += TR) put(j, splits > 1 ? 0 : key_of(NEG_INF, 0));
      }
      if (!fits) {
        const bool ends = piece == 0;
        plain_top<DT, TR>(vec.row, ends ? 0 : vec.first(v0), vec.first(v1), ends ? vec.n - vec.tail() : vec.n, vec.n, top_k, sp.best, tid,
                      [&](int j, u64 k) { put(j, k || splits > 1 ? k : key_of(NEG_INF, 0)); });
      }
    }
  }
}

// The pieces of a row: sums joined in order; of the sorted lists, the k-th of their first ceil(k / splits) entries each is a
// bound that k classes reach.
template <int DT>
__global__ __launch_bounds__(256) void logprobs_join_kernel(LogitsView x, const int64_t* __restrict__ targets,
                                                            const uint8_t* __restrict__ select, int top_k, LogprobsOut out,
                                                            const char* __restrict__ pieces, int splits) {
  typedef typename Elem<DT>::T T;
  __shared__ u64 keys[64 * TOP_MAX];
  __shared__ alignas(16) u64 firsts[64 + TOP_MAX + 8];
  __shared__ alignas(16) u64 found[64 * TOP_MAX + 8];
  __shared__ u64 tau;
  __shared__ int n_found;
  __shared__ float plain_space[768];
  const int tid = threadIdx.x;
  for (long r = blockIdx.x; r < x.rows; r += gridDim.x) {
    if (select && !select[r]) {
      skip_row(out, r, top_k, tid, 256);
      continue;
    }
    const T* row = row_of<T>(x, r);
    const char* src = pieces + r * splits * piece_bytes(top_k);
    __syncthreads();
    if (tid == 0) {
      tau = 0;
      n_found = 0;
    }
    const int64_t t = targets ? targets[r] : -1;  // (its value and the pieces are on their way together)
    const float target_value = targets && t >= 0 && t < x.n ? Elem<DT>::get(row[t]) : 0.f;
    const int depth = top_k ? (top_k + splits - 1) / splits : 0, n_firsts = depth * splits;  // < splits + top_k <= 96
    for (int i = tid; i < splits * top_k; i += 256) {
      const int s = i / top_k, j = i - s * top_k;
      const u64 k = ((const u64*)(src + s * piece_bytes(top_k) + sizeof(Piece)))[j];
      keys[i] = k;
      if (j < depth) firsts[s * depth + j] = k;
    }
    if (tid < 8) firsts[n_firsts + tid] = 0;
    Sums2 a{NEG_INF, R_MIN, 0.f, 0.f};  // every wave joins all pieces, one a lane
    if ((tid & 63) < splits) a = ((const Piece*)(src + (tid & 63) * piece_bytes(top_k)))->sums;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const Sums2 b{__shfl_xor(a.m, o), __shfl_xor(a.r, o), __shfl_xor(a.s, o), __shfl_xor(a.t, o)};
      a.join(b);
    }
    const bool plain = (a.m > PLAIN_FROM || a.m < -PLAIN_FROM) && a.m != NEG_INF;
    const RowEnd res = plain ? RowEnd(plain_sums<DT, 256>(row, x.n, plain_space, tid)) : RowEnd(a);
    if (tid == 0) {
      if (targets) out.logprob[r] = t < 0 || t >= x.n ? __builtin_nanf("") : res.logprob(target_value);
      out.entropy[r] = res.entropy;
      if (out.stats) put_stats(out.stats + 2 * r, res.mark(), res.log_s);
    }
    if (top_k == 0) continue;
    __syncthreads();
    if (tid < n_firsts) {
      const u64 k = firsts[tid];
      int rank = 0;
      for (int j = 0; j < n_firsts; j += 8) {
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
          const ulonglong2 two = *(const ulonglong2*)(firsts + j + e);
          rank += (two.x > k) + (two.y > k);
        }
      }
      if (rank == top_k - 1 && k) tau = k;
    }
    __syncthreads();
    const u64 floor = tau;
    for (int i = tid; i < splits * top_k; i += 256)
      if (keys[i] && keys[i] >= floor) found[atomicAdd(&n_found, 1)] = keys[i];
    __syncthreads();
    auto put = [&](int rank, u64 k) {
      out.top_logprob[r * top_k + rank] = res.logprob(key_value(k));
      out.top_token[r * top_k + rank] = key_index(k);
    };
    const int n = n_found;
    rank_found<256>(found, n, top_k, tid, put);
    for (int j = n + tid; j < top_k; j += 256) put(j, key_of(NEG_INF, 0));
  }
}

// ---------------------------------------------------------------------------------------------------
// Gradient: a value in, a value out.  log p comes from the row's saved maximum and log sum; the few classes that are named
// (target, top alternatives) get the whole sum for their class, in a fixed order.
// ---------------------------------------------------------------------------------------------------
struct GradRow {
  float m, log_s, h, weight, g_h;
  bool skip;
  __device__ __forceinline__ float at(float x) const {
    const float lp = (x - m) - log_s, p = __builtin_amdgcn_exp2f(lp * LOG2E);
    // From log p = -200 on p is 0, far under the least value of the type; held there, the other factor stays finite for incoming
    // gradients up to 1e36: a forbidden class gets nothing, not nothing times infinity.
    return -p * fmaf(g_h, max_nan(lp, -200.0f) + h, weight);
  }
};
__device__ __forceinline__ GradRow grad_row(const LogitsView& x, const int64_t* targets, const uint8_t* select,
                                            const LogprobsGrad& g, long r) {  // (weight: without the top alternatives)
  GradRow a;
  a.m = g.stats[2 * r];
  a.log_s = g.stats[2 * r + 1];
  a.skip = (select && !select[r]) || a.m == NEG_INF;
  a.h = g.entropy[r];
  a.weight = g.g_logprob ? g.g_logprob[r] : 0.f;
  a.g_h = g.g_entropy ? g.g_entropy[r] : 0.f;
  // (a target that is no class: its log probability is NaN, and so is a gradient that comes through it; no other does)
  if (a.weight != 0.f && targets && (targets[r] < 0 || targets[r] >= x.n)) a.weight = __builtin_nanf("");
  return a;
}
// what the named classes of row r add to class v
__device__ __forceinline__ float named(const int64_t* targets, int top_k, const LogprobsGrad& g, long r, int64_t v) {
  float d = g.g_logprob && targets[r] == v ? g.g_logprob[r] : 0.f;
  if (g.g_top)
    for (int j = 0; j < top_k; ++j)
      if (g.top_token[r * top_k + j] == v) d += g.g_top[r * top_k + j];
  return d;
}

// A workgroup per `per` tiles of 256 vectors of a row, 16 bytes of the destination each: loads, the next tile's in flight, at whatever
// alignment the source has there (the last 32000 of 32001 columns, 4096 rows, bf16: 99 us, class by class 295), and aligned stores.
// The stores pass by the caches (the reader behind is a product over the whole gradient): 4096 x 32000 bf16 117 -> 90 us (5.8 TB/s
// in and out), 1024 x 32000 fp32 56 -> 43.  The named classes of the piece are listed in shared memory while the first loads fly,
// with a bit for each vector that holds one.
constexpr int GRAD_TILES = 8;  // at most, of a workgroup
template <int DT>
__global__ __launch_bounds__(256) void logprobs_grad_kernel(LogitsView x, const int64_t* __restrict__ targets,
                                                            const uint8_t* __restrict__ select, int top_k,
                                                            LogprobsGrad g, int pieces, int per) {
  typedef typename Elem<DT>::T T;
  constexpr int EPV = 16 / sizeof(T), U = 2;
  typedef __attribute__((ext_vector_type(EPV))) T VT;
  typedef VT Loose __attribute__((aligned(sizeof(T))));
  __shared__ int64_t cls[TOP_MAX + 1];  // named classes and their gradients, in order
  __shared__ float cls_g[TOP_MAX + 1];
  __shared__ int name_at[TOP_MAX + 1];  // those of this piece, each once, and their sums
  __shared__ float name_add[TOP_MAX + 1];
  __shared__ int n_names;
  __shared__ unsigned hot[GRAD_TILES * 8];
  const int tid = threadIdx.x;
  const long items = x.rows * pieces;
  for (long item = blockIdx.x; item < items; item += gridDim.x) {
    const long r = item / pieces;
    const int piece = (int)(item - r * pieces);
    const T* row = row_of<T>(x, r);
    T* dst = (T*)g.dlogits + r * g.columns;
    const int head = (int)((16 - (reinterpret_cast<uintptr_t>(dst) & 15)) & 15) / (int)sizeof(T);
    // the vectors of this piece, all of them classes; columns beside vectors are the first and the last piece's
    const int vectors = x.n > head ? (x.n - head) / EPV : 0;
    const int v0 = piece * per * 256 < vectors ? piece * per * 256 : vectors;
    const int v1 = v0 + per * 256 < vectors && piece + 1 < pieces ? v0 + per * 256 : vectors;
    auto edges = [&](auto one) {  // one(column) for those of this piece that no vector holds
      if (vectors > 0) {
        if (piece == 0 && tid < head) one(tid);
        if (piece + 1 == pieces)
          for (long v = head + (long)vectors * EPV + tid; v < g.columns; v += 256) one(v);
      } else {
        const long span = (g.columns + pieces - 1) / pieces, to = (piece + 1) * span < g.columns ? (piece + 1) * span : g.columns;
        for (long v = piece * span + tid; v < to; v += 256) one(v);
      }
    };
    if (select && !select[r]) {  // left out: nothing of the row is read (4096 x 32000 bf16 with half of them 70 -> 55 us)
      for (int vec = v0 + tid; vec < v1; vec += 256) __builtin_nontemporal_store(VT{}, (VT*)(dst + head + (long)vec * EPV));
      edges([&](long v) { dst[v] = Elem<DT>::put(0.f); });
      continue;
    }
    uint4 next[U];
    auto load = [&](int at) {
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (at + u * 256 + tid < v1) next[u] = __builtin_bit_cast(uint4, *(const Loose*)(row + head + (long)(at + u * 256 + tid) * EPV));
    };
    load(v0);
    GradRow a = grad_row(x, targets, select, g, r);
    const int has_target = g.g_logprob ? 1 : 0, names = has_target + (g.g_top ? top_k : 0);
    __syncthreads();  // the row before is done with the shared memory
    if (tid < names) {
      const bool target = has_target && tid == 0;
      const long at = r * top_k + tid - has_target;
      cls[tid] = target ? targets[r] : g.top_token[at];
      cls_g[tid] = target ? g.g_logprob[r] : g.g_top[at];
    }
    if (tid == 0) n_names = 0;
    if (tid < GRAD_TILES * 8) hot[tid] = 0;
    __syncthreads();
    for (int j = has_target; j < names; ++j) a.weight += cls_g[j];
    if (tid < names) {
      const int64_t v = cls[tid], vec = (v - head) / EPV;
      const bool inside = v >= head && vec < vectors;
      if (v >= 0 && v < x.n && (!inside || (vec >= v0 && vec < v1))) {
        float d = 0.f;
        bool first = true;
        for (int j = 0; j < names; ++j)
          if (cls[j] == v) {
            first &= j >= tid;
            d += cls_g[j];
          }
        if (first) {
          const int slot = atomicAdd(&n_names, 1);
          name_at[slot] = (int)v;
          name_add[slot] = d;
          if (inside) atomicOr(&hot[(vec - v0) >> 5], 1u << ((vec - v0) & 31));
        }
      }
    }
    __syncthreads();
    const int listed = n_names;
    for (int at = v0; at < v1; at += 256 * U) {
      uint4 raw[U];
#pragma unroll
      for (int u = 0; u < U; ++u) raw[u] = next[u];
      load(at + 256 * U);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int vec = at + u * 256 + tid;
        if (vec >= v1) continue;
        const int first = head + vec * EPV;
        float f[EPV];
        unpack<DT>(raw[u], f);
#pragma unroll
        for (int i = 0; i < EPV; ++i) f[i] = a.at(f[i]);
        if (hot[(vec - v0) >> 5] >> ((vec - v0) & 31) & 1)
          for (int j = 0; j < listed; ++j) {
            const int off = name_at[j] - first;
#pragma unroll
            for (int i = 0; i < EPV; ++i) f[i] += off == i ? name_add[j] : 0.f;
          }
        VT o;
#pragma unroll
        for (int i = 0; i < EPV; ++i) o[i] = Elem<DT>::put(a.skip ? 0.f : f[i]);
        __builtin_nontemporal_store(o, (VT*)(dst + first));
      }
    }
    edges([&](long v) {
      float d = 0.f;
      if (!a.skip && v < x.n) {
        d = a.at(Elem<DT>::get(row[v]));
        for (int j = 0; j < listed; ++j)
          if (name_at[j] == v) {
            d += name_add[j];
            break;
          }
      }
      dst[v] = Elem<DT>::put(d);
    });
  }
}

// Few columns: a thread per value, rows behind each other (16384 x 31 fp32 5 us, most of it the launch).
template <int DT>
__global__ __launch_bounds__(256) void logprobs_grad_flat_kernel(LogitsView x, const int64_t* __restrict__ targets,
                                                                 const uint8_t* __restrict__ select, int top_k,
                                                                 LogprobsGrad g) {
  typedef typename Elem<DT>::T T;
  const long count = x.rows * g.columns;
  for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < count; i += (long)gridDim.x * 256) {
    const long r = i / g.columns;
    const int v = (int)(i - r * g.columns);
    GradRow a = grad_row(x, targets, select, g, r);
    if (g.g_top)
      for (int j = 0; j < top_k; ++j) a.weight += g.g_top[r * top_k + j];
    float d = 0.f;
    if (!a.skip && v < x.n) d = a.at(Elem<DT>::get(row_of<T>(x, r)[v])) + named(targets, top_k, g, r, v);
    ((T*)g.dlogits)[i] = Elem<DT>::put(d);
  }
}

}  // namespace

// A wave a row instead of a workgroup, with no barrier anywhere: rows enough to fill the chip that way (4096 x 50257 bf16 top 5
// 97 us against 113, 16384 x 4096 55 against 130), or too short to share.
static bool wave_rows(int64_t rows, int64_t n) { return rows >= 2048 || n <= 4096; }

// Pieces of a row: one where the rows alone give every CU two workgroups; else as many as bring the grid there, none under 4096
// classes (under two 16-byte loads a thread a piece costs more than it saves), at most 64.
static int row_splits(int64_t rows, int64_t n) {
  if (wave_rows(rows, n)) return 1;
  const int64_t want = (512 + rows - 1) / rows, most = (n + 4095) / 4096;
  const int64_t s = want < most ? want : most;
  return s < 1 ? 1 : s > 64 ? 64 : (int)s;
}

int64_t token_logprobs_workspace(int64_t rows, int64_t n, int top_k) {
  const int splits = row_splits(rows, n);
  return splits > 1 ? rows * splits * piece_bytes(top_k) : 0;
}

template <int DT>
static hipError_t launch_logprobs(const LogitsView& x, const int64_t* targets, const uint8_t* select, int top_k,
                                  const LogprobsOut& out, void* workspace, hipStream_t stream) {
  auto blocks = [&](long n) { return dim3((unsigned)(n < (1 << 20) ? n : 1 << 20)); };
#define ED_GROUP(G, E)                                                                                                     \
  hipLaunchKernelGGL((logprobs_group_kernel<DT, G, E>), blocks((x.rows + 256 / G - 1) / (256 / G)), dim3(256), 0, stream, x, \
                     targets, select, top_k, out)
  if (x.n <= 32) ED_GROUP(4, 8);
  else if (x.n <= 64) ED_GROUP(8, 8);
  else if (x.n <= 256) ED_GROUP(16, 16);
  else if (x.n <= 512 && top_k <= 4) ED_GROUP(64, 8);  // (few passes over registers: 16384 x 300 bf16 top 1 13 us, top 5 on the other form 33)
  else {
    const int splits = row_splits(x.rows, x.n);
#define ED_STREAM(TOP, TR)                                                                                                \
  hipLaunchKernelGGL((logprobs_stream_kernel<DT, TOP, TR>), blocks(TR == 256 ? x.rows * splits : (x.rows + 3) / 4), dim3(256), 0, stream, x, \
                     targets, select, top_k, out, (char*)workspace, splits)
    if (wave_rows(x.rows, x.n)) {
      if (top_k > 0) ED_STREAM(true, 64);
      else ED_STREAM(false, 64);
    } else {
      if (top_k > 0) ED_STREAM(true, 256);
      else ED_STREAM(false, 256);
    }
#undef ED_STREAM
    if (splits > 1) {
      const hipError_t e = hipGetLastError();
      if (e != hipSuccess) return e;
      hipLaunchKernelGGL((logprobs_join_kernel<DT>), blocks(x.rows), dim3(256), 0, stream, x, targets, select, top_k, out,
                         (const char*)workspace, splits);
    }
  }
#undef ED_GROUP
  return hipGetLastError();
}

hipError_t launch_token_logprobs(const LogitsView& x, const int64_t* targets, const uint8_t* select, int top_k,
                                 const LogprobsOut& out, void* workspace, hipStream_t stream) {
  if (x.dt == DT_FP32) return launch_logprobs<DT_FP32>(x, targets, select, top_k, out, workspace, stream);
  if (x.dt == DT_BF16) return launch_logprobs<DT_BF16>(x, targets, select, top_k, out, workspace, stream);
  return launch_logprobs<DT_FP16>(x, targets, select, top_k, out, workspace, stream);
}

template <int DT>
static hipError_t launch_grad(const LogitsView& x, const int64_t* targets, const uint8_t* select, int top_k, const LogprobsGrad& g,
                              hipStream_t stream) {
  auto blocks = [&](long n) { return dim3((unsigned)(n < (1 << 20) ? n : 1 << 20)); };
  if (g.columns <= 256) {
    hipLaunchKernelGGL((logprobs_grad_flat_kernel<DT>), blocks((x.rows * g.columns + 255) / 256), dim3(256), 0, stream, x, targets,
                       select, top_k, g);
  } else {
    // tiles of 256 vectors in a workgroup: eight where the rows are many (the row's scalars and names are read once for
    // them), down to two so that few rows still fill the chip eight workgroups a CU deep
    const long tiles = (g.columns / (16 / dt_bytes(DT)) + 255) / 256;
    int per = GRAD_TILES;
    while (per > 2 && x.rows * ((tiles + per - 1) / per) < 2048) per /= 2;
    const int pieces = (int)((tiles + per - 1) / per);
    hipLaunchKernelGGL((logprobs_grad_kernel<DT>), blocks(x.rows * pieces), dim3(256), 0, stream, x, targets, select, top_k, g, pieces, per);
  }
  return hipGetLastError();
}

hipError_t launch_token_logprobs_backward(const LogitsView& x, const int64_t* targets, const uint8_t* select, int top_k,
                                          const LogprobsGrad& g, hipStream_t stream) {
  if (x.dt == DT_FP32) return launch_grad<DT_FP32>(x, targets, select, top_k, g, stream);
  if (x.dt == DT_BF16) return launch_grad<DT_BF16>(x, targets, select, top_k, g, stream);
  return launch_grad<DT_FP16>(x, targets, select, top_k, g, stream);
}

}  // namespace ed
