// Block-scaled 8-bit floating point (OCP e4m3) on gfx950: quantisation and the product.
//
// A block of 128 values - 128 channels of a row, or 128 x 128 weights - shares a scale 2^s, s the smallest whole number with
// max |x| <= 448 * 2^s (448: the largest e4m3 value).  Powers of two cost no precision in a floating format (only range at
// the small end), are exact to apply, and are what the matrix instruction takes beside its operands (E8M0 bytes): the
// product needs no vector instruction for its scales.
#include "ops.hpp"

#include <hip/hip_fp16.h>

namespace ed {
namespace {

typedef __attribute__((ext_vector_type(8))) int i32x8;
typedef __attribute__((ext_vector_type(4))) int i32x4;
typedef __attribute__((ext_vector_type(4))) float f32x4;

template <int DT>
struct Elem;
template <>
struct Elem<DT_FP32> { typedef float T; };
template <>
struct Elem<DT_BF16> { typedef __bf16 T; };
template <>
struct Elem<DT_FP16> { typedef _Float16 T; };

// E8M0 byte of the scale for a block whose largest magnitude has these bits: 448 = 2^8 * (1 + 0x600000 / 2^23).
__device__ __forceinline__ int scale_byte(unsigned amax) {
  const int e = (int)(amax >> 23) - 8 + ((amax & 0x7fffffu) > 0x600000u ? 1 : 0);
  return e < 1 ? 1 : e > 254 ? 254 : e;
}
__device__ __forceinline__ float inverse_scale(int byte) { return __uint_as_float((unsigned)(254 - byte) << 23); }  // 2^(127 - byte)

// Eight values of a row at column k0 (a multiple of 8): zeros behind K.
template <int DT>
__device__ __forceinline__ void load8(const typename Elem<DT>::T* row, long k0, long K, bool wide, float (&v)[8]) {
  typedef typename Elem<DT>::T T;
  typedef __attribute__((ext_vector_type(8))) T V8;
  if (wide && k0 + 8 <= K) {
    const V8 raw = *(const V8*)(row + k0);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = (float)raw[i];
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = k0 + i < K ? (float)row[k0 + i] : 0.f;
  }
}
// largest magnitude (as bits) of eight values; Inf and NaN do not count and become NaN
__device__ __forceinline__ unsigned amax8(float (&v)[8]) {
  unsigned a = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const unsigned b = __float_as_uint(v[i]) & 0x7fffffffu;
    if (b >= 0x7f800000u) v[i] = __builtin_nanf("");
    else a = b > a ? b : a;
  }
  return a;
}
__device__ __forceinline__ uint2 pack8(const float (&v)[8], float inv) {
  uint2 r;
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(v[0] * inv, v[1] * inv, 0, false);
  r.x = (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(v[2] * inv, v[3] * inv, w, true);
  w = __builtin_amdgcn_cvt_pk_fp8_f32(v[4] * inv, v[5] * inv, 0, false);
  r.y = (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(v[6] * inv, v[7] * inv, w, true);
  return r;
}

// 16 lanes own a block of 128.
template <int DT>
__global__ __launch_bounds__(256) void quantize_rows_kernel(const void* __restrict__ x, long row_stride, long blocks,
                                                            int kb, long K, bool wide, uint8_t* __restrict__ q,
                                                            uint8_t* __restrict__ scale) {
  const long blk = (long)blockIdx.x * 16 + (threadIdx.x >> 4);
  if (blk >= blocks) return;
  const int l = threadIdx.x & 15;
  const long row = blk / kb;
  const int b = (int)(blk - row * kb);
  float v[8];
  load8<DT>((const typename Elem<DT>::T*)x + row * row_stride, (long)b * FP8_BLOCK + l * 8, K, wide, v);
  unsigned a = amax8(v);
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) {
    const unsigned c = (unsigned)__shfl_xor((int)a, o);
    a = c > a ? c : a;
  }
  const int byte = scale_byte(a);
  *(uint2*)(q + blk * FP8_BLOCK + l * 8) = pack8(v, inverse_scale(byte));
  if (l == 0) scale[blk] = (uint8_t)byte;
}

// One workgroup per 128 x 128 weights: thread (r, c) holds columns 8c .. 8c + 7 of rows r, r + 16, ...
template <int DT>
__global__ __launch_bounds__(256) void quantize_weight_kernel(const void* __restrict__ w, long row_stride, long N, int kb,
                                                              long K, bool wide, uint8_t* __restrict__ q,
                                                              uint8_t* __restrict__ scale) {
  __shared__ unsigned red[4];
  const int l = threadIdx.x & 15, r0 = threadIdx.x >> 4;
  const long nb = blockIdx.x / kb;
  const int b = (int)(blockIdx.x - nb * kb);
  float v[8][8];
  unsigned a = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const long row = nb * FP8_BLOCK + r0 + i * 16;
    if (row < N) {
      load8<DT>((const typename Elem<DT>::T*)w + row * row_stride, (long)b * FP8_BLOCK + l * 8, K, wide, v[i]);
      const unsigned c = amax8(v[i]);
      a = c > a ? c : a;
    }
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const unsigned c = (unsigned)__shfl_xor((int)a, o);
    a = c > a ? c : a;
  }
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = a;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 4; ++i) a = red[i] > a ? red[i] : a;
  const int byte = scale_byte(a);
  const float inv = inverse_scale(byte);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const long row = nb * FP8_BLOCK + r0 + i * 16;
    if (row < N) *(uint2*)(q + (row * kb + b) * FP8_BLOCK + l * 8) = pack8(v[i], inv);
  }
  if (threadIdx.x == 0) scale[nb * kb + b] = (uint8_t)byte;
}

template <int OUT_DT>
__device__ __forceinline__ void store_out(void* out, long at, float v) {
  ((typename Elem<OUT_DT>::T*)out)[at] = (typename Elem<OUT_DT>::T)v;
}

// 16 bytes of K at chunk c (of 8) of a block row
__device__ __forceinline__ i32x8 load_fragment(const uint8_t* row, int fq) {
  const i32x4 a = *(const i32x4*)(row + fq * 16), b = *(const i32x4*)(row + 64 + fq * 16);
  return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
}

// Eight products at a time, the 8-bit matrix instructions (scaled or not, any shape) align to the largest and drop what lies
// under 2^-13 of it: results are 4e-5 to 6e-5 (2-norm) from the exact sum at any K, well under half a step of bf16 (2e-3) or fp16
// (2e-4), which those outputs are rounded by anyway.  fp32 outputs take the exact form: e4m3 values are exact in bf16, so are
// their products in fp32, and the bf16 instruction keeps fp32 sums; it has half the rate.
typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8;
typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2;

// values 8 s2 .. 8 s2 + 7 of a fragment times 2^(byte - 127) as bf16 (exact; magnitudes under 2^-126 vanish)
__device__ __forceinline__ bf16x8 widen(const i32x8& v, int s2, float scale) {
  bf16x8 r;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const bf16x2 lo = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((unsigned)v[2 * s2 + i], scale, false);
    const bf16x2 hi = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((unsigned)v[2 * s2 + i], scale, true);
    r[4 * i] = lo[0]; r[4 * i + 1] = lo[1]; r[4 * i + 2] = hi[0]; r[4 * i + 3] = hi[1];
  }
  return r;
}
__device__ __forceinline__ float scale_of(int byte) {  // 2^(byte - 127)
  return byte == 0 ? __uint_as_float(0x400000u) : byte == 255 ? __builtin_nanf("") : __uint_as_float((unsigned)byte << 23);
}

// A wave per 32 x 32 results, operands straight from memory.  The weights are the instruction's row operand: a lane then
// holds four consecutive channels of one row.  Rows and channels past the end read the last one and are not stored.
template <int OUT_DT>
__global__ __launch_bounds__(256) void gemm_kernel(Fp8Gemm g) {
  const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6;
  const int fr = lane & 15, fq = lane >> 4;
  const long tiles_n = (g.N + 63) / 64;
  const long m0 = blockIdx.x / tiles_n * 64 + (wid >> 1) * 32, n0 = blockIdx.x % tiles_n * 64 + (wid & 1) * 32;
  const long pitch = (long)g.kb * FP8_BLOCK;
  long rm[2], rn[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    rm[i] = m0 + i * 16 + fr < g.M ? m0 + i * 16 + fr : g.M - 1;
    rn[i] = n0 + i * 16 + fr < g.N ? n0 + i * 16 + fr : g.N - 1;
  }
  f32x4 acc[2][2] = {};
  for (int b = 0; b < g.kb; ++b) {
    i32x8 w[2], x[2];
    int sw[2], sx[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      w[i] = load_fragment(g.wq + rn[i] * pitch + (long)b * FP8_BLOCK, fq);
      x[i] = load_fragment(g.xq + rm[i] * pitch + (long)b * FP8_BLOCK, fq);
      sw[i] = g.ws[(rn[i] >> 7) * g.kb + b];
      sx[i] = g.xs[rm[i] * g.kb + b];
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j)
        if constexpr (OUT_DT != DT_FP32) {
          acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w[i], x[j], acc[i][j], 0, 0, 0, sw[i], 0, sx[j]);
        } else {
#pragma unroll
          for (int s2 = 0; s2 < 4; ++s2)
            acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(widen(w[i], s2, scale_of(sw[i])), widen(x[j], s2, scale_of(sx[j])), acc[i][j], 0, 0, 0);
        }
  }
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const long m = m0 + j * 16 + fr;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const long n = n0 + i * 16 + fq * 4 + e;
        if (m < g.M && n < g.N) store_out<OUT_DT>(g.out, m * g.N + n, acc[i][j][e] + (g.bias ? g.bias[n] : 0.f));
      }
    }
}

bool wide_rows(const void* p, int dt, int64_t row_stride) {  // every row starts on eight aligned elements
  const int64_t align = 8 * dt_bytes(dt) < 16 ? 8 * dt_bytes(dt) : 16;
  return (reinterpret_cast<uintptr_t>(p) % align) == 0 && (row_stride * dt_bytes(dt)) % align == 0;
}

}  // namespace

hipError_t launch_fp8_quantize_rows(const void* x, int dt, int64_t row_stride, int64_t rows, int64_t K, uint8_t* q,
                                    uint8_t* scale, hipStream_t stream) {
  const int kb = (int)fp8_blocks(K);
  const long blocks = rows * kb;
  const dim3 grid((unsigned)((blocks + 15) / 16));
  const bool wide = wide_rows(x, dt, row_stride);
#define ED_GO(DT) hipLaunchKernelGGL((quantize_rows_kernel<DT>), grid, dim3(256), 0, stream, x, (long)row_stride, blocks, kb, (long)K, wide, q, scale)
  if (dt == DT_FP32) ED_GO(DT_FP32);
  else if (dt == DT_BF16) ED_GO(DT_BF16);
  else ED_GO(DT_FP16);
#undef ED_GO
  return hipGetLastError();
}

hipError_t launch_fp8_quantize_weight(const void* w, int dt, int64_t row_stride, int64_t N, int64_t K, uint8_t* q,
                                      uint8_t* scale, hipStream_t stream) {
  const int kb = (int)fp8_blocks(K);
  const dim3 grid((unsigned)(fp8_blocks(N) * kb));
  const bool wide = wide_rows(w, dt, row_stride);
#define ED_GO(DT) hipLaunchKernelGGL((quantize_weight_kernel<DT>), grid, dim3(256), 0, stream, w, (long)row_stride, (long)N, kb, (long)K, wide, q, scale)
  if (dt == DT_FP32) ED_GO(DT_FP32);
  else if (dt == DT_BF16) ED_GO(DT_BF16);
  else ED_GO(DT_FP16);
#undef ED_GO
  return hipGetLastError();
}

static hipError_t launch_gemm(const Fp8Gemm& g, hipStream_t stream) {
  const dim3 grid((unsigned)(((g.N + 63) / 64) * ((g.M + 63) / 64)));
  if (g.out_dt == DT_FP32) hipLaunchKernelGGL((gemm_kernel<DT_FP32>), grid, dim3(256), 0, stream, g);
  else if (g.out_dt == DT_BF16) hipLaunchKernelGGL((gemm_kernel<DT_BF16>), grid, dim3(256), 0, stream, g);
  else hipLaunchKernelGGL((gemm_kernel<DT_FP16>), grid, dim3(256), 0, stream, g);
  return hipGetLastError();
}

// workspace: the quantised rows, then their scales
int64_t fp8_linear_workspace(int64_t M, int64_t N, int64_t K, bool quantised) {
  return quantised ? 0 : M * fp8_blocks(K) * (FP8_BLOCK + 1);
}

hipError_t launch_fp8_linear(const Fp8Linear& p, hipStream_t stream) {
  const int kb = (int)fp8_blocks(p.K);
  Fp8Gemm g{(const uint8_t*)p.x, p.x_scale, p.w, p.w_scale, p.bias, p.out, p.out_dt, p.M, p.N, kb};
  if (p.x_dt != DT_E4M3) {
    uint8_t* q = (uint8_t*)p.workspace;
    uint8_t* scale = q + p.M * kb * FP8_BLOCK;
    const hipError_t e = launch_fp8_quantize_rows(p.x, p.x_dt, p.row_stride, p.M, p.K, q, scale, stream);
    if (e != hipSuccess) return e;
    g.xq = q;
    g.xs = scale;
  }
  return launch_gemm(g, stream);
}

}  // namespace ed
