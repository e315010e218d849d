// Block-scaled 8-bit floating point (OCP e4m3) on gfx950: quantisation and the product.
//
// A block of 128 values - 128 channels of a row, or 128 x 128 weights - shares a scale 2^s, s the smallest whole number with
// max |x| <= 448 * 2^s (448: the largest e4m3 value).  Powers of two cost no precision in a floating format (only range at
// the small end), are exact to apply, and are what the matrix instruction takes beside its operands (E8M0 bytes): the
// product needs no vector instruction for its scales.
#include "ops.hpp"

#include <hip/hip_fp16.h>

#include <type_traits>

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

// 16 lanes own a block of 128; a workgroup takes U blocks of 16 rows, all loads first.  TURNED: scales go to (kb, rows), as the
// product reads them (16 rows' bytes side by side), instead of (rows, kb).
template <int DT, int U, bool TURNED>
__global__ __launch_bounds__(256) void quantize_rows_kernel(const void* __restrict__ x, long row_stride, long rows, int kb, long K,
                                                            bool wide, uint8_t* __restrict__ q, uint8_t* __restrict__ scale) {
  const int chunks = (kb + U - 1) / U;
  const long row = blockIdx.x / chunks * 16 + (threadIdx.x >> 4);
  const int b0 = (int)(blockIdx.x % chunks) * U, l = threadIdx.x & 15;
  if (row >= rows) return;
  const typename Elem<DT>::T* src = (const typename Elem<DT>::T*)x + row * row_stride;
  float v[U][8];
#pragma unroll
  for (int u = 0; u < U; ++u) load8<DT>(src, (long)(b0 + u) * FP8_BLOCK + l * 8, K, wide, v[u]);
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int b = b0 + u;
    if (b >= kb) break;
    unsigned a = amax8(v[u]);
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) {
      const unsigned c = (unsigned)__shfl_xor((int)a, o);
      a = c > a ? c : a;
    }
    const int byte = scale_byte(a);
    *(uint2*)(q + (row * kb + b) * FP8_BLOCK + l * 8) = pack8(v[u], inverse_scale(byte));
    if (l == 0) scale[TURNED ? b * rows + row : row * kb + b] = (uint8_t)byte;
  }
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

// Memory -> LDS copies and the scale loads are buffer instructions: they are bounded by the buffer (bytes past it read as zero:
// rows behind the last need no clamp), take the step of K as a scalar offset, and unlike global ones leave the waits
// for LDS reads countable.
typedef __amdgpu_buffer_rsrc_t buffer_t;
__device__ __forceinline__ buffer_t buffer_of(const uint8_t* p, long bytes) {
  return __builtin_amdgcn_make_buffer_rsrc((void*)p, 0, (int)(unsigned)(bytes < 0xfffffff0L ? bytes : 0xfffffff0L), 0x00020000);
}
__device__ __forceinline__ void copy16(buffer_t src, unsigned lane_off, unsigned off, char* lds) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(src, (__attribute__((address_space(3))) void*)lds, 16, (int)lane_off, (int)off, 0, 0);
}
__device__ __forceinline__ int load_byte(buffer_t src, unsigned lane_off, unsigned off) {
  return __builtin_amdgcn_raw_buffer_load_b8(src, (int)lane_off, (int)off, 0);
}

// ---------------------------------------------------------------------------------------------------
// Tiled product.  Four waves, 2 (rows) x 2 (channels), own a tile of 32 WTM rows x 32 WTN channels, a wave 16 WTM x 16 WTN as
// WTN x WTM instructions of 16 x 16 x 128: one per block of K and pair of fragments, its scales beside it.
//
// Step of K (one block): rows of 128 bytes of both operands, copied memory -> LDS a step ahead into one of two stages.  The
// 16-byte chunk c of tile row r lies at chunk c ^ (r >> 1 & 7) (the copy's source addresses are permuted, its image is
// lane-linear): the 16 rows of a fragment read then fall on 16 different slots of the banks.
//
// Order inside a step.  A wave's channel fragments pass through a ring of four, its row fragments stay for the step.  Once
// the last channel fragment of the step is read (row of instructions JB), the one barrier of the step: behind it the next
// stage has landed and this one is free.  The rows of instructions left cover the reads of the next step's first fragments and
// the copies of the step after, so that neither the barrier nor a read leaves the matrix pipe without work.  The
// order is pinned (sched_barrier): at most two auxiliary instructions behind each matrix instruction.
//
// The channels of an LDS tile are permuted within 32 so that two instructions give a lane eight consecutive ones: 16-byte stores.
// ---------------------------------------------------------------------------------------------------
template <int WTM, int WTN, int OUT_DT>
__global__ __launch_bounds__(256, 1) void tile_kernel(Fp8Gemm g, int tiles_m, int tiles_n) {
  constexpr int BM = 32 * WTM, BN = 32 * WTN, STAGE = (BM + BN) * 128;
  constexpr int GX = BM / 32, GW = BN / 32, NG = GX + GW;  // 8-row copies a wave makes of each operand
  constexpr int RING = 4, JB = WTN > 4 ? WTN - 3 : WTN - 2;  // the barrier stands before row JB of instructions
  static_assert(JB >= WTN - RING + 1 && JB >= 1, "every channel fragment of a step is read in front of its barrier");
  __shared__ __attribute__((aligned(1024))) char lds[2 * STAGE];
  const int lane = threadIdx.x & 63, wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int fr = lane & 15, fq = lane >> 4, wr = wid >> 1, wc = wid & 1;

  // Tiles: workgroups id, id + 8, ... share an XCD and its L2; each XCD takes a run of the order in which four tile rows are
  // walked column by column, so that what it holds at a time is a compact block.
  int tile_m, tile_n;
  {
    const int total = tiles_m * tiles_n, id = blockIdx.x, q = total >> 3, r = total & 7, xcd = id & 7;
    const int at = (xcd < r ? xcd * (q + 1) : r * (q + 1) + (xcd - r) * q) + (id >> 3);
    const int per = 4 * tiles_n, band = at / per, in = at - band * per, high = min(tiles_m - 4 * band, 4);
    tile_n = in / high;
    tile_m = 4 * band + in - tile_n * high;
  }
  const long m0 = (long)tile_m * BM, n0 = (long)tile_n * BN, pitch = (long)g.kb * FP8_BLOCK;
  const int T = g.kb;

  // copies: lane -> (row of 8, physical chunk)
  const int chunk0 = ((lane & 7) ^ (lane >> 4)) * 16, chunk1 = ((lane & 7) ^ (4 + (lane >> 4))) * 16;
  unsigned off[NG];
#pragma unroll
  for (int j = 0; j < GX; ++j) {
    const int row = (wid * GX + j) * 8 + (lane >> 3);
    off[j] = (unsigned)(row * pitch) + ((wid * GX + j) & 1 ? chunk1 : chunk0);
  }
#pragma unroll
  for (int j = 0; j < GW; ++j) {
    const int lr = (wid * GW + j) * 8 + (lane >> 3);
    const int ch = (lr & ~31) + 8 * ((lr & 15) >> 2) + 4 * ((lr >> 4) & 1) + (lr & 3);
    off[GX + j] = (unsigned)(ch * pitch) + ((wid * GW + j) & 1 ? chunk1 : chunk0);
  }
  const buffer_t x_src = buffer_of(g.xq + m0 * pitch, (g.M - m0) * pitch);
  const buffer_t w_src = buffer_of(g.wq + n0 * pitch, (g.N - n0) * pitch);
  auto copy = [&](int j, unsigned at, char* stage) {  // piece j of the step at byte `at` of the rows
    if (j < GX) copy16(x_src, off[j], at, stage + (wid * GX + j) * 1024);
    else copy16(w_src, off[j], at, stage + BM * 128 + (wid * GW + j - GX) * 1024);
  };

  // scales: a lane's row in each of the WTM fragments; the wave's channels lie in one block of 128
  const unsigned mw = (unsigned)(m0 + wr * 16 * WTM + fr);
  const long nw = n0 + wc * 16 * WTN;
  const buffer_t sx_src = buffer_of(g.xs, g.M * (long)T);  // (kb, M)
  const buffer_t sw_src = buffer_of(g.ws + ((nw < g.N ? nw : g.N - 1) >> 7) * g.kb, T);

  const int swz = (fq ^ ((fr >> 1) & 7)) << 4;
  const int x_rd = (wr * 16 * WTM + fr) * 128, w_rd = BM * 128 + (wc * 16 * WTN + fr) * 128;
  auto read = [&](const char* stage, int base, int half) { return *(const i32x4*)(stage + base + ((half << 6) ^ swz)); };
  auto put = [](i32x8& f, int half, i32x4 v) {
    if (half == 0) { f[0] = v[0]; f[1] = v[1]; f[2] = v[2]; f[3] = v[3]; }
    else { f[4] = v[0]; f[5] = v[1]; f[6] = v[2]; f[7] = v[3]; }
  };

  f32x4 acc[WTN][WTM] = {};
  i32x8 X[WTM], W[RING];
  int sx[WTM], sx_next[WTM], sw, sw_next;

  // step 0, its first fragments, step 1's copies
#pragma unroll
  for (int j = 0; j < NG; ++j) copy(j, 0, lds);
#pragma unroll
  for (int i = 0; i < WTM; ++i) sx[i] = load_byte(sx_src, mw + i * 16, 0);
  sw = load_byte(sw_src, 0, 0);
  __syncthreads();
#pragma unroll
  for (int i = 0; i < WTM; ++i) { put(X[i], 0, read(lds, x_rd + i * 2048, 0)); put(X[i], 1, read(lds, x_rd + i * 2048, 1)); }
#pragma unroll
  for (int j = 0; j < 2; ++j) { put(W[j], 0, read(lds, w_rd + j * 2048, 0)); put(W[j], 1, read(lds, w_rd + j * 2048, 1)); }
  // The copies run two steps ahead; past the last step they repeat its block (in bounds, into a stage nobody reads).
  const unsigned last = (unsigned)(T - 1);
  unsigned at = (last < 1 ? last : 1) * FP8_BLOCK;
#pragma unroll
  for (int j = 0; j < NG; ++j) copy(j, at, lds + STAGE);

  for (int t = 0; t < T; ++t) {
    char* const here = lds + (t & 1) * STAGE;
    const char* const there = lds + (1 - (t & 1)) * STAGE;
    const unsigned next = (unsigned)t < last ? t + 1 : last;
    const unsigned sx_at = next * (unsigned)g.M;
    at = ((unsigned)t + 2 < last ? t + 2 : last) * FP8_BLOCK;
#pragma unroll
    for (int j = 0; j < WTN; ++j) {
      if (j == JB) {
        __builtin_amdgcn_sched_barrier(0);
        __syncthreads();  // (drains this wave's copies and reads)
        __builtin_amdgcn_sched_barrier(0);
      }
#pragma unroll
      for (int i = 0; i < WTM; ++i) {
        acc[j][i] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(W[j % RING], X[i], acc[j][i], 0, 0, 0, sw, 0, sx[i]);
        const int slot = j * WTM + i;
        if (j < JB) {
          // channel fragments 2 .. WTN - 1, two reads each, as soon as their slot of the ring is free
#pragma unroll
          for (int r = 0; r < 2 * (WTN - 2); ++r) {
            const int f = 2 + r / 2, want = f < RING ? r : (f - RING + 1) * WTM + (r & 1);
            if (want == slot) put(W[f % RING], r & 1, read(here, w_rd + f * 2048, r & 1));
          }
          if (slot >= 4 && slot < 4 + WTM) sx_next[slot - 4] = load_byte(sx_src, mw + (slot - 4) * 16, sx_at);  // the next step's scales
          if (slot == 4) sw_next = load_byte(sw_src, 0, next);
        } else {
          constexpr int COPY_SLOTS = (WTN - JB) * WTM;
          const int after = slot - JB * WTM;
#pragma unroll
          for (int c = after * NG / COPY_SLOTS; c < (after + 1) * NG / COPY_SLOTS; ++c) copy(c, at, here);
          // the next step's first two channel fragments: slot 0 is free, slot 1 too unless row JB of instructions reads it
          constexpr int W1_AT = JB % RING == 1 ? WTM : 2;
          if (after < 2) put(W[0], after, read(there, w_rd, after));
          if (after >= W1_AT && after < W1_AT + 2) put(W[1], after - W1_AT, read(there, w_rd + 2048, after - W1_AT));
          if (j == WTN - 1) {
            put(X[i], 0, read(there, x_rd + i * 2048, 0));  // in place: X[i] has done its last instruction of the step
            put(X[i], 1, read(there, x_rd + i * 2048, 1));
            sx[i] = sx_next[i];
          }
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    sw = sw_next;
  }
  __syncthreads();  // (no copy may land once this workgroup's shared memory is another's)

  // ---- results: acc[2 J][i], acc[2 J + 1][i] are channels nw + 32 J + 8 fq + 0 .. 3, 4 .. 7 of row i * 16 + fr
  typedef typename Elem<OUT_DT>::T T_out;
  typedef __attribute__((ext_vector_type(8))) T_out V8;
  T_out* const out = (T_out*)g.out;
  const bool wide = (g.N & 7) == 0 && (reinterpret_cast<uintptr_t>(out) & 15) == 0;
#pragma unroll
  for (int J = 0; J < WTN / 2; ++J) {
    const long n = nw + 32 * J + 8 * fq;
    float b[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) b[e] = g.bias && n + e < g.N ? g.bias[n + e] : 0.f;
#pragma unroll
    for (int i = 0; i < WTM; ++i) {
      const long m = m0 + wr * 16 * WTM + i * 16 + fr;
      if (m >= g.M) continue;
      T_out* const to = out + m * g.N + n;
      if (wide && n + 8 <= g.N) {
        V8 v;
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = (T_out)(acc[2 * J + (e >> 2)][i][e & 3] + b[e]);
        *(V8*)to = v;
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (n + e < g.N) to[e] = (T_out)(acc[2 * J + (e >> 2)][i][e & 3] + b[e]);
      }
    }
  }
}

// Any shape, operands straight from memory, a wave per 32 x 32 results; row scales as in the tiled kernel.
__device__ __forceinline__ i32x8 load_fragment(const uint8_t* row, int fq) {
  const i32x4 a = *(const i32x4*)(row + fq * 16), b = *(const i32x4*)(row + 64 + fq * 16);
  return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
}
template <int OUT_DT>
__device__ __forceinline__ void store_out(void* out, long at, float v) {
  ((typename Elem<OUT_DT>::T*)out)[at] = (typename Elem<OUT_DT>::T)v;
}
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
      sx[i] = g.xs[b * g.M + rm[i]];
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

// scale (rows, kb) -> (kb, rows)
__global__ __launch_bounds__(256) void turn_scales_kernel(const uint8_t* __restrict__ scale, uint8_t* __restrict__ turned, long rows, int kb) {
  const long count = rows * kb;
  for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < count; i += (long)gridDim.x * 256) {
    const long b = i / rows;
    turned[i] = scale[(i - b * rows) * kb + b];
  }
}

bool wide_rows(const void* p, int dt, int64_t row_stride) {  // every row starts on eight aligned elements
  const int64_t align = 8 * dt_bytes(dt) < 16 ? 8 * dt_bytes(dt) : 16;
  return (reinterpret_cast<uintptr_t>(p) % align) == 0 && (row_stride * dt_bytes(dt)) % align == 0;
}

}  // namespace

template <bool TURNED>
static hipError_t quantize_rows(const void* x, int dt, int64_t row_stride, int64_t rows, int64_t K, uint8_t* q, uint8_t* scale,
                                hipStream_t stream) {
  const int kb = (int)fp8_blocks(K);
  const bool wide = wide_rows(x, dt, row_stride);
  // four blocks a thread where that still leaves every CU eight workgroups, else one
  const int64_t bands = (rows + 15) / 16;
  const int u = bands * ((kb + 3) / 4) >= 2048 ? 4 : 1;
  const dim3 grid((unsigned)(bands * ((kb + u - 1) / u)));
#define ED_GO(DT)                                                                                                          \
  if (u == 4) ED_GO_U(DT, 4);                                                                                              \
  else ED_GO_U(DT, 1)
#define ED_GO_U(DT, U) hipLaunchKernelGGL((quantize_rows_kernel<DT, U, TURNED>), grid, dim3(256), 0, stream, x, (long)row_stride, (long)rows, kb, (long)K, wide, q, scale)
  if (dt == DT_FP32) {
    ED_GO(DT_FP32);
  } else if (dt == DT_BF16) {
    ED_GO(DT_BF16);
  } else {
    ED_GO(DT_FP16);
  }
#undef ED_GO_U
#undef ED_GO
  return hipGetLastError();
}
hipError_t launch_fp8_quantize_rows(const void* x, int dt, int64_t row_stride, int64_t rows, int64_t K, uint8_t* q,
                                    uint8_t* scale, hipStream_t stream) {
  return quantize_rows<false>(x, dt, row_stride, rows, K, q, scale, stream);
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

template <int WTM, int WTN, int OUT_DT>
static hipError_t launch_tile(const Fp8Gemm& g, hipStream_t stream) {
  const int tiles_m = (int)((g.M + 32 * WTM - 1) / (32 * WTM)), tiles_n = (int)((g.N + 32 * WTN - 1) / (32 * WTN));
  hipLaunchKernelGGL((tile_kernel<WTM, WTN, OUT_DT>), dim3((unsigned)(tiles_m * tiles_n)), dim3(256), 0, stream, g, tiles_m, tiles_n);
  return hipGetLastError();
}

template <int OUT_DT>
static hipError_t launch_gemm(const Fp8Gemm& g, hipStream_t stream) {
  if constexpr (OUT_DT != DT_FP32) {
    const int64_t big = ((g.M + 255) / 256) * ((g.N + 255) / 256);
    if (big >= 200) return launch_tile<8, 8, OUT_DT>(g, stream);
    if (g.M > 64) return launch_tile<4, 4, OUT_DT>(g, stream);
  }
  const dim3 grid((unsigned)(((g.N + 63) / 64) * ((g.M + 63) / 64)));
  hipLaunchKernelGGL((gemm_kernel<OUT_DT>), grid, dim3(256), 0, stream, g);
  return hipGetLastError();
}

// workspace: the quantised rows (a multiple of 128 bytes), then their scales, (kb, rows)
int64_t fp8_linear_workspace(int64_t M, int64_t N, int64_t K, bool quantised) {
  return M * fp8_blocks(K) * (quantised ? 1 : FP8_BLOCK + 1);
}

hipError_t launch_fp8_linear(const Fp8Linear& p, hipStream_t stream) {
  const int kb = (int)fp8_blocks(p.K);
  const uint8_t* xq = (const uint8_t*)p.x;
  uint8_t* xs = (uint8_t*)p.workspace;
  hipError_t e;
  if (p.x_dt == DT_E4M3) {
    const long blocks = (p.M * kb + 255) / 256;
    hipLaunchKernelGGL(turn_scales_kernel, dim3((unsigned)(blocks < 4096 ? blocks : 4096)), dim3(256), 0, stream, p.x_scale, xs, (long)p.M, kb);
    e = hipGetLastError();
  } else {
    uint8_t* q = (uint8_t*)p.workspace;
    xs = q + p.M * kb * FP8_BLOCK;
    e = quantize_rows<true>(p.x, p.x_dt, p.row_stride, p.M, p.K, q, xs, stream);
    xq = q;
  }
  if (e != hipSuccess) return e;
  const Fp8Gemm g{xq, xs, p.w, p.w_scale, p.bias, p.out, p.out_dt, p.M, p.N, kb};
  if (p.out_dt == DT_FP32) return launch_gemm<DT_FP32>(g, stream);
  if (p.out_dt == DT_BF16) return launch_gemm<DT_BF16>(g, stream);
  return launch_gemm<DT_FP16>(g, stream);
}

}  // namespace ed
