// Block-scaled 8-bit floating point (OCP e4m3) on gfx950: quantisation and the product.
//
// A block of 128 values - 128 channels of a row, or 128 x 128 weights - shares a scale 2^s, s the smallest whole number with
// max |x| <= 448 * 2^s (448: the largest e4m3 value).  Powers of two cost no precision in a floating format (only range at
// the small end), are exact to apply, and are what the matrix instruction takes beside its operands (E8M0 bytes): the
// product needs no vector instruction for its scales.
#include "ops.hpp"
#include "fp8_block.hpp"

#include <hip/hip_fp16.h>

#include <algorithm>
#include <cmath>

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

// Vectors that are aligned to their element alone: the memory instructions take any address, so that odd widths and strides move 16
// bytes at a time as others do (4452 x 3354 x 2092 fp16, 8-bit sums, 53 us, value by value 85).
template <typename T, int N>
struct Loose {
  typedef __attribute__((ext_vector_type(N))) T V;
  typedef V U __attribute__((aligned(sizeof(T))));
  static __device__ __forceinline__ V get(const T* p) { return *(const U*)p; }
  static __device__ __forceinline__ void put(T* p, V v) { *(U*)p = v; }
};

// Eight values of a row at column k0 (a multiple of 8): zeros behind K.
template <int DT>
__device__ __forceinline__ void load8(const typename Elem<DT>::T* row, long k0, long K, float (&v)[8]) {
  typedef typename Elem<DT>::T T;
  if (k0 + 8 <= K) {
    const auto raw = Loose<T, 8>::get(row + k0);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = (float)raw[i];
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = k0 + i < K ? (float)row[k0 + i] : 0.f;
  }
}
// 16 lanes own a block of 128, its largest magnitude found with moves inside them (no shared memory); a workgroup takes U blocks
// of 16 rows, all loads first.  Bound by HBM: 16384 x 1280 bf16 11.7 us, 5.4 TB/s in and out (a copy: 4.7).  TURNED: scales go
// to (kb, rows), as the product reads them (16 rows' bytes side by side), instead of (rows, kb).
template <int DT, int U, bool TURNED>
__global__ __launch_bounds__(256) void quantize_rows_kernel(const void* __restrict__ x, long row_stride, long rows, int kb, long K,
                                                            uint8_t* __restrict__ q, uint8_t* __restrict__ scale) {
  const int chunks = (kb + U - 1) / U;
  const long row = blockIdx.x / chunks * 16 + (threadIdx.x >> 4);
  const int b0 = (int)(blockIdx.x % chunks) * U, l = threadIdx.x & 15;
  if (row >= rows) return;
  const typename Elem<DT>::T* src = (const typename Elem<DT>::T*)x + row * row_stride;
  float v[U][8];
#pragma unroll
  for (int u = 0; u < U; ++u) load8<DT>(src, (long)(b0 + u) * FP8_BLOCK + l * 8, K, v[u]);
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int b = b0 + u;
    if (b >= kb) break;
    const unsigned a = max16(amax8(v[u]));
    const int byte = scale_byte(a);
    *(uint2*)(q + (row * kb + b) * FP8_BLOCK + l * 8) = pack8(v[u], inverse_scale(byte));
    if (l == 0) scale[TURNED ? b * rows + row : row * kb + b] = (uint8_t)byte;
  }
}

// One workgroup per 128 x 128 weights: thread (r, c) holds columns 8c .. 8c + 7 of rows r, r + 16, ..., read once and kept in
// registers while the largest magnitude goes round.  Bound by HBM: 6400 x 1280 fp32 8.1 us, 5.1 TB/s in and out.
template <int DT>
__global__ __launch_bounds__(256) void quantize_weight_kernel(const void* __restrict__ w, long row_stride, long N, int kb,
                                                              long K, uint8_t* __restrict__ q,
                                                              uint8_t* __restrict__ scale, int kb_row, int b_first) {
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
      load8<DT>((const typename Elem<DT>::T*)w + row * row_stride, (long)b * FP8_BLOCK + l * 8, K, v[i]);
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
    if (row < N) *(uint2*)(q + (row * kb_row + b_first + b) * FP8_BLOCK + l * 8) = pack8(v[i], inv);
  }
  if (threadIdx.x == 0) scale[nb * kb_row + b_first + b] = (uint8_t)byte;
}


// Eight products at a time, the 8-bit matrix instructions (scaled or not, any shape) align to the largest and drop what lies
// under 2^-13 of it: results are 4e-5 to 6e-5 (2-norm) from the exact sum at any K, and where a large product cancels against
// another group's, what stood beside it is gone.  So a product takes the exact form, whatever its output's type: e4m3 values are exact in
// bf16, so are their products in fp32, and the bf16 instruction, at half the rate, keeps fp32 sums.  The 8-bit instruction is for
// callers that ask for it: ED_FAST_SUMS, and the model at ED_PREC_FP8, whose operands' rounding (3 % a product) is far above it.
typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8;

// values 8 s2 .. 8 s2 + 7 of a fragment as bf16 (exact: the upper halves of their fp32 forms; a NaN stays one).  Four full-rate
// instructions for four values; the scaled conversion straight to bf16 takes over three times as long.
__device__ __forceinline__ bf16x8 widen(const i32x8& v, int s2) {
  typedef __attribute__((ext_vector_type(2))) float f32x2;
  i32x4 r;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8(v[2 * s2 + i], false), hi = __builtin_amdgcn_cvt_pk_f32_fp8(v[2 * s2 + i], true);
    r[2 * i] = (int)__builtin_amdgcn_perm(__float_as_uint(lo.y), __float_as_uint(lo.x), 0x07060302u);
    r[2 * i + 1] = (int)__builtin_amdgcn_perm(__float_as_uint(hi.y), __float_as_uint(hi.x), 0x07060302u);
  }
  return __builtin_bit_cast(bf16x8, r);
}
// acc += part * 2^(sx + sw - 254) (a byte of 255 is a NaN)
__device__ __forceinline__ void add_scaled(f32x4& acc, const f32x4& part, int sx, int sw) {
  const int e = sx + sw - 254;
  const bool bad = sx == 255 || sw == 255;
#pragma unroll
  for (int i = 0; i < 4; ++i) acc[i] += bad ? __builtin_nanf("") : __builtin_amdgcn_ldexpf(part[i], e);
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
// Tiled product.  WM x 2 waves (rows x channels) own a tile of 16 WM WTM rows x 32 WTN channels, a wave 16 WTM x 16 WTN as
// WTN x WTM instructions of 16 x 16 x 128: one per block of K and pair of fragments, its scales beside it.
//
// Step of K (one block): rows of 128 bytes of both operands, copied memory -> LDS into a ring of S stages, S - 1 steps ahead.
// The 16-byte chunk c of tile row r lies at chunk c ^ (r >> 1 & 7) (the copy's source addresses are permuted, its image is
// lane-linear): the 16 rows of a fragment read then fall on 16 different slots of the banks.
//
// Order inside a step.  A wave's channel fragments pass through a ring of four, its row fragments stay for the step and are
// replaced in place during the last row of instructions.  Once the last channel fragment of the step is read (row of
// instructions JB), the one barrier of the step: behind it the next stage has landed (the copies of the steps after it
// stay in flight: they are counted, not drained) and this one is free.  The rows of instructions left cover the reads
// of the next step's first fragments and the copies into the free stage, so that neither the barrier nor a read leaves the
// matrix pipe without work.  The order is pinned (sched_barrier): at most a few auxiliary instructions behind each matrix one.
//
// EXACT: the fragments are widened to bf16 and multiplied four times K = 32; a block's sums are scaled as they are added.
// A cut K loop (gridDim.y > 1) stores its part of the sums, fp32 without bias, to out + blockIdx.y * M * N.
//
// The channels of an LDS tile are permuted within 32 so that two instructions give a lane eight consecutive ones: 16-byte stores.
// ---------------------------------------------------------------------------------------------------
//
// TAPS: the rows are positions of sequences and every one is multiplied from `ntaps` of them (a dilated convolution): K runs over
// taps, then blocks; a tap moves the row operand by `dilation` rows of its padded layout, whose rows around a sequence hold
// zeros.  Taps that move a whole tile outside its sequence are left out.
//
// Measured on rows in 8 bits, ten calls in a captured graph, a call with its scales turned: 8-bit sums 8192^3 386 us, 2850 TFLOP/s (a
// library's product on the same values 402 us: the matrix pipe under that chip's clock), 16384 x 1280 x 1280 33 us, 1630 (ten steps
// of K: a third of the time is the tile's start and its stores); EXACT 1266 us, 870, and 73 us, 730: bound by its vector
// instructions, some 16 to widen (shared by a wave's tile) and a dozen to scale and add for four matrix ones.  Under a kernel trace
// the large products take a tenth longer.  A convolution of five taps, 1280 channels and 16384 positions 121 us, 2200 counting all taps.
template <int WM, int WTM, int WTN, int S, int OUT_DT, bool EXACT, bool TAPS>
__global__ __launch_bounds__(128 * WM, WM / 2) void tile_kernel(Fp8Gemm g, int tiles_m, int tiles_n) {
  constexpr int WAVES = 2 * WM, BM = 16 * WM * WTM, BN = 32 * WTN, STAGE = (BM + BN) * 128;
  constexpr int GX = BM / 8 / WAVES, GW = BN / 8 / WAVES, NG = GX + GW;  // 8-row copies a wave makes of each operand
  static_assert(GX * 8 * WAVES == BM && GW * 8 * WAVES == BN, "the copies cover the tile");
  constexpr int RING = 4, JB = WTN > 4 ? WTN - 3 : WTN > 2 ? WTN - 2 : 1;  // the barrier stands before row JB of instructions
  static_assert(JB >= WTN - RING + 1 && JB >= 1, "every channel fragment of a step is read in front of its barrier");
  // the next step's channel fragment f (0 or 1) is read once no row of instructions needs its slot: from this row on (WTN: behind the last)
  constexpr int FREE0 = (WTN - 1) / RING * RING + 1, FREE1 = (WTN - 2) / RING * RING + 2;
  constexpr int W0_AT = FREE0 > JB ? FREE0 : JB, W1_AT = FREE1 > JB ? FREE1 : JB;
  constexpr int NSW = 16 * WTN > 128 ? 2 : 1;  // blocks of channels that a wave's lie in
  static_assert((S & (S - 1)) == 0 && S >= 2, "the ring index is masked");
  __shared__ __attribute__((aligned(1024))) char lds[S * STAGE];
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
  const long m0 = (long)tile_m * BM, n0 = (long)tile_n * BN;
  const long x_pitch = (long)g.kb * FP8_BLOCK;
  const int kb_all = TAPS ? g.kb * g.ntaps : g.kb;  // blocks of a weight row
  const long w_pitch = (long)kb_all * FP8_BLOCK;
  // blocks of K of this workgroup (never none: the launcher cuts into no more pieces than there are)
  int first = (int)((long)kb_all * blockIdx.y / gridDim.y), T = (int)((long)kb_all * (blockIdx.y + 1) / gridDim.y) - first;
  // row of x that output row m reads at tap 0
  auto x_row = [&](long m) -> long {
    if constexpr (!TAPS) return m;
    const unsigned seq = (unsigned)m / (unsigned)g.L, l = (unsigned)m - seq * (unsigned)g.L;
    return (long)seq * g.x_seq_pitch + g.x_row0 + l - (long)g.center * g.dilation;
  };
  if constexpr (TAPS) {
    const int l0 = (int)(m0 % g.L);
    if (l0 + BM <= g.L) {  // the tile lies in one sequence
      int lo = 0, hi = g.ntaps - 1;
      while (lo < g.center && l0 + BM + (lo - g.center) * g.dilation <= 0) ++lo;
      while (hi > g.center && l0 + (hi - g.center) * g.dilation >= g.L) --hi;
      first = lo * g.kb;
      T = (hi - lo + 1) * g.kb;
    }
  }

  // copies: lane -> (row of 8, physical chunk)
  const int chunk0 = ((lane & 7) ^ (lane >> 4)) * 16, chunk1 = ((lane & 7) ^ (4 + (lane >> 4))) * 16;
  const long x_first = x_row(m0);
  unsigned off[NG];
#pragma unroll
  for (int j = 0; j < GX; ++j) {
    const int row = (wid * GX + j) * 8 + (lane >> 3);
    const long m = TAPS && m0 + row >= g.M ? g.M - 1 : m0 + row;
    off[j] = (unsigned)((x_row(m) - x_first) * x_pitch) + ((wid * GX + j) & 1 ? chunk1 : chunk0);
  }
#pragma unroll
  for (int j = 0; j < GW; ++j) {
    const int lr = (wid * GW + j) * 8 + (lane >> 3);
    const int ch = (lr & ~31) + 8 * ((lr & 15) >> 2) + 4 * ((lr >> 4) & 1) + (lr & 3);
    off[GX + j] = (unsigned)(ch * w_pitch) + ((wid * GW + j) & 1 ? chunk1 : chunk0);
  }
  // Where the copies stand, bytes into a row of each operand; past the last step they repeat its block (in bounds, into a
  // stage nobody reads).  The scales are read a step ahead and stand at their own place.
  const int last = T - 1;
  const unsigned first_tap = TAPS ? (unsigned)first / (unsigned)g.kb : 0, first_k = (unsigned)first - first_tap * (unsigned)g.kb;
  struct Place {
    unsigned x, w;  // of the row operand, of the weights
    int k, t;       // block of the tap, step
  };
  Place at{first_tap * (unsigned)(TAPS ? g.dilation : 0) * (unsigned)x_pitch + first_k * FP8_BLOCK, (unsigned)first * FP8_BLOCK, (int)first_k, 0};
  const unsigned x_rows = (unsigned)(TAPS ? g.x_rows : g.M);
  Place sc{first_k * x_rows + first_tap * (unsigned)(TAPS ? g.dilation : 0), (unsigned)first, (int)first_k, 0};
  auto advance = [&](Place& p, unsigned x_block, unsigned x_tap, unsigned w_block) {
    if (p.t >= last) return;
    ++p.t;
    p.w += w_block;
    if (TAPS && ++p.k == g.kb) {
      p.k = 0;
      p.x += x_tap - (unsigned)(g.kb - 1) * x_block;
    } else {
      p.x += x_block;
    }
  };
  auto advance_copies = [&]() { advance(at, FP8_BLOCK, TAPS ? (unsigned)g.dilation * (unsigned)x_pitch : 0, FP8_BLOCK); };
  auto advance_scales = [&]() { advance(sc, x_rows, TAPS ? (unsigned)g.dilation : 0, 1); };
  const buffer_t x_src = buffer_of(g.xq + x_first * x_pitch, ((long)x_rows - x_first) * x_pitch);
  const buffer_t w_src = buffer_of(g.wq + n0 * w_pitch, (g.N - n0) * w_pitch);
  auto copy = [&](int j, char* stage) {  // piece j of the step the copies stand at
    if (j < GX) copy16(x_src, off[j], at.x, stage + (wid * GX + j) * 1024);
    else copy16(w_src, off[j], at.w, stage + BM * 128 + (wid * GW + j - GX) * 1024);
  };

  // scales: a lane's row in each of the WTM fragments; the wave's channels lie in NSW blocks of 128
  unsigned sx_row[TAPS ? WTM : 1];
  if constexpr (TAPS)
#pragma unroll
    for (int i = 0; i < WTM; ++i) {
      const long m = m0 + wr * 16 * WTM + i * 16 + fr;
      sx_row[i] = (unsigned)x_row(m < g.M ? m : g.M - 1);
    }
  else
    sx_row[0] = (unsigned)(m0 + wr * 16 * WTM + fr);
  const long nw = n0 + wc * 16 * WTN;
  const buffer_t sx_src = buffer_of(g.xs, (long)x_rows * g.kb);  // (kb, rows)
  // (past the last channel the byte reads as zero, or is another block's: those channels are not stored)
  const buffer_t sw_src = buffer_of(g.ws + ((nw < g.N ? nw : g.N - 1) >> 7) * kb_all, ((g.N + 127) / 128 - ((nw < g.N ? nw : g.N - 1) >> 7)) * kb_all);
  const int in_first = (int)(128 - (nw & 127)) >> 5;  // 32-channel pairs of fragments in the first of two blocks
  auto row_scale = [&](int i) { return load_byte(sx_src, TAPS ? sx_row[TAPS ? i : 0] : sx_row[0] + i * 16, sc.x); };  // of fragment i
  auto channel_scale_byte = [&](int k) { return load_byte(sw_src, 0, sc.w + (unsigned)(k * kb_all)); };

  const int swz = (fq ^ ((fr >> 1) & 7)) << 4;
  const int x_rd = (wr * 16 * WTM + fr) * 128, w_rd = BM * 128 + (wc * 16 * WTN + fr) * 128;
  auto read = [&](const char* stage, int base, int half) { return *(const i32x4*)(stage + base + ((half << 6) ^ swz)); };
  auto put = [](i32x8& f, int half, i32x4 v) {
    if (half == 0) { f[0] = v[0]; f[1] = v[1]; f[2] = v[2]; f[3] = v[3]; }
    else { f[4] = v[0]; f[5] = v[1]; f[6] = v[2]; f[7] = v[3]; }
  };

  f32x4 acc[WTN][WTM] = {};
  i32x8 X[WTM], W[RING];
  bf16x8 XW[EXACT ? WTM : 1][4], WW[4];
  f32x4 part[2];
  int sx_now[WTM];
  int sx[WTM], sx_next[WTM], sw[NSW], sw_next[NSW];
  auto channel_scale = [&](int j) { return NSW == 1 || (j >> 1) < in_first ? sw[0] : sw[NSW - 1]; };

  // step 0 and its first fragments, copies of the S - 1 steps behind it
#pragma unroll
  for (int j = 0; j < NG; ++j) copy(j, lds);
#pragma unroll
  for (int i = 0; i < WTM; ++i) sx[i] = row_scale(i);
#pragma unroll
  for (int k = 0; k < NSW; ++k) sw[k] = channel_scale_byte(k);
  asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" ::: "memory");
#pragma unroll
  for (int k = 1; k < S; ++k) {
    advance_copies();
#pragma unroll
    for (int j = 0; j < NG; ++j) copy(j, lds + k * STAGE);
  }
#pragma unroll
  for (int i = 0; i < WTM; ++i) { put(X[i], 0, read(lds, x_rd + i * 2048, 0)); put(X[i], 1, read(lds, x_rd + i * 2048, 1)); }
#pragma unroll
  for (int j = 0; j < 2; ++j) { put(W[j], 0, read(lds, w_rd + j * 2048, 0)); put(W[j], 1, read(lds, w_rd + j * 2048, 1)); }

  for (int t = 0; t < T; ++t) {
    char* const here = lds + (t & (S - 1)) * STAGE;
    const char* const there = lds + ((t + 1) & (S - 1)) * STAGE;
    advance_copies();
    advance_scales();
    if constexpr (EXACT)
#pragma unroll
      for (int i = 0; i < WTM; ++i) sx_now[i] = sx[i];  // (sx becomes the next step's during the last row of instructions)
#pragma unroll
    for (int j = 0; j < WTN; ++j) {
      if (j == JB) {
        // Behind the copies of step t + 1 at least those of S - 2 steps and this step's scale loads were issued: with no more
        // than that many outstanding they have landed.  This wave's reads of the stage are in registers.
        __builtin_amdgcn_sched_barrier(0);
        constexpr int OUT = (S - 2) * NG + WTM + NSW;
        static_assert(OUT < 64, "the counter has six bits");
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(OUT) : "memory");
        __builtin_amdgcn_sched_barrier(0);
      }
#pragma unroll
      for (int i = 0; i < WTM; ++i) {
        if constexpr (EXACT) {
          if (i == 0)
#pragma unroll
            for (int h = 0; h < 4; ++h) WW[h] = widen(W[j % RING], h);
          if (j == 0)
#pragma unroll
            for (int h = 0; h < 4; ++h) XW[i][h] = widen(X[i], h);
          // this block's sums from zero; they are scaled and added under the next fragments' instructions
          f32x4& now = part[(j * WTM + i) & 1];
          now = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int h = 0; h < 4; ++h) now = __builtin_amdgcn_mfma_f32_16x16x32_bf16(WW[h], XW[i][h], now, 0, 0, 0);
          if (j * WTM + i > 0) {
            const int before = j * WTM + i - 1;
            add_scaled(acc[before / WTM][before % WTM], part[before & 1], sx_now[before % WTM], channel_scale(before / WTM));
          }
        } else {
          acc[j][i] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(W[j % RING], X[i], acc[j][i], 0, 0, 0, channel_scale(j), 0, sx[i]);
        }
        const int slot = j * WTM + i;
        if (j < JB) {
          // channel fragments 2 .. WTN - 1, two reads each, as soon as their slot of the ring is free
#pragma unroll
          for (int r = 0; r < 2 * (WTN - 2); ++r) {
            const int f = 2 + r / 2, want = f < RING ? (r < JB * WTM ? r : JB * WTM - 1) : (f - RING + 1) * WTM + (r & 1);
            if (want == slot) put(W[f % RING], r & 1, read(here, w_rd + f * 2048, r & 1));
          }
          constexpr int AT = JB * WTM >= 4 + WTM ? 4 : 0;  // the next step's scales
          if (slot >= AT && slot < AT + WTM) sx_next[slot - AT] = row_scale(slot - AT);
          if (slot == AT)
#pragma unroll
            for (int k = 0; k < NSW; ++k) sw_next[k] = channel_scale_byte(k);
        } else {
          constexpr int COPY_SLOTS = (WTN - JB) * WTM;
          const int after = slot - JB * WTM;
#pragma unroll
          for (int c = after * NG / COPY_SLOTS; c < (after + 1) * NG / COPY_SLOTS; ++c) copy(c, here);
          const int from0 = slot - W0_AT * WTM, from1 = slot - W1_AT * WTM - (W1_AT == W0_AT ? 2 : 0);
          if (from0 == 0 || from0 == 1) put(W[0], from0, read(there, w_rd, from0));
          if (from1 == 0 || from1 == 1) put(W[1], from1, read(there, w_rd + 2048, from1));
          if (j == WTN - 1) {
            put(X[i], 0, read(there, x_rd + i * 2048, 0));  // in place: X[i] has done its last instruction of the step
            put(X[i], 1, read(there, x_rd + i * 2048, 1));
            sx[i] = sx_next[i];
            if (W1_AT == WTN && i == WTM - 1) {
              put(W[1], 0, read(there, w_rd + 2048, 0));
              put(W[1], 1, read(there, w_rd + 2048, 1));
            }
          }
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    if constexpr (EXACT) add_scaled(acc[WTN - 1][WTM - 1], part[(WTN * WTM - 1) & 1], sx_now[WTM - 1], channel_scale(WTN - 1));
#pragma unroll
    for (int k = 0; k < NSW; ++k) sw[k] = sw_next[k];
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // (no copy may land once this workgroup's shared memory is another's)

  // ---- results: acc[2 J][i], acc[2 J + 1][i] are channels nw + 32 J + 8 fq + 0 .. 3, 4 .. 7 of row i * 16 + fr
  typedef typename Elem<OUT_DT>::T T_out;
  T_out* const out = (T_out*)g.out + (gridDim.y > 1 ? (long)blockIdx.y * g.M * g.N : 0);
  const buffer_t bias = buffer_of((const uint8_t*)g.bias, g.bias ? g.N * 4 : 0);  // (reads as zero behind its end)
  f32x4 b[WTN];
#pragma unroll
  for (int j = 0; j < WTN; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e)
      b[j][e] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(bias, (int)((nw + 32 * (j >> 1) + 8 * fq + 4 * (j & 1) + e) * 4), 0, 0));
#pragma unroll
  for (int i = 0; i < WTM; ++i) {
    const long m = m0 + wr * 16 * WTM + i * 16 + fr;
    if (m >= g.M) continue;
#pragma unroll
    for (int J = 0; J < WTN / 2; ++J) {
      const long n = nw + 32 * J + 8 * fq;
      T_out* const to = out + m * g.N + n;
      if constexpr (OUT_DT == DT_FP32 && !EXACT)
        if (g.resid) {  // (may be the output: a lane reads what it writes)
          const float* const from = g.resid + m * g.N + n;
          if (n + 8 <= g.N) {
            acc[2 * J][i] += Loose<float, 4>::get(from);
            acc[2 * J + 1][i] += Loose<float, 4>::get(from + 4);
          } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
              if (n + e < g.N) acc[2 * J + (e >> 2)][i][e & 3] += from[e];
          }
        }
      if (n + 8 <= g.N) {
        typename Loose<T_out, 8>::V v;
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = (T_out)(acc[2 * J + (e >> 2)][i][e & 3] + b[2 * J + (e >> 2)][e & 3]);
        Loose<T_out, 8>::put(to, v);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (n + e < g.N) to[e] = (T_out)(acc[2 * J + (e >> 2)][i][e & 3] + b[2 * J + (e >> 2)][e & 3]);
      }
    }
  }
}

// ---------------------------------------------------------------------------------------------------
// Few rows (up to 16: the weights are streamed once and bound the time), or little work: latency bounds it.  A workgroup owns
// 16 rows and 16 NF channels, its waves share the blocks of K (wave w: w, w + waves, ...): a wave reads a block's weights as fragments straight from memory, the next
// block's in flight, and brings plain rows to 8 bits in registers - the four lanes that hold a row's block find its
// largest magnitude with two exchanges.  The waves' sums meet in shared memory, in order.
// Measured, calls in a captured graph, exact (8-bit sums): 8 x 8192 x 8192 on rows in 8 bits 18.2 us (17.7), 67 MB of weights at 3.7 TB/s (a
// copy: 4.7; the start and the join of a single round of workgroups are the rest); 1 x 1280 x 1280 5.0 us (4.7), where a launch
// alone takes 2 to 3.
// ---------------------------------------------------------------------------------------------------
// 32 values of a row: columns k0 .. k0 + 15 and k0 + 64 .. k0 + 79, zeros behind K
template <int DT>
struct RowPart {
  float v[4][8];
  __device__ __forceinline__ void load(const void* x, long row_at, long k0, long K, bool on) {
    typedef typename Elem<DT>::T T;
    const T* row = (const T*)x + row_at;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (on) load8<DT>(row, k0 + (i >> 1) * 64 + (i & 1) * 8, K, v[i]);
      else
#pragma unroll
        for (int e = 0; e < 8; ++e) v[i][e] = 0.f;
    }
  }
  __device__ __forceinline__ int quantise(i32x8& f) {  // -> scale byte
    unsigned a = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const unsigned c = amax8(v[i]);
      a = c > a ? c : a;
    }
#pragma unroll
    for (int o = 16; o < 64; o <<= 1) {
      const unsigned c = (unsigned)__shfl_xor((int)a, o);
      a = c > a ? c : a;
    }
    const int byte = scale_byte(a);
    const float inv = inverse_scale(byte);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint2 p = pack8(v[i], inv);
      f[2 * i] = (int)p.x;
      f[2 * i + 1] = (int)p.y;
    }
    return byte;
  }
};

struct FewRows {
  const void* x;
  long row_stride, K;
  const uint8_t* x_scale;  // x in 8 bits only: (M, kb)
};

template <int DT, bool EXACT, int NF>
__global__ __launch_bounds__(1024) void few_rows_kernel(Fp8Gemm g, FewRows r) {
  __shared__ f32x4 sums[16][NF][64];
  const int tid = threadIdx.x, lane = tid & 63, wid = __builtin_amdgcn_readfirstlane(tid >> 6), waves = (int)blockDim.x >> 6;
  const int fr = lane & 15, fq = lane >> 4;
  const long n0 = (long)blockIdx.x * 16 * NF, m = (long)blockIdx.y * 16 + fr, pitch = (long)g.kb * FP8_BLOCK;
  // (channels and rows past the end repeat one that is there, unstored)
  const bool on = m < g.M;
  const long mf = on ? m : g.M - 1;
  const uint8_t *w_row[NF], *ws_row[NF];
  f32x4 acc[NF];
  i32x4 w_next[NF][2];
  int sw_next[NF];
#pragma unroll
  for (int f = 0; f < NF; ++f) {
    const long n = n0 + 16 * f + fr, nf = n < g.N ? n : g.N - 1;
    w_row[f] = g.wq + nf * pitch + fq * 16;
    ws_row[f] = g.ws + (nf >> 7) * g.kb;
    acc[f] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  auto fetch = [&](int b) {
    if (b >= g.kb) return;
#pragma unroll
    for (int f = 0; f < NF; ++f) {
      w_next[f][0] = *(const i32x4*)(w_row[f] + (long)b * FP8_BLOCK);
      w_next[f][1] = *(const i32x4*)(w_row[f] + (long)b * FP8_BLOCK + 64);
      sw_next[f] = ws_row[f][b];
    }
  };
  fetch(wid);
  for (int b = wid; b < g.kb; b += waves) {
    i32x8 X;
    int sx;
    if constexpr (DT == DT_E4M3) {
      const uint8_t* q = (const uint8_t*)r.x + mf * pitch + (long)b * FP8_BLOCK + fq * 16;
      X = __builtin_shufflevector(*(const i32x4*)q, *(const i32x4*)(q + 64), 0, 1, 2, 3, 4, 5, 6, 7);
      sx = r.x_scale[mf * g.kb + b];
    } else {
      RowPart<DT> part;
      part.load(r.x, mf * r.row_stride, (long)b * FP8_BLOCK + fq * 16, r.K, on);
      sx = part.quantise(X);
    }
    i32x8 W[NF];
    int sw[NF];
#pragma unroll
    for (int f = 0; f < NF; ++f) {
      W[f] = __builtin_shufflevector(w_next[f][0], w_next[f][1], 0, 1, 2, 3, 4, 5, 6, 7);
      sw[f] = sw_next[f];
    }
    fetch(b + waves);
#pragma unroll
    for (int f = 0; f < NF; ++f) {
      if constexpr (EXACT) {
        f32x4 part = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int h = 0; h < 4; ++h) part = __builtin_amdgcn_mfma_f32_16x16x32_bf16(widen(W[f], h), widen(X, h), part, 0, 0, 0);
        add_scaled(acc[f], part, sx, sw[f]);
      } else {
        acc[f] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(W[f], X, acc[f], 0, 0, 0, sw[f], 0, sx);
      }
    }
  }
#pragma unroll
  for (int f = 0; f < NF; ++f) sums[wid][f][lane] = acc[f];
  __syncthreads();
  for (int j = wid; j < NF; j += waves) {  // wave j joins fragment j
    if (!on) break;
    f32x4 y = sums[0][j][lane];
    for (int w = 1; w < waves; ++w) y += sums[w][j][lane];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const long n = n0 + 16 * j + fq * 4 + e;
      if (n >= g.N) break;
      const float v = y[e] + (g.bias ? g.bias[n] : 0.f);
      const long o = m * g.N + n;
      if (g.out_dt == DT_FP32) ((float*)g.out)[o] = v;
      else if (g.out_dt == DT_BF16) ((__bf16*)g.out)[o] = (__bf16)v;
      else ((_Float16*)g.out)[o] = (_Float16)v;
    }
  }
}

// out = bias + the parts of a cut K loop, added in order; four values a thread (bound by the parts' way through memory)
template <int OUT_DT>
__global__ __launch_bounds__(256) void join_kernel(const float* __restrict__ part, int parts, const float* __restrict__ bias,
                                                   void* __restrict__ out, long M, long N) {
  typedef typename Elem<OUT_DT>::T T_out;
  const long count = M * N;
  for (long i = ((long)blockIdx.x * 256 + threadIdx.x) * 4; i < count; i += (long)gridDim.x * 1024) {
    float v[4] = {0.f, 0.f, 0.f, 0.f};
    if (i + 4 <= count && (count & 3) == 0) {
#pragma unroll 4
      for (int z = 0; z < parts; ++z) {
        const f32x4 p = *(const f32x4*)(part + z * count + i);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] += p[e];
      }
    } else {
      for (int z = 0; z < parts; ++z)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (i + e < count) v[e] += part[z * count + i + e];
    }
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (i + e < count) ((T_out*)out)[i + e] = (T_out)(v[e] + (bias ? bias[(i + e) % N] : 0.f));
  }
}

// scale (rows, kb) -> (kb, rows): a hundredth of the product's bytes, once per call on rows that were quantised before
__global__ __launch_bounds__(256) void turn_scales_kernel(const uint8_t* __restrict__ scale, uint8_t* __restrict__ turned, long rows, int kb) {
  const long count = rows * kb;
  for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < count; i += (long)gridDim.x * 256) {
    const long b = i / rows;
    turned[i] = scale[(i - b * rows) * kb + b];
  }
}

}  // namespace

template <bool TURNED>
static hipError_t quantize_rows(const void* x, int dt, int64_t row_stride, int64_t rows, int64_t K, uint8_t* q, uint8_t* scale,
                                hipStream_t stream) {
  const int kb = (int)fp8_blocks(K);
  // four blocks a thread where that still leaves every CU eight workgroups, else one
  const int64_t bands = (rows + 15) / 16;
  const int u = bands * ((kb + 3) / 4) >= 2048 ? 4 : 1;
  const dim3 grid((unsigned)(bands * ((kb + u - 1) / u)));
#define ED_GO(DT)                                                                                                          \
  if (u == 4) ED_GO_U(DT, 4);                                                                                              \
  else ED_GO_U(DT, 1)
#define ED_GO_U(DT, U) hipLaunchKernelGGL((quantize_rows_kernel<DT, U, TURNED>), grid, dim3(256), 0, stream, x, (long)row_stride, (long)rows, kb, (long)K, q, scale)
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
                                      uint8_t* scale, hipStream_t stream, int kb_row, int b_first) {
  const int kb = (int)fp8_blocks(K);
  if (kb_row == 0) kb_row = kb;
  const dim3 grid((unsigned)(fp8_blocks(N) * kb));
#define ED_GO(DT) hipLaunchKernelGGL((quantize_weight_kernel<DT>), grid, dim3(256), 0, stream, w, (long)row_stride, (long)N, kb, (long)K, q, scale, kb_row, b_first)
  if (dt == DT_FP32) ED_GO(DT_FP32);
  else if (dt == DT_BF16) ED_GO(DT_BF16);
  else ED_GO(DT_FP16);
#undef ED_GO
  return hipGetLastError();
}

// How a product is cut: tiles of 32 `size` x 32 `size` (10: 256 x 320), and the pieces of its K loop.
struct Plan {
  int size, parts;
};
// The cheapest by what was measured of the tiles (microseconds).  A step of K takes a tile no less than `step` alone on its CU (its
// latency), all tiles at work together no less than their copies take at 16 GB/ms of L2 and their products at `rate`; a round of
// tiles has 2 to 3 us of start and end, and its results to write.  A cut K loop adds a launch and its sums' way through
// memory.  Sides measured with 8-bit sums: 16384 x 1280 x 1280 tiles of 256 x 320 34 us, 256 x 256 47, 128 x 128 41; 4096^3 67, 55 and 69; 512 x 8192 x 8192 128-tiles
// 46, 64-tiles 59; 1024 x 1280 x 1280 12.1 and 11.2; 128 x 8192 x 8192 64-tiles whole 28.6, K cut in two 25.5 - there the cost errs: it
// says 19.0 and 26.5, and takes the first.  What the exact form takes and the cost says: 32 x 8192 x 8192 27.5 (20), 128 rows 44 (34), 512
// rows 133 (102), 16384 x 1280 x 1280 73 (88), 8192^3 1266 (1510).
static Plan plan_of(int64_t M, int64_t N, int kb, bool exact, bool whole_k = false) {
  struct Kind {
    int size, bm, bn, resident;
    double step;
  };
  static const Kind fast[4] = {{10, 256, 320, 1, 1.3}, {8, 256, 256, 1, 1.1}, {4, 128, 128, 2, 0.6}, {2, 64, 64, 2, 0.24}},
                    wide[2] = {{4, 128, 128, 2, 1.55}, {2, 64, 64, 2, 0.75}};
  const double rate = exact ? 0.75e9 : 2.6e9, l2 = 16e6, hbm = 4.5e6;  // per microsecond
  Plan best{2, 1};
  double least = 1e30;
  for (int k = 0; k < (exact ? 2 : 4); ++k) {
    const Kind& t = exact ? wide[k] : fast[k];
    const double area = (double)t.bm * t.bn, slots = 256.0 * t.resident;
    const double whole = (double)((M + t.bm - 1) / t.bm) * (double)((N + t.bn - 1) / t.bn);
    for (int parts = 1; parts <= 16; parts *= 2) {
      if (parts > 1 && (whole_k || kb < 4 * parts || whole * parts > 1024)) break;
      const double work = whole * parts, steps = (double)((kb + parts - 1) / parts);
      auto round = [&](double n) {
        if (n <= 0) return 0.0;
        const double step = std::max({t.step, n * (t.bm + t.bn) * 128 / l2, n * area * 256 / rate});
        return steps * step + (t.resident > 1 ? 2.0 : 3.0) + n * area * (parts > 1 || exact ? 4 : 2) / hbm / t.resident;
      };
      const double full = std::floor(work / slots);
      double cost = full * round(slots) + round(work - full * slots);
      if (parts > 1) cost += 4.0 + (double)M * N * (4.0 * parts + 4) / hbm;
      if (cost < least) {
        least = cost;
        best = Plan{t.size, parts};
      }
    }
  }
  return best;
}

template <int WM, int WTM, int WTN, int S, int OUT_DT, bool EXACT, bool TAPS = false>
static hipError_t launch_tile(const Fp8Gemm& g, int parts, hipStream_t stream) {
  const int tiles_m = (int)((g.M + 16 * WM * WTM - 1) / (16 * WM * WTM)), tiles_n = (int)((g.N + 32 * WTN - 1) / (32 * WTN));
  hipLaunchKernelGGL((tile_kernel<WM, WTM, WTN, S, OUT_DT, EXACT, TAPS>), dim3((unsigned)(tiles_m * tiles_n), (unsigned)parts), dim3(128 * WM), 0,
                     stream, g, tiles_m, tiles_n);
  return hipGetLastError();
}

template <int OUT_DT, bool EXACT>
static hipError_t launch_plan(const Fp8Gemm& g, const Plan& p, hipStream_t stream) {
  if constexpr (!EXACT) {
    if (p.size == 10) return launch_tile<4, 4, 10, 2, OUT_DT, EXACT>(g, p.parts, stream);
    if (p.size == 8) return launch_tile<2, 8, 8, 2, OUT_DT, EXACT>(g, p.parts, stream);
  }
  if (p.size == 4) return launch_tile<2, 4, 4, 2, OUT_DT, EXACT>(g, p.parts, stream);
  return launch_tile<2, 2, 2, 4, OUT_DT, EXACT>(g, p.parts, stream);
}

// The few-rows kernel takes up to 16 rows always, and more where 16 x 16 outputs by 128 channels make no more than FEW_WORK pieces
// and a wave no more than four steps: one launch, no wait between the steps of K.  Sides measured (us, rows already in 8 bits, 8-bit
// and exact sums; the tiles need the scales turned first): 64 x 1280 x 1280 6.8 and 6.4, tiles 10.6 and 13.3; 300 x 1111 x 1000
// (10640 pieces) 8.4 and 9.1, tiles 10.6 and 13.4; plain rows there 11.2 and 11.7, tiles 10.6 and 13.8; 1024 x 640 x 640 (12800) 12.4
// and 13.1, tiles 10.3 and 10.4.  One limit for both sums, by the exact ones (plain rows with 8-bit sums would turn a little sooner).
constexpr int FEW_ROWS = 16, FEW_WORK = 11000, FEW_K = 64;
static int64_t few_work(int64_t M, int64_t N, int64_t kb) { return ((M + 15) / 16) * ((N + 15) / 16) * kb; }
static bool few_rows(int64_t M, int64_t N, int64_t kb) { return M <= FEW_ROWS || (kb <= FEW_K && few_work(M, N, kb) <= FEW_WORK); }
// Plain rows are brought to 8 bits inside that kernel (every workgroup does it again) up to this many blocks of K (8 x 2560 x 2560
// 7.6 us against 10.3 with a launch of its own, 4 x 5120 x 5120 16.6 against 12.3) and, beyond 16 rows, pieces (8-bit and exact sums: 4096 x
// 31 x 1280, 5120 pieces, 6.6 and 6.7 against 10.0 and 10.4; 128 x 640 x 2560, 6400 pieces, 7.8 and 10.3 against 10.2 and 10.4;
// 300 x 1111 x 1000, 10640 pieces, 10.0 and 11.2 against 10.4 and 11.0).
constexpr int FEW_BLOCKS = 24, FEW_INSIDE = 8000;
static bool quantised_inside(int64_t M, int64_t N, int64_t kb) {
  return kb <= FEW_BLOCKS && (M <= FEW_ROWS || few_work(M, N, kb) <= FEW_INSIDE);
}

template <int DT, int NF>
static hipError_t launch_few(const Fp8Gemm& g, const FewRows& r, bool exact, hipStream_t stream) {
  const dim3 grid((unsigned)((g.N + 16 * NF - 1) / (16 * NF)), (unsigned)((g.M + 15) / 16));
  const dim3 block(64 * (g.kb < 16 ? g.kb : 16));  // (no wave without a block of K)
  if (exact) hipLaunchKernelGGL((few_rows_kernel<DT, true, NF>), grid, block, 0, stream, g, r);
  else hipLaunchKernelGGL((few_rows_kernel<DT, false, NF>), grid, block, 0, stream, g, r);
  return hipGetLastError();
}
// 16 channels a workgroup, so that as many as there can be read the weights (8 x 8192 x 8192 17.7 us against 18.5 with 32); 32 where
// more than 16 rows are brought to 8 bits inside, which each workgroup does (128 x 1280 x 1280 8.6 us against 9.5).
template <int DT>
static hipError_t launch_few_rows(const Fp8Gemm& g, const FewRows& r, bool exact, hipStream_t stream) {
  if constexpr (DT != DT_E4M3)
    if (g.M > FEW_ROWS) return launch_few<DT, 2>(g, r, exact, stream);
  return launch_few<DT, 1>(g, r, exact, stream);
}

template <int OUT_DT, bool EXACT>
static hipError_t launch_gemm(const Fp8Gemm& g, void* partial, hipStream_t stream) {
  const Plan p = plan_of(g.M, g.N, g.kb, EXACT);
  if (p.parts == 1) return launch_plan<OUT_DT, EXACT>(g, p, stream);
  Fp8Gemm part = g;
  part.out = partial;
  part.bias = nullptr;
  const hipError_t e = launch_plan<DT_FP32, EXACT>(part, p, stream);
  if (e != hipSuccess) return e;
  const long blocks = (g.M * g.N + 1023) / 1024;
  hipLaunchKernelGGL((join_kernel<OUT_DT>), dim3((unsigned)(blocks < 4096 ? blocks : 4096)), dim3(256), 0, stream, (const float*)partial,
                     p.parts, g.bias, g.out, (long)g.M, (long)g.N);
  return hipGetLastError();
}

hipError_t launch_fp8_gemm(const Fp8Gemm& g, hipStream_t stream) {
  const Plan p = plan_of(g.M, g.N, g.kb * g.ntaps, false, true);
  if (g.ntaps > 1) {
    if (g.out_dt != DT_BF16 || g.resid) return hipErrorInvalidValue;
    if (p.size == 10) return launch_tile<4, 4, 10, 2, DT_BF16, false, true>(g, 1, stream);
    if (p.size == 8) return launch_tile<2, 8, 8, 2, DT_BF16, false, true>(g, 1, stream);
    if (p.size == 4) return launch_tile<2, 4, 4, 2, DT_BF16, false, true>(g, 1, stream);
    return launch_tile<2, 2, 2, 4, DT_BF16, false, true>(g, 1, stream);
  }
  if (g.out_dt == DT_BF16) return g.resid ? hipErrorInvalidValue : launch_plan<DT_BF16, false>(g, p, stream);
  return g.out_dt == DT_FP32 ? launch_plan<DT_FP32, false>(g, p, stream) : hipErrorInvalidValue;
}

// workspace: the quantised rows (a multiple of 128 bytes), their scales, (kb, rows), up to 16 bytes, then the parts of a cut K loop
static int64_t scales_end(int64_t M, int64_t kb, bool quantised) {
  return (M * kb * (quantised ? 1 : FP8_BLOCK + 1) + 15) / 16 * 16;
}
int64_t fp8_linear_workspace(int64_t M, int64_t N, int64_t K, bool quantised, bool exact) {
  const int64_t kb = fp8_blocks(K);
  if (few_rows(M, N, kb)) return quantised || quantised_inside(M, N, kb) ? 0 : M * kb * (FP8_BLOCK + 1);
  const Plan p = plan_of(M, N, (int)kb, exact);
  return scales_end(M, kb, quantised) + (p.parts > 1 ? p.parts * M * N * 4 : 0);
}

hipError_t launch_fp8_linear(const Fp8Linear& p, hipStream_t stream) {
  const int kb = (int)fp8_blocks(p.K);
  const bool exact = !p.fast;
  if (few_rows(p.M, p.N, kb)) {
    const Fp8Gemm g{nullptr, nullptr, p.w, p.w_scale, p.bias, p.out, p.out_dt, p.M, p.N, kb};
    FewRows r{p.x, (long)p.row_stride, (long)p.K, p.x_scale};
    if (p.x_dt != DT_E4M3) {
      if (quantised_inside(p.M, p.N, kb)) {
        if (p.x_dt == DT_FP32) return launch_few_rows<DT_FP32>(g, r, exact, stream);
        if (p.x_dt == DT_BF16) return launch_few_rows<DT_BF16>(g, r, exact, stream);
        return launch_few_rows<DT_FP16>(g, r, exact, stream);
      }
      uint8_t* const q = (uint8_t*)p.workspace;
      uint8_t* const scale = q + p.M * kb * FP8_BLOCK;
      const hipError_t e = quantize_rows<false>(p.x, p.x_dt, p.row_stride, p.M, p.K, q, scale, stream);
      if (e != hipSuccess) return e;
      r.x = q;
      r.x_scale = scale;
    }
    return launch_few_rows<DT_E4M3>(g, r, exact, stream);
  }
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
  void* const partial = (char*)p.workspace + scales_end(p.M, kb, p.x_dt == DT_E4M3);
  if (p.out_dt == DT_FP32) return exact ? launch_gemm<DT_FP32, true>(g, partial, stream) : hipErrorInvalidValue;
  if (p.out_dt == DT_BF16) return exact ? launch_gemm<DT_BF16, true>(g, partial, stream) : launch_gemm<DT_BF16, false>(g, partial, stream);
  return exact ? launch_gemm<DT_FP16, true>(g, partial, stream) : launch_gemm<DT_FP16, false>(g, partial, stream);
}

}  // namespace ed
