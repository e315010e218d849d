// Internal launcher interface of the model-free operators (fp8.hip, logprobs.hip): block-scaled 8-bit quantisation, the
// product on it, and log probabilities of given tokens.  As in kernels.hpp: asynchronous on `stream`, nothing allocated,
// nothing synchronised, so a caller may capture them; the C-ABI layer (api.hip) has checked every argument.
#pragma once
#include "kernels.hpp"

namespace ed {

enum { DT_FP32 = 0, DT_BF16 = 1, DT_FP16 = 2 };  // = ED_DT_* of the C ABI
inline int dt_bytes(int dt) { return dt == DT_FP32 ? 4 : 2; }

constexpr int FP8_BLOCK = 128;  // values that share a scale (and the K of one matrix instruction)
inline int64_t fp8_blocks(int64_t k) { return (k + FP8_BLOCK - 1) / FP8_BLOCK; }

// x (rows, K) -> q (rows, Kb * 128) e4m3 bytes, zeros behind K, and scale (rows, Kb) E8M0 bytes; row_stride in elements.
hipError_t launch_fp8_quantize_rows(const void* x, int dt, int64_t row_stride, int64_t rows, int64_t K, uint8_t* q,
                                    uint8_t* scale, hipStream_t stream);
// w (N, K) -> q (N, Kb * 128) and scale (ceil(N / 128), Kb): one scale for 128 x 128 weights
// (kb_row > 0: into rows of kb_row blocks, from block b_first on - the taps of a convolution side by side)
hipError_t launch_fp8_quantize_weight(const void* w, int dt, int64_t row_stride, int64_t N, int64_t K, uint8_t* q,
                                      uint8_t* scale, hipStream_t stream, int kb_row = 0, int b_first = 0);
// zeros, by a kernel (bytes: a multiple of 16)
hipError_t launch_clear(void* p, size_t bytes, hipStream_t stream);
// q, scale (kb, q_rows) <- act(LayerNorm(in)) in 8 bits: row r of `in` (fp32 or bf16, C channels) goes to row
// (r / L) * seq_pitch + row0 + r % L.  act: 1 GELU (the bf16 path's fit), 2 ReLU.
hipError_t launch_ln_act_fp8(const void* in, bool in_bf16, const float* gamma, const float* beta, int rows, int C, int act, uint8_t* q,
                             uint8_t* scale, long q_rows, int L, long seq_pitch, long row0, hipStream_t stream);

// out[m][n] = bias[n] + sum_b 2^(xs[b][m] + ws[n / 128][b] - 254) sum_{k in block b} xq[m][k] * wq[n][k]
struct Fp8Gemm {
  const uint8_t *xq, *xs;  // (M, Kb * 128), (Kb, M)
  const uint8_t *wq, *ws;  // (N, Kb * 128), (ceil(N / 128), Kb)
  const float* bias;       // nullptr or [N]
  void* out;               // (M, N) of type out_dt
  int out_dt;
  int64_t M, N;
  int kb;                  // blocks along K (of one tap)
  const float* resid = nullptr;  // fp32 (M, N) added to an fp32 result (may be out)
  // A dilated convolution (ntaps > 1): output row m = (sequence, l) = (m / L, m % L) reads rows sequence * x_seq_pitch + x_row0 + l +
  // (tap - center) * dilation of the x_rows rows of x, and weight rows hold ntaps * kb blocks, tap by tap.
  int ntaps = 1, dilation = 1, center = 0, L = 1;
  long x_seq_pitch = 0, x_row0 = 0, x_rows = 0;
};
// Without a workspace (K whole): bf16 results, fp32 results with or without a residual (rounded as the 8-bit instruction does),
// bf16 results of a convolution.
hipError_t launch_fp8_gemm(const Fp8Gemm& g, hipStream_t stream);

// The product on plain or quantised rows (x_dt DT_E4M3: x_scale is read, row_stride is Kb * 128).
enum { DT_E4M3 = 3 };  // = ED_DT_E4M3
struct Fp8Linear {
  const void* x;
  int x_dt;
  int64_t row_stride;
  const uint8_t* x_scale;
  const uint8_t *w, *w_scale;
  const float* bias;
  void* out;
  int out_dt;
  int64_t M, N, K;
  void* workspace;  // fp8_linear_workspace bytes, 16-byte aligned
  bool fast;        // sums as the 8-bit instruction takes them (16-bit outputs only), else fp32
};
int64_t fp8_linear_workspace(int64_t M, int64_t N, int64_t K, bool quantised, bool exact);  // exact: not fast
hipError_t launch_fp8_linear(const Fp8Linear& p, hipStream_t stream);

// Rows of logits: row r = (o, i) = (r / inner, r % inner) starts at o * outer_stride + i * inner_stride (elements).
struct LogitsView {
  const void* p;
  int dt;
  int64_t rows, inner, inner_stride, outer_stride;
  int n;  // classes
};
struct LogprobsOut {
  float *logprob, *entropy;  // [rows]
  float* stats;              // [rows][2]: the row's maximum and log sum exp(x - max); may be nullptr
  float* top_logprob;        // [rows][top_k]
  int64_t* top_token;        // [rows][top_k]
};
int64_t token_logprobs_workspace(int64_t rows, int64_t n, int top_k);
hipError_t launch_token_logprobs(const LogitsView& x, const int64_t* targets, const uint8_t* select, int top_k,
                                 const LogprobsOut& out, void* workspace, hipStream_t stream);
struct LogprobsGrad {
  const float *stats, *entropy;   // as the forward wrote them
  const int64_t* top_token;       // [rows][top_k]
  const float *g_logprob, *g_entropy, *g_top;  // nullptr = zero
  void* dlogits;                  // (rows, columns) of the logits' type, contiguous; columns >= n get zeros
  int64_t columns;
};
hipError_t launch_token_logprobs_backward(const LogitsView& x, const int64_t* targets, const uint8_t* select, int top_k,
                                          const LogprobsGrad& g, hipStream_t stream);

}  // namespace ed
