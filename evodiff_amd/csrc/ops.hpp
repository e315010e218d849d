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
hipError_t launch_fp8_quantize_weight(const void* w, int dt, int64_t row_stride, int64_t N, int64_t K, uint8_t* q,
                                      uint8_t* scale, hipStream_t stream);

// out[m][n] = bias[n] + sum_b 2^(xs[b][m] + ws[n / 128][b] - 254) sum_{k in block b} xq[m][k] * wq[n][k]
struct Fp8Gemm {
  const uint8_t *xq, *xs;  // (M, Kb * 128), (Kb, M)
  const uint8_t *wq, *ws;  // (N, Kb * 128), (ceil(N / 128), Kb)
  const float* bias;       // nullptr or [N]
  void* out;               // (M, N) of type out_dt
  int out_dt;
  int64_t M, N;
  int kb;                  // blocks along K
};

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
};
int64_t fp8_linear_workspace(int64_t M, int64_t N, int64_t K, bool quantised, bool exact);  // exact: fp32 output
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
