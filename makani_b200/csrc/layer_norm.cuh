// Layer norm over the last dimension of tokens, forward and backward, with or without a residual sum in front (layer_norm.cu).
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace mk {

constexpr int LN_CHANNELS = 8192;      // most channels of a row
constexpr int LN_HALF_PARAMS = 1024;   // most channels with weights and biases in bf16 (their gradients may be bf16 at any width)

// y = (x - mean) rstd w + b for every row, biased variance; with `r` the row is s = x + r, rounded to the type of x, which is written too.
// Types: bf16 (0) or fp32 (1), of x and s (`x_f32`), of r (`r_f32`, not above that of x), of y (`y_f32`), of w and of b (either may be null).
// Row i of x begins at (i / inner) * outer_stride + (i % inner) * inner_stride elements; the others are dense.
struct LnForward {
  const void* x;
  const void* r;
  void* s;
  void* y;
  const void* w;
  const void* b;
  float2* stats;           // (mean, rstd) of every row, or null
  long long rows;
  int C;
  long long inner, outer_stride, inner_stride;
  float eps;
  uint8_t x_f32, r_f32, y_f32, w_f32, b_f32;
};
cudaError_t layer_norm_fwd(const LnForward& p, cudaStream_t s);

// dx (type of x; a copy in bf16 in `dr`, if there is one) = rstd (g - mean(g) - xh mean(g xh)) (+ ds), g = dy w (dy: type of y); dw = sum of dy xh, db = sum
// of dy over the rows (both or none; `dw_f32`, `db_f32`: their types, rounded once).  `part`: layer_norm_scratch() floats.  The sums are added up in one fixed order.
struct LnBackward {
  const void* x;
  const void* dy;
  const void* ds;
  void* dx;
  void* dr;
  const void* w;
  const float2* stats;
  void* dw;
  void* db;
  float* part;
  long long rows;
  int C;
  long long inner, outer_stride, inner_stride;
  // (bytes: three integers more, and the compiler spills ten times as much in the kernel of ragged long rows)
  uint8_t x_f32, y_f32, w_f32, dw_f32, db_f32;
};
long long layer_norm_scratch(long long rows, int C);
cudaError_t layer_norm_bwd(const LnBackward& p, int* launches, cudaStream_t s);

}  // namespace mk
