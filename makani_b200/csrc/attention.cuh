// Softmax attention of tokens with themselves: whole prompts, causal or not, grouped heads, batches or packed sequences (attention.cu).
#pragma once
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace mk {

constexpr int ATTN_WIDTH = 128;        // most channels of a head (a multiple of 8)

// A tensor [B, N, heads, D] in elements; D is dense, strides are multiples of 8 and the base is 16-byte aligned
struct AttnTensor {
  __nv_bfloat16* ptr;
  long long token, head, batch;
};

struct AttnShape {
  int B, N, H, Hk, D;        // H: heads of q and o; Hk: of k and v, H / Hk of q share one
  int causal;
  float scale;               // > 0
  // packed sequences (B = 1): sequence i has the tokens offsets[i] .. offsets[i + 1], not decreasing, within N; null: one sequence per batch.
  // What the offsets do not cover is written as zeros behind the last sequence.
  const int* offsets;
  int sequences;
};

// o [B, N, H, D] dense.  For a backward pass (both or none): lse [B, H, N], log2 of the sum of exponentials of every row, and o_rest, like o, what the
// rounding of o has left out, rounded in its turn.  `scratch`: attention_scratch() floats (none: nothing is split over the keys), 16-byte aligned.
// `launches` counts.
long long attention_scratch(const AttnShape& p);
cudaError_t attention_fwd(const AttnShape& p, const AttnTensor& q, const AttnTensor& k, const AttnTensor& v, __nv_bfloat16* o, __nv_bfloat16* o_rest,
                          float* lse, float* scratch, int* launches, int* err, cudaStream_t s);
// dq, dk, dv from o, o_rest and d_o (dense, like o); delta [B, H, N]: room for the row sums of o d_o.  `scratch`: attention_bwd_scratch() floats.  Two launches,
// with the sums of what is split four, and no atomics.
long long attention_bwd_scratch(const AttnShape& p);
cudaError_t attention_bwd(const AttnShape& p, const AttnTensor& q, const AttnTensor& k, const AttnTensor& v, const __nv_bfloat16* o,
                          const __nv_bfloat16* o_rest, const __nv_bfloat16* d_o, const float* lse, float* delta, const AttnTensor& dq,
                          const AttnTensor& dk, const AttnTensor& dv, float* scratch, int* launches, int* err, cudaStream_t s);

}  // namespace mk
