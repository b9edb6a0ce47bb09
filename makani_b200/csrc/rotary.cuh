// Rotary positions with several axes for queries and keys, alone or behind a norm of every head's channels, forward and backward (rotary.cu).
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace mk {

constexpr int ROT_WIDTH = 256;         // most channels of a head (a multiple of 8)
constexpr int ROT_AXES = 4;            // most axes

// A tensor [B, N, heads, D] in elements: D is dense, strides are multiples of 8 and the base is 16-byte aligned
struct RotTensor {
  void* ptr;
  long long token, head, batch;
};

// Queries, or keys
struct RotPart {
  RotTensor x;             // input (null in a backward pass without a norm)
  RotTensor dy;            // gradient of the result (backward)
  RotTensor out;           // result, or gradient of x; may be dy
  int heads;
  const float *w, *b;      // [D] of the norm; null: one and zero
  float *dw, *db;          // [D] (backward; both or none)
};

enum { ROT_POS_I32 = 0, ROT_POS_I64 = 1, ROT_POS_F32 = 2, ROT_POS_F64 = 3 };
enum { ROT_NORM_NONE = 0, ROT_NORM_LAYER = 1, ROT_NORM_RMS = 2 };

struct RotShape {
  RotPart part[2];
  int parts;               // 1 or 2
  int B, N, D;
  uint8_t f32;             // type of x, dy and out: fp32, or bf16
  uint8_t norm;
  uint8_t interleaved;     // pairs are neighbours (2i, 2i + 1) of a band, else its halves (i, i + band / 2)
  uint8_t inverse;         // turned the other way
  float eps;
  // positions [N, axes], or [B, N, axes]: null for no rotation
  const void* positions;
  int position_type;
  long long position_batch;      // elements between two samples; 0: shared
  int axes;
  const int* limit;              // (backward) tokens from *limit on, in the only sample, are left as they are and add nothing to dw, db; null: none
  int band[ROT_AXES];            // channels of an axis, one after the other from channel 0 on; even
  double turns[ROT_WIDTH / 2];   // turns per unit of position of every pair
};

// Result: x normed, turned.  Backward: dy turned back, through the norm; `sums`: rotary_scratch() floats where dw is asked for.
cudaError_t rotary_fwd(const RotShape& p, cudaStream_t s);
long long rotary_scratch(const RotShape& p);
cudaError_t rotary_bwd(const RotShape& p, float* sums, int* launches, cudaStream_t s);

}  // namespace mk
