// Dropout from a counter-based generator, with or without a residual sum behind it (dropout.cu).
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace mk {

// Where a call's random words come from: the key (64 bits) and the number of the call, read on the device where there is a pointer (a captured graph reads
// what stands there at its replay).  number = (*offset or 0, plus `more`) >> shift.
struct DropSource {
  const int64_t* key_at;
  const int64_t* offset_at;
  uint64_t key, more;
  int shift;
  int64_t* kept;           // (key, number) as they were used, or null
};

// out = (word_i > last ? x * factor : 0) (+ r) for every element i of dense tensors; `copy`: x rounded to bf16 (a residual's gradient), or null.
// Types: bf16 (0) or fp32 (1) of x, r and out: out has the wider of x and r, or (no r) any that is not wider than x.
struct DropParams {
  const void* x;
  const void* r;
  void* out;
  void* copy;
  long long n;
  uint32_t last;           // words up to this one are dropped
  float factor;
  DropSource source;
  uint8_t x_f32, r_f32, out_f32;
};
cudaError_t dropout(const DropParams& p, cudaStream_t s);

}  // namespace mk
