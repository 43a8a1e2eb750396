// The norms between a decoder's blocks, as the kernels take them (include/gguf_decoder.h: contract).
#pragma once

#include "dec_common.h"

namespace gguf_dec {

// strides of a row (token, head), in elements; its values are adjacent
struct RowStride {
  int64_t t, h;
};

enum { kActNone = 0, kActSigmoid = 1, kActSilu = 2 };

struct NormArgs {
  const void* x;
  const void* residual;  // or null
  const void* gate;      // or null
  const float* inner;    // or null: no norm of x
  const float* outer;    // or null: no norm of h
  void* hidden;          // [rows, n]
  void* out;             // [rows, n], where there is an outer weight
  RowStride xs, rs, gs;
  int64_t rows;          // tokens * heads
  int heads, n, act;
  float scale, eps;
};

}  // namespace gguf_dec
