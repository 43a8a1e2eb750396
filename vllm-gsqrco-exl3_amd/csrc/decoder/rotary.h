// Position rotation on the way into the 8-bit cache, and the moves within it, as the kernels take them
// (include/gguf_decoder.h: contract).
#pragma once

#include "dec_common.h"

namespace gguf_dec {

constexpr int kMostKept = 1024;  // rows of a path

struct RotaryArgs {
  Kv8 c;
  const void *q, *k, *v;
  int64_t qt, qh, kt, kh, vt, vh;  // strides of a token and a head, in elements
  const float *qw, *kw;            // weights of the heads' norms, or null
  float eps;
  const float* table;              // [positions, rot]: cosines, then sines
  int64_t table_stride;
  int64_t positions;
  const int64_t* at;               // [tokens]
  int rot;
  bool pairs;                      // dims (2i, 2i + 1) turn together, else (i, i + rot / 2)
  const int32_t* lens;
  Ragged rows;
  int hq;
  void* out;                       // [tokens, hq, d]
};

}  // namespace gguf_dec
