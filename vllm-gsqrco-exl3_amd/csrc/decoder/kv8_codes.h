// Codes of the 8-bit cache as its writers make them (kv8.hip says how they are defined).
#pragma once

#include "dec_common.h"

namespace gguf_dec {

// round to nearest even, at most 127 in magnitude; NaN (0 * inf of a page that is not finite) -> 0
__device__ __forceinline__ int code_of(float x) {
  const float r = rintf(x);
  return r != r ? 0 : (int)fminf(fmaxf(r, -127.0f), 127.0f);
}

__device__ __forceinline__ uint32_t rescale4(uint32_t w, float ratio) {
  uint32_t out = 0;
#pragma unroll
  for (int b = 0; b < 4; ++b) out |= (uint32_t)(code_of((float)(int8_t)(w >> 8 * b) * ratio) & 0xFF) << 8 * b;
  return out;
}

// A (page, head)'s new scale, its inverse, and what older codes are multiplied by where it is another one (`shrink`).
struct Rescale {
  float scale, inv, ratio;
  bool shrink;
};

// from the old scale and the scale that fresh values need: never less than the old one; a NaN on either side is kept
__device__ __forceinline__ Rescale grown(float was, float fresh) {
  const float now = fresh <= was ? was : fresh;  // a NaN of fresh's is kept here, was's as was > 0 fails
  Rescale r;
  r.scale = was != was ? was : now;
  r.inv = r.scale > 0.0f ? 1.0f / r.scale : 0.0f;
  r.shrink = !(r.scale == was);
  r.ratio = r.shrink ? was / r.scale : 1.0f;
  return r;
}

// from the old scale and the largest magnitude of fresh values
__device__ __forceinline__ Rescale rescale_of(float was, float amax) {
  const float fresh = amax / 127.0f;
  return grown(was, fresh < kLeastScale ? 0.0f : fresh);
}

}  // namespace gguf_dec
