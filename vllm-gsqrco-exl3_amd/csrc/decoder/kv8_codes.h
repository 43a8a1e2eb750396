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

// Writes tokens [lo, hi) of a (page, head) of V, whose tokens are innermost: a thread turns 16 tokens x 8 dims in its registers.
// `base`: where the page's token 0 would lie in x. 16-token groups without new tokens are touched only where the scale grew.
template <int DT, int D, int THREADS>
__device__ __forceinline__ void put_v(int8_t* codes, int page, int lo, int hi, int older, const void* x, int64_t base,
                                      int64_t stride, const Rescale& s) {
  constexpr int per = D / 8;
  const bool shrink = older > 0 && s.shrink;
  const int g0 = shrink ? 0 : lo / 16, g1 = (hi + 15) / 16;
  for (int i = threadIdx.x; i < (g1 - g0) * per; i += THREADS) {
    const int t0 = 16 * (g0 + i / per), at = 8 * (i % per);
    uint32_t w[8][4];
    const bool whole = lo <= t0 && t0 + 16 <= hi;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      uint4 o = make_uint4(0, 0, 0, 0);
      if (!whole) o = *(const uint4*)(codes + (int64_t)(at + e) * page + t0);
      w[e][0] = o.x; w[e][1] = o.y; w[e][2] = o.z; w[e][3] = o.w;
    }
#pragma unroll
    for (int t = 0; t < 16; ++t) {
      float v[8];
      const bool is_new = t0 + t >= lo && t0 + t < hi;
      const bool is_old = shrink && t0 + t < older;
      if (is_new) load8<DT>(x, base + (t0 + t) * stride + at, v);
      if (is_new || is_old) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float y = is_new ? v[e] * s.inv : (float)(int8_t)(w[e][t >> 2] >> 8 * (t & 3)) * s.ratio;
          w[e][t >> 2] = (w[e][t >> 2] & ~(0xFFu << 8 * (t & 3))) | (uint32_t)(code_of(y) & 0xFF) << 8 * (t & 3);
        }
      }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) *(uint4*)(codes + (int64_t)(at + e) * page + t0) = make_uint4(w[e][0], w[e][1], w[e][2], w[e][3]);
  }
}

}  // namespace gguf_dec
