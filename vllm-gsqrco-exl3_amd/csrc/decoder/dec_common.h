// Types and small device helpers shared by the decoder operators' kernels (include/gguf_decoder.h).
#pragma once

#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../gguf_common.h"

namespace gguf_dec {

using gguf::kBF16;
using gguf::kF16;
using gguf::kF32;

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef short short8 __attribute__((ext_vector_type(8)));
typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef uint32_t uintx4 __attribute__((ext_vector_type(4)));

// scales of the 8-bit cache below this count as zero, so that 1 / s stays finite
constexpr float kLeastScale = 0x1p-100f;

// The paged 8-bit KV cache as the kernels take it.
struct Kv8 {
  int8_t* k;       // [pages, heads, page, d]
  int8_t* v;       // [pages, heads, d, page]
  float* ks;       // [pages, heads]
  float* vs;
  const int32_t* table;  // [seqs, max_pages]
  int64_t table_stride;
  int pages, heads, page, d, max_pages;
};

// A ragged batch: offsets of each sequence's rows among `tokens`.
struct Ragged {
  const int32_t* cu;  // [seqs + 1]
  int seqs, tokens;
};

// rows [lo, hi) of sequence s, cut to the tensors' rows (offsets in device memory are not trusted)
__device__ __forceinline__ void rows_of(const Ragged& r, int s, int& lo, int& hi) {
  lo = min(max(r.cu[s], 0), r.tokens);
  hi = min(max(r.cu[s + 1], lo), r.tokens);
}

// 8 consecutive elements of type DT as fp32 (16-byte aligned)
template <int DT>
__device__ __forceinline__ void load8(const void* p, int64_t i, float (&v)[8]) {
  if constexpr (DT == kF32) {
    const float4 a = *(const float4*)((const float*)p + i), b = *(const float4*)((const float*)p + i + 4);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  } else {
    const uint4 a = *(const uint4*)((const uint16_t*)p + i);
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if constexpr (DT == kF16) {
        v[2 * e] = gguf::half_bits_to_float(w[e] & 0xFFFF);
        v[2 * e + 1] = gguf::half_bits_to_float(w[e] >> 16);
      } else {
        v[2 * e] = __uint_as_float(w[e] << 16);
        v[2 * e + 1] = __uint_as_float(w[e] & 0xFFFF0000u);
      }
    }
  }
}

template <int DT>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if constexpr (DT == kF16) {
    return (uint32_t)__half_as_ushort(__float2half_rn(a)) | (uint32_t)__half_as_ushort(__float2half_rn(b)) << 16;
  } else {
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    const bf16x2 v = {(__bf16)a, (__bf16)b};  // one v_cvt_pk_bf16_f32, to nearest even
    return __builtin_bit_cast(uint32_t, v);
  }
}

// 4 / 8 consecutive fp32 values rounded to DT (aligned)
template <int DT>
__device__ __forceinline__ void store4(void* p, int64_t i, const float (&v)[4]) {
  if constexpr (DT == kF32) {
    *(float4*)((float*)p + i) = make_float4(v[0], v[1], v[2], v[3]);
  } else {
    *(uint2*)((uint16_t*)p + i) = make_uint2(pack2<DT>(v[0], v[1]), pack2<DT>(v[2], v[3]));
  }
}

template <int DT>
__device__ __forceinline__ void store8(void* p, int64_t i, const float (&v)[8]) {
  if constexpr (DT == kF32) {
    *(float4*)((float*)p + i) = make_float4(v[0], v[1], v[2], v[3]);
    *(float4*)((float*)p + i + 4) = make_float4(v[4], v[5], v[6], v[7]);
  } else {
    *(uint4*)((uint16_t*)p + i) =
        make_uint4(pack2<DT>(v[0], v[1]), pack2<DT>(v[2], v[3]), pack2<DT>(v[4], v[5]), pack2<DT>(v[6], v[7]));
  }
}

template <int DT>
__device__ __forceinline__ void store1(void* p, int64_t i, float v) {
  if constexpr (DT == kF32) ((float*)p)[i] = v;
  else if constexpr (DT == kF16) ((_Float16*)p)[i] = (_Float16)v;
  else ((__bf16*)p)[i] = (__bf16)v;
}

template <int DT>
__device__ __forceinline__ float load1(const void* p, int64_t i) {
  return gguf::load_x(p, i, DT);
}

}  // namespace gguf_dec

// CALL(DT) for the element type of a tensor
#define GGUF_DEC_FLOATS(dtype, CALL)      \
  switch (dtype) {                        \
    case gguf_dec::kF32: CALL(gguf_dec::kF32); break;   \
    case gguf_dec::kF16: CALL(gguf_dec::kF16); break;   \
    default: CALL(gguf_dec::kBF16); break;  \
  }
