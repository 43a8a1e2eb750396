// What the attention kernels over the 8-bit cache share: operand layouts, conversions and the
// softmax's statistics.
//
// Both products are transposed, so that a lane keeps one query row all through:
//   S^T [tokens x rows] = K [tokens x d] . Q^T [d x rows]        v_mfma_f32_16x16x32_f16
//   O^T [d x rows]     += V^T [d x tokens] . P^T [tokens x rows]
// With lane = 16 g + n, an A operand holds row n's values 8g .. 8g + 7 of 32 along the sum, a B
// operand column n's, and the result's element i is row 4g + i of column n. Which values the 32 places
// stand for is free as long as both operands agree:
//   - along d, lane group g takes 16 bytes at 64 s + 16 g of a key: the first eight are its part of
//     product 2s, the others of 2s + 1;
//   - a tile is 64 tokens, in chunks of 16 (a chunk never leaves its page). Row 4c + i of the
//     tile's K operand tt is token 16 c + 4 tt + i, so lane group g receives the scores of chunk g,
//     tokens 4 tt + i, and these are, in place, the P^T operand for the 16 tokens of V's chunk g, which lie in
//     one 16-byte piece of a dim's row. Scores never cross lanes.
#pragma once

#include "dec_common.h"

namespace gguf_dec {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kNoScore = -3e38f;  // the running maximum before any score; finite, so that differences are numbers
// Weights enter the second product in fp16, times this: the maximum lags by at most 2^8, so they end at 2^15, and keep
// all bits down to 2^-21 of the largest, some down to 2^-32 (without it 2^-14 and 2^-25, where half a million tokens
// of 2^-26 each, a hundredth of a row's sum, were lost).
constexpr float kWeight = 128.0f;

// 4 codes -> 4 fp16, exact: a byte u under 0x64 is fp16 1024 + u
__device__ __forceinline__ void codes_to_half(uint32_t w, uint32_t& lo, uint32_t& hi) {
  const uint32_t u = w ^ 0x80808080u;  // code + 128
  const half2v off = {(_Float16)1152.0f, (_Float16)1152.0f};
  lo = __builtin_bit_cast(uint32_t, __builtin_bit_cast(half2v, __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u)) - off);
  hi = __builtin_bit_cast(uint32_t, __builtin_bit_cast(half2v, __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u)) - off);
}

__device__ __forceinline__ half8 codes8(uint32_t a, uint32_t b) {
  uint4 w;
  codes_to_half(a, w.x, w.y);
  codes_to_half(b, w.z, w.w);
  return __builtin_bit_cast(half8, w);
}

// max over the four lane groups (lanes n, n + 16, n + 32, n + 48)
__device__ __forceinline__ float group_max(float v) {
  v = fmaxf(v, __shfl_xor(v, 16, 64));
  return fmaxf(v, __shfl_xor(v, 32, 64));
}

__device__ __forceinline__ float group_sum(float v) {
  v += __shfl_xor(v, 16, 64);
  return v + __shfl_xor(v, 32, 64);
}

// The power of two that brings a row's largest magnitude into [1, 2) ([2, 4) from 2^127 on), so that bf16 queries of
// any size fit fp16 exactly (but for values 2^-14 below the row's largest, rounded there); 1 for an all-zero row.
__device__ __forceinline__ float row_factor(float amax) {
  const int e = (int)((__float_as_uint(amax) >> 23) & 0xFF);
  return amax > 0.0f && e >= 1 && e <= 254 ? __uint_as_float((uint32_t)max(254 - e, 1) << 23) : 1.0f;
}

// Where a 16-token chunk lies (page * heads + head, first token in the page), and its scales.
struct Chunk {
  int ph, off;
  float ks, vs;
};

// Chunk ch of a sequence. One past position `see` has scales of 0; a page out of range reads as NaN, and a V scale
// that is not finite is NaN for the rows that see it and no measure for the others. ph is always a page's.
__device__ __forceinline__ Chunk chunk_of(const Kv8& c, const int32_t* table, int page16, int head, int64_t ch, int see) {
  const bool seen = see >= 0 && ch <= see / 16;
  const int pi = seen ? (int)ch / page16 : 0;
  const int pid = table[pi];
  const bool ok = seen && pid >= 0 && pid < c.pages;
  Chunk r;
  r.ph = (ok ? pid : 0) * c.heads + head;
  r.off = seen ? ((int)ch - pi * page16) * 16 : 0;
  const float none = seen ? __builtin_nanf("") : 0.0f;
  r.ks = ok ? c.ks[r.ph] : none;
  r.vs = ok ? c.vs[r.ph] : none;
  if (!(r.vs <= 3.0e38f)) r.vs = __builtin_nanf("");
  if (fabsf(r.vs) < kLeastScale) r.vs = 0.0f;
  return r;
}

// max over lanes l and l ^ 32
__device__ __forceinline__ float half_max(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

// What a call is made of.
struct AttnArgs {
  Kv8 c;
  const void* q;
  int64_t qt, qh;  // strides of a token and a head, in elements
  const int32_t* lens;
  Ragged rows;
  int hq, group;   // query heads; query heads a KV head
  float scale;     // times log2 e
  int span;        // tokens of a split, a multiple of 256 (the last split takes what is left)
  int splits;
  void* out;       // [tokens, hq, d]
  float* part;     // of a split call: [splits][tokens * hq][d] sums, then m and l: [splits][tokens * hq][2]
  float* stat;
};

// attention_rows.hip: many rows
constexpr int kRowsTile = 128;  // rows of a workgroup
hipError_t launch_attend_rows(const AttnArgs& a, int dtype, int64_t row_tiles, hipStream_t stream);

}  // namespace gguf_dec
