// The gated delta rule's arguments and the layout of its chunked form's workspace.
#pragma once

#include "dec_common.h"

namespace gguf_dec {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

constexpr float kNormEps = 1e-6f;
constexpr int kRecurrent = 32;  // the most tokens that the recurrent form takes where there is a workspace

struct DeltaArgs {
  const void *q, *k, *v;
  int64_t qt, qh, kt, kh, vt, vh;  // strides of a token and a head, in elements
  const float *g, *beta;
  int64_t gt, bt;
  float* state;  // [nslots, hv, dv, dk]
  int64_t nslots;
  const int32_t *slots, *out_slots;
  int64_t out_stride;
  int steps;  // 0: the last state goes to out_slots[seq]; else each of the first `steps` tokens' states goes to its own
  int hk, hv, dv, rep;
  float scale;
  int l2norm;
  Ragged rows;
  void* out;  // [tokens, hv, dv]
};

struct ChunkWs {
  char* kq;  // [chunk slots][hk][Layout::kKq]
  char* t;   // [chunk slots][hv][Layout::kT]
};

// Chunks of 64 tokens of bf16; of 32 where keys take two or three planes, whose LDS would not hold 64.
template <int DT>
struct Chunk {
  static constexpr int C = DT == kBF16 ? 64 : 32;
};

// What a chunk's scan takes, as it lies in LDS. Rows are padded by 16 bytes against bank conflicts.
template <int DT, int DK, int C>
struct Layout {
  static constexpr int NK = DT == kBF16 ? 1 : DT == kF16 ? 2 : 3;  // planes of a key or query
  static constexpr int NA = DT == kF32 ? 3 : 2;                    // planes of A
  static constexpr int KR = DK + 8, CR = C + 8;                    // row lengths
  // bytes: keys [NK][C][KR], queries alike, keys turned [NK][DK][CR]
  static constexpr int kK = 0, kQ = NK * C * KR * 2, kKT = 2 * kQ, kKq = kKT + NK * DK * CR * 2;
  // T [3][C][CR], A [NA][C][CR], factors float4 [C + 1]
  static constexpr int kTt = 0, kA = 3 * C * CR * 2, kFactors = kA + NA * C * CR * 2, kT = kFactors + (C + 1) * 16;
  static_assert(kKq % 16 == 0 && kT % 16 == 0 && kKq + kT <= 160 * 1024, "LDS");
};

}  // namespace gguf_dec
