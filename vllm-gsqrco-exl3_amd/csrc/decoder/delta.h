// The gated delta rule's arguments and the layout of its chunked form's workspace.
#pragma once

#include "dec_common.h"

namespace gguf_dec {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

constexpr float kNormEps = 1e-6f;
// The most tokens that the recurrent form takes where there is a workspace: between where one sequence and where many
// cross. Calls in us, recurrent / chunked, 16 and 48 bf16 heads of 128: one sequence of 16 tokens 21.4 / 20.8, of 32 tokens
// 38.7 / 21.0; eight of 24 tokens 40.3 / 58.1, of 48 tokens 73.2 / 61.0; 32 of 32 tokens 120 / 157, of 64 tokens 225 / 185.
constexpr int kRecurrent = 32;

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
  static constexpr int NA = DT == kF32 ? 3 : 2;                    // planes of A that the output takes
  static constexpr int KR = DK + 8;                                // row length of keys and queries
  // bytes: keys [NK][C][KR], queries alike; whole KB
  static constexpr int kK = 0, kQ = NK * C * KR * 2, kKq = (2 * kQ + 1023) / 1024 * 1024;
  static constexpr int kPrep = NK * C * KR * 2 > C * (C + 4) * 4 ? NK * C * KR * 2 : C * (C + 4) * 4;  // half of prep_kernel's LDS
  // T and A in fp32, by steps of 32 columns, of which step s has the rows from 32 s on (above they are 0):
  // row i, column j lies at kTt + 4 tri(i, j)
  static constexpr int RS = 36;
  static constexpr __host__ __device__ int tri(int i, int j) {
    const int s = j / 32;
    return (s * C - 16 * s * (s - 1) + i - 32 * s) * RS + j % 32;
  }
  static constexpr int kTri = (tri(C - 1, C - 1) + 1 + 4) / 4 * 4 * 4;
  // T, A, factors float4 [C + 1]; whole KB, shared out evenly with the above over the scan's waves, which copy
  // 1 KB at a time
  static constexpr int kTt = 0, kA = kTri, kFactors = 2 * kTri;
  static constexpr int ND = DT == kF16 ? 4 : 2;     // groups of 16 values of a head that a workgroup of the scan takes
  static constexpr int WAVES = C / 16 * ND, kPart = WAVES * 1024;
  static constexpr int kT = (kKq + kFactors + (C + 1) * 16 + kPart - 1) / kPart * kPart - kKq;
  // behind them in LDS: the planes of S, X and U as right operands, 1 KB for 32 places of the sum
  static constexpr int NU = DT == kF32 ? 6 : 5;     // U's planes: three for S, the others for the output
  static constexpr int kS = kKq + kT, kX = kS + ND * 3 * (DK / 32) * 1024, kU = kX + ND * 3 * (C / 32) * 1024;
  static constexpr int kLds = kU + ND * NU * (C / 32) * 1024;
  static_assert(kLds + ND * 16 * 4 <= 160 * 1024, "LDS");
};

}  // namespace gguf_dec
