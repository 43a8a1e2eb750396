// Rotation of queries and keys by their positions, with the norms of their heads before it, and the keys' and values' way into
// the 8-bit paged cache, in one launch (include/gguf_decoder.h: contract; kv8.hip: the codes).
//
// A head's row is D / 16 items, a lane each: two pieces of 8 values that turn together, the i-th and the (i + rot / 2)-th
// dims of a piece, or that hold whole pairs. So a row's lanes need each other for the norm's sum only.
#include <algorithm>

#include "kv8_codes.h"
#include "rotary.h"

namespace gguf_dec {

namespace {

constexpr int kThreads = 256;

// lanes of a row (a power of two; of 192 dims four of 16 idle)
template <int D>
constexpr int kLanes = D == 64 ? 4 : D == 128 ? 8 : 16;

// where an item's pieces lie in the row, and its first cosine (-1: it does not turn)
struct Item {
  int o0, o1, turn;
};

__device__ __forceinline__ Item item_of(int i, int rot, bool pairs) {
  if (16 * i >= rot || pairs) return Item{16 * i, 16 * i + 8, 16 * i < rot ? 8 * i : -1};
  return Item{8 * i, rot / 2 + 8 * i, 8 * i};
}

// A row's item, normed and turned, in fp32. Every lane of the row comes here.
template <int DT, int D>
__device__ __forceinline__ void turned(const RotaryArgs& a, const void* x, int64_t row, const Item& it, bool mine,
                                       const float (*w)[8], int64_t token, bool ok, float (&v)[2][8]) {
#pragma unroll
  for (int e = 0; e < 8; ++e) v[0][e] = v[1][e] = 0.0f;
  float c[8], s[8];
  const bool turn = mine && ok && it.turn >= 0;
  if (turn) {
    const int64_t at = a.at[token];
    if (at >= 0 && at < a.positions) {
      load8<kF32>(a.table, at * a.table_stride + it.turn, c);
      load8<kF32>(a.table, at * a.table_stride + a.rot / 2 + it.turn, s);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) c[e] = s[e] = __builtin_nanf("");
    }
  }
  if (mine && ok) {
    load8<DT>(x, row + it.o0, v[0]);
    load8<DT>(x, row + it.o1, v[1]);
  }
  if (w) {
    float sum = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; ++e) sum += v[0][e] * v[0][e] + v[1][e] * v[1][e];
#pragma unroll
    for (int off = 1; off < kLanes<D>; off <<= 1) sum += __shfl_xor(sum, off, 64);
    const float by = rsqrtf(sum * (1.0f / D) + a.eps);
#pragma unroll
    for (int p = 0; p < 2; ++p)
#pragma unroll
      for (int e = 0; e < 8; ++e) v[p][e] *= by * w[p][e];
  }
  if (!turn) return;
  if (a.pairs) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int p = e >> 2, i = 2 * (e & 3);
      const float x0 = v[p][i], x1 = v[p][i + 1];
      v[p][i] = x0 * c[e] - x1 * s[e];
      v[p][i + 1] = x1 * c[e] + x0 * s[e];
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float x0 = v[0][e], x1 = v[1][e];
      v[0][e] = x0 * c[e] - x1 * s[e];
      v[1][e] = x1 * c[e] + x0 * s[e];
    }
  }
}

// 8 values as codes of 1 / scale
__device__ __forceinline__ uint2 codes_of(const float (&v)[8], float inv) {
  uint32_t w[2] = {0, 0};
#pragma unroll
  for (int e = 0; e < 8; ++e) w[e >> 2] |= (uint32_t)(code_of(v[e] * inv) & 0xFF) << 8 * (e & 3);
  return make_uint2(w[0], w[1]);
}

// The first `blocks` workgroups take the cache's (sequence, page, head)s of K and V, one at a time, so that a scale has one
// writer; the others take the queries' rows.
template <int DT, int D>
__global__ void __launch_bounds__(kThreads) rotary_kernel(RotaryArgs a, int blocks, int page_blocks) {
  constexpr int L = kLanes<D>;
  const Kv8& c = a.c;
  const int tid = threadIdx.x, lane = tid % L;
  const bool mine = 16 * lane < D;
  const Item it = item_of(mine ? lane : 0, a.rot, a.pairs);
  if ((int)blockIdx.x >= blocks) {
    float w[2][8];
    if (a.qw) {
      load8<kF32>(a.qw, it.o0, w[0]);
      load8<kF32>(a.qw, it.o1, w[1]);
    }
    const int64_t all = (int64_t)a.rows.tokens * a.hq, per = kThreads / L;
    for (int64_t r0 = ((int64_t)blockIdx.x - blocks) * per; r0 < all; r0 += (int64_t)(gridDim.x - blocks) * per) {
      const int64_t r = r0 + tid / L, token = r / a.hq;
      const bool ok = r < all;
      float v[2][8];
      turned<DT, D>(a, a.q, token * a.qt + (r - token * a.hq) * a.qh, it, mine, a.qw ? w : nullptr, token, ok, v);
      if (mine && ok) {
        store8<DT>(a.out, r * D + it.o0, v[0]);
        store8<DT>(a.out, r * D + it.o1, v[1]);
      }
    }
    return;
  }

  const int b = blockIdx.x / page_blocks, head = b / 2 % c.heads, seq = b / 2 / c.heads;
  const bool is_v = b & 1;
  int r0, r1;
  rows_of(a.rows, seq, r0, r1);
  const int64_t room = (int64_t)c.max_pages * c.page;
  const int64_t len = a.lens[seq], start = len - (r1 - r0);  // position of row r0; rows before position 0 are dropped
  const int64_t end = min(len, room);
  if (r1 == r0 || end <= 0) return;
  const int page = c.page;
  const int first = (int)(max(start, (int64_t)0) / page), last = (int)((end - 1) / page);
  __shared__ uint32_t most[kThreads / 64];
  float w[2][8];
  if (!is_v && a.kw) {
    load8<kF32>(a.kw, it.o0, w[0]);
    load8<kF32>(a.kw, it.o1, w[1]);
  }

  for (int p = first + (int)blockIdx.x % page_blocks; p <= last; p += page_blocks) {
    const int pid = c.table[(int64_t)seq * c.table_stride + p];
    if (pid < 0 || pid >= c.pages) continue;  // uniform
    const int64_t p0 = (int64_t)p * page;
    const int lo = (int)(max(start, p0) - p0), hi = (int)(min(end, p0 + page) - p0);  // new tokens of the page
    const int64_t row0 = r0 + (p0 - start);                                           // row of the page's token 0
    const int older = start > p0 ? lo : 0;
    int8_t* codes = (is_v ? c.v : c.k) + ((int64_t)pid * c.heads + head) * page * D;

    // the new values' largest magnitude (as bits of |x|: unsigned order puts inf and NaN on top, so they reach the scale)
    uint32_t big = 0;
    const auto key = [&](int t, float (&v)[2][8]) __attribute__((always_inline)) {
      const int64_t token = row0 + t;
      turned<DT, D>(a, a.k, token * a.kt + head * a.kh, it, mine, a.kw ? w : nullptr, token, t < hi, v);
    };
    if (!is_v) {
      for (int t0 = lo; t0 < hi; t0 += kThreads / L) {
        float v[2][8];
        key(t0 + tid / L, v);
#pragma unroll
        for (int e = 0; e < 8; ++e) big = max(big, max(__float_as_uint(v[0][e]) & 0x7FFFFFFFu, __float_as_uint(v[1][e]) & 0x7FFFFFFFu));
      }
    } else {
      for (int i = tid; i < (hi - lo) * (D / 8); i += kThreads) {
        float v[8];
        load8<DT>(a.v, (row0 + lo + i / (D / 8)) * a.vt + head * a.vh + 8 * (i % (D / 8)), v);
#pragma unroll
        for (int e = 0; e < 8; ++e) big = max(big, __float_as_uint(v[e]) & 0x7FFFFFFFu);
      }
    }
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) big = max(big, (uint32_t)__shfl_xor((int)big, off, 64));
    __syncthreads();  // the previous page's `most` has been read
    if ((tid & 63) == 0) most[tid >> 6] = big;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kThreads / 64; ++i) big = max(big, most[i]);

    float* scale = (is_v ? c.vs : c.ks) + (int64_t)pid * c.heads + head;
    const float was = older > 0 ? *scale : 0.0f;
    const Rescale s = rescale_of(was, __uint_as_float(big));
    __syncthreads();  // every thread has read the old scale
    if (tid == 0) *scale = s.scale;

    if (!is_v) {
      if (s.shrink && older > 0)
        for (int i = tid; i < older * D / 4; i += kThreads) ((uint32_t*)codes)[i] = rescale4(((uint32_t*)codes)[i], s.ratio);
      for (int t0 = lo; t0 < hi; t0 += kThreads / L) {
        const int t = t0 + tid / L;
        float v[2][8];
        key(t, v);
        if (!mine || t >= hi) continue;
        *(uint2*)(codes + (int64_t)t * D + it.o0) = codes_of(v[0], s.inv);
        *(uint2*)(codes + (int64_t)t * D + it.o1) = codes_of(v[1], s.inv);
      }
    } else {
      put_v<DT, D, kThreads>(codes, page, lo, hi, older, a.v, row0 * a.vt + head * a.vh, a.vt, s);
    }
  }
}

}  // namespace

hipError_t launch_kv8_rotary(const RotaryArgs& a, int dtype, int64_t max_new, hipStream_t stream) {
  // a page more than the tokens fill: they may start inside one. A grid holds fewer than 2^24 workgroups of 256 threads: of
  // many pages a workgroup takes several in turn
  const int64_t groups = 2LL * a.c.heads * a.rows.seqs;
  int64_t pages = (max_new + a.c.page - 2) / a.c.page + 1;
  pages = std::max<int64_t>(1, std::min(pages, (1 << 23) / groups));
  const int64_t blocks = groups * pages;
#define GGUF_DEC_ROTARY(DT, D)                                                                       \
  {                                                                                                  \
    constexpr int per = kThreads / kLanes<D>;                                                        \
    const int64_t rows = ((int64_t)a.rows.tokens * a.hq + per - 1) / per;                            \
    const int64_t grid = blocks + std::min<int64_t>(rows, 1 << 22);                                  \
    rotary_kernel<DT, D><<<(unsigned)grid, kThreads, 0, stream>>>(a, (int)blocks, (int)pages);       \
  }
#define GGUF_DEC_ROTARY_D(DT)                  \
  switch (a.c.d) {                             \
    case 64: GGUF_DEC_ROTARY(DT, 64) break;    \
    case 128: GGUF_DEC_ROTARY(DT, 128) break;  \
    case 192: GGUF_DEC_ROTARY(DT, 192) break;  \
    default: GGUF_DEC_ROTARY(DT, 256) break;   \
  }
  GGUF_DEC_FLOATS(dtype, GGUF_DEC_ROTARY_D)
#undef GGUF_DEC_ROTARY_D
#undef GGUF_DEC_ROTARY
  return hipGetLastError();
}

}  // namespace gguf_dec
