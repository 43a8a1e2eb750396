// Rotation of queries and keys by their positions, with the norms of their heads before it, and the keys' and values' way into
// the 8-bit paged cache, in one launch (include/gguf_decoder.h: contract; kv8.hip: the codes).
//
// A head's row is D / 16 items, a lane each: two pieces of 8 values that turn together, the i-th and the (i + rot / 2)-th
// dims of a piece, or that hold whole pairs. So a row's lanes need each other for the norm's sum only.
//
// What bounds it: a step of single tokens the chain lens -> table -> page -> codes (32 sequences, 24 + 4 heads of 256 dims in
// bf16: 7.2 us a call in a graph, kv8_append alone 5.4, where no page's scale grows; where all do and older codes are rounded again, the
// kernel takes 9.8 us for 8.1, 16 fp16 drafts of 8 sequences 9.1 for 8.0, a prompt no longer); a prompt the memory (8192 tokens of 24 + 4 heads of 256: 252 MB read and
// written in 71 us, 3.6 TB/s, a copy reaches 5; in a loop, where the last level of cache holds a part, in 55). Times of that loop:
// - The two passes over a page's new values, for the scale and for the codes, run forwards and backwards, so that the last rows
//   are at hand for the second: of a page of 64 tokens of 256 dims half of K's and all of V's are read once. Holding all of K's
//   costs registers that spill (2 x 2 pieces: 69 us the prompt, 10.0 us the step).
// - V's codes, tokens innermost, turn in LDS, 64 tokens at a time; written a byte each they took the prompt to 100 us.
// - 512 threads and 128 registers; with 168 registers half the waves: 77 us; with 256 threads 58.
#include <algorithm>

#include "kv8_codes.h"
#include "rotary.h"

namespace gguf_dec {

namespace {

constexpr int kThreads = 512;
constexpr int kChunk = 64;  // tokens of V that are turned at a time

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
                                       bool norm, const float (&w)[2][8], int64_t token, bool ok, float (&v)[2][8]) {
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
  if (norm) {
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
// A (page, head)'s new values go through registers for its scale and then for the codes: the last kThreads / kLanes of its keys (32 of 256
// dims) and the last 64 of its values stay there, what it has beyond that is read (keys: normed and turned) again. V's codes, whose tokens
// are innermost, turn in LDS.
template <int DT, int D>
__global__ void __launch_bounds__(kThreads, 4) rotary_kernel(RotaryArgs a, int blocks, int page_blocks) {
  constexpr int L = kLanes<D>, ROWS = kThreads / L;  // rows that the workgroup takes at a time
  const Kv8& c = a.c;
  const int tid = threadIdx.x, lane = tid % L;
  const bool mine = 16 * lane < D;
  const Item it = item_of(mine ? lane : 0, a.rot, a.pairs);
  if ((int)blockIdx.x >= blocks) {
    float w[2][8] = {};
    if (a.qw) {
      load8<kF32>(a.qw, it.o0, w[0]);
      load8<kF32>(a.qw, it.o1, w[1]);
    }
    const int64_t all = (int64_t)a.rows.tokens * a.hq;
    for (int64_t r0 = ((int64_t)blockIdx.x - blocks) * ROWS; r0 < all; r0 += (int64_t)(gridDim.x - blocks) * ROWS) {
      const int64_t r = r0 + tid / L, token = all <= UINT32_MAX ? (int64_t)((uint32_t)r / (uint32_t)a.hq) : r / a.hq;
      float v[2][8];
      turned<DT, D>(a, a.q, token * a.qt + (r - token * a.hq) * a.qh, it, mine, a.qw != nullptr, w, token, r < all, v);
      if (!mine || r >= all) continue;
      store8<DT>(a.out, r * D + it.o0, v[0]);
      store8<DT>(a.out, r * D + it.o1, v[1]);
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
  const int first = (int)max(start, (int64_t)0) / page, last = (int)(end - 1) / page;
  __shared__ uint32_t most[kThreads / 64];
  float w[2][8] = {};
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
    float* scale = (is_v ? c.vs : c.ks) + (int64_t)pid * c.heads + head;

    // the page's scale from the new values' largest magnitude (as bits of |x|: unsigned order puts inf and NaN on top, so they
    // reach the scale)
    const float was = older > 0 ? *scale : 0.0f;
    const auto rescale = [&](uint32_t big) __attribute__((always_inline)) {
#pragma unroll
      for (int off = 32; off > 0; off >>= 1) big = max(big, (uint32_t)__shfl_xor((int)big, off, 64));
      __syncthreads();  // the previous page's `most` has been read
      if ((tid & 63) == 0) most[tid >> 6] = big;
      __syncthreads();  // (and every thread has read the old scale)
#pragma unroll
      for (int i = 0; i < kThreads / 64; ++i) big = max(big, most[i]);
      const Rescale s = rescale_of(was, __uint_as_float(big));
      if (tid == 0) *scale = s.scale;
      return s;
    };

    if (!is_v) {
      const auto key = [&](int t, float (&v)[2][8]) __attribute__((always_inline)) {
        const int64_t token = row0 + t;
        turned<DT, D>(a, a.k, token * a.kt + head * a.kh, it, mine, a.kw != nullptr, w, token, t < hi, v);
      };
      const auto most_of = [](const float (&v)[2][8]) __attribute__((always_inline)) {
        uint32_t big = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) big = max(big, max(__float_as_uint(v[0][e]) & 0x7FFFFFFFu, __float_as_uint(v[1][e]) & 0x7FFFFFFFu));
        return big;
      };
      float v[2][8];
      uint32_t big = 0;
      int t0 = lo;  // the last pass's rows stay in v
      while (true) {
        key(t0 + tid / L, v);
        big = max(big, most_of(v));
        if (t0 + ROWS >= hi) break;
        t0 += ROWS;
      }
      const Rescale s = rescale(big);
      if (s.shrink && older > 0)
        for (int i = tid; i < older * D / 4; i += kThreads) ((uint32_t*)codes)[i] = rescale4(((uint32_t*)codes)[i], s.ratio);
      while (true) {
        const int t = t0 + tid / L;
        if (mine && t < hi) {
          *(uint2*)(codes + (int64_t)t * D + it.o0) = codes_of(v[0], s.inv);
          *(uint2*)(codes + (int64_t)t * D + it.o1) = codes_of(v[1], s.inv);
        }
        t0 -= ROWS;
        if (t0 < lo) break;
        key(t0 + tid / L, v);
      }
    } else {
      constexpr int PER = D / 8, HELD = (kChunk * PER + kThreads - 1) / kThreads, ROW = D + 4;  // (4 more bytes, for LDS's banks)
      __shared__ __align__(16) uint32_t turn[kChunk * ROW / 4];
      const int g0 = lo / 16 * 16, g1 = (hi + 15) / 16 * 16;
      const int64_t base = row0 * a.vt + head * a.vh;
      // piece i of a chunk of tokens from t0 on: 8 dims of token t0 + i / PER
      const auto fetch = [&](int t0, int i, float (&x)[8]) __attribute__((always_inline)) {
        const int t = t0 + i / PER;
        const bool is_new = i < kChunk * PER && t >= lo && t < hi;
        if (is_new) {
          load8<DT>(a.v, base + t * a.vt + 8 * (i % PER), x);
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) x[e] = 0.0f;
        }
      };
      const auto most_of = [](const float (&x)[8]) __attribute__((always_inline)) {
        uint32_t big = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) big = max(big, __float_as_uint(x[e]) & 0x7FFFFFFFu);
        return big;
      };
      float held[HELD][8];
      uint32_t big = 0;
      int t0 = g0;  // the last chunk stays in `held`
      while (true) {
#pragma unroll
        for (int j = 0; j < HELD; ++j) {
          fetch(t0, j * kThreads + tid, held[j]);
          big = max(big, most_of(held[j]));
        }
        if (t0 + kChunk >= hi) break;
        t0 += kChunk;
      }
      const Rescale s = rescale(big);
      const bool shrink = s.shrink && older > 0;
      if (shrink)  // the groups of older tokens alone
        for (int i = tid; i < g0 / 16 * D; i += kThreads) {
          uint4* to = (uint4*)(codes + (int64_t)(i / (g0 / 16)) * page + 16 * (i % (g0 / 16)));
          const uint4 o = *to;
          *to = make_uint4(rescale4(o.x, s.ratio), rescale4(o.y, s.ratio), rescale4(o.z, s.ratio), rescale4(o.w, s.ratio));
        }
      while (true) {
#pragma unroll
        for (int j = 0; j < HELD; ++j) {
          const int i = j * kThreads + tid;
          if (i < kChunk * PER) {
            const uint2 w2 = codes_of(held[j], s.inv);
            uint32_t* to = turn + (i / PER) * (ROW / 4) + 2 * (i % PER);
            to[0] = w2.x;
            to[1] = w2.y;
          }
        }
        __syncthreads();
        // four dims of 16 tokens a thread, the groups of a dim side by side: a chunk's are no more than the workgroup's threads
        static_assert(kChunk / 16 * D / 4 <= kThreads, "one turn");
        const int groups = min(kChunk, g1 - t0) / 16;
        if (tid < groups * (D / 4)) {
          const int q = tid / groups, t = 16 * (tid - q * groups);
          uint32_t out[4][4];
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            uint32_t in[4];
#pragma unroll
            for (int y = 0; y < 4; ++y) in[y] = turn[(t + 4 * x + y) * (ROW / 4) + q];
            // a 4 x 4 block of bytes, turned
            const uint32_t a0 = __builtin_amdgcn_perm(in[1], in[0], 0x05010400u), a1 = __builtin_amdgcn_perm(in[1], in[0], 0x07030602u);
            const uint32_t b0 = __builtin_amdgcn_perm(in[3], in[2], 0x05010400u), b1 = __builtin_amdgcn_perm(in[3], in[2], 0x07030602u);
            out[0][x] = __builtin_amdgcn_perm(b0, a0, 0x05040100u);
            out[1][x] = __builtin_amdgcn_perm(b0, a0, 0x07060302u);
            out[2][x] = __builtin_amdgcn_perm(b1, a1, 0x05040100u);
            out[3][x] = __builtin_amdgcn_perm(b1, a1, 0x07060302u);
          }
          // what is not new stays, rescaled where it is older and the scale grew (the tokens before lo are all older)
          const bool whole = lo <= t0 + t && t0 + t + 16 <= hi;
          uint32_t before[4], fresh[4];  // bytes of tokens before lo, of new ones
          if (!whole) {
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              const int at = t0 + t + 4 * x, n0 = min(max(lo - at, 0), 4), n1 = min(max(hi - at, 0), 4);
              before[x] = (uint32_t)((1ull << 8 * n0) - 1);
              fresh[x] = (uint32_t)((1ull << 8 * n1) - 1) & ~before[x];
            }
          }
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            uint4* to = (uint4*)(codes + (int64_t)(4 * q + e) * page + t0 + t);
            if (!whole) {
              const uint4 o = *to;
              const uint32_t old[4] = {o.x, o.y, o.z, o.w};
#pragma unroll
              for (int x = 0; x < 4; ++x) {
                const uint32_t kept = shrink ? (old[x] & ~before[x]) | (rescale4(old[x], s.ratio) & before[x]) : old[x];
                out[e][x] = (out[e][x] & fresh[x]) | (kept & ~fresh[x]);
              }
            }
            *to = make_uint4(out[e][0], out[e][1], out[e][2], out[e][3]);
          }
        }
        t0 -= kChunk;
        if (t0 < g0) break;
        __syncthreads();
        for (int j = 0; j < HELD; ++j) fetch(t0, j * kThreads + tid, held[j]);
      }
    }
  }
}

}  // namespace

hipError_t launch_kv8_rotary(const RotaryArgs& a, int dtype, int64_t max_new, hipStream_t stream) {
  // a page more than the tokens fill: they may start inside one. A grid holds fewer than 2^23 workgroups of 512 threads: of
  // many pages a workgroup takes several in turn
  const int64_t groups = 2LL * a.c.heads * a.rows.seqs;
  int64_t pages = (max_new + a.c.page - 2) / a.c.page + 1;
  pages = std::max<int64_t>(1, std::min(pages, (1 << 22) / groups));
  const int64_t blocks = groups * pages;
#define GGUF_DEC_ROTARY(DT, D)                                                                       \
  {                                                                                                  \
    constexpr int per = kThreads / kLanes<D>;                                                        \
    const int64_t rows = ((int64_t)a.rows.tokens * a.hq + per - 1) / per;                            \
    const int64_t grid = blocks + std::min<int64_t>(rows, 1 << 21);                                  \
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
