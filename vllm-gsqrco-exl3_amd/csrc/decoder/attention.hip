// Causal attention over the 8-bit paged cache (attend.h: layouts; include/gguf_decoder.h: contract).
#include <algorithm>

#include "attend.h"

namespace gguf_dec {

namespace {

constexpr int kTile = 64;   // tokens a wave takes at a time
constexpr int kWaves = 4;
constexpr int kSegment = 64;  // tiles whose chunks are looked up at a time

// One workgroup takes RT = 16 NT query rows (token, head of the KV head's group) of one sequence and
// KV head, and one split of its tokens; its waves take the split's tiles in turn, straight from the cache into
// operand registers (each byte is read by one lane, so LDS would only add a hop), with statistics and
// accumulators of their own, joined through LDS at the end. Softmax is online: a wave keeps, for each row, the maximum m so
// far, its lanes' sums of 2^(s - m), and O scaled to m.
// The scale of a V chunk goes into P: p * kWeight * vs / ref, where ref is the largest vs of the chunks that the row has met and
// sees, so that P stays within fp16's range whatever the scales are, and what a row does not see takes no bits from it. P is rounded to fp16 (11 bits; the output
// has 8 or 11), everything else is fp32.
//
// Bound: HBM, 2 bytes a (token, head, dim). Measured, 24 query and 4 KV heads of 256: 64 ragged sequences of up to
// 16384 tokens 235 us a call (989 MB, 4.2 TB/s; before a wave's next tile was fetched ahead 444); one of 701 tokens 14 us,
// of which this kernel is 12, latency. At head sizes from 128 on a workgroup takes 16 rows: of 256, 32 spill, and this kernel took 148 us for 8
// sequences of 4 rows over up to 32768 tokens, 104 (the call 117) with the cache read for two row tiles; see attn_plan for the others.
//
// TREE: the rows are drafts. They see the positions before the sequence's own rows, and of these what their mask says.
template <int DT, int D, int NT, bool TREE>
__global__ void __launch_bounds__(64 * kWaves, 1) attend_kernel(AttnArgs a) {
  constexpr int S = D / 64, DD = D / 16;
  extern __shared__ __align__(16) float lds[];  // [kWaves][DD][NT][64][4]
  __shared__ float stat[kWaves][NT * 16][2];
  __shared__ Chunk chunks[4 * kSegment];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, n = lane & 15, g = lane >> 4;
  // row tiles of one (sequence, head, split) read the same tokens: a stride of gridDim.x apart, they run on as few XCDs as
  // there are, and share their L2. Later splits, which short sequences do not have, come last.
  const int head = blockIdx.x % a.c.heads, seq = blockIdx.x / a.c.heads % a.rows.seqs;
  const int split = blockIdx.x / a.c.heads / a.rows.seqs, splits = a.splits;
  int r0, r1;
  rows_of(a.rows, seq, r0, r1);
  const int64_t nrows = (int64_t)(r1 - r0) * a.group;
  const int len0 = a.lens[seq];
  const int64_t room = (int64_t)a.c.max_pages * a.c.page;
  const int page16 = a.c.page / 16;
  const int32_t* table = a.c.table + (int64_t)seq * a.c.table_stride;
  const int64_t base = (int64_t)len0 - (r1 - r0);  // position of the sequence's first row
  const int64_t drafts = TREE ? min((int64_t)(r1 - r0), (int64_t)64 * a.words) : 0;

  for (int64_t tile0 = (int64_t)blockIdx.y * 16 * NT; tile0 < nrows; tile0 += (int64_t)gridDim.y * 16 * NT) {
    // what the tile's rows see at most: they are in order of their tokens
    const int64_t rlast = min(nrows, tile0 + 16 * NT) - 1;
    const int see = (int)max(min(TREE ? (int64_t)len0 - 1 : (int64_t)len0 - (r1 - r0) + rlast / a.group, room - 1), (int64_t)-1);
    const int ntiles = (see + kTile) / kTile;  // see = -1: none
    const int tb = (int)min((int64_t)split * (a.span / kTile), (int64_t)ntiles);
    const int te = split == splits - 1 ? ntiles : min(ntiles, tb + a.span / kTile);
    const auto find_chunks = [&](int from, int to) __attribute__((always_inline)) {
      for (int i = tid; i < 4 * (to - from); i += 64 * kWaves)
        chunks[i] = chunk_of(a.c, table, page16, head, (int64_t)4 * from + i, see);
    };
    find_chunks(tb, min(tb + kSegment, te));  // (the previous rows are through: see the loop's end)
    // rows of this tile: row -> (token, head); last: the last position that it sees (of a tree: before the mask's)
    int64_t qrow[NT];
    const int64_t* mask[NT];
    int last[NT];
    int all = 0x7FFFFFFF;  // the last position that every row sees
    half8 q[NT][2 * S];
    float qs[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const int64_t r = tile0 + 16 * t + n;
      const bool ok = r < nrows;
      const int tok = ok ? (int)(r / a.group) : 0, h = head * a.group + (ok ? (int)(r % a.group) : 0);
      qrow[t] = ok ? (int64_t)(r0 + tok) * a.hq + h : -1;
      const int64_t l = ok ? (int64_t)len0 - (r1 - r0) + (TREE ? -1 : tok) : -1;
      if constexpr (TREE) mask[t] = a.mask + (int64_t)(r0 + tok) * a.mask_stride;
      last[t] = (int)(l < room ? l : room - 1);
      if (ok) all = min(all, last[t]);
      float amax = 0.0f;
      float v[2 * S][8];
#pragma unroll
      for (int s = 0; s < S; ++s)
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
          if (ok) {
            load8<DT>(a.q, (int64_t)(r0 + tok) * a.qt + (int64_t)h * a.qh + 64 * s + 16 * g + 8 * hf, v[2 * s + hf]);
          } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[2 * s + hf][e] = 0.0f;
          }
#pragma unroll
          for (int e = 0; e < 8; ++e) amax = fmaxf(amax, fabsf(v[2 * s + hf][e]));
        }
      amax = group_max(amax);
      const float f = DT == kBF16 ? row_factor(amax) : 1.0f;
      qs[t] = amax < __builtin_inff() ? a.scale / f : __builtin_nanf("");  // also where every score would be -inf
#pragma unroll
      for (int s = 0; s < 2 * S; ++s)
#pragma unroll
        for (int e = 0; e < 8; ++e) q[t][s][e] = (_Float16)(v[s][e] * f);
    }
#pragma unroll
    for (int off = 1; off < 16; off <<= 1) {
      all = min(all, __shfl_xor(all, off, 64));
    }
    if (splits > 1 && tb >= te) {  // uniform: nothing of these rows lies in the split
#pragma unroll
      for (int t = 0; t < NT; ++t)
        if (wave == 0 && g == 0 && qrow[t] >= 0)
          *(float2*)(a.stat + (split * (int64_t)a.rows.tokens * a.hq + qrow[t]) * 2) = make_float2(kNoScore, 0.0f);
      continue;
    }

    floatx4 o[DD][NT];
    float m[NT], l[NT];
    float ref[NT], inv_ref[NT];
    int seg = tb;  // chunks[0] is of this tile
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      m[t] = kNoScore;
      l[t] = ref[t] = inv_ref[t] = 0.0f;
#pragma unroll
      for (int i = 0; i < DD; ++i) o[i][t] = floatx4{0, 0, 0, 0};
    }

    // K and V of a wave's next tile are on their way while it works on this one. Lane group g looks after chunk g; the K
    // operand's rows lie in chunk n >> 2.
    uintx4 kw[4][S], vw[DD];
    const auto load_k = [&](int tile) __attribute__((always_inline)) {
      const Chunk& c = chunks[4 * (tile - seg) + (n >> 2)];
      const int8_t* kp = a.c.k + ((int64_t)c.ph * a.c.page + c.off + (n & 3)) * D + 16 * g;
#pragma unroll
      for (int tt = 0; tt < 4; ++tt)
#pragma unroll
        for (int i = 0; i < S; ++i) kw[tt][i] = *(const uintx4*)(kp + 4 * tt * D + 64 * i);
    };
    const auto load_v = [&](int tile) __attribute__((always_inline)) {
      const Chunk& c = chunks[4 * (tile - seg) + g];
      const int8_t* vp = a.c.v + ((int64_t)c.ph * D + n) * a.c.page + c.off;
#pragma unroll
      for (int i = 0; i < DD; ++i) vw[i] = *(const uintx4*)(vp + (uint32_t)(16 * i * a.c.page));
    };
    const auto work = [&](int tile, int then) __attribute__((always_inline)) {
      const float ks = chunks[4 * (tile - seg) + g].ks, vs = chunks[4 * (tile - seg) + g].vs;
      floatx4 sc[4][NT];
#pragma unroll
      for (int tt = 0; tt < 4; ++tt) {
#pragma unroll
        for (int t = 0; t < NT; ++t) sc[tt][t] = floatx4{0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < S; ++i) {
          const half8 k0 = codes8(kw[tt][i][0], kw[tt][i][1]), k1 = codes8(kw[tt][i][2], kw[tt][i][3]);
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            sc[tt][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k0, q[t][2 * i], sc[tt][t], 0, 0, 0);
            sc[tt][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k1, q[t][2 * i + 1], sc[tt][t], 0, 0, 0);
          }
        }
      }
      load_k(then);

      const bool masked = kTile * tile + kTile - 1 > all;
      float nm[NT], own[NT];  // own: the V scale of the lane's chunk, if the row sees it
      uint32_t bits[NT];      // of a tree: the tokens of the lane's chunk that the row sees
      bool grown = false;
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const float f = qs[t] * ks;
        float mx = kNoScore;
        if constexpr (TREE) bits[t] = masked ? tree_bits(mask[t], kTile * tile + 16 * g, base, drafts, room) : 0xFFFF;
#pragma unroll
        for (int tt = 0; tt < 4; ++tt)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            float x = sc[tt][t][i] * f;
            if (TREE ? !(bits[t] >> (4 * tt + i) & 1) : masked && kTile * tile + 16 * g + 4 * tt + i > last[t]) x = -__builtin_inff();
            sc[tt][t][i] = x;
            mx = fmaxf(mx, x);
          }
        // the maximum may lag: weights stay below 2^8, and the sums are scaled again only where it does not do, or
        // where the largest V scale grew
        mx = group_max(mx);
        nm[t] = mx > m[t] + 8.0f ? mx : m[t];
        own[t] = (TREE ? bits[t] == 0 : masked && kTile * tile + 16 * g > last[t]) ? 0.0f : vs;
        grown = grown || nm[t] != m[t] || own[t] > ref[t];
      }
      if (__any(grown)) {
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          const float nref = fmaxf(ref[t], group_max(own[t]));
          const float shrink = nref > ref[t] ? ref[t] / nref : 1.0f;
          ref[t] = nref;
          inv_ref[t] = nref > 0.0f ? kWeight / nref : 0.0f;
          const float al = __builtin_amdgcn_exp2f(m[t] - nm[t]);
          m[t] = nm[t];
          l[t] *= al;
#pragma unroll
          for (int i = 0; i < DD; ++i) o[i][t] *= al * shrink;
        }
      }
      half8 p[NT][2];
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const float vr = vs * inv_ref[t];
#pragma unroll
        for (int tt = 0; tt < 4; ++tt)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float x = sc[tt][t][i];
            const float e = __builtin_amdgcn_exp2f(x - m[t]);
            l[t] += e;
            // a masked place adds nothing, also where its page's scale is not finite
            p[t][tt >> 1][4 * (tt & 1) + i] = (_Float16)(masked && x == -__builtin_inff() ? 0.0f : e * vr);
          }
      }
#pragma unroll
      for (int i = 0; i < DD; ++i) {
        const half8 v0 = codes8(vw[i][0], vw[i][1]), v1 = codes8(vw[i][2], vw[i][3]);
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          o[i][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v0, p[t][0], o[i][t], 0, 0, 0);
          o[i][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v1, p[t][1], o[i][t], 0, 0, 0);
        }
      }
      load_v(then);
    };
    for (seg = tb; seg < te; seg += kSegment) {
      const int stop = min(seg + kSegment, te);
      if (seg != tb) {
        __syncthreads();
        find_chunks(seg, stop);
      }
      __syncthreads();
      int tile = seg + wave;
      if (tile < stop) {
        load_k(tile);
        load_v(tile);
      }
      // past the wave's last tile it is loaded again, for nobody
      for (; tile < stop; tile += kWaves) work(tile, tile + kWaves < stop ? tile + kWaves : tile);
    }

    // join the waves: the common maximum, then the scaled sums
    __syncthreads();
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const float sum = group_sum(l[t]);
      if (g == 0) {
        stat[wave][16 * t + n][0] = m[t];
        stat[wave][16 * t + n][1] = sum;
      }
#pragma unroll
      for (int i = 0; i < DD; ++i)
        *(floatx4*)(lds + ((((size_t)wave * DD + i) * NT + t) * 64 + lane) * 4) = o[i][t] * (ref[t] / kWeight);
    }
    __syncthreads();
    for (int i = wave; i < DD; i += kWaves) {
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const int64_t row = qrow[t];
        float mx = kNoScore, sum = 0.0f;
        floatx4 acc = {0, 0, 0, 0};
#pragma unroll
        for (int w = 0; w < kWaves; ++w) mx = fmaxf(mx, stat[w][16 * t + n][0]);
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
          const float f = __builtin_amdgcn_exp2f(stat[w][16 * t + n][0] - mx);
          sum += stat[w][16 * t + n][1] * f;
          acc += *(const floatx4*)(lds + ((((size_t)w * DD + i) * NT + t) * 64 + lane) * 4) * f;
        }
        if (row < 0) continue;
        if (splits == 1) {
          const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
          const float y[4] = {acc[0] * inv, acc[1] * inv, acc[2] * inv, acc[3] * inv};
          store4<DT>(a.out, row * D + 16 * i + 4 * g, y);
        } else {
          const int64_t all_rows = (int64_t)a.rows.tokens * a.hq;
          *(floatx4*)(a.part + (split * all_rows + row) * D + 16 * i + 4 * g) = acc;
          if (i == 0 && g == 0) *(float2*)(a.stat + (split * all_rows + row) * 2) = make_float2(mx, sum);
        }
      }
    }
    __syncthreads();  // lds is written again for the next rows
  }
}

// Joins the splits of a row. One workgroup a row: its waves take the splits in turn, 4 dims a lane, and join through LDS.
template <int DT, int D>
__global__ void __launch_bounds__(256) join_kernel(const float* __restrict__ part, const float* __restrict__ stat,
                                                   int64_t rows, int splits, void* __restrict__ out) {
  __shared__ floatx4 sums[4][64];
  __shared__ float ls[4];
  const int64_t row = blockIdx.x;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t at = min(4 * lane, D - 4);
  float mx = kNoScore;
  for (int s = lane; s < splits; s += 64) mx = fmaxf(mx, stat[(s * rows + row) * 2]);
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) mx = fmaxf(mx, __shfl_xor(mx, off, 64));
  float sum = 0.0f;
  floatx4 acc = {0, 0, 0, 0};
#pragma unroll 4
  for (int s = wave; s < splits; s += 4) {
    const float2 ml = *(const float2*)(stat + (s * rows + row) * 2);
    const floatx4 x = *(const floatx4*)(part + (s * rows + row) * D + at);
    const float f = ml.y == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(ml.x - mx);
    sum += ml.y * f;
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[e] += ml.y == 0.0f ? 0.0f : x[e] * f;  // an empty split's sums are not written
  }
  sums[wave][lane] = acc;
  if (lane == 0) ls[wave] = sum;
  __syncthreads();
  if (wave == 0 && 4 * lane < D) {
    sum = ls[0] + ls[1] + ls[2] + ls[3];
    acc = sums[0][lane] + sums[1][lane] + sums[2][lane] + sums[3][lane];
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    const float y[4] = {acc[0] * inv, acc[1] * inv, acc[2] * inv, acc[3] * inv};
    store4<DT>(out, row * D + 4 * lane, y);
  }
}

template <int DT, int D, int NT, bool TREE>
hipError_t launch_attend(const AttnArgs& a, dim3 grid, hipStream_t stream) {
  constexpr int lds = kWaves * D * 16 * NT * 4;
  int dev = 0;
  hipError_t e = hipGetDevice(&dev);
  if (e != hipSuccess) return e;
  struct Tag {};
  gguf::once_per_device<Tag>(dev, [&] {
    (void)hipFuncSetAttribute((const void*)attend_kernel<DT, D, NT, TREE>, hipFuncAttributeMaxDynamicSharedMemorySize, lds);
  });
  attend_kernel<DT, D, NT, TREE><<<grid, 64 * kWaves, lds, stream>>>(a);
  return hipGetLastError();
}

}  // namespace

// How a call is cut: rows of a workgroup, and tokens of a split so that the CUs have two workgroups each, in
// steps of a tile a wave.
// Many rows: from 64 on, about where the two forms cross in long contexts. Calls in us, few / many, at up to 16384 tokens: head
// size 256, one sequence of 24 rows 29.9 / 31.9, of 66 rows 39.8 / 34.0, eight of 24 rows 68.8 / 115, of 48 rows 114 / 120,
// of 66 rows 158 / 120; head size 128, one of 64 rows 24.1 / 28.7, of 96 rows 39.3 / 31.8, eight of 32 rows 55.3 / 97.2, of
// 64 rows 97.0 / 98.7, of 96 rows 116 / 101. (Over 2048 tokens one sequence stays quicker with few: of 66 rows 16.4 / 27.9.)
// Two row tiles a workgroup (32 rows): only at head size 64 does the cache read once make up for the waves' registers.
// Calls in us, one / two tiles, at up to 16384 tokens: head size 64, eight sequences of 64 rows 67.5 / 55.7, of 24 rows
// 39.2 / 35.6; head size 128, eight of 32 rows 55.3 / 62.6, one of 32 rows 19.4 / 27.8; head size 192, one of 24 rows
// 15.0 / 18.0, eight of 60 rows 37.9 / 40.4, of 36 rows 45.8 / 38.1.
// A tree takes its form for many rows (attention_tree.hip) by its work, since that form's fixed costs are larger: from 33 rows of a
// (sequence, KV head) on (65 of heads of 64), and 2^23 of rows times tokens over all of them (3 * 2^23 of heads up to 128). Calls in us,
// few / many: head size 256, four KV heads, 96 rows of one sequence of 16000 tokens 45.8 / 48.7, of one of 32768 84.5 / 49.2, of two of
// 16000 76.2 / 52.4, of four of 4000 61.1 / 52.4, of eight 76.7 / 50.1; 48 rows of four of 4000 36.6 / 42.7, of eight of 16000 131 / 99.6; 24 rows of
// eight of 16000 94.0 / 94.6, of 32 of 8000 196 / 168, of 64 of 16000 709 / 597; 384 rows of one of 2000 35.5 / 38.3. Head size 192, one KV head,
// 96 rows of eight of 16000 60.1 / 47.1, 192 of four of 4000 28.5 / 39.9. Head size 128, eight KV heads, 128 rows of two of 8000 37.7 /
// 54.1, of four 61.3 / 51.9, of eight of 4000 55.1 / 51.6, of 32 of 4000 306 / 117; 48 rows of eight of 16000 117 / 105, 32 rows
// 87.3 / 101. Head size 64, eight KV heads, 128 rows of two of 8000 30.9 / 46.0, of 32 of 4000 136 / 81.3; 64 rows of 32 of 2000
// 43.0 / 50.6, of 16 of 16000 133 / 129.
// At three of these points, of heads of 256, the rule takes the slower side: 96 rows of four sequences of 4000 (6.1 million rows times tokens),
// and 24 rows of 32 and of 64 sequences (as 30 rows of 32 of 16000: 371 / 311).
static bool tree_many(int d, int64_t rows, int64_t groups, int64_t max_len) {
  return rows > (d == 64 ? 64 : 32) && (double)rows * (double)groups * (double)max_len >= (d > 128 ? 1 : 3) * 8388608.0;
}

struct AttnPlan {
  bool many;
  int nt, span, splits;
  int64_t row_tiles;
};

static AttnPlan attn_plan(int d, int64_t rows, int64_t groups, int64_t max_len, int64_t most, bool tree) {
  AttnPlan p;
  p.many = !tree && rows > 64;
  p.nt = rows > 16 && d < 128 ? 2 : 1;
  const int64_t tile = p.many ? kRowsTile : 16 * p.nt;
  p.row_tiles = (rows + tile - 1) / tile;
  const int64_t blocks = groups * p.row_tiles, step = kTile * kWaves;
  const int64_t steps = (max_len + step - 1) / step;
  int64_t want = (2 * gguf::device_cus() + blocks - 1) / blocks;
  if (want > most) want = most;
  if (want < 1) want = 1;
  const int64_t each = (steps + want - 1) / want;
  p.span = (int)(each * step < (1 << 30) ? each * step : (1 << 30));
  p.splits = (int)((steps + each - 1) / each);
  if (p.splits < 1) p.splits = 1;
  return p;
}

// splits of a call of that many rows: join_kernel's grid, a workgroup a row, holds fewer than 2^32 threads
static int64_t most_splits(int64_t rows) { return rows < (1 << 24) ? 512 : 1; }

size_t kv8_attention_workspace(int d, int heads, int hq, int64_t tokens, int64_t seqs, int64_t max_new,
                               int64_t max_len, bool tree) {
  if (tree && tree_many(d, max_new * (hq / heads), seqs * heads, max_len))
    return tree_workspace(d, max_new * (hq / heads), tokens, hq, seqs, heads, max_len);
  const AttnPlan p = attn_plan(d, max_new * (hq / heads), seqs * heads, max_len, most_splits(tokens * hq), tree);
  return p.splits == 1 ? 0 : (size_t)p.splits * tokens * hq * (d + 2) * sizeof(float);
}

hipError_t launch_kv8_attention(const Kv8& c, int dtype, const void* q, int64_t qt, int64_t qh, int hq,
                                const int32_t* lens, const Ragged& rows, int64_t max_new, int64_t max_len, float scale,
                                const int64_t* mask, int64_t mask_stride, int words, void* out, void* ws, size_t ws_bytes,
                                hipStream_t stream) {
  if (mask && tree_many(c.d, max_new * (hq / c.heads), (int64_t)rows.seqs * c.heads, max_len)) {
    const AttnArgs a{c, q, qt, qh, lens, rows, hq, hq / c.heads, scale * kLog2e, 0, 0, out, nullptr, nullptr, mask, mask_stride, words, dtype};
    return launch_attend_tree(a, max_new * (hq / c.heads), max_len, ws, stream);
  }
  const int64_t all = (int64_t)rows.tokens * hq;
  const int64_t fit = (int64_t)(ws_bytes / sizeof(float)) / (all * (c.d + 2));
  const AttnPlan p = attn_plan(c.d, max_new * (hq / c.heads), (int64_t)rows.seqs * c.heads, max_len,
                               fit < 2 ? 1 : std::min(fit, most_splits(all)), mask != nullptr);
  const AttnArgs a{c, q, qt, qh, lens, rows, hq, hq / c.heads, scale * kLog2e, p.span, p.splits, out, (float*)ws,
                   (float*)ws + (size_t)p.splits * all * c.d, mask, mask_stride, words, dtype};
  const dim3 grid((unsigned)(rows.seqs * c.heads * p.splits), (unsigned)(p.row_tiles < 65535 ? p.row_tiles : 65535));
  hipError_t e = hipSuccess;
  if (p.many) e = launch_attend_rows(a, dtype, p.row_tiles, stream);
#define GGUF_DEC_ATTEND(DT, D)                                                                                         \
  {                                                                                                                    \
    if (!p.many && p.nt == 1) e = mask ? launch_attend<DT, D, 1, true>(a, grid, stream) : launch_attend<DT, D, 1, false>(a, grid, stream); \
    if constexpr (D < 128)                                                                                             \
      if (!p.many && p.nt == 2) e = mask ? launch_attend<DT, D, 2, true>(a, grid, stream) : launch_attend<DT, D, 2, false>(a, grid, stream); \
    if (e == hipSuccess && p.splits > 1)                                                                               \
      join_kernel<DT, D><<<(unsigned)all, 256, 0, stream>>>(a.part, a.stat, all, p.splits, out);           \
  }
#define GGUF_DEC_ATTEND_D(DT)                 \
  switch (c.d) {                              \
    case 64: GGUF_DEC_ATTEND(DT, 64) break;   \
    case 128: GGUF_DEC_ATTEND(DT, 128) break; \
    case 192: GGUF_DEC_ATTEND(DT, 192) break; \
    default: GGUF_DEC_ATTEND(DT, 256) break;  \
  }
  if (dtype == kF16) {
    GGUF_DEC_ATTEND_D(kF16)
  } else {
    GGUF_DEC_ATTEND_D(kBF16)
  }
#undef GGUF_DEC_ATTEND_D
#undef GGUF_DEC_ATTEND
  return e == hipSuccess ? hipGetLastError() : e;
}

}  // namespace gguf_dec
