// Attention for trees of drafts over the 8-bit paged cache, for many rows a KV head: some ten to some hundred rows that all see a
// long context, and of each other what their masks say.
//
// Both products are transposed, S^T = K Q^T and O^T += V^T P^T, in fp16 with 32 x 32 MFMAs, so that a lane keeps one query row. With
// lane = 32 h + n, a result's element i is row 8 (i >> 2) + 4 h + (i & 3) of column n; the 32 tokens of a block stand in K's rows in
// such an order that the lane's 8 scores i = 8 c .. 8 c + 7 are its places of the c-th step of the second product: tokens 16 c +
// 8 h + 0 .. 7. Scores never cross lanes. Codes become fp16 on the way to LDS, exactly.
//   - A tile is 64 tokens. Up to 128 dims a wave takes 32 rows for itself; beyond, two waves share 32 rows (PAIR), either with half
//     of the output's dims, so that two waves fit a SIMD, and each takes 32 scores a row; weights and running maxima go to the partner
//     through LDS. A maximum lags its scores by up to 2^8 and is a whole number, so that a partner's weights are brought to the larger
//     of the two by a power of two, exactly.
//   - A wave's tile is two steps, products and weights, and the two waves of a SIMD are a step apart: one's matrix instructions run
//     beside the other's softmax and conversions. (32 sequences of 64 drafts at 8192 tokens, 32 query and 8 KV heads of 128: 413 us,
//     in step 455; at 256 dims, where partners wait for each other anyway, no difference.)
//   - The tiles of all (sequence, head, row tile)s in a line are cut into equal shares, one a workgroup and CU, whatever the lengths
//     are. A workgroup whose share begins or ends inside a group leaves its sums to join_tree_kernel; a group that lies in one share is
//     written at once.
// Queries are exact in fp16, but for bf16 elements below 2^-14 of the row's largest, and weights are rounded to fp16; scores, sums of
// weights and outputs are fp32. As integers in two int8 planes, queries cost two instructions more a score and as much matrix time:
// up to 128 dims slower (502 us to 419, the case above), beyond quicker (206 to 217, 21 drafts of 8 sequences of 32768 tokens, 24 query and
// 4 KV heads of 256), where a second set of operands and rounded queries were not worth it.
//
// Weights are in fp16 as the matrix instructions take 16 bits: bf16 would leave them 8 bits for 11, and a second plane of them would double the
// second product. Against 64 bits this takes the error of fp16 outputs from their own rounding's 2.1e-4 (relative, all of an output) to
// 2.9e-4; bf16 outputs' stays 1.7e-3.
//
// What bounds it: by clock values stored by each workgroup, a step takes 2200 to 2600 cycles, the products' 32 matrix instructions 1024 of them on
// a SIMD; the weights' 270 to 300 vector instructions, 16 or 32 of them exponentials, with their waits for LDS and each other the rest.
// Outside the steps a piece (a share's part of one group) takes some 17500 cycles for its start, where places, K's first tiles and the
// queries are loaded one behind the other, and 7500 for its last product and its sums: 14 of 76 us on average where a share is one
// piece (16 drafts of 8 ragged sequences to 32768 tokens, 24 query and 4 KV heads of 256: 101 us a call), 14 of 58 (47 drafts of 4 to 16000:
// 83), 24 of 156 at two pieces (64 drafts of 32 to 8192, 32 query and 8 KV heads of 128: 224). The products alone take 28, 20 and 88 at a
// library product's rate.
#include <algorithm>
#include <type_traits>

#include "attend.h"

namespace gguf_dec {

namespace {

typedef float floatx16 __attribute__((ext_vector_type(16)));

constexpr int kToks = 64;                // tokens of a tile
constexpr int kVRow = 2 * kToks + 16;    // bytes of a dim's row of V in LDS; 16 more than its values, for the banks
constexpr int kAhead = 16;               // tiles whose chunks are looked up at a time
constexpr int kPlaces = 4 * 2 * kAhead;  // places of chunks that are held: those of tile t at 4 (t % (2 kAhead))
constexpr int kLeastTiles = 4;           // of a workgroup's share
constexpr int kParts = 32;               // of a group that is cut, for a wave

// v, made again where it is needed: what comes of a thread's number (its places in LDS and memory) would otherwise be kept over the
// tiles, in registers that the products need
__device__ __forceinline__ int again(int v) {
  asm volatile("" : "+v"(v));
  return v;
}

// Where a chunk's K and V lie, and its scales.
struct Place {
  int64_t k, v;
  float ks, vs;
};

// A group of tiles that lies in several shares, from share `first` on (it begins there) to `last`, and what its rows are.
struct Cut {
  int first, last, own;  // own: it is the first of share `first`
  int head, r0;          // KV head; the sequence's first token
  int64_t row0;          // the group's first row among the sequence's of the head
  int rows;
};

// Queries as the products take them, and the line of all tiles, cut: what prep_tree_kernel leaves.
struct Prep {
  _Float16* q;     // [tokens * hq][d]: bf16 times a power of two that brings the row's largest to 1 .. 2; and the call's scale's sign
  float* qs;       // [tokens * hq]: what they are multiplied by, with the call's scale
  int64_t* line;   // [seqs + 1]: tiles before a sequence's
  int* begins;     // [shares]: the sequence in which a share begins
  int* cuts;       // how many groups are cut
  Cut* cut;        // [shares]
};

// PAIR: two waves share 32 rows
template <int D, int NW>
struct Lay {
  static constexpr bool kPair = D > 128;
  static constexpr int kThreads = 64 * NW, kRows = kPair ? 16 * NW : 32 * NW;
  static constexpr int kKRow = 2 * D + 16;                       // bytes of a token's row of K
  static constexpr int kK = 0;                                   // [2][64][kKRow]
  static constexpr int kV = kK + 2 * kToks * kKRow;              // [2][D][kVRow]
  static constexpr int kP = kV + 2 * D * kVRow;                  // [waves][2][64] x 16 bytes, of pairs
  static constexpr int kPlace = kP + (kPair ? NW * 2048 : 0);    // Place [kPlaces]
  static constexpr int kStat = kPlace + 24 * kPlaces;            // float [waves][32], of pairs
  static constexpr int kBytes = kStat + (kPair ? NW * 128 : 0);
};

// tiles of a sequence's rows: 0 without rows, at least one with them (it writes the zeros of rows that see nothing)
struct Seq {
  int r0, n, tiles, row_tiles;
  int64_t len;
};

__device__ __forceinline__ Seq seq_of(const AttnArgs& a, int s, int rows) {
  Seq q;
  int r1;
  rows_of(a.rows, s, q.r0, r1);
  q.n = r1 - q.r0;
  q.len = a.lens[s];
  const int64_t room = (int64_t)a.c.max_pages * a.c.page;
  const int64_t see = min(q.len, room);
  q.tiles = q.n == 0 ? 0 : (int)max((see + kToks - 1) / kToks, (int64_t)1);
  q.row_tiles = (int)(((int64_t)q.n * a.group + rows - 1) / rows);
  return q;
}

// The two words of a row's mask that hold the tile at position `at`; nothing is read beyond the mask's `count` rows.
struct Words {
  uint64_t lo, hi;
};

__device__ __forceinline__ Words words_of(const int64_t* mask, int at, int base, int count) {
  const int64_t from = (int64_t)at - base, i = from >> 6;  // (the tile begins in word i, or before the first)
  Words w{0, 0};
  if (i >= 0 && 64 * i < count) w.lo = (uint64_t)mask[i];
  if (i + 1 >= 0 && 64 * (i + 1) < count) w.hi = (uint64_t)mask[i + 1];
  return w;
}

// What the row sees of the tile, a bit a token (attend.h: tree_bits).
__device__ __forceinline__ uint64_t seen_of(const Words& w, int at, int base, int count, int room) {
  const auto below = [](int64_t n) { return n >= 64 ? ~0ull : n <= 0 ? 0ull : (1ull << n) - 1; };
  const int64_t from = (int64_t)at - base;
  const int shift = (int)(from & 63);
  const uint64_t own = shift ? w.lo >> shift | w.hi << (64 - shift) : w.lo;
  return ((own & below(count - from)) | below(-from)) & below((int64_t)room - at);
}

// How the line of all tiles is cut: share w of `shares` is [w total / shares, (w + 1) total / shares).
struct Line {
  int64_t total, shares;
  __device__ Line(int64_t all, int64_t most) : total(all) {
    shares = min(most, max((total + kLeastTiles - 1) / kLeastTiles, (int64_t)1));
  }
  __device__ int64_t begin(int64_t w) const { return w * total / shares; }
};

// Queries in fp16, four values a lane; and, by the first workgroup, the tiles before each sequence's, where the
// shares begin, and which groups they cut.
template <int DT, int D>
__global__ void __launch_bounds__(256) prep_tree_kernel(AttnArgs a, Prep p, int rows, int64_t most) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  if (blockIdx.x == 0) {
    constexpr int HELD = 1024;  // sequences whose line is looked up in LDS
    __shared__ int64_t part[4], held[HELD];
    int64_t total = 0;
    for (int s0 = 0; s0 < a.rows.seqs; s0 += 256) {
      const int s = s0 + tid;
      int64_t cost = 0;
      if (s < a.rows.seqs) {
        const Seq q = seq_of(a, s, rows);
        cost = (int64_t)a.c.heads * q.row_tiles * q.tiles;
      }
      int64_t x = cost;
#pragma unroll
      for (int off = 1; off < 64; off <<= 1) {
        const int64_t y = __shfl_up(x, off, 64);
        if (lane >= off) x += y;
      }
      __syncthreads();
      if (lane == 63) part[wave] = x;
      __syncthreads();
      int64_t before = total;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        if (w < wave) before += part[w];
        total += part[w];
      }
      if (s < a.rows.seqs) p.line[s] = before + x - cost;
      if (s < HELD) held[s] = before + x - cost;
    }
    if (tid == 0) p.line[a.rows.seqs] = total, *p.cuts = 0;
    __syncthreads();
    const Line line(total, most);
    const bool all_held = a.rows.seqs <= HELD;
    for (int64_t w = tid; w < line.shares && total > 0; w += 256) {
      const int64_t at = line.begin(w);
      int s = 0;  // the last sequence with line[s] <= at: one that has tiles
      for (int lo = 0, hi = a.rows.seqs - 1; lo <= hi;) {
        const int mid = lo + (hi - lo) / 2;
        if ((all_held ? held[mid] : p.line[mid]) <= at) s = mid, lo = mid + 1;
        else hi = mid - 1;
      }
      p.begins[w] = s;
      if (w == 0) continue;
      const Seq q = seq_of(a, s, rows);
      const int64_t from = all_held ? held[s] : p.line[s], group = (at - from) / q.tiles, lo = from + group * q.tiles, hi = lo + q.tiles;
      if (at == lo || line.begin(w - 1) > lo) continue;  // it begins with the group, or an earlier share's begin lies inside it
      const int64_t last = (hi * line.shares + line.total - 1) / line.total - 1;  // the last share that begins before hi
      const int64_t row0 = group % q.row_tiles * rows;
      p.cut[atomicAdd(p.cuts, 1)] = Cut{(int)w - 1, (int)last, line.begin(w - 1) == lo, (int)(group / q.row_tiles), q.r0, row0,
                                        (int)min((int64_t)rows, (int64_t)q.n * a.group - row0)};
    }
    return;
  }
  constexpr int L = D == 192 ? 64 : D / 4, ROWS = 256 / L;  // lanes of a row (of 192 dims some idle), rows a workgroup
  const int64_t all = (int64_t)a.rows.tokens * a.hq;
  const int at = min(4 * (tid % L), D - 4);
  for (int64_t r0 = ((int64_t)blockIdx.x - 1) * ROWS; r0 < all; r0 += (int64_t)(gridDim.x - 1) * ROWS) {
    const int64_t r = min(r0 + tid / L, all - 1), tok = r / a.hq;  // (lanes past the last row take it again)
    const uint2 w = *(const uint2*)((const uint16_t*)a.q + tok * a.qt + (r - tok * a.hq) * a.qh + at);
    const uint32_t bits[4] = {w.x & 0xFFFF, w.x >> 16, w.y & 0xFFFF, w.y >> 16};
    float v[4];
    uint32_t big = 0;  // NaN and inf on top: then the row's scores are NaN
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      v[e] = DT == kF16 ? gguf::half_bits_to_float(bits[e]) : __uint_as_float(bits[e] << 16);
      big = max(big, __float_as_uint(v[e]) & 0x7FFFFFFFu);
    }
#pragma unroll
    for (int off = 1; off < L; off <<= 1) big = max(big, (uint32_t)__shfl_xor((int)big, off, 64));
    // fp16 queries as they are: scaled, elements 2^-15 of the row's largest would become subnormal and lose bits
    const float amax = __uint_as_float(big), by = DT == kBF16 ? row_factor(amax) : 1.0f, to = a.scale < 0.0f ? -by : by;
    *(uint2*)(p.q + r * D + at) = make_uint2(pack2<kF16>(v[0] * to, v[1] * to), pack2<kF16>(v[2] * to, v[3] * to));
    // not negative: the scale's sign is the queries'
    if (tid % L == 0) p.qs[r] = amax < __builtin_inff() ? fabsf(a.scale) / by : __builtin_nanf("");
  }
}

// A workgroup's share. Sums of a group that it does not have alone: slot 2 w of one in which share w begins, 2 w + 1 of a later one.
//
// A tile is two steps of a wave: products (the tile before's O^T += V^T P^T, then S^T = K Q^T), and weights (softmax, and the tiles' way
// to LDS), with a barrier behind each. The first four waves, one a SIMD, and the others (LAG: there are others) are a step apart,
// so that on a SIMD one wave's products run beside the other's weights. The first bring V: tile t's in the step of its weights, over
// tile t - 2's, which the others have read a step before. The others bring K: tile t + 2's in the step of tile t's weights, over tile t's.
template <int D, int NW>
__global__ void __launch_bounds__(64 * NW) __attribute__((amdgpu_waves_per_eu(NW > 4 || D <= 128 ? 2 : 1, NW > 4 || D <= 128 ? 2 : 1)))
attend_tree_kernel(AttnArgs a, Prep prep, int64_t most) {
  using L = Lay<D, NW>;
  constexpr bool LAG = NW > 4, PAIR = L::kPair;
  constexpr int KS = D / 16;                    // steps of the first product
  constexpr int DD = PAIR ? D / 64 : D / 32;    // 32-dim tiles of the wave's dims: of a pair's wave half of all
  constexpr int B = PAIR ? 1 : 2;               // the wave's blocks of 32 tokens of a tile
  constexpr int PIECES = 4 * D;                 // 16-byte pieces of a tile's K, and of its V
  constexpr int FIRST = L::kThreads / 2;        // threads that bring V, and as many K
  constexpr int NP = PIECES / FIRST;
  static_assert(PIECES % FIRST == 0, "whole turns");
  extern __shared__ __align__(16) char lds[];
  Place* places = (Place*)(lds + L::kPlace);
  float* stat = (float*)(lds + L::kStat);
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), n = lane & 31, h = lane >> 5;
  const int rg = PAIR ? wave >> 1 : wave, half = PAIR ? wave & 1 : 0;
  const bool brings_v = wave < FIRST / 64, late = LAG && !brings_v;
  const int room = (int)min((int64_t)a.c.max_pages * a.c.page, (int64_t)INT32_MAX);

  const Line line(prep.line[a.rows.seqs], most);
  if ((int64_t)blockIdx.x >= line.shares || line.total == 0) return;
  const int64_t begin = line.begin(blockIdx.x), end = line.begin((int64_t)blockIdx.x + 1);
  int seq = prep.begins[blockIdx.x];

  for (int64_t pos = begin; pos < end;) {
    while (pos >= prep.line[seq + 1]) ++seq;  // (sequences without rows cost nothing)
    const Seq q = seq_of(a, seq, L::kRows);
    const int64_t in_seq = pos - prep.line[seq], group = in_seq / q.tiles;
    const int tb = (int)(in_seq - group * q.tiles), te = (int)min((int64_t)q.tiles, tb + (end - pos));
    const int head = (int)(group / q.row_tiles), rt = (int)(group - (int64_t)head * q.row_tiles);
    const bool whole = tb == 0 && te == q.tiles, first = pos == begin;
    pos += te - tb;

    const int32_t* table = a.c.table + (int64_t)seq * a.c.table_stride;
    const int see = (int)min(q.len, (int64_t)room) - 1;
    // position of the sequence's first row; below -2^30 no position is one of its rows (their masks hold 2^30 bits at most)
    const int base = (int)max(q.len - q.n, -((int64_t)1 << 30));
    const int drafts = (int)min((int64_t)q.n, (int64_t)64 * a.words);
    const int open = min(base, room);  // positions that every row sees
    const int tlast = te - 1;
    const auto places_of = [&](int t) __attribute__((always_inline)) { return places + 4 * (t & (2 * kAhead - 1)); };
    const auto find_places = [&](int from, int tiles, int threads) __attribute__((always_inline)) {
      for (int i = again(tid); i < 4 * tiles; i += threads) {
        const Chunk c = chunk_of(a.c, table, a.c.page / 16, head, (int64_t)4 * from + i, see);
        places_of(from + (i >> 2))[i & 3] =
            Place{((int64_t)c.ph * a.c.page + c.off) * D, (int64_t)c.ph * a.c.page * D + c.off, c.ks, c.vs};
      }
    };

    // A thread's pieces, j * FIRST + me, of V (chunk p & 3 of dim p >> 2) or of K (row p / (D / 16)), on their way.
    uintx4 raw[NP];
    const auto load_v = [&](int t) __attribute__((always_inline)) {
      const int me = again(tid);
      const int8_t* from = a.c.v + places_of(t)[me & 3].v;
#pragma unroll
      for (int j = 0; j < NP; ++j) raw[j] = *(const uintx4*)(from + (uint32_t)((j * (FIRST / 4) + (me >> 2)) * a.c.page));
    };
    const auto load_k = [&](int t) __attribute__((always_inline)) {
      const int me = again(tid - FIRST);
      const Place* at = places_of(t);
#pragma unroll
      for (int j = 0; j < NP; ++j) {
        const uint32_t p = j * FIRST + me, row = p / (D / 16);
        raw[j] = *(const uintx4*)(a.c.k + at[row >> 4].k + (row & 15) * D + 16 * (p % (D / 16)));
      }
    };
    const auto put_v = [&](int t) __attribute__((always_inline)) {
      const int me = again(tid);
      char* to = lds + L::kV + (t & 1) * D * kVRow + (me >> 2) * kVRow + 32 * (me & 3);
#pragma unroll
      for (int j = 0; j < NP; ++j) {
        *(half8*)(to + j * (FIRST / 4) * kVRow) = codes8(raw[j][0], raw[j][1]);
        *(half8*)(to + j * (FIRST / 4) * kVRow + 16) = codes8(raw[j][2], raw[j][3]);
      }
    };
    const auto put_k = [&](int t) __attribute__((always_inline)) {
      const int me = again(tid - FIRST);
#pragma unroll
      for (int j = 0; j < NP; ++j) {
        const uint32_t p = j * FIRST + me;
        char* to = lds + L::kK + (t & 1) * kToks * L::kKRow + p / (D / 16) * L::kKRow + 32 * (p % (D / 16));
        *(half8*)to = codes8(raw[j][0], raw[j][1]);
        *(half8*)(to + 16) = codes8(raw[j][2], raw[j][3]);
      }
    };
    __syncthreads();  // what the last piece left in LDS has been read
    find_places(tb, 2 * kAhead, L::kThreads);
    __syncthreads();

    const int64_t row0 = (int64_t)rt * L::kRows;
    const int tok0 = (int)(row0 / a.group), head0 = (int)(row0 - (int64_t)tok0 * a.group);
    const int left = (int)min((int64_t)q.n * a.group - row0, (int64_t)L::kRows);
    // the lane's row: its token (of the first row if it is none), and its place among all rows
    struct Row {
      bool ok;
      int tok;
      int64_t at;
    };
    const auto row_of = [&]() __attribute__((always_inline)) {
      const int r = 32 * rg + (again(lane) & 31);
      Row x;
      x.ok = r < left;
      const uint32_t y = head0 + (x.ok ? r : 0), z = y / (uint32_t)a.group;
      x.tok = q.r0 + tok0 + (int)z;
      x.at = (int64_t)x.tok * a.hq + head * a.group + (int)(y - z * a.group);
      return x;
    };

    half8 qf[KS];
    const Row row = row_of();
    const float qs = prep.qs[row.at];
    const _Float16* qp = prep.q + row.at * D + 8 * h;
#pragma unroll
    for (int i = 0; i < KS; ++i) qf[i] = *(const half8*)(qp + 16 * i);
    if (brings_v) {
      load_v(tb);
    } else {
      load_k(tb);
      put_k(tb);
      load_k(min(tb + 1, tlast));
      put_k(tb + 1);
      load_k(min(tb + 2, tlast));
    }
    floatx16 o[DD];
    float m = kNoScore, l = 0.0f, ref = 0.0f, inv_ref = 0.0f;
#pragma unroll
    for (int i = 0; i < DD; ++i)
#pragma unroll
      for (int e = 0; e < 16; ++e) o[i][e] = 0.0f;
#pragma unroll
    for (int i = 0; i < KS; ++i) asm volatile("" : "+v"(qf[i]));  // here: not waited for with the tiles' loads

    half8* const weights = (half8*)(lds + L::kP);  // [waves][2][64]: for the waves' partners
    const int krow = 32 * half + 16 * (n >> 4) + 8 * ((n >> 2) & 1) + 4 * ((n >> 3) & 1) + (n & 3);  // token of K's row n
    const char* const k0 = lds + L::kK + krow * L::kKRow + 16 * h;
    const char* const v0 = lds + L::kV + (half * (D / 2) + n) * kVRow + 16 * h;
    half8 p[4];  // the weights of a tile: the wave's own, then its partner's
    // The products of a step, two MFMAs at a time: O^T of tile t - 1 (the wave's dims; its own tokens' weights, then its
    // partner's), then S^T of the wave's tokens of tile t. Operands are read two pairs ahead.
    // BACK: the first, FRONT: the second.
    floatx16 s[B];
    const auto products = [&](int t, auto back, auto front) __attribute__((always_inline)) {
      constexpr bool BACK = decltype(back)::value, FRONT = decltype(front)::value;
      constexpr int P2 = BACK ? 2 * DD : 0, PAIRS = P2 + (FRONT ? B * KS / 2 : 0);
      const char* const vt = v0 + ((t - 1) & 1) * D * kVRow;
      const char* const kt = k0 + (t & 1) * kToks * L::kKRow;
      half8 v[BACK ? 4 * DD : 1];
      half8 k[B * KS];  // of a block of tokens, or of two in turn
      const auto fetch = [&](int r) __attribute__((always_inline)) {  // the operands of pair r
        if (r < P2) {
#pragma unroll
          for (int f = 2 * r; f < 2 * r + 2; ++f)
            v[f] = *(const half8*)(vt + 64 * (half ^ (f / DD >> 1)) + 32 * (f / DD & 1) + 32 * (f % DD) * kVRow);
        } else if (r < PAIRS) {
#pragma unroll
          for (int f = 2 * (r - P2); f < 2 * (r - P2) + 2; ++f) k[f] = *(const half8*)(kt + f % B * 32 * L::kKRow + 32 * (f / B));
        }
      };
      if constexpr (BACK && PAIR) {
        const int me = again(lane);
        const float other = stat[32 * (wave ^ 1) + (me & 31)];
        const half8* const theirs = weights + 64 * 2 * (wave ^ 1) + me;
        p[2] = theirs[0];
        p[3] = theirs[64];
        fetch(0);
        fetch(1);
        if (__any(other != m)) {  // one of the partners has raised its maximum: both go on with the larger
          const float nm = fmaxf(m, other), al = __builtin_amdgcn_exp2f(m - nm), be = __builtin_amdgcn_exp2f(other - nm);
          m = nm;
          l *= al;
#pragma unroll
          for (int i = 0; i < DD; ++i) o[i] *= al;
#pragma unroll
          for (int c = 0; c < 4; ++c) p[c] *= (_Float16)(c < 2 ? al : be);  // by powers of two: the maxima are whole numbers
        }
      } else {
        fetch(0);
        fetch(1);
      }
      if constexpr (FRONT) {
#pragma unroll
        for (int c = 0; c < B; ++c)
#pragma unroll
          for (int e = 0; e < 16; ++e) s[c][e] = 0.0f;
      }
#pragma unroll
      for (int r = 0; r < PAIRS; ++r) {
        fetch(r + 2);
        __builtin_amdgcn_sched_barrier(0);
        if (r < P2) {
#pragma unroll
          for (int f = 2 * r; f < 2 * r + 2; ++f)
            o[f % DD] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v[f], p[f / DD], o[f % DD], 0, 0, 0);
        } else {
#pragma unroll
          for (int f = 2 * (r - P2); f < 2 * (r - P2) + 2; ++f)
            s[f % B] = __builtin_amdgcn_mfma_f32_32x32x16_f16(k[f], qf[f / B], s[f % B], 0, 0, 0);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    };

    __syncthreads();
    if (late) __syncthreads();
    for (int t = tb; t < te; ++t) {
      const bool masked = kToks * t + kToks > open;  // some row does not see all
      Words words{0, 0};
      if (masked) words = words_of(a.mask + row_of().tok * a.mask_stride, kToks * t, base, drafts);
      if (t > tb) products(t, std::true_type(), std::true_type());
      else products(t, std::false_type(), std::true_type());
      const Place* at = places_of(t);
      float own[2 * B], f[2 * B];  // of the wave's chunks
#pragma unroll
      for (int c = 0; c < 2 * B; ++c) {
        own[c] = at[2 * half + c].vs;
        f[c] = qs * at[2 * half + c].ks;
      }
      // the largest V scale of the chunks that the row sees (a NaN counts for nothing)
      float highest = fmaxf(fmaxf(at[0].vs, at[1].vs), fmaxf(at[2].vs, at[3].vs));
      __syncthreads();

      if (brings_v) {
        put_v(t);
        load_v(min(t + 1, tlast));
        if (((t - tb) & (kAhead - 1)) == 0 && t != tb && t + kAhead <= tlast) find_places(t + kAhead, kAhead, FIRST);
      } else {
        put_k(t);  // tile t + 2's, in tile t's place
        load_k(min(t + 3, tlast));
      }
      // scores are s f. Where some row does not see all, or scores are so large that an fma's rest would pass any weight, they are
      // multiplied for themselves, and f is 1.
      const auto scaled = [&](int c, int e) __attribute__((always_inline)) {
        float x = s[c][e] * f[2 * c + (e >> 3)];
        asm("" : "+v"(x));
        return x;
      };
      if (masked) {
        const uint64_t seen = seen_of(words, kToks * t, base, drafts, room);
        highest = 0.0f;
#pragma unroll
        for (int c = 0; c < 4; ++c)
          if (seen >> 16 * c & 0xFFFF) highest = fmaxf(highest, at[c].vs);
#pragma unroll
        for (int c = 0; c < 2 * B; ++c) {
          const uint32_t bits = (uint32_t)(seen >> (32 * half + 16 * c)) & 0xFFFF;
          if (bits == 0) own[c] = 0.0f;  // also where the page's scale is not finite
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float x = scaled(c >> 1, 8 * (c & 1) + e);
            s[c >> 1][8 * (c & 1) + e] = bits >> (8 * h + e) & 1 ? x : -__builtin_inff();
          }
          f[c] = 1.0f;
        }
      }
      float mx = kNoScore;
#pragma unroll
      for (int c = 0; c < 2 * B; ++c) {
        float big = s[c >> 1][8 * (c & 1)];
#pragma unroll
        for (int e = 1; e < 8; ++e) big = fmaxf(big, s[c >> 1][8 * (c & 1) + e]);
        mx = fmaxf(mx, big * f[c]);
      }
      mx = half_max(mx);
      // the maximum may lag: weights stay below 2^8, and the sums are scaled again only where it does not do, or
      // where the largest V scale grew
      const bool raise = mx > m + 8.0f;
      if (__any(raise || highest > ref)) {
        const float nref = fmaxf(ref, highest), nm = raise ? ceilf(mx) : m, al = __builtin_amdgcn_exp2f(m - nm);
        const float by = nref > ref ? al * (ref / nref) : al;
        l *= al;
#pragma unroll
        for (int i = 0; i < DD; ++i) o[i] *= by;
        m = nm;
        ref = nref;
        inv_ref = nref > 0.0f ? kWeight / nref : 0.0f;
      }
      if (__any(fabsf(m) > 0x1p20f)) {
#pragma unroll
        for (int c = 0; c < 2 * B; ++c) {
#pragma unroll
          for (int e = 0; e < 8; ++e) s[c >> 1][8 * (c & 1) + e] = scaled(c >> 1, 8 * (c & 1) + e);
          f[c] = 1.0f;
        }
      }
#pragma unroll
      for (int c = 0; c < 2 * B; ++c) {
        const float vr = own[c] * inv_ref;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float w = __builtin_amdgcn_exp2f(__builtin_fmaf(s[c >> 1][8 * (c & 1) + e], f[c], -m));
          l += w;
          p[c][e] = (_Float16)(w * vr);
        }
      }
      if constexpr (PAIR) {
        const int me = again(lane);
        half8* const ours = weights + 64 * 2 * wave + me;
        stat[32 * wave + (me & 31)] = m;
        ours[0] = p[0];
        ours[64] = p[1];
      }
      __syncthreads();
    }
    products(te, std::true_type(), std::false_type());
    __syncthreads();
    if (LAG && !late) __syncthreads();

    // the rows' sums over both halves of the tokens
    l += __shfl_xor(l, 32, 64);
    if constexpr (PAIR) {
      if (h == 0) stat[32 * wave + n] = l;
      __syncthreads();
      l += stat[32 * (wave ^ 1) + n];
    }
    const Row mine = row_of();
    if (!mine.ok) continue;
    const float by = ref / kWeight;
    if (whole) {
      const float inv = l == 0.0f ? 0.0f : by / l;
#pragma unroll
      for (int i = 0; i < DD; ++i)
#pragma unroll
        for (int e = 0; e < 16; e += 4) {
          const int64_t to = mine.at * D + half * (D / 2) + 32 * i + 2 * e + 4 * h;
          const float y[4] = {o[i][e] * inv, o[i][e + 1] * inv, o[i][e + 2] * inv, o[i][e + 3] * inv};
          if (a.dtype == kF16) store4<kF16>(a.out, to, y);
          else store4<kBF16>(a.out, to, y);
        }
    } else {
      const int64_t r = (2 * (int64_t)blockIdx.x + !first) * L::kRows + 32 * rg + n;
#pragma unroll
      for (int i = 0; i < DD; ++i)
#pragma unroll
        for (int e = 0; e < 16; e += 4)
          *(floatx4*)(a.part + r * D + half * (D / 2) + 32 * i + 2 * e + 4 * h) =
              floatx4{o[i][e] * by, o[i][e + 1] * by, o[i][e + 2] * by, o[i][e + 3] * by};
      if (h == 0 && half == 0) *(float2*)(a.stat + r * 2) = make_float2(m, l);
    }
  }
}

// Joins the rows of the groups that are cut. Of up to kParts parts a wave takes some rows at a time, AT parts' loads under way at once; of
// more a workgroup takes a row, its waves the parts in turn. Bound by memory: two groups' sums a share at most, some 30 MB of the first
// case above and 60 of the last, in 10 and 13 us.
template <int D>
__global__ void __launch_bounds__(256) join_tree_kernel(AttnArgs a, Prep prep, int rows, int most) {
  constexpr int E = D / 64, AT = 4;
  __shared__ float sums[4][64][E];
  __shared__ float ls[4];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int cuts = *prep.cuts;
  for (int i = blockIdx.y; i < most; i += gridDim.y) {
    const Cut cut = prep.cut[i];  // fetched beside their number
    if (i >= cuts) break;
    const auto slot = [&](int w, int64_t r) { return (2 * (int64_t)w + (w == cut.first && !cut.own)) * rows + r; };
    const auto store = [&](int64_t r, int at, auto& v, float sum) __attribute__((always_inline)) {
      const int64_t row = cut.row0 + r;
      const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
      const int64_t to = ((int64_t)(cut.r0 + row / a.group) * a.hq + cut.head * a.group + row % a.group) * D + at;
#pragma unroll
      for (int e = 0; e < (int)(sizeof(v) / 4); ++e) {
        if (a.dtype == kF16) store1<kF16>(a.out, to + e, v[e] * inv);
        else store1<kBF16>(a.out, to + e, v[e] * inv);
      }
    };
    if (cut.last - cut.first < kParts) {  // uniform
      constexpr int L = D == 192 ? 64 : D / 4;  // lanes of a row, four dims each (of 192 some do another's over)
      const int at = min(4 * (lane % L), D - 4);
      for (int64_t r = ((int64_t)blockIdx.x * 4 + wave) * (64 / L) + lane / L; r < cut.rows; r += (int64_t)gridDim.x * (256 / L)) {
        float mx = kNoScore, sum = 0.0f, acc[4] = {};
        for (int w0 = cut.first; w0 <= cut.last; w0 += AT) {
          float2 ml[AT];
          floatx4 v[AT];
#pragma unroll
          for (int j = 0; j < AT; ++j) {
            const bool ok = w0 + j <= cut.last;
            const int64_t from = slot(ok ? w0 + j : w0, r);
            ml[j] = ok ? *(const float2*)(a.stat + from * 2) : make_float2(kNoScore, 0.0f);
            v[j] = ok ? *(const floatx4*)(a.part + from * D + at) : floatx4{0, 0, 0, 0};
          }
          float nm = mx;
#pragma unroll
          for (int j = 0; j < AT; ++j) nm = fmaxf(nm, ml[j].x);
          const float al = __builtin_amdgcn_exp2f(mx - nm);
          mx = nm;
          sum *= al;
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[e] *= al;
#pragma unroll
          for (int j = 0; j < AT; ++j) {
            const float f = __builtin_amdgcn_exp2f(ml[j].x - mx);
            sum += ml[j].y * f;
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[e] += v[j][e] * f;
          }
        }
        store(r, at, acc, sum);
      }
      continue;
    }
    for (int64_t r = blockIdx.x; r < cut.rows; r += gridDim.x) {
      float mx = kNoScore;
      for (int w = cut.first + lane; w <= cut.last; w += 64) mx = fmaxf(mx, a.stat[slot(w, r) * 2]);
#pragma unroll
      for (int off = 32; off > 0; off >>= 1) mx = fmaxf(mx, __shfl_xor(mx, off, 64));
      float sum = 0.0f, acc[E];
#pragma unroll
      for (int e = 0; e < E; ++e) acc[e] = 0.0f;
#pragma unroll 4
      for (int w = cut.first + wave; w <= cut.last; w += 4) {
        const float2 ml = *(const float2*)(a.stat + slot(w, r) * 2);
        const float f = __builtin_amdgcn_exp2f(ml.x - mx);
        sum += ml.y * f;
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] += a.part[slot(w, r) * D + E * lane + e] * f;
      }
#pragma unroll
      for (int e = 0; e < E; ++e) sums[wave][lane][e] = acc[e];
      if (lane == 0) ls[wave] = sum;
      __syncthreads();
      if (wave == 0) {
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] = sums[0][lane][e] + sums[1][lane][e] + sums[2][lane][e] + sums[3][lane][e];
        store(r, E * lane, acc, ls[0] + ls[1] + ls[2] + ls[3]);
      }
      __syncthreads();
    }
  }
}

struct Plan {
  int waves;         // of a workgroup
  int64_t shares;
  int64_t heads;     // (sequence, head, row tile)s, at most a workgroup's share each
  size_t q, qs, line, begins, cuts, cut, part, stat, bytes;  // parts of the workspace, and its size
};

size_t padded(size_t n) { return (n + 255) / 256 * 256; }

// `rows`: of a KV head. As few workgroups a KV head as there can be, of as few rows; shares of a workgroup a CU, or two of four waves
// of up to 128 dims.
Plan plan_of(int d, int64_t rows, int64_t tokens, int hq, int64_t seqs, int heads, int64_t max_len) {
  Plan p;
  const bool pair = d > 128;
  const int64_t units = std::max<int64_t>(1, (rows + 31) / 32), most = pair ? 4 : 8, row_tiles = (units + most - 1) / most;
  p.waves = (units + row_tiles - 1) / row_tiles <= most / 2 ? 4 : 8;
  const int cus = gguf::device_cus() * (!pair && p.waves == 4 ? 2 : 1);
  const int64_t tiles = std::max<int64_t>(1, (max_len + kToks - 1) / kToks);
  // (each factor is capped where the product is beyond every number of workgroups)
  const int64_t work = std::min<int64_t>(seqs * heads, 1 << 20) * std::min<int64_t>(row_tiles, 1 << 20) * std::min<int64_t>(tiles, 1 << 20);
  p.shares = std::max<int64_t>(1, std::min<int64_t>(cus, (work + kLeastTiles - 1) / kLeastTiles));
  p.q = 0;
  p.qs = p.q + padded((size_t)tokens * hq * 2 * d);
  p.line = p.qs + padded((size_t)tokens * hq * sizeof(float));
  p.heads = std::min<int64_t>(std::min<int64_t>(seqs * heads, 1 << 20) * std::min<int64_t>(row_tiles, 1 << 20), p.shares);
  p.begins = p.line + padded((size_t)(seqs + 1) * sizeof(int64_t));
  p.cuts = p.begins + padded((size_t)p.shares * sizeof(int));
  p.cut = p.cuts + 256;
  p.part = p.cut + padded((size_t)p.shares * sizeof(Cut));
  const size_t slots = p.shares == 1 ? 0 : 2 * (size_t)p.shares * (pair ? 16 : 32) * p.waves;
  p.stat = p.part + slots * d * sizeof(float);
  p.bytes = p.stat + slots * 2 * sizeof(float);
  return p;
}

template <int D, int NW>
hipError_t launch(const AttnArgs& a, const Prep& prep, const Plan& p, hipStream_t stream) {
  using L = Lay<D, NW>;
  int dev = 0;
  hipError_t e = hipGetDevice(&dev);
  if (e != hipSuccess) return e;
  struct Tag {};
  gguf::once_per_device<Tag>(dev, [&] {
    (void)hipFuncSetAttribute((const void*)attend_tree_kernel<D, NW>, hipFuncAttributeMaxDynamicSharedMemorySize, L::kBytes);
  });
  constexpr int per = D == 192 ? 4 : 1024 / D;
  const int64_t rows = ((int64_t)a.rows.tokens * a.hq + per - 1) / per;
  const unsigned blocks = (unsigned)std::min<int64_t>(rows, 1 << 20) + 1;
  if (a.dtype == kF16) prep_tree_kernel<kF16, D><<<blocks, 256, 0, stream>>>(a, prep, L::kRows, p.shares);
  else prep_tree_kernel<kBF16, D><<<blocks, 256, 0, stream>>>(a, prep, L::kRows, p.shares);
  attend_tree_kernel<D, NW><<<(unsigned)p.shares, L::kThreads, L::kBytes, stream>>>(a, prep, p.shares);
  if (p.shares > 1) {  // some thousand workgroups, of a row or more
    const int64_t each = std::min<int64_t>(L::kRows, std::max<int64_t>(L::kRows / 16, 4096 / p.heads));
    join_tree_kernel<D><<<dim3((unsigned)each, (unsigned)p.heads), 256, 0, stream>>>(a, prep, L::kRows, (int)p.shares);
  }
  return hipGetLastError();
}

}  // namespace

size_t tree_workspace(int d, int64_t rows, int64_t tokens, int hq, int64_t seqs, int heads, int64_t max_len) {
  return plan_of(d, rows, tokens, hq, seqs, heads, max_len).bytes;
}

hipError_t launch_attend_tree(AttnArgs a, int64_t rows, int64_t max_len, void* ws, hipStream_t stream) {
  const Plan p = plan_of(a.c.d, rows, a.rows.tokens, a.hq, a.rows.seqs, a.c.heads, max_len);
  char* w = (char*)ws;
  const Prep prep{(_Float16*)w, (float*)(w + p.qs), (int64_t*)(w + p.line), (int*)(w + p.begins), (int*)(w + p.cuts), (Cut*)(w + p.cut)};
  a.part = (float*)(w + p.part);
  a.stat = (float*)(w + p.stat);
#define GGUF_DEC_TREE(D) return p.waves == 4 ? launch<D, 4>(a, prep, p, stream) : launch<D, 8>(a, prep, p, stream);
  switch (a.c.d) {
    case 64: GGUF_DEC_TREE(64)
    case 128: GGUF_DEC_TREE(128)
    case 192: GGUF_DEC_TREE(192)
    default: GGUF_DEC_TREE(256)
  }
#undef GGUF_DEC_TREE
}

}  // namespace gguf_dec
