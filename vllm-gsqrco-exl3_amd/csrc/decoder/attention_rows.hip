// Causal attention over the 8-bit paged cache for many rows a sequence (a prompt's chunk): the form of
// attention.hip with the tiles shared through LDS and 32 x 32 MFMAs, which reach more of the matrix cores' rate here
// (in loops without loads f16 32x32x16 1.71 PFLOP/s, 16x16x32 1.37, i8 32x32x32 4.8).
//
// Both products are transposed, S^T = K Q^T and O^T += V^T P^T, so that a lane keeps one query row. With lane = 32 h + n,
// a result's element i is row 8 (i >> 2) + 4 h + (i & 3) of column n. The 32 tokens of a tile stand in K's rows in
// such an order (token_of) that the 8 scores i = 8 c .. 8 c + 7 of a lane are its 8 consecutive places of the c-th step
// of the second product: tokens 16 c + 8 h + 0 .. 7.
//
// K stays in 8 bits: the first product is int8, with Q as 15-bit integers q = s (128 hi + lo), s the row's
// largest magnitude / 16256, in two products whose int32 sums are exact (128 * 127 * 127 * 256 < 2^30). What rounding Q
// changes of a score is below 2^-15 of the largest |q| times |k|, where the weights are rounded to fp16 (2^-12)
// and outputs to 8 or 11 bits. Beside two fp16 steps this halves what the waves read of K from LDS, which bounds the kernel
// next to the matrix cores, and K needs no conversion.
// V is converted to fp16 once a workgroup, from registers to LDS.
//
// Measured, 24 query and 4 KV heads of 256: a call of 2048 rows at positions up to 8192 590 us, 611 TFLOP/s (1453 us in the
// form for few rows). By counters the matrix cores are busy for 25 % of the kernel's time and VALU instructions issue
// for 35 %: the softmax and the operand reads are not hidden, with one wave a SIMD (D = 256: 128 accumulator and 64 query
// registers; two workgroups a CU spill, 1,065 us).
#include <type_traits>

#include "attend.h"

namespace gguf_dec {

namespace {

typedef int intx4 __attribute__((ext_vector_type(4)));
typedef int intx16 __attribute__((ext_vector_type(16)));
typedef float floatx16 __attribute__((ext_vector_type(16)));

constexpr int kToks = 32;  // tokens of a tile
constexpr int kRowWaves = kRowsTile / 32;
constexpr int kSegment = 128;  // tiles whose chunks are looked up at a time

// place of a 16-byte piece c of a key's row in LDS: rows that are read together fall into different banks
template <int D>
__device__ __forceinline__ int k_place(int row, int c) {
  const int x = D == 256 ? row & 15 : D == 128 ? row & 7 : (row >> 2) & 3;
  return row * D + 16 * (c ^ x);
}

// where a tile's two chunks lie, and their scales (the same in all lanes)
struct Tile {
  int ph[2], off[2];
  float ks[2], vs[2];
};

template <int DT, int D>
__global__ void __launch_bounds__(64 * kRowWaves, D <= 128 ? 2 : 1) attend_rows_kernel(AttnArgs a) {
  constexpr int KS = D / 32, DD = D / 32;   // steps of the first product, 32-dim tiles of the second
  constexpr int VROW = 2 * kToks + 16;      // bytes of a dim's row of V in LDS
  constexpr int VP = (2 * D + 64 * kRowWaves - 1) / (64 * kRowWaves);  // 16-byte pieces of V a lane
  __shared__ __align__(16) int8_t kl[2][kToks * D];
  __shared__ __align__(16) char vl[2][D * VROW];
  __shared__ __align__(16) Chunk chunks[2 * (kSegment + 3)];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), n = lane & 31, h = lane >> 5;
  // workgroups of one (sequence, head, split) take the same tiles: a stride of gridDim.x apart, they run on as few XCDs as
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
  const int64_t row_tiles = (nrows + kRowsTile - 1) / kRowsTile;

  // the last rows, which see most, first
  for (int64_t rt = row_tiles - 1 - blockIdx.y; rt >= 0; rt -= gridDim.y) {
    const int64_t r = rt * kRowsTile + wave * 32 + n;
    const bool row_ok = r < nrows;
    const int tok = row_ok ? (int)(r / a.group) : 0, hd = head * a.group + (row_ok ? (int)(r % a.group) : 0);
    const int64_t orow = row_ok ? (int64_t)(r0 + tok) * a.hq + hd : -1;
    const int64_t lst = row_ok ? (int64_t)len0 - (r1 - r0) + tok : -1;
    const int last = (int)(lst < room ? lst : room - 1);
    // what the tile's rows see: rows are in order of their tokens
    const int64_t rlast = min(nrows, (rt + 1) * kRowsTile) - 1;
    const int64_t see64 = min((int64_t)len0 - (r1 - r0) + rlast / a.group, room - 1);
    const int see = (int)max(see64, (int64_t)-1);
    const int ntiles = (see + kToks) / kToks;
    const int tb = (int)min((int64_t)split * (a.span / kToks), (int64_t)ntiles);
    const int te = split == splits - 1 ? ntiles : min(ntiles, tb + a.span / kToks);
    const int64_t all_rows = (int64_t)a.rows.tokens * a.hq;
    if (tb >= te) {  // uniform: the rows see nothing of the split, or nothing at all
      if (splits == 1) {
        const float none[4] = {0, 0, 0, 0};
        for (int i = 4 * h; i < D && orow >= 0; i += 8) store4<DT>(a.out, orow * D + i, none);
      } else if (h == 0 && orow >= 0) *(float2*)(a.stat + (split * all_rows + orow) * 2) = make_float2(kNoScore, 0.0f);
      continue;
    }

    // Q as integers
    intx4 qhi[KS], qlo[KS];
    float qs;
    {
      float v[KS][16];
      uint32_t big = 0;
#pragma unroll
      for (int s = 0; s < KS; ++s)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          float w[8];
          if (row_ok) {
            load8<DT>(a.q, (int64_t)(r0 + tok) * a.qt + (int64_t)hd * a.qh + 32 * s + 16 * h + 8 * half, w);
          } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) w[e] = 0.0f;
          }
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            v[s][8 * half + e] = w[e];
            big = max(big, __float_as_uint(w[e]) & 0x7FFFFFFFu);
          }
        }
      big = max(big, (uint32_t)__shfl_xor((int)big, 32, 64));
      const float amax = __uint_as_float(big);  // NaN and inf on top: then the row's scores are NaN
      // a row of magnitudes below 2^-100 has scores of 0
      const float inv = amax >= 0x1p-100f && amax < __builtin_inff() ? (a.scale < 0.0f ? -16256.0f : 16256.0f) / amax : 0.0f;
      // not negative (the scale's sign is Q's), so that the largest product is the largest score
      qs = amax < __builtin_inff() ? fabsf(a.scale) * (amax * (1.0f / 16256.0f)) : __builtin_nanf("");
#pragma unroll
      for (int s = 0; s < KS; ++s)
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          uint32_t hi = 0, lo = 0;
#pragma unroll
          for (int b = 0; b < 4; ++b) {
            const int x = (int)rintf(v[s][4 * w + b] * inv);
            const int top = (x + 64) >> 7;
            hi |= (uint32_t)(top & 0xFF) << 8 * b;
            lo |= (uint32_t)((x - 128 * top) & 0xFF) << 8 * b;
          }
          qhi[s][w] = (int)hi;
          qlo[s][w] = (int)lo;
        }
    }

    floatx16 o[DD];
#pragma unroll
    for (int i = 0; i < DD; ++i)
#pragma unroll
      for (int e = 0; e < 16; ++e) o[i][e] = 0.0f;
    float m = kNoScore, l = 0.0f, ref = 0.0f, inv_ref = 0.0f;

    // tile t's chunks, from LDS, the same in all lanes
    int seg = tb;  // chunks[0] is of this tile
    const auto find = [&](int t) __attribute__((always_inline)) {
      Tile r;
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const Chunk x = chunks[2 * (t - seg) + c];
        r.ph[c] = __builtin_amdgcn_readfirstlane(x.ph);
        r.off[c] = __builtin_amdgcn_readfirstlane(x.off);
        r.ks[c] = __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(x.ks)));
        r.vs[c] = __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(x.vs)));
      }
      return r;
    };
    const auto find_chunks = [&](int from) __attribute__((always_inline)) {
      __syncthreads();
      seg = from;
      for (int i = tid; i < 2 * (kSegment + 3); i += 64 * kRowWaves)
        chunks[i] = chunk_of(a.c, table, page16, head, (int64_t)2 * from + i, see);
      __syncthreads();
    };
    // this thread's j-th 16-byte piece of K (row p / (D / 16)) and of V (half p & 1 of dim p >> 1); where a tile does
    // not go round evenly some are taken twice, so that nothing branches
    constexpr int KP = VP;
    const auto piece = [&](int j) __attribute__((always_inline)) {
      const int p = j * 64 * kRowWaves + tid;
      return D % 128 == 0 ? p : D == 64 ? tid & 127 : p < 2 * D ? p : p - 64 * kRowWaves;
    };
    uintx4 kraw[KP], vraw[VP];
    const auto load_k = [&](const Tile& x) __attribute__((always_inline)) {
      const int8_t* k0 = a.c.k + ((int64_t)x.ph[0] * a.c.page + x.off[0]) * D;
      const int8_t* k1 = a.c.k + ((int64_t)x.ph[1] * a.c.page + x.off[1]) * D;
#pragma unroll
      for (int j = 0; j < KP; ++j) {
        const int p = piece(j), row = p / (D / 16), c = p % (D / 16);
        kraw[j] = *(const uintx4*)((row >> 4 ? k1 : k0) + (uint32_t)((row & 15) * D + 16 * c));
      }
    };
    const auto load_v = [&](const Tile& x) __attribute__((always_inline)) {
      const int8_t* v0 = a.c.v + (int64_t)x.ph[0] * a.c.page * D + x.off[0];
      const int8_t* v1 = a.c.v + (int64_t)x.ph[1] * a.c.page * D + x.off[1];
#pragma unroll
      for (int j = 0; j < VP; ++j) {
        const int p = piece(j);
        vraw[j] = *(const uintx4*)((p & 1 ? v1 : v0) + (uint32_t)((p >> 1) * a.c.page));
      }
    };
    const auto put_k = [&](int b) __attribute__((always_inline)) {
#pragma unroll
      for (int j = 0; j < KP; ++j) {
        const int p = piece(j);
        *(uintx4*)(kl[b] + k_place<D>(p / (D / 16), p % (D / 16))) = kraw[j];
      }
    };
    const auto put_v = [&](int b) __attribute__((always_inline)) {
#pragma unroll
      for (int j = 0; j < VP; ++j) {
        const int p = piece(j), d = p >> 1, u = p & 1;
        *(half8*)(vl[b] + d * VROW + 32 * u) = codes8(vraw[j][0], vraw[j][1]);
        *(half8*)(vl[b] + d * VROW + 32 * u + 16) = codes8(vraw[j][2], vraw[j][3]);
      }
    };
    const int krow = 16 * (n >> 4) + 8 * ((n >> 2) & 1) + 4 * ((n >> 3) & 1) + (n & 3);  // token of K's row n
    // S^T of the tile in buffer b, before its scales
    const auto product = [&](int b, intx16& s) __attribute__((always_inline)) {
      intx4 k[KS];
#pragma unroll
      for (int i = 0; i < KS; ++i) k[i] = *(const intx4*)(kl[b] + k_place<D>(krow, 2 * i + h));
      intx16 lo;
#pragma unroll
      for (int e = 0; e < 16; ++e) s[e] = lo[e] = 0;
#pragma unroll
      for (int i = 0; i < KS; ++i) {
        s = __builtin_amdgcn_mfma_i32_32x32x32_i8(k[i], qhi[i], s, 0, 0, 0);
        lo = __builtin_amdgcn_mfma_i32_32x32x32_i8(k[i], qlo[i], lo, 0, 0, 0);
      }
#pragma unroll
      for (int e = 0; e < 16; ++e) s[e] = (s[e] << 7) + lo[e];
    };
    const int first_last = (int)min((int64_t)len0 - (r1 - r0) + rt * kRowsTile / a.group, room - 1);  // of the first row

    // Turn t multiplies tile t + 1's K beside tile t's softmax, then tile t's V, so that the matrix cores run on while a
    // wave works on its scores: it is alone on its SIMD (at D = 256 a wave needs some 400 registers). What a turn
    // loads is put to LDS at the next one's start. Past the end the last tile is taken again, to buffers that nobody reads.
    const int tlast = te - 1;
    intx16 s;
    find_chunks(tb);  // (and the previous rows' last tile has been read)
    Tile x0 = find(tb), x1 = find(min(tb + 1, tlast)), x2 = find(min(tb + 2, tlast));
    load_k(x0);
    put_k(0);
    load_k(x1);
    load_v(x0);
    put_k(1);
    put_v(0);
    load_k(x2);
    load_v(x1);
    __syncthreads();
    product(0, s);
    // a turn; `masked`: some row does not see all of the tile
    const auto turn = [&](int t, auto masked) __attribute__((always_inline)) {
      constexpr bool kMasked = decltype(masked)::value;
      const int b = (t - tb) & 1;
      const Tile x3 = find(min(t + 3, tlast));
      __syncthreads();
      // here: K of t + 1 and V of t in LDS, K of t + 2 and V of t + 1 in registers

      // the rows' statistics
      const int seen = last - (kToks * t + 8 * h);  // place 16 c + e of the lane is seen if it is at most this
      // the largest V scale of the chunks that the row sees; a NaN counts for nothing
      const float top = fmaxf(!kMasked || last >= kToks * t ? x0.vs[0] : 0.0f, !kMasked || last >= kToks * t + 16 ? x0.vs[1] : 0.0f);
      const float f[2] = {qs * x0.ks[0], qs * x0.ks[1]};
      float mx = kNoScore;
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        int big = INT32_MIN;
#pragma unroll
        for (int e = 0; e < 8; ++e) big = max(big, !kMasked || 16 * c + e <= seen ? s[8 * c + e] : INT32_MIN);
        if (!kMasked || big != INT32_MIN) mx = fmaxf(mx, (float)big * f[c]);
      }
      mx = half_max(mx);
      // the maximum may lag: weights stay below 2^8, and the sums are scaled again only where it does not do, or
      // where the largest V scale grew
      const float nm = mx > m + 8.0f ? mx : m;
      if (__any(nm != m || top > ref)) {
        const float nref = fmaxf(ref, top);
        const float al = __builtin_amdgcn_exp2f(m - nm);
        const float by = nref > ref ? al * (ref / nref) : al;
        l *= al;
#pragma unroll
        for (int i = 0; i < DD; ++i) o[i] *= by;
        m = nm;
        ref = nref;
        inv_ref = ref > 0.0f ? kWeight / ref : 0.0f;
      }

      // from here on straight, for the scheduler: tile t + 1's K beside the weights
      intx16 sn;
      product(b ^ 1, sn);
      half8 p[2];
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const float vr = x0.vs[c] * inv_ref;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          float x = (float)s[8 * c + e] * f[c];
          asm("" : "+v"(x));  // rounded as it was for the maximum: of scores beyond 2^24 an fma's rest would pass any weight
          float w = __builtin_amdgcn_exp2f(x - m);
          float y = w * vr;
          if (kMasked && 16 * c + e > seen) w = y = 0.0f;  // also where the page's scale is not finite
          l += w;
          p[c][e] = (_Float16)y;
        }
      }
      // O^T, beside the next tile's way to LDS
#pragma unroll
      for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int i = 0; i < DD; ++i) {
          const half8 v = *(const half8*)(vl[b] + (32 * i + n) * VROW + 32 * c + 16 * h);
          o[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, p[c], o[i], 0, 0, 0);
        }
      put_k(b);
      put_v(b ^ 1);
      load_k(x3);
      load_v(x2);
      s = sn;
      x0 = x1;
      x1 = x2;
      x2 = x3;
    };
    for (int t = tb; t < te;) {
      if (t != tb) find_chunks(t);
      const int stop = min(t + kSegment, te);
      for (; t < stop && kToks * t + kToks - 1 <= first_last; ++t) turn(t, std::false_type());
      for (; t < stop; ++t) turn(t, std::true_type());
    }

    l += __shfl_xor(l, 32, 64);
    if (orow >= 0) {
      const float by = ref / kWeight, inv = splits == 1 ? (l == 0.0f ? 0.0f : by / l) : by;
#pragma unroll
      for (int i = 0; i < DD; ++i)
#pragma unroll
        for (int e = 0; e < 16; e += 4) {
          const int at = 32 * i + 2 * e + 4 * h;
          if (splits == 1) {
            const float y[4] = {o[i][e] * inv, o[i][e + 1] * inv, o[i][e + 2] * inv, o[i][e + 3] * inv};
            store4<DT>(a.out, orow * D + at, y);
          } else {
            *(floatx4*)(a.part + (split * all_rows + orow) * D + at) =
                floatx4{o[i][e] * inv, o[i][e + 1] * inv, o[i][e + 2] * inv, o[i][e + 3] * inv};
          }
        }
      if (splits > 1 && h == 0) *(float2*)(a.stat + (split * all_rows + orow) * 2) = make_float2(m, l);
    }
  }
}

}  // namespace

hipError_t launch_attend_rows(const AttnArgs& a, int dtype, int64_t row_tiles, hipStream_t stream) {
  const dim3 grid((unsigned)(a.rows.seqs * a.c.heads * a.splits), (unsigned)(row_tiles < 65535 ? row_tiles : 65535));
#define GGUF_DEC_ROWS(DT)                                                                         \
  switch (a.c.d) {                                                                                \
    case 64: attend_rows_kernel<DT, 64><<<grid, 64 * kRowWaves, 0, stream>>>(a); break;           \
    case 128: attend_rows_kernel<DT, 128><<<grid, 64 * kRowWaves, 0, stream>>>(a); break;         \
    case 192: attend_rows_kernel<DT, 192><<<grid, 64 * kRowWaves, 0, stream>>>(a); break;         \
    default: attend_rows_kernel<DT, 256><<<grid, 64 * kRowWaves, 0, stream>>>(a); break;          \
  }
  if (dtype == kF16) {
    GGUF_DEC_ROWS(kF16)
  } else {
    GGUF_DEC_ROWS(kBF16)
  }
#undef GGUF_DEC_ROWS
  return hipGetLastError();
}

}  // namespace gguf_dec
