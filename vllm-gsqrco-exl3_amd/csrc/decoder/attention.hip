// Causal attention over the 8-bit paged cache (attend.h: layouts; include/gguf_decoder.h: contract).
#include "attend.h"

namespace gguf_dec {

namespace {

constexpr int kTile = 64;   // tokens a wave takes at a time
constexpr int kWaves = 4;

// One workgroup takes RT = 16 NT query rows (token, head of the KV head's group) of one sequence and
// KV head, and one split of its tokens; its waves take the split's tiles in turn, straight from the cache into
// operand registers (each byte is read by one lane, so LDS would only add a hop), with statistics and
// accumulators of their own, joined through LDS at the end. Softmax is online: a wave keeps, for each row, the maximum m so
// far, its lanes' sums of 2^(s - m), and O scaled to m.
// The scale of a V chunk goes into P: p * vs / ref, where ref is the largest vs the wave has met, so
// that P stays within fp16's range whatever the scales are. P is rounded to fp16 (11 bits; the output
// has 8 or 11), everything else is fp32.
//
// Bound: HBM for few rows. 2 bytes a (token, head, dim).
template <int DT, int D, int NT>
__global__ void __launch_bounds__(64 * kWaves, 1) attend_kernel(AttnArgs a) {
  constexpr int S = D / 64, DD = D / 16;
  extern __shared__ __align__(16) float lds[];  // [kWaves][DD][NT][64][4]
  __shared__ float stat[kWaves][NT * 16][2], refs[kWaves];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, n = lane & 15, g = lane >> 4;
  const int seqs = a.rows.seqs;
  const int head = blockIdx.y % a.c.heads, seq = blockIdx.y / a.c.heads, split = blockIdx.z, splits = gridDim.z;
  int r0, r1;
  rows_of(a.rows, seq, r0, r1);
  const int64_t nrows = (int64_t)(r1 - r0) * a.group;
  const int len0 = a.lens[seq];
  const int64_t room = (int64_t)a.c.max_pages * a.c.page;
  const int page16 = a.c.page / 16;
  const int32_t* table = a.c.table + (int64_t)seq * a.c.table_stride;

  for (int64_t tile0 = (int64_t)blockIdx.x * 16 * NT; tile0 < nrows; tile0 += (int64_t)gridDim.x * 16 * NT) {
    // rows of this tile: row -> (token, head); last: the last position that it sees
    int64_t qrow[NT];
    int last[NT];
    int see = -1, all = 0x7FFFFFFF;  // the last position that any / every row sees
    half8 q[NT][2 * S];
    float qs[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const int64_t r = tile0 + 16 * t + n;
      const bool ok = r < nrows;
      const int tok = ok ? (int)(r / a.group) : 0, h = head * a.group + (ok ? (int)(r % a.group) : 0);
      qrow[t] = ok ? (int64_t)(r0 + tok) * a.hq + h : -1;
      const int64_t l = ok ? (int64_t)len0 - (r1 - r0) + tok : -1;
      last[t] = (int)(l < room ? l : room - 1);
      see = max(see, last[t]);
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
      const float f = DT == kBF16 ? row_factor(group_max(amax)) : 1.0f;
      qs[t] = a.scale / f;
#pragma unroll
      for (int s = 0; s < 2 * S; ++s)
#pragma unroll
        for (int e = 0; e < 8; ++e) q[t][s][e] = (_Float16)(v[s][e] * f);
    }
#pragma unroll
    for (int off = 1; off < 16; off <<= 1) {
      see = max(see, __shfl_xor(see, off, 64));
      all = min(all, __shfl_xor(all, off, 64));
    }
    const int ntiles = (see + kTile) / kTile;  // see = -1: none
    const int tb = (int)min((int64_t)split * (a.span / kTile), (int64_t)ntiles);
    const int te = split == splits - 1 ? ntiles : min(ntiles, tb + a.span / kTile);
    if (splits > 1 && tb >= te) {  // uniform: nothing of these rows lies in the split
#pragma unroll
      for (int t = 0; t < NT; ++t)
        if (wave == 0 && g == 0 && qrow[t] >= 0)
          *(float2*)(a.stat + (split * (int64_t)a.rows.tokens * a.hq + qrow[t]) * 2) = make_float2(kNoScore, 0.0f);
      continue;
    }

    floatx4 o[DD][NT];
    float m[NT], l[NT];
    float ref = 0.0f;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      m[t] = kNoScore;
      l[t] = 0.0f;
#pragma unroll
      for (int i = 0; i < DD; ++i) o[i][t] = floatx4{0, 0, 0, 0};
    }

    for (int tile = tb + wave; tile < te; tile += kWaves) {
      // chunk g of the tile: its page, scales; the K operand's rows lie in chunk n >> 2
      const Chunk ck = chunk_of(a.c, table, page16, head, (int64_t)4 * tile + g, see);
      const int64_t ph = ck.ph;
      const int off = ck.off;
      const float ks = ck.ks, vs = ck.vs;
      const int8_t* vp = a.c.v + ph * a.c.page * D + (int64_t)n * a.c.page + off;
      const int64_t koff = (ph * a.c.page + off) * D;
      const int64_t kc = __shfl(koff, 16 * (n >> 2), 64);
      const int8_t* kp = a.c.k + kc + (n & 3) * D + 16 * g;

      floatx4 sc[4][NT];
#pragma unroll
      for (int tt = 0; tt < 4; ++tt) {
#pragma unroll
        for (int t = 0; t < NT; ++t) sc[tt][t] = floatx4{0, 0, 0, 0};
#pragma unroll
        for (int s = 0; s < S; ++s) {
          const uint4 w = *(const uint4*)(kp + 4 * tt * D + 64 * s);
          const half8 k0 = codes8(w.x, w.y), k1 = codes8(w.z, w.w);
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            sc[tt][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k0, q[t][2 * s], sc[tt][t], 0, 0, 0);
            sc[tt][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k1, q[t][2 * s + 1], sc[tt][t], 0, 0, 0);
          }
        }
      }

      const float top = group_max(vs);
      const float nref = fmaxf(ref, top);
      const float shrink = nref > ref ? ref / nref : 1.0f;
      ref = nref;
      const float vr = ref > 0.0f ? vs / ref : vs;  // vs is 0 (or NaN) where ref is 0
      const bool masked = kTile * tile + kTile - 1 > all;
      half8 p[NT][2];
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const float f = qs[t] * ks;
        float mx = kNoScore;
#pragma unroll
        for (int tt = 0; tt < 4; ++tt)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            float x = sc[tt][t][i] * f;
            if (masked && kTile * tile + 16 * g + 4 * tt + i > last[t]) x = -__builtin_inff();
            sc[tt][t][i] = x;
            mx = fmaxf(mx, x);
          }
        mx = fmaxf(group_max(mx), m[t]);
        const float al = __builtin_amdgcn_exp2f(m[t] - mx);
        m[t] = mx;
        float sum = 0.0f;
#pragma unroll
        for (int tt = 0; tt < 4; ++tt)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float x = sc[tt][t][i];
            const float e = __builtin_amdgcn_exp2f(x - mx);
            sum += e;
            // a masked place adds nothing, also where its page's scale is not finite
            p[t][tt >> 1][4 * (tt & 1) + i] = (_Float16)(x == -__builtin_inff() ? 0.0f : e * vr);
          }
        l[t] = l[t] * al + sum;
        const float r = al * shrink;
        if (__any(r != 1.0f)) {
#pragma unroll
          for (int i = 0; i < DD; ++i) o[i][t] *= r;
        }
      }
#pragma unroll
      for (int i = 0; i < DD; ++i) {
        const uint4 w = *(const uint4*)(vp + (int64_t)16 * i * a.c.page);
        const half8 v0 = codes8(w.x, w.y), v1 = codes8(w.z, w.w);
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          o[i][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v0, p[t][0], o[i][t], 0, 0, 0);
          o[i][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v1, p[t][1], o[i][t], 0, 0, 0);
        }
      }
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
        *(floatx4*)(lds + ((((size_t)wave * DD + i) * NT + t) * 64 + lane) * 4) = o[i][t] * ref;
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

// Joins the splits of a row: one wave a row, 4 dims a lane and turn.
template <int DT, int D>
__global__ void __launch_bounds__(256) join_kernel(const float* __restrict__ part, const float* __restrict__ stat,
                                                   int64_t rows, int splits, void* __restrict__ out) {
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= rows) return;
  const int lane = threadIdx.x & 63;
  float mx = kNoScore;
  for (int s = 0; s < splits; ++s) mx = fmaxf(mx, stat[(s * rows + row) * 2]);
  float sum = 0.0f;
  floatx4 acc = {0, 0, 0, 0};
  for (int s = 0; s < splits; ++s) {
    const float l = stat[(s * rows + row) * 2 + 1];
    const float f = __builtin_amdgcn_exp2f(stat[(s * rows + row) * 2] - mx);
    if (l == 0.0f) continue;
    sum += l * f;
    if (4 * lane < D) acc += *(const floatx4*)(part + (s * rows + row) * D + 4 * lane) * f;
  }
  const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
  const float y[4] = {acc[0] * inv, acc[1] * inv, acc[2] * inv, acc[3] * inv};
  if (4 * lane < D) store4<DT>(out, row * D + 4 * lane, y);
}

template <int DT, int D, int NT>
hipError_t launch_attend(const AttnArgs& a, dim3 grid, hipStream_t stream) {
  constexpr int lds = kWaves * D * 16 * NT * 4;
  int dev = 0;
  hipError_t e = hipGetDevice(&dev);
  if (e != hipSuccess) return e;
  struct Tag {};
  gguf::once_per_device<Tag>(dev, [&] {
    (void)hipFuncSetAttribute((const void*)attend_kernel<DT, D, NT>, hipFuncAttributeMaxDynamicSharedMemorySize, lds);
  });
  attend_kernel<DT, D, NT><<<grid, 64 * kWaves, lds, stream>>>(a);
  return hipGetLastError();
}

}  // namespace

// How a call is cut: rows of a workgroup, and tokens of a split so that the CUs have two workgroups each, in
// steps of a tile a wave.
struct AttnPlan {
  bool many;
  int nt, span, splits;
  int64_t row_tiles;
};

static AttnPlan attn_plan(int64_t rows, int64_t groups, int64_t max_len, int64_t most_splits) {
  AttnPlan p;
  p.many = rows > 64;
  p.nt = rows > 16 ? 2 : 1;
  const int64_t tile = p.many ? kRowsTile : 16 * p.nt;
  p.row_tiles = (rows + tile - 1) / tile;
  const int64_t blocks = groups * p.row_tiles, step = kTile * kWaves;
  const int64_t steps = (max_len + step - 1) / step;
  int64_t want = (2 * gguf::device_cus() + blocks - 1) / blocks;
  if (want > 512) want = 512;
  if (want > most_splits) want = most_splits;
  if (want < 1) want = 1;
  const int64_t each = (steps + want - 1) / want;
  p.span = (int)(each * step < (1 << 30) ? each * step : (1 << 30));
  p.splits = (int)((steps + each - 1) / each);
  if (p.splits < 1) p.splits = 1;
  return p;
}

size_t kv8_attention_workspace(int d, int heads, int hq, int64_t tokens, int64_t seqs, int64_t max_new,
                               int64_t max_len) {
  const AttnPlan p = attn_plan(max_new * (hq / heads), seqs * heads, max_len, 512);
  return p.splits == 1 ? 0 : (size_t)p.splits * tokens * hq * (d + 2) * sizeof(float);
}

hipError_t launch_kv8_attention(const Kv8& c, int dtype, const void* q, int64_t qt, int64_t qh, int hq,
                                const int32_t* lens, const Ragged& rows, int64_t max_new, int64_t max_len, float scale,
                                void* out, void* ws, size_t ws_bytes, hipStream_t stream) {
  const int64_t all = (int64_t)rows.tokens * hq;
  const int64_t fit = (int64_t)(ws_bytes / sizeof(float)) / (all * (c.d + 2));
  const AttnPlan p = attn_plan(max_new * (hq / c.heads), (int64_t)rows.seqs * c.heads, max_len, fit < 2 ? 1 : fit);
  const AttnArgs a{c, q, qt, qh, lens, rows, hq, hq / c.heads, scale * kLog2e, p.span, p.splits, out, (float*)ws,
                   (float*)ws + (size_t)p.splits * all * c.d};
  const dim3 grid((unsigned)(p.row_tiles < 65535 ? p.row_tiles : 65535), (unsigned)(rows.seqs * c.heads), p.splits);
  hipError_t e = hipSuccess;
  if (p.many) e = launch_attend_rows(a, dtype, p.row_tiles, stream);
#define GGUF_DEC_ATTEND(DT, D)                                                                                         \
  {                                                                                                                    \
    if (!p.many) e = p.nt == 1 ? launch_attend<DT, D, 1>(a, grid, stream) : launch_attend<DT, D, 2>(a, grid, stream);  \
    if (e == hipSuccess && p.splits > 1)                                                                               \
      join_kernel<DT, D><<<(unsigned)((all + 3) / 4), 256, 0, stream>>>(a.part, a.stat, all, p.splits, out);           \
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
