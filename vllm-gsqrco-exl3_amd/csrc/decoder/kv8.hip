// Writing and reading a paged KV cache in 8 bits (include/gguf_decoder.h states its layout).
//
// A (page, head) of K or of V has one scale s = amax / 127 and codes round(x / s). A page that is
// filled over several calls keeps s >= every earlier scale, so older codes are only ever rounded
// again to a coarser step: round(code * s_old / s_new).
#include "kv8_codes.h"

namespace gguf_dec {

namespace {

constexpr int kThreads = 256;

// One workgroup writes the new tokens of one (sequence, page, head) of K (blockIdx.y even) or of V
// (odd), so no two workgroups share a scale and nothing is atomic. First the new values' largest
// magnitude (as bits of |x|: unsigned order puts inf and NaN on top, so they reach the scale), then,
// where the scale grew, the older codes, then the new ones. The second read of the values is from L2.
//
// Bound: HBM, 2 B in and 1 B out a value, and for a prompt the second pass, in which of V half of the threads have no piece
// (pages of 64, heads of 256); at a token a sequence the launch's latency. Measured: 8192 tokens of 4 heads of 256 in bf16
// 24 us, 50 MB, 2.1 TB/s; 32 sequences of one token 5.5 us.
template <int DT>
__global__ void __launch_bounds__(kThreads) append_kernel(Kv8 c, const void* __restrict__ key, int64_t kt, int64_t kh,
                                                          const void* __restrict__ value, int64_t vt, int64_t vh,
                                                          const int32_t* __restrict__ lens, Ragged rows) {
  const int seq = blockIdx.z, head = blockIdx.y >> 1;
  const bool is_v = blockIdx.y & 1;
  int r0, r1;
  rows_of(rows, seq, r0, r1);
  const int64_t room = (int64_t)c.max_pages * c.page;
  const int64_t len = lens[seq], start = len - (r1 - r0);  // position of row r0; rows before position 0 are dropped
  const int64_t end = min(len, room);
  if (r1 == r0 || end <= 0) return;
  const int tid = threadIdx.x, d = c.d, page = c.page;
  const int first = (int)(max(start, (int64_t)0) / page), last = (int)((end - 1) / page);
  const void* x = is_v ? value : key;
  const int64_t st = is_v ? vt : kt;
  const int64_t base = (int64_t)head * (is_v ? vh : kh);
  __shared__ uint32_t most[kThreads / 64];

  for (int p = first + blockIdx.x; p <= last; p += gridDim.x) {
    const int pid = c.table[(int64_t)seq * c.table_stride + p];
    if (pid < 0 || pid >= c.pages) continue;  // uniform
    const int64_t p0 = (int64_t)p * page;
    const int lo = (int)(max(start, p0) - p0), hi = (int)(min(end, p0 + page) - p0);  // new tokens of the page
    const int64_t row0 = r0 + (p0 - start);                                           // row of the page's token 0
    const int older = start > p0 ? lo : 0;

    const int per = d / 8;  // 8-value pieces a token
    uint32_t big = 0;
    for (int i = tid; i < (hi - lo) * per; i += kThreads) {
      float v[8];
      load8<DT>(x, (row0 + lo + i / per) * st + base + 8 * (i % per), v);
#pragma unroll
      for (int e = 0; e < 8; ++e) big = max(big, __float_as_uint(v[e]) & 0x7FFFFFFFu);
    }
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) big = max(big, (uint32_t)__shfl_xor((int)big, off, 64));
    __syncthreads();  // the previous page's `most` has been read
    if ((tid & 63) == 0) most[tid >> 6] = big;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kThreads / 64; ++w) big = max(big, most[w]);

    float* scale = (is_v ? c.vs : c.ks) + (int64_t)pid * c.heads + head;
    const Rescale s = rescale_of(older > 0 ? *scale : 0.0f, __uint_as_float(big));
    const bool shrink = older > 0 && s.shrink;
    __syncthreads();  // every thread has read the old scale
    if (tid == 0) *scale = s.scale;

    int8_t* codes = (is_v ? c.v : c.k) + ((int64_t)pid * c.heads + head) * page * d;
    if (!is_v) {
      if (shrink)
        for (int i = tid; i < older * d / 4; i += kThreads) ((uint32_t*)codes)[i] = rescale4(((uint32_t*)codes)[i], s.ratio);
      for (int i = tid; i < (hi - lo) * per; i += kThreads) {
        const int t = lo + i / per, at = 8 * (i % per);
        float v[8];
        load8<DT>(x, (row0 + t) * st + base + at, v);
        uint32_t w[2] = {0, 0};
#pragma unroll
        for (int e = 0; e < 8; ++e) w[e >> 2] |= (uint32_t)(code_of(v[e] * s.inv) & 0xFF) << 8 * (e & 3);
        *(uint2*)(codes + (int64_t)t * d + at) = make_uint2(w[0], w[1]);
      }
    } else {
      // a thread turns 16 tokens x 8 dims in its registers; 16-token groups without new tokens are
      // touched only where the scale grew
      const int g0 = shrink ? 0 : lo / 16, g1 = (hi + 15) / 16;
      for (int i = tid; i < (g1 - g0) * per; i += kThreads) {
        const int t0 = 16 * (g0 + i / per), at = 8 * (i % per);
        uint32_t w[8][4];
        const bool whole = lo <= t0 && t0 + 16 <= hi;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          uint4 o = make_uint4(0, 0, 0, 0);
          if (!whole) o = *(const uint4*)(codes + (int64_t)(at + e) * page + t0);
          w[e][0] = o.x; w[e][1] = o.y; w[e][2] = o.z; w[e][3] = o.w;
        }
#pragma unroll
        for (int t = 0; t < 16; ++t) {
          float v[8];
          const bool is_new = t0 + t >= lo && t0 + t < hi;
          const bool is_old = shrink && t0 + t < older;
          if (is_new) load8<DT>(x, (row0 + t0 + t) * st + base + at, v);
          if (is_new || is_old) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const float y = is_new ? v[e] * s.inv : (float)(int8_t)(w[e][t >> 2] >> 8 * (t & 3)) * s.ratio;
              w[e][t >> 2] = (w[e][t >> 2] & ~(0xFFu << 8 * (t & 3))) | (uint32_t)(code_of(y) & 0xFF) << 8 * (t & 3);
            }
          }
        }
#pragma unroll
        for (int e = 0; e < 8; ++e)
          *(uint4*)(codes + (int64_t)(at + e) * page + t0) = make_uint4(w[e][0], w[e][1], w[e][2], w[e][3]);
      }
    }
  }
}

// One workgroup reads 64 cache positions, aligned to 16, of one (sequence, head) of K or V. A thread takes 16 positions x 8 dims: of K
// eight bytes a position, of V sixteen a dim, turned in its registers. Bound: HBM, 1 B in, 2 B out a value (16-bit rows).
// Measured: 8192 tokens of 4 heads of 256 as bf16 12 us, 50 MB, 4.1 TB/s.
template <int DT>
__global__ void __launch_bounds__(kThreads) read_kernel(Kv8 c, const int32_t* __restrict__ starts, Ragged rows,
                                                        void* __restrict__ kout, void* __restrict__ vout) {
  const int seq = blockIdx.z, head = blockIdx.y >> 1;
  const bool is_v = blockIdx.y & 1;
  int r0, r1;
  rows_of(rows, seq, r0, r1);
  const int64_t room = (int64_t)c.max_pages * c.page;
  const int64_t start = starts[seq], end = start + (r1 - r0);
  const int d = c.d, page = c.page, per = d / 8;
  const int64_t g0 = start >= 0 ? start / 16 : -((15 - start) / 16), g1 = (end + 15 + (end < 0 ? -15 : 0)) / 16;
  void* out = is_v ? vout : kout;
  for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < (g1 - g0) * per; i += (int64_t)gridDim.x * kThreads) {
    const int64_t t0 = 16 * (g0 + i / per);
    const int at = 8 * (int)(i % per);
    int pid = -1;
    if (t0 >= 0 && t0 < room) pid = c.table[(int64_t)seq * c.table_stride + t0 / page];
    const bool ok = pid >= 0 && pid < c.pages;
    uint32_t w[16][2] = {};  // of K: 8 codes of each position; of V: 16 codes of each of the 8 dims, as [2 e + half]
    float s = __builtin_nanf("");
    if (ok) {
      s = (is_v ? c.vs : c.ks)[(int64_t)pid * c.heads + head];
      const int8_t* codes = (is_v ? c.v : c.k) + ((int64_t)pid * c.heads + head) * page * d;
      const int off = (int)(t0 % page);
      if (is_v) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const uint4 o = *(const uint4*)(codes + (int64_t)(at + e) * page + off);
          w[2 * e][0] = o.x; w[2 * e][1] = o.y; w[2 * e + 1][0] = o.z; w[2 * e + 1][1] = o.w;
        }
      } else {
#pragma unroll
        for (int t = 0; t < 16; ++t) {
          const uint2 o = *(const uint2*)(codes + (int64_t)(off + t) * d + at);
          w[t][0] = o.x; w[t][1] = o.y;
        }
      }
    }
#pragma unroll
    for (int t = 0; t < 16; ++t) {
      if (t0 + t < start || t0 + t >= end) continue;
      float v[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const uint32_t b = is_v ? w[2 * e + (t >> 3)][(t >> 2) & 1] >> 8 * (t & 3) : w[t][e >> 2] >> 8 * (e & 3);
        v[e] = (float)(int8_t)b * s;
        asm("" : "+v"(v[e]));  // rounded to fp32 here: not joined with the rounding to fp16
      }
      store8<DT>(out, ((int64_t)(r0 + (t0 + t - start)) * c.heads + head) * d + at, v);
    }
  }
}

}  // namespace

hipError_t launch_kv8_append(const Kv8& c, int dtype, const void* key, int64_t kt, int64_t kh, const void* value,
                             int64_t vt, int64_t vh, const int32_t* lens, const Ragged& rows, int64_t max_new,
                             hipStream_t stream) {
  // a page more than the tokens fill: they may start inside one
  const int64_t pages = (max_new + c.page - 2) / c.page + 1;
  const dim3 grid((unsigned)(pages < 1024 ? pages : 1024), 2 * c.heads, rows.seqs);
#define GGUF_DEC_APPEND(DT) append_kernel<DT><<<grid, kThreads, 0, stream>>>(c, key, kt, kh, value, vt, vh, lens, rows)
  GGUF_DEC_FLOATS(dtype, GGUF_DEC_APPEND)
#undef GGUF_DEC_APPEND
  return hipGetLastError();
}

hipError_t launch_kv8_read(const Kv8& c, int dtype, const int32_t* starts, const Ragged& rows, int64_t max_tokens,
                           void* kout, void* vout, hipStream_t stream) {
  const int64_t items = ((max_tokens + 14) / 16 + 1) * (c.d / 8), blocks = (items + kThreads - 1) / kThreads;
  const dim3 grid((unsigned)(blocks < 4096 ? blocks : 4096), 2 * c.heads, rows.seqs);
#define GGUF_DEC_READ(DT) read_kernel<DT><<<grid, kThreads, 0, stream>>>(c, starts, rows, kout, vout)
  GGUF_DEC_FLOATS(dtype, GGUF_DEC_READ)
#undef GGUF_DEC_READ
  return hipGetLastError();
}

}  // namespace gguf_dec
