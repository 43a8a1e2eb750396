// Moves a sequence's accepted draft rows together in the 8-bit cache (include/gguf_decoder.h: contract; kv8.hip: the codes).
#include "kv8_codes.h"
#include "rotary.h"

namespace gguf_dec {

namespace {

constexpr int kThreads = 256;

// One workgroup takes one (sequence, head) of K or V, so a scale has one writer. Row path[j] goes to place j. The path grows
// strictly, so from its first j with path[j] != j on every row moves down, and pages in ascending order never lose a row that
// is still to move: what a page receives comes from itself or from later pages, which are as they were. A page's scale grows to what
// the rows from other pages need, its codes are rounded again, then rows are read, waited for and written, some at a time;
// a later row's source lies behind every place written before.
//
// Bound: latency of a few dependent loads (lengths, path, table, scales, codes); a path is some rows of some hundred bytes. 8 drafts of one
// sequence 5.7 us, 64 drafts of 64 sequences over pages of 16 tokens 9.8; where pages' scales have to grow 9.9.
__global__ void __launch_bounds__(kThreads) keep_kernel(Kv8 c, const int32_t* __restrict__ path, int64_t path_stride, int m,
                                                        const int32_t* __restrict__ lens, Ragged rows) {
  __shared__ int ph[kMostKept], off[kMostKept], from[kMostKept];  // a row's (page, head), place in it, and page of the table
  __shared__ float src[kMostKept];                                // and scale
  __shared__ int cut, moved;
  __shared__ uint32_t most[kThreads / 64];
  const int tid = threadIdx.x;
  const bool is_v = blockIdx.x & 1;
  const int head = blockIdx.x / 2 % c.heads, seq = blockIdx.x / 2 / c.heads;
  int r0, r1;
  rows_of(rows, seq, r0, r1);
  const int n = r1 - r0, page = c.page, d = c.d;
  const int64_t room = (int64_t)c.max_pages * page;
  const int64_t base = (int64_t)lens[seq] - n;
  const int32_t* own = path + seq * path_stride;
  const int32_t* table = c.table + (int64_t)seq * c.table_stride;
  float* scales = is_v ? c.vs : c.ks;
  int8_t* codes = is_v ? c.v : c.k;
  if (tid == 0) cut = moved = m;
  __syncthreads();
  for (int j = tid; j < m; j += kThreads) {
    const int r = own[j];
    if (r < 0 || r >= n || (j > 0 && r <= own[j - 1])) {
      atomicMin(&cut, j);
    } else {
      if (r != j) atomicMin(&moved, j);
      const int64_t at = base + r;
      const int p = at >= 0 && at < room ? (int)(at / page) : -1;
      const int pid = p >= 0 ? table[p] : -1;
      const bool ok = pid >= 0 && pid < c.pages;
      from[j] = p;
      ph[j] = ok ? pid * c.heads + head : -1;
      off[j] = p >= 0 ? (int)(at - (int64_t)p * page) : 0;
      src[j] = ok ? scales[ph[j]] : __builtin_nanf("");
    }
  }
  __syncthreads();
  const int64_t lo = max(base + moved, (int64_t)0), hi = min(base + cut, room);  // places that receive rows
  for (int64_t p0 = lo / page * page; p0 < hi; p0 += page) {
    const int p = (int)(p0 / page), pid = table[p];
    if (pid < 0 || pid >= c.pages) continue;  // uniform
    const int at = pid * c.heads + head;
    const int j0 = (int)(max(lo, p0) - base), count = (int)(min(hi, p0 + page) - max(lo, p0)), t0 = (int)(max(lo, p0) - p0);
    int8_t* mine = codes + (int64_t)at * page * d;
    const int words = is_v ? d : d / 4, items = count * words;
    // K: item i is word i % words of row i / words; V: dim i / count of row i % count, whose place is a byte
    const auto read = [&](int i, int& j) __attribute__((always_inline)) {
      j = is_v ? i % count : i / words;
      const int x = is_v ? i / count : i - j * words, row = j0 + j;
      if (ph[row] < 0) return 0u;
      const int8_t* q = codes + (int64_t)ph[row] * page * d;
      return is_v ? (uint32_t)(uint8_t)q[(int64_t)x * page + off[row]] : *(const uint32_t*)(q + (int64_t)off[row] * d + 4 * x);
    };

    // what the rows from other pages need of the scale
    uint32_t big = 0;
    for (int i = tid; i < items; i += kThreads) {
      int j;
      const uint32_t w = read(i, j);
      if (from[j0 + j] == p) continue;
      int a = 0;
#pragma unroll
      for (int b = 0; b < 4; ++b) a = max(a, abs((int)(int8_t)(w >> 8 * b)));
      const float from_scale = src[j0 + j];  // one that is not finite goes on, whatever the codes
      const float need = from_scale <= 3.4e38f ? (float)a / 127.0f * from_scale : from_scale;
      big = max(big, __float_as_uint(need) & 0x7FFFFFFFu);
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) big = max(big, (uint32_t)__shfl_xor((int)big, o, 64));
    const float was = scales[at];
    __syncthreads();  // the previous page's `most` has been read
    if ((tid & 63) == 0) most[tid >> 6] = big;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kThreads / 64; ++w) big = max(big, most[w]);
    const float fresh = __uint_as_float(big);
    const Rescale s = grown(was, fresh < kLeastScale ? 0.0f : fresh);
    if (s.shrink) {
      for (int i = tid; i < page * d / 4; i += kThreads) ((uint32_t*)mine)[i] = rescale4(((uint32_t*)mine)[i], s.ratio);
      if (tid == 0) scales[at] = s.scale;
      __syncthreads();
    }
    for (int i0 = 0; i0 < items; i0 += kThreads) {
      const int i = i0 + tid;
      int j = 0;
      uint32_t w = 0;
      if (i < items) {
        w = read(i, j);
        if (from[j0 + j] != p) w = rescale4(w, src[j0 + j] / s.scale);
      }
      __syncthreads();
      if (i < items) {
        if (is_v) mine[(int64_t)(i / count) * page + t0 + j] = (int8_t)w;
        else *(uint32_t*)(mine + (int64_t)(t0 + j) * d + 4 * (i - j * words)) = w;
      }
    }
    __syncthreads();  // a row that comes from the next page is read by what wrote here
  }
}

}  // namespace

hipError_t launch_kv8_keep(const Kv8& c, const int32_t* path, int64_t path_stride, int m, const int32_t* lens,
                           const Ragged& rows, hipStream_t stream) {
  keep_kernel<<<(unsigned)(2 * rows.seqs * c.heads), kThreads, 0, stream>>>(c, path, path_stride, m, lens, rows);
  return hipGetLastError();
}

}  // namespace gguf_dec
