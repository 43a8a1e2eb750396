// Log probability, rank, entropy and best tokens of rows of logits (include/gguf_decoder.h).
//
// With m the row's maximum, Z = sum e^{x - m} and A = sum (x - m) e^{x - m}: logprob(x) = x - m -
// log Z, entropy = log Z - A / Z. Each row is cut into chunks; a workgroup holds a chunk in registers,
// so the logits are read once, and leaves its m, Z, A, the tokens before the given one and its best
// `top`; merge_kernel joins a row's chunks in order.
//
// The best of a chunk: values are ordered by one 64-bit key, (value in an order-preserving
// unsigned form) << 32 | ~index, so that all keys differ and equal values go by index. The k-th
// largest of the threads' own maxima bounds the k-th largest key from below, and exactly k threads can hold keys at
// or above it: those (at most k times the values a thread) go to a list, and each finds its place by counting
// the larger ones.
#include "dec_common.h"

namespace gguf_dec {

namespace {

constexpr int kThreads = 256;
constexpr float kLog2e = 1.4426950408889634f;

// order-preserving: a < b as floats <=> key(a) < key(b); -0 = +0; NaN above +inf
__device__ __forceinline__ uint32_t order_key(float x) {
  if (x != x) return 0xFFFFFFFFu;
  const uint32_t b = __float_as_uint(x + 0.0f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}

// the value of an order key (not 0)
__device__ __forceinline__ float value_of(uint32_t key) {
  if (key == 0xFFFFFFFFu) return __builtin_nanf("");
  return __uint_as_float(key & 0x80000000u ? key & 0x7FFFFFFFu : ~key);
}

__device__ __forceinline__ uint64_t full_key(float x, uint32_t index) {
  return (uint64_t)order_key(x) << 32 | (0xFFFFFFFFu - index);
}

__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v = fmaxf(v, __shfl_xor(v, off, 64));
  return v;
}

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
  return v;
}

__device__ __forceinline__ int wave_sum(int v) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
  return v;
}

// The k largest of the workgroup's keys, E a thread (0: none; all others distinct), as emit(place, key) for
// places 0 .. ; fewer where there are fewer. list: E * k keys of LDS, most: kThreads.
template <int E, class F>
__device__ __forceinline__ void select_top(const uint64_t (&key)[E], int k, uint64_t* most, uint64_t* list, F&& emit) {
  __shared__ uint64_t least;
  __shared__ int count;
  const int tid = threadIdx.x;
  uint64_t mine = 0;
#pragma unroll
  for (int e = 0; e < E; ++e) mine = key[e] > mine ? key[e] : mine;
  __syncthreads();
  most[tid] = mine;
  if (tid == 0) {
    least = 1;
    count = 0;
  }
  __syncthreads();
  if (mine) {
    int above = 0;
    for (int i = 0; i < kThreads; i += 2) {
      const ulonglong2 o = *(const ulonglong2*)(most + i);
      above += (o.x > mine) + (o.y > mine);
    }
    if (above == k - 1) least = mine;
  }
  __syncthreads();
  if (mine >= least) {
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (key[e] >= least) list[atomicAdd(&count, 1)] = key[e];
  }
  __syncthreads();
  const int n = count;
  for (int i = tid; i < n; i += kThreads) {
    const uint64_t x = list[i];
    int above = 0;
    for (int j = 0; j < n; ++j) above += list[j] > x;
    if (above < k) emit(above, x);
  }
}

// what a chunk leaves: m, Z, A, and the tokens before the given one
struct Part {
  float m, z, a;
  int before;
};

// the next float below x (x finite)
__device__ __forceinline__ float below(float x) {
  const uint32_t b = __float_as_uint(x + 0.0f);  // -0 -> +0
  return b == 0 ? __uint_as_float(0x80000001u) : __uint_as_float(b & 0x80000000u ? b + 1 : b - 1);
}

// One workgroup a chunk of E values a thread. VALU-bound (512 bf16 rows of 248320: 98 us, 2.6 TB/s, by counters 24 VALU
// instructions a value, issuing for 80 % of the time; 200 us with a 64-bit key for every value), so what is done for every
// value is kept short. The rank is one comparison against the given value, or the next one below it for pieces before
// the given token, whose equal values count too. The best
// tokens go by the threads' maxima: the top-th largest of a wave's bounds the chunk's top-th best from below, and
// only what reaches it is looked at by key. Where ties make that too many for the list, keys decide from the start
// (select_top).
template <int DT, int E>
__global__ void __launch_bounds__(kThreads) chunk_kernel(const void* __restrict__ x, int64_t stride, int vocab,
                                                         const int64_t* __restrict__ ids, int64_t id_stride, int top,
                                                         Part* __restrict__ parts, uint64_t* __restrict__ keys) {
  constexpr int VEC = 8, WAVES = kThreads / 64;
  constexpr int SIZE = DT == kF32 ? 4 : 2;
  extern __shared__ __align__(16) uint64_t lds[];  // most, list
  __shared__ float fs[4][WAVES];
  __shared__ int is[WAVES], count;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t row = blockIdx.y, chunk = blockIdx.x, chunks = gridDim.x;
  const char* base = (const char*)x + row * stride * SIZE;
  // chunks are cut on the 16-byte grid of memory: the row begins `skip` elements into the first piece
  const int skip = (int)((uintptr_t)base % (VEC * SIZE)) / SIZE;

  float v[E];
  int first[E / VEC];  // index of each piece's first value
#pragma unroll
  for (int p = 0; p < E / VEC; ++p) {
    const int64_t at = (chunk * (E / VEC) + p) * kThreads * VEC + tid * VEC - skip;
    first[p] = (int)(at < vocab ? at : vocab);
    float w[8];
    if (at >= 0 && at + VEC <= vocab) {
      load8<DT>(base, at, w);
    } else {
#pragma unroll
      for (int e = 0; e < VEC; ++e) w[e] = at + e >= 0 && at + e < vocab ? load1<DT>(base, at + e) : -__builtin_inff();
    }
#pragma unroll
    for (int e = 0; e < VEC; ++e) v[p * VEC + e] = w[e];
  }
  const int64_t id = ids[row * id_stride];
  const bool has = id >= 0 && id < vocab;
  const float given = has ? load1<DT>(base, id) : 0.0f;

  float mine = -__builtin_inff();
#pragma unroll
  for (int e = 0; e < E; ++e) mine = fmaxf(mine, v[e]);
  float m = wave_max(mine);
  // the wave's bound: the top-th largest of its lanes' maxima, bit by bit of its order key
  float bound = -__builtin_inff();
  if (top > 0) {
    const uint32_t order = order_key(mine);
    uint32_t key = 0;
#pragma unroll
    for (int bit = 31; bit >= 0; --bit) {
      const uint32_t next = key | 1u << bit;
      if (__popcll(__ballot(order >= next)) >= top) key = next;
    }
    if (key) bound = value_of(key);
  }
  if (lane == 0) {
    fs[0][wave] = m;
    fs[3][wave] = bound;
  }
  if (tid == 0) count = 0;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < WAVES; ++w) {
    m = fmaxf(m, fs[0][w]);
    bound = fmaxf(bound, fs[3][w]);
  }
  // a chunk of -inf alone has Z = A = 0
  const float mm = m == -__builtin_inff() ? 0.0f : m;
  float z = 0.0f, a = 0.0f;
  int before = 0;
  const bool plain = given > -__builtin_inff() && given < __builtin_inff();
#pragma unroll
  for (int p = 0; p < E / VEC; ++p) {
    const float than = first[p] + VEC <= id ? below(given) : given;
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      const float y = v[p * VEC + e];
      const float d = y - mm;  // before the change of base: m log2 e rounded would shift every weight alike
      const float t = __builtin_amdgcn_exp2f(d * kLog2e);
      z += t;
      a = fmaf(t, fmaxf(d, -1000.0f), a);  // also where d is -inf; a NaN is in z
      before += y > than;
    }
    if (!plain || (first[p] <= id && id < first[p] + VEC)) {  // the piece of the given token, or a given value that has no next one
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const int i = first[p] + e;
        const float y = v[p * VEC + e];
        before -= y > than;
        before += i >= 0 && i < vocab && (y > given || (y == given && i < id));
      }
    }
  }
  z = wave_sum(z);
  a = wave_sum(a);
  before = wave_sum(before);
  if (lane == 0) {
    fs[1][wave] = z;
    fs[2][wave] = a;
    is[wave] = before;
  }
  uint64_t* out = keys + (row * chunks + chunk) * top;
  uint64_t* list = lds + kThreads;
  if (top > 0) {
    if (tid < top) out[tid] = 0;
    // NaN is above everything: a thread's maximum does not show it
    const bool odd = z != z;
    if (mine >= bound || odd) {
      uint32_t reach = 0;
#pragma unroll
      for (int e = 0; e < E; ++e) reach |= (uint32_t)!(v[e] < bound) << e;
      // (a value of the padding, -inf, reaches a bound of -inf only)
#pragma unroll
      for (int p = 0; p < E / VEC; ++p)
#pragma unroll
        for (int e = 0; e < VEC; ++e)
          if (first[p] < 0 || first[p] + VEC > vocab)
            if (first[p] + e < 0 || first[p] + e >= vocab) reach &= ~(1u << (p * VEC + e));
      int at = atomicAdd(&count, __popc(reach));
      for (; reach; reach &= reach - 1, ++at) {
        const int e = __ffs(reach) - 1, i = (int)((chunk * (E / VEC) + e / VEC) * kThreads * VEC + tid * VEC - skip) + e % VEC;
        if (at < E * top) list[at] = full_key(load1<DT>(base, i), i);  // read again: few are
      }
    }
  }
  __syncthreads();
  if (tid == 0) {
    Part p = {m, 0.0f, 0.0f, 0};
    for (int w = 0; w < WAVES; ++w) {
      p.z += fs[1][w];
      p.a += fs[2][w];
      p.before += is[w];
    }
    parts[row * chunks + chunk] = p;
  }
  if (top == 0) return;
  const int n = count;
  if (n <= E * top) {
    for (int i = tid; i < n; i += kThreads) {
      const uint64_t k = list[i];
      int above = 0;
      for (int j = 0; j < n; ++j) above += list[j] > k;
      if (above < top) out[above] = k;
    }
  } else {  // uniform
    uint64_t key[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int i = first[e / VEC] + e % VEC;
      key[e] = i >= 0 && i < vocab ? full_key(v[e], i) : 0;
    }
    select_top(key, top, lds, list, [&](int place, uint64_t k) { out[place] = k; });
  }
}

// One workgroup a row. The best of all are among the chunks' best.
template <int E>
__global__ void __launch_bounds__(kThreads) merge_kernel(const Part* __restrict__ parts, const uint64_t* __restrict__ keys,
                                                         int chunks, int top, const void* __restrict__ x, int64_t stride,
                                                         int dtype, int vocab, const int64_t* __restrict__ ids,
                                                         int64_t id_stride, float* __restrict__ logprobs,
                                                         int32_t* __restrict__ ranks, float* __restrict__ entropy,
                                                         float* __restrict__ top_logprobs, int32_t* __restrict__ top_ids) {
  extern __shared__ __align__(16) uint64_t lds[];
  __shared__ float lse_s[2];
  const int tid = threadIdx.x;
  const int64_t row = blockIdx.x;
  if (tid < 64) {  // the first wave: each lane some chunks, then over the lanes
    const Part* p = parts + row * chunks;
    float m = -__builtin_inff();
    for (int i = tid; i < chunks; i += 64) m = fmaxf(m, p[i].m);
    m = wave_max(m);
    float z = 0.0f, a = 0.0f;
    int before = 0;
    for (int i = tid; i < chunks; i += 64) {
      before += p[i].before;
      if (p[i].z == 0.0f) continue;  // -inf alone
      const float d = p[i].m - m, f = __expf(d);
      if (f == 0.0f && p[i].z == p[i].z) continue;  // far below: z d may pass fp32's range. A NaN, which m does not show, stays
      z += p[i].z * f;
      a += (p[i].a + p[i].z * d) * f;
    }
    z = wave_sum(z);
    a = wave_sum(a);
    before = wave_sum(before);
    if (tid == 0) {
      const float lz = logf(z);  // Z = 0 (a row of -inf): NaN below, as -inf - (-inf)
      const int64_t id = ids[row * id_stride];
      const bool has = id >= 0 && id < vocab;
      const bool none = z == 0.0f;
      logprobs[row] = has && !none ? gguf::load_x(x, row * stride + id, dtype) - m - lz : __builtin_nanf("");
      ranks[row] = has ? before + 1 : 0;
      entropy[row] = none ? __builtin_nanf("") : lz - a / z;
      lse_s[0] = none ? __builtin_nanf("") : m;
      lse_s[1] = lz;
    }
  }
  if (top == 0) return;
  __syncthreads();
  const float m = lse_s[0], lz = lse_s[1];
  const int64_t n = (int64_t)chunks * top;
  uint64_t key[E];
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int64_t i = (int64_t)e * kThreads + tid;
    key[e] = i < n ? keys[row * n + i] : 0;
  }
  select_top(key, top, lds, lds + kThreads, [&](int place, uint64_t k) {
    top_logprobs[row * top + place] = value_of((uint32_t)(k >> 32)) - m - lz;
    top_ids[row * top + place] = (int32_t)(0xFFFFFFFFu - (uint32_t)k);
  });
}

constexpr int kMergeMost = 64;  // keys a thread of merge_kernel, at most

int64_t chunks_of(int64_t vocab, int per) {  // one piece more: a row may begin inside a 16-byte piece
  const int64_t size = (int64_t)kThreads * per;
  return (vocab + 7 + size - 1) / size;
}

// values of a chunk a thread: 32, or 8 where chunks of 32 would not give every CU a workgroup and the best of the
// smaller ones, four times as many, still fit merge_kernel. Calls in us, 32 / 8 values, 20 best of bf16 logits: of 151936
// one row 15.5 / 14.7, 8 rows 15.9 / 16.0, 16 rows 16.5 / 17.3, 64 rows 20.1 / 29.7; of 32000 one row 15.2 / 13.9, 64 rows
// 15.8 / 15.8, 128 rows 16.4 / 19.0.
int per_thread(int64_t rows, int64_t vocab, int64_t top) {
  return rows * chunks_of(vocab, 32) < gguf::device_cus() && vocab < (1 << 20) &&
                 chunks_of(vocab, 8) * top <= kMergeMost * kThreads
             ? 8
             : 32;
}

}  // namespace

// the largest vocabulary whose chunks of 32 values a thread leave no more keys than merge_kernel holds
int64_t logprobs_most_vocab(int64_t top) {
  return top == 0 ? INT32_MAX - 65536 : (int64_t)(kMergeMost * kThreads / top) * kThreads * 32 - 8;
}

size_t logprobs_workspace(int64_t rows, int64_t vocab, int64_t top) {
  return (size_t)rows * chunks_of(vocab, per_thread(rows, vocab, top)) * (sizeof(Part) + top * sizeof(uint64_t));
}

hipError_t launch_logprobs(const void* x, int dtype, int64_t stride, int64_t rows, int64_t vocab, const int64_t* ids,
                           int64_t id_stride, int top, float* logprobs, int32_t* ranks, float* entropy,
                           float* top_logprobs, int32_t* top_ids, void* ws, hipStream_t stream) {
  const int per = per_thread(rows, vocab, top);
  const int64_t chunks = chunks_of(vocab, per);
  if (chunks * top > kMergeMost * kThreads) return hipErrorInvalidValue;  // past logprobs_most_vocab
  uint64_t* keys = (uint64_t*)ws;  // first: 8-byte aligned
  Part* parts = (Part*)(keys + rows * chunks * top);
  constexpr int64_t kRows = 65535;  // of a launch
  for (int64_t r = 0; r < rows; r += kRows) {
    const int64_t n = rows - r < kRows ? rows - r : kRows;
    const int size = dtype == kF32 ? 4 : 2;
    const void* xr = (const char*)x + r * stride * size;
    Part* pr = parts + r * chunks;
    uint64_t* kr = keys + r * chunks * top;
    const int64_t* ir = ids + r * id_stride;
    const size_t lds = top ? (kThreads + (size_t)per * top) * 8 : 0;
    const dim3 grid((unsigned)chunks, (unsigned)n);
#define GGUF_DEC_CHUNK(DT)                                                                                          \
  if (per == 8) chunk_kernel<DT, 8><<<grid, kThreads, lds, stream>>>(xr, stride, (int)vocab, ir, id_stride, top, pr, kr); \
  else chunk_kernel<DT, 32><<<grid, kThreads, lds, stream>>>(xr, stride, (int)vocab, ir, id_stride, top, pr, kr)
    GGUF_DEC_FLOATS(dtype, GGUF_DEC_CHUNK)
#undef GGUF_DEC_CHUNK
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
#define GGUF_DEC_MERGE(E)                                                                                            \
  merge_kernel<E><<<(unsigned)n, kThreads, top ? (kThreads + (size_t)E * top) * 8 : 0, stream>>>(                    \
      pr, kr, (int)chunks, top, xr, stride, dtype, (int)vocab, ir, id_stride, logprobs + r, ranks + r, entropy + r, \
      top ? top_logprobs + r * top : nullptr, top ? top_ids + r * top : nullptr)
    const int64_t each = (chunks * top + kThreads - 1) / kThreads;  // keys a thread
    if (each <= 2) {
      GGUF_DEC_MERGE(2);
    } else if (each <= 8) {
      GGUF_DEC_MERGE(8);
    } else {
      GGUF_DEC_MERGE(kMergeMost);
    }
#undef GGUF_DEC_MERGE
    if ((e = hipGetLastError()) != hipSuccess) return e;
  }
  return hipSuccess;
}

}  // namespace gguf_dec
