// The norm behind a block, its gate and residual scale, and the next block's norm, in one pass:
//   u = x;  u = u rsqrt(mean u^2 + eps) w_in;  u = u act(gate);  h = residual + scale u;
//   out = h rsqrt(mean h^2 + eps) w_out
// (every part but x optional). A row's values stay in registers from the loads to the stores, so each input is read and
// each output written once; sums of squares are fp32, and only h and out are rounded.
//
// Bound by memory for many rows, by the launch and a row's chain of loads, sums and stores for few: 8192 rows of 5120 values, all
// bf16, both norms: 76 us (4.4 TB/s; a copy reaches 4.9 to 5.2); 8192 x 48 heads of 128 with a gate: 56 us (5.3
// TB/s); 4 rows of 5120: 3.4 us in a graph, 6.7 by itself, where the host takes the time.
#include <algorithm>

#include "norm.h"

namespace gguf_dec {

namespace {

constexpr float kLog2e = 1.4426950408889634f, kLog2eRest = 1.9259629911e-8f, kLn2 = 0.6931471805599453f;

// Where h is rounded to 8 or 11 bits: by the hardware's 2^x of an argument rounded to fp32, off by up to 2^-24 of the argument (2^-17 of the
// result), and 0 where the sigmoid is subnormal (g below -87). Where h is fp32: sigmoid(g) = t^[g < 0] / (1 + t), t = e^-|g|, to some steps of
// fp32 and down to its least number. What rounding the argument left, lo, goes into t = 2^hi (1 + lo ln 2); and as the hardware's 2^x has no
// subnormal results, below 2^-100 (where 1 + t is 1) it is taken of hi + 64, and 2^-64 multiplied in last. For all types that would take
// 8192 x 48 heads of 128 from 61 to 72 us in bf16; in fp32 they take 104 instead of 103, 8192 rows of 4097 values 164 instead of 152.
template <int RT>
__device__ __forceinline__ float act_of(float g, int act) {
#pragma clang fp contract(off)  // hi + 64 is of the rounded hi
  if constexpr (RT != kF32) {
    const float s = __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-kLog2e * g));  // of -inf: 1 / inf
    return act == kActSilu ? g * s : act == kActSigmoid ? s : g;
  }
  const float a = fabsf(g) > 200.0f ? 200.0f : fabsf(g);  // e^-200 is 0; a NaN stays
  const float hi = -a * kLog2e, lo = __builtin_fmaf(-a, kLog2eRest, __builtin_fmaf(-a, kLog2e, -hi));
  const bool least = g < 0.0f && hi < -100.0f;
  const float e = __builtin_amdgcn_exp2f(least ? hi + 64.0f : hi);
  const float t = __builtin_fmaf(e, lo * kLn2, e);
  const float x = act == kActSilu ? g : 1.0f;
  const float y = (g < 0.0f ? x * t : x) * (least ? 0x1p-64f : __builtin_amdgcn_rcpf(1.0f + t));
  return act == kActNone ? g : y;
}

// Sum over the row's lanes (a power of two up to 64, aligned) or over the workgroup, of whose waves each holds ITEMS parts. Each
// 64 pieces are summed for themselves, then these sums, in one order, so that a row has the same bits in every form that takes it.
template <bool WG, int ITEMS>
__device__ __forceinline__ float row_sum(const float (&sums)[ITEMS], int lanes, float* part) {
  if constexpr (!WG) {
    float v = sums[0];
    for (int off = 1; off < lanes; off <<= 1) v += __shfl_xor(v, off, 64);
    return v;
  } else {
    const int waves = blockDim.x >> 6, wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    // the sums of ITEMS values together: after the first steps lane l holds a part of the (l % ITEMS)-th alone
    float s[ITEMS];
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) s[i] = sums[i];
#pragma unroll
    for (int left = ITEMS; left > 1; left /= 2) {
      const int off = ITEMS / left;
      const bool odd = lane & off;
#pragma unroll
      for (int i = 0; i < left / 2; ++i) {
        const float mine = odd ? s[2 * i + 1] : s[2 * i], other = odd ? s[2 * i] : s[2 * i + 1];
        s[i] = mine + __shfl_xor(other, off, 64);
      }
    }
#pragma unroll
    for (int off = ITEMS; off < 64; off <<= 1) s[0] += __shfl_xor(s[0], off, 64);
    __syncthreads();  // the last sum's parts have been read
    if (lane < ITEMS) part[lane * waves + wave] = s[0];
    __syncthreads();
    float v = part[0];
    for (int g = 1; g < ITEMS * waves; ++g) v += part[g];
    return v;
  }
}

__device__ __forceinline__ void at_row(const RowStride& s, int64_t token, int head, int64_t& at) {
  at = token * s.t + head * s.h;
}

// A row is ITEMS pieces of 8 values a lane: `lanes` lanes of a wave take it, or (WG) the whole workgroup. Weights are held over
// the rows that a lane takes; of four pieces a lane, weights and gates are read as they are needed, for the registers.
template <int DT, int RT, int ITEMS, bool WG>
__global__ void __launch_bounds__(WG ? 1024 : 256) norm_kernel(NormArgs a, int lanes) {
  __shared__ float part[64];
  const int per = WG ? 1 : blockDim.x / lanes;  // rows a workgroup at a time
  const int lane = WG ? threadIdx.x : threadIdx.x % lanes, width = WG ? blockDim.x : lanes;
  const int mine = WG ? 0 : threadIdx.x / lanes;
  const float over = 1.0f / (float)a.n;
  constexpr bool HELD = ITEMS < 4;
  float wi[HELD ? ITEMS : 1][8], wo[HELD ? ITEMS : 1][8];
  const auto weight = [&](const float* from, int c, float (&w)[8]) __attribute__((always_inline)) {
#pragma unroll
    for (int e = 0; e < 8; ++e) w[e] = 0.0f;
    if (from && c < a.n) load8<kF32>(from, c, w);
  };
  if constexpr (HELD) {
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      weight(a.inner, 8 * (lane + i * width), wi[i]);
      weight(a.outer, 8 * (lane + i * width), wo[i]);
    }
  }
  for (int64_t r0 = (int64_t)blockIdx.x * per; r0 < a.rows; r0 += (int64_t)gridDim.x * per) {
    const bool ok = r0 + mine < a.rows;
    const int64_t row = ok ? r0 + mine : a.rows - 1;  // lanes past the last row take it again, and store nothing
    const int64_t token = a.heads == 1 ? row : row / a.heads;
    const int head = a.heads == 1 ? 0 : (int)(row - token * a.heads);
    int64_t xa, ra, ga;
    at_row(a.xs, token, head, xa);
    at_row(a.rs, token, head, ra);
    at_row(a.gs, token, head, ga);
    float u[ITEMS][8], g[HELD ? ITEMS : 1][8], h[ITEMS][8];
    const auto gate = [&](int c, float (&to)[8]) __attribute__((always_inline)) {
#pragma unroll
      for (int e = 0; e < 8; ++e) to[e] = 1.0f;
      if (a.gate && c < a.n) load8<DT>(a.gate, ga + c, to);
    };
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      const int c = 8 * (lane + i * width);
#pragma unroll
      for (int e = 0; e < 8; ++e) u[i][e] = h[i][e] = 0.0f;
      if constexpr (HELD) gate(c, g[i]);
      if (c < a.n) {
        load8<DT>(a.x, xa + c, u[i]);
        if (a.residual) load8<RT>(a.residual, ra + c, h[i]);
      }
    }
    if (a.inner) {
      float sum[ITEMS] = {};
#pragma unroll
      for (int i = 0; i < ITEMS; ++i)
#pragma unroll
        for (int e = 0; e < 8; ++e) sum[i] += u[i][e] * u[i][e];
      const float by = rsqrtf(row_sum<WG>(sum, lanes, part) * over + a.eps);
#pragma unroll
      for (int i = 0; i < ITEMS; ++i) {
        if constexpr (!HELD) weight(a.inner, 8 * (lane + i * width), wi[0]);
#pragma unroll
        for (int e = 0; e < 8; ++e) u[i][e] *= by * wi[HELD ? i : 0][e];
      }
    }
    float sum[ITEMS] = {};
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      const int c = 8 * (lane + i * width);
      if constexpr (!HELD) gate(c, g[0]);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        if (a.gate) u[i][e] *= act_of<RT>(g[HELD ? i : 0][e], a.act);
        h[i][e] += a.scale * u[i][e];
        if (c < a.n) sum[i] += h[i][e] * h[i][e];
      }
      if (c < a.n && ok) store8<RT>(a.hidden, row * a.n + c, h[i]);
    }
    if (a.outer) {
      const float by = rsqrtf(row_sum<WG>(sum, lanes, part) * over + a.eps);
#pragma unroll
      for (int i = 0; i < ITEMS; ++i) {
        const int c = 8 * (lane + i * width);
        if constexpr (!HELD) weight(a.outer, c, wo[0]);
#pragma unroll
        for (int e = 0; e < 8; ++e) h[i][e] *= by * wo[HELD ? i : 0][e];
        if (c < a.n && ok) store8<DT>(a.out, row * a.n + c, h[i]);
      }
    }
  }
}

// Rows of any length up to ITEMS values a thread, and of any alignment: a workgroup a row, whose values stay in registers. Loads and
// stores of single values bound it: 8192 rows of 4097 values in bf16 108 us (2.5 TB/s), in fp32 108 (5.0). Weights are read as they are
// needed: held, they left two workgroups a CU (179 us in bf16).
template <int DT, int RT, int ITEMS>
__global__ void __launch_bounds__(1024) norm_odd_kernel(NormArgs a) {
  __shared__ float part[16];
  const float over = 1.0f / (float)a.n;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const int64_t token = row / a.heads;
    const int head = (int)(row - token * a.heads);
    int64_t xa, ra, ga;
    at_row(a.xs, token, head, xa);
    at_row(a.rs, token, head, ra);
    at_row(a.gs, token, head, ga);
    float u[ITEMS], g[ITEMS], h[ITEMS], sum[1] = {};
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      const int c = threadIdx.x + i * blockDim.x;
      u[i] = h[i] = 0.0f, g[i] = 1.0f;
      if (c < a.n) {
        u[i] = load1<DT>(a.x, xa + c);
        if (a.residual) h[i] = load1<RT>(a.residual, ra + c);
        if (a.gate) g[i] = load1<DT>(a.gate, ga + c);
      }
      sum[0] += u[i] * u[i];
    }
    if (a.inner) {
      const float by = rsqrtf(row_sum<true>(sum, 64, part) * over + a.eps);
#pragma unroll
      for (int i = 0; i < ITEMS; ++i) {
        const int c = threadIdx.x + i * blockDim.x;
        if (c < a.n) u[i] *= by * a.inner[c];
      }
    }
    sum[0] = 0.0f;
    if (a.gate) {
#pragma unroll
      for (int i = 0; i < ITEMS; ++i) u[i] *= act_of<RT>(g[i], a.act);
    }
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      const int c = threadIdx.x + i * blockDim.x;
      h[i] += a.scale * u[i];
      if (c < a.n) {
        sum[0] += h[i] * h[i];
        store1<RT>(a.hidden, row * a.n + c, h[i]);
      }
    }
    if (a.outer) {
      const float by = rsqrtf(row_sum<true>(sum, 64, part) * over + a.eps);
#pragma unroll
      for (int i = 0; i < ITEMS; ++i) {
        const int c = threadIdx.x + i * blockDim.x;
        if (c < a.n) store1<DT>(a.out, row * a.n + c, h[i] * (by * a.outer[c]));
      }
    }
  }
}

// Rows of any length and alignment, value by value, read again for each sum: a workgroup a row. 2048 rows of 20001 values in bf16 234 us
// (1.4 TB/s).
template <int DT, int RT>
__global__ void __launch_bounds__(256) norm_any_kernel(NormArgs a) {
  __shared__ float part[16];
  const float over = 1.0f / (float)a.n;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const int64_t token = row / a.heads;
    const int head = (int)(row - token * a.heads);
    int64_t xa, ra, ga;
    at_row(a.xs, token, head, xa);
    at_row(a.rs, token, head, ra);
    at_row(a.gs, token, head, ga);
    float by = 1.0f, sum[1] = {};
    if (a.inner) {
      for (int c = threadIdx.x; c < a.n; c += blockDim.x) {
        const float v = load1<DT>(a.x, xa + c);
        sum[0] += v * v;
      }
      by = rsqrtf(row_sum<true>(sum, 64, part) * over + a.eps);
    }
    const auto hidden = [&](int c) __attribute__((always_inline)) {
      float u = load1<DT>(a.x, xa + c);
      if (a.inner) u *= by * a.inner[c];
      if (a.gate) u *= act_of<RT>(load1<DT>(a.gate, ga + c), a.act);
      return (a.residual ? load1<RT>(a.residual, ra + c) : 0.0f) + a.scale * u;
    };
    sum[0] = 0.0f;
    for (int c = threadIdx.x; c < a.n; c += blockDim.x) {
      const float h = hidden(c);
      sum[0] += h * h;
      store1<RT>(a.hidden, row * a.n + c, h);
    }
    if (a.outer) {
      const float f = rsqrtf(row_sum<true>(sum, 64, part) * over + a.eps);
      for (int c = threadIdx.x; c < a.n; c += blockDim.x) store1<DT>(a.out, row * a.n + c, hidden(c) * (f * a.outer[c]));
    }
  }
}

template <int DT, int RT>
hipError_t launch(const NormArgs& a, bool wide, hipStream_t stream) {
  const int64_t most = 1 << 22;  // workgroups: a grid holds fewer than 2^32 threads
  const int pieces = (a.n + 7) / 8;
  // Read again for each sum instead (norm_any_kernel), in us: 8192 rows of 4097 values in bf16 135 to 108, 4 rows 12.3 to 6.2, 16384 rows
  // of 100 values 23.2 to 8.9; two values a thread up to 1024, eight beyond (sixteen: 115, 6.9).
  if (!wide && a.n <= 8 * 1024) {
    const auto threads = [&](int items) { return 64 * ((a.n + 64 * items - 1) / (64 * items)); };
    const unsigned rows = (unsigned)std::min(a.rows, most / 4);
    if (a.n <= 1024) norm_odd_kernel<DT, RT, 2><<<rows, threads(2), 0, stream>>>(a);
    else norm_odd_kernel<DT, RT, 8><<<rows, threads(8), 0, stream>>>(a);
    return hipGetLastError();
  }
  if (!wide || pieces > 4 * 1024) {
    norm_any_kernel<DT, RT><<<(unsigned)std::min(a.rows, most), 256, 0, stream>>>(a);
    return hipGetLastError();
  }
  if (pieces <= 64) {  // a row is at most one piece of each lane of a wave
    int lanes = 8;
    while (lanes < pieces) lanes *= 2;
    const int64_t blocks = (a.rows * lanes + 255) / 256;
    norm_kernel<DT, RT, 1, false><<<(unsigned)std::min(blocks, most), 256, 0, stream>>>(a, lanes);
    return hipGetLastError();
  }
  const int64_t rows = std::min(a.rows, most / 4);
  const auto threads = [&](int items) { return 64 * ((pieces + 64 * items - 1) / (64 * items)); };
  // Few rows take as many waves as there are, for the latency; of many rows smaller workgroups keep the loads of one under way while
  // another waits for its sum. Four pieces a lane against one or two, in us, with the gate and both norms (with one norm), bf16:
  //   rows of 5120 values:  512: 8.6 : 7.3 (6.5 : 5.5), 1024: 11.3 : 14.1 (8.8 : 9.9), 4096: 36.8 : 41.0 (30.7 : 28.2)
  //   rows of 8192 values:  512: 10.3 : 11.2 (8.0 : 7.9), 1024: 15.9 : 20.7 (12.6 : 15.5), 4096: 50.9 : 71.8 (43.9 : 47.4)
  //   rows of 16384 values: 4: 7.9 : 7.1 (5.5 : 4.8), 1024: 30.3 : 36.5 (23.9 : 27.8), 4096: 123 : 152 (104 : 104)
  // and 4096 rows of 4096 values: 28.7 : 27.3 (24.1 : 22.5).
  if (pieces > 2048 || (pieces > 512 && a.rows >= 1024)) norm_kernel<DT, RT, 4, true><<<(unsigned)rows, threads(4), 0, stream>>>(a, 64);
  else if (pieces <= 1024) norm_kernel<DT, RT, 1, true><<<(unsigned)rows, threads(1), 0, stream>>>(a, 64);
  else norm_kernel<DT, RT, 2, true><<<(unsigned)rows, threads(2), 0, stream>>>(a, 64);
  return hipGetLastError();
}

}  // namespace

// wide: rows are a multiple of 8 long and 16-byte aligned, as are the weights
hipError_t launch_norm(const NormArgs& a, int dtype, int residual_dtype, bool wide, hipStream_t stream) {
  if (residual_dtype == kF32) {
    switch (dtype) {
      case kF32: return launch<kF32, kF32>(a, wide, stream);
      case kF16: return launch<kF16, kF32>(a, wide, stream);
      default: return launch<kBF16, kF32>(a, wide, stream);
    }
  }
  return dtype == kF16 ? launch<kF16, kF16>(a, wide, stream) : launch<kBF16, kBF16>(a, wide, stream);
}

}  // namespace gguf_dec
