// The gated delta rule (include/gguf_decoder.h states the contract). For each v head, with the fp32
// state S [dv, dk], its decay exp(g) and step beta,
//   S <- exp(g) S,   u = beta (v - S k),   S <- S + u k^T,   o = scale S q.
// Sequences of up to kRecurrent tokens take these steps one by one (recurrent_kernel); longer ones
// take chunks of C tokens (prep_kernel, scan_kernel).
#include "delta.h"

namespace gguf_dec {

namespace {

__device__ __forceinline__ float row16_sum(float v) {  // over 16 lanes, in all of them
  v += __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), 0x128, 0xF, 0xF, true));  // row_ror:8
  v += __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), 0x124, 0xF, 0xF, true));
  v += __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), 0x122, 0xF, 0xF, true));
  v += __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), 0x121, 0xF, 0xF, true));
  return v;
}

template <int DT>
__device__ __forceinline__ void load4(const void* p, int64_t i, float (&v)[4]) {
  if constexpr (DT == kF32) {
    const float4 a = *(const float4*)((const float*)p + i);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
  } else {
    const uint2 a = *(const uint2*)((const uint16_t*)p + i);
    const uint32_t w[2] = {a.x, a.y};
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      v[2 * e] = DT == kF16 ? gguf::half_bits_to_float(w[e] & 0xFFFF) : __uint_as_float(w[e] << 16);
      v[2 * e + 1] = DT == kF16 ? gguf::half_bits_to_float(w[e] >> 16) : __uint_as_float(w[e] & 0xFFFF0000u);
    }
  }
}

// One wave holds 4 R rows of a head's state in registers: 16 lanes a row, lane sub with the keys
// 64 c + 4 sub .. + 3. Rows are independent, so nothing leaves the wave. A token's two products with
// the state, S k and S q, are summed over the 16 lanes together: S' q = S q + u (k . q), so the output need
// not wait for the update.
// Bound: HBM, the state in and out (2 x 64 KB a head of 128 x 128); at one sequence latency. Measured, 48 heads of
// 128 x 128: 32 sequences of 4 tokens with every state kept 104 us (508 MB, 4.9 TB/s), one token 8 us.
template <int DT, int DK, int R>
__global__ void __launch_bounds__(256) recurrent_kernel(DeltaArgs a, int most) {
  constexpr int P = DK / 64;
  const int lane = threadIdx.x & 63, sub = lane & 15, rr = lane >> 4;
  const int seq = blockIdx.z, h = blockIdx.y, hk = h / a.rep;
  const int row0 = ((int)blockIdx.x * 4 + (threadIdx.x >> 6)) * 4 * R;
  if (row0 >= a.dv) return;
  int r0, r1;
  rows_of(a.rows, seq, r0, r1);
  if (r1 - r0 > most) return;  // the chunked form's
  const int from = a.slots[seq];
  const int64_t head = (int64_t)a.dv * DK, slot = (int64_t)a.hv * head;
  float s[R][P][4];
  int row[R];
#pragma unroll
  for (int j = 0; j < R; ++j) {
    row[j] = row0 + 4 * j + rr;
    const bool have = from >= 0 && from < a.nslots && row[j] < a.dv;
#pragma unroll
    for (int c = 0; c < P; ++c) {
      if (have) {
        load4<kF32>(a.state, from * slot + h * head + (int64_t)row[j] * DK + 64 * c + 4 * sub, s[j][c]);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) s[j][c][e] = 0.0f;
      }
    }
  }
  const auto put = [&](int to) {
    if (to < 0 || to >= a.nslots) return;
#pragma unroll
    for (int j = 0; j < R; ++j)
      if (row[j] < a.dv)
#pragma unroll
        for (int c = 0; c < P; ++c)
          *(float4*)(a.state + to * slot + h * head + (int64_t)row[j] * DK + 64 * c + 4 * sub) =
              make_float4(s[j][c][0], s[j][c][1], s[j][c][2], s[j][c][3]);
  };

  for (int t = r0; t < r1; ++t) {
    float k[P][4], q[P][4], v[R];
#pragma unroll
    for (int c = 0; c < P; ++c) {
      load4<DT>(a.k, t * a.kt + hk * a.kh + 64 * c + 4 * sub, k[c]);
      load4<DT>(a.q, t * a.qt + hk * a.qh + 64 * c + 4 * sub, q[c]);
    }
#pragma unroll
    for (int j = 0; j < R; ++j) v[j] = load1<DT>(a.v, t * a.vt + h * a.vh + min(row[j], a.dv - 1));
    const float eg = expf(a.g[t * a.gt + h]), beta = a.beta[t * a.bt + h];
    float kk = 0.0f, qq = 0.0f, kq = 0.0f;
#pragma unroll
    for (int c = 0; c < P; ++c)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        kk = fmaf(k[c][e], k[c][e], kk);
        qq = fmaf(q[c][e], q[c][e], qq);
        kq = fmaf(k[c][e], q[c][e], kq);
      }
    kq = row16_sum(kq);
    float rk = 1.0f, rq = a.scale;
    if (a.l2norm) {
      rk = 1.0f / sqrtf(row16_sum(kk) + kNormEps);
      rq = a.scale / sqrtf(row16_sum(qq) + kNormEps);
    }
#pragma unroll
    for (int j = 0; j < R; ++j) {
      float sk = 0.0f, sq = 0.0f;
#pragma unroll
      for (int c = 0; c < P; ++c)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          s[j][c][e] *= eg;
          sk = fmaf(s[j][c][e], k[c][e], sk);
          sq = fmaf(s[j][c][e], q[c][e], sq);
        }
      sk = row16_sum(sk);
      sq = row16_sum(sq);
      const float u = beta * (v[j] - rk * sk) * rk;
      const float o = rq * fmaf(u, kq, sq);
#pragma unroll
      for (int c = 0; c < P; ++c)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[j][c][e] = fmaf(u, k[c][e], s[j][c][e]);
      if (sub == 0 && row[j] < a.dv) store1<DT>(a.out, ((int64_t)t * a.hv + h) * a.dv + row[j], o);
    }
    if (a.steps > 0 && t - r0 < a.steps) put(a.out_slots[(int64_t)seq * a.out_stride + (t - r0)]);
  }
  if (a.steps == 0) put(a.out_slots[(int64_t)seq * a.out_stride]);
}

// ---------------------------------------------------------------------------------------------
// Chunks. With G_i the sum of g up to token i of the chunk (its last: G_c), u_i = beta_i (v_i -
// S_i k_i) for the state before token i's update solves (I + L) U = X,
//   L_ij = beta_i e^{G_i - G_j} k_i.k_j (j < i),   X_i = beta_i (v_i - e^{G_i} S k_i)
// and with T = (I + L)^-1, U = T X,
//   o_i = scale (e^{G_i} S q_i + sum_{j <= i} e^{G_i - G_j} (q_i.k_j) u_j),
//   S  <- e^{G_c} S + sum_j e^{G_c - G_j} u_j k_j^T.
// T and A_ij = scale e^{G_i - G_j} q_i.k_j need no state: prep_kernel makes them for all chunks at
// once. scan_kernel goes through a sequence's chunks, with S in registers.
//
// Precision: products are bf16 MFMAs with fp32 sums. A bf16 key or query is exact (its norm is
// applied to the sums), fp16 and fp32 ones are two and three bf16 planes; fp32 values on
// the way (S, X, U, T) are split into three planes hi + mid + lo, 24 bits, and of the products of planes i and j those
// with i + j <= 2 are kept: what is dropped is below 2^-24. The output's own products (S q and A U)
// keep i + j <= 1, below 2^-16, where the output is rounded to 16 bits. Differences of G are taken in 64 bits: G
// may reach thousands where only differences near 0 matter.

// What a token that is not finite reaches: its own and later tokens, of its columns. The products meet it with the
// zeros of T and A above the diagonal as well, where 0 NaN would reach earlier tokens; so such values are taken as 0 there,
// and the first token of a column to have one is kept, from which on the column is NaN.

// finite, and within bf16's range
__device__ __forceinline__ bool finite(float x) { return fabsf(x) <= 3.38e38f; }

// min over the four lane groups (lanes n, n + 16, n + 32, n + 48)
__device__ __forceinline__ int groups_min(int v) {
  v = min(v, __shfl_xor(v, 16, 64));
  return min(v, __shfl_xor(v, 32, 64));
}

// P planes of 8 fp32 values, two a conversion
template <int P>
__device__ __forceinline__ void split(const float (&x)[8], bf16x8 (&planes)[P]) {
  typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
  float r[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) r[e] = x[e];
#pragma unroll
  for (int p = 0; p < P; ++p) {
    uint32_t w[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const bf16x2 v = {(__bf16)r[2 * e], (__bf16)r[2 * e + 1]};
      w[e] = __builtin_bit_cast(uint32_t, v);
      if (p + 1 < P) {
        r[2 * e] -= __uint_as_float(w[e] << 16);
        r[2 * e + 1] -= __uint_as_float(w[e] & 0xFFFF0000u);
      }
    }
    planes[p] = __builtin_bit_cast(bf16x8, uintx4{w[0], w[1], w[2], w[3]});
  }
}

// an element's bits, their value, and access through a buffer descriptor
template <int DT>
struct Bits {
  typedef uint16_t type;
  static __device__ __forceinline__ float value(uint16_t b) {
    return DT == kF16 ? gguf::half_bits_to_float(b) : __uint_as_float((uint32_t)b << 16);
  }
  static __device__ __forceinline__ uint16_t load(__amdgpu_buffer_rsrc_t r, uint32_t at) {
    return (uint16_t)__builtin_amdgcn_raw_buffer_load_b16(r, at, 0, 0);
  }
  static __device__ __forceinline__ void store(__amdgpu_buffer_rsrc_t r, uint32_t at, float v) {
    const uint16_t b = DT == kF16 ? __builtin_bit_cast(uint16_t, (_Float16)v) : __builtin_bit_cast(uint16_t, (__bf16)v);
    __builtin_amdgcn_raw_buffer_store_b16(b, r, at, 0, 0);
  }
};
template <>
struct Bits<kF32> {
  typedef float type;
  static __device__ __forceinline__ float value(float b) { return b; }
  static __device__ __forceinline__ float load(__amdgpu_buffer_rsrc_t r, uint32_t at) {
    return __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(r, at, 0, 0));
  }
  static __device__ __forceinline__ void store(__amdgpu_buffer_rsrc_t r, uint32_t at, float v) {
    __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(v), r, at, 0, 0);
  }
};

struct Lane8 {
  float x[8];
};

__device__ __forceinline__ Lane8 lane8(floatx4 a, floatx4 b) {
  return Lane8{{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]}};
}

template <int P>
__device__ __forceinline__ void split(const Lane8& x, bf16x8 (&planes)[P]) {
  split(x.x, planes);
}

typedef short short4v __attribute__((ext_vector_type(4)));

__device__ __forceinline__ short4v turned(const __bf16* p) {
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) short4v*)p);
}

__device__ __forceinline__ bf16x8 join(short4v a, short4v b) {
  return __builtin_bit_cast(bf16x8, short8{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]});
}

// P planes of 4 fp32 values
template <int P>
__device__ __forceinline__ void split4(const floatx4& x, uint2 (&planes)[P]) {
  typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
  floatx4 r = x;
#pragma unroll
  for (int p = 0; p < P; ++p) {
    const bf16x2 a = {(__bf16)r[0], (__bf16)r[1]}, b = {(__bf16)r[2], (__bf16)r[3]};
    planes[p] = make_uint2(__builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, b));
    if (p + 1 < P) {
      r[0] -= __uint_as_float(planes[p].x << 16);
      r[1] -= __uint_as_float(planes[p].x & 0xFFFF0000u);
      r[2] -= __uint_as_float(planes[p].y << 16);
      r[3] -= __uint_as_float(planes[p].y & 0xFFFF0000u);
    }
  }
}

// (chunk slot, v head): one workgroup. Measured: 121 us for the 128 chunks x 48 heads of an 8192-token
// prompt; with LDS of their own for T and L, two workgroups a CU, 169.
template <int DT, int DK, int C>
__global__ void __launch_bounds__(256) prep_kernel(DeltaArgs a, int most, ChunkWs ws) {
  typedef Layout<DT, DK, C> Lay;
  constexpr int NK = Lay::NK, CT = C / 16;
  constexpr int KR = Lay::KR;
  extern __shared__ __align__(16) char lds[];
  // [NK][C][KR] keys, then queries; once they are multiplied, T and L [C][C + 4] in their places, so that four
  // workgroups share a CU
  __bf16* kp = (__bf16*)lds;
  __bf16* qp = (__bf16*)(lds + Lay::kPrep);
  float *T = (float*)kp, *L = (float*)qp;
  __shared__ double G[C];
  __shared__ float beta[C], rk[C], rq[C];
  constexpr int LS = C + 4;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, n = lane & 15, g = lane >> 4;
  const int h = blockIdx.y, hk = h / a.rep;

  // the chunk: slot base(s) + c, base(s) = cu[s] / C + s (rows_of's offsets are never negative)
  int seq, r0, r1, c;
  {
    int lo = 0, hi = a.rows.seqs - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) / 2;
      const int b = min(max(a.rows.cu[mid], 0), a.rows.tokens) / C + mid;
      if (b <= (int)blockIdx.x) lo = mid; else hi = mid - 1;
    }
    seq = lo;
    rows_of(a.rows, seq, r0, r1);
    c = (int)blockIdx.x - (r0 / C + seq);
  }
  if (r1 - r0 <= most || c < 0 || c * C >= r1 - r0) return;
  const int t0 = r0 + c * C, nt = min(C, r1 - t0);

  // keys and queries as planes, with their norms: 256 / C threads a row
  constexpr int TR = 256 / C, PER = DK / TR / 8;  // threads a row, 8-value pieces a thread
  {
    const int i = tid / TR, part = tid % TR;
    float kk = 0.0f, qq = 0.0f;
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      float sum = 0.0f;
#pragma unroll
      for (int p = 0; p < PER; ++p) {
        const int at = 8 * (part + TR * p);
        float v[8] = {0, 0, 0, 0, 0, 0, 0, 0};
        if (i < nt) {
          if (x == 0) load8<DT>(a.k, (int64_t)(t0 + i) * a.kt + hk * a.kh + at, v);
          else load8<DT>(a.q, (int64_t)(t0 + i) * a.qt + hk * a.qh + at, v);
        }
        bf16x8 w[NK];
        split(v, w);
#pragma unroll
        for (int e = 0; e < 8; ++e) sum = fmaf(v[e], v[e], sum);
#pragma unroll
        for (int pl = 0; pl < NK; ++pl) *(bf16x8*)((x ? qp : kp) + (pl * C + i) * KR + at) = w[pl];
      }
      (x ? qq : kk) = sum;
    }
#pragma unroll
    for (int off = 1; off < TR; off <<= 1) {
      kk += __shfl_xor(kk, off, 64);
      qq += __shfl_xor(qq, off, 64);
    }
    if (part == 0) {
      rk[i] = a.l2norm ? 1.0f / sqrtf(kk + kNormEps) : 1.0f;
      rq[i] = a.l2norm ? a.scale / sqrtf(qq + kNormEps) : a.scale;
    }
  }
  if (wave == 0) {
    // a decay below e^-1e5 is 0 in fp32; cut there, sums and differences stay finite
    double s = 0.0;
    if (lane < nt) {
      const float gv = a.g[(int64_t)(t0 + lane) * a.gt + h];
      s = gv < -1e5f ? -1e5 : (double)gv;
    }
#pragma unroll
    for (int off = 1; off < C; off <<= 1) {
      const double o = __shfl_up(s, off, 64);
      if (lane >= off) s += o;
    }
    if (lane < C) {
      G[lane] = s;
      beta[lane] = lane < nt ? a.beta[(int64_t)(t0 + lane) * a.bt + h] : 0.0f;
    }
  }
  __syncthreads();

  char* kq = ws.kq + ((int64_t)blockIdx.x * a.hk + hk) * Lay::kKq;
  char* tp = ws.t + ((int64_t)blockIdx.x * a.hv + h) * Lay::kT;
  // factors of a token: beta, of S k in X, of S q in o, of u in S; and the chunk's decay
  if (tid < C) {
    float4 f;
    const float eg = expf((float)G[tid]);
    f.x = beta[tid];
    f.y = beta[tid] * eg * rk[tid];
    f.z = eg * rq[tid];
    f.w = expf((float)(G[C - 1] - G[tid])) * rk[tid];
    ((float4*)(tp + Lay::kFactors))[tid] = f;
    if (tid == 0) ((float4*)(tp + Lay::kFactors))[C] = make_float4(expf((float)G[C - 1]), 0, 0, 0);
  }
  if (h % a.rep == 0) {  // keys and queries, once a k head
    for (int i = tid; i < NK * C * (DK / 8); i += 256) {
      const int row = i / (DK / 8), at = 8 * (i % (DK / 8));
      *(bf16x8*)((__bf16*)(kq + Lay::kK) + row * KR + at) = *(const bf16x8*)(kp + row * KR + at);
      *(bf16x8*)((__bf16*)(kq + Lay::kQ) + row * KR + at) = *(const bf16x8*)(qp + row * KR + at);
    }
  }

  // k k^T and q k^T, 16 rows a wave
  float* Ap = (float*)(tp + Lay::kA);
  const int it = wave;
  floatx4 kk[CT], qk[CT];
#pragma unroll
  for (int jt = 0; jt < CT; ++jt) kk[jt] = qk[jt] = floatx4{0, 0, 0, 0};
  if (it < CT) {
#pragma unroll
    for (int s = 0; s < DK / 32; ++s) {
      bf16x8 ka[NK], qa[NK];
#pragma unroll
      for (int p = 0; p < NK; ++p) {
        ka[p] = *(const bf16x8*)(kp + (p * C + 16 * it + n) * KR + 32 * s + 8 * g);
        qa[p] = *(const bf16x8*)(qp + (p * C + 16 * it + n) * KR + 32 * s + 8 * g);
      }
#pragma unroll
      for (int jt = 0; jt < CT; ++jt) {
        if (jt > it) continue;
#pragma unroll
        for (int p = 0; p < NK; ++p) {
          const bf16x8 b = *(const bf16x8*)(kp + (p * C + 16 * jt + n) * KR + 32 * s + 8 * g);
#pragma unroll
          for (int o = 0; o + p < 3 && o < NK; ++o) {
            kk[jt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ka[o], b, kk[jt], 0, 0, 0);
            qk[jt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(qa[o], b, qk[jt], 0, 0, 0);
          }
        }
      }
    }
  }
  __syncthreads();
  if (it < CT) {
#pragma unroll
    for (int jt = 0; jt < CT; ++jt)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int i = 16 * it + 4 * g + e, j = 16 * jt + n;
        const float w = j <= i ? expf((float)(G[i] - G[j])) * rk[j] : 0.0f;
        L[i * LS + j] = j < i ? beta[i] * rk[i] * w * kk[jt][e] : 0.0f;
        if (j / 32 <= i / 32) Ap[Lay::tri(i, j)] = j <= i ? rq[i] * w * qk[jt][e] : 0.0f;
      }
  }
  __syncthreads();

  // T: the 16 x 16 blocks on the diagonal by forward substitution, a lane a column
  if (tid < C) {
    const int b = 16 * (tid / 16), col = tid % 16;
    float t[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      float v = i == col ? 1.0f : 0.0f;
#pragma unroll
      for (int j = 0; j < i; ++j) v = fmaf(-L[(b + i) * LS + b + j], t[j], v);
      t[i] = v;
      T[(b + i) * LS + b + col] = v;
    }
  }
  __syncthreads();
  // below it, a wave a column of blocks: T_IJ = -T_II sum_{J <= K < I} L_IK T_KJ, in fp32 MFMAs. Sum place g
  // of step s stands for 4 g + s, so that a result is the next product's right operand as it is.
  for (int J = wave; J < CT; J += 4) {
    floatx4 col[CT];
#pragma unroll
    for (int e = 0; e < 4; ++e) col[0][e] = T[(16 * J + 4 * g + e) * LS + 16 * J + n];
    for (int I = 0; I < J; ++I)  // nothing above
#pragma unroll
      for (int e = 0; e < 4; ++e) T[(16 * I + 4 * g + e) * LS + 16 * J + n] = 0.0f;
#pragma unroll
    for (int x = 1; x < CT; ++x) {
      const int I = J + x;
      if (I >= CT) break;
      floatx4 m = {0, 0, 0, 0};
#pragma unroll
      for (int y = 0; y < x; ++y) {
        const floatx4 l = *(const floatx4*)(L + (16 * I + n) * LS + 16 * (J + y) + 4 * g);
#pragma unroll
        for (int s = 0; s < 4; ++s) m = __builtin_amdgcn_mfma_f32_16x16x4f32(l[s], col[y][s], m, 0, 0, 0);
      }
      const floatx4 d = *(const floatx4*)(T + (16 * I + n) * LS + 16 * I + 4 * g);
      // rows before one that is not finite meet it with T_II's zeros, which must not make them NaN
      int first = 16;
#pragma unroll
      for (int e = 3; e >= 0; --e)
        if (!finite(m[e])) {
          first = 4 * g + e;
          m[e] = 0.0f;
        }
      floatx4 r = {0, 0, 0, 0};
#pragma unroll
      for (int s = 0; s < 4; ++s) r = __builtin_amdgcn_mfma_f32_16x16x4f32(-d[s], m[s], r, 0, 0, 0);
      if (__any(first < 16)) {
        first = groups_min(first);
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (4 * g + e >= first) r[e] = __builtin_nanf("");
      }
      col[x] = r;
#pragma unroll
      for (int e = 0; e < 4; ++e) T[(16 * I + 4 * g + e) * LS + 16 * J + n] = r[e];
    }
  }
  __syncthreads();
  float* Tp = (float*)(tp + Lay::kTt);
  for (int i = tid; i < C * C / 4; i += 256) {
    const int row = i / (C / 4), at = 4 * (i % (C / 4));
    if (at / 32 <= row / 32) *(floatx4*)(Tp + Lay::tri(row, at)) = *(const floatx4*)(T + row * LS + at);
  }
}

// A workgroup takes 16 ND columns (values) of a head through the sequence's chunks in turn. Wave (wt, wd) has of
// its 16 columns wd: the wt-th 16 tokens of X, U and the output, and the wt-th part of S's rows (keys).
// The chunk's left operands lie in LDS as prep_kernel left them. S, X and U become right operands: each wave splits
// its own part into planes, and all read them from LDS; three barriers a chunk.
//
// With lane = 16 g + n, a result has column n = value n, and row 4g + e of its tile t stands for place
// 32 (t >> 1) + 8 g + 4 (t & 1) + e of its dimension (keys or tokens): tiles 2s and 2s + 1 hold, in place, the lane's
// 8 consecutive values of step s of a right operand, so planes are written as they are read, 16
// bytes a lane; only the left operands' rows are taken in that order.
//
// Bound: for one sequence of 48 heads (192 workgroups), latency: the chain S k -> X -> U -> S, with the fetch of a chunk's
// 64 KB of operands beside its second half only; by counters the matrix cores of its CUs are busy for 16 % of the time.
// Measured: 493 us for 8192 tokens, 3.9 us a chunk; one wave for 16 columns, without the barriers but with all of a chunk's
// work on one SIMD, took 650.
template <int DT, int DK, int C>
__global__ void __launch_bounds__((64 * Layout<DT, DK, C>::WAVES), 1) scan_kernel(DeltaArgs a, int most, ChunkWs ws) {
  typedef Layout<DT, DK, C> Lay;
  constexpr int NK = Lay::NK, NA = Lay::NA, KR = Lay::KR, WAVES = Lay::WAVES;
  constexpr int TT = C / 16, TS = C / 32, KT = DK / 16, KS = DK / 32, KW = KT / TT;
  constexpr int MAXO = DT == kF32 ? 2 : 1;  // highest plane sum kept for the output
  extern __shared__ __align__(16) char lds[];
  __shared__ int dead[Lay::ND][16];  // of each column: its first token that is not finite (in later chunks 0: S is NaN)
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), n = lane & 15, g = lane >> 4;
  const int wt = wave % TT, wd = wave / TT;
  const int seq = blockIdx.z, h = blockIdx.x, hk = h / a.rep;
  int r0, r1;
  rows_of(a.rows, seq, r0, r1);
  if (r1 - r0 <= most) return;
  const int dv = ((int)blockIdx.y * Lay::ND + wd) * 16 + n;  // dv % 16 == 0: a wave is in or out as one
  const bool in = dv < a.dv;
  const int from = a.slots[seq];
  const int64_t head = (int64_t)a.dv * DK, slot = (int64_t)a.hv * head;
  const int64_t at = h * head + (int64_t)dv * DK + 8 * g;
  const auto key = [&](int t) { return 32 * ((wt * KW + t) >> 1) + 4 * ((wt * KW + t) & 1); };  // of the wave's tile t, less 8 g
  floatx4 S[KW];
#pragma unroll
  for (int t = 0; t < KW; ++t)
    S[t] = in && from >= 0 && from < a.nslots ? *(const floatx4*)(a.state + from * slot + at + key(t)) : floatx4{0, 0, 0, 0};
  const int chunks = (r1 - r0 + C - 1) / C, base = r0 / C + seq;
  const int rown = 8 * (n >> 2) + (n & 3);  // row n of an even tile of a left operand
  const int tok0 = 32 * (wt >> 1) + 4 * (wt & 1);  // the wave's tokens are tok0 + 8 g + e

  // v and out through buffer descriptors over the chunk's rows: a lane without a token (or column) reads 0 and its
  // stores are dropped, without branches, across which the compiler would wait for every load and store in flight
  constexpr uint32_t ES = DT == kF32 ? 4 : 2, kNowhere = 0x7FFFFF00u;
  const uint32_t vt = (uint32_t)a.vt * ES, ot = (uint32_t)(a.hv * a.dv) * ES;
  const auto place = [&](int e, int nt, uint32_t stride) __attribute__((always_inline)) {
    const int i = tok0 + 8 * g + e;
    return in && i < nt ? (uint32_t)i * stride + (uint32_t)dv * ES : kNowhere;
  };
  // The next chunk's operands go to LDS, and its v to registers, during this one's last products: by then
  // this one's are in registers.
  typename Bits<DT>::type vnext[4];  // as they are: converting them here would wait for them here
  const auto fetch = [&](int c) __attribute__((always_inline)) {
    const char* kq = ws.kq + ((int64_t)(base + c) * a.hk + hk) * Lay::kKq;
    const char* tp = ws.t + ((int64_t)(base + c) * a.hv + h) * Lay::kT - Lay::kKq;
#pragma unroll
    for (int i = 0; i < (Lay::kKq + Lay::kT) / Lay::kPart; ++i) {
      const int o = (WAVES * i + wave) * 1024;
      __builtin_amdgcn_global_load_lds((const void*)((o < Lay::kKq ? kq : tp) + o + 16 * lane),
                                       (__attribute__((address_space(3))) void*)(lds + o), 16, 0, 0);
    }
    const int nt = min(C, r1 - r0 - c * C);
    const __amdgpu_buffer_rsrc_t rs = gguf::buffer_rsrc((const char*)a.v + ((int64_t)(r0 + c * C) * a.vt + h * a.vh) * ES, (C - 1) * vt + a.dv * ES);
#pragma unroll
    for (int e = 0; e < 4; ++e) vnext[e] = Bits<DT>::load(rs, place(e, nt, vt));
  };
  const __bf16* K = (const __bf16*)(lds + Lay::kK);
  const __bf16* Q = (const __bf16*)(lds + Lay::kQ);
  const float* Tm = (const float*)(lds + Lay::kKq + Lay::kTt);
  const float* Am = (const float*)(lds + Lay::kKq + Lay::kA);
  const float4* F = (const float4*)(lds + Lay::kKq + Lay::kFactors);
  // plane p, step s of the wave's columns
  char* const sl = lds + Lay::kS + wd * 3 * KS * 1024 + 16 * lane;
  char* const xl = lds + Lay::kX + wd * 3 * TS * 1024 + 16 * lane;
  char* const ul = lds + Lay::kU + wd * Lay::NU * TS * 1024 + 16 * lane;

  if (tid < 16 * Lay::ND) dead[tid / 16][n] = C;
  fetch(0);
  __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0)

  for (int c = 0; c < chunks; ++c) {
    const int nt = min(C, r1 - r0 - c * C);  // tokens of the chunk
    float v[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = Bits<DT>::value(vnext[e]);
#pragma unroll
    for (int t = 0; t < KW; ++t) {
      uint2 w[3];
      split4(S[t], w);
#pragma unroll
      for (int p = 0; p < 3; ++p) *(uint2*)(sl + (p * KS + (wt * KW + t) / 2) * 1024 + 8 * ((wt * KW + t) & 1)) = w[p];
    }
    __syncthreads();

    // S k and S q
    floatx4 X[3] = {}, O[2] = {};  // sums of their own: MFMAs that follow each other do not wait for each other
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      bf16x8 sp[3];
#pragma unroll
      for (int p = 0; p < 3; ++p) sp[p] = *(const bf16x8*)(sl + (p * KS + s) * 1024);
#pragma unroll
      for (int p = 0; p < NK; ++p) {
        const bf16x8 k = *(const bf16x8*)(K + (p * C + tok0 + rown) * KR + 32 * s + 8 * g);
        const bf16x8 q = *(const bf16x8*)(Q + (p * C + tok0 + rown) * KR + 32 * s + 8 * g);
#pragma unroll
        for (int o = 0; o + p <= 2; ++o) {
          X[o] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k, sp[o], X[o], 0, 0, 0);
          if (o + p <= MAXO) O[o & 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(q, sp[o], O[o & 1], 0, 0, 0);
        }
      }
    }
    // X
    floatx4 x, f2;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float4 f = F[tok0 + 8 * g + e];
      x[e] = f.x * v[e] - f.y * (X[0][e] + (X[1][e] + X[2][e]));
      O[0][e] = (O[0][e] + O[1][e]) * f.z;
      O[1][e] = 0.0f;
      f2[e] = f.w;
    }
    const float dec = F[C].x;
    int first = C;  // the lane's first token whose u is not finite
    const auto clean = [&](floatx4& y) __attribute__((always_inline)) {
      // where a branch costs less than the selects (8192 bf16 tokens, 48 heads: 605 us against 618; 2048 of fp16 263, 249)
      if (DT == kBF16 && !__any(!finite(fabsf(y[0]) + fabsf(y[1]) + fabsf(y[2]) + fabsf(y[3])))) return;
#pragma unroll
      for (int e = 3; e >= 0; --e)
        if (!finite(y[e])) {
          first = min(first, tok0 + 8 * g + e);
          y[e] = 0.0f;
        }
    };
    // K^T's rows are keys: the transposing read gives a lane 4 tokens of its key, from the 4 rows that its group of 16
    // lanes addresses (lane 4 r + c: 4 keys of row r)
    bf16x8 tm[TS][3], am[TS][NA], km[NK][TS][KW];
#pragma unroll
    for (int s = 0; s < TS; ++s) {
      if (s <= wt / 2) {
        const int o = Lay::tri(tok0 + rown, 32 * s + 8 * g);
        split(lane8(*(const floatx4*)(Tm + o), *(const floatx4*)(Tm + o + 4)), tm[s]);
        split(lane8(*(const floatx4*)(Am + o), *(const floatx4*)(Am + o + 4)), am[s]);
      }
#pragma unroll
      for (int p = 0; p < NK; ++p)
#pragma unroll
        for (int t = 0; t < KW; ++t) {
          const __bf16* k = K + (p * C + 32 * s + 8 * g + (n >> 2)) * KR + key(t) + 8 * (n & 3);
          km[p][s][t] = join(turned(k), turned(k + 4 * KR));
        }
    }
    clean(x);
    {
      uint2 w[3];
      split4(x, w);
#pragma unroll
      for (int p = 0; p < 3; ++p) *(uint2*)(xl + (p * TS + wt / 2) * 1024 + 8 * (wt & 1)) = w[p];
    }
    __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0): the chunk's operands are here
    __syncthreads();
    fetch(min(c + 1, chunks - 1));  // taken within this turn, so that its wait does not take in the stores

    // U = T X; T is 0 above its diagonal
    floatx4 U[3] = {};
#pragma unroll
    for (int s = 0; s < TS; ++s) {
      if (s > wt / 2) break;
      bf16x8 xp[3];
#pragma unroll
      for (int p = 0; p < 3; ++p) xp[p] = *(const bf16x8*)(xl + (p * TS + s) * 1024);
#pragma unroll
      for (int p = 0; p < 3; ++p)
#pragma unroll
        for (int o = 0; o + p <= 2; ++o) U[o] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(tm[s][p], xp[o], U[o], 0, 0, 0);
    }
    floatx4 u = U[0] + (U[1] + U[2]);
    clean(u);
    if (DT != kBF16 || __any(first < C)) atomicMin(&dead[wd][n], first);
    {
      uint2 w[3], o[MAXO + 1];
      split4(u * f2, w);
      split4(u, o);
#pragma unroll
      for (int p = 0; p < 3; ++p) *(uint2*)(ul + (p * TS + wt / 2) * 1024 + 8 * (wt & 1)) = w[p];
#pragma unroll
      for (int p = 0; p <= MAXO; ++p) *(uint2*)(ul + ((3 + p) * TS + wt / 2) * 1024 + 8 * (wt & 1)) = o[p];
    }
    __syncthreads();

    // S = e^{G_c} S + K^T (e^{G_c - G} U);   O += A U
    first = dead[wd][n];
#pragma unroll
    for (int t = 0; t < KW; ++t) S[t] *= first < C ? __builtin_nanf("") : dec;
#pragma unroll
    for (int s = 0; s < TS; ++s) {
      bf16x8 wp[3], up[MAXO + 1];
#pragma unroll
      for (int p = 0; p < 3; ++p) wp[p] = *(const bf16x8*)(ul + (p * TS + s) * 1024);
#pragma unroll
      for (int p = 0; p <= MAXO; ++p) up[p] = *(const bf16x8*)(ul + ((3 + p) * TS + s) * 1024);
#pragma unroll
      for (int p = 0; p < NK; ++p)
#pragma unroll
        for (int o = 0; o + p <= 2; ++o)
#pragma unroll
          for (int t = 0; t < KW; ++t) S[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(km[p][s][t], wp[o], S[t], 0, 0, 0);
      if (s > wt / 2) continue;  // A is 0 above its diagonal
#pragma unroll
      for (int p = 0; p < NA; ++p)
#pragma unroll
        for (int o = 0; o + p <= MAXO; ++o)
          O[(o + p) & 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(am[s][p], up[o], O[(o + p) & 1], 0, 0, 0);
    }
    const __amdgpu_buffer_rsrc_t rs = gguf::buffer_rsrc((char*)a.out + (int64_t)(r0 + c * C) * ot + (int64_t)h * a.dv * ES, (C - 1) * ot + a.dv * ES);
#pragma unroll
    for (int e = 0; e < 4; ++e)
      Bits<DT>::store(rs, place(e, nt, ot), tok0 + 8 * g + e >= first ? __builtin_nanf("") : O[0][e] + O[1][e]);
    __builtin_amdgcn_s_waitcnt(0x0F74);  // vmcnt(4): all but these stores
  }
  const int to = a.out_slots[(int64_t)seq * a.out_stride];
  if (in && to >= 0 && to < a.nslots)
#pragma unroll
    for (int t = 0; t < KW; ++t) *(floatx4*)(a.state + to * slot + at + key(t)) = S[t];
}

template <int DT, int DK>
hipError_t launch(const DeltaArgs& a, int64_t max_new, void* wsp, hipStream_t stream) {
  const bool chunked = wsp != nullptr;
  const int most = chunked ? kRecurrent : 0x7FFFFFFF;
  constexpr int R = 4;
  recurrent_kernel<DT, DK, R><<<dim3((a.dv + 16 * R - 1) / (16 * R), a.hv, a.rows.seqs), 256, 0, stream>>>(a, most);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || !chunked) return e;
  constexpr int C = Chunk<DT>::C;
  typedef Layout<DT, DK, C> Lay;
  const int64_t slots = a.rows.tokens / C + a.rows.seqs;
  ChunkWs ws{(char*)wsp, (char*)wsp + slots * a.hk * Lay::kKq};
  constexpr int prep_lds = 2 * Lay::kPrep, scan_lds = Lay::kLds;
  int dev = 0;
  if ((e = hipGetDevice(&dev)) != hipSuccess) return e;
  struct Tag {};
  gguf::once_per_device<Tag>(dev, [&] {
    (void)hipFuncSetAttribute((const void*)prep_kernel<DT, DK, C>, hipFuncAttributeMaxDynamicSharedMemorySize, prep_lds);
    (void)hipFuncSetAttribute((const void*)scan_kernel<DT, DK, C>, hipFuncAttributeMaxDynamicSharedMemorySize, scan_lds);
  });
  prep_kernel<DT, DK, C><<<dim3((unsigned)slots, a.hv), 256, prep_lds, stream>>>(a, most, ws);
  if ((e = hipGetLastError()) != hipSuccess) return e;
  // heads first: workgroups of one head, which share its operands, then run on one XCD where heads are a multiple of 8
  scan_kernel<DT, DK, C><<<dim3(a.hv, (a.dv + 16 * Lay::ND - 1) / (16 * Lay::ND), a.rows.seqs), 64 * Lay::WAVES, scan_lds, stream>>>(a, most, ws);
  return hipGetLastError();
}

template <int DT>
size_t ws_bytes(int dk, int hk, int hv, int64_t tokens, int64_t seqs) {
  constexpr int C = Chunk<DT>::C;
  const int64_t slots = tokens / C + seqs;
  const size_t kq = dk == 64 ? Layout<DT, 64, C>::kKq : Layout<DT, 128, C>::kKq;
  const size_t t = dk == 64 ? Layout<DT, 64, C>::kT : Layout<DT, 128, C>::kT;
  return slots * (hk * kq + hv * t);
}

}  // namespace

size_t delta_workspace(int dtype, int dk, int hk, int hv, int64_t tokens, int64_t seqs, int64_t max_new, bool steps) {
  if (steps || max_new <= kRecurrent) return 0;
  return dtype == kF32   ? ws_bytes<kF32>(dk, hk, hv, tokens, seqs)
         : dtype == kF16 ? ws_bytes<kF16>(dk, hk, hv, tokens, seqs)
                         : ws_bytes<kBF16>(dk, hk, hv, tokens, seqs);
}

// ws: of delta_workspace's bytes, or null: every sequence in the recurrent form
hipError_t launch_delta(const DeltaArgs& a, int dtype, int dk, int64_t max_new, void* ws, hipStream_t stream) {
#define GGUF_DEC_DELTA(DT) return dk == 64 ? launch<DT, 64>(a, max_new, ws, stream) : launch<DT, 128>(a, max_new, ws, stream)
  switch (dtype) {
    case kF32: GGUF_DEC_DELTA(kF32);
    case kF16: GGUF_DEC_DELTA(kF16);
    default: GGUF_DEC_DELTA(kBF16);
  }
#undef GGUF_DEC_DELTA
}

}  // namespace gguf_dec
