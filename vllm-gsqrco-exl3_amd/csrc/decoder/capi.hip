// C ABI of libgguf_decoder.so (include/gguf_decoder.h): checks and dispatch. Host code only.
#include <hip/hip_runtime.h>

#include <climits>
#include <cmath>
#include <cstdarg>
#include <cstdio>

#include "../../../include/gguf_decoder.h"
#include "delta.h"
#include "norm.h"
#include "rotary.h"

namespace gguf_dec {
hipError_t launch_kv8_append(const Kv8& c, int dtype, const void* key, int64_t kt, int64_t kh, const void* value,
                             int64_t vt, int64_t vh, const int32_t* lens, const Ragged& rows, int64_t max_new,
                             hipStream_t stream);
hipError_t launch_kv8_read(const Kv8& c, int dtype, const int32_t* starts, const Ragged& rows, int64_t max_tokens,
                           void* kout, void* vout, hipStream_t stream);
size_t kv8_attention_workspace(int d, int heads, int hq, int64_t tokens, int64_t seqs, int64_t max_new,
                               int64_t max_len, bool tree);
hipError_t launch_kv8_attention(const Kv8& c, int dtype, const void* q, int64_t qt, int64_t qh, int hq,
                                const int32_t* lens, const Ragged& rows, int64_t max_new, int64_t max_len, float scale,
                                const int64_t* mask, int64_t mask_stride, int words, void* out, void* ws, size_t ws_bytes,
                                hipStream_t stream);
hipError_t launch_kv8_rotary(const RotaryArgs& a, int dtype, int64_t max_new, hipStream_t stream);
hipError_t launch_kv8_keep(const Kv8& c, const int32_t* path, int64_t path_stride, int m, const int32_t* lens,
                           const Ragged& rows, hipStream_t stream);
hipError_t launch_norm(const NormArgs& a, int dtype, int residual_dtype, bool wide, hipStream_t stream);
size_t delta_workspace(int dtype, int dk, int hk, int hv, int64_t tokens, int64_t seqs, int64_t max_new, bool steps);
hipError_t launch_delta(const DeltaArgs& a, int dtype, int dk, int64_t max_new, void* ws, hipStream_t stream);
int64_t logprobs_most_vocab(int64_t top);
size_t logprobs_workspace(int64_t rows, int64_t vocab, int64_t top);
hipError_t launch_logprobs(const void* x, int dtype, int64_t stride, int64_t rows, int64_t vocab, const int64_t* ids,
                           int64_t id_stride, int top, float* logprobs, int32_t* ranks, float* entropy,
                           float* top_logprobs, int32_t* top_ids, void* ws, hipStream_t stream);
}  // namespace gguf_dec

namespace {

using gguf_dec::Kv8;
using gguf_dec::Ragged;

thread_local char g_err[512];  // no allocation, so no exception at the C boundary

int fail(const char* fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(g_err, sizeof(g_err), fmt, ap);
  va_end(ap);
  return GGUF_DEC_EINVAL;
}

int hip_fail(hipError_t e, const char* op) {
  snprintf(g_err, sizeof(g_err), "%s: HIP error: %s", op, hipGetErrorString(e));
  return GGUF_DEC_EHIP;
}

int begin() {
  g_err[0] = 0;
  return GGUF_DEC_OK;
}

bool is_float(int dt) { return dt == GGUF_DEC_F32 || dt == GGUF_DEC_F16 || dt == GGUF_DEC_BF16; }
bool is_half(int dt) { return dt == GGUF_DEC_F16 || dt == GGUF_DEC_BF16; }
int64_t size_of(int dt) {
  return dt == GGUF_DEC_I64 ? 8 : dt == GGUF_DEC_F32 || dt == GGUF_DEC_I32 ? 4 : is_half(dt) ? 2 : 1;
}

bool aligned(const gguf_tensor* t, int64_t bytes) { return reinterpret_cast<uintptr_t>(t->data) % bytes == 0; }

int64_t numel(const gguf_tensor* t) {
  int64_t n = 1;
  for (int i = 0; i < t->ndim; ++i) n *= t->size[i];
  return n;
}

bool contiguous(const gguf_tensor* t) {
  if (numel(t) == 0) return true;
  int64_t want = 1;
  for (int i = t->ndim - 1; i >= 0; --i) {
    if (t->size[i] != 1 && t->stride[i] != want) return false;
    want *= t->size[i];
  }
  return true;
}

// stride of dimension i, or what a contiguous tensor would have where it has one element there
int64_t stride_of(const gguf_tensor* t, int i) {
  if (t->size[i] != 1) return t->stride[i];
  int64_t n = 1;
  for (int j = i + 1; j < t->ndim; ++j) n *= t->size[j];
  return n;
}

bool shaped(const gguf_tensor* t, int ndim) {
  if (!t || t->ndim != ndim) return false;
  for (int i = 0; i < ndim; ++i)
    if (t->size[i] < 0 || t->size[i] > INT_MAX || t->stride[i] < 0 || (t->ndim == 3 && i < 2 && t->size[i] > 1 && t->stride[i] > INT_MAX)) return false;
  return true;
}

// [tokens, heads, d] rows that kernels read 16 bytes at a time
bool rows_ok(const gguf_tensor* t) {
  const int64_t es = size_of(t->dtype);
  return (t->size[2] == 1 || t->stride[2] == 1) && aligned(t, 16) && stride_of(t, 0) * es % 16 == 0 &&
         stride_of(t, 1) * es % 16 == 0;
}

// a hint as the launch takes it: at least 1 and at most what there can be, so that no arithmetic on it overflows
int64_t bounded(int64_t hint, int64_t most) { return hint > most ? (most < 1 ? 1 : most) : hint < 1 ? 1 : hint; }

struct DeviceScope {
  int prev = -1;
  hipError_t err = hipSuccess;
  explicit DeviceScope(int device) {
    int cur = -1;
    err = hipGetDevice(&cur);
    if (err == hipSuccess && cur != device) {
      err = hipSetDevice(device);
      if (err == hipSuccess) prev = cur;
    }
  }
  ~DeviceScope() {
    if (prev >= 0) (void)hipSetDevice(prev);
  }
};

template <class... T>
bool same_device(int dev, const T*... t) {
  bool same = true;
  ((same = same && (!t || t->device == dev)), ...);
  return same;
}

// tensors that have elements have memory
template <class... T>
bool present(const T*... t) {
  bool all = true;
  ((all = all && (!t || t->data || numel(t) == 0)), ...);
  return all;
}

// cu_seqlens: int32 [seqs + 1], contiguous
int check_cu(const char* op, const gguf_tensor* cu, int64_t tokens, Ragged* out) {
  if (!shaped(cu, 1) || cu->dtype != GGUF_DEC_I32 || !contiguous(cu)) return fail("%s: cu_seqlens must be a contiguous 1-D int32 tensor", op);
  if (cu->size[0] < 2 || cu->size[0] > 65536) return fail("%s: cu_seqlens must hold 1 to 65535 sequences and one offset more", op);
  *out = Ragged{(const int32_t*)cu->data, (int)(cu->size[0] - 1), (int)tokens};
  return 0;
}

int check_seq_ints(const char* op, const char* name, const gguf_tensor* t, int seqs) {
  if (!shaped(t, 1) || t->dtype != GGUF_DEC_I32 || !contiguous(t) || t->size[0] != seqs)
    return fail("%s: %s must be a contiguous int32 tensor of %d sequences", op, name, seqs);
  return 0;
}

int check_cache(const char* op, const gguf_kv8_cache* c, const gguf_tensor* table, int seqs, Kv8* out) {
  if (!c || !shaped(&c->k, 4) || !shaped(&c->v, 4) || !shaped(&c->k_scale, 2) || !shaped(&c->v_scale, 2))
    return fail("%s: the cache has k and v of 4 dimensions, k_scale and v_scale of 2", op);
  if (c->k.dtype != GGUF_DEC_I8 || c->v.dtype != GGUF_DEC_I8) return fail("%s: k and v of the cache must be int8", op);
  if (c->k_scale.dtype != GGUF_DEC_F32 || c->v_scale.dtype != GGUF_DEC_F32) return fail("%s: k_scale and v_scale must be fp32", op);
  const int64_t p = c->k.size[0], h = c->k.size[1], page = c->k.size[2], d = c->k.size[3];
  if (p < 1 || h < 1 || page < 16 || page % 16) return fail("%s: the cache needs pages, heads and pages of a multiple of 16 tokens, got [%lld, %lld, %lld, ...]", op, (long long)p, (long long)h, (long long)page);
  if (d != 64 && d != 128 && d != 192 && d != 256) return fail("%s: head size %lld is not 64, 128, 192 or 256", op, (long long)d);
  if (p * h > INT_MAX || h > 16384 || page * d > (1 << 28)) return fail("%s: cache of too many heads or too large pages", op);
  if (c->v.size[0] != p || c->v.size[1] != h || c->v.size[2] != d || c->v.size[3] != page)
    return fail("%s: v of the cache must be [pages, heads, head size, page]", op);
  if (c->k_scale.size[0] != p || c->k_scale.size[1] != h || c->v_scale.size[0] != p || c->v_scale.size[1] != h)
    return fail("%s: k_scale and v_scale must be [pages, heads]", op);
  if (!contiguous(&c->k) || !contiguous(&c->v) || !contiguous(&c->k_scale) || !contiguous(&c->v_scale))
    return fail("%s: the cache must be contiguous", op);
  if (!aligned(&c->k, 16) || !aligned(&c->v, 16) || !aligned(&c->k_scale, 4) || !aligned(&c->v_scale, 4))
    return fail("%s: the cache must be 16-byte aligned", op);
  if (!shaped(table, 2) || table->dtype != GGUF_DEC_I32 || table->size[0] != seqs || (table->size[1] > 1 && table->stride[1] != 1))
    return fail("%s: block_table must be int32 [sequences, pages] with unit inner stride", op);
  if (table->size[1] < 1) return fail("%s: block_table has no pages", op);
  if (table->size[1] * page > INT_MAX - 1024) return fail("%s: block_table of too many pages", op);
  if (!same_device(c->k.device, &c->v, &c->k_scale, &c->v_scale, table)) return fail("%s: tensors on different devices", op);
  if (!present(&c->k, &c->v, &c->k_scale, &c->v_scale, table)) return fail("%s: a tensor has no data", op);
  *out = Kv8{(int8_t*)c->k.data, (int8_t*)c->v.data, (float*)c->k_scale.data, (float*)c->v_scale.data,
             (const int32_t*)table->data, stride_of(table, 0), (int)p, (int)h, (int)page, (int)d, (int)table->size[1]};
  return 0;
}

}  // namespace

extern "C" {

const char* gguf_decoder_last_error(void) { return g_err; }

int gguf_kv8_append(const gguf_kv8_cache* cache, const gguf_tensor* key, const gguf_tensor* value,
                    const gguf_tensor* block_table, const gguf_tensor* seq_lens, const gguf_tensor* cu_seqlens,
                    int64_t max_new, void* stream) {
  begin();
  const char* op = "kv8_append";
  if (!shaped(key, 3) || !shaped(value, 3)) return fail("%s: key and value must be [tokens, heads, head size]", op);
  if (!is_float(key->dtype) || value->dtype != key->dtype) return fail("%s: key and value must share one float dtype", op);
  Ragged rows;
  Kv8 c;
  if (check_cu(op, cu_seqlens, key->size[0], &rows) || check_cache(op, cache, block_table, rows.seqs, &c) ||
      check_seq_ints(op, "seq_lens", seq_lens, rows.seqs))
    return GGUF_DEC_EINVAL;
  for (const gguf_tensor* t : {key, value})
    if (t->size[0] != key->size[0] || t->size[1] != c.heads || t->size[2] != c.d)
      return fail("%s: key and value must be [tokens, %d, %d] for this cache", op, c.heads, c.d);
  if (key->size[0] > 0 && (!rows_ok(key) || !rows_ok(value)))
    return fail("%s: key and value need unit inner stride and 16-byte aligned rows", op);
  if (max_new < 0) return fail("%s: max_new must not be negative", op);
  if (!same_device(key->device, value, &cache->k, seq_lens, cu_seqlens)) return fail("%s: tensors on different devices", op);
  if (!present(key, value, seq_lens, cu_seqlens)) return fail("%s: a tensor has no data", op);
  if (key->device < 0) return fail("%s: tensors must be CUDA tensors", op);
  if (key->size[0] == 0) return GGUF_DEC_OK;
  const DeviceScope scope(key->device);
  if (scope.err != hipSuccess) return hip_fail(scope.err, op);
  const hipError_t e = gguf_dec::launch_kv8_append(c, key->dtype, key->data, stride_of(key, 0), stride_of(key, 1), value->data,
                                                   stride_of(value, 0), stride_of(value, 1), (const int32_t*)seq_lens->data, rows,
                                                   bounded(max_new, key->size[0]), (hipStream_t)stream);
  return e == hipSuccess ? GGUF_DEC_OK : hip_fail(e, op);
}

int gguf_kv8_read(const gguf_kv8_cache* cache, const gguf_tensor* block_table, const gguf_tensor* starts,
                  const gguf_tensor* cu_seqlens, int64_t max_tokens, const gguf_tensor* k_out, const gguf_tensor* v_out,
                  void* stream) {
  begin();
  const char* op = "kv8_read";
  if (!shaped(k_out, 3) || !shaped(v_out, 3)) return fail("%s: outputs must be [tokens, heads, head size]", op);
  if (!is_float(k_out->dtype) || v_out->dtype != k_out->dtype) return fail("%s: outputs must share one float dtype", op);
  Ragged rows;
  Kv8 c;
  if (check_cu(op, cu_seqlens, k_out->size[0], &rows) || check_cache(op, cache, block_table, rows.seqs, &c) ||
      check_seq_ints(op, "starts", starts, rows.seqs))
    return GGUF_DEC_EINVAL;
  for (const gguf_tensor* t : {k_out, v_out})
    if (t->size[0] != k_out->size[0] || t->size[1] != c.heads || t->size[2] != c.d || !contiguous(t) || (t->size[0] > 0 && !aligned(t, 16)))
      return fail("%s: outputs must be contiguous, 16-byte aligned [tokens, %d, %d] for this cache", op, c.heads, c.d);
  if (max_tokens < 0) return fail("%s: max_tokens must not be negative", op);
  if (!same_device(k_out->device, v_out, &cache->k, starts, cu_seqlens)) return fail("%s: tensors on different devices", op);
  if (!present(k_out, v_out, starts, cu_seqlens)) return fail("%s: a tensor has no data", op);
  if (k_out->device < 0) return fail("%s: tensors must be CUDA tensors", op);
  if (k_out->size[0] == 0) return GGUF_DEC_OK;
  const DeviceScope scope(k_out->device);
  if (scope.err != hipSuccess) return hip_fail(scope.err, op);
  const hipError_t e = gguf_dec::launch_kv8_read(c, k_out->dtype, (const int32_t*)starts->data, rows, bounded(max_tokens, k_out->size[0]),
                                                 k_out->data, v_out->data, (hipStream_t)stream);
  return e == hipSuccess ? GGUF_DEC_OK : hip_fail(e, op);
}

static size_t attention_workspace(const gguf_kv8_cache* cache, const gguf_tensor* query, int64_t seqs, int64_t max_new,
                                  int64_t max_len, bool tree) {
  if (!cache || cache->k.ndim != 4 || !query || query->ndim != 3 || seqs < 1 || cache->k.size[1] < 1 || query->size[0] < 1 ||
      query->size[1] % cache->k.size[1] || query->size[1] < 1)
    return 0;
  const DeviceScope scope(query->device < 0 ? 0 : query->device);
  return gguf_dec::kv8_attention_workspace((int)cache->k.size[3], (int)cache->k.size[1], (int)query->size[1],
                                           query->size[0], seqs, bounded(max_new, query->size[0]), bounded(max_len, INT_MAX), tree);
}

size_t gguf_kv8_attention_workspace_bytes(const gguf_kv8_cache* cache, const gguf_tensor* query, int64_t seqs,
                                          int64_t max_new, int64_t max_len) {
  return attention_workspace(cache, query, seqs, max_new, max_len, false);
}

size_t gguf_kv8_tree_attention_workspace_bytes(const gguf_kv8_cache* cache, const gguf_tensor* query, int64_t seqs,
                                               int64_t max_new, int64_t max_len) {
  return attention_workspace(cache, query, seqs, max_new, max_len, true);
}

// kv8_attention, or with a mask kv8_tree_attention
static int attention(const char* op, const gguf_tensor* query, const gguf_kv8_cache* cache, const gguf_tensor* mask, bool tree,
                     const gguf_tensor* block_table, const gguf_tensor* seq_lens, const gguf_tensor* cu_seqlens, int64_t max_new,
                     int64_t max_len, float scale, const gguf_tensor* out, void* workspace, size_t workspace_bytes,
                     void* stream) {
  begin();
  if (!shaped(query, 3) || !shaped(out, 3)) return fail("%s: query and out must be [tokens, heads, head size]", op);
  if (!is_half(query->dtype)) return fail("%s: query must be fp16 or bf16", op);
  Ragged rows;
  Kv8 c;
  if (check_cu(op, cu_seqlens, query->size[0], &rows) || check_cache(op, cache, block_table, rows.seqs, &c) ||
      check_seq_ints(op, "seq_lens", seq_lens, rows.seqs))
    return GGUF_DEC_EINVAL;
  if (query->size[2] != c.d) return fail("%s: query has head size %lld, the cache %d", op, (long long)query->size[2], c.d);
  if (query->size[1] < 1 || query->size[1] % c.heads) return fail("%s: %lld query heads are no multiple of the cache's %d", op, (long long)query->size[1], c.heads);
  if ((int64_t)rows.seqs * c.heads >= (1 << 24))  // a grid holds fewer than 2^32 threads, 256 each
    return fail("%s: sequences times heads must be below 2^24", op);
  if (query->size[0] > 0 && !rows_ok(query)) return fail("%s: query needs unit inner stride and 16-byte aligned rows", op);
  if (tree && (!shaped(mask, 2) || mask->dtype != GGUF_DEC_I64 || mask->size[0] != query->size[0] || mask->size[1] < 1 ||
               mask->size[1] > (1 << 24) || (mask->size[1] > 1 && mask->stride[1] != 1)))
    return fail("%s: tree_mask must be int64 [tokens, words] with unit inner stride", op);
  if (tree && !aligned(mask, 8)) return fail("%s: tree_mask must be 8-byte aligned", op);
  if (out->dtype != query->dtype || out->size[0] != query->size[0] || out->size[1] != query->size[1] || out->size[2] != query->size[2] ||
      !contiguous(out) || (out->size[0] > 0 && !aligned(out, 16)))
    return fail("%s: out must be contiguous, 16-byte aligned, with query's shape and dtype", op);
  if (max_new < 0 || max_len < 0) return fail("%s: max_new and max_len must not be negative", op);
  if (!std::isfinite(scale)) return fail("%s: scale must be finite", op);
  if (reinterpret_cast<uintptr_t>(workspace) % 16) return fail("%s: workspace must be 16-byte aligned", op);
  if (!same_device(query->device, out, &cache->k, seq_lens, cu_seqlens, mask)) return fail("%s: tensors on different devices", op);
  if (!present(query, out, seq_lens, cu_seqlens, mask)) return fail("%s: a tensor has no data", op);
  if (query->device < 0) return fail("%s: tensors must be CUDA tensors", op);
  if (query->size[0] == 0) return GGUF_DEC_OK;
  const size_t need = tree ? gguf_kv8_tree_attention_workspace_bytes(cache, query, rows.seqs, max_new, max_len) : 0;
  if (need > 0 && (!workspace || workspace_bytes < need)) return fail("%s: workspace of %zu bytes needed, got %zu", op, need, workspace_bytes);
  const DeviceScope scope(query->device);
  if (scope.err != hipSuccess) return hip_fail(scope.err, op);
  const hipError_t e = gguf_dec::launch_kv8_attention(
      c, query->dtype, query->data, stride_of(query, 0), stride_of(query, 1), (int)query->size[1], (const int32_t*)seq_lens->data,
      rows, bounded(max_new, query->size[0]), bounded(max_len, INT_MAX), scale, tree ? (const int64_t*)mask->data : nullptr,
      tree ? stride_of(mask, 0) : 0, tree ? (int)mask->size[1] : 0, out->data, workspace, workspace ? workspace_bytes : 0,
      (hipStream_t)stream);
  return e == hipSuccess ? GGUF_DEC_OK : hip_fail(e, op);
}

int gguf_kv8_attention(const gguf_tensor* query, const gguf_kv8_cache* cache, const gguf_tensor* block_table,
                       const gguf_tensor* seq_lens, const gguf_tensor* cu_seqlens, int64_t max_new, int64_t max_len,
                       float scale, const gguf_tensor* out, void* workspace, size_t workspace_bytes, void* stream) {
  return attention("kv8_attention", query, cache, nullptr, false, block_table, seq_lens, cu_seqlens, max_new, max_len, scale, out,
                   workspace, workspace_bytes, stream);
}

int gguf_kv8_tree_attention(const gguf_tensor* query, const gguf_kv8_cache* cache, const gguf_tensor* tree_mask,
                            const gguf_tensor* block_table, const gguf_tensor* seq_lens, const gguf_tensor* cu_seqlens,
                            int64_t max_new, int64_t max_len, float scale, const gguf_tensor* out, void* workspace,
                            size_t workspace_bytes, void* stream) {
  return attention("kv8_tree_attention", query, cache, tree_mask, true, block_table, seq_lens, cu_seqlens, max_new, max_len, scale,
                   out, workspace, workspace_bytes, stream);
}

int gguf_kv8_rotary_append(const gguf_kv8_cache* cache, const gguf_tensor* query, const gguf_tensor* key,
                           const gguf_tensor* value, const gguf_tensor* cos_sin, const gguf_tensor* positions,
                           const gguf_tensor* block_table, const gguf_tensor* seq_lens, const gguf_tensor* cu_seqlens,
                           int64_t max_new, int interleaved, const gguf_tensor* q_weight, const gguf_tensor* k_weight, float eps,
                           const gguf_tensor* query_out, void* stream) {
  begin();
  const char* op = "kv8_rotary_append";
  if (!shaped(query, 3) || !shaped(key, 3) || !shaped(value, 3)) return fail("%s: query, key and value must be [tokens, heads, head size]", op);
  if (!is_float(key->dtype) || value->dtype != key->dtype || query->dtype != key->dtype) return fail("%s: query, key and value must share one float dtype", op);
  const int64_t t = key->size[0];
  Ragged rows;
  Kv8 c;
  if (check_cu(op, cu_seqlens, t, &rows) || check_cache(op, cache, block_table, rows.seqs, &c) ||
      check_seq_ints(op, "seq_lens", seq_lens, rows.seqs))
    return GGUF_DEC_EINVAL;
  for (const gguf_tensor* x : {key, value})
    if (x->size[0] != t || x->size[1] != c.heads || x->size[2] != c.d)
      return fail("%s: key and value must be [tokens, %d, %d] for this cache", op, c.heads, c.d);
  if (query->size[0] != t || query->size[1] < 1 || query->size[2] != c.d) return fail("%s: query must be [tokens, heads, %d] with key's tokens", op, c.d);
  if (t > 0 && (!rows_ok(query) || !rows_ok(key) || !rows_ok(value)))
    return fail("%s: query, key and value need unit inner stride and 16-byte aligned rows", op);
  if ((int64_t)rows.seqs * c.heads >= (1 << 21)) return fail("%s: sequences times heads must be below 2^21", op);
  if (!shaped(cos_sin, 2) || cos_sin->dtype != GGUF_DEC_F32 || cos_sin->size[0] < 1 || cos_sin->size[1] < 16 || cos_sin->size[1] % 16 ||
      cos_sin->size[1] > c.d || cos_sin->stride[1] != 1 || !aligned(cos_sin, 16) || stride_of(cos_sin, 0) % 4)
    return fail("%s: cos_sin must be fp32 [positions, 16 .. %d in steps of 16] with unit inner stride and 16-byte aligned rows", op, c.d);
  if (!shaped(positions, 1) || positions->dtype != GGUF_DEC_I64 || positions->size[0] != t || !contiguous(positions) || !aligned(positions, 8))
    return fail("%s: positions must be a contiguous int64 [tokens]", op);
  for (const gguf_tensor* w : {q_weight, k_weight})
    if (w && (!shaped(w, 1) || w->dtype != GGUF_DEC_F32 || w->size[0] != c.d || !contiguous(w) || !aligned(w, 16)))
      return fail("%s: q_weight and k_weight must be contiguous, 16-byte aligned fp32 of %d values", op, c.d);
  if (!(eps >= 0.0f) || !std::isfinite(eps)) return fail("%s: eps must be finite and not negative", op);
  if (!shaped(query_out, 3) || query_out->dtype != query->dtype || query_out->size[0] != t || query_out->size[1] != query->size[1] ||
      query_out->size[2] != c.d || !contiguous(query_out) || (t > 0 && !aligned(query_out, 16)))
    return fail("%s: query_out must be contiguous, 16-byte aligned, with query's shape and dtype", op);
  if (max_new < 0) return fail("%s: max_new must not be negative", op);
  if (!same_device(key->device, query, value, cos_sin, positions, &cache->k, seq_lens, cu_seqlens, q_weight, k_weight, query_out))
    return fail("%s: tensors on different devices", op);
  if (!present(query, key, value, cos_sin, positions, seq_lens, cu_seqlens, q_weight, k_weight, query_out)) return fail("%s: a tensor has no data", op);
  if (key->device < 0) return fail("%s: tensors must be CUDA tensors", op);
  if (t == 0) return GGUF_DEC_OK;
  const DeviceScope scope(key->device);
  if (scope.err != hipSuccess) return hip_fail(scope.err, op);
  const gguf_dec::RotaryArgs a{c, query->data, key->data, value->data, stride_of(query, 0), stride_of(query, 1), stride_of(key, 0),
                               stride_of(key, 1), stride_of(value, 0), stride_of(value, 1), q_weight ? (const float*)q_weight->data : nullptr,
                               k_weight ? (const float*)k_weight->data : nullptr, eps, (const float*)cos_sin->data, stride_of(cos_sin, 0),
                               cos_sin->size[0], (const int64_t*)positions->data, (int)cos_sin->size[1], interleaved != 0,
                               (const int32_t*)seq_lens->data, rows, (int)query->size[1], query_out->data};
  const hipError_t e = gguf_dec::launch_kv8_rotary(a, key->dtype, bounded(max_new, t), (hipStream_t)stream);
  return e == hipSuccess ? GGUF_DEC_OK : hip_fail(e, op);
}

int gguf_kv8_keep(const gguf_kv8_cache* cache, const gguf_tensor* path, const gguf_tensor* block_table, const gguf_tensor* seq_lens,
                  const gguf_tensor* cu_seqlens, void* stream) {
  begin();
  const char* op = "kv8_keep";
  Ragged rows;
  Kv8 c;
  if (check_cu(op, cu_seqlens, INT_MAX, &rows) || check_cache(op, cache, block_table, rows.seqs, &c) ||
      check_seq_ints(op, "seq_lens", seq_lens, rows.seqs))
    return GGUF_DEC_EINVAL;
  if (!shaped(path, 2) || path->dtype != GGUF_DEC_I32 || path->size[0] != rows.seqs || (path->size[1] > 1 && path->stride[1] != 1))
    return fail("%s: path must be int32 [sequences, rows] with unit inner stride", op);
  if (path->size[1] > gguf_dec::kMostKept) return fail("%s: a path of %lld rows is longer than %d", op, (long long)path->size[1], gguf_dec::kMostKept);
  if ((int64_t)rows.seqs * c.heads >= (1 << 22)) return fail("%s: sequences times heads must be below 2^22", op);
  if (!same_device(cache->k.device, path, seq_lens, cu_seqlens)) return fail("%s: tensors on different devices", op);
  if (!present(path, seq_lens, cu_seqlens)) return fail("%s: a tensor has no data", op);
  if (cache->k.device < 0) return fail("%s: tensors must be CUDA tensors", op);
  if (path->size[1] == 0) return GGUF_DEC_OK;
  const DeviceScope scope(cache->k.device);
  if (scope.err != hipSuccess) return hip_fail(scope.err, op);
  const hipError_t e = gguf_dec::launch_kv8_keep(c, (const int32_t*)path->data, stride_of(path, 0), (int)path->size[1],
                                                 (const int32_t*)seq_lens->data, rows, (hipStream_t)stream);
  return e == hipSuccess ? GGUF_DEC_OK : hip_fail(e, op);
}

int gguf_residual_norm(const gguf_tensor* x, const gguf_tensor* residual, const gguf_tensor* gate, int act,
                       const gguf_tensor* inner_weight, const gguf_tensor* weight, float scale, float eps, const gguf_tensor* hidden,
                       const gguf_tensor* out, void* stream) {
  begin();
  const char* op = "residual_norm";
  const int nd = x && x->ndim == 3 ? 3 : 2;
  if (!shaped(x, nd) || !is_float(x->dtype)) return fail("%s: x must be a float [rows, n] or [rows, heads, n]", op);
  const int64_t n = x->size[nd - 1], heads = nd == 3 ? x->size[1] : 1;
  if (n < 1 || heads < 1) return fail("%s: x has no columns", op);
  if (n > (1 << 30) || x->size[0] > INT_MAX / heads) return fail("%s: x has too many rows or columns", op);
  const int64_t rows = x->size[0] * heads;
  const auto like = [&](const gguf_tensor* t) {
    if (!shaped(t, nd)) return false;
    for (int i = 0; i < nd; ++i)
      if (t->size[i] != x->size[i]) return false;
    return true;
  };
  if (gate && (!like(gate) || gate->dtype != x->dtype)) return fail("%s: gate must have x's shape and dtype", op);
  if (act < 0 || act > 2) return fail("%s: act=%d is not 0 (none), 1 (sigmoid) or 2 (silu)", op, act);
  if (residual && (!like(residual) || (residual->dtype != x->dtype && residual->dtype != GGUF_DEC_F32)))
    return fail("%s: residual must have x's shape, and its dtype or fp32", op);
  for (const gguf_tensor* w : {inner_weight, weight})
    if (w && (!shaped(w, 1) || w->dtype != GGUF_DEC_F32 || w->size[0] != n || !contiguous(w) || !aligned(w, 4)))
      return fail("%s: weights must be contiguous fp32 of %lld values", op, (long long)n);
  const int rdt = residual ? residual->dtype : x->dtype;
  if (!like(hidden) || hidden->dtype != rdt || !contiguous(hidden) || !aligned(hidden, size_of(rdt)))
    return fail("%s: hidden must be contiguous, with x's shape and residual's dtype", op);
  if (weight && (!like(out) || out->dtype != x->dtype || !contiguous(out) || !aligned(out, size_of(x->dtype))))
    return fail("%s: out must be contiguous, with x's shape and dtype", op);
  for (const gguf_tensor* t : {x, residual, gate})
    if (t && ((n > 1 && t->stride[nd - 1] != 1) || !aligned(t, size_of(t->dtype))))
      return fail("%s: x, residual and gate need unit inner stride and alignment to their elements", op);
  if (!std::isfinite(scale) || !(eps >= 0.0f) || !std::isfinite(eps)) return fail("%s: scale must be finite, eps finite and not negative", op);
  if (!weight) out = nullptr;
  if (!same_device(x->device, residual, gate, inner_weight, weight, hidden, out)) return fail("%s: tensors on different devices", op);
  if (!present(x, residual, gate, inner_weight, weight, hidden, out)) return fail("%s: a tensor has no data", op);
  if (x->device < 0) return fail("%s: tensors must be CUDA tensors", op);
  if (rows == 0) return GGUF_DEC_OK;
  bool wide = n % 8 == 0;
  for (const gguf_tensor* t : {x, residual, gate, inner_weight, weight, hidden, out}) {
    if (!t) continue;
    wide = wide && aligned(t, 16);
    for (int i = 0; i + 1 < t->ndim; ++i) wide = wide && stride_of(t, i) * size_of(t->dtype) % 16 == 0;
  }
  const auto strides = [&](const gguf_tensor* t) {
    return t ? gguf_dec::RowStride{stride_of(t, 0), nd == 3 ? stride_of(t, 1) : 0} : gguf_dec::RowStride{0, 0};
  };
  const auto data = [](const gguf_tensor* t) { return t ? t->data : nullptr; };
  const DeviceScope scope(x->device);
  if (scope.err != hipSuccess) return hip_fail(scope.err, op);
  const gguf_dec::NormArgs a{x->data, data(residual), data(gate), (const float*)data(inner_weight), (const float*)data(weight),
                             hidden->data, data(out), strides(x), strides(residual), strides(gate), rows, (int)heads, (int)n,
                             act, scale, eps};
  const hipError_t e = gguf_dec::launch_norm(a, x->dtype, rdt, wide, (hipStream_t)stream);
  return e == hipSuccess ? GGUF_DEC_OK : hip_fail(e, op);
}

size_t gguf_gated_delta_rule_workspace_bytes(const gguf_tensor* q, const gguf_tensor* v, int64_t seqs, int64_t max_new,
                                             int steps) {
  if (!q || !v || q->ndim != 3 || v->ndim != 3 || seqs < 1 || q->size[0] < 1) return 0;
  return gguf_dec::delta_workspace(q->dtype, (int)q->size[2], (int)q->size[1], (int)v->size[1], q->size[0], seqs, max_new,
                                   steps != 0);
}

int gguf_gated_delta_rule(const gguf_tensor* q, const gguf_tensor* k, const gguf_tensor* v, const gguf_tensor* g,
                          const gguf_tensor* beta, const gguf_tensor* state, const gguf_tensor* slots,
                          const gguf_tensor* out_slots, const gguf_tensor* cu_seqlens, int64_t max_new, float scale,
                          int l2norm, const gguf_tensor* out, void* workspace, size_t workspace_bytes, void* stream) {
  begin();
  const char* op = "gated_delta_rule";
  if (!shaped(q, 3) || !shaped(k, 3) || !shaped(v, 3)) return fail("%s: q, k and v must be [tokens, heads, head size]", op);
  if (!is_float(q->dtype) || k->dtype != q->dtype || v->dtype != q->dtype) return fail("%s: q, k and v must share one float dtype", op);
  const int64_t t = q->size[0], hk = q->size[1], dk = q->size[2], hv = v->size[1], dv = v->size[2];
  if (k->size[0] != t || v->size[0] != t || k->size[1] != hk || k->size[2] != dk)
    return fail("%s: q and k must have one shape, and v as many tokens", op);
  if (dk != 64 && dk != 128) return fail("%s: key head size %lld is not 64 or 128", op, (long long)dk);
  if (dv < 16 || dv % 16 || dv > 65536) return fail("%s: value head size %lld is not a multiple of 16", op, (long long)dv);
  if (hk < 1 || hv < 1 || hv % hk || hv > 65535) return fail("%s: %lld value heads are no multiple of %lld key heads", op, (long long)hv, (long long)hk);
  if (t > 0 && (!rows_ok(q) || !rows_ok(k) || !rows_ok(v))) return fail("%s: q, k and v need unit inner stride and 16-byte aligned rows", op);
  if (hv * dv > (1 << 22) || (t > 1 && v->stride[0] > (1 << 22)))  // 64 rows are addressed by 32-bit byte offsets
    return fail("%s: rows of v and out must be at most 2^22 elements apart", op);
  for (const gguf_tensor* x : {g, beta})
    if (!shaped(x, 2) || x->dtype != GGUF_DEC_F32 || x->size[0] != t || x->size[1] != hv || (hv > 1 && x->stride[1] != 1) || !aligned(x, 4))
      return fail("%s: g and beta must be fp32 [tokens, value heads] with unit inner stride", op);
  Ragged rows;
  if (check_cu(op, cu_seqlens, t, &rows)) return GGUF_DEC_EINVAL;
  if (!shaped(state, 4) || state->dtype != GGUF_DEC_F32 || state->size[0] < 1 || state->size[1] != hv || state->size[2] != dv ||
      state->size[3] != dk || !contiguous(state) || !aligned(state, 16))
    return fail("%s: state must be a contiguous, 16-byte aligned fp32 [slots, %lld, %lld, %lld]", op, (long long)hv, (long long)dv, (long long)dk);
  if (check_seq_ints(op, "slots", slots, rows.seqs)) return GGUF_DEC_EINVAL;
  int steps = 0;
  const int32_t* outs = (const int32_t*)slots->data;
  int64_t out_stride = 1;
  if (out_slots) {
    const bool two = out_slots->ndim == 2;
    if (!shaped(out_slots, two ? 2 : 1) || out_slots->dtype != GGUF_DEC_I32 || !contiguous(out_slots) ||
        out_slots->size[0] != rows.seqs || (two && out_slots->size[1] < 1))
      return fail("%s: out_slots must be a contiguous int32 [sequences] or [sequences, tokens]", op);
    outs = (const int32_t*)out_slots->data;
    if (two) {
      steps = (int)out_slots->size[1];
      out_stride = steps;
    }
  }
  if (!shaped(out, 3) || out->dtype != q->dtype || out->size[0] != t || out->size[1] != hv || out->size[2] != dv ||
      !contiguous(out) || !aligned(out, 4))
    return fail("%s: out must be a contiguous [tokens, %lld, %lld] in q's dtype", op, (long long)hv, (long long)dv);
  if (max_new < 0) return fail("%s: max_new must not be negative", op);
  if (!std::isfinite(scale)) return fail("%s: scale must be finite", op);
  if (!same_device(q->device, k, v, g, beta, state, slots, out_slots, cu_seqlens, out)) return fail("%s: tensors on different devices", op);
  if (!present(q, k, v, g, beta, state, slots, out_slots, cu_seqlens, out)) return fail("%s: a tensor has no data", op);
  if (q->device < 0) return fail("%s: tensors must be CUDA tensors", op);
  const size_t need = t ? gguf_dec::delta_workspace(q->dtype, (int)dk, (int)hk, (int)hv, t, rows.seqs, max_new, steps > 0) : 0;
  if (need > 0 && (workspace_bytes < need || !workspace)) return fail("%s: workspace of %zu bytes needed, got %zu", op, need, workspace_bytes);
  if (reinterpret_cast<uintptr_t>(workspace) % 16) return fail("%s: workspace must be 16-byte aligned", op);
  const DeviceScope scope(q->device);
  if (scope.err != hipSuccess) return hip_fail(scope.err, op);
  const gguf_dec::DeltaArgs a{q->data, k->data, v->data, stride_of(q, 0), stride_of(q, 1), stride_of(k, 0), stride_of(k, 1),
                              stride_of(v, 0), stride_of(v, 1), (const float*)g->data, (const float*)beta->data, stride_of(g, 0),
                              stride_of(beta, 0), (float*)state->data, state->size[0], (const int32_t*)slots->data, outs, out_stride,
                              steps, (int)hk, (int)hv, (int)dv, (int)(hv / hk), scale, l2norm != 0, rows, out->data};
  const hipError_t e = gguf_dec::launch_delta(a, q->dtype, (int)dk, max_new, need ? workspace : nullptr, (hipStream_t)stream);
  return e == hipSuccess ? GGUF_DEC_OK : hip_fail(e, op);
}

size_t gguf_token_logprobs_workspace_bytes(int64_t rows, int64_t vocab, int64_t top) {
  return rows < 1 || vocab < 1 || top < 0 ? 0 : gguf_dec::logprobs_workspace(rows, vocab, top);
}

int gguf_token_logprobs(const gguf_tensor* logits, const gguf_tensor* token_ids, int64_t top, const gguf_tensor* logprobs,
                        const gguf_tensor* ranks, const gguf_tensor* entropy, const gguf_tensor* top_logprobs,
                        const gguf_tensor* top_ids, void* workspace, size_t workspace_bytes, void* stream) {
  begin();
  const char* op = "token_logprobs";
  if (!shaped(logits, 2) || !is_float(logits->dtype)) return fail("%s: logits must be a float [rows, vocab]", op);
  const int64_t rows = logits->size[0], vocab = logits->size[1];
  if (vocab < 1) return fail("%s: logits have no columns", op);
  if (vocab > 1 && logits->stride[1] != 1) return fail("%s: logits need unit inner stride", op);
  if (!aligned(logits, size_of(logits->dtype))) return fail("%s: logits must be aligned to their elements", op);
  if (!shaped(token_ids, 1) || token_ids->dtype != GGUF_DEC_I64 || token_ids->size[0] != rows) return fail("%s: token_ids must be int64 [rows]", op);
  if (top < 0 || top > 64 || top > vocab) return fail("%s: top=%lld must be 0 to 64 and at most the vocabulary", op, (long long)top);
  if (vocab > gguf_dec::logprobs_most_vocab(top)) return fail("%s: a vocabulary of %lld is too large for top=%lld", op, (long long)vocab, (long long)top);
  const struct { const gguf_tensor* t; int dt, nd; const char* name; } outs[] = {
      {logprobs, GGUF_DEC_F32, 1, "logprobs"}, {ranks, GGUF_DEC_I32, 1, "ranks"}, {entropy, GGUF_DEC_F32, 1, "entropy"},
      {top_logprobs, GGUF_DEC_F32, 2, "top_logprobs"}, {top_ids, GGUF_DEC_I32, 2, "top_ids"}};
  for (const auto& o : outs)
    if (!shaped(o.t, o.nd) || o.t->dtype != o.dt || o.t->size[0] != rows || (o.nd == 2 && o.t->size[1] != top) || !contiguous(o.t))
      return fail("%s: %s must be contiguous %s of %lld rows", op, o.name, o.dt == GGUF_DEC_F32 ? "fp32" : "int32", (long long)rows);
  if (!same_device(logits->device, token_ids, logprobs, ranks, entropy, top_logprobs, top_ids)) return fail("%s: tensors on different devices", op);
  if (!present(logits, token_ids, logprobs, ranks, entropy, top_logprobs, top_ids)) return fail("%s: a tensor has no data", op);
  if (logits->device < 0) return fail("%s: tensors must be CUDA tensors", op);
  if (rows == 0) return GGUF_DEC_OK;
  const size_t need = gguf_dec::logprobs_workspace(rows, vocab, top);
  if (workspace_bytes < need || !workspace) return fail("%s: workspace of %zu bytes needed, got %zu", op, need, workspace_bytes);
  if (reinterpret_cast<uintptr_t>(workspace) % 16) return fail("%s: workspace must be 16-byte aligned", op);
  const DeviceScope scope(logits->device);
  if (scope.err != hipSuccess) return hip_fail(scope.err, op);
  const hipError_t e = gguf_dec::launch_logprobs(logits->data, logits->dtype, stride_of(logits, 0), rows, vocab, (const int64_t*)token_ids->data,
                                                 stride_of(token_ids, 0), (int)top, (float*)logprobs->data, (int32_t*)ranks->data,
                                                 (float*)entropy->data, (float*)top_logprobs->data, (int32_t*)top_ids->data, workspace,
                                                 (hipStream_t)stream);
  return e == hipSuccess ? GGUF_DEC_OK : hip_fail(e, op);
}

}  // extern "C"
