// The decoder operators as torch.ops._C_gguf (a fragment of the namespace beside torch_ops.cpp's
// product ops), over the C ABI of libgguf_decoder.so (include/gguf_decoder.h). Host code only: each op
// describes its tensors, takes outputs and workspace from torch's caching allocator on its
// input's device (safe under graph capture) and calls the library on torch's current stream there. A
// check that fails raises RuntimeError with the library's message. Registered for CUDA (HIP tensors)
// and for CPU, where the checks run and the call ends with "must be CUDA tensors".
#include <ATen/ATen.h>
#include <c10/hip/HIPStream.h>
#include <torch/library.h>

#include <optional>
#include <tuple>

#include "../../../include/gguf_decoder.h"

namespace {

using at::Tensor;

int32_t dtype_code(const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return GGUF_DEC_F32;
    case at::kHalf: return GGUF_DEC_F16;
    case at::kBFloat16: return GGUF_DEC_BF16;
    case at::kByte: return GGUF_DEC_U8;
    case at::kChar: return GGUF_DEC_I8;
    case at::kInt: return GGUF_DEC_I32;
    case at::kLong: return GGUF_DEC_I64;
    default: return GGUF_DEC_OTHER;
  }
}

gguf_tensor desc(const Tensor& t) {
  gguf_tensor v{};
  v.data = t.numel() ? t.data_ptr() : nullptr;
  v.dtype = dtype_code(t);
  v.ndim = (int32_t)t.dim();
  for (int64_t i = 0; i < std::min<int64_t>(4, t.dim()); ++i) {
    v.size[i] = t.size(i);
    v.stride[i] = t.stride(i);
  }
  v.device = t.is_cuda() ? (int32_t)t.get_device() : -1;
  return v;
}

void check(int rc) { TORCH_CHECK(rc == GGUF_DEC_OK, gguf_decoder_last_error()); }

void* stream_of(const Tensor& t) {
  return t.is_cuda() ? (void*)c10::hip::getCurrentHIPStream(t.get_device()).stream() : nullptr;
}

Tensor workspace(const Tensor& like, size_t bytes) {
  return at::empty({(int64_t)bytes}, like.options().dtype(at::kByte));
}

void* data_of(const Tensor& t) { return t.numel() ? t.data_ptr() : nullptr; }

gguf_kv8_cache cache_of(const Tensor& k, const Tensor& v, const Tensor& ks, const Tensor& vs) {
  return gguf_kv8_cache{desc(k), desc(v), desc(ks), desc(vs)};
}

void kv8_append(const Tensor& key, const Tensor& value, const Tensor& k, const Tensor& v, const Tensor& ks,
                const Tensor& vs, const Tensor& block_table, const Tensor& seq_lens, const Tensor& cu_seqlens,
                int64_t max_new) {
  const gguf_kv8_cache c = cache_of(k, v, ks, vs);
  const gguf_tensor a = desc(key), b = desc(value), t = desc(block_table), l = desc(seq_lens), cu = desc(cu_seqlens);
  check(gguf_kv8_append(&c, &a, &b, &t, &l, &cu, max_new, stream_of(key)));
}

std::tuple<Tensor, Tensor> kv8_read(const Tensor& k, const Tensor& v, const Tensor& ks, const Tensor& vs,
                                    const Tensor& block_table, const Tensor& starts, const Tensor& cu_seqlens,
                                    int64_t tokens, int64_t max_tokens, at::ScalarType dtype) {
  const gguf_kv8_cache c = cache_of(k, v, ks, vs);
  TORCH_CHECK(k.dim() == 4 && tokens >= 0, "kv8_read: a cache of 4 dimensions and a number of tokens are needed");
  Tensor ko = at::empty({tokens, k.size(1), k.size(3)}, k.options().dtype(dtype)), vo = at::empty_like(ko);
  const gguf_tensor t = desc(block_table), s = desc(starts), cu = desc(cu_seqlens), a = desc(ko), b = desc(vo);
  check(gguf_kv8_read(&c, &t, &s, &cu, max_tokens, &a, &b, stream_of(k)));
  return {ko, vo};
}

Tensor kv8_attention(const Tensor& query, const Tensor& k, const Tensor& v, const Tensor& ks, const Tensor& vs,
                     const Tensor& block_table, const Tensor& seq_lens, const Tensor& cu_seqlens, int64_t max_new,
                     int64_t max_len, double scale) {
  const gguf_kv8_cache c = cache_of(k, v, ks, vs);
  Tensor out = at::empty(query.sizes(), query.options());
  const gguf_tensor q = desc(query), t = desc(block_table), l = desc(seq_lens), cu = desc(cu_seqlens), o = desc(out);
  const size_t bytes = gguf_kv8_attention_workspace_bytes(&c, &q, cu_seqlens.numel() - 1, max_new, max_len);
  const Tensor ws = workspace(query, bytes);
  check(gguf_kv8_attention(&q, &c, &t, &l, &cu, max_new, max_len, (float)scale, &o, data_of(ws), bytes, stream_of(query)));
  return out;
}

Tensor kv8_tree_attention(const Tensor& query, const Tensor& k, const Tensor& v, const Tensor& ks, const Tensor& vs,
                          const Tensor& tree_mask, const Tensor& block_table, const Tensor& seq_lens, const Tensor& cu_seqlens,
                          int64_t max_new, int64_t max_len, double scale) {
  const gguf_kv8_cache c = cache_of(k, v, ks, vs);
  Tensor out = at::empty(query.sizes(), query.options());
  const gguf_tensor q = desc(query), m = desc(tree_mask), t = desc(block_table), l = desc(seq_lens), cu = desc(cu_seqlens),
                    o = desc(out);
  const size_t bytes = gguf_kv8_tree_attention_workspace_bytes(&c, &q, cu_seqlens.numel() - 1, max_new, max_len);
  const Tensor ws = workspace(query, bytes);
  check(gguf_kv8_tree_attention(&q, &c, &m, &t, &l, &cu, max_new, max_len, (float)scale, &o, data_of(ws), bytes, stream_of(query)));
  return out;
}

// a tensor that may be missing, as the library takes it
struct Maybe {
  gguf_tensor t{};
  const gguf_tensor* p = nullptr;
  explicit Maybe(const std::optional<Tensor>& x) {
    if (x) {
      t = desc(*x);
      p = &t;
    }
  }
};

Tensor kv8_rotary_append(const Tensor& query, const Tensor& key, const Tensor& value, const Tensor& k, const Tensor& v,
                         const Tensor& ks, const Tensor& vs, const Tensor& cos_sin, const Tensor& positions,
                         const Tensor& block_table, const Tensor& seq_lens, const Tensor& cu_seqlens, int64_t max_new,
                         bool interleaved, const std::optional<Tensor>& q_weight, const std::optional<Tensor>& k_weight,
                         double eps) {
  const gguf_kv8_cache c = cache_of(k, v, ks, vs);
  Tensor out = at::empty(query.sizes(), query.options());
  const gguf_tensor a = desc(query), b = desc(key), x = desc(value), cs = desc(cos_sin), p = desc(positions), t = desc(block_table),
                    l = desc(seq_lens), cu = desc(cu_seqlens), o = desc(out);
  const Maybe qw(q_weight), kw(k_weight);
  check(gguf_kv8_rotary_append(&c, &a, &b, &x, &cs, &p, &t, &l, &cu, max_new, interleaved, qw.p, kw.p, (float)eps, &o, stream_of(key)));
  return out;
}

void kv8_keep(const Tensor& k, const Tensor& v, const Tensor& ks, const Tensor& vs, const Tensor& path,
              const Tensor& block_table, const Tensor& seq_lens, const Tensor& cu_seqlens) {
  const gguf_kv8_cache c = cache_of(k, v, ks, vs);
  const gguf_tensor p = desc(path), t = desc(block_table), l = desc(seq_lens), cu = desc(cu_seqlens);
  check(gguf_kv8_keep(&c, &p, &t, &l, &cu, stream_of(k)));
}

std::tuple<Tensor, Tensor> residual_norm(const Tensor& x, const std::optional<Tensor>& residual, const std::optional<Tensor>& gate,
                                         int64_t act, const std::optional<Tensor>& inner_weight,
                                         const std::optional<Tensor>& weight, double scale, double eps) {
  Tensor hidden = at::empty(x.sizes(), residual ? x.options().dtype(residual->dtype()) : x.options());
  Tensor out = weight ? at::empty(x.sizes(), x.options()) : at::empty({0}, x.options());
  const gguf_tensor a = desc(x), h = desc(hidden), o = desc(out);
  const Maybe r(residual), g(gate), wi(inner_weight), w(weight);
  check(gguf_residual_norm(&a, r.p, g.p, act < 0 || act > 2 ? -1 : (int)act, wi.p, w.p, (float)scale, (float)eps, &h, w.p ? &o : nullptr,
                           stream_of(x)));
  return {out, hidden};
}

Tensor gated_delta_rule(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& g, const Tensor& beta,
                        const Tensor& state, const Tensor& slots, const Tensor& cu_seqlens, int64_t max_new,
                        const std::optional<Tensor>& out_slots, double scale, bool l2norm) {
  const gguf_tensor dq = desc(q), dk = desc(k), dv = desc(v), dg = desc(g), db = desc(beta), ds = desc(state),
                    sl = desc(slots), cu = desc(cu_seqlens);
  gguf_tensor os{};
  if (out_slots) os = desc(*out_slots);
  Tensor out = at::empty(v.sizes(), v.options());
  const gguf_tensor o = desc(out);
  const size_t bytes = gguf_gated_delta_rule_workspace_bytes(&dq, &dv, cu_seqlens.numel() - 1, max_new,
                                                             out_slots && out_slots->dim() == 2);
  const Tensor ws = workspace(q, bytes);
  check(gguf_gated_delta_rule(&dq, &dk, &dv, &dg, &db, &ds, &sl, out_slots ? &os : nullptr, &cu, max_new, (float)scale,
                              l2norm, &o, data_of(ws), bytes, stream_of(q)));
  return out;
}

std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor> token_logprobs(const Tensor& logits, const Tensor& token_ids,
                                                                  int64_t top) {
  TORCH_CHECK(logits.dim() == 2 && top >= 0, "token_logprobs: logits must be [rows, vocab] and top not negative");
  const int64_t rows = logits.size(0);
  const auto f = logits.options().dtype(at::kFloat), i = logits.options().dtype(at::kInt);
  Tensor lp = at::empty({rows}, f), rank = at::empty({rows}, i), ent = at::empty({rows}, f);
  Tensor tlp = at::empty({rows, top}, f), tid = at::empty({rows, top}, i);
  const gguf_tensor x = desc(logits), t = desc(token_ids), a = desc(lp), b = desc(rank), c = desc(ent), d = desc(tlp),
                    e = desc(tid);
  const size_t bytes = gguf_token_logprobs_workspace_bytes(rows, logits.size(1), top);
  const Tensor ws = workspace(logits, bytes);
  check(gguf_token_logprobs(&x, &t, top, &a, &b, &c, &d, &e, data_of(ws), bytes, stream_of(logits)));
  return {lp, rank, ent, tlp, tid};
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(_C_gguf, m) {
  m.def("kv8_append(Tensor key, Tensor value, Tensor(a!) k_cache, Tensor(b!) v_cache, Tensor(c!) k_scale, "
        "Tensor(d!) v_scale, Tensor block_table, Tensor seq_lens, Tensor cu_seqlens, int max_new) -> ()");
  m.def("kv8_read(Tensor k_cache, Tensor v_cache, Tensor k_scale, Tensor v_scale, Tensor block_table, Tensor starts, "
        "Tensor cu_seqlens, int tokens, int max_tokens, ScalarType dtype) -> (Tensor, Tensor)");
  m.def("kv8_attention(Tensor query, Tensor k_cache, Tensor v_cache, Tensor k_scale, Tensor v_scale, "
        "Tensor block_table, Tensor seq_lens, Tensor cu_seqlens, int max_new, int max_len, float scale) -> Tensor");
  m.def("kv8_tree_attention(Tensor query, Tensor k_cache, Tensor v_cache, Tensor k_scale, Tensor v_scale, Tensor tree_mask, "
        "Tensor block_table, Tensor seq_lens, Tensor cu_seqlens, int max_new, int max_len, float scale) -> Tensor");
  m.def("kv8_rotary_append(Tensor query, Tensor key, Tensor value, Tensor(a!) k_cache, Tensor(b!) v_cache, "
        "Tensor(c!) k_scale, Tensor(d!) v_scale, Tensor cos_sin, Tensor positions, Tensor block_table, Tensor seq_lens, "
        "Tensor cu_seqlens, int max_new, bool interleaved, Tensor? q_weight, Tensor? k_weight, float eps) -> Tensor");
  m.def("kv8_keep(Tensor(a!) k_cache, Tensor(b!) v_cache, Tensor(c!) k_scale, Tensor(d!) v_scale, Tensor path, "
        "Tensor block_table, Tensor seq_lens, Tensor cu_seqlens) -> ()");
  m.def("residual_norm(Tensor x, Tensor? residual, Tensor? gate, int act, Tensor? inner_weight, Tensor? weight, float scale, "
        "float eps) -> (Tensor, Tensor)");
  m.def("gated_delta_rule(Tensor q, Tensor k, Tensor v, Tensor g, Tensor beta, Tensor(a!) state, Tensor slots, "
        "Tensor cu_seqlens, int max_new, Tensor? out_slots, float scale, bool l2norm) -> Tensor");
  m.def("token_logprobs(Tensor logits, Tensor token_ids, int top) -> (Tensor, Tensor, Tensor, Tensor, Tensor)");
}

#define GGUF_DEC_IMPLS(KEY)                           \
  TORCH_LIBRARY_IMPL(_C_gguf, KEY, m) {               \
    m.impl("kv8_append", &kv8_append);                \
    m.impl("kv8_read", &kv8_read);                    \
    m.impl("kv8_attention", &kv8_attention);          \
    m.impl("kv8_tree_attention", &kv8_tree_attention); \
    m.impl("kv8_rotary_append", &kv8_rotary_append);  \
    m.impl("kv8_keep", &kv8_keep);                    \
    m.impl("residual_norm", &residual_norm);          \
    m.impl("gated_delta_rule", &gated_delta_rule);    \
    m.impl("token_logprobs", &token_logprobs);        \
  }
GGUF_DEC_IMPLS(CUDA)
GGUF_DEC_IMPLS(CPU)
#undef GGUF_DEC_IMPLS
