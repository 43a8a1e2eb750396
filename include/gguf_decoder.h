/* C ABI of libgguf_decoder.so: the MI355X (gfx950) operators that stand between a decoder's GGUF
 * linear layers (libgguf_mi355x.so) and behind its head.
 *
 *   gguf_kv8_append, gguf_kv8_read, gguf_kv8_attention   a paged KV cache in 8 bits, and attention over it
 *   gguf_kv8_rotary_append                               the position rotation on the way into that cache
 *   gguf_kv8_tree_attention, gguf_kv8_keep               attention for a tree of drafts, and keeping a path of it
 *   gguf_residual_norm                                   norms before and after a block, its gate and residual
 *   gguf_gated_delta_rule                                linear attention: recurrent and chunked
 *   gguf_token_logprobs                                  log probabilities, entropy and best tokens
 *
 * Conventions, as in gguf_mi355x.h: plain pointers, sizes and strides; the caller gives outputs,
 * workspace and stream; the library allocates nothing, never synchronises the host and keeps no
 * state between calls. Rows that belong to no sequence (before cu_seqlens[0] or past its last offset) are left unwritten or
 * unspecified. Every check that the host can make runs before any GPU access and returns
 * GGUF_DEC_EINVAL with a message in gguf_decoder_last_error() (per thread). What lies in device
 * memory (lengths, page numbers, slots, token ids) is checked by the kernels: a length is cut to what
 * its tensors hold, and what each entry point says happens for a page, slot or token id out of
 * range. max_new and max_len are hints: they size the grid, and choose between forms of a call that compute the same
 * and round differently, as its entry point says (kv8_attention up to 64 rows a KV head and above,
 * gated_delta_rule by tokens and by chunks). Any number is allowed. Calls are safe under stream capture.
 *
 * cu_seqlens [seqs + 1] (int32) holds the offsets of each sequence's rows in the ragged tensors, and
 * sequence s has n_s = cu_seqlens[s + 1] - cu_seqlens[s] rows.
 */
#ifndef GGUF_DECODER_H
#define GGUF_DECODER_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#if defined(__GNUC__)
#define GGUF_DEC_API __attribute__((visibility("default")))
#else
#define GGUF_DEC_API
#endif

#define GGUF_DEC_OK 0
#define GGUF_DEC_EINVAL 1
#define GGUF_DEC_EHIP 2

/* element types; the first five as in gguf_mi355x.h */
enum {
  GGUF_DEC_F32 = 0,
  GGUF_DEC_F16 = 1,
  GGUF_DEC_BF16 = 2,
  GGUF_DEC_U8 = 3,
  GGUF_DEC_OTHER = 4,
  GGUF_DEC_I8 = 5,
  GGUF_DEC_I32 = 6,
  GGUF_DEC_I64 = 7
};

/* A strided tensor of up to four dimensions. Sizes and strides in elements; device: GPU index, or
 * -1 for host memory (rejected after the shape checks, which so run without a GPU). */
typedef struct gguf_tensor {
  void* data;
  int32_t dtype;
  int32_t ndim;
  int64_t size[4];
  int64_t stride[4];
  int32_t device;
} gguf_tensor;

/* A paged KV cache in 8 bits. Pages hold `page` tokens (a multiple of 16) of every KV head; a code
 * stands for code * scale, with one fp32 scale for each (page, head) of K and of V:
 *   k        int8 [pages, heads, page, d]     contiguous, 16-byte aligned
 *   v        int8 [pages, heads, d, page]     (tokens innermost: the order in which attention's
 *                                              second product takes them)
 *   k_scale  fp32 [pages, heads], v_scale fp32 [pages, heads]      contiguous
 * A V scale below 2^-100 counts as 0 in attention. d is 64, 128, 192 or 256. A sequence's tokens
 * 0 .. len - 1 lie in the pages block_table[s, 0 ..] (int32 [seqs, max_pages], unit inner stride). */
typedef struct gguf_kv8_cache {
  gguf_tensor k, v, k_scale, v_scale;
} gguf_kv8_cache;

/* Last error message of the calling thread ("" if none). */
GGUF_DEC_API const char* gguf_decoder_last_error(void);

/* Appends the rows of key and value (fp32 / fp16 / bf16 [tokens, heads, d], unit inner stride, rows
 * 16-byte aligned) to the cache: sequence s's n_s rows become its positions seq_lens[s] - n_s ..
 * seq_lens[s] - 1. A (page, head)'s scale is its largest magnitude / 127 (0 below 2^-100) and its codes
 * round(x / scale); where the page holds older tokens its scale never falls, and where it grows
 * their codes are rounded again to the new scale. No page may be written for two sequences at once.
 * Values that are not finite make the scale so, and the (page, head) reads as NaN. Rows past the
 * table's capacity or of a page number out of range are dropped.
 * max_new: the largest n_s, a hint. */
GGUF_DEC_API int gguf_kv8_append(const gguf_kv8_cache* cache, const gguf_tensor* key, const gguf_tensor* value,
                                 const gguf_tensor* block_table, const gguf_tensor* seq_lens,
                                 const gguf_tensor* cu_seqlens, int64_t max_new, void* stream);

/* The cached values of positions starts[s] .. starts[s] + n_s - 1 of every sequence, as dense rows:
 * k_out and v_out [tokens, heads, d] (contiguous, fp32 / fp16 / bf16, 16-byte aligned). Positions
 * before 0 or past the table's capacity, or in a page whose number is out of range, read as NaN.
 * max_tokens: the largest n_s, a hint. */
GGUF_DEC_API int gguf_kv8_read(const gguf_kv8_cache* cache, const gguf_tensor* block_table, const gguf_tensor* starts,
                               const gguf_tensor* cu_seqlens, int64_t max_tokens, const gguf_tensor* k_out,
                               const gguf_tensor* v_out, void* stream);

/* Causal attention of the rows of query (fp16 / bf16 [tokens, q_heads, d], unit inner stride, rows
 * 16-byte aligned; q_heads a multiple of the cache's heads; sequences times heads below 2^24) over the cache, which
 * holds their own tokens already: row i of sequence s sees positions 0 .. seq_lens[s] - n_s + i, so
 * out = softmax(scale * q k^T) v. A row that sees nothing is 0; one that sees a page whose number is
 * out of range is NaN. out: contiguous, like query. The workspace holds the partial results of a
 * cache split over workgroups; with fewer bytes than gguf_kv8_attention_workspace_bytes (0 included) the
 * call is split less. max_new, max_len: the largest n_s and seq_lens[s], hints.
 * Precision: sums and the softmax's statistics are fp32. A weight times its page's V scale enters the second product
 * in fp16: to 2^-11 of itself down to 2^-21 of the row's largest weight times the largest V scale that the row sees, below
 * that to 2^-32 of these. Queries: where max_new * q_heads / heads is at most 64, exact but for bf16 elements below 2^-14
 * of the row's largest; above, integers of 15 bits, to 2^-15 of the row's largest magnitude (0 where that is below 2^-100).
 * A query row with an infinity or a NaN is NaN. */
GGUF_DEC_API size_t gguf_kv8_attention_workspace_bytes(const gguf_kv8_cache* cache, const gguf_tensor* query,
                                                       int64_t seqs, int64_t max_new, int64_t max_len);
GGUF_DEC_API int gguf_kv8_attention(const gguf_tensor* query, const gguf_kv8_cache* cache,
                                    const gguf_tensor* block_table, const gguf_tensor* seq_lens,
                                    const gguf_tensor* cu_seqlens, int64_t max_new, int64_t max_len, float scale,
                                    const gguf_tensor* out, void* workspace, size_t workspace_bytes, void* stream);

/* kv8_append with the position rotation of keys, and of the queries beside them, on the way, after the norms of their heads
 * where these have weights. query [tokens, q_heads, d] (any number of heads), key, value: one float dtype, unit inner stride, rows
 * 16-byte aligned; the sequences times the cache's heads below 2^21. For a head's row x of query (w = q_weight) or key
 * (w = k_weight; fp32 [d], 16-byte aligned; NULL: no norm)
 *   x = x / sqrt(mean(x^2) + eps) * w
 *   x_i, x_j = x_i c - x_j s, x_j c + x_i s   for the pairs (i, j = i + r / 2), i < r / 2; interleaved: (2 i', j = 2 i' + 1)
 * with c and s at cos_sin[positions[token], i] and [.., r / 2 + i] (i' where interleaved). cos_sin: fp32 [positions, r], r a
 * multiple of 16 up to d (dims from r on do not turn), unit inner stride, rows 16-byte aligned; positions: int64 [tokens],
 * where a tree of drafts has its depths. A position out of the table's range turns by NaN. Everything is fp32; query_out (contiguous, 16-byte
 * aligned, like query) is rounded once, a key is rounded to its code only. Squares are summed as in gguf_residual_norm. All rows of query are turned,
 * those of no sequence too. Keys and values enter the cache as by gguf_kv8_append. */
GGUF_DEC_API int gguf_kv8_rotary_append(const gguf_kv8_cache* cache, const gguf_tensor* query, const gguf_tensor* key,
                                        const gguf_tensor* value, const gguf_tensor* cos_sin, const gguf_tensor* positions,
                                        const gguf_tensor* block_table, const gguf_tensor* seq_lens,
                                        const gguf_tensor* cu_seqlens, int64_t max_new, int interleaved,
                                        const gguf_tensor* q_weight, const gguf_tensor* k_weight, float eps,
                                        const gguf_tensor* query_out, void* stream);

/* kv8_attention for a tree of drafts: row i of sequence s sees positions 0 .. b - 1, b = seq_lens[s] - n_s, and of the sequence's
 * own rows j (at positions b + j) those with bit j % 64 of tree_mask[row, j / 64] set (int64 [tokens, words], unit inner
 * stride; rows past 64 * words are not seen). Usually these are a draft's ancestors and itself, but any bits are allowed. Otherwise
 * as gguf_kv8_attention, but for the workspace, which is needed whole, and for queries, which never become integers: bf16 elements
 * below 2^-14 of the row's largest alone are rounded. */
GGUF_DEC_API size_t gguf_kv8_tree_attention_workspace_bytes(const gguf_kv8_cache* cache, const gguf_tensor* query,
                                                            int64_t seqs, int64_t max_new, int64_t max_len);
GGUF_DEC_API int gguf_kv8_tree_attention(const gguf_tensor* query, const gguf_kv8_cache* cache, const gguf_tensor* tree_mask,
                                         const gguf_tensor* block_table, const gguf_tensor* seq_lens,
                                         const gguf_tensor* cu_seqlens, int64_t max_new, int64_t max_len, float scale,
                                         const gguf_tensor* out, void* workspace, size_t workspace_bytes, void* stream);

/* Keeps a path of a tree of drafts: of sequence s's n_s last positions b .. seq_lens[s] - 1, row path[s, j] moves to position
 * b + j, in the cache alone (int32 [sequences, m], unit inner stride, m up to 1024; sequences times heads below 2^22). A path grows strictly and ends
 * before its first entry that is out of range or does not; what lies behind its last place is no longer the sequence's (the
 * caller's next seq_lens says so) and may have changed. Within a page codes move as they are; from another page they are rounded
 * to the page's scale, which grows where the moved rows need it, and the page's other codes then are rounded again to it, as
 * by gguf_kv8_append. A row from a page whose number is out of range makes the page that receives it NaN; one that would go to such a page is dropped. */
GGUF_DEC_API int gguf_kv8_keep(const gguf_kv8_cache* cache, const gguf_tensor* path, const gguf_tensor* block_table,
                               const gguf_tensor* seq_lens, const gguf_tensor* cu_seqlens, void* stream);

/* The norm behind a block, its gate, the residual, and the next block's norm, row by row over the last dimension n of x
 * (fp32 / fp16 / bf16 [rows, n] or [rows, heads, n], unit inner stride; any other strides, 0 included). Each part may be NULL:
 *   u = x;   u = u / sqrt(mean(u^2) + eps) * inner_weight;   u = u * act(gate);   h = residual + scale * u
 *   out = h / sqrt(mean(h^2) + eps) * weight
 * act: 0 the gate itself, 1 its sigmoid, 2 silu; without a gate it is not looked at. gate: like x (other strides); residual: x's shape, x's dtype or fp32; weights: fp32 [n].
 * hidden (h): contiguous, residual's dtype (x's without one), written by every call; out: contiguous, x's dtype, not read or written without weight. Neither
 * overlaps an input. Everything between is fp32: out comes from h before its rounding. Where hidden is not fp32, a sigmoid is
 * known to 2^-17 of itself and may be 0 for gates below -87; where it is, to some steps of fp32. Squares are summed in fp32, so a row of
 * magnitudes beyond 2^63 is taken for infinite, and without eps one below 2^-63 loses bits of its mean. */
GGUF_DEC_API int gguf_residual_norm(const gguf_tensor* x, const gguf_tensor* residual, const gguf_tensor* gate, int act,
                                    const gguf_tensor* inner_weight, const gguf_tensor* weight, float scale, float eps,
                                    const gguf_tensor* hidden, const gguf_tensor* out, void* stream);

/* The gated delta rule over ragged sequences. q, k: [tokens, hk, dk], v: [tokens, hv, dv] of one
 * float dtype (unit inner stride, rows 16-byte aligned; hv a multiple of hk; dk 64 or 128, dv a
 * multiple of 16); g (log of the decay), beta: fp32 [tokens, hv] (unit inner stride). For each v
 * head, with the fp32 state S [dv, dk] of its sequence, token by token,
 *   S = exp(g) S;   S = S + beta (v - S k) k^T;   out = scale S q
 * where l2norm first divides q and k by sqrt(|x|^2 + 1e-6). state: fp32 [slots, hv, dv, dk],
 * contiguous, 16-byte aligned. Sequence s starts from state[slots[s]], or from zero where slots[s]
 * is out of range (-1). out_slots (int32) says where states go: [seqs]: after the sequence's last
 * token; [seqs, m]: after each of its first m tokens, as a verify pass needs that may keep only some of
 * them; NULL: back to slots. A slot out of range keeps nothing, and a sequence of no tokens
 * copies its state to a [seqs] slot. No slot may be written twice, or written for one sequence and read
 * for another. out: [tokens, hv, dv] contiguous, in q's dtype. Token strides are at most 2^22 elements. What a
 * token that is not finite reaches (a value's column, a key's, gate's or beta's head, from that token on) is
 * not finite, and nothing else is.
 * Precision: states are fp32 throughout, products carry 24 bits. In the chunked form (more than 32 tokens) the two
 * products that make an fp16 or bf16 output, S q and A u, keep 2^-16 of their terms.
 * max_new: the largest n_s, a hint; the workspace is for sequences of more tokens than the recurrent form
 * takes (gguf_gated_delta_rule_workspace_bytes). */
GGUF_DEC_API size_t gguf_gated_delta_rule_workspace_bytes(const gguf_tensor* q, const gguf_tensor* v, int64_t seqs,
                                                          int64_t max_new, int steps);
GGUF_DEC_API int gguf_gated_delta_rule(const gguf_tensor* q, const gguf_tensor* k, const gguf_tensor* v,
                                       const gguf_tensor* g, const gguf_tensor* beta, const gguf_tensor* state,
                                       const gguf_tensor* slots, const gguf_tensor* out_slots,
                                       const gguf_tensor* cu_seqlens, int64_t max_new, float scale, int l2norm,
                                       const gguf_tensor* out, void* workspace, size_t workspace_bytes, void* stream);

/* For each row of logits (fp32 / fp16 / bf16 [rows, vocab], unit inner stride): the log probability
 * of token_ids[row] (int64), its rank (1 + the tokens before it in descending order, equal ones by
 * index), the entropy of the row's distribution, and the `top` (0 .. 64, at most vocab) best tokens'
 * log probabilities and ids in that order. A token id out of range has log probability NaN and rank 0;
 * a row with a NaN or +inf, or of -inf alone, has NaN log probabilities, as log_softmax has.
 * logprobs, entropy: fp32 [rows]; ranks: int32 [rows]; top_logprobs fp32, top_ids int32 [rows, top];
 * all contiguous (data of the last two may be NULL where top is 0). */
GGUF_DEC_API size_t gguf_token_logprobs_workspace_bytes(int64_t rows, int64_t vocab, int64_t top);
GGUF_DEC_API int gguf_token_logprobs(const gguf_tensor* logits, const gguf_tensor* token_ids, int64_t top,
                                     const gguf_tensor* logprobs, const gguf_tensor* ranks, const gguf_tensor* entropy,
                                     const gguf_tensor* top_logprobs, const gguf_tensor* top_ids, void* workspace,
                                     size_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* GGUF_DECODER_H */
