/*
 * hephserve.h - the ops of a batched serving step around the W8A8 linears:
 * q/k norm + rotation into a paged KV cache, attention of a batch over that
 * cache with shared prefixes computed once, page copies (each with one scale
 * for a whole layer's head, or one for each page found while it is written),
 * the low-rank adapters of many requests beside one projection, and the pick
 * of the next tokens from a batch's logits. Same conventions as
 * hephfp8.h: device pointers unless an argument says host, a hipStream_t as
 * void* (NULL = default stream), HEPH_* status codes, no allocation, no
 * synchronization, capturable into a HIP graph.
 *
 * bf16 tensors are passed as their 16-bit patterns. Head size is 128. What
 * only the device sees (positions, slots, page ids, lengths, adapter ids) is
 * clamped or skipped there as stated below: no value makes an op read or
 * write outside its buffers.
 */
#ifndef HEPHSERVE_H
#define HEPHSERVE_H

#include <stddef.h>
#include <stdint.h>

#include "hephdecode.h"

#ifdef __cplusplus
extern "C" {
#endif

/*
 * The paged cache (E4M3 codes, head_dim 128): pages of HEPH_PAGE_KEYS keys,
 * 8192 bytes a kv head in each of two pools.
 *   K: [n_pages][n_kv_heads][2][64 keys][64 dims]: key j, dim d at
 *      d/64 * 4096 + j * 64 + d%64.
 *   V: [n_pages][n_kv_heads][128 dims][64 places]: key j, dim d at
 *      d * 64 + place(j), place(j) = j/4%4 * 16 + j/32 * 8 + j/16%2 * 4 + j%4.
 * A slot is page * 64 + key. The 16 bytes a lane loads are the operands of
 * two matrix instructions (K: 16 dims of a key; V: 16 keys of a dim, in the
 * order in which the scores of those keys lie in that lane).
 */
#define HEPH_PAGE_KEYS 64
/* Most sequences of one attention call. */
#define HEPH_PAGES_MAX_SEQS 1024

/*
 * Rotation table: table[pos][p] = (cos, sin) of pair p < head_dim/2 at
 * position pos < n_pos in f32, the angle pos * theta^(-2p/head_dim) in
 * double (2 * n_pos * head_dim/2 floats). head_dim 128, table 16-byte
 * aligned.
 */
int heph_rope_table_f32(float* table, int n_pos, int head_dim, double theta, void* stream);

/*
 * The batch form of heph_qk_norm_rope_kv on a paged cache. For token t < n_tok
 * at qkv + t * qkv_stride ([n_heads + 2*n_kv_heads, 128]; strides in elements,
 * multiples of 8): per-head RMSNorm of q (q_gamma) and k (k_gamma) and the
 * rotation of both by rope_table's row positions[t], q to q_out + t * q_stride
 * ([n_heads, 128] bf16); k and v as e4m3(clamp(x * kv_inv_scale[h], +-448))
 * into slot slots[t] of the pools (kv_inv_scale: n_kv_heads K entries, then V; a
 * NaN is clamped to -448, as heph_qk_norm_rope_kv does).
 * Norm and rotation are computed in f32 and rounded once (heph_qk_norm_rope_kv
 * rounds every step to bf16, as the reference's single-token path does).
 * A token whose position is outside [0, n_rope_pos) is skipped: its q and its
 * slot stay as they were (padding rows: position -1). A slot outside
 * [0, 64 * n_pages) is not written; q is. n_pages < 2^25. The slots of a call's tokens are
 * distinct. q_out may be qkv itself with the same stride (q in place), and
 * overlaps it in no other way.
 * Replaces, for a batch, the q/k norms, rotation and cache write of the
 * reference's batched decode (src/hephaestus/forward.mojo:618-871).
 */
int heph_qk_norm_rope_pages(void* q_out_bf16, int64_t q_stride, const void* qkv_bf16,
                            int64_t qkv_stride, const void* q_gamma, const void* k_gamma,
                            uint8_t* k_pages, uint8_t* v_pages, int n_pages,
                            const float* kv_inv_scale, const float* rope_table, int n_rope_pos,
                            const int32_t* positions, const int32_t* slots, int n_tok,
                            int n_heads, int n_kv_heads, int head_dim, float eps, void* stream);

/*
 * Attention of a batch over the paged cache. Sequence s has kv_len[s] keys,
 * key j in page page_table[s * table_pages + j/64]; its tokens are rows
 * q_start[s] .. q_start[s+1]-1 of q and out (q_start: n_seqs + 1 entries, not
 * decreasing) and are its newest keys, already in the cache: token i of n
 * attends to keys 0 .. kv_len[s] - n + i.
 *   out[t, h] = sum_j softmax_j(q . k_j * sk / sqrt(128)) v_j sv
 * with kv_scale (n_kv_heads K entries, then V). Scores, softmax statistics and
 * sums are f32; the unnormalized probabilities are rounded to bf16 for the
 * product with V, and out once to bf16. A token without keys gives a zero row.
 * n_heads is a multiple of n_kv_heads, at most 64 times it; n_seqs is at most
 * HEPH_PAGES_MAX_SEQS. kv_scale > 0. A token whose every score is -inf gives a
 * zero row.
 *
 * Shared prefixes: group g is the sequences group_start[g] ..
 * group_start[g+1]-1 (n_groups + 1 entries, not decreasing), whose first
 * shared_pages[g] page-table entries are the same pages. Their keys are read
 * once for the group's rows together, from the table row of the group's first
 * sequence, if two or more of its sequences have less than 64 rows (tokens x
 * heads a kv head), or enough of them 64 behind a long prefix, and longer
 * prompts' rows would not pay more for it than that saves; else for each sequence
 * from its own table row, with the same answer up to the order of sums. Sequences in no
 * group, or n_groups = 0 with both NULL: nothing shared. A shared_pages beyond a
 * sequence's own keys is allowed.
 *
 * heph_pages_attention_plan (one small launch) lays out a step's work from
 * the lengths in device memory; one plan serves the attention of every layer
 * of the step. The attention takes the same sizes as its plan; with others it
 * writes nothing. plan and ws: device buffers of the two _bytes functions,
 * 16-byte aligned; calls that share a ws are ordered by the caller. A larger
 * ws is not used.
 *
 * On the device: q_start is clamped to [0, n_tok], kv_len to [0, 64 *
 * table_pages]; the keys of a page id outside [0, n_pages) are left out as if
 * masked. Rows of no sequence are left as they were; rows that a decreasing
 * q_start gives to two sequences, or that a decreasing group_start gives to two
 * groups, are undefined.
 * q + t * q_stride: [n_heads, 128] (q_stride in elements, a multiple of 8);
 * out: [n_tok, n_heads, 128], not overlapping q (q's own address: HEPH_ERR_SHAPE).
 * Replaces, for a batch, attention (src/hephaestus/kernels.mojo:923-1240) as
 * forward_fp8_batched_decode calls it per sequence
 * (src/hephaestus/forward.mojo:618-871).
 */
size_t heph_pages_attention_plan_bytes(int n_tok, int n_seqs, int n_groups, int n_heads,
                                       int n_kv_heads);
size_t heph_pages_attention_ws_bytes(int n_tok, int n_seqs, int n_groups, int n_heads,
                                     int n_kv_heads);
int heph_pages_attention_plan(void* plan, size_t plan_bytes, const int32_t* q_start,
                              const int32_t* kv_len, const int32_t* group_start,
                              const int32_t* shared_pages, int n_tok, int n_seqs, int n_groups,
                              int table_pages, int n_heads, int n_kv_heads, void* stream);
int heph_pages_attention(void* out_bf16, const void* q_bf16, int64_t q_stride,
                         const uint8_t* k_pages, const uint8_t* v_pages, int n_pages,
                         const float* kv_scale, const int32_t* page_table, int table_pages,
                         const void* plan, size_t plan_bytes, void* ws, size_t ws_bytes,
                         int n_tok, int n_seqs, int n_groups, int n_heads, int n_kv_heads,
                         int head_dim, void* stream);

/*
 * Page src[i] of every layer's K and V pool copied to page dst[i], i < n
 * (pools [n_layers][n_pages][n_kv_heads * 8192] bytes). src and dst are HOST
 * arrays, read before the call returns (a captured call keeps their values).
 * A source may feed several destinations; a destination that repeats or is a
 * source too gives HEPH_ERR_SHAPE, since the copies run at once. n = 0 does
 * nothing.
 */
int heph_copy_pages(uint8_t* k_pages, uint8_t* v_pages, int n_layers, int n_pages,
                    int n_kv_heads, const int32_t* src, const int32_t* dst, int n, void* stream);

/*
 * The same cache with a scale for each block: a page's 64 keys of one kv head,
 * K and V apart. page_scale [n_pages][2 * n_kv_heads] (a page's K heads, then
 * its V heads), all powers of two 2^e, -117 <= e <= 119: a code c stands for
 * c * 2^e, a bf16 value. Nothing has to be calibrated: the ops below find the
 * scales from what they write. Pages, slots, positions and the remaining
 * arguments are as in the ops of the same names without _scaled.
 *
 * heph_qk_norm_rope_pages_scaled: a block's scale becomes the least 2^e with
 * |x| <= 448 * 2^e for its new keys' finite values x (computed in f32; e is
 * held to the range above and values past 448 * 2^119 are clamped), and no less
 * than it was, unless the page's key 0 is among the call's tokens: they begin
 * the page anew, whatever it held. Where a scale grows by 2^n, the codes of all
 * 64 keys are divided by 2^n (exactly, but for those that leave E4M3's normal
 * range, which are rounded to its subnormal ones); new codes are
 * e4m3(x * 2^-e), and a NaN or an infinity, which E4M3 has not, is the code of
 * NaN. A scale outside the range (memory that was never written) counts as the
 * nearest one in it; a page that begins behind its key 0 has its scales set to
 * 0 first.
 * The tokens of a page are neighbours among the call's rows, as a sequence's
 * newest tokens are (tokens that are skipped, for their position or their slot, may
 * stand between them), no two of them with one slot, and a page belongs to one
 * sequence while it is written; a page among whose tokens one of another page
 * stands gets codes of more than one scale, and of two tokens for one slot either
 * may be left out.
 * Writes no page and no scale without a token of the call.
 *
 * heph_pages_attention_scaled takes a plan of heph_pages_attention_plan and the
 * workspace of heph_pages_attention_ws_bytes. Of a page_scale only the exponent
 * is used. V's scales may lie anywhere in the range above: sums are kept relative to
 * the largest one (values 2^200 times smaller than a run's largest may be lost
 * beside it). Scores q . k are f32 numbers, and have to be finite as such.
 *
 * heph_copy_pages_scaled copies the pages' scales with them (page_scale
 * [n_layers][n_pages][2 * n_kv_heads]).
 * No counterpart in the reference, whose cache is bf16.
 */
int heph_qk_norm_rope_pages_scaled(void* q_out_bf16, int64_t q_stride, const void* qkv_bf16,
                                   int64_t qkv_stride, const void* q_gamma, const void* k_gamma,
                                   uint8_t* k_pages, uint8_t* v_pages, int n_pages,
                                   float* page_scale, const float* rope_table, int n_rope_pos,
                                   const int32_t* positions, const int32_t* slots, int n_tok,
                                   int n_heads, int n_kv_heads, int head_dim, float eps,
                                   void* stream);
int heph_pages_attention_scaled(void* out_bf16, const void* q_bf16, int64_t q_stride,
                                const uint8_t* k_pages, const uint8_t* v_pages, int n_pages,
                                const float* page_scale, const int32_t* page_table, int table_pages,
                                const void* plan, size_t plan_bytes, void* ws, size_t ws_bytes,
                                int n_tok, int n_seqs, int n_groups, int n_heads, int n_kv_heads,
                                int head_dim, void* stream);
int heph_copy_pages_scaled(uint8_t* k_pages, uint8_t* v_pages, float* page_scale, int n_layers,
                           int n_pages, int n_kv_heads, const int32_t* src, const int32_t* dst,
                           int n, void* stream);

/*
 * Keys read back: row t < n_rows of k_out and v_out ([n_rows, n_kv_heads, 128]
 * bf16) gets the key and value of slots[t]: code * scale in f32, rounded to bf16
 * (both exact with page_scale, two roundings with kv_scale). One of kv_scale
 * (2 * n_kv_heads, of all pages) and page_scale is given, the other NULL. Rows of a
 * slot outside [0, 64 * n_pages) are left as they were; n_pages < 2^25. Slots may
 * repeat and come in any order; consecutive ones are read together. k_out and v_out
 * do not overlap.
 */
int heph_read_pages(void* k_out_bf16, void* v_out_bf16, const uint8_t* k_pages,
                    const uint8_t* v_pages, int n_pages, const float* kv_scale,
                    const float* page_scale, const int32_t* slots, int n_rows, int n_kv_heads,
                    int head_dim, void* stream);

/*
 * Low-rank adapters of many requests beside one projection:
 *   c[m, :] = base[m, :] + scale[i] * (x[m, :] @ a[i]^T) @ b[i]^T,  i = ids[m],
 * x bf16 [M, K], a bf16 [n_adapters, rank, K], b bf16 [n_adapters, N, rank],
 * scale f32 [n_adapters], base and c of c_dtype [M, N] (c may be base: the
 * projection's output updated in place). Rows with an id outside
 * [0, n_adapters) have no adapter: c = base. Sums are f32; x @ a^T is kept to
 * 16 bits of mantissa (a bf16 and a bf16 of its remainder) for the product
 * with b; c is rounded once.
 * N % 16 == 0, K % 16 == 0, rank % 8 == 0 and 8 <= rank <= 128 (adapters of
 * less rank are padded with zeros); n_adapters at most HEPH_LORA_MAX_ADAPTERS.
 * base and c are the same buffer or do not overlap.
 *
 * heph_lora_plan (one small launch) groups the rows by adapter from the ids in
 * device memory; one plan serves every projection of a step. heph_lora_add
 * takes the M and n_adapters of its plan; with others it writes nothing.
 * plan and ws: device buffers of the two _bytes functions, 16-byte aligned;
 * calls that share a ws are ordered by the caller.
 * No counterpart in the reference.
 */
#define HEPH_LORA_MAX_ADAPTERS 4096
size_t heph_lora_plan_bytes(int M, int n_adapters);
size_t heph_lora_ws_bytes(int M, int n_adapters, int K, int rank);
int heph_lora_plan(void* plan, size_t plan_bytes, const int32_t* ids, int M, int n_adapters,
                   void* stream);
int heph_lora_add(void* c, int c_dtype, const void* base, const uint16_t* x_bf16,
                  const uint16_t* a_bf16, const uint16_t* b_bf16, const float* scale,
                  const void* plan, size_t plan_bytes, void* ws, size_t ws_bytes, int M, int N,
                  int K, int rank, int n_adapters, void* stream);

/*
 * The pick: each row's next token from its logits, after the rules of its
 * request. For row r of logits ([rows, vocab], rows logits_stride elements
 * apart, f32 or bf16) and s = slots[r], the request's place in the rules, in f32:
 *   penalties[s] = (repetition, presence, frequency)
 *   seen t (in history[s][0 .. length[s])):  l = l > 0 ? l / repetition
 *                                                      : l * repetition
 *   answered n > 0 times (from n_prompt[s] on): l = l - (n * frequency + presence)
 *   in bias_ids[s][0 .. n_bias[s]):          l = l + bias (of an id that is
 *                                            there twice, its last entry's)
 *   bit t % 32 of masks[mask_ids[r]][t / 32] is 0:  l = -inf
 * tokens[r] is the lowest index of the largest l, NaN left out; -1 if none is
 * above -inf. logprob[r] is its log-probability under the softmax of all l:
 * -inf where tokens[r] is -1, NaN where an l is NaN or +inf. out (the type of
 * logits, rows out_stride apart; may be logits itself with the same stride, and
 * overlaps it in no other way) gets the l's, rounded once. Each of tokens, logprob and
 * out may be NULL, but not tokens and out both; with flags HEPH_PICK_APPEND (tokens not
 * NULL) a token >= 0 is then written behind its request's history while that has
 * room, and length[s] grows by one; the rows' slots are then distinct.
 * A row has no rules if rules or slots is NULL or its slot is outside
 * [0, n_slots); no mask if masks or mask_ids is NULL or its id is outside [0, n_masks).
 *
 * heph_token_rules: device pointers, row by row: history [n_slots][max_tokens],
 * bias_ids and bias [n_slots][max_bias] (bias_ids, bias and n_bias may be NULL
 * with max_bias 0), masks [n_masks][(vocab + 31) / 32]. max_tokens up to
 * 262144, max_bias up to HEPH_PICK_MAX_BIAS. Lengths are clamped to their
 * buffers on the device, ids outside the vocabulary are passed over.
 * ws: heph_pick_ws_bytes(rows, vocab) bytes (which are enough for fewer rows and
 * smaller vocabularies too), 16-byte aligned; calls that share it are ordered by
 * the caller.
 * Replaces, for a batch with rules, argmax (src/hephaestus/kernels.mojo:1376-1433),
 * which rounds logits to bf16 first.
 */
#define HEPH_PICK_APPEND 0x1
#define HEPH_PICK_MAX_BIAS 4095
typedef struct heph_token_rules {
    int n_slots, max_tokens, max_bias;
    int32_t* history;
    int32_t* length;
    const int32_t* n_prompt;
    const float* penalties;
    const int32_t* bias_ids;
    const float* bias;
    const int32_t* n_bias;
} heph_token_rules;
size_t heph_pick_ws_bytes(int rows, int vocab);
int heph_pick_tokens(int32_t* tokens, float* logprob, void* out, int64_t out_stride,
                     const void* logits, int64_t logits_stride, int dtype, int rows, int vocab,
                     const heph_token_rules* rules, const int32_t* slots, const uint32_t* masks,
                     int n_masks, const int32_t* mask_ids, int flags, void* ws, size_t ws_bytes,
                     void* stream);

#ifdef __cplusplus
}
#endif

#endif /* HEPHSERVE_H */
