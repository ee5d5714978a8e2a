/*
 * hephserve.h - the ops of a batched serving step around the W8A8 linears:
 * q/k norm + rotation into a paged KV cache, attention of a batch over that
 * cache with shared prefixes computed once, page copies, and the low-rank
 * adapters of many requests beside one projection. Same conventions as
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

#ifdef __cplusplus
}
#endif

#endif /* HEPHSERVE_H */
