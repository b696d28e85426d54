/*
 * mesh_moe_cache.h -- C ABI of the part of libmesh_moe_hip.so that keeps the keys and
 * values of sequences in pages: writing rows, reading them back, and attention of one new
 * token over them.
 *
 * The conventions are those of mesh_moe.h: device pointers owned by the caller, one
 * asynchronous call on `stream`, 0 or a negative MESH_MOE_E_* code, the reason from
 * mesh_moe_last_error().  Nothing is allocated or kept between calls: every call can be
 * recorded into a HIP graph, and calls on different streams do not meet unless they share
 * a workspace, an output or pages.
 *
 * A cache is
 *   k_pages, v_pages [N,HK,S,D]  N pages of S rows (S a power of two) for each of HK key /
 *                      value heads of D values: of `dtype`, or e4m3 numbers where k_scales
 *                      and v_scales are given
 *   k_scales, v_scales [N,HK,S,DB]  a byte for each block of 128 values of a row, DB = D /
 *                      128 rounded up (a row's last block may be shorter), or both NULL.
 *                      Value i of a row stands for page[i] * 2^(scale[i / 128] - 127);
 *                      exponents, roundings and blocks that are not finite as in
 *                      mesh_moe_fp8.h.  Bytes from 10 to 254 are taken; the calls make
 *                      these.
 * (v_pages NULL: keys and values are the same tensor, mesh_tensorflow/transformer/
 * attention.py:499-515; v_scales is NULL then, too.)  Where a sequence's rows lie is told
 * by
 *   table [B,P] int32  position p of sequence b is row p % S of page table[b][p / S]
 * Entries outside 0 .. N - 1 are pages that are not there, and so are all positions from P
 * * S on: rows for them are not written, read as zeros, and are not attended to.  A page may
 * be named several times, by sequences or by one, where the rows that they have of it are
 * only read; what a call leaves in a row that it is told to write twice, or reads of a row
 * that it writes for another place of the table, is unspecified.
 *
 * Limits: D up to 256, HK up to 65536, T and P * S up to 2^30.  Attention of H query heads
 * takes B * H up to 2^24 - 1 with D below 16.  From 16 on it takes U = B * HK * (H / HK / 16
 * rounded up) up to that, and U * (P * S / R + 1, rounded up) up to 2^31 - 1; R is 256 for
 * 8-bit pages with bfloat16 queries and D up to 128, and 64 or 128 otherwise.  The buffers
 * of a cache do not overlap each other.  Tensors lie on their elements' size; the calls are
 * fastest on 16 bytes, with D of 64, 128 or 256 and pages of 16 rows and more.
 *
 * The reference keeps recurrent states as whole tensors (mesh_tensorflow/transformer/
 * transformer_layers.py:231-254); these calls are a form of what it does with them.
 */
#ifndef MESH_MOE_CACHE_H_
#define MESH_MOE_CACHE_H_

#include "mesh_moe.h"

#ifdef __cplusplus
extern "C" {
#endif

/* (counted up with every change of a declaration, and of what a call accepts) */
#define MESH_MOE_CACHE_ABI_VERSION 2

int mesh_moe_cache_abi_version(void);

/*
 * Rows of keys and values into a cache: row t of sequence b becomes position
 * position[b] + t.
 *   k, v [B,T,HK*D] dtype (v NULL together with v_pages)
 *   position [B] int32 (rows for positions below 0 are not written)
 *   count [B] int32 or NULL: only the first count[b] rows (clamped to 0 .. T); the others
 *     are not read
 */
int mesh_moe_cache_write(const void* k, const void* v, const int32_t* table,
                         const int32_t* position, const int32_t* count, void* k_pages,
                         void* v_pages, uint8_t* k_scales, uint8_t* v_scales, int B,
                         int T, int HK, int D, int N, int S, int P, int dtype,
                         void* stream);

/*
 * The way back: row t of sequence b is what position position[b] + t stands for, exact in
 * float32 and bfloat16; zeros from count[b] on, and for positions that are not there.
 *   k, v [B,T,HK*D] dtype (v NULL together with v_pages)
 */
int mesh_moe_cache_read(const void* k_pages, const void* v_pages,
                        const uint8_t* k_scales, const uint8_t* v_scales,
                        const int32_t* table, const int32_t* position,
                        const int32_t* count, void* k, void* v, int B, int T, int HK,
                        int D, int N, int S, int P, int dtype, void* stream);

/*
 * One decoding step of self-attention over a cache (mesh_moe_attention_decode is its form
 * on whole tensors): the query of sequence b sees its positions 0 .. position[b], as many
 * of them as are there.  H query heads in HK groups of H / HK that follow each other; a
 * group shares a key / value head.
 *   logit[h][j] = q[h] . k[j] + rel_values[h][rel_bucket[j - position[b] + reach - 1]]
 *   out[h] = sum_j w[h][j] v[j] with the softmax w of the logits over j
 * The logits, the softmax and its sums are float32; with bfloat16 the weights are rounded
 * to it, unnormalised, and the sum of those that were multiplied divides the result.
 * out[h] is 0 where nothing is seen (position[b] < 0) or all logits are -infinity.
 * Calls with the same sizes and positions give the same bits; a sequence's last bits may
 * depend on the others' lengths, by which its sums are divided.
 *   q, out [B,H*D] dtype
 *   k_new, v_new [B,HK*D] dtype or NULL: the step's own row, written to position[b] first
 *     (mesh_moe_cache_write with T = 1); v_new is NULL also where v_pages is
 *   rel_values [H,num_buckets] dtype and rel_bucket [2*reach-1] int32, or both NULL: a
 *     relative attention bias as in mesh_moe_attention_decode; positions farther than
 *     reach - 1 back have the bias of that distance
 *   workspace: mesh_moe_cache_attention_workspace_bytes bytes, which may be 0 (and are for
 *     sizes that the call refuses)
 */
size_t mesh_moe_cache_attention_workspace_bytes(int B, int H, int HK, int D, int S,
                                                int P, int dtype, int eight_bit);
int mesh_moe_cache_attention(const void* q, const void* k_new, const void* v_new,
                             void* k_pages, void* v_pages, uint8_t* k_scales,
                             uint8_t* v_scales, const int32_t* table,
                             const int32_t* position, const void* rel_values,
                             const int32_t* rel_bucket, int num_buckets, int reach,
                             void* out, int B, int H, int HK, int D, int N, int S, int P,
                             int dtype, void* workspace, size_t workspace_bytes,
                             void* stream);

#ifdef __cplusplus
}
#endif
#endif  /* MESH_MOE_CACHE_H_ */
