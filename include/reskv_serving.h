/* Operators for serving sequences of different lengths: causal attention of packed
 * prompts, and a paged cache of 4-bit keys and values with the attention that reads it.
 *
 * They stand beside the prompt attention of reskv_llama.h (equal lengths) and the
 * decode calls of reskv_hip.h (clustered or dense fp16 caches, one length for the
 * whole batch); the reference has no counterpart.
 *
 * Conventions as in reskv_hip.h: fp16 tensors are passed as void*, every call returns
 * 0 on success and non-zero on error (reskv_last_error() says why), `stream` is a
 * hipStream_t, nothing is allocated and nothing synchronises.  Offsets, lengths and
 * page tables are int32 in device memory; what they hold is bounds-checked by the
 * kernels: offsets are clamped into their tensors, lengths to the table's capacity, and a
 * page number outside the pool stands for tokens that are not there.
 *
 * Pages.  A pool holds `pages` pages; a page is [Hk][page_tokens / 32] blocks of 32
 * tokens of one KV head, RESKV_INT4_BLOCK_BYTES each.  Every token's row of 128 channels
 * is four groups of 32; a group has a lowest value `low` and a `scale`, both fp16, and a
 * value is code * scale + low with codes 0 .. 15.  A block is, in order (t: token of the
 * block, c: channel, g = c / 32; nibble(e) of eight values e = 0 .. 7: e / 2 + 4 (e % 2)):
 *   K codes    2048 B, dword ((t/16 * 4 + c%32/8) * 16 + t%16) * 4 + g, nibble(c % 8)
 *   K scaling   512 B, dword (t/16 * 4 + g) * 16 + t%16: scale, then low
 *   V codes    2048 B, dword (c/64 * 64 + t/8 * 16 + c%16) * 4 + c/16%4, nibble(t % 8)
 *   V scale     256 B, half g * 32 + t
 *   V low       256 B, half g * 32 + t
 * which is the order in which the lanes of a wave take them as operands of the matrix cores. */
#ifndef RESKV_SERVING_H
#define RESKV_SERVING_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define RESKV_INT4_BLOCK_BYTES 5120 /* 32 tokens x (64 + 16) bytes, K and V */

/* Causal attention of S packed sequences.  Sequence s has the query rows
 * [q_offsets[s], q_offsets[s+1]) and the key rows [k_offsets[s], k_offsets[s+1]);
 * with nq and nk of them, query i sees the keys 0 .. i + nk - nq (none: zeros).
 * q fp16 [Nq, Hq, 128], k, v [Nk, Hk, 128]: strides[0..5] are the token and head strides of q,
 * k and v in elements (channel stride 1, rows 16-byte aligned, token strides below 2^23, those of k and v
 * at least 128);
 * out [Nq, Hq, 128] contiguous.  Query rows of no sequence are left as they are, or set to
 * zero with clear_rest.  max_keys bounds the keys of a sequence (it only steers how the work
 * is split); workspace as reskv_packed_workspace_bytes says (may be NULL when that is 0). */
int64_t reskv_packed_workspace_bytes(int S, int64_t Nq, int Hq, int Hk, int64_t max_keys);
int reskv_packed_attention(const void* q, const void* k, const void* v, void* out, const int32_t* q_offsets,
                           const int32_t* k_offsets, int S, int64_t Nq, int64_t Nk, int Hq, int Hk,
                           const int64_t* strides, float scaling, int64_t max_keys, int clear_rest, void* workspace,
                           int64_t workspace_bytes, void* stream);

/* Quantises rows of k and v (fp16 [N, Hk, 128]; strides[0..3] the token and head strides of k and v)
 * into pages: row offsets[s] + i becomes token starts[s] + i of sequence s, whose pages are
 * table[s * table_width ...].  offsets NULL: one row per sequence (N == S).  A group that holds a
 * value that is not finite is stored as NaN.  Rows of no sequence or page are left out.  Two
 * sequences of one call must not write to the same page. */
int reskv_int4_append(void* pages, int64_t num_pages, int page_tokens, int Hk, const int32_t* table, int table_width,
                      int S, const int32_t* starts, const int32_t* offsets, const void* k, const void* v, int64_t N,
                      const int64_t* strides, void* stream);

/* The way back: rows k_out, v_out fp16 [N, Hk, 128] (contiguous), fp16(code * scale + low) of the same
 * tokens.  Rows of no sequence or page are left as they are, or set to zero with clear_rest. */
int reskv_int4_gather(const void* pages, int64_t num_pages, int page_tokens, int Hk, const int32_t* table,
                      int table_width, int S, const int32_t* starts, const int32_t* offsets, void* k_out, void* v_out,
                      int64_t N, int clear_rest, void* stream);

/* One token of each of B sequences: q fp16 [B, Hq, 128] against the first lengths[b] tokens of
 * sequence b, out fp16 [B, Hq, 128] (zeros for a sequence without tokens), both contiguous.
 * max_length bounds the lengths (longer ones are clamped to it); the workspace is always needed. */
int64_t reskv_int4_workspace_bytes(int B, int Hq, int Hk, int64_t max_length);
int reskv_int4_attention(const void* q, const void* pages, int64_t num_pages, int page_tokens, const int32_t* table,
                         int table_width, const int32_t* lengths, int B, int Hq, int Hk, float scaling,
                         int64_t max_length, void* out, void* workspace, int64_t workspace_bytes, void* stream);

/* Copies page source[i] to page target[i] in each of `layers` pools of num_pages pages of
 * page_bytes bytes (a multiple of 16) that lie one behind the other.  source and target are
 * host arrays; no target may be a source or occur twice. */
int reskv_copy_pages(void* pages, int layers, int64_t num_pages, int64_t page_bytes, const int32_t* source,
                     const int32_t* target, int n, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* RESKV_SERVING_H */
