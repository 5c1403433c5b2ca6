/* Operators of drafted decoding over the paged 4-bit cache of reskv_serving.h: several tokens of a sequence, a chain
 * or a tree of drafts, go through the model at once, and those that the model agrees with are kept.
 *
 * A tree has up to RESKV_DRAFT_NODES nodes per sequence, parents before children.  Node 0 is its root, the token that
 * was sampled last and is not in the cache yet; the others are drafts.  With `context` tokens before the tree, node
 * i is token context + i of its sequence in the pages, at position context + (its depth).
 *
 * Conventions as in reskv_serving.h: offsets, lengths, tables, parents and paths are int32 in device memory, what they
 * hold is bounds-checked by the kernels, and what lies outside is left out; nothing is allocated and nothing
 * synchronises. */
#ifndef RESKV_DRAFTS_H
#define RESKV_DRAFTS_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define RESKV_DRAFT_NODES 64

/* reskv_int4_append of rows whose keys are rotated to their positions first, with the queries rotated beside them:
 * of every head's first `rotary` channels (a multiple of 16), the pairs (a, b) = (x[i], x[i + rotary / 2]), or
 * (x[2 i], x[2 i + 1]) with `interleaved`, become fp16(a c - b s), fp16(b c + a s), products and sums rounded to fp32,
 * with c = cos[p, i] and s = sin[p, i] (fp32 [rows, rotary / 2], contiguous) of the row's position p: positions[row], or the
 * token's place in its sequence where positions is NULL.  q fp16 [N, Hq, 128] may be NULL; strides[0..5] are the
 * token and head strides of q, k and v; q_out [N, Hq, 128] contiguous.  Rows whose position is outside the tables are not
 * stored; their rows of q_out, and those of no sequence, are left as they are, or set to zero with clear_rest. */
int reskv_int4_append_rope(void* pages, int64_t num_pages, int page_tokens, int Hk, const int32_t* table, int table_width,
                           int S, const int32_t* starts, const int32_t* offsets, const int32_t* positions, const void* q,
                           int Hq, const void* k, const void* v, int64_t N, const int64_t* strides, const float* cos,
                           const float* sin, int rows, int rotary, int interleaved, void* q_out, int clear_rest,
                           void* stream);

/* Masks and positions of trees: node i of sequence s (row offsets[s] + i) has parents[row] < i as its parent (anything
 * else: none).  seen[row] has bit i and the bits of its ancestors; positions[row] = starts[s] + the number of its
 * ancestors.  starts and positions may be NULL.  Rows of no sequence, and nodes from RESKV_DRAFT_NODES on, are left as they are. */
int reskv_draft_tree(const int32_t* parents, const int32_t* offsets, const int32_t* starts, int S, int64_t N, uint64_t* seen,
                     int32_t* positions, void* stream);

/* Attention of the trees' nodes over the pages: sequence s has the rows [offsets[s], offsets[s+1]) of q fp16 [N, Hq, 128]
 * (contiguous), n of them; its first lengths[s] tokens count, the last n of which are the nodes.  A node sees every token
 * before them, and node j where bit j of seen[row] is set (seen NULL: the nodes up to itself).  out [N, Hq, 128]: zeros
 * where a node sees nothing; rows of no sequence and nodes from max_nodes <= RESKV_DRAFT_NODES on are left as they are, or set
 * to zero with clear_rest.  max_length as in reskv_int4_attention; scaling > 0. */
int64_t reskv_int4_tree_workspace_bytes(int S, int64_t N, int Hq, int Hk, int64_t max_length, int max_nodes);
int reskv_int4_tree_attention(const void* q, const void* pages, int64_t num_pages, int page_tokens, const int32_t* table,
                              int table_width, const int32_t* lengths, const int32_t* offsets, const uint64_t* seen, int S,
                              int64_t N, int Hq, int Hk, float scaling, int64_t max_length, int max_nodes, int clear_rest,
                              void* out, void* workspace, int64_t workspace_bytes, void* stream);

/* Which drafts the target model accepts.  logits [N, V] (fp16, or fp32 with logits_fp32; rows row_stride elements apart): row i of
 * a sequence is what the target says behind node i.  The walk starts at the root with r = softmax(logits / temperature) and
 * goes through the nodes in their order; at node x, a child of the node reached, with q the distribution that x's
 * token t was drawn from (draft[row], fp32 [N, V], draft_stride apart; draft NULL: all of it at t):
 *   accept[row] * q(t) < r(t) / sum r: x is reached, and r is its softmax;
 *   else r becomes max(r / sum r - q, 0), or stays where that leaves nothing.
 * temperature is 0, or 1e-30 and more.
 * path[s] [RESKV_DRAFT_NODES] lists the nodes reached, the root first, and -1 behind them; counts[s] says how many;
 * token[s] is the first t with r(0) + .. + r(t) > sample[s] * sum r.  With temperature 0, r has one token, the
 * argmax (the lowest of equals), and accept, sample and draft are not read.  Sums are 64 bits.  A node whose token is outside the
 * vocabulary is passed over.  token[s] = -1 where the row reached has no distribution (a NaN; without temperature 0 also
 * plus infinity, or nothing but minus infinity), and where a sequence has no nodes (then counts[s] = 0). */
int64_t reskv_verify_workspace_bytes(int S, int64_t N, int64_t V);
int reskv_verify_drafts(const void* logits, int logits_fp32, int64_t row_stride, const int64_t* tokens, const int32_t* parents,
                        const int32_t* offsets, const float* accept, const float* sample, const float* draft,
                        int64_t draft_stride, double temperature, int S, int64_t N, int64_t V, int32_t* path, int32_t* counts,
                        int64_t* token, void* workspace, int64_t workspace_bytes, void* stream);

/* The accepted nodes' tokens move together: in each of `layers` pools of num_pages pages that lie one behind the other,
 * token starts[s] + path[s * width + j] of sequence s becomes its token starts[s] + j, for j < counts[s], all of them at
 * once (width <= RESKV_DRAFT_NODES).  Entries outside 0 .. RESKV_DRAFT_NODES - 1, and tokens without a page, are left out.  No
 * two sequences may have these tokens in one page. */
int reskv_int4_keep(void* pages, int layers, int64_t num_pages, int page_tokens, int Hk, const int32_t* table,
                    int table_width, int S, const int32_t* starts, const int32_t* path, int width, const int32_t* counts,
                    void* stream);

#ifdef __cplusplus
}
#endif

#endif /* RESKV_DRAFTS_H */
