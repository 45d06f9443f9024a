/*
 * tv_draft.h -- C ABI of draft verification on MI355X (gfx950): several drafted
 * tokens of every sequence, a tree of them, go through the model at once.  The
 * reference (jonirajala/tinyvllm) decodes one token a step and has no
 * counterpart of these.
 *
 * A tree has up to `nodes` nodes a sequence, tree_lens[b] of them in use.  Node 0
 * is the token that the sequence has last got (its K/V are not cached yet);
 * parents[b, i] is a lower index of the same tree, anything else stands for no
 * parent.  Node i's K/V lie at cache position context_lens[b] + i of the sequence
 * and are rotated to position context_lens[b] + its depth.
 *
 * Conventions are those of tv_attn.h (device pointers but where noted, caller-owned
 * buffers, nothing allocated, stream = hipStream_t, return 0 or a TV_E* code with
 * tv_last_error()).  Lengths are clamped: context_lens below 0 count as 0, tree_lens to
 * 0 .. nodes.  The caches are those of a 16- or 32-bit KVCache: in an 8-bit cache a
 * rejected row would have changed its block's scale.
 */
#ifndef TV_DRAFT_H
#define TV_DRAFT_H

#include <stddef.h>
#include <stdint.h>

#include "tv_attn.h"

#ifdef __cplusplus
extern "C" {
#endif

#define TV_DRAFT_MAX_NODES 256

/*
 * What every node sees, where it stands and where its K/V go.
 *   mask      [num_seqs, nodes, ceil(nodes/64)] uint64: bit t % 64 of word t / 64 is
 *             set for t = i and every ancestor of i
 *   positions [num_seqs, nodes] int32: context_lens[b] + depth
 *   slots     [num_seqs, nodes] int32: slot of position context_lens[b] + i by the
 *             block table; -1 where the table does not reach it or names a block
 *             outside the cache
 * Nodes at tree_lens[b] and beyond get mask 0, position 0 and slot -1.
 * 1 <= nodes <= TV_DRAFT_MAX_NODES; mask 8-byte aligned.
 */
int tv_draft_tree_layout(uint64_t* mask, int32_t* positions, int32_t* slots, const int32_t* parents,
                         const int32_t* tree_lens, const int32_t* context_lens, const int32_t* block_tables,
                         int num_seqs, int nodes, int bt_stride, int block_size, int num_blocks, void* stream);

/*
 * Rotates q and k of num_tokens tokens to their positions and writes k and v into
 * the paged caches [num_blocks, block_size, num_kv_heads, head_dim].
 * q [num_tokens, num_heads, head_dim], k / v [num_tokens, num_kv_heads, head_dim] at
 * strides (elements) between tokens; q_out like q and allowed to be q.
 * rope [rope_len, rope_dim/2, 2] float: cos and sin of pair i at a position.  Pairs are
 * elements (2i, 2i + 1), or with halves != 0 (i, i + rope_dim/2), of the first rope_dim
 * (even, <= head_dim) of a head; the others stay as they are:
 *   (a, b) -> (a cos - b sin, a sin + b cos), in fp32, rounded once.
 * A negative slot is padding: K/V are not written.  A slot past the cache is counted
 * in err_count (may be NULL) and not written.  A position outside [0, rope_len)
 * makes the token's q NaN, is counted, and not written.  Slots of one call differ.
 */
int tv_rope_and_cache(void* q_out, void* k_cache, void* v_cache, const void* q, const void* k, const void* v,
                      const int32_t* slots, const int32_t* positions, const float* rope, int rope_len, int rope_dim,
                      int halves, int num_tokens, int num_heads, int num_kv_heads, int head_dim, int block_size,
                      int num_blocks, int64_t q_out_stride, int64_t q_stride, int64_t k_stride, int64_t v_stride,
                      int dtype, uint32_t* err_count, void* stream);

/*
 * Attention of a tree's nodes over the paged cache:
 *   out[b, i, h] = softmax_j((q[b, i, h] . K[j]) * scale) V[j]
 * over j < context_lens[b] and over j = context_lens[b] + t for the set bits t of
 * mask[b, i] with t < tree_lens[b]; positions past max_blocks * block_size do not
 * exist.  Nodes at tree_lens[b] and beyond, and nodes that see nothing, get zeros.
 * A block id outside the cache, a NaN in K, a score of +inf, or a NaN or infinity in V makes
 * values of the nodes that see it NaN or infinite and reaches no others (a score of -inf
 * has weight 0).  Rows past the tree are not looked at.
 * queries: head rows of head_dim elements, dense in a token; strides in elements
 * between sequences and nodes (multiples of 16 bytes).  mask [num_seqs, nodes,
 * ceil(nodes/64)], or with mask_shared != 0 one [nodes, ceil(nodes/64)] for all.
 * out [num_seqs, nodes, num_heads, head_dim] of dtype or TV_F32 (out_dtype).
 * head_dim 64, 128 or 256; any block size; any number of query heads per KV head.
 * work_groups: 0 gives every (sequence, KV head, tile of rows) a work-group.  n > 0 deals
 * the keys of all of them evenly to n work-groups (as many for every KV head, one at least) by the lengths on the device, and joins what
 * that cuts through `workspace` (16-byte aligned, of tv_paged_tree_workspace_bytes bytes,
 * one per launch that may overlap); results then depend on the batch in their last digits.
 */
size_t tv_paged_tree_workspace_bytes(int num_seqs, int nodes, int num_heads, int num_kv_heads, int head_dim, int dtype,
                                     int work_groups);
/* work_groups for the current device; negative: bad arguments. */
int tv_paged_tree_work_groups(int num_seqs, int nodes, int num_heads, int num_kv_heads, int head_dim, int max_blocks,
                              int block_size, int dtype);
int tv_paged_tree(void* out, const void* queries, const void* k_cache, const void* v_cache,
                  const int32_t* block_tables, const int32_t* context_lens, const int32_t* tree_lens,
                  const uint64_t* mask, int mask_shared, int num_seqs, int nodes, int num_heads, int num_kv_heads,
                  int head_dim, int block_size, int num_blocks, int block_table_stride, int max_blocks,
                  int64_t q_seq_stride, int64_t q_node_stride, float scale, int dtype, int out_dtype,
                  int work_groups, void* workspace, size_t workspace_bytes, void* stream);

/*
 * The path through a tree that the model's logits accept.
 *   path        [num_seqs, nodes] int32: accepted nodes from node 0 on, -1 behind them
 *   counts      [num_seqs] int32: their number (0 for an empty tree)
 *   next_tokens [num_seqs] int32: the token after them (-1 for an empty tree)
 * From node 0 on, greedy (temperatures NULL, or its entry below 2^-126): the path goes to
 * the child, of lowest index, whose token is the first maximum of the node's logits;
 * without one it ends, and the maximum is the next token.  Sampled (entry of at least
 * 2^-126, finite): p = softmax(logits / temperature) and u = uniforms[b, node] in [0, 1); the path
 * goes to the first child at which the children's probabilities sum, in the order
 * of their indexes, to more than u.  Without one the next token is the first at which
 * the probabilities of the tokens that no child has sum to more than (u - c) / (1 - c) of
 * theirs, c being the children's: child or not, a token is drawn with its p.
 * Of children with one token the first counts; a token outside [0, vocab) is never
 * taken.  A node whose logits have a NaN or no number above -inf (sampled: or +inf) ends
 * the path, and the next token is -1.
 * logits [num_seqs * nodes, vocab] of dtype at row_stride elements.  Exponentials and sums are fp32
 * where u is not next to a bound, and else, and for the draw, fp64.  workspace: 16-byte aligned, one per
 * launch that may overlap.
 */
size_t tv_verify_draft_tree_workspace_bytes(int num_seqs, int nodes, int vocab, int dtype);
int tv_verify_draft_tree(int32_t* path, int32_t* counts, int32_t* next_tokens, const void* logits,
                         const int32_t* tokens, const int32_t* parents, const int32_t* tree_lens,
                         const float* temperatures, const float* uniforms, int num_seqs, int nodes, int vocab,
                         int64_t row_stride, int dtype, void* workspace, size_t workspace_bytes, void* stream);

/*
 * Moves the K/V of accepted nodes to where the sequence goes on, in all layers:
 * cache position context_lens[b] + path[b, j] -> context_lens[b] + j for j < counts[b]
 * (clamped to 0 .. nodes).  k_caches / v_caches: host arrays of num_layers device
 * pointers.  path rises from node to node, as tv_verify_draft_tree gives it; an entry
 * outside [j, nodes), or a position that the table does not reach or whose block is outside
 * the cache, is not moved.
 */
int tv_keep_draft_rows(void* const* k_caches, void* const* v_caches, int num_layers, const int32_t* path,
                       const int32_t* counts, const int32_t* context_lens, const int32_t* block_tables, int num_seqs,
                       int nodes, int bt_stride, int num_kv_heads, int head_dim, int block_size, int num_blocks,
                       int dtype, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* TV_DRAFT_H */
