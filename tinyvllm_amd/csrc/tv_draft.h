// Launch parameter blocks of draft verification (include/tv_draft.h).
#pragma once

#include "tv_common.h"

namespace tv {

constexpr int kDraftMaxNodes = 256;
constexpr int kKeepLayers = 64;          // layers of one launch (their pointers are kernel arguments)

typedef unsigned long long u64;

struct DraftLayoutParams {
  u64* mask;                 // [B, nodes, words]
  int* positions;            // [B, nodes]
  int* slots;
  const int* parents;
  const int* tree_lens;      // [B]
  const int* context_lens;
  const int* block_tables;   // [B, bt_stride]
  int num_seqs, nodes, words, bt_stride, block_size, num_blocks;
};

struct RopeCacheParams {
  void* q_out;
  void* k_cache;             // [NB, bs, Hkv, D]
  void* v_cache;
  const void* q;
  const void* k;
  const void* v;
  const int* slots;
  const int* positions;
  const float* rope;         // [rope_len, rope_dim / 2, 2]
  int rope_len, rope_dim;
  int num_tokens, num_heads, num_kv_heads, head_dim;
  long long num_slots;
  long long q_out_stride, q_stride, k_stride, v_stride;   // elements between tokens
  unsigned* err_count;       // may be null
};

struct TreeParams {
  void* out;                 // [B, nodes, Hq, D] in out_dtype
  const void* q;
  const void* k_cache;       // [NB, bs, Hkv, D]
  const void* v_cache;
  const int* block_tables;   // [B, bt_stride]
  const int* context_lens;
  const int* tree_lens;
  const u64* mask;
  long long mask_seq_stride; // words between sequences (0: one mask for all)
  long long q_seq_stride, q_node_stride;   // elements
  int num_seqs, nodes, words, num_kv_heads, group;
  int block_size, bs_log2;   // log2 or -1
  int num_blocks, bt_stride;
  int width;                 // max_blocks * block_size
  float scale;
  int out_dtype;
  int row_tiles;
  // 0: a work-group per row tile of a (sequence, KV head).  Else the key tiles of all sequences' row tiles, one after the
  // other, are dealt evenly to groups, at least least_tiles each; a group is a work-group for every KV head.  A second
  // kernel joins what is cut.
  int work_groups, groups, least_tiles;
  int tile_rows, tile_keys;
  float* part_o;             // [work_groups, 2, tile_rows, D] normalised parts: of a work-group's first unit, of a later one
  float* part_ml;            // [work_groups, 2, tile_rows, 2] (max in log2 units, sum)
  int* first_tiles;          // [B + 1] tiles of the sequences before; then the tiles of a group
};

struct VerifyParams {
  int* path;
  int* counts;
  int* next_tokens;
  const void* logits;
  const int* tokens;
  const int* parents;
  const int* tree_lens;
  const float* temperatures; // may be null
  const float* uniforms;
  int num_seqs, nodes, vocab;
  long long row_stride;
  void* workspace;
  int draw_chunks;           // of a row, for the draw
  int stat_size, stat_parts; // elements of a part, and parts, of a row that is read beforehand (0: none is)
  int chain_rows;            // greedy: work-groups for the rows of a chain (0: all rows are read)
  double unsure;             // sampled: how near to a bound, of the row's sum, fp32 sums do not decide
};

struct KeepParams {
  void* k[kKeepLayers];
  void* v[kKeepLayers];
  const int* path;
  const int* counts;
  const int* context_lens;
  const int* block_tables;
  int num_seqs, nodes, bt_stride, row_vecs, block_size, num_blocks;
};

void launch_draft_layout(const DraftLayoutParams& p, hipStream_t s);
void launch_rope_cache(const RopeCacheParams& p, int dtype, bool halves, bool wide, hipStream_t s);
// The tile of so many rows: its rows, its keys, and the work-groups that are resident at once.
struct TreeShapeInfo {
  int tile_rows, tile_keys;
  long long (*resident)();
};
void launch_tree_f32(const TreeParams& p, int head_dim, hipStream_t s);
void launch_tree_f16(const TreeParams& p, int head_dim, hipStream_t s);
void launch_tree_bf16(const TreeParams& p, int head_dim, hipStream_t s);
TreeShapeInfo tree_info_f32(long long rows, int head_dim);
TreeShapeInfo tree_info_f16(long long rows, int head_dim);
TreeShapeInfo tree_info_bf16(long long rows, int head_dim);
size_t verify_workspace_bytes(int num_seqs, int nodes, int vocab, int dtype);
void launch_verify(VerifyParams p, int dtype, hipStream_t s);
void launch_keep(const KeepParams& p, int layers, int vec_bytes, hipStream_t s);

}  // namespace tv
