// extern "C" entry points of draft verification (declared in include/tv_draft.h).
// Host-side validation lives here; kernels assume validated arguments.
#include <algorithm>

#include "../../include/tv_draft.h"
#include "tv_device_cache.h"
#include "tv_draft.h"
#include "tv_error.h"

namespace {

using tv::check_launch;
using tv::fail;
using tv::ok;

static_assert(TV_DRAFT_MAX_NODES == tv::kDraftMaxNodes, "nodes");

bool valid_dtype(int d) { return d == TV_F32 || d == TV_F16 || d == TV_BF16; }
bool valid_head_dim(int d) { return d == 64 || d == 128 || d == 256; }
bool aligned(const void* p, int n) { return (uintptr_t)p % n == 0; }
int elem_size(int dtype) { return dtype == TV_F32 ? 4 : 2; }
int log2_or_minus1(int x) { return (x & (x - 1)) ? -1 : __builtin_ctz(x); }

// The arguments that every call over trees shares; blocks: whether it has a block table.
int check_trees(const char* who, int num_seqs, int nodes) {
  if (num_seqs < 0 || num_seqs > 65535) return fail(TV_EINVAL, "%s: num_seqs %d outside 0..65535", who, num_seqs);
  if (nodes < 1 || nodes > TV_DRAFT_MAX_NODES)
    return fail(TV_EINVAL, "%s: nodes %d outside 1..%d", who, nodes, TV_DRAFT_MAX_NODES);
  return TV_OK;
}

tv::TreeShapeInfo tree_info(long long rows, int head_dim, int dtype) {
  return dtype == TV_F32   ? tv::tree_info_f32(rows, head_dim)
         : dtype == TV_F16 ? tv::tree_info_f16(rows, head_dim)
                           : tv::tree_info_bf16(rows, head_dim);
}

int check_blocks(const char* who, int bt_stride, int block_size, int num_blocks) {
  if (bt_stride <= 0 || block_size <= 0 || num_blocks <= 0)
    return fail(TV_EINVAL, "%s: bad block table or cache (table width %d, block_size %d, num_blocks %d)", who, bt_stride,
                block_size, num_blocks);
  if ((long long)num_blocks * block_size > 0x7fffffffLL)
    return fail(TV_EINVAL, "%s: %d blocks of %d have slots past 32 bits", who, num_blocks, block_size);
  return TV_OK;
}

}  // namespace

extern "C" {

int tv_draft_tree_layout(uint64_t* mask, int32_t* positions, int32_t* slots, const int32_t* parents,
                         const int32_t* tree_lens, const int32_t* context_lens, const int32_t* block_tables,
                         int num_seqs, int nodes, int bt_stride, int block_size, int num_blocks, void* stream) {
  const char* who = "tv_draft_tree_layout";
  int rc = check_trees(who, num_seqs, nodes);
  if (rc == TV_OK) rc = check_blocks(who, bt_stride, block_size, num_blocks);
  if (rc != TV_OK) return rc;
  if (num_seqs == 0) return ok();
  if (!mask || !positions || !slots || !parents || !tree_lens || !context_lens || !block_tables)
    return fail(TV_EINVAL, "%s: null pointer argument", who);
  if (!aligned(mask, 8) || !aligned(positions, 4) || !aligned(slots, 4) || !aligned(parents, 4) ||
      !aligned(tree_lens, 4) || !aligned(context_lens, 4) || !aligned(block_tables, 4))
    return fail(TV_EINVAL, "%s: misaligned pointer", who);
  tv::DraftLayoutParams p{};
  p.mask = reinterpret_cast<tv::u64*>(mask);
  p.positions = positions;
  p.slots = slots;
  p.parents = parents;
  p.tree_lens = tree_lens;
  p.context_lens = context_lens;
  p.block_tables = block_tables;
  p.num_seqs = num_seqs;
  p.nodes = nodes;
  p.words = (nodes + 63) / 64;
  p.bt_stride = bt_stride;
  p.block_size = block_size;
  p.num_blocks = num_blocks;
  tv::launch_draft_layout(p, reinterpret_cast<hipStream_t>(stream));
  return check_launch(who);
}

int tv_rope_and_cache(void* q_out, void* k_cache, void* v_cache, const void* q, const void* k, const void* v,
                      const int32_t* slots, const int32_t* positions, const float* rope, int rope_len, int rope_dim,
                      int halves, int num_tokens, int num_heads, int num_kv_heads, int head_dim, int block_size,
                      int num_blocks, int64_t q_out_stride, int64_t q_stride, int64_t k_stride, int64_t v_stride,
                      int dtype, uint32_t* err_count, void* stream) {
  const char* who = "tv_rope_and_cache";
  if (!valid_dtype(dtype)) return fail(TV_EINVAL, "%s: bad dtype %d", who, dtype);
  if (num_tokens < 0) return fail(TV_EINVAL, "%s: num_tokens %d", who, num_tokens);
  if (num_heads <= 0 || num_kv_heads <= 0 || head_dim <= 0 || head_dim > 4096 || num_heads > 4096 || num_kv_heads > 4096)
    return fail(TV_EINVAL, "%s: bad heads (%d, %d of %d)", who, num_heads, num_kv_heads, head_dim);
  int rc = check_blocks(who, 1, block_size, num_blocks);
  if (rc != TV_OK) return rc;
  if (rope_len <= 0 || rope_dim < 2 || rope_dim % 2 || rope_dim > head_dim)
    return fail(TV_EINVAL, "%s: rope table of %d positions for %d of %d elements (an even number of them)", who, rope_len,
                rope_dim, head_dim);
  const long long q_row = (long long)num_heads * head_dim, kv_row = (long long)num_kv_heads * head_dim;
  if (q_stride < q_row || q_out_stride < q_row || k_stride < kv_row || v_stride < kv_row)
    return fail(TV_EINVAL, "%s: token stride smaller than a row", who);
  if (num_tokens == 0) return ok();
  if (!q_out || !k_cache || !v_cache || !q || !k || !v || !slots || !positions || !rope)
    return fail(TV_EINVAL, "%s: null pointer argument", who);
  const int es = elem_size(dtype);
  if (!aligned(q_out, es) || !aligned(k_cache, es) || !aligned(v_cache, es) || !aligned(q, es) || !aligned(k, es) ||
      !aligned(v, es) || !aligned(slots, 4) || !aligned(positions, 4) || !aligned(rope, 8))
    return fail(TV_EINVAL, "%s: misaligned pointer", who);
  if (num_tokens >= 1 << 24) return fail(TV_EINVAL, "%s: grid too large", who);   // 256 threads each in one dimension
  // 16-byte vectors where every row, and what is rotated of it, is made of whole ones
  const int vec = 16 / es;
  const bool wide = aligned(q_out, 16) && aligned(k_cache, 16) && aligned(v_cache, 16) && aligned(q, 16) &&
                    aligned(k, 16) && aligned(v, 16) && q_out_stride % vec == 0 && q_stride % vec == 0 &&
                    k_stride % vec == 0 && v_stride % vec == 0 && head_dim % vec == 0 &&
                    rope_dim % (halves ? 2 * vec : vec) == 0;
  if (!wide && !halves && head_dim % 2) return fail(TV_EUNSUPPORTED, "%s: odd head_dim %d with adjacent pairs", who, head_dim);
  tv::RopeCacheParams p{};
  p.q_out = q_out;
  p.k_cache = k_cache;
  p.v_cache = v_cache;
  p.q = q;
  p.k = k;
  p.v = v;
  p.slots = slots;
  p.positions = positions;
  p.rope = rope;
  p.rope_len = rope_len;
  p.rope_dim = rope_dim;
  p.num_tokens = num_tokens;
  p.num_heads = num_heads;
  p.num_kv_heads = num_kv_heads;
  p.head_dim = head_dim;
  p.num_slots = (long long)num_blocks * block_size;
  p.q_out_stride = q_out_stride;
  p.q_stride = q_stride;
  p.k_stride = k_stride;
  p.v_stride = v_stride;
  p.err_count = err_count;
  tv::launch_rope_cache(p, dtype, halves != 0, wide, reinterpret_cast<hipStream_t>(stream));
  return check_launch(who);
}

size_t tv_paged_tree_workspace_bytes(int num_seqs, int nodes, int num_heads, int num_kv_heads, int head_dim, int dtype,
                                     int work_groups) {
  if (num_seqs <= 0 || nodes <= 0 || num_heads <= 0 || num_kv_heads <= 0 || num_heads % num_kv_heads != 0 ||
      !valid_head_dim(head_dim) || !valid_dtype(dtype) || work_groups <= 0)
    return 0;
  const int rows = tree_info((long long)nodes * (num_heads / num_kv_heads), head_dim, dtype).tile_rows;
  const size_t groups = std::max(1, work_groups / num_kv_heads);
  return 2 * groups * num_kv_heads * rows * (head_dim + 2) * sizeof(float) + ((size_t)num_seqs + 1) * sizeof(int);
}

int tv_paged_tree_work_groups(int num_seqs, int nodes, int num_heads, int num_kv_heads, int head_dim, int max_blocks,
                              int block_size, int dtype) {
  const char* who = "tv_paged_tree_work_groups";
  if (num_seqs <= 0 || nodes <= 0 || nodes > TV_DRAFT_MAX_NODES || num_heads <= 0 || num_kv_heads <= 0 ||
      num_heads % num_kv_heads != 0 || max_blocks <= 0 || block_size <= 0 ||
      (long long)max_blocks * block_size > (1LL << 30) || !valid_dtype(dtype))
    return fail(TV_EINVAL, "%s: bad arguments", who), -1;
  if (!valid_head_dim(head_dim))
    return fail(TV_EUNSUPPORTED, "%s: head_dim %d not supported (64/128/256)", who, head_dim), -1;
  const long long rows = (long long)nodes * (num_heads / num_kv_heads);
  const tv::TreeShapeInfo shape = tree_info(rows, head_dim, dtype);
  const long long resident = shape.resident();
  const long long units = (rows + shape.tile_rows - 1) / shape.tile_rows * num_kv_heads * num_seqs;
  const long long tiles = ((long long)max_blocks * block_size + shape.tile_keys - 1) / shape.tile_keys;
  // In tiles that a work-group takes one after the other: undealt, its rounds of whole units; dealt, its share and
  // what dealing and joining cost (8 us).  Long units are dealt in any case: their lengths are rarely equal, and few of them end a
  // launch on a few CUs; a batch that fills the card gains nothing by it.  MI355X, us, undealt / dealt, 32 / 8 heads of 128 in fp16: 16 x 8 nodes over 100..500 tokens 15 / 17,
  // over 500..2000 44 / 26; 64 x 8 over 500..1000 41 / 48; 64 x 16 over 512..4096 126 / 125; 256 x 4 over 500..2000
  // 244 / 245, over 512..4096 444 / 430; 32 / 4 heads of 64: 64 x 8 over 200..1000 18 / 21, 1 x 32 over 1000 23 / 15,
  // 1 x 64 over 8000 125 / 25; in fp32 4 x 8 over 17..250 16 / 11.
  const long long cost = dtype == TV_F32 ? 6 : head_dim == 64 ? 12 : 8;
  const long long undealt = (units + resident - 1) / resident * tiles, dealt = units * tiles / resident + cost;
  const bool counted = ((long long)max_blocks * block_size / 16 + 1) * ((rows + 63) / 64) * num_seqs <= 0x7fffffff;
  if (!counted || !(dealt < undealt || tiles >= 6 * cost)) return 0;
  // Two on a CU load as fast as more do and leave fewer parts; only several tiles of rows in 16 bits, which wait for their own
  // arithmetic, take as many as are resident.  MI355X, us, two a CU / all, 32 / 4 heads of 64 over 1000..4000 tokens in fp16:
  // 64 x 8 nodes 38 / 44, 32 x 16 34 / 36, 32 x 32 47 / 48, 32 x 61 over 1000..6000 98 / 93; in fp32 over 500..2000 tokens 16 x 16 38 / 42.
  const long long two = 2LL * std::max(tv::device_cus(), 1);
  return (int)(rows > 128 && dtype != TV_F32 ? resident : std::min(resident, two));
}

int tv_paged_tree(void* out, const void* queries, const void* k_cache, const void* v_cache,
                  const int32_t* block_tables, const int32_t* context_lens, const int32_t* tree_lens,
                  const uint64_t* mask, int mask_shared, int num_seqs, int nodes, int num_heads, int num_kv_heads,
                  int head_dim, int block_size, int num_blocks, int block_table_stride, int max_blocks,
                  int64_t q_seq_stride, int64_t q_node_stride, float scale, int dtype, int out_dtype,
                  int work_groups, void* workspace, size_t workspace_bytes, void* stream) {
  const char* who = "tv_paged_tree";
  int rc = check_trees(who, num_seqs, nodes);
  if (rc == TV_OK) rc = check_blocks(who, block_table_stride, block_size, num_blocks);
  if (rc != TV_OK) return rc;
  if (!valid_dtype(dtype) || !(out_dtype == dtype || out_dtype == TV_F32))
    return fail(TV_EINVAL, "%s: bad dtype %d / out_dtype %d", who, dtype, out_dtype);
  if (num_heads <= 0 || num_kv_heads <= 0 || num_heads % num_kv_heads != 0)
    return fail(TV_EINVAL, "%s: bad head counts (%d, %d)", who, num_heads, num_kv_heads);
  if (!valid_head_dim(head_dim))
    return fail(TV_EUNSUPPORTED, "%s: head_dim %d not supported (64/128/256)", who, head_dim);
  if (max_blocks <= 0 || max_blocks > block_table_stride)
    return fail(TV_EINVAL, "%s: bad block table (stride=%d, max_blocks=%d)", who, block_table_stride, max_blocks);
  const long long width = (long long)max_blocks * block_size;
  if (width > (1LL << 30)) return fail(TV_EINVAL, "%s: context width too large", who);
  if (work_groups < 0 || work_groups > 1 << 16)
    return fail(TV_EINVAL, "%s: work_groups %d outside 0..%d", who, work_groups, 1 << 16);
  if ((long long)block_size * num_kv_heads * head_dim * elem_size(dtype) > 0x7fffffffLL)
    return fail(TV_EUNSUPPORTED, "%s: blocks of 2 GiB and more", who);
  const int vec = 16 / elem_size(dtype);
  if (q_node_stride < (int64_t)num_heads * head_dim || q_node_stride % vec || q_seq_stride % vec ||
      (num_seqs > 1 && q_seq_stride < 0))
    return fail(TV_EINVAL, "%s: query strides must cover a token's heads and be multiples of 16 bytes", who);
  if (num_seqs == 0) return ok();
  if (!out || !queries || !k_cache || !v_cache || !block_tables || !context_lens || !tree_lens || !mask)
    return fail(TV_EINVAL, "%s: null pointer argument", who);
  if (!aligned(out, 16) || !aligned(queries, 16) || !aligned(k_cache, 16) || !aligned(v_cache, 16) || !aligned(mask, 8) ||
      !aligned(block_tables, 4) || !aligned(context_lens, 4) || !aligned(tree_lens, 4))
    return fail(TV_EINVAL, "%s: queries, caches and out must be 16-byte aligned, the mask 8-byte aligned", who);
  const size_t need = tv_paged_tree_workspace_bytes(num_seqs, nodes, num_heads, num_kv_heads, head_dim, dtype, work_groups);
  if (work_groups && (!workspace || workspace_bytes < need || !aligned(workspace, 16)))
    return fail(TV_EINVAL, "%s: workspace of %zu bytes, 16-byte aligned, required (got %zu)", who, need, workspace_bytes);
  const long long rows = (long long)nodes * (num_heads / num_kv_heads);
  const long long units = (rows + 63) / 64 * num_kv_heads * num_seqs;
  // 256 threads each in one dimension of fewer than 2^32; tiles are counted in 32 bits
  if (num_kv_heads > 65535 || rows > 1 << 22 || units >= 1 << 23 ||
      (work_groups && (width / 16 + 1) * (units / num_kv_heads) > 0x7fffffff))
    return fail(TV_EINVAL, "%s: grid too large", who);
  tv::TreeParams p{};
  p.out = out;
  p.q = queries;
  p.k_cache = k_cache;
  p.v_cache = v_cache;
  p.block_tables = block_tables;
  p.context_lens = context_lens;
  p.tree_lens = tree_lens;
  p.mask = reinterpret_cast<const tv::u64*>(mask);
  p.num_seqs = num_seqs;
  p.nodes = nodes;
  p.words = (nodes + 63) / 64;
  p.mask_seq_stride = mask_shared ? 0 : (long long)nodes * p.words;
  p.q_seq_stride = q_seq_stride;
  p.q_node_stride = q_node_stride;
  p.num_kv_heads = num_kv_heads;
  p.group = num_heads / num_kv_heads;
  p.block_size = block_size;
  p.bs_log2 = log2_or_minus1(block_size);
  p.num_blocks = num_blocks;
  p.bt_stride = block_table_stride;
  p.width = (int)width;
  p.scale = scale;
  p.out_dtype = out_dtype;
  p.work_groups = work_groups;
  p.least_tiles = dtype == TV_F32 ? 1 : 2;   // 4 x 8 nodes over 500..1000 tokens (32 / 8 heads of 128, fp16), us: 1 16.3, 2 15.0, 4 16.9
  p.part_o = reinterpret_cast<float*>(workspace);
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (dtype == TV_F32) tv::launch_tree_f32(p, head_dim, s);
  else if (dtype == TV_F16) tv::launch_tree_f16(p, head_dim, s);
  else tv::launch_tree_bf16(p, head_dim, s);
  return check_launch(who);
}

size_t tv_verify_draft_tree_workspace_bytes(int num_seqs, int nodes, int vocab, int dtype) {
  if (num_seqs <= 0 || nodes <= 0 || nodes > TV_DRAFT_MAX_NODES || vocab <= 0 || !valid_dtype(dtype)) return 0;
  return tv::verify_workspace_bytes(num_seqs, nodes, vocab, dtype);
}

int tv_verify_draft_tree(int32_t* path, int32_t* counts, int32_t* next_tokens, const void* logits,
                         const int32_t* tokens, const int32_t* parents, const int32_t* tree_lens,
                         const float* temperatures, const float* uniforms, int num_seqs, int nodes, int vocab,
                         int64_t row_stride, int dtype, void* workspace, size_t workspace_bytes, void* stream) {
  const char* who = "tv_verify_draft_tree";
  int rc = check_trees(who, num_seqs, nodes);
  if (rc != TV_OK) return rc;
  if (!valid_dtype(dtype)) return fail(TV_EINVAL, "%s: bad dtype %d", who, dtype);
  if (vocab < 1 || vocab > 1 << 24 || row_stride < vocab)
    return fail(TV_EINVAL, "%s: bad shape (vocab %d, row stride %lld)", who, vocab, (long long)row_stride);
  if (num_seqs == 0) return ok();
  if (!path || !counts || !next_tokens || !logits || !tokens || !parents || !tree_lens)
    return fail(TV_EINVAL, "%s: null pointer argument", who);
  if (temperatures && !uniforms) return fail(TV_EINVAL, "%s: temperatures without uniforms", who);
  if (!aligned(path, 4) || !aligned(counts, 4) || !aligned(next_tokens, 4) || !aligned(logits, elem_size(dtype)) ||
      !aligned(tokens, 4) || !aligned(parents, 4) || !aligned(tree_lens, 4) || !aligned(temperatures, 4) ||
      !aligned(uniforms, 4))
    return fail(TV_EINVAL, "%s: misaligned pointer", who);
  const size_t need = tv::verify_workspace_bytes(num_seqs, nodes, vocab, dtype);
  if (need && (!workspace || workspace_bytes < need || !aligned(workspace, 16)))
    return fail(TV_EINVAL, "%s: workspace of %zu bytes, 16-byte aligned, required (got %zu)", who, need, workspace_bytes);
  tv::VerifyParams p{};
  p.path = path;
  p.counts = counts;
  p.next_tokens = next_tokens;
  p.logits = logits;
  p.tokens = tokens;
  p.parents = parents;
  p.tree_lens = tree_lens;
  p.temperatures = temperatures;
  p.uniforms = uniforms;
  p.num_seqs = num_seqs;
  p.nodes = nodes;
  p.vocab = vocab;
  p.row_stride = row_stride;
  p.workspace = workspace;
  tv::launch_verify(p, dtype, reinterpret_cast<hipStream_t>(stream));
  return check_launch(who);
}

int tv_keep_draft_rows(void* const* k_caches, void* const* v_caches, int num_layers, const int32_t* path,
                       const int32_t* counts, const int32_t* context_lens, const int32_t* block_tables, int num_seqs,
                       int nodes, int bt_stride, int num_kv_heads, int head_dim, int block_size, int num_blocks,
                       int dtype, void* stream) {
  const char* who = "tv_keep_draft_rows";
  int rc = check_trees(who, num_seqs, nodes);
  if (rc == TV_OK) rc = check_blocks(who, bt_stride, block_size, num_blocks);
  if (rc != TV_OK) return rc;
  if (!valid_dtype(dtype)) return fail(TV_EINVAL, "%s: bad dtype %d", who, dtype);
  if (num_layers < 0 || num_kv_heads <= 0 || head_dim <= 0 || (long long)num_kv_heads * head_dim > 1 << 20)
    return fail(TV_EINVAL, "%s: bad cache shape (%d layers, %d heads of %d)", who, num_layers, num_kv_heads, head_dim);
  if (num_seqs == 0 || num_layers == 0) return ok();
  if (!k_caches || !v_caches || !path || !counts || !context_lens || !block_tables)
    return fail(TV_EINVAL, "%s: null pointer argument", who);
  if (!aligned(path, 4) || !aligned(counts, 4) || !aligned(context_lens, 4) || !aligned(block_tables, 4))
    return fail(TV_EINVAL, "%s: misaligned pointer", who);
  const long long row = (long long)num_kv_heads * head_dim * elem_size(dtype);
  int vec = 16;
  for (int i = 0; i < num_layers; ++i) {
    if (!k_caches[i] || !v_caches[i]) return fail(TV_EINVAL, "%s: null pointer argument (layer %d)", who, i);
    if (!aligned(k_caches[i], elem_size(dtype)) || !aligned(v_caches[i], elem_size(dtype)))
      return fail(TV_EINVAL, "%s: misaligned cache (layer %d)", who, i);
    while (row % vec || !aligned(k_caches[i], vec) || !aligned(v_caches[i], vec)) vec /= 2;
  }
  tv::KeepParams p{};
  p.path = path;
  p.counts = counts;
  p.context_lens = context_lens;
  p.block_tables = block_tables;
  p.num_seqs = num_seqs;
  p.nodes = nodes;
  p.bt_stride = bt_stride;
  p.row_vecs = (int)(row / vec);
  p.block_size = block_size;
  p.num_blocks = num_blocks;
  for (int at = 0; at < num_layers; at += tv::kKeepLayers) {
    const int n = std::min(tv::kKeepLayers, num_layers - at);
    for (int i = 0; i < n; ++i) {
      p.k[i] = k_caches[at + i];
      p.v[i] = v_caches[at + i];
    }
    tv::launch_keep(p, n, vec, reinterpret_cast<hipStream_t>(stream));
  }
  return check_launch(who);
}

}  // extern "C"
