// extern "C" entry points of the 8-bit K/V cache (declared in include/tv_attn.h).
// Host-side validation lives here; kernels assume validated arguments.
#include <algorithm>

#include "../../include/tv_attn.h"
#include "paged_decode.cuh"
#include "tv_device_cache.h"
#include "tv_error.h"
#include "tv_fp8.h"

namespace {

using tv::check_launch;
using tv::fail;
using tv::ok;

bool valid_dtype(int d) { return d == TV_F32 || d == TV_F16 || d == TV_BF16; }
bool valid_head_dim(int d) { return d == 64 || d == 128 || d == 256; }
bool aligned(const void* p, int n) { return (uintptr_t)p % n == 0; }
int log2_or_minus1(int x) { return (x & (x - 1)) ? -1 : __builtin_ctz(x); }

// The arguments that every call on the 8-bit cache shares.
int check_cache(const char* who, const void* k_cache, const void* v_cache, const void* k_scale, const void* v_scale,
                int num_kv_heads, int head_dim, int block_size, int num_blocks, int dtype) {
  if (!k_cache || !v_cache || !k_scale || !v_scale) return fail(TV_EINVAL, "%s: null pointer argument", who);
  if (!valid_dtype(dtype)) return fail(TV_EINVAL, "%s: bad dtype %d", who, dtype);
  if (num_kv_heads <= 0 || head_dim <= 0 || block_size <= 0 || num_blocks <= 0)
    return fail(TV_EINVAL, "%s: bad cache shape (num_blocks=%d, num_kv_heads=%d, block_size=%d, head_dim=%d)", who,
                num_blocks, num_kv_heads, block_size, head_dim);
  if (!valid_head_dim(head_dim))
    return fail(TV_EUNSUPPORTED, "%s: head_dim %d not supported (64/128/256)", who, head_dim);
  if (block_size > tv::kFp8MaxBlock)
    return fail(TV_EUNSUPPORTED, "%s: block_size %d above %d", who, block_size, tv::kFp8MaxBlock);
  if (!aligned(k_cache, 16) || !aligned(v_cache, 16) || !aligned(k_scale, 4) || !aligned(v_scale, 4))
    return fail(TV_EINVAL, "%s: caches must be 16-byte aligned, scales 4-byte aligned", who);
  return TV_OK;
}

int write_common(const char* who, void* k_cache, void* v_cache, float* k_scale, float* v_scale, const void* k,
                 const void* v, const int32_t* slots, int base_slot, int num_tokens, int num_kv_heads, int head_dim,
                 int block_size, int num_blocks, int64_t k_stride, int64_t v_stride, int dtype, uint32_t* err_count,
                 void* stream) {
  if (num_tokens < 0) return fail(TV_EINVAL, "%s: num_tokens %d", who, num_tokens);
  int rc = check_cache(who, k_cache, v_cache, k_scale, v_scale, num_kv_heads, head_dim, block_size, num_blocks, dtype);
  if (rc != TV_OK) return rc;
  const int es = dtype == TV_F32 ? 4 : 2;
  const long long row = (long long)num_kv_heads * head_dim;
  if (k_stride < row || v_stride < row) return fail(TV_EINVAL, "%s: token stride smaller than a row", who);
  if (num_tokens == 0) return ok();
  if (!k || !v) return fail(TV_EINVAL, "%s: null pointer argument", who);
  if (!aligned(k, es) || !aligned(v, es) || (slots && !aligned(slots, 4)))
    return fail(TV_EINVAL, "%s: misaligned input", who);
  // a launch holds fewer than 2^32 threads per dimension: 16 tokens per work-group of 256
  if ((num_kv_heads + 1) / 2 > 65535 || num_tokens >= 1 << 28) return fail(TV_EINVAL, "%s: grid too large", who);
  tv::KVWriteFp8Params p{};
  p.k_cache = static_cast<uint8_t*>(k_cache);
  p.v_cache = static_cast<uint8_t*>(v_cache);
  p.k_scale = k_scale;
  p.v_scale = v_scale;
  p.k = k;
  p.v = v;
  p.slots = slots;
  p.base_slot = base_slot;
  p.num_tokens = num_tokens;
  p.num_kv_heads = num_kv_heads;
  p.head_dim = head_dim;
  p.block_size = block_size;
  p.num_blocks = num_blocks;
  p.k_stride = k_stride;
  p.v_stride = v_stride;
  p.aligned = aligned(k, 16) && aligned(v, 16) && k_stride * es % 16 == 0 && v_stride * es % 16 == 0;
  p.err_count = err_count;
  tv::launch_kv_write_fp8(p, dtype, reinterpret_cast<hipStream_t>(stream));
  return check_launch(who);
}

// Unsplit launches of this many sequences run longest first.
constexpr int kOrderMinSeqs = 32;
constexpr int kOrderMaxSeqs = 1024;

// Compute units of the current device, asked for once per device.
int device_cus() {
  static std::atomic<int> known[tv::kMaxDevices];
  int dev = 0, cus = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0) return 0;
  if (dev < tv::kMaxDevices && (cus = known[dev].load(std::memory_order_relaxed)) > 0) return cus;
  if (hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess) return 0;
  if (dev < tv::kMaxDevices) known[dev].store(cus, std::memory_order_relaxed);
  return cus;
}

long long decode_rows(int num_seqs, int num_heads, int num_kv_heads) {
  const int group = num_heads / num_kv_heads;
  return (long long)num_seqs * num_kv_heads * ((group + 15) / 16);
}

}  // namespace

extern "C" {

int tv_reshape_and_cache_fp8(void* k_cache, void* v_cache, float* k_scale, float* v_scale, const void* k,
                             const void* v, const int32_t* slot_mapping, int num_tokens, int num_kv_heads,
                             int head_dim, int block_size, int num_blocks, int64_t k_stride, int64_t v_stride,
                             int dtype, uint32_t* err_count, void* stream) {
  if (!slot_mapping && num_tokens > 0) return fail(TV_EINVAL, "tv_reshape_and_cache_fp8: null slot_mapping");
  return write_common("tv_reshape_and_cache_fp8", k_cache, v_cache, k_scale, v_scale, k, v, slot_mapping, 0,
                      num_tokens, num_kv_heads, head_dim, block_size, num_blocks, k_stride, v_stride, dtype,
                      err_count, stream);
}

int tv_write_kv_fp8(void* k_cache, void* v_cache, float* k_scale, float* v_scale, const void* k, const void* v,
                    int block_id, int start_offset, int num_tokens, int num_kv_heads, int head_dim, int block_size,
                    int num_blocks, int64_t k_stride, int64_t v_stride, int dtype, void* stream) {
  if (block_id < 0 || block_id >= num_blocks)
    return fail(TV_EINVAL, "tv_write_kv_fp8: block_id %d outside [0, %d)", block_id, num_blocks);
  if (start_offset < 0 || num_tokens < 0 || (long long)start_offset + num_tokens > block_size)
    return fail(TV_EINVAL, "tv_write_kv_fp8: rows [%d, %lld) do not fit a block of %d", start_offset,
                (long long)start_offset + num_tokens, block_size);
  if ((long long)num_blocks * block_size > 0x7fffffffLL)
    return fail(TV_EINVAL, "tv_write_kv_fp8: %d blocks of %d have slots past 32 bits", num_blocks, block_size);
  return write_common("tv_write_kv_fp8", k_cache, v_cache, k_scale, v_scale, k, v, nullptr,
                      block_id * block_size + start_offset, num_tokens, num_kv_heads, head_dim, block_size,
                      num_blocks, k_stride, v_stride, dtype, nullptr, stream);
}

int tv_read_kv_blocks_fp8(void* k_out, void* v_out, const void* k_cache, const void* v_cache, const float* k_scale,
                          const float* v_scale, const int32_t* block_ids, int num_block_ids, int context_len,
                          int num_kv_heads, int head_dim, int block_size, int num_blocks, int dtype, void* stream) {
  const char* who = "tv_read_kv_blocks_fp8";
  int rc = check_cache(who, k_cache, v_cache, k_scale, v_scale, num_kv_heads, head_dim, block_size, num_blocks, dtype);
  if (rc != TV_OK) return rc;
  if (context_len < 0 || num_block_ids < 0 || (long long)context_len > (long long)num_block_ids * block_size)
    return fail(TV_EINVAL, "%s: context_len %d exceeds %d blocks of %d", who, context_len, num_block_ids, block_size);
  if (context_len == 0) return ok();
  if (!k_out || !v_out || !block_ids) return fail(TV_EINVAL, "%s: null pointer argument", who);
  if (!aligned(k_out, 16) || !aligned(v_out, 16) || !aligned(block_ids, 4))
    return fail(TV_EINVAL, "%s: outputs must be 16-byte aligned", who);
  tv::KVGatherFp8Params p{};
  p.k_out = k_out;
  p.v_out = v_out;
  p.k_cache = static_cast<const uint8_t*>(k_cache);
  p.v_cache = static_cast<const uint8_t*>(v_cache);
  p.k_scale = k_scale;
  p.v_scale = v_scale;
  p.block_ids = block_ids;
  p.context_len = context_len;
  p.num_kv_heads = num_kv_heads;
  p.head_dim = head_dim;
  p.block_size = block_size;
  p.num_blocks = num_blocks;
  tv::launch_kv_gather_fp8(p, dtype, reinterpret_cast<hipStream_t>(stream));
  return check_launch(who);
}

size_t tv_paged_decode_fp8_workspace_bytes(int num_seqs, int num_heads, int head_dim, int max_blocks, int block_size,
                                           int partition_size) {
  if (num_seqs <= 0 || num_heads <= 0 || head_dim <= 0 || max_blocks <= 0 || block_size <= 0 || partition_size <= 0)
    return 0;
  const long long width = (long long)max_blocks * block_size;
  const long long parts = (width + partition_size - 1) / partition_size;
  if (parts <= 1)
    return num_seqs >= kOrderMinSeqs && num_seqs <= kOrderMaxSeqs
               ? ((size_t)(num_seqs + 1) * sizeof(int) + 255) & ~(size_t)255
               : 0;
  return (size_t)num_seqs * num_heads * parts * (head_dim + 2) * sizeof(float);
}

int tv_paged_decode_fp8_partition_size(int num_seqs, int num_heads, int num_kv_heads, int head_dim, int max_blocks,
                                       int block_size, int dtype) {
  const char* who = "tv_paged_decode_fp8_partition_size";
  if (num_seqs <= 0 || num_heads <= 0 || num_kv_heads <= 0 || num_heads % num_kv_heads != 0 || max_blocks <= 0 ||
      block_size <= 0 || (long long)max_blocks * block_size > (1LL << 30) || !valid_dtype(dtype))
    return fail(TV_EINVAL, "%s: bad arguments", who), 0;
  if (!valid_head_dim(head_dim))
    return fail(TV_EUNSUPPORTED, "%s: head_dim %d not supported (64/128/256)", who, head_dim), 0;
  const int cus = device_cus();
  if (cus < 1) return fail(TV_EHIP, "%s: no device", who), 0;
  const long long width = (long long)max_blocks * block_size;
  const int whole = (int)((width + 31) / 32 * 32);
  const long long rows = decode_rows(num_seqs, num_heads, num_kv_heads);
  if (rows >= 2LL * cus || width <= tv::kFp8WideTokens) return whole;
  // Enough parts that every CU has one (of 32 KiB and more; two parts gain less
  // than joining them costs), and, for contexts of more than 256 KiB a head, four
  // per CU, whose ends even out.  MI355X, us, whole / this rule (equal lengths, and
  // lengths down to half): 40 x 8000 tokens of 32 / 8 heads of 128 143 / 113, 121 /
  // 94; 20 x 16000 138 / 113, 130 / 99; 24 x 4000 39 / 39, 37 / 40; 60 x 12000 234 /
  // 245, 209 / 195; 16 x 32768 in 2 parts 171, in 8 175; 1 x 8000 30 / 11; 32 / 4
  // heads of 64: 32 x 1000 stays whole, 9.4, in 2 parts 11.2.
  const long long least = std::max(1LL, width * head_dim / 16384);
  long long fill = std::min(cus / rows, least);
  if (fill < 3) fill = 1;
  const long long even = std::min((4LL * cus + rows - 1) / rows, (width * head_dim + 131071) / 131072);
  const long long parts = std::max({1LL, fill, even});
  long long p = (width + parts - 1) / parts;
  p = std::max(128LL, (p + 31) / 32 * 32);
  return p < whole ? (int)p : whole;
}

int tv_paged_decode_fp8(void* out, const void* queries, const void* k_cache, const void* v_cache,
                        const float* k_scale, const float* v_scale, const int32_t* block_tables,
                        const int32_t* context_lens, int num_seqs, int num_heads, int num_kv_heads, int head_dim,
                        int block_size, int num_blocks, int block_table_stride, int max_blocks, float scale,
                        int dtype, int out_dtype, int partition_size, void* workspace, size_t workspace_bytes,
                        void* stream) {
  const char* who = "tv_paged_decode_fp8";
  if (!out || !queries || !block_tables || !context_lens) return fail(TV_EINVAL, "%s: null pointer argument", who);
  int rc = check_cache(who, k_cache, v_cache, k_scale, v_scale, num_kv_heads, head_dim, block_size, num_blocks, dtype);
  if (rc != TV_OK) return rc;
  if (!(out_dtype == dtype || out_dtype == TV_F32))
    return fail(TV_EINVAL, "%s: bad dtype %d / out_dtype %d", who, dtype, out_dtype);
  if (num_seqs <= 0 || num_heads <= 0 || num_heads % num_kv_heads != 0)
    return fail(TV_EINVAL, "%s: bad head counts (num_seqs=%d, num_heads=%d, num_kv_heads=%d)", who, num_seqs,
                num_heads, num_kv_heads);
  if (block_table_stride < 0 || max_blocks <= 0 || (block_table_stride > 0 && max_blocks > block_table_stride))
    return fail(TV_EINVAL, "%s: bad block table (stride=%d, max_blocks=%d)", who, block_table_stride, max_blocks);
  const long long width = (long long)max_blocks * block_size;
  if (width > (1LL << 30)) return fail(TV_EINVAL, "%s: context width too large", who);
  if (partition_size <= 0 || partition_size % 32 != 0)
    return fail(TV_EINVAL, "%s: partition_size must be a positive multiple of 32 (got %d)", who, partition_size);
  if (!aligned(out, 16) || !aligned(queries, 16) || !aligned(block_tables, 4) || !aligned(context_lens, 4))
    return fail(TV_EINVAL, "%s: queries/out must be 16-byte aligned", who);
  const int max_parts = (int)((width + partition_size - 1) / partition_size);
  const size_t need = tv_paged_decode_fp8_workspace_bytes(num_seqs, num_heads, head_dim, max_blocks, block_size,
                                                          partition_size);
  if (max_parts > 1 && (!workspace || workspace_bytes < need || !aligned(workspace, 4)))
    return fail(TV_EINVAL, "%s: workspace of %zu bytes required (got %zu)", who, need, workspace_bytes);
  // Longest first, at the cost of a launch, where work-groups wait for others to end
  // (two are resident per CU).  MI355X, us, lengths from a quarter up, with / without:
  // 32 / 8 heads of 128: 128 sequences to 4096 tokens 113 / 132, 256 230 / 247, 512 to
  // 1152 144 / 148, 128 to 1152 39.3 / 39.9; 32 / 4 heads of 64, 256 to 4096 67 / 76,
  // and with 256 work-groups (64 to 1152) 15.4 / 10.0.
  const bool ordered = max_parts == 1 && need > 0 && workspace && workspace_bytes >= need && aligned(workspace, 4) &&
                       decode_rows(num_seqs, num_heads, num_kv_heads) > 2LL * device_cus() &&
                       decode_rows(num_seqs, num_heads, num_kv_heads) < 1LL << 24;   // 256 threads each in one dimension
  const int group = num_heads / num_kv_heads;
  const int chunks = (group + 15) / 16;
  if (num_seqs > 65535 || max_parts > 65535 || num_heads > 0x7fffffff / 256)
    return fail(TV_EINVAL, "%s: grid too large", who);

  tv::DecodeFp8Params p{};
  p.out = out;
  p.q = queries;
  p.k_cache = static_cast<const uint8_t*>(k_cache);
  p.v_cache = static_cast<const uint8_t*>(v_cache);
  p.k_scale = k_scale;
  p.v_scale = v_scale;
  p.block_tables = block_tables;
  p.context_lens = context_lens;
  p.num_seqs = num_seqs;
  p.num_heads = num_heads;
  p.num_kv_heads = num_kv_heads;
  p.head_chunks = chunks;
  p.block_size = block_size;
  p.bs_log2 = log2_or_minus1(block_size);
  p.num_blocks = num_blocks;
  p.bt_stride = block_table_stride;
  p.max_blocks = max_blocks;
  p.scale = scale;
  p.partition_size = partition_size;
  p.max_parts = max_parts;
  p.out_dtype = out_dtype;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (max_parts > 1) {
    p.part_o = reinterpret_cast<float*>(workspace);
    p.part_ml = p.part_o + (size_t)num_seqs * num_heads * max_parts * head_dim;
  }
  if (ordered) {
    int* sched = reinterpret_cast<int*>(workspace);
    p.sched = sched;
    hipLaunchKernelGGL(tv::decode_order_kernel, dim3(1), dim3(1024), 0, s, context_lens, num_seqs, (int)width, 0,
                       sched);
  }
  // Eight waves where a CU has one work-group of few tiles.  MI355X, us, 8 / 4 waves,
  // 32 / 4 heads of 64: 1 x 500 tokens 5.8 / 6.5, 8 x 250 5.1 / 5.4, 32 x 500 6.3 /
  // 6.9; with heads of 128 the larger merge takes it back: 1 x 500 7.7 / 7.5, 32 x
  // 500 8.3 / 7.9.
  const bool wide = !ordered && max_parts == 1 && head_dim == 64 && width <= tv::kFp8WideTokens &&
                    decode_rows(num_seqs, num_heads, num_kv_heads) <= device_cus();
  tv::launch_paged_decode_fp8(p, head_dim, dtype, wide, s);
  return check_launch(who);
}

size_t tv_flash_prefill_paged_fp8_workspace_bytes(int q_len, int start_pos, int num_heads, int num_kv_heads,
                                                  int head_dim) {
  if (q_len <= 0 || start_pos < 0 || num_heads <= 0 || num_kv_heads <= 0 || num_heads % num_kv_heads != 0 ||
      !valid_head_dim(head_dim))
    return 0;
  const int splits = tv::prefill_fp8_splits(q_len, start_pos, num_heads, num_kv_heads, head_dim, device_cus());
  return splits > 1 ? (size_t)splits * q_len * num_heads * (head_dim + 2) * sizeof(float) : 0;
}

int tv_flash_prefill_paged_fp8(void* out, const void* q, const void* k_cache, const void* v_cache,
                               const float* k_scale, const float* v_scale, const int32_t* block_table,
                               int num_blocks, int block_size, int q_len, int start_pos, int num_heads,
                               int num_kv_heads, int head_dim, int64_t q_stride, int64_t out_stride, int causal,
                               float scale, int dtype, int out_dtype, void* workspace, size_t workspace_bytes,
                               void* stream) {
  const char* who = "tv_flash_prefill_paged_fp8";
  if (!out || !q || !block_table) return fail(TV_EINVAL, "%s: null pointer argument", who);
  int rc = check_cache(who, k_cache, v_cache, k_scale, v_scale, num_kv_heads, head_dim, block_size, num_blocks, dtype);
  if (rc != TV_OK) return rc;
  if (!(out_dtype == dtype || out_dtype == TV_F32))
    return fail(TV_EINVAL, "%s: bad dtype %d / out_dtype %d", who, dtype, out_dtype);
  if (dtype == TV_F32) return fail(TV_EUNSUPPORTED, "%s: fp16 / bf16 queries only", who);
  if (q_len <= 0 || start_pos < 0 || (long long)start_pos + q_len > (1LL << 30))
    return fail(TV_EINVAL, "%s: bad sizes (q_len=%d, start_pos=%d)", who, q_len, start_pos);
  if (num_heads <= 0 || num_heads % num_kv_heads != 0)
    return fail(TV_EINVAL, "%s: bad head counts (%d, %d)", who, num_heads, num_kv_heads);
  if (q_stride < (int64_t)num_heads * head_dim || out_stride < (int64_t)num_heads * head_dim)
    return fail(TV_EINVAL, "%s: token stride smaller than a token row", who);
  if (!aligned(q, 16) || q_stride % 8 || !aligned(out, 16) || out_stride % 4 || !aligned(block_table, 4))
    return fail(TV_EINVAL, "%s: query and output rows must be 16-byte aligned", who);
  const int group = num_heads / num_kv_heads;
  if ((long long)q_len * group > 65535LL * 64) return fail(TV_EINVAL, "%s: grid too large", who);
  const size_t need = tv_flash_prefill_paged_fp8_workspace_bytes(q_len, start_pos, num_heads, num_kv_heads, head_dim);
  if (workspace && (workspace_bytes < need || !aligned(workspace, 16)))
    return fail(TV_EINVAL, "%s: workspace of %zu bytes, 16-byte aligned, required (got %zu)", who, need, workspace_bytes);
  tv::PrefillFp8Params p{};
  p.out = out;
  p.q = q;
  p.k_cache = static_cast<const uint8_t*>(k_cache);
  p.v_cache = static_cast<const uint8_t*>(v_cache);
  p.k_scale = k_scale;
  p.v_scale = v_scale;
  p.block_table = block_table;
  p.q_len = q_len;
  p.start_pos = start_pos;
  p.num_kv_heads = num_kv_heads;
  p.group = group;
  p.block_size = block_size;
  p.bs_log2 = log2_or_minus1(block_size);
  p.num_blocks = num_blocks;
  p.q_stride = q_stride;
  p.out_stride = out_stride;
  p.causal = causal ? 1 : 0;
  p.scale = scale;
  p.out_dtype = out_dtype;
  p.splits = 1;
  if (workspace && need) {
    p.splits = tv::prefill_fp8_splits(q_len, start_pos, num_heads, num_kv_heads, head_dim, device_cus());
    p.part_o = reinterpret_cast<float*>(workspace);
    p.part_ml = p.part_o + (size_t)p.splits * q_len * num_heads * head_dim;
  }
  tv::launch_prefill_fp8(p, head_dim, dtype, device_cus(), reinterpret_cast<hipStream_t>(stream));
  return check_launch(who);
}

}  // extern "C"
