// The 8-bit K/V cache: number format, scales and launch parameter blocks.
//
// A cache element is an e4m3 number (no infinities, 0x7f / 0xff are NaN, largest
// 448) that stands for q * 2^e; e is held once per (block, KV head), K and V each
// for itself, as the fp32 number 2^e.  A scale is a power of two so that x * 2^-e
// and q * 2^e are exact: the only rounding is the one to e4m3, rescaling held
// rows is exact above e4m3's subnormals, and e4m3, being a floating-point format,
// gains nothing from the finer scales that an integer format would need.
//
// Layout: [num_blocks, Hkv, block_size, D].  The rows of one head in a block are
// contiguous (2 KiB at D 128, block 16), so the work-group of one head reads
// whole lines; in [num_blocks, block_size, Hkv, D] an 8-bit row of head_dim 64
// would be half a line.
#pragma once

#include "tv_common.h"

namespace tv {

typedef float f32x2 __attribute__((ext_vector_type(2)));

constexpr int kFp8MinExp = -100;       // least scale exponent (blocks of zeros, and blocks never written)
constexpr int kFp8MaxBlock = 1024;     // rows of a block (the write kernel's row list in LDS)
constexpr int kFp8WideTokens = 512;    // contexts of at most this many tokens stay unsplit, whatever the batch
constexpr uint32_t kFp8Nan = 0x7f;

// Exponent of the scale for rows whose largest magnitude is amax (finite, >= 0):
// the least e >= kFp8MinExp with amax <= 448 * 2^e; 448 = 1.75 * 2^8.
__device__ __forceinline__ int fp8_scale_exp(float amax) {
  const uint32_t u = __builtin_bit_cast(uint32_t, amax);
  const int e = (int)(u >> 23) - 127 - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
  return e > kFp8MinExp ? e : kFp8MinExp;
}
__device__ __forceinline__ float exp2_int(int e) { return __builtin_bit_cast(float, (uint32_t)(e + 127) << 23); }
// Exponent of a stored scale.  Anything below the least one (a zeroed scale) counts as the least.
__device__ __forceinline__ int fp8_scale_exp_of(float scale) {
  const int e = (int)((__builtin_bit_cast(uint32_t, scale) >> 23) & 255u) - 127;
  return e > kFp8MinExp ? e : kFp8MinExp;
}

// What no kernel writes while this one runs, at a wave-uniform address: a scalar load.
template <typename V> __device__ __forceinline__ V uniform_load(const V* p) {
  return *(const __attribute__((address_space(4))) V*)(p);
}

// Four e4m3 numbers to fp32, exactly.
__device__ __forceinline__ f32x4 fp8_to_f32x4(uint32_t w) {
  const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false);
  const f32x2 b = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
  return f32x4{a[0], a[1], b[0], b[1]};
}
// Four fp32 numbers of at most 448 in magnitude to e4m3, to nearest, ties to
// even.  An infinity (which the format lacks) becomes NaN, as a NaN does.
__device__ __forceinline__ uint32_t f32x4_to_fp8(f32x4 x) {
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = fabsf(x[i]) <= 448.0f ? x[i] : __builtin_nanf("");
  int r = __builtin_amdgcn_cvt_pk_fp8_f32(x[0], x[1], 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(x[2], x[3], r, true);
}
// Two e4m3 numbers (the low or the high half of a word) to two packed 16-bit
// numbers: both formats hold every e4m3 number.
template <typename T, bool HI> __device__ __forceinline__ uint32_t fp8_to_pair(uint32_t w) {
  if constexpr (sizeof(T) == 2 && ElemTraits<T>::kCode == kF16)
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, HI));
  else
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, HI));
}

// The largest finite number of T.  A value's rounding to e4m3, of up to 2^-4, can
// lift it past that number (65504 becomes 65536, 3.3e38 becomes 2^128), and an
// infinity in V would reach rows that give it a weight of zero: what is read back
// as T is limited to it.  Only scales above kSafeScale need the comparison.
template <typename T> constexpr float kLargest =
    ElemTraits<T>::kCode == kF16 ? 65504.0f : ElemTraits<T>::kCode == kBF16 ? 0x1.fep127f : 0x1.fffffep127f;
template <typename T> constexpr float kSafeScale = ElemTraits<T>::kCode == kF16 ? 0x1p7f : 0x1p119f;   // 448 times it is in range

template <typename T> __device__ __forceinline__ f32x4 limited(f32x4 x) {
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (fabsf(x[i]) > kLargest<T>) x[i] = __builtin_copysignf(kLargest<T>, x[i]);   // NaN stays
  return x;
}

// An output that averages cached values.  Rounding to e4m3 can lift a value near
// fp16's largest past it (65504 becomes 65536), so fp16 outputs are limited to it.
__device__ __forceinline__ void store_limited(void* base, size_t idx, float v, int dtype) {
  if (dtype == kF16 && fabsf(v) > 65504.0f) v = __builtin_copysignf(65504.0f, v);
  store_as(base, idx, v, dtype);
}

// 8-bit cache write and gather (kv_cache_fp8.hip).
struct KVWriteFp8Params {
  uint8_t* k_cache;
  uint8_t* v_cache;
  float* k_scale;
  float* v_scale;
  const void* k;
  const void* v;
  const int* slots;      // may be null: token t goes to slot base_slot + t
  int base_slot;
  int num_tokens;
  int num_kv_heads;
  int head_dim;
  int block_size;
  int num_blocks;
  long long k_stride;    // elements between consecutive tokens
  long long v_stride;
  int heads_per_group;   // KV heads of one work-group
  int tokens_per_group;  // tokens whose blocks one work-group looks after
  bool aligned;          // rows of k and v start at multiples of 16 bytes
  unsigned* err_count;   // may be null
};

struct KVGatherFp8Params {
  void* k_out;
  void* v_out;
  const uint8_t* k_cache;
  const uint8_t* v_cache;
  const float* k_scale;
  const float* v_scale;
  const int* block_ids;
  int context_len;
  int num_kv_heads;
  int head_dim;
  int block_size;
  int num_blocks;
};

// Attention of one token per sequence over the 8-bit cache (paged_decode_fp8.hip).
struct DecodeFp8Params {
  void* out;                 // [B, Hq, D] in out_dtype
  float* part_o;             // [B, Hq, max_parts, D] normalised partition outputs
  float* part_ml;            // [B, Hq, max_parts, 2] (max in log2 units, sum)
  const void* q;             // [B, Hq, D]
  const uint8_t* k_cache;    // [NB, Hkv, bs, D]
  const uint8_t* v_cache;
  const float* k_scale;      // [NB, Hkv]
  const float* v_scale;
  const int* block_tables;   // [B, bt_stride]
  const int* context_lens;   // [B]
  int num_seqs;
  int num_heads;
  int num_kv_heads;
  int head_chunks;           // ceil((Hq / Hkv) / 16)
  int block_size;
  int bs_log2;               // log2(block_size) or -1
  int num_blocks;
  int bt_stride;
  int max_blocks;            // table columns used (<= bt_stride, or bt_stride 0)
  float scale;
  int partition_size;        // tokens per work-group, a multiple of 32
  int max_parts;
  int out_dtype;
  const int* sched;          // unsplit launch of many sequences: [1 ..] their longest-first order
};

void launch_paged_decode_fp8(const DecodeFp8Params& p, int head_dim, int dtype, bool wide, hipStream_t stream);

// Attention of a chunk's rows over the 8-bit cache (flash_prefill_fp8.hip).
struct PrefillFp8Params {
  void* out;
  const void* q;             // [q_len, Hq, D], token stride q_stride
  const uint8_t* k_cache;    // [NB, Hkv, bs, D]
  const uint8_t* v_cache;
  const float* k_scale;      // [NB, Hkv]
  const float* v_scale;
  const int* block_table;
  int q_len;
  int start_pos;
  int num_kv_heads;
  int group;                 // query heads of a KV head
  int block_size;
  int bs_log2;               // log2(block_size) or -1
  int num_blocks;
  long long q_stride;        // elements between consecutive tokens
  long long out_stride;
  int causal;
  float scale;
  int out_dtype;
  int splits;                // work-groups that share a row tile's keys
  float* part_o;             // [splits, Hkv, q_len * group, D] normalised parts
  float* part_ml;            // [splits, Hkv, q_len * group, 2] (max in log2 units, sum)
};

int prefill_fp8_splits(int q_len, int start_pos, int num_heads, int num_kv_heads, int head_dim, int cus);
void launch_prefill_fp8(const PrefillFp8Params& p, int head_dim, int dtype, int cus, hipStream_t stream);

void launch_kv_write_fp8(KVWriteFp8Params p, int dtype, hipStream_t stream);
void launch_kv_gather_fp8(const KVGatherFp8Params& p, int dtype, hipStream_t stream);

}  // namespace tv
