// Rotation of q and k to their positions and the write of k and v into the paged
// cache, in one pass (tv_rope_and_cache).
//
// With the table's (cos, sin) of pair i at a token's position,
//   (a, b) -> (a cos - b sin, a sin + b cos)
// in fp32, rounded once to the cache's type.  Every element is read and written once: bound by
// HBM, and by the launch for a decode step's tokens.  A work-group has 256 vectors of one token, so that its position and slot are the
// same in all lanes.  MI355X: 64 sequences of up to 32 nodes, 32 / 8 heads of 128 in bf16 (45 MB) 9.0 us, 5.0 TB/s; 4 x 8 nodes, 32 / 4 heads of
// 64 in fp32 2.8 us.
#include "tv_draft.h"

#include <algorithm>

namespace tv {

namespace {

constexpr int kThreads = 256;

// VEC consecutive elements of T as fp32.  WIDE: 16 bytes at a 16-byte boundary.
template <typename T, int VEC, bool WIDE> struct Vec {
  float x[VEC];
  __device__ __forceinline__ void load(const T* p) {
    if constexpr (WIDE) {
      const u32x4 w = *reinterpret_cast<const u32x4*>(p);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (sizeof(T) == 4) x[i] = u32_as_f32(w[i]);
        else unpack2<T>(w[i], x[2 * i], x[2 * i + 1]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < VEC; ++i) x[i] = to_float<T>(p[i]);
    }
  }
  __device__ __forceinline__ void store(T* p) const {
    if constexpr (WIDE) {
      u32x4 w;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (sizeof(T) == 4) w[i] = __builtin_bit_cast(uint32_t, (float)x[i]);
        else w[i] = pack2<T>(x[2 * i], x[2 * i + 1]);
      }
      *reinterpret_cast<u32x4*>(p) = w;
    } else {
#pragma unroll
      for (int i = 0; i < VEC; ++i) p[i] = from_float<T>(x[i]);
    }
  }
};

// Units of a head of q or k: with adjacent pairs its vectors; with halves first the
// vectors of the first half, each with its partner, then those that are not rotated.
// Units of a head of v: its vectors, which go as they are (bit for bit).
template <typename T, int VEC, bool WIDE, bool HALVES>
__global__ void __launch_bounds__(kThreads) rope_cache_kernel(const RopeCacheParams p) {
  const int t = blockIdx.x;
  const int pos = p.positions[t];
  const int slot = p.slots[t];
  const bool known = (unsigned)pos < (unsigned)p.rope_len;
  const bool write = known && slot >= 0 && slot < p.num_slots;
  if (blockIdx.y == 0 && threadIdx.x == 0 && p.err_count && (!known || slot >= p.num_slots)) atomicAdd(p.err_count, 1u);
  const int D = p.head_dim, half = p.rope_dim / 2;
  const int rotated = HALVES ? half / VEC : p.rope_dim / VEC;
  const int units = rotated + (D - p.rope_dim) / VEC;
  const int turned = (p.num_heads + p.num_kv_heads) * units;
  const int total = turned + p.num_kv_heads * (D / VEC);
  const float* table = p.rope + (size_t)(known ? pos : 0) * p.rope_dim;
  const T* q = reinterpret_cast<const T*>(p.q) + (size_t)t * p.q_stride;
  const T* k = reinterpret_cast<const T*>(p.k) + (size_t)t * p.k_stride;
  const T* v = reinterpret_cast<const T*>(p.v) + (size_t)t * p.v_stride;
  T* q_out = reinterpret_cast<T*>(p.q_out) + (size_t)t * p.q_out_stride;
  const size_t row = (size_t)(write ? slot : 0) * p.num_kv_heads * D;
  T* k_out = reinterpret_cast<T*>(p.k_cache) + row;
  T* v_out = reinterpret_cast<T*>(p.v_cache) + row;
  for (int i = blockIdx.y * kThreads + threadIdx.x; i < total; i += gridDim.y * kThreads) {
    if (i >= turned) {
      const int at = (i - turned) * VEC;
      if (!write) continue;
      if constexpr (WIDE) {
        *reinterpret_cast<u32x4*>(v_out + at) = *reinterpret_cast<const u32x4*>(v + at);
      } else {
#pragma unroll
        for (int e = 0; e < VEC; ++e) v_out[at + e] = v[at + e];
      }
      continue;
    }
    const int head = i / units, u = i - head * units;
    const bool is_q = head < p.num_heads;
    if (!is_q && !write) continue;
    const T* src = is_q ? q + (size_t)head * D : k + (size_t)(head - p.num_heads) * D;
    T* dst = is_q ? q_out + (size_t)head * D : k_out + (size_t)(head - p.num_heads) * D;
    Vec<T, VEC, WIDE> a, b;
    if (u >= rotated) {
      const int at = p.rope_dim + (u - rotated) * VEC;
      a.load(src + at);
      if (!known) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) a.x[e] = __builtin_nanf("");
      }
      a.store(dst + at);
    } else if constexpr (HALVES) {
      const int at = u * VEC;
      a.load(src + at);
      b.load(src + half + at);
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const float2 cs = reinterpret_cast<const float2*>(table)[at + e];
        const float x = a.x[e], y = b.x[e];
        a.x[e] = known ? x * cs.x - y * cs.y : __builtin_nanf("");
        b.x[e] = known ? x * cs.y + y * cs.x : __builtin_nanf("");
      }
      a.store(dst + at);
      b.store(dst + half + at);
    } else {
      const int at = u * VEC;
      a.load(src + at);
#pragma unroll
      for (int e = 0; e < VEC; e += 2) {
        const float2 cs = reinterpret_cast<const float2*>(table)[(at + e) / 2];
        const float x = a.x[e], y = a.x[e + 1];
        a.x[e] = known ? x * cs.x - y * cs.y : __builtin_nanf("");
        a.x[e + 1] = known ? x * cs.y + y * cs.x : __builtin_nanf("");
      }
      a.store(dst + at);
    }
  }
}

template <typename T> void launch_of(const RopeCacheParams& p, bool halves, bool wide, hipStream_t s) {
  constexpr int W = 16 / (int)sizeof(T);
  const int per = wide ? W : halves ? 1 : 2;
  const long long items = (long long)(p.num_heads + 2 * p.num_kv_heads) * p.head_dim / per;
  const dim3 grid(p.num_tokens, (unsigned)std::min<long long>((items + kThreads - 1) / kThreads, 64));
  if (wide && halves) hipLaunchKernelGGL((rope_cache_kernel<T, W, true, true>), grid, dim3(kThreads), 0, s, p);
  else if (wide) hipLaunchKernelGGL((rope_cache_kernel<T, W, true, false>), grid, dim3(kThreads), 0, s, p);
  else if (halves) hipLaunchKernelGGL((rope_cache_kernel<T, 1, false, true>), grid, dim3(kThreads), 0, s, p);
  else hipLaunchKernelGGL((rope_cache_kernel<T, 2, false, false>), grid, dim3(kThreads), 0, s, p);
}

}  // namespace

void launch_rope_cache(const RopeCacheParams& p, int dtype, bool halves, bool wide, hipStream_t s) {
  if (dtype == kF32) launch_of<float>(p, halves, wide, s);
  else if (dtype == kF16) launch_of<_Float16>(p, halves, wide, s);
  else launch_of<__bf16>(p, halves, wide, s);
}

}  // namespace tv
