// Writing and reading the 8-bit paged cache (format, scales and layout: tv_fp8.h).
//
// kv_write_fp8_kernel.  Token t's K and V rows go to slot s_t, block s_t /
// block_size, row s_t % block_size.  Per block touched, KV head and cache:
//   amax   the largest finite magnitude among the rows that the call writes there
//   e      the least exponent with amax <= 448 * 2^e; not below the block's
//          present one, unless the call writes row 0: that starts the block anew
//   rows   x * 2^-e rounded to e4m3; held rows are rounded again by 2^(old - e)
//          where the exponent grew, and become zero where the block starts anew
// A block's scale depends on all of the call's rows for it, so one work-group
// owns a block (for heads_per_group of its heads) and no atomics are needed: the
// work-group of the first token whose slot lies in the block.  It finds the
// others by reading the slot list, which also settles a slot that is named twice
// (the last token wins).  Only tokens whose predecessor lies in another block
// read the list, one per 16 tokens of a prompt, from L2.
// Bound: the rows' bytes for long prompts, launch and the chain slots -> list ->
// scale and rows -> maximum for short ones.  MI355X: 8192 fp16 or bf16 rows of 8
// heads of 128, K and V, 50 MB read and written, 16.7 us (3.0 TB/s), 16384 24.4
// (4.1 TB/s); 64 rows of a step 5.4.
// Wave w takes (head, cache) pairs w, w + 4, ...: D / 8 lanes cover a row with
// eight elements each, and up to kWriteHold rows a lane stay in registers from
// the maximum to the rounding.
#include "tv_fp8.h"

namespace tv {

constexpr int kWriteThreads = 256;
constexpr int kWriteHold = 4;
constexpr int kWriteFewTokens = 512;
constexpr long long kWriteGroups = 512;   // work-groups that a long prompt's write keeps

struct Row8 {
  f32x4 a, b;
};

// Eight elements as they lie in memory.  `aligned` (uniform over the launch):
// their addresses are multiples of 16 bytes.
template <typename T> struct Raw8 { u32x4 w[sizeof(T) == 4 ? 2 : 1]; };

template <typename T> __device__ __forceinline__ Raw8<T> load_row8(const T* p, bool aligned) {
  Raw8<T> r;
  if (aligned) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) r.w[i] = reinterpret_cast<const u32x4*>(p)[i];
  } else if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < 8; ++i) r.w[i >> 2][i & 3] = reinterpret_cast<const uint32_t*>(p)[i];
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      r.w[0][i] = reinterpret_cast<const uint16_t*>(p)[2 * i] | (uint32_t)reinterpret_cast<const uint16_t*>(p)[2 * i + 1] << 16;
  }
  return r;
}

template <typename T> __device__ __forceinline__ Row8 as_floats(const Raw8<T>& raw) {
  Row8 r;
  if constexpr (sizeof(T) == 4) {
    r.a = __builtin_bit_cast(f32x4, raw.w[0]);
    r.b = __builtin_bit_cast(f32x4, raw.w[1]);
  } else {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      float x, y;
      unpack2<T>(raw.w[0][i], x, y);
      r.a[2 * i] = x; r.a[2 * i + 1] = y;
      unpack2<T>(raw.w[0][2 + i], x, y);
      r.b[2 * i] = x; r.b[2 * i + 1] = y;
    }
  }
  return r;
}

__device__ __forceinline__ float finite_abs(float x) {
  const float a = fabsf(x);
  return a < __builtin_inff() ? a : 0.0f;
}
__device__ __forceinline__ float amax8(const Row8& r, float m) {
#pragma unroll
  for (int i = 0; i < 4; ++i) m = fmaxf(m, fmaxf(finite_abs(r.a[i]), finite_abs(r.b[i])));
  return m;
}
__device__ __forceinline__ u32x2 round_row8(const Row8& r, float inv) {
  return u32x2{f32x4_to_fp8(r.a * inv), f32x4_to_fp8(r.b * inv)};
}

// Marks the rows of the block that starts at slot `first` with their tokens (winner[r] becomes the last
// token of row r) and returns whether any is before token t.  Sixteen slots a thread are on the way at once.
__device__ __forceinline__ bool find_rows(const KVWriteFp8Params& p, int t, int first, int* winner) {
  constexpr int kStep = 4;
  const int n = p.num_tokens;
  bool earlier = false;
  const bool vec = (uintptr_t)p.slots % 16 == 0;
  for (int i0 = threadIdx.x * 4; i0 < n; i0 += kWriteThreads * 4 * kStep) {
    u32x4 s[kStep];
#pragma unroll
    for (int u = 0; u < kStep; ++u) {
      const int i = i0 + u * kWriteThreads * 4;
      if (vec && i + 4 <= n) {
        s[u] = *reinterpret_cast<const u32x4*>(p.slots + i);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) s[u][e] = (uint32_t)p.slots[min(i + e, n - 1)];
      }
    }
#pragma unroll
    for (int u = 0; u < kStep; ++u) {
      s[u] -= (uint32_t)first;
      const uint32_t least = min(min(s[u][0], s[u][1]), min(s[u][2], s[u][3]));
      if (least < (unsigned)p.block_size) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int i = i0 + u * kWriteThreads * 4 + e;
          if (i < n && s[u][e] < (unsigned)p.block_size) {
            earlier |= i < t;
            atomicMax(&winner[s[u][e]], i);
          }
        }
      }
    }
  }
  return earlier;
}

template <typename T, int D>
__global__ void __launch_bounds__(kWriteThreads) kv_write_fp8_kernel(const KVWriteFp8Params p) {
  constexpr int LPR = D / 8;        // lanes of a row
  constexpr int RPI = 64 / LPR;     // rows a wave covers at once
  constexpr int NW = kWriteThreads / 64;
  __shared__ int winner[kFp8MaxBlock];   // token that writes row r of the block, or -1
  const int bs = p.block_size;
  const long long num_slots = (long long)p.num_blocks * bs;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  const int lr = lane / LPR;
  const int lc = (lane % LPR) * 8;
  const int h0 = blockIdx.y * p.heads_per_group;
  const int units = 2 * min(p.heads_per_group, p.num_kv_heads - h0);

  // first tokens of runs in one block, found by every wave for the tokens that the work-group looks after
  const int t0 = blockIdx.x * p.tokens_per_group;
  int my_slot = -1;
  bool head = false;
  if (lane < p.tokens_per_group && t0 + lane < p.num_tokens) {
    const int t = t0 + lane;
    my_slot = p.slots ? p.slots[t] : p.base_slot + t;
    const int before = t == 0 ? -1 : p.slots ? p.slots[t - 1] : my_slot - 1;
    if (my_slot >= num_slots) {
      if (wave == 0 && blockIdx.y == 0 && p.err_count) atomicAdd(p.err_count, 1u);
    } else if (my_slot >= 0) {
      const int first = my_slot / bs * bs;          // the block's slots: first .. first + bs - 1
      head = (unsigned)before - (unsigned)first >= (unsigned)bs;
    }
  }
  unsigned long long heads = __builtin_amdgcn_ballot_w64(head);
  while (heads) {
    const int at = __builtin_ctzll(heads);
    heads &= heads - 1;
    const int t = t0 + at;
    const int slot = __builtin_amdgcn_readlane(my_slot, at);
    const int blk = slot / bs;
    const int first = blk * bs;
    __syncthreads();                                // the run before is done with winner
    for (int r = threadIdx.x; r < bs; r += kWriteThreads) {
      const int from_base = r - (slot - first);
      winner[r] = !p.slots && from_base >= 0 && from_base < p.num_tokens ? from_base : -1;
    }
    __syncthreads();
    if (__syncthreads_or(p.slots && find_rows(p, t, first, winner) ? 1 : 0)) continue;

    const bool restart = winner[0] >= 0;
    struct Rows {
      Raw8<T> x[kWriteHold];
      float scale;
    };
    auto source = [&](int u) {
      return reinterpret_cast<const T*>(u & 1 ? p.v : p.k) + (size_t)(h0 + (u >> 1)) * D + lc;
    };
    auto scale_of = [&](int u) {
      return (u & 1 ? p.v_scale : p.k_scale) + (size_t)blk * p.num_kv_heads + h0 + (u >> 1);
    };
    auto request = [&](int u, Rows& rows) {
      const T* src = source(u);
      const long long stride = u & 1 ? p.v_stride : p.k_stride;
      rows.scale = *scale_of(u);
#pragma unroll
      for (int j = 0; j < kWriteHold; ++j) {
        const int r = j * RPI + lr;
        const int w = r < bs ? winner[r] : -1;
        if (w >= 0) rows.x[j] = load_row8<T>(src + (size_t)w * stride, p.aligned);
      }
    };
    auto write = [&](int u, const Rows& rows) {
      const T* src = source(u);
      const long long stride = u & 1 ? p.v_stride : p.k_stride;
      uint8_t* dst = (u & 1 ? p.v_cache : p.k_cache) + ((size_t)blk * p.num_kv_heads + h0 + (u >> 1)) * bs * D + lc;
      const int old_e = fp8_scale_exp_of(rows.scale);
      float m = 0.0f;
#pragma unroll
      for (int j = 0; j < kWriteHold; ++j) {
        const int r = j * RPI + lr;
        if (r < bs && winner[r] >= 0) m = amax8(as_floats<T>(rows.x[j]), m);
      }
      for (int r = kWriteHold * RPI + lr; r < bs; r += RPI) {
        const int w = winner[r];
        if (w >= 0) m = amax8(as_floats<T>(load_row8<T>(src + (size_t)w * stride, p.aligned)), m);
      }
      m = group_max<64>(m);
      const int own_e = fp8_scale_exp(m);
      const int e = restart ? own_e : max(own_e, old_e);
      const float inv = exp2_int(-e);
      const float again = exp2_int(max(old_e - e, -126));   // of held rows, where the exponent grew

      auto put = [&](int r, const Row8& x) {
        *reinterpret_cast<u32x2*>(dst + (size_t)r * D) = round_row8(x, inv);
      };
      auto keep = [&](int r) {
        u32x2* q = reinterpret_cast<u32x2*>(dst + (size_t)r * D);
        if (restart) {
          *q = u32x2{0, 0};
        } else if (e != old_e) {
          const u32x2 w = *q;
          *q = u32x2{f32x4_to_fp8(fp8_to_f32x4(w[0]) * again), f32x4_to_fp8(fp8_to_f32x4(w[1]) * again)};
        }
      };
#pragma unroll
      for (int j = 0; j < kWriteHold; ++j) {
        const int r = j * RPI + lr;
        if (r < bs) {
          if (winner[r] >= 0) put(r, as_floats<T>(rows.x[j]));
          else keep(r);
        }
      }
      for (int r = kWriteHold * RPI + lr; r < bs; r += RPI) {
        const int w = winner[r];
        if (w >= 0) put(r, as_floats<T>(load_row8<T>(src + (size_t)w * stride, p.aligned)));
        else keep(r);
      }
      if (lane == 0) *scale_of(u) = exp2_int(e);
    };
    // the wave's next (head, cache) pair is on its way while one is rounded
    if (wave < units) {
      Rows ra, rb;
      request(wave, ra);
      for (int u = wave;; u += 2 * NW) {
        if (u + NW < units) request(u + NW, rb);
        write(u, ra);
        if (u + NW >= units) break;
        if (u + 2 * NW < units) request(u + 2 * NW, ra);
        write(u + NW, rb);
        if (u + 2 * NW >= units) break;
      }
    }
  }
}

// Row t of the listed blocks as values q * 2^e, limited to T's largest finite
// number.  Ids outside the cache read as 0.  Eight elements a lane, both caches.  Bound: HBM;
// 8192 rows as above back to fp16 10.3 us (4.9 TB/s).
template <typename T>
__global__ void __launch_bounds__(256) kv_gather_fp8_kernel(const KVGatherFp8Params p) {
  const int vec = p.head_dim / 8;
  const long long row = (long long)p.num_kv_heads * vec;
  const long long total = (long long)p.context_len * row;
  for (long long idx = (long long)blockIdx.x * blockDim.x + threadIdx.x; idx < total;
       idx += (long long)gridDim.x * blockDim.x) {
    const int t = (int)(idx / row);
    const int rest = (int)(idx - (long long)t * row);
    const int h = rest / vec;
    const int c = (rest - h * vec) * 8;
    const int bi = t / p.block_size;
    const int blk = p.block_ids[bi];
    const bool ok = (unsigned)blk < (unsigned)p.num_blocks;
    const size_t unit = (size_t)(ok ? blk : 0) * p.num_kv_heads + h;
    const size_t at = (unit * p.block_size + (t - bi * p.block_size)) * p.head_dim + c;
    const float f[2] = {ok ? exp2_int(fp8_scale_exp_of(p.k_scale[unit])) : 0.0f,
                        ok ? exp2_int(fp8_scale_exp_of(p.v_scale[unit])) : 0.0f};
    u32x2 w[2] = {u32x2{0, 0}, u32x2{0, 0}};
    if (ok) {
      w[0] = *reinterpret_cast<const u32x2*>(p.k_cache + at);
      w[1] = *reinterpret_cast<const u32x2*>(p.v_cache + at);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      f32x4 a = fp8_to_f32x4(w[i][0]) * f[i], b = fp8_to_f32x4(w[i][1]) * f[i];
      if (f[i] > kSafeScale<T>) {
        a = limited<T>(a);
        b = limited<T>(b);
      }
      T* out = reinterpret_cast<T*>(i ? p.v_out : p.k_out) + idx * 8;
      if constexpr (sizeof(T) == 4) {
        *reinterpret_cast<f32x4*>(out) = a;
        *reinterpret_cast<f32x4*>(out + 4) = b;
      } else {
        *reinterpret_cast<u32x4*>(out) =
            u32x4{pack2<T>(a[0], a[1]), pack2<T>(a[2], a[3]), pack2<T>(b[0], b[1]), pack2<T>(b[2], b[3])};
      }
    }
  }
}

namespace {

template <typename T>
void write_of(const KVWriteFp8Params& p, dim3 grid, hipStream_t stream) {
  if (p.head_dim == 64) hipLaunchKernelGGL((kv_write_fp8_kernel<T, 64>), grid, dim3(kWriteThreads), 0, stream, p);
  else if (p.head_dim == 128) hipLaunchKernelGGL((kv_write_fp8_kernel<T, 128>), grid, dim3(kWriteThreads), 0, stream, p);
  else hipLaunchKernelGGL((kv_write_fp8_kernel<T, 256>), grid, dim3(kWriteThreads), 0, stream, p);
}

}  // namespace

void launch_kv_write_fp8(KVWriteFp8Params p, int dtype, hipStream_t stream) {
  // A step's tokens lie in blocks of their own: one token and four (head, cache)
  // pairs, one a wave, per work-group.  A prompt's are in runs: sixteen tokens.  The
  // host sees only their number.  MI355X, us, one / sixteen, 8 heads of 128, bf16:
  // steps of 128 sequences 5.7 / 45, 512 11 / 42, 1024 20 / 43; prompts of 128 tokens
  // 6.4 / 5.8, 512 14 / 6, 1024 26 / 6, 8192 178 / 17.
  // Sixteen tokens take more heads a work-group, as long as two work-groups a CU
  // remain, since each reads the slots.  8 heads of 128, rule / two heads: 8192
  // tokens 16.7 / 17.0, 16384 24.4 / 33.8; 32 heads of 128 fp16: 4096 24 / 26, 8192
  // 44 / 53, 16384 90 / 140; 4 heads of 64 fp32, 8192 7.9 / 9.9.
  p.tokens_per_group = p.num_tokens <= kWriteFewTokens ? 1 : 16;
  const int groups = (p.num_tokens + p.tokens_per_group - 1) / p.tokens_per_group;
  p.heads_per_group = 2;
  while (p.tokens_per_group > 1 && p.heads_per_group < p.num_kv_heads &&
         (long long)groups * p.num_kv_heads >= kWriteGroups * 2 * p.heads_per_group)
    p.heads_per_group *= 2;
  const dim3 grid(groups, (p.num_kv_heads + p.heads_per_group - 1) / p.heads_per_group);
  if (dtype == kF32) write_of<float>(p, grid, stream);
  else if (dtype == kF16) write_of<_Float16>(p, grid, stream);
  else write_of<__bf16>(p, grid, stream);
}

void launch_kv_gather_fp8(const KVGatherFp8Params& p, int dtype, hipStream_t stream) {
  const long long total = (long long)p.context_len * p.num_kv_heads * (p.head_dim / 8);
  const long long g = (total + 255) / 256;
  const dim3 grid((unsigned)(g > 65536 ? 65536 : g));
  if (dtype == kF32) hipLaunchKernelGGL(kv_gather_fp8_kernel<float>, grid, dim3(256), 0, stream, p);
  else if (dtype == kF16) hipLaunchKernelGGL(kv_gather_fp8_kernel<_Float16>, grid, dim3(256), 0, stream, p);
  else hipLaunchKernelGGL(kv_gather_fp8_kernel<__bf16>, grid, dim3(256), 0, stream, p);
}

}  // namespace tv
