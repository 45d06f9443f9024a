// Attention of a draft tree's nodes over the paged cache (tv_paged_tree).
//
// The rows of a work-group are nodes times the query heads of one KV head, row r =
// head r % G of node r / G, so that all heads that read a key share it.  A
// work-group walks tiles of BN keys: S^T = K Q^T with the key rows as operand A; its
// accumulator layout is the B operand of O^T = V^T P^T, so P stays in registers.
// Every row sees every context key; only the tiles that reach past the context look
// at the nodes' mask, shifted to the tile.
//
// Numbers: scores, maxima, sums and accumulators are fp32.  For 16-bit types a weight is
// rounded to the type for the second product (at most half a step of it, as in the
// prefill kernels) and the row sum is that of the rounded weights; fp32 stays
// fp32 throughout (v_mfma_f32_16x16x4_f32).
// In a tile past the context rows differ in what they see, and a weight of zero would
// not hide a NaN or infinity in V: there such a value is zero in LDS and its key's score
// NaN, which the mask replaces for the rows that do not see the key.
#pragma once

#include "tv_draft.h"
#include "tv_fp8.h"

#include <algorithm>

namespace tv {

namespace {

constexpr int kTreeThreads = 256;

template <typename T> constexpr uint32_t kTreeNan = sizeof(T) == 4 ? 0x7FC00000u
                                                  : ElemTraits<T>::kCode == kF16 ? 0x7E007E00u : 0x7FC07FC0u;
// Exponent bits of a word's elements: all set in an infinity or NaN.
template <typename T> constexpr uint32_t kExpBits = sizeof(T) == 4 ? 0x7F800000u
                                                  : ElemTraits<T>::kCode == kF16 ? 0x7C007C00u : 0x7F807F80u;

// The bits of a word whose elements are infinite or NaN.
template <typename T> __device__ __forceinline__ uint32_t not_finite(uint32_t w) {
  if constexpr (sizeof(T) == 4) {
    return (w & kExpBits<T>) == kExpBits<T> ? ~0u : 0u;
  } else {
    constexpr uint32_t lo = kExpBits<T> & 0xffffu, hi = kExpBits<T> & 0xffff0000u;
    return ((w & lo) == lo ? 0xffffu : 0u) | ((w & hi) == hi ? 0xffff0000u : 0u);
  }
}

__device__ __forceinline__ float tree_max4(f32x4 x) {
  return __builtin_elementwise_maximum(__builtin_elementwise_maximum(x[0], x[1]), __builtin_elementwise_maximum(x[2], x[3]));
}

// Keys per tile.
template <typename T, int D> constexpr int kTreeKeys = sizeof(T) == 4 ? (D == 256 ? 16 : 32) : (D == 256 ? 32 : 64);

// UB: the block size is 16 or a larger power of two: the rows that a wave stages at
// once lie in one block, whose id and address are then scalar.
template <typename T, int D, int RB, bool UB>
__global__ void __launch_bounds__(kTreeThreads) tree_attention_kernel(const TreeParams p) {
  constexpr bool F32 = sizeof(T) == 4;
  constexpr int BM = 64 * RB;
  constexpr int BN = kTreeKeys<T, D>;
  constexpr int KB = BN / 16;
  constexpr int DB = D / 16;
  constexpr int VEC = 16 / (int)sizeof(T);
  constexpr int CPR = D / VEC;                 // 16-byte vectors of a row
  constexpr int P = F32 ? D + 4 : D + 16;      // LDS row pitch (elements)
  constexpr int SKT = BN * P;
  constexpr int NV = BN * CPR / kTreeThreads;  // vectors per thread and tile, each of K and V
  constexpr int RPP = kTreeThreads / CPR;      // tile rows of one pass over the threads
  static_assert(NV * kTreeThreads == BN * CPR && NV >= 1, "tile shape");
  __shared__ __attribute__((aligned(16))) T smem[2][2 * SKT];

  const int tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lane = tid & 63;
  const int g = lane >> 4, col = lane & 15;
  int unit = blockIdx.x;
  const int rt = unit % p.row_tiles;
  unit /= p.row_tiles;
  const int kh = unit % p.num_kv_heads;
  unit /= p.num_kv_heads;
  const int b = unit % p.num_seqs;
  const int part = unit / p.num_seqs;

  const int G = p.group;
  const int ctx = min(max(p.context_lens[b], 0), p.width);
  const int len = min(max(p.tree_lens[b], 0), p.nodes);
  const int keys = min(ctx + len, p.width);
  const int parts = max(1, (keys + p.partition - 1) / p.partition);
  if (part >= parts) return;
  const int rows = p.nodes * G;
  const int row0 = rt * BM + wave * RB * 16;
  const int t0 = part * (p.partition / BN);
  // a tile without a live node has nothing to attend, and writes its zeros
  const int t1 = rt * BM < len * G ? min(t0 + p.partition / BN, (keys + BN - 1) / BN) : t0;

  int qrow[RB], node[RB];
  constexpr int QF = F32 ? D / 16 : D / 32;
  u32x4 qf[RB][QF];
#pragma unroll
  for (int r = 0; r < RB; ++r) {
    qrow[r] = row0 + r * 16 + col;
    node[r] = qrow[r] / G;
    const T* qg = reinterpret_cast<const T*>(p.q) + (size_t)b * p.q_seq_stride + (size_t)node[r] * p.q_node_stride +
                  (size_t)(kh * G + qrow[r] - node[r] * G) * D;
    // fp32: k index of step 4 f + e, lane g: 16 f + 4 g + e, on both operands
#pragma unroll
    for (int f = 0; f < QF; ++f)
      qf[r][f] = node[r] < len ? *reinterpret_cast<const u32x4*>(qg + (F32 ? 16 * f + 4 * g : 32 * f + 8 * g))
                               : u32x4{0, 0, 0, 0};
  }

  // staging: this thread's vectors are chunk ch of tile rows sr + RPP i
  const int sr = tid / CPR, ch = tid % CPR;
  const int wr = wave * (64 / CPR);            // first of the wave's rows
  const int bs = p.block_size;
  const size_t rs = (size_t)p.num_kv_heads * D;
  const int* table = p.block_tables + (size_t)b * p.bt_stride;
  const T* kc = reinterpret_cast<const T*>(p.k_cache) + (size_t)kh * D;
  const T* vc = reinterpret_cast<const T*>(p.v_cache) + (size_t)kh * D;
  auto key_of = [&](int t, int i) { return min(t * BN + (UB ? wr : sr) + RPP * i, keys - 1); };
  struct Ids { int id[NV]; };
  struct Stage { u32x4 k[NV], v[NV]; int ok[NV]; };
  auto ids_of = [&](int t, Ids& x) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int key = key_of(t, i);
      x.id[i] = UB ? uniform_load(table + (key >> p.bs_log2)) : table[key / bs];
    }
  };
  auto gload = [&](int t, const Ids& x, Stage& s) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int id = UB ? __builtin_amdgcn_readfirstlane(x.id[i]) : x.id[i];
      s.ok[i] = (unsigned)id < (unsigned)p.num_blocks ? -1 : 0;
      const size_t block = (size_t)(id & s.ok[i]) * bs;
      if constexpr (UB) {
        // a wave's rows start at a multiple of their number: those past the last key are the block's own
        const int first = (t * BN + wr + RPP * i) & (bs - 1);
        const size_t at = (block + first) * rs;
        const size_t lane_at = (size_t)(sr - wr) * rs + ch * VEC;
        s.k[i] = *reinterpret_cast<const u32x4*>(kc + at + lane_at);
        s.v[i] = *reinterpret_cast<const u32x4*>(vc + at + lane_at);
      } else {
        const int key = key_of(t, i);
        const size_t at = (block + key % bs) * rs + ch * VEC;
        s.k[i] = *reinterpret_cast<const u32x4*>(kc + at);
        s.v[i] = *reinterpret_cast<const u32x4*>(vc + at);
      }
    }
  };
  auto lstore = [&](const Stage& s, int buf, int t) {
    T* sk = smem[buf] + sr * P + ch * VEC;
    bool plain = (t + 1) * BN <= ctx;
#pragma unroll
    for (int i = 0; i < NV; ++i) plain = plain && s.ok[i];
    if (__builtin_amdgcn_ballot_w64(!plain) == 0) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        *reinterpret_cast<u32x4*>(sk + RPP * i * P) = s.k[i];
        *reinterpret_cast<u32x4*>(sk + RPP * i * P + SKT) = s.v[i];
      }
      return;
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      u32x4 k = s.k[i], v = s.v[i];
      const bool in = t * BN + sr + RPP * i < keys;
      if (!in || !s.ok[i]) k = v = u32x4{0, 0, 0, 0};
      bool poison = in && !s.ok[i];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t bad = not_finite<T>(v[j]);
        poison = poison || bad != 0;
        v[j] &= ~bad;
      }
      if (poison) k[0] = kTreeNan<T>;
      *reinterpret_cast<u32x4*>(sk + RPP * i * P) = k;
      *reinterpret_cast<u32x4*>(sk + RPP * i * P + SKT) = v;
    }
  };

  // Bits of the keys k0 .. k0 + 63 that a live node sees.
  auto seen_from = [&](int n, int k0) -> u64 {
    const u64* words = p.mask + (size_t)b * p.mask_seq_stride + (size_t)n * p.words;
    const int left = keys - k0;
    u64 bits;
    if (k0 >= ctx) {
      const int w = (k0 - ctx) >> 6, s = (k0 - ctx) & 63;
      bits = w < p.words ? words[w] >> s : 0;
      if (s && w + 1 < p.words) bits |= words[w + 1] << (64 - s);
    } else {
      const int s = ctx - k0;                  // context keys of the tile
      bits = s >= 64 ? ~0ull : ((1ull << s) - 1) | words[0] << s;
    }
    return left >= 64 ? bits : left > 0 ? bits & ((1ull << left) - 1) : 0;
  };

  f32x4 oacc[RB][DB];
  f32x4 sums[RB];                              // 16-bit: every lane's row sum; fp32: of the lane's own keys, in [0]
  float m[RB];
#pragma unroll
  for (int r = 0; r < RB; ++r) {
#pragma unroll
    for (int db = 0; db < DB; ++db) oacc[r][db] = f32x4{0.f, 0.f, 0.f, 0.f};
    sums[r] = f32x4{0.f, 0.f, 0.f, 0.f};
    m[r] = kNegInf;
  }
  const float c = p.scale * kLog2e;

  auto compute = [&](int buf, int t) {
    const T* sk = smem[buf];
    const T* sv = sk + SKT;
    const int k0 = t * BN;
    f32x4 st[RB][KB];
#pragma unroll
    for (int r = 0; r < RB; ++r)
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) st[r][kb] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int f = 0; f < QF; ++f)
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) {
        const u32x4 kf = *reinterpret_cast<const u32x4*>(sk + (kb * 16 + col) * P + (F32 ? 16 * f + 4 * g : 32 * f + 8 * g));
#pragma unroll
        for (int r = 0; r < RB; ++r) {
          if constexpr (F32) {
#pragma unroll
            for (int e = 0; e < 4; ++e)
              st[r][kb] = __builtin_amdgcn_mfma_f32_16x16x4f32(u32_as_f32(kf[e]), u32_as_f32(qf[r][f][e]), st[r][kb], 0, 0, 0);
          } else {
            st[r][kb] = mfma16x16x32<T>(kf, qf[r][f], st[r][kb]);
          }
        }
      }
    float base[RB], mt[RB];
    bool need = false;
#pragma unroll
    for (int r = 0; r < RB; ++r) {
      base[r] = m[r] == kNegInf ? 0.0f : m[r];
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int i = 0; i < 4; ++i) st[r][kb][i] = fmaf(st[r][kb][i], c, -base[r]);
    }
    if (k0 + BN > ctx) {
#pragma unroll
      for (int r = 0; r < RB; ++r) {
        const u64 bits = node[r] < len ? seen_from(node[r], k0) >> (4 * g) : 0;
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
          for (int i = 0; i < 4; ++i) st[r][kb][i] = bits >> (kb * 16 + i) & 1 ? st[r][kb][i] : kNegInf;
      }
    }
    // the running maximum is raised only when a tile passes it by 2^8
#pragma unroll
    for (int r = 0; r < RB; ++r) {
      mt[r] = tree_max4(st[r][0]);
#pragma unroll
      for (int kb = 1; kb < KB; ++kb) mt[r] = __builtin_elementwise_maximum(mt[r], tree_max4(st[r][kb]));
      need |= mt[r] > (m[r] == kNegInf ? kNegInf : 8.0f);
    }
    if (__builtin_amdgcn_ballot_w64(need) != 0) {
      __asm__ volatile("" ::: "memory");       // keeps this rare block a branch
#pragma unroll
      for (int r = 0; r < RB; ++r) {
        const float mm = max_over_g(mt[r]);    // relative to base
        const bool raise = mm > (m[r] == kNegInf ? kNegInf : 8.0f);
        const float delta = raise ? mm : 0.0f;
        const float alpha = raise && m[r] != kNegInf ? fast_exp2(-delta) : 1.0f;
        m[r] = raise ? base[r] + delta : m[r];
#pragma unroll
        for (int db = 0; db < DB; ++db) oacc[r][db] *= alpha;
        sums[r] *= alpha;
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) st[r][kb] -= delta;
      }
    }
#pragma unroll
    for (int r = 0; r < RB; ++r)
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int i = 0; i < 4; ++i) st[r][kb][i] = fast_exp2(st[r][kb][i]);
    if constexpr (F32) {
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) {
#pragma unroll
        for (int r = 0; r < RB; ++r) sums[r][0] += (st[r][kb][0] + st[r][kb][1]) + (st[r][kb][2] + st[r][kb][3]);
#pragma unroll
        for (int i = 0; i < 4; ++i)            // keys 4 g + i of the block
#pragma unroll
          for (int db = 0; db < DB; ++db) {
            const float v = sv[(kb * 16 + 4 * g + i) * P + db * 16 + col];
#pragma unroll
            for (int r = 0; r < RB; ++r)
              oacc[r][db] = __builtin_amdgcn_mfma_f32_16x16x4f32(v, st[r][kb][i], oacc[r][db], 0, 0, 0);
          }
      }
    } else {
      const u32x4 ones = u32x4{kOnes2<T>, kOnes2<T>, kOnes2<T>, kOnes2<T>};
#pragma unroll
      for (int x = 0; x < BN / 32; ++x) {
        u32x4 pf[RB];
        // reduction index 8g + j: key 4g + j of block 2 x (j < 4), 4g + j - 4 of block 2 x + 1
#pragma unroll
        for (int r = 0; r < RB; ++r)
          pf[r] = u32x4{pack2<T>(st[r][2 * x][0], st[r][2 * x][1]), pack2<T>(st[r][2 * x][2], st[r][2 * x][3]),
                        pack2<T>(st[r][2 * x + 1][0], st[r][2 * x + 1][1]), pack2<T>(st[r][2 * x + 1][2], st[r][2 * x + 1][3])};
#pragma unroll
        for (int db = 0; db < DB; ++db) {
          const T* a = sv + (x * 32 + 4 * g + (col >> 2)) * P + db * 16 + 4 * (col & 3);
          const u32x2 lo = lds_read_tr16(reinterpret_cast<const uint16_t*>(a));
          const u32x2 hi = lds_read_tr16(reinterpret_cast<const uint16_t*>(a + 16 * P));
          const u32x4 vf = u32x4{lo[0], lo[1], hi[0], hi[1]};
#pragma unroll
          for (int r = 0; r < RB; ++r) oacc[r][db] = mfma16x16x32<T>(vf, pf[r], oacc[r][db]);
        }
#pragma unroll
        for (int r = 0; r < RB; ++r) sums[r] = mfma16x16x32<T>(ones, pf[r], sums[r]);
      }
    }
  };

  if (t0 < t1) {
    Ids ids;
    Stage s;
    ids_of(t0, ids);
    gload(t0, ids, s);
    ids_of(t0 + 1, ids);
    lstore(s, 0, t0);
    gload(t0 + 1, ids, s);
    ids_of(t0 + 2, ids);
    lds_barrier();
    for (int t = t0; t < t1; ++t) {
      compute((t - t0) & 1, t);
      if (t + 1 < t1) {
        lstore(s, ((t - t0) & 1) ^ 1, t + 1);
        gload(t + 2, ids, s);
        ids_of(t + 3, ids);
      }
      lds_barrier();
    }
  }

#pragma unroll
  for (int r = 0; r < RB; ++r) {
    if (qrow[r] >= rows) continue;
    const bool live = node[r] < len;
    const float l = F32 ? sum_over_g(sums[r][0]) : sums[r][0];
    const float inv = l != 0.0f ? 1.0f / l : 0.0f;       // a row that sees nothing is zero
    if (parts == 1) {
      const size_t at = (((size_t)b * p.nodes + node[r]) * p.num_kv_heads * G + (size_t)kh * G + qrow[r] - node[r] * G) * D + 4 * g;
#pragma unroll
      for (int db = 0; db < DB; ++db) {
        const f32x4 x = live ? oacc[r][db] * inv : f32x4{0.f, 0.f, 0.f, 0.f};
        if (F32 || p.out_dtype == kF32)
          *reinterpret_cast<f32x4*>(reinterpret_cast<float*>(p.out) + at + db * 16) = x;
        else if constexpr (!F32)
          *reinterpret_cast<u32x2*>(reinterpret_cast<uint16_t*>(p.out) + at + db * 16) =
              u32x2{pack2<T>(x[0], x[1]), pack2<T>(x[2], x[3])};
      }
    } else if (live) {
      const size_t slot = (((size_t)part * p.num_seqs + b) * p.num_kv_heads + kh) * rows + qrow[r];
      if (g == 0) {
        p.part_ml[2 * slot] = m[r];
        p.part_ml[2 * slot + 1] = l;           // zero: no keys of this row, and no output row
      }
      if (l != 0.0f) {
#pragma unroll
        for (int db = 0; db < DB; ++db) *reinterpret_cast<f32x4*>(p.part_o + slot * D + db * 16 + 4 * g) = oacc[r][db] * inv;
      }
    }
  }
}

// Joins the parts of a split sequence's rows: out = sum w_s o_s / sum w_s, w_s = l_s 2^(m_s - max m).
template <typename T, int D>
__global__ void __launch_bounds__(256) tree_merge_kernel(const TreeParams p) {
  constexpr int TPR = D / 4;                   // threads of a row
  const int b = blockIdx.z, kh = blockIdx.y;
  const int G = p.group;
  const int rows = p.nodes * G;
  const int ctx = min(max(p.context_lens[b], 0), p.width);
  const int len = min(max(p.tree_lens[b], 0), p.nodes);
  const int keys = min(ctx + len, p.width);
  const int parts = (keys + p.partition - 1) / p.partition;
  if (parts <= 1) return;                      // written already
  const int row = blockIdx.x * (256 / TPR) + threadIdx.x / TPR;
  if (row >= rows) return;
  const int d = (threadIdx.x % TPR) * 4;
  const int node = row / G;
  f32x4 x = f32x4{0.f, 0.f, 0.f, 0.f};
  if (node < len) {
    const size_t step = (size_t)p.num_seqs * p.num_kv_heads * rows;
    const size_t slot0 = ((size_t)b * p.num_kv_heads + kh) * rows + row;
    constexpr int U = 8;                       // parts on the way at once
    float M = kNegInf;
    for (int s0 = 0; s0 < parts; s0 += U) {
      float mv[U];
#pragma unroll
      for (int u = 0; u < U; ++u) mv[u] = p.part_ml[2 * (slot0 + min(s0 + u, parts - 1) * step)];
#pragma unroll
      for (int u = 0; u < U; ++u) M = fmaxf(M, mv[u]);
    }
    float den = 0.0f;
    for (int s0 = 0; s0 < parts; s0 += U) {
      float mv[U], lv[U];
      f32x4 o[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const size_t slot = slot0 + min(s0 + u, parts - 1) * step;
        mv[u] = p.part_ml[2 * slot];
        lv[u] = p.part_ml[2 * slot + 1];
        o[u] = *reinterpret_cast<const f32x4*>(p.part_o + slot * D + d);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (s0 + u >= parts || lv[u] == 0.0f) continue;  // no keys of this row: its part was not written
        const float w = lv[u] * (M == kNegInf ? 1.0f : fast_exp2(mv[u] - M));   // without a maximum: only NaN
        den += w;
        x += o[u] * w;
      }
    }
    x *= den != 0.0f ? 1.0f / den : 0.0f;
  }
  const size_t at = (((size_t)b * p.nodes + node) * p.num_kv_heads * G + (size_t)kh * G + row - node * G) * D + d;
  if (sizeof(T) == 4 || p.out_dtype == kF32)
    *reinterpret_cast<f32x4*>(reinterpret_cast<float*>(p.out) + at) = x;
  else if constexpr (sizeof(T) == 2)
    *reinterpret_cast<u32x2*>(reinterpret_cast<uint16_t*>(p.out) + at) = u32x2{pack2<T>(x[0], x[1]), pack2<T>(x[2], x[3])};
}

template <typename T, int D, int RB> void tree_launch_of(TreeParams p, hipStream_t s) {
  const int rows = p.nodes * p.group;
  p.row_tiles = (rows + 64 * RB - 1) / (64 * RB);
  const dim3 grid((unsigned)((long long)p.row_tiles * p.num_kv_heads * p.num_seqs * p.max_parts));
  if (p.bs_log2 >= 4) hipLaunchKernelGGL((tree_attention_kernel<T, D, RB, true>), grid, dim3(kTreeThreads), 0, s, p);
  else hipLaunchKernelGGL((tree_attention_kernel<T, D, RB, false>), grid, dim3(kTreeThreads), 0, s, p);
  if (p.max_parts > 1) {
    constexpr int per = 256 / (D / 4);
    hipLaunchKernelGGL((tree_merge_kernel<T, D>), dim3((rows + per - 1) / per, p.num_kv_heads, p.num_seqs), dim3(256), 0, s, p);
  }
}

}  // namespace

template <typename T> void tree_launch(const TreeParams& p, int head_dim, hipStream_t s) {
  if (head_dim == 64) tree_launch_of<T, 64, 1>(p, s);
  else if (head_dim == 128) tree_launch_of<T, 128, 1>(p, s);
  else tree_launch_of<T, 256, 1>(p, s);
}

}  // namespace tv
