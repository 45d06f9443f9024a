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
//
// Tiles come by LDS DMA, one that is read and one on the way: loads into registers made a wave wait for all of them
// wherever it reused one.  Work is dealt by the lengths on the device (work_groups): what a launch of whole units takes
// is its longest unit's time.  MI355X, kernel and merge, us; GB/s and TFLOP/s of the keys and products that cannot be left out:
//   64 sequences x 16 nodes over 512..4096 tokens, 32 / 8 heads of 128, fp16       117 +  9   4.7 TB/s   loads
//   2 x 32 over 31000..32700, 32 / 8 of 128, bf16                                   55 +  9   4.2 TB/s   loads
//   32 x 61 over 1000..6000, 32 / 4 of 64, bf16                                     87 + 10   470 TFLOP/s
//   16 x 32 over 2000, 32 / 8 of 128, fp32                                         166        103 TFLOP/s   matrix units
// (a large read reaches 7.0 TB/s, a large product 1140 TFLOP/s, 153 in fp32).  One tile on the way, drained before the next is
// requested, is what bounds the first two: the loads alone take 113 and 50 us, 5.1 and 5.3 TB/s.  In the third the matrix units are busy for
// 27% of the cycles and the vector units for 42%: a head of 64 has 128 products a weight, and its exponential, scaling,
// maximum and conversion cost more cycles than those; its four row tiles read 382 MB past the L2 caches, since
// they are at different keys at a time.  Without loads it takes 74 us, without the softmax 70, with loads alone 65.  Its
// instance (heads of 64, 32 rows a wave) spills 14 vector registers, used where a unit begins and ends.
#pragma once

#include "tv_device_cache.h"
#include "tv_draft.h"
#include "tv_fp8.h"
#include "tv_tile_dma.h"

#include <algorithm>
#include <type_traits>

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

// The chunk permutation of a tile's row r (16-byte chunks, by exclusive or): without it all rows of a column
// lie in the same banks.
template <int CPR> __device__ __forceinline__ int tree_perm(int r) {
  if constexpr (CPR == 8) return (((r >> 1) & 3) << 1) | ((r >> 3) & 1);
  else return ((r & 7) << 1) | ((r >> 3) & 1);
}

// A row tile of a sequence: its lengths, and the tiles of its keys.
struct TreeUnit { int b, rt, ctx, len, keys, tiles; };

// Four waves, 16 RB rows a wave.  BN keys a tile, two tiles in LDS: one that is read and one on the way.
// UB: the block size is 16 or a larger power of two: the rows of a load lie in one
// block, whose id and address are then scalar, and whose range ends at the last key.
template <typename T, int D, int RB, int BN, int EU, bool NT, bool UB>
__global__ void __launch_bounds__(kTreeThreads, EU) tree_attention_kernel(const TreeParams p) {
  constexpr bool F32 = sizeof(T) == 4;
  constexpr int THREADS = kTreeThreads;
  constexpr int WAVES = THREADS / 64;
  constexpr int BM = 64 * RB;
  constexpr int KB = BN / 16;
  constexpr int DB = D / 16;
  constexpr int VEC = 16 / (int)sizeof(T);
  constexpr int CPR = D / VEC;                 // 16-byte chunks of a row
  constexpr int ROW = D * (int)sizeof(T);      // bytes of a row
  constexpr int TILE = BN * ROW;
  constexpr int STAGE = 2 * TILE;              // K tile, then V tile
  constexpr int NV = BN * CPR / THREADS;       // loads of a wave for a tile, each of K and V
  constexpr int RPI = 64 / CPR;                // rows of a load
  constexpr int RPP = WAVES * RPI;             // rows of all waves' loads
  static_assert(NV * THREADS == BN * CPR && NV >= 1 && NV <= 32, "tile shape");
  __shared__ __attribute__((aligned(16))) unsigned char smem[2 * STAGE];
  __shared__ int wave_tiles[WAVES];
  __shared__ int start_seq, start_tile;        // the work-group's first tile

  const uint32_t smem_at = sgpr((uint32_t)(uintptr_t)(__attribute__((address_space(3))) unsigned char*)smem);
  const int tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lane = tid & 63;
  const int g = lane >> 4, col = lane & 15;
  const int G = p.group;
  const int rows = p.nodes * G;

  // The walk's state is the same in all lanes; saying so keeps it in scalar registers.
  auto uniform = [](int x) { return __builtin_amdgcn_readfirstlane(x); };
  auto unit_of = [&](int b) {
    TreeUnit u;
    u.b = uniform(b);
    u.rt = 0;
    u.ctx = uniform(min(max(uniform_load(p.context_lens + u.b), 0), p.width));
    u.len = uniform(min(max(uniform_load(p.tree_lens + u.b), 0), p.nodes));
    u.keys = uniform(min(u.ctx + u.len, p.width));
    u.tiles = uniform((u.keys + BN - 1) / BN);
    return u;
  };

  // ---- this work-group's tiles: `left` of them from tile `tile` of unit cu on, of one KV head ----
  TreeUnit cu;
  int tile = 0, left = 0, kh;
  int wg = blockIdx.x;
  if (p.work_groups) {
    // the heads of a group read the same keys' neighbouring slices of the cache's rows at about the same time
    const int group = wg / p.num_kv_heads;
    kh = wg - group * p.num_kv_heads;
    // prefix sums of the sequences' tiles (fewer than 2^31): a thread has `per` consecutive sequences
    const int per = (p.num_seqs + THREADS - 1) / THREADS;
    auto tiles_of = [&](int b) -> int {
      if (b >= p.num_seqs) return 0;
      const int ctx = min(max(p.context_lens[b], 0), p.width), len = min(max(p.tree_lens[b], 0), p.nodes);
      return (min(ctx + len, p.width) + BN - 1) / BN * ((len * G + BM - 1) / BM);
    };
    const int one = tiles_of(tid * per);
    int mine = one;
    for (int k = 1; k < per; ++k) mine += tiles_of(tid * per + k);
    int upto = mine;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      const int other = __builtin_amdgcn_ds_bpermute((lane - d) << 2, upto);
      if (lane >= d) upto += other;
    }
    if (lane == 63) wave_tiles[wave] = upto;
    if (tid == 0) start_seq = -1;
    __syncthreads();
    int total = 0, before = upto - mine;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      if (w < wave) before += wave_tiles[w];
      total += wave_tiles[w];
    }
    const int share = max((int)(((unsigned)total + p.groups - 1) / (unsigned)p.groups), p.least_tiles);
    const long long from = (long long)share * group;
    const int here = from < total ? (int)from : total;       // a group past the last tile has none
    for (int k = 0; k < per; ++k) {
      const int b = tid * per + k, n = k ? tiles_of(b) : one;
      if (wg == 0 && b < p.num_seqs) p.first_tiles[b] = before;
      if (here >= before && here < before + n) {
        start_seq = b;
        start_tile = here - before;
      }
      before += n;
    }
    if (wg == 0 && tid == 0) p.first_tiles[p.num_seqs] = share;
    __syncthreads();
    const int b0 = __builtin_amdgcn_readfirstlane(start_seq);
    if (b0 < 0) return;                        // no tiles are left for it
    left = uniform(min(share, total - here));
    tile = __builtin_amdgcn_readfirstlane(start_tile);
    cu = unit_of(b0);
    cu.rt = uniform(tile / cu.tiles);
    tile = uniform(tile - cu.rt * cu.tiles);
  } else {
    const int rt = wg % p.row_tiles;
    wg /= p.row_tiles;
    kh = wg % p.num_kv_heads;
    cu = unit_of(wg / p.num_kv_heads);
    cu.rt = rt;
    left = rt * BM < cu.len * G ? cu.tiles : 0;          // nothing to attend: zeros
  }
  // The next row tile, or the first of the next sequence that has a node.
  auto advance = [&](TreeUnit& u) {
    u.rt = uniform(u.rt + 1);
    if (u.rt * BM < u.len * G) return;
    do u = unit_of(u.b + 1);
    while (uniform(u.b + 1 < p.num_seqs && u.len == 0));
  };

  // The wave's place among the tile's rows.  Few rows leave waves without any, which only load; work-groups 256 apart mostly
  // share a CU (8 XCDs of 32), and their rows go to different SIMDs.  MI355X, us, all waves in their places at work / so, over
  // 500..2000 tokens: 16 rows 61 / 55 (64 x 2 nodes, 32 / 4 heads of 64, fp32), 32 rows 68 / 65 (64 x 8, 32 / 8 of 128, fp16), 48 rows
  // 70 / 66 and 64 rows 69 / 71 (16 x 12 and 16 x 16, 32 / 8 of 128, fp32).
  const int part = (wave + (rows <= 16 ? 1 : 2) * (blockIdx.x >> 8)) & 3;
  int qrow[RB], node[RB];
  constexpr int QF = F32 ? D / 16 : D / 32;
  u32x4 qf[RB][QF];
  f32x4 oacc[RB][DB];
  f32x4 sums[RB];                              // 16-bit: every lane's row sum; fp32: of the lane's own keys, in [0]
  float m[RB];
  auto begin_unit = [&]() {
#pragma unroll
    for (int r = 0; r < RB; ++r) {
      qrow[r] = cu.rt * BM + (part * RB + r) * 16 + col;
      node[r] = qrow[r] / G;
      const T* qg = reinterpret_cast<const T*>(p.q) + (size_t)cu.b * p.q_seq_stride + (size_t)node[r] * p.q_node_stride +
                    (size_t)(kh * G + qrow[r] - node[r] * G) * D;
      // fp32: k index of step 4 f + e, lane g: 16 f + 4 g + e, on both operands
#pragma unroll
      for (int f = 0; f < QF; ++f)
        qf[r][f] = node[r] < cu.len ? *reinterpret_cast<const u32x4*>(qg + (F32 ? 16 * f + 4 * g : 32 * f + 8 * g))
                                    : u32x4{0, 0, 0, 0};
#pragma unroll
      for (int db = 0; db < DB; ++db) oacc[r][db] = f32x4{0.f, 0.f, 0.f, 0.f};
      sums[r] = f32x4{0.f, 0.f, 0.f, 0.f};
      m[r] = kNegInf;
    }
  };

  // loading: load i of a wave fills tile rows wr + RPP i .. + RPI - 1, a lane chunk lane % CPR of row lane / CPR of them
  const int wr = wave * RPI;
  const int lr = lane / CPR;
  const int bs = p.block_size;
  const long long row_bytes = (long long)p.num_kv_heads * ROW;
  const uint32_t block_bytes = (uint32_t)(bs * row_bytes);
  const u64 kc = reinterpret_cast<u64>(p.k_cache) + (u64)kh * ROW, vc = reinterpret_cast<u64>(p.v_cache) + (u64)kh * ROW;
  uint32_t voff[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i)
    voff[i] = (UB ? (uint32_t)(lr * row_bytes) : 0u) + (((lane % CPR) ^ tree_perm<CPR>(wr + RPP * i + lr)) * 16);
  // The next tile to request: tile lt of unit lu, with `to_load` to come; its block ids are looked up a tile ahead.
  TreeUnit lu = cu;
  int lt = tile, to_load = left;
  // UB: load i's in lane i, by a vector load: it arrives with the tile before, where a scalar load would have every read
  // from LDS wait for it.  Else each lane's own.
  struct Ids { int id[UB ? 1 : NV]; } ids;
  auto look_up = [&]() {
    if (to_load <= 0) return;
    const int* table = p.block_tables + (size_t)lu.b * p.bt_stride;
    if constexpr (UB) {
      ids.id[0] = table[min(lt * BN + wr + RPP * (lane % NV), lu.keys - 1) >> p.bs_log2];
    } else {
#pragma unroll
      for (int i = 0; i < NV; ++i) ids.id[i] = table[min(lt * BN + wr + RPP * i + lr, lu.keys - 1) / bs];
    }
  };
  // Requests it into a stage and moves on; returns bit i for a load whose block is outside the cache.  Where no tile is
  // left the requests are empty, so that their number is the same every time.
  auto issue = [&](int stage) -> uint32_t {
    uint32_t bad = 0;
    uint32_t range[NV];                        // bytes of a load; rows past the last key arrive as zeros
#pragma unroll
    for (int i = 0; i < NV; ++i) range[i] = (uint32_t)((RPI - 1) * row_bytes + ROW);
    if (UB && !(to_load > 0 && (lt + 1) * BN <= lu.keys)) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int count = to_load > 0 ? min(RPI, lu.keys - (lt * BN + wr + RPP * i)) : 0;
        range[i] = count > 0 ? (uint32_t)((count - 1) * row_bytes + ROW) : 0u;
      }
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const uint32_t at = sgpr(smem_at + stage * STAGE + (wr + RPP * i) * ROW);
      if constexpr (UB) {
        const uint32_t id = __builtin_amdgcn_readlane(ids.id[0], i);
        const bool ok = id < (uint32_t)p.num_blocks;
        const u64 off = (u64)(ok ? id : 0) * block_bytes + (uint32_t)((lt * BN + wr + RPP * i) & (bs - 1)) * (uint32_t)row_bytes;
        const u64 ka = kc + off, va = vc + off;
        const uint32_t n = sgpr(ok ? range[i] : 0u);
        const u32x4 kr = u32x4{sgpr((uint32_t)ka), sgpr((uint32_t)(ka >> 32)), n, 0x00020000u};
        const u32x4 vr = u32x4{sgpr((uint32_t)va), sgpr((uint32_t)(va >> 32)), n, 0x00020000u};
        if constexpr (NT) {
          load_lds16_nt(kr, at, voff[i]);
          load_lds16_nt(vr, sgpr(at + TILE), voff[i]);
        } else {
          load_lds16(kr, at, voff[i]);
          load_lds16(vr, sgpr(at + TILE), voff[i]);
        }
        bad |= ok ? 0u : 1u << i;
      } else {
        const bool ok = (unsigned)ids.id[i] < (unsigned)p.num_blocks;
        const int key = min(lt * BN + wr + RPP * i + lr, lu.keys - 1);
        const long long off = ((long long)(ok ? ids.id[i] : 0) * bs + key % bs) * row_bytes + voff[i];
        load_lds16_at(reinterpret_cast<const void*>(kc + off), at);
        load_lds16_at(reinterpret_cast<const void*>(vc + off), sgpr(at + TILE));
        bad |= ok ? 0u : 1u << i;
      }
    }
    if (--to_load > 0 && ++lt == lu.tiles) {
      lt = 0;
      advance(lu);
    }
    return bad;
  };
  // A wave's own loads of a tile that not all rows see in the same way.
  auto amend = [&](int t, uint32_t bad, int stage) {   // of unit cu
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      u32x4* kp = reinterpret_cast<u32x4*>(smem + stage * STAGE + (wr + RPP * i) * ROW + lane * 16);
      u32x4* vp = kp + TILE / 16;
      u32x4 k = *kp, v = *vp;
      const bool in = t * BN + wr + RPP * i + lr < cu.keys;
      const bool lost = bad >> i & 1;
      if (!in || lost) k = v = u32x4{0, 0, 0, 0};
      bool poison = in && lost;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t w = not_finite<T>(v[j]);
        poison = poison || w != 0;
        v[j] &= ~w;
      }
      if (poison) k[0] = kTreeNan<T>;
      *kp = k;
      *vp = v;
    }
  };

  // Bits of the keys k0 .. k0 + 63 that a live node sees.
  auto seen_from = [&](int n, int k0) -> u64 {
    const u64* words = p.mask + (size_t)cu.b * p.mask_seq_stride + (size_t)n * p.words;
    const int left = cu.keys - k0;
    u64 bits;
    if (k0 >= cu.ctx) {
      const int w = (k0 - cu.ctx) >> 6, s = (k0 - cu.ctx) & 63;
      bits = w < p.words ? words[w] >> s : 0;
      if (s && w + 1 < p.words) bits |= words[w + 1] << (64 - s);
    } else {
      const int s = cu.ctx - k0;                  // context keys of the tile
      bits = s >= 64 ? ~0ull : ((1ull << s) - 1) | words[0] << s;
    }
    return left >= 64 ? bits : left > 0 ? bits & ((1ull << left) - 1) : 0;
  };

  const float c = p.scale * kLog2e;

  auto compute = [&](int stage, int t) {
    const unsigned char* sk = smem + stage * STAGE;
    const unsigned char* sv = sk + TILE;
    const int k0 = t * BN;
    f32x4 st[RB][KB];
    // reads first, then products, so that one wait covers many reads
    constexpr int FM = F32 && D == 256 ? 8 : 16, FG = QF * KB > FM ? FM / KB : QF;      // reads of at most FM fragments at once
#pragma unroll
    for (int f0 = 0; f0 < QF; f0 += FG) {
      u32x4 kf[FG][KB];
#pragma unroll
      for (int f = 0; f < FG; ++f)
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
          kf[f][kb] = *reinterpret_cast<const u32x4*>(sk + (kb * 16 + col) * ROW + ((4 * (f0 + f) + g) ^ tree_perm<CPR>(col)) * 16);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int f = 0; f < FG; ++f)
#pragma unroll
        for (int e = 0; e < (F32 ? 4 : 1); ++e)
#pragma unroll
          for (int kb = 0; kb < KB; ++kb)
#pragma unroll
            for (int r = 0; r < RB; ++r) {
              const f32x4 acc = f0 + f + e ? st[r][kb] : f32x4{0.f, 0.f, 0.f, 0.f};
              if constexpr (F32)
                st[r][kb] = __builtin_amdgcn_mfma_f32_16x16x4f32(u32_as_f32(kf[f][kb][e]), u32_as_f32(qf[r][f0 + f][e]), acc, 0, 0, 0);
              else
                st[r][kb] = mfma16x16x32<T>(kf[f][kb], qf[r][f0 + f], acc);
            }
    }
    __builtin_amdgcn_sched_barrier(0);
    // V^T operands of the first 32 keys: from LDS while the softmax runs
    u32x4 vf[F32 ? 1 : 2][F32 ? 1 : DB];
    auto values = [&](int x) {
#pragma unroll
      for (int db = 0; db < DB; ++db) {
        const int r = x * 32 + 4 * g + (col >> 2);      // and 16 rows on, whose permutation is the same
        const unsigned char* at = sv + r * ROW + ((db * 2 + ((col & 3) >> 1)) ^ tree_perm<CPR>(r)) * 16 + (col & 1) * 8;
        const u32x2 lo = lds_read_tr16(reinterpret_cast<const uint16_t*>(at));
        const u32x2 hi = lds_read_tr16(reinterpret_cast<const uint16_t*>(at + 16 * ROW));
        vf[x & 1][db] = u32x4{lo[0], lo[1], hi[0], hi[1]};
      }
    };
    // fp32: element e of vector b of a row is A row col of accumulator 4 b + e, which so holds d = 64 b + 4 col + e
    constexpr int VS = !F32 ? 1 : D == 256 ? 2 : 4 * KB;      // rows on the way: all, where there are registers for them
    f32x4 vw[VS][F32 ? D / 64 : 1];
    auto value_row = [&](int y) {              // key 4 g + y % 4 of block y / 4
#pragma unroll
      for (int b = 0; b < D / 64; ++b) {
        const int r = y / 4 * 16 + 4 * g + y % 4;
        vw[y % VS][b] = *reinterpret_cast<const f32x4*>(sv + r * ROW + ((b * 16 + col) ^ tree_perm<CPR>(r)) * 16);
      }
    };
    if constexpr (F32) {
#pragma unroll
      for (int y = 0; y < VS; ++y) value_row(y);
    } else {
      values(0);
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
    if (k0 + BN > cu.ctx) {
#pragma unroll
      for (int r = 0; r < RB; ++r) {
        const u64 bits = node[r] < cu.len ? seen_from(node[r], k0) >> (4 * g) : 0;
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
        for (int i = 0; i < 4; ++i) {
          const int y = 4 * kb + i;
#pragma unroll
          for (int db = 0; db < DB; ++db)
#pragma unroll
            for (int r = 0; r < RB; ++r)
              oacc[r][db] = __builtin_amdgcn_mfma_f32_16x16x4f32(vw[y % VS][db / 4][db % 4], st[r][kb][i], oacc[r][db], 0, 0, 0);
          if (y + VS < 4 * KB) value_row(y + VS);
        }
      }
    } else {
      const u32x4 ones = u32x4{kOnes2<T>, kOnes2<T>, kOnes2<T>, kOnes2<T>};
#pragma unroll
      for (int x = 0; x < BN / 32; ++x) {
        if (x + 1 < BN / 32) values(x + 1);
        u32x4 pf[RB];
        // reduction index 8g + j: key 4g + j of block 2 x (j < 4), 4g + j - 4 of block 2 x + 1
#pragma unroll
        for (int r = 0; r < RB; ++r)
          pf[r] = u32x4{pack2<T>(st[r][2 * x][0], st[r][2 * x][1]), pack2<T>(st[r][2 * x][2], st[r][2 * x][3]),
                        pack2<T>(st[r][2 * x + 1][0], st[r][2 * x + 1][1]), pack2<T>(st[r][2 * x + 1][2], st[r][2 * x + 1][3])};
#pragma unroll
        for (int db = 0; db < DB; ++db)
#pragma unroll
          for (int r = 0; r < RB; ++r) oacc[r][db] = mfma16x16x32<T>(vf[x & 1][db], pf[r], oacc[r][db]);
#pragma unroll
        for (int r = 0; r < RB; ++r) sums[r] = mfma16x16x32<T>(ones, pf[r], sums[r]);
      }
    }
  };

  // Four consecutive outputs of a lane's row, and their place: the 16-element block and the element in it.
  auto four = [&](int r, int db) -> f32x4 {
    const int b = db & ~3, i = db & 3;
    if constexpr (F32) return f32x4{oacc[r][b][i], oacc[r][b + 1][i], oacc[r][b + 2][i], oacc[r][b + 3][i]};
    else return oacc[r][db];
  };
  auto block_of = [&](int db) { return F32 ? (db & ~3) + g : db; };
  auto element_of = [&](int db) { return F32 ? 4 * (db & 3) : 4 * g; };
  // A unit's rows go out, or, where other work-groups have tiles of it, its part of them.
  auto end_unit = [&](int first, int past, int slot) {
    const bool whole = first == 0 && past == cu.tiles;
#pragma unroll
    for (int r = 0; r < RB; ++r) {
      const float l = F32 ? sum_over_g(sums[r][0]) : sums[r][0];
      const bool live = node[r] < cu.len;
      if (!(live || (!p.work_groups && qrow[r] < rows))) continue;
      const float inv = l != 0.0f ? 1.0f / l : 0.0f;     // a row that sees nothing is zero
      if (whole) {
        const size_t at = (((size_t)cu.b * p.nodes + node[r]) * p.num_kv_heads * G + (size_t)kh * G + qrow[r] - node[r] * G) * D;
#pragma unroll
        for (int db = 0; db < DB; ++db) {
          const f32x4 x = live ? four(r, db) * inv : f32x4{0.f, 0.f, 0.f, 0.f};
          const size_t to = at + block_of(db) * 16 + element_of(db);
          if (F32 || p.out_dtype == kF32)
            *reinterpret_cast<f32x4*>(reinterpret_cast<float*>(p.out) + to) = x;
          else if constexpr (!F32)
            *reinterpret_cast<u32x2*>(reinterpret_cast<uint16_t*>(p.out) + to) =
                u32x2{pack2<T>(x[0], x[1]), pack2<T>(x[2], x[3])};
        }
      } else {
        const size_t at = (size_t)slot * BM + (part * RB + r) * 16 + col;
        if (g == 0) {
          p.part_ml[2 * at] = m[r];
          p.part_ml[2 * at + 1] = l;           // zero: no keys of this row
        }
#pragma unroll
        for (int db = 0; db < DB; ++db)
          *reinterpret_cast<f32x4*>(p.part_o + (at - col) * D + block_of(db) * 256 + col * 16 + element_of(db)) = four(r, db) * inv;
      }
    }
  };

  begin_unit();
  if (left <= 0) {
    end_unit(0, cu.tiles, 0);
    return;
  }
  look_up();
  uint32_t lost = issue(0);
  look_up();
  int first = tile, slot = 2 * wg;
  int stage = 0;
  while (true) {
    wait_vmcnt<0>();
    if (__builtin_amdgcn_ballot_w64((tile + 1) * BN > cu.ctx || lost != 0) != 0) {
      __asm__ volatile("" ::: "memory");
      amend(tile, lost, stage);
    }
    lds_barrier();                             // the tile is there; the one before has been read
    lost = issue(stage ^ 1);
    look_up();
    if (cu.rt * BM + part * RB * 16 < cu.len * G) compute(stage, tile);
    stage ^= 1;
    ++tile;
    --left;
    if (tile == cu.tiles || left == 0) {
      end_unit(first, tile, slot);
      if (left == 0) break;
      advance(cu);
      begin_unit();
      first = tile = 0;
      slot |= 1;
    }
  }
  wait_vmcnt<0>();                             // (empty requests write zeros)
}

// Joins the parts of a unit's rows that several work-groups have: out = sum w_s o_s / sum w_s, w_s = l_s 2^(m_s - max m).
// A work-group has 16 rows of a row tile, whose parts are the same for all its threads, in the order in which the kernel's
// accumulators left them, [D / 16][16 rows][16].
template <typename T, int D, int TILE_ROWS>
__global__ void __launch_bounds__(256) tree_merge_kernel(const TreeParams p) {
  constexpr int R = D / 64;                    // 16-byte vectors a thread, of one row
  const int b = blockIdx.z, kh = blockIdx.y;
  const int G = p.group;
  const int len = min(max(uniform_load(p.tree_lens + b), 0), p.nodes);
  const int ctx = min(max(uniform_load(p.context_lens + b), 0), p.width);
  const int share = uniform_load(p.first_tiles + p.num_seqs), first = uniform_load(p.first_tiles + b);
  const int tid = threadIdx.x;
  const int row = blockIdx.x * 16 + tid / 4 % 16;
  if (row >= p.nodes * G) return;
  const int node = row / G;
  const int d = tid / 64 * 16 + tid % 4 * 4;   // and 64 on, for every further vector
  const size_t out_at = (((size_t)b * p.nodes + node) * p.num_kv_heads * G + (size_t)kh * G + row - node * G) * D + d;
  auto store = [&](int r, f32x4 x) {
    if (sizeof(T) == 4 || p.out_dtype == kF32)
      *reinterpret_cast<f32x4*>(reinterpret_cast<float*>(p.out) + out_at + 64 * r) = x;
    else if constexpr (sizeof(T) == 2)
      *reinterpret_cast<u32x2*>(reinterpret_cast<uint16_t*>(p.out) + out_at + 64 * r) =
          u32x2{pack2<T>(x[0], x[1]), pack2<T>(x[2], x[3])};
  };
  f32x4 x[R];
#pragma unroll
  for (int r = 0; r < R; ++r) x[r] = f32x4{0.f, 0.f, 0.f, 0.f};
  if (node < len) {                            // else padding: zeros
    const unsigned tiles = (unsigned)(min(ctx + len, p.width) + p.tile_keys - 1) / p.tile_keys;
    const unsigned rt = blockIdx.x * 16 / TILE_ROWS;
    const unsigned from = first + rt * tiles;
    const int g0 = from / (unsigned)share, g1 = (from + tiles - 1) / (unsigned)share;
    if (g0 == g1) return;                      // written already
    const int parts = g1 - g0 + 1;
    // a part that begins where its work-group does is that one's first, others its second
    const bool second = from > (unsigned)share * g0;
    auto place = [&](int s) -> size_t {        // of the 16 rows
      const unsigned slot = 2 * ((unsigned)(g0 + s) * p.num_kv_heads + kh) + (s == 0 && second ? 1 : 0);
      return (size_t)slot * TILE_ROWS + (blockIdx.x * 16 - rt * TILE_ROWS);
    };
    float den = 0.0f, M = kNegInf;
    // U parts on the way at once; past the last one they are read again and weigh nothing
    auto join = [&](auto count) {
      constexpr int U = decltype(count)::value;
      for (int s0 = 0; s0 < parts; s0 += U) {
        float mv[U], lv[U];
        f32x4 o[U][R];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const size_t at = place(min(s0 + u, parts - 1));
          const float2 ml = reinterpret_cast<const float2*>(p.part_ml)[at + tid / 4 % 16];
          mv[u] = ml.x;
          lv[u] = ml.y;
#pragma unroll
          for (int r = 0; r < R; ++r) o[u][r] = reinterpret_cast<const f32x4*>(p.part_o + at * D)[tid + 256 * r];
        }
        float top = M;
#pragma unroll
        for (int u = 0; u < U; ++u) top = fmaxf(top, mv[u]);
        const float f = M == kNegInf ? 1.0f : fast_exp2(M - top);    // (without a maximum: nothing, or NaN)
        den *= f;
#pragma unroll
        for (int r = 0; r < R; ++r) x[r] *= f;
        M = top;
#pragma unroll
        for (int u = 0; u < U; ++u) {
          if (s0 + u >= parts || lv[u] == 0.0f) continue;            // no keys of this row
          const float w = lv[u] * (mv[u] == kNegInf ? 1.0f : fast_exp2(mv[u] - M));
          den += w;
#pragma unroll
          for (int r = 0; r < R; ++r) x[r] += o[u][r] * w;
        }
      }
    };
    if (parts <= 2) join(std::integral_constant<int, 2>());
    else join(std::integral_constant<int, (D == 256 ? 4 : 8)>());
    const float inv = den != 0.0f ? 1.0f / den : 0.0f;
#pragma unroll
    for (int r = 0; r < R; ++r) x[r] *= inv;
  }
#pragma unroll
  for (int r = 0; r < R; ++r) store(r, x[r]);
}

// What a (type, head size, number of rows) runs as.  A wave of 32 rows reads a key or value from LDS once for both its row
// blocks, but is half empty at 64 rows, and holds twice the registers; keys that one row tile reads bypass the
// caches, those that several read do not.  MI355X, us, 16 rows a wave / 16 cached / 32 / 32 cached, fp16, 32 / 8 heads of 128 over
// 500..2000 tokens: 64 x 16 nodes (64 rows) 74 / 81 / 89 / 95, 32 x 32 (128) 67 / 62 / 56 / 60, 16 x 48 (192) 59 / 55 / 53 / 47,
// 16 x 64 (256) 75 / 65 / 57 / 52.
template <typename T, int D, int RB, int BN, int EU, bool NT> struct TreeShape {
  static constexpr int kRows = 64 * RB, kKeys = BN;

  static void launch(TreeParams p, hipStream_t s) {
    const int rows = p.nodes * p.group;
    p.tile_rows = kRows;
    p.tile_keys = BN;
    p.row_tiles = (rows + kRows - 1) / kRows;
    if (p.work_groups) {
      p.groups = std::max(1, p.work_groups / p.num_kv_heads);
      p.work_groups = p.groups * p.num_kv_heads;
      p.part_ml = p.part_o + (size_t)2 * p.work_groups * kRows * D;
      p.first_tiles = reinterpret_cast<int*>(p.part_ml + (size_t)4 * p.work_groups * kRows);
    }
    const dim3 grid(p.work_groups ? p.work_groups : (unsigned)((long long)p.row_tiles * p.num_kv_heads * p.num_seqs));
    if (p.bs_log2 >= 4)
      hipLaunchKernelGGL((tree_attention_kernel<T, D, RB, BN, EU, NT, true>), grid, dim3(kTreeThreads), 0, s, p);
    else
      hipLaunchKernelGGL((tree_attention_kernel<T, D, RB, BN, EU, NT, false>), grid, dim3(kTreeThreads), 0, s, p);
    if (p.work_groups)
      hipLaunchKernelGGL((tree_merge_kernel<T, D, kRows>), dim3((rows + 15) / 16, p.num_kv_heads, p.num_seqs), dim3(256), 0, s, p);
  }
  static long long resident() {
    static std::atomic<long long> slots[kMaxDevices];
    return resident_work_groups(slots, tree_attention_kernel<T, D, RB, BN, EU, NT, true>, kTreeThreads);
  }
};

// Calls f with the shape for so many rows (nodes times query heads of a KV head).
template <typename T, int D, typename F> auto tree_shape(long long rows, F f) {
  if constexpr (sizeof(T) == 4) {
    constexpr int BN = D == 256 ? 16 : 32;
    return rows <= 64 ? f(TreeShape<T, D, 1, BN, 2, true>()) : f(TreeShape<T, D, 1, BN, 2, false>());
  } else if constexpr (D == 256) {
    return rows <= 64 ? f(TreeShape<T, D, 1, 32, 2, true>()) : f(TreeShape<T, D, 1, 32, 2, false>());
  } else {
    constexpr int BN = D == 64 ? 64 : 32, EU = D == 64 ? 3 : 2;
    if (rows <= 64) return f(TreeShape<T, D, 1, 64, (D == 64 ? 4 : 2), true>());
    return rows <= 128 ? f(TreeShape<T, D, 2, BN, EU, true>()) : f(TreeShape<T, D, 2, BN, EU, false>());
  }
}
template <typename T, typename F> auto tree_shape(long long rows, int head_dim, F f) {
  if (head_dim == 64) return tree_shape<T, 64>(rows, f);
  if (head_dim == 128) return tree_shape<T, 128>(rows, f);
  return tree_shape<T, 256>(rows, f);
}

}  // namespace

template <typename T> void tree_launch(const TreeParams& p, int head_dim, hipStream_t s) {
  tree_shape<T>((long long)p.nodes * p.group, head_dim, [&](auto shape) { shape.launch(p, s); });
}
template <typename T> TreeShapeInfo tree_info(long long rows, int head_dim) {
  return tree_shape<T>(rows, head_dim, [](auto shape) {
    return TreeShapeInfo{decltype(shape)::kRows, decltype(shape)::kKeys, [] { return decltype(shape)::resident(); }};
  });
}

}  // namespace tv
