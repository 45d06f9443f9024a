// Attention of a prompt's chunk over the 8-bit paged cache (format, scales and
// layout: tv_fp8.h): query row i at position start_pos + i attends keys j <=
// start_pos + i (causal) or all start_pos + q_len keys.
//
// Bound: the matrix cores, 4 D operations per (row, query head, key), and the
// vector unit (an exponential per score), which two to four waves a SIMD overlap in
// part only.  An 8-bit key or value costs a
// conversion more than a 16-bit one, so it is made once per work-group, on the
// way from registers to LDS, and the work-group's rows are as many as the shape
// has: the query heads of a KV head are packed into one row index, row r = query
// r / G of head r % G, so that a chunk of few rows still fills its tiles and all
// G heads share one conversion.  MI355X, 32 / 8 heads of 128, bf16, 2048 rows after
// 6144 cached ones: 255 us, 942 TFLOP/s, matrix cores busy 38% of the cycles and the
// vector unit 41%; the products and the exponentials alone take 200 and the staging
// alone 105 (copies of the kernel with the other part taken out): both use LDS, and
// more of either's overlap was not to be had by offsetting the key groups against
// each other.
//
// A work-group of 4 waves owns BM = 64 RB rows of one KV head, RB blocks of 16 a
// wave, and walks tiles of BN keys: S^T = K Q^T with the key rows as operand A;
// its accumulator layout is the B operand of O^T = V^T P^T (V read transposed
// from LDS), so P stays in registers.  Tiles are double-buffered in LDS and one
// more is on the way in registers: one barrier a tile.  Where the tiles of rows
// are too few for the GPU, the keys are split between work-groups and a second
// kernel joins their parts.
// Numbers: K and V enter as their dequantised values in T, exact but for its range
// (values are limited to T's largest number; below fp16's normal numbers they are
// rounded as fp16 inputs that small are).  Scores, maxima, sums, accumulators are
// fp32; a weight is rounded to T for the second product, as in the 16-bit prefill
// kernels, and the row sum is that of the rounded weights.  That rounding is the
// largest error beside the output's own: against 64 bits 2.3e-3 in bf16 and 2.7e-4
// in fp16, with weights of two parts 1.7e-3 and 2.1e-4, the output's rounding alone.
// Two parts (as the decode kernel has, where bytes leave the time for them) cost a
// quarter: 322 against 257 us for the rows above, 36.7 against 28.4 for 512 fp16
// rows of 64-wide heads after 3584.
// A NaN in a key or value and a block id outside the cache show in the rows that
// attend that key and in no others: the key's score becomes NaN, which the mask
// replaces for rows that do not see it, and a NaN value is zero in LDS, since a
// weight of zero would not hide it.  (The row is then NaN in every dim.)
#include "tv_fp8.h"

#include <algorithm>

namespace tv {

namespace {

constexpr int kThreads = 256;

template <typename T> constexpr uint32_t kNan2 = ElemTraits<T>::kCode == kF16 ? 0x7E007E00u : 0x7FC07FC0u;

// Two e4m3 numbers times a power of two in T.
template <typename T, bool HI> __device__ __forceinline__ uint32_t scaled_pair(uint32_t w, float scale) {
  if constexpr (ElemTraits<T>::kCode == kF16)
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, scale, HI));
  else
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, HI));
}

// Four e4m3 numbers as T, limited to its range.
template <typename T> __device__ __forceinline__ u32x2 dequant4(uint32_t w, float scale) {
  if (scale > kSafeScale<T>) {
    const f32x4 x = limited<T>(fp8_to_f32x4(w) * scale);
    return u32x2{pack2<T>(x[0], x[1]), pack2<T>(x[2], x[3])};
  }
  return u32x2{scaled_pair<T, false>(w, scale), scaled_pair<T, true>(w, scale)};
}

__device__ __forceinline__ uint32_t nan_bytes(uint32_t w) { return ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; }

// NaN stays NaN (v_maximum3_f32): fmaxf would first have every operand made quiet.
// A query with a NaN score raises no maximum; its row is NaN whatever the others are.
__device__ __forceinline__ float max4(f32x4 x) {
  return __builtin_elementwise_maximum(__builtin_elementwise_maximum(x[0], x[1]), __builtin_elementwise_maximum(x[2], x[3]));
}

// UB: the block size is 16 or a larger power of two.  The rows that a wave stages
// at once (4, 8 or 16, from a multiple of their number) then lie in one block, so
// the block id, its scales and its address are scalar and cost no vector work.
template <typename T, int D, int RB, int BN, int KS, bool UB>
__global__ void __launch_bounds__(kThreads * KS, KS == 1 ? 2 : KS) prefill_fp8_kernel(const PrefillFp8Params p) {
  constexpr int BM = 64 * RB;
  constexpr int KB = BN / 16;
  constexpr int KSD = D / 32;
  constexpr int DB = D / 16;
  constexpr int P = D + 16;               // LDS row pitch (elements): conflict-free reads of both operands
  constexpr int SKT = BN * P;
  constexpr int BUF = 2 * SKT;            // K tile, then V tile
  constexpr int CPR = D / 16;             // 16-number vectors of a row
  constexpr int NV = BN * CPR / kThreads; // vectors per thread and tile, each of K and V
  constexpr int RPP = kThreads / CPR;     // tile rows of one pass over the threads
  static_assert(NV * kThreads == BN * CPR && NV >= 1, "tile shape");
  constexpr int MP = D + 4;               // row pitch (floats) of the merge of two key groups
  static_assert((KS - 1) * BM * (MP + 2) * 2 <= KS * 2 * BUF, "the merge fits the tiles' space");
  __shared__ __attribute__((aligned(16))) uint16_t smem_all[KS * 2 * BUF];

  const int grp = __builtin_amdgcn_readfirstlane(threadIdx.x / kThreads);
  const int tid = threadIdx.x % kThreads;
  uint16_t* const smem = smem_all + grp * 2 * BUF;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lane = tid & 63;
  const int g = lane >> 4, col = lane & 15;
  const int kh = blockIdx.x;
  // the longest rows first: later row tiles see more keys
  const int rt = gridDim.y - 1 - blockIdx.y;
  const int split = blockIdx.z;
  const int G = p.group;
  const int rows = p.q_len * G;
  const int kv_len = p.start_pos + p.q_len;
  const int last_pos = min((rt + 1) * BM, rows) - 1;
  const int kfull = p.causal ? min(kv_len, p.start_pos + last_pos / G + 1) : kv_len;
  const int nkt = (kfull + BN - 1) / BN;
  const int per = (nkt + p.splits - 1) / p.splits;
  const int t0 = split * per, t1 = min(t0 + per, nkt);
  const int row0 = rt * BM + wave * RB * 16;

  int qrow[RB], qpos[RB];
  u32x4 qf[RB][KSD];
#pragma unroll
  for (int r = 0; r < RB; ++r) {
    qrow[r] = row0 + r * 16 + col;
    qpos[r] = qrow[r] / G;
    const T* qg = reinterpret_cast<const T*>(p.q) + (size_t)qpos[r] * p.q_stride +
                  (size_t)(kh * G + qrow[r] - qpos[r] * G) * D + g * 8;
#pragma unroll
    for (int ks = 0; ks < KSD; ++ks)
      qf[r][ks] = qrow[r] < rows ? *reinterpret_cast<const u32x4*>(qg + ks * 32) : u32x4{0, 0, 0, 0};
  }

  // staging: this thread's vectors are chunk ch of tile rows sr + RPP i
  const int sr = tid / CPR, ch = tid % CPR;
  const int wr = wave * (64 / CPR);       // first of the wave's rows
  const int bs = p.block_size;
  const size_t unit_bytes = (size_t)bs * D;
  auto column = [&](int key) { return UB ? key >> p.bs_log2 : key / bs; };
  // the key whose block a vector's rows are looked up by, and that key kept inside the sequence
  auto key_of = [&](int t, int i) { return t * BN + (UB ? wr : sr) + RPP * i; };
  struct Ids { int id[NV]; };
  struct Stage { u32x4 k[NV], v[NV]; float ks[NV], vs[NV]; int ok[NV]; };
  auto ids_of = [&](int t, Ids& x) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int* at = p.block_table + column(min(key_of(t, i), kv_len - 1));
      x.id[i] = UB ? uniform_load(at) : *at;
    }
  };
  auto gload = [&](int t, const Ids& x, Stage& s) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int id = UB ? __builtin_amdgcn_readfirstlane(x.id[i]) : x.id[i];
      s.ok[i] = (unsigned)id < (unsigned)p.num_blocks ? -1 : 0;
      const size_t unit = (size_t)(id & s.ok[i]) * p.num_kv_heads + kh;
      if constexpr (UB) {
        // rows past the sequence's end are the block's own (whatever it holds there)
        const size_t at = unit * unit_bytes + (size_t)(key_of(t, i) & (bs - 1)) * D;
        const int lane_at = (sr - wr) * D + ch * 16;
        s.k[i] = *reinterpret_cast<const u32x4*>(p.k_cache + at + lane_at);
        s.v[i] = *reinterpret_cast<const u32x4*>(p.v_cache + at + lane_at);
        s.ks[i] = uniform_load(p.k_scale + unit);
        s.vs[i] = uniform_load(p.v_scale + unit);
      } else {
        const int key = min(key_of(t, i), kv_len - 1);
        const size_t at = unit * unit_bytes + (size_t)(key - column(key) * bs) * D + ch * 16;
        s.k[i] = *reinterpret_cast<const u32x4*>(p.k_cache + at);
        s.v[i] = *reinterpret_cast<const u32x4*>(p.v_cache + at);
        s.ks[i] = p.k_scale[unit];
        s.vs[i] = p.v_scale[unit];
      }
    }
  };
  auto put = [&](int b, int i, const u32x2 (&kw)[4], const u32x2 (&vw)[4]) {
    uint16_t* dk = smem + b * BUF + (sr + RPP * i) * P + ch * 16;
    *reinterpret_cast<u32x4*>(dk) = u32x4{kw[0][0], kw[0][1], kw[1][0], kw[1][1]};
    *reinterpret_cast<u32x4*>(dk + 8) = u32x4{kw[2][0], kw[2][1], kw[3][0], kw[3][1]};
    *reinterpret_cast<u32x4*>(dk + SKT) = u32x4{vw[0][0], vw[0][1], vw[1][0], vw[1][1]};
    *reinterpret_cast<u32x4*>(dk + SKT + 8) = u32x4{vw[2][0], vw[2][1], vw[3][0], vw[3][1]};
  };
  auto lstore = [&](const Stage& s, int b, int t) {
    // Nearly every tile: all of its keys inside the sequence, in blocks of the cache, no NaN among the
    // values and scales whose values T holds.
    uint32_t nan = 0;
    uint32_t largest = (t + 1) * BN > kv_len ? ~0u : 0u;   // of the scales, as bits: uniform where they are
#pragma unroll
    for (int i = 0; i < NV; ++i) {
#pragma unroll
      for (int j = 0; j < 4; ++j) nan |= (s.v[i][j] & 0x7f7f7f7fu) + 0x01010101u;
      largest = max(largest, max(__builtin_bit_cast(uint32_t, s.ks[i]), __builtin_bit_cast(uint32_t, s.vs[i])) | ~s.ok[i]);
    }
    uint64_t special = __builtin_amdgcn_ballot_w64((nan & 0x80808080u) != 0);
    special |= __builtin_amdgcn_ballot_w64(largest > __builtin_bit_cast(uint32_t, kSafeScale<T>));
    if (special == 0) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        u32x2 kw[4], vw[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          kw[j] = u32x2{scaled_pair<T, false>(s.k[i][j], s.ks[i]), scaled_pair<T, true>(s.k[i][j], s.ks[i])};
          vw[j] = u32x2{scaled_pair<T, false>(s.v[i][j], s.vs[i]), scaled_pair<T, true>(s.v[i][j], s.vs[i])};
        }
        put(b, i, kw, vw);
      }
      return;
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      u32x4 k = s.k[i], v = s.v[i];
      const bool in = t * BN + sr + RPP * i < kv_len;
      if (!in) k = v = u32x4{0, 0, 0, 0};        // masked, and their values zero
      const bool poison = in && (s.ok[i] == 0 || (nan_bytes(v[0]) | nan_bytes(v[1]) | nan_bytes(v[2]) | nan_bytes(v[3])));
      u32x2 kw[4], vw[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t bad = (nan_bytes(v[j]) >> 7) * 0xffu;
        kw[j] = dequant4<T>(k[j], s.ks[i]);
        vw[j] = dequant4<T>(s.ok[i] ? v[j] & ~bad : 0u, s.vs[i]);
      }
      if (poison) kw[0][0] = kNan2<T>;
      put(b, i, kw, vw);
    }
  };

  f32x4 oacc[RB][DB + 1];
  float m[RB];
#pragma unroll
  for (int r = 0; r < RB; ++r) {
#pragma unroll
    for (int db = 0; db <= DB; ++db) oacc[r][db] = f32x4{0.f, 0.f, 0.f, 0.f};
    m[r] = kNegInf;
  }
  const u32x4 ones = u32x4{kOnes2<T>, kOnes2<T>, kOnes2<T>, kOnes2<T>};
  const float c = p.scale * kLog2e;
  const int first_seen = p.causal ? p.start_pos + row0 / G : kv_len - 1;   // last key that all of the wave's rows see

  auto compute = [&](int b, int t) {
    const uint16_t* sk = smem + b * BUF;
    const uint16_t* sv = sk + SKT;
    const int k0 = t * BN;
    f32x4 st[RB][KB];
    // independent products next to each other: the sums of one score are KB RB apart
#pragma unroll
    for (int ks = 0; ks < KSD; ++ks) {
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) {
        const u32x4 kf = *reinterpret_cast<const u32x4*>(sk + (kb * 16 + col) * P + ks * 32 + g * 8);
#pragma unroll
        for (int r = 0; r < RB; ++r)
          st[r][kb] = mfma16x16x32<T>(kf, qf[r][ks], ks ? st[r][kb] : f32x4{0.f, 0.f, 0.f, 0.f});
      }
    }
    __builtin_amdgcn_sched_barrier(0);   // all products before the first use of one: no waits between them
    // V^T operands of the first 32 keys: from LDS while the softmax runs
    u32x4 vf[DB];
    auto values = [&](int x) {
#pragma unroll
      for (int db = 0; db < DB; ++db) {
        const uint16_t* a = sv + (x * 32 + 4 * g + (col >> 2)) * P + db * 16 + 4 * (col & 3);
        const u32x2 lo = lds_read_tr16(a);
        const u32x2 hi = lds_read_tr16(a + 16 * P);
        vf[db] = u32x4{lo[0], lo[1], hi[0], hi[1]};
      }
    };
    values(0);
    float base[RB];
    bool need = false;
#pragma unroll
    for (int r = 0; r < RB; ++r) {
      base[r] = m[r] == kNegInf ? 0.0f : m[r];
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int i = 0; i < 4; ++i) st[r][kb][i] = fmaf(st[r][kb][i], c, -base[r]);
    }
    if (k0 + BN - 1 > first_seen) {
      __asm__ volatile("");                // a branch, not 32 selects in every tile
#pragma unroll
      for (int r = 0; r < RB; ++r) {
        const int rel = (p.causal ? min(kv_len - 1, p.start_pos + qpos[r]) : kv_len - 1) - (k0 + 4 * g);
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
          for (int i = 0; i < 4; ++i) st[r][kb][i] = kb * 16 + i <= rel ? st[r][kb][i] : kNegInf;
      }
    }
    // the running maximum is raised only when a tile passes it by 2^8
    float mt[RB];
#pragma unroll
    for (int r = 0; r < RB; ++r) {
      mt[r] = max4(st[r][0]);
#pragma unroll
      for (int kb = 1; kb < KB; ++kb) mt[r] = __builtin_elementwise_maximum(mt[r], max4(st[r][kb]));
      need |= mt[r] > (m[r] == kNegInf ? kNegInf : 8.0f);
    }
    if (__builtin_amdgcn_ballot_w64(need) != 0) {
      __asm__ volatile("" ::: "memory");   // keeps this rare block a branch
#pragma unroll
      for (int r = 0; r < RB; ++r) {
        const float mm = max_over_g(mt[r]);               // relative to base
        const bool raise = mm > (m[r] == kNegInf ? kNegInf : 8.0f);
        const float delta = raise ? mm : 0.0f;
        const float alpha = raise && m[r] != kNegInf ? fast_exp2(-delta) : 1.0f;
        m[r] = raise ? base[r] + delta : m[r];
#pragma unroll
        for (int db = 0; db <= DB; ++db) oacc[r][db] *= alpha;
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) st[r][kb] -= delta;
      }
    }
    u32x4 pf[RB][BN / 32];
#pragma unroll
    for (int r = 0; r < RB; ++r)
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) {
        // reduction index 8g + j: key 4g + j of block 2 x (j < 4), 4g + j - 4 of block 2 x + 1
        pf[r][kb >> 1][(kb & 1) * 2] = pack2<T>(fast_exp2(st[r][kb][0]), fast_exp2(st[r][kb][1]));
        pf[r][kb >> 1][(kb & 1) * 2 + 1] = pack2<T>(fast_exp2(st[r][kb][2]), fast_exp2(st[r][kb][3]));
      }
#pragma unroll
    for (int x = 0; x < BN / 32; ++x) {
#pragma unroll
      for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int r = 0; r < RB; ++r) oacc[r][db] = mfma16x16x32<T>(vf[db], pf[r][x], oacc[r][db]);
      if (x + 1 < BN / 32) values(x + 1);
#pragma unroll
      for (int r = 0; r < RB; ++r) oacc[r][DB] = mfma16x16x32<T>(ones, pf[r][x], oacc[r][DB]);
    }
  };

  // group grp takes tiles t0 + grp, t0 + grp + KS, ...
  const int steps = (t1 - t0 + KS - 1) / KS;
  if (steps > 0) {
    Ids ids;
    Stage s;
    const int first = t0 + grp;
    ids_of(first, ids);
    gload(first, ids, s);
    ids_of(first + KS, ids);
    lstore(s, 0, first);
    gload(first + KS, ids, s);
    ids_of(first + 2 * KS, ids);
    lds_barrier();
    for (int j = 0; j < steps; ++j) {
      const int t = first + j * KS;
      if (t < t1) compute(j & 1, t);
      if (j + 1 < steps) {
        lstore(s, (j & 1) ^ 1, t + KS);
        gload(t + 2 * KS, ids, s);
        ids_of(t + 3 * KS, ids);
      }
      lds_barrier();
    }
  }
  if constexpr (KS > 1) {
    // the other groups' rows join the first's through LDS
    float* so = reinterpret_cast<float*>(smem_all);
    float* sml = so + (KS - 1) * BM * MP;
    if (grp > 0) {
#pragma unroll
      for (int r = 0; r < RB; ++r) {
        const int row = (grp - 1) * BM + (wave * RB + r) * 16 + col;
#pragma unroll
        for (int db = 0; db < DB; ++db) *reinterpret_cast<f32x4*>(so + row * MP + db * 16 + 4 * g) = oacc[r][db];
        if (g == 0) {
          sml[2 * row] = m[r];
          sml[2 * row + 1] = oacc[r][DB][0];
        }
      }
    }
    lds_barrier();
    if (grp > 0) return;
#pragma unroll
    for (int r = 0; r < RB; ++r) {
#pragma unroll
      for (int k = 0; k < KS - 1; ++k) {
        const int row = k * BM + (wave * RB + r) * 16 + col;
        const float m1 = sml[2 * row], l1 = sml[2 * row + 1];
        const float M = fmaxf(m[r], m1);
        // without a maximum a group has no keys of this row (zeros) or only NaN
        const float f0 = m[r] == kNegInf ? 1.0f : fast_exp2(m[r] - M);
        const float f1 = m1 == kNegInf ? 1.0f : fast_exp2(m1 - M);
        m[r] = M;
#pragma unroll
        for (int db = 0; db < DB; ++db)
          oacc[r][db] = oacc[r][db] * f0 + *reinterpret_cast<const f32x4*>(so + row * MP + db * 16 + 4 * g) * f1;
        oacc[r][DB][0] = oacc[r][DB][0] * f0 + l1 * f1;
      }
    }
  }

#pragma unroll
  for (int r = 0; r < RB; ++r) {
    if (qrow[r] >= rows) continue;
    const float l = oacc[r][DB][0];
    const float inv = 1.0f / l;
    if (p.splits == 1) {
      const size_t at = (size_t)qpos[r] * p.out_stride + (size_t)(kh * G + qrow[r] - qpos[r] * G) * D + 4 * g;
#pragma unroll
      for (int db = 0; db < DB; ++db) {
        const f32x4 x = oacc[r][db] * inv;
        if (p.out_dtype == kF32)
          *reinterpret_cast<f32x4*>(reinterpret_cast<float*>(p.out) + at + db * 16) = x;
        else
          *reinterpret_cast<u32x2*>(reinterpret_cast<uint16_t*>(p.out) + at + db * 16) =
              u32x2{pack2<T>(x[0], x[1]), pack2<T>(x[2], x[3])};
      }
    } else {
      const size_t slot = ((size_t)split * p.num_kv_heads + kh) * rows + qrow[r];
      if (g == 0) {
        p.part_ml[2 * slot] = m[r];
        p.part_ml[2 * slot + 1] = l;      // zero: no keys of this row, and no output row
      }
      if (l != 0.0f) {
#pragma unroll
        for (int db = 0; db < DB; ++db)
          *reinterpret_cast<f32x4*>(p.part_o + slot * D + db * 16 + 4 * g) = oacc[r][db] * inv;
      }
    }
  }
}

// Joins the key splits of a row: out = sum w_s o_s / sum w_s, w_s = l_s 2^(m_s - max m).
template <typename T, int D>
__global__ void __launch_bounds__(256) prefill_fp8_merge_kernel(const PrefillFp8Params p) {
  constexpr int TPR = D / 4;              // threads of a row
  const int rows = p.q_len * p.group;
  const long long item = (long long)blockIdx.x * (256 / TPR) + threadIdx.x / TPR;
  if (item >= (long long)rows * p.num_kv_heads) return;
  const int kh = (int)(item / rows), row = (int)(item - (long long)kh * rows);
  const int d = (threadIdx.x % TPR) * 4;
  const size_t step = (size_t)p.num_kv_heads * rows;
  const size_t slot0 = (size_t)kh * rows + row;
  constexpr int U = 8;                    // parts on the way at once; past the last one they are read again and weigh nothing
  float M = kNegInf;
  for (int s0 = 0; s0 < p.splits; s0 += U) {
    float mv[U];
#pragma unroll
    for (int u = 0; u < U; ++u) mv[u] = p.part_ml[2 * (slot0 + min(s0 + u, p.splits - 1) * step)];
#pragma unroll
    for (int u = 0; u < U; ++u) M = fmaxf(M, mv[u]);
  }
  f32x4 num = f32x4{0.f, 0.f, 0.f, 0.f};
  float den = 0.0f;
  for (int s0 = 0; s0 < p.splits; s0 += U) {
    float mv[U], lv[U];
    f32x4 o[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const size_t slot = slot0 + min(s0 + u, p.splits - 1) * step;
      mv[u] = p.part_ml[2 * slot];
      lv[u] = p.part_ml[2 * slot + 1];
      o[u] = *reinterpret_cast<const f32x4*>(p.part_o + slot * D + d);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (s0 + u >= p.splits || lv[u] == 0.0f) continue;   // no keys of this row: its part was not written
      const float w = lv[u] * fast_exp2(mv[u] - M);
      den += w;
      num += o[u] * w;
    }
  }
  const f32x4 x = num * (1.0f / den);
  const int pos = row / p.group;
  const size_t at = (size_t)pos * p.out_stride + (size_t)(kh * p.group + row - pos * p.group) * D + d;
  if (p.out_dtype == kF32)
    *reinterpret_cast<f32x4*>(reinterpret_cast<float*>(p.out) + at) = x;
  else
    *reinterpret_cast<u32x2*>(reinterpret_cast<uint16_t*>(p.out) + at) = u32x2{pack2<T>(x[0], x[1]), pack2<T>(x[2], x[3])};
}

int tile_keys(int head_dim) { return head_dim == 256 ? 32 : 64; }

template <typename T, int D, int RB, int BN, int KS>
void launch_of(const PrefillFp8Params& p, hipStream_t stream) {
  const long long rows = (long long)p.q_len * p.group;
  const dim3 grid(p.num_kv_heads, (unsigned)((rows + 64 * RB - 1) / (64 * RB)), p.splits);
  if (p.bs_log2 >= 4)
    hipLaunchKernelGGL((prefill_fp8_kernel<T, D, RB, BN, KS, true>), grid, dim3(kThreads * KS), 0, stream, p);
  else
    hipLaunchKernelGGL((prefill_fp8_kernel<T, D, RB, BN, KS, false>), grid, dim3(kThreads * KS), 0, stream, p);
  if (p.splits > 1) {
    const long long items = rows * p.num_kv_heads, per = 256 / (D / 4);
    hipLaunchKernelGGL((prefill_fp8_merge_kernel<T, D>), dim3((unsigned)((items + per - 1) / per)), dim3(256), 0, stream, p);
  }
}

template <typename T> void launch_dims(const PrefillFp8Params& p, int head_dim, bool wide, hipStream_t stream) {
  if (head_dim == 64) wide ? launch_of<T, 64, 2, 64, 2>(p, stream) : launch_of<T, 64, 1, 64, 4>(p, stream);
  else if (head_dim == 128) wide ? launch_of<T, 128, 2, 64, 2>(p, stream) : launch_of<T, 128, 1, 32, 4>(p, stream);
  else launch_of<T, 256, 1, 32, 1>(p, stream);
}

// 128-row work-groups of two key groups (8 waves) where they give nearly every CU
// one, else 64 rows and four key groups (16 waves).  A CU holds one of either.
// MI355X, bf16, us, 128 rows / 64 rows: 32 / 8 heads of 128, 1024 rows after 4000
// cached ones (256 tiles of 128) 94 / 109, with 128 rows in one group of 4 waves 134;
// 512 after 2000 50 / 33; 2048 after 6144 255 / 322, in one group 252; 32 / 4 heads of
// 64, 512 after 3584 46 / 28, with two groups of 64 rows 37.  Heads of 256 have 64
// rows and one group: 512 after 3584 (32 / 8) 125, 2048 after 6144 690 (697 TFLOP/s).
bool wide_rows(long long rows, int num_kv_heads, int head_dim, int cus) {
  return head_dim != 256 && (rows + 127) / 128 * num_kv_heads * 8 >= 7LL * cus;
}

}  // namespace

// Key splits: as many as give every CU its work-groups, each of at least four key tiles.
int prefill_fp8_splits(int q_len, int start_pos, int num_heads, int num_kv_heads, int head_dim, int cus) {
  const long long rows = (long long)q_len * (num_heads / num_kv_heads);
  if (wide_rows(rows, num_kv_heads, head_dim, cus)) return 1;
  const long long wgs = (rows + 63) / 64 * num_kv_heads;
  const int tiles = (int)(((long long)start_pos + q_len + tile_keys(head_dim) - 1) / tile_keys(head_dim));
  const long long want = (head_dim == 256 ? 2LL : 1LL) * cus / std::max(1LL, wgs);
  return (int)std::max(1LL, std::min({want, (long long)tiles / 4, 64LL}));
}

void launch_prefill_fp8(const PrefillFp8Params& p, int head_dim, int dtype, int cus, hipStream_t stream) {
  const bool wide = p.splits == 1 && wide_rows((long long)p.q_len * p.group, p.num_kv_heads, head_dim, cus);
  if (dtype == kF16) launch_dims<_Float16>(p, head_dim, wide, stream);
  else launch_dims<__bf16>(p, head_dim, wide, stream);
}

}  // namespace tv
