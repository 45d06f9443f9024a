// Attention of one query token per sequence over the 8-bit paged cache (format,
// scales and layout: tv_fp8.h):
//   out = sum_j softmax_j(scale * 2^ek q.k_j) 2^ev v_j,  j < context_lens[b]
// with ek, ev the exponents of key j's block.  A context of no tokens gives zeros.
//
// Bound: HBM, 2 D bytes per token and KV head; half of a 16-bit cache's, while
// the arithmetic per token stays.  MI355X, 32 / 8 heads of 128: 256 sequences of 512
// to 4096 tokens (1.25 GB) 200 us, 6.2 TB/s; 16 of 32768 (1.07 GB) 173 us, 6.2 TB/s.  On the vector unit a token of D 128 and four
// query heads is 14 instructions a wave with dot2 / fma, which at 8 bits would
// leave no slack over the conversions; both products go to the matrix cores.
//
// A work-group of NW waves attends one sequence for one KV head and up to 16
// query heads of its group (the columns of a 16 x 16 x 32 product; unused ones
// are zero); wave w takes tiles w, w + NW, ... of 32 tokens.
//   S^T = K Q^T: a 16-token half tile is the A operand.  Lane (c = lane % 16, g =
//     lane / 16) reads token c, bytes 64 i + 16 g .. + 15, so one load
//     instruction takes 64 contiguous bytes of each of 16 rows; the reduction
//     index of step 2 i + h is dim 64 i + 16 g + 8 h + j, and Q is read the same way.
//   O^T = V^T P^T: S^T leaves lane (n, g) with tokens 4 g .. 4 g + 3 of query n,
//     which is the B operand for reduction index 8 g + j = token 4 g + j % 4 of
//     half j / 4.  Lane (c, g) reads dims c D / 16 .. of tokens 4 g .. 4 g + 3 and
//     transposes their bytes with v_perm_b32, so neither P nor V crosses lanes.
// e4m3 is exact in fp16 and bf16, so products of K with a 16-bit Q are exact; an
// fp32 Q enters as three bf16 parts.  The scales are applied in fp32: 2^ek to the
// scores, 2^ev to the weights, which then enter the product as two bf16 parts
// (2^-17 of a weight; three, 2^-25, for fp32 queries) whatever the range of the
// scales.  Maxima, sums and accumulators are fp32.
// The running maximum is raised only when a tile exceeds it by 2^8 (as in the
// 16-bit kernel), so most tiles rescale nothing.  A tile's rows are read through
// buffer resources that end at the last attended row: rows past it are zeros,
// whatever the block holds there.  The next tile is requested before the present
// one is used, and its block ids one tile before that.
#include "tv_fp8.h"

#include "tv_split.h"

namespace tv {

namespace {

constexpr int kTT = 32;            // tokens of a wave's tile
constexpr int kCols = 16;          // query heads of a work-group
constexpr float kSlack = 8.0f;     // log2 units by which a tile may exceed the running maximum

// 16-bit type of the score product: the query's own, bf16 parts of an fp32 one.
template <typename T> struct ScoreType { using type = T; };
template <> struct ScoreType<float> { using type = __bf16; };

template <int BYTES> struct VecOf;
template <> struct VecOf<4> { using type = uint32_t; };
template <> struct VecOf<8> { using type = u32x2; };
template <> struct VecOf<16> { using type = u32x4; };

template <int BYTES>
__device__ __forceinline__ void buffer_load_v(__amdgpu_buffer_rsrc_t r, int off, uint32_t (&w)[BYTES / 4]) {
  if constexpr (BYTES == 4) {
    w[0] = __builtin_amdgcn_raw_buffer_load_b32(r, off, 0, 2);
  } else if constexpr (BYTES == 8) {
    const auto x = __builtin_amdgcn_raw_buffer_load_b64(r, off, 0, 2);
    w[0] = x[0]; w[1] = x[1];
  } else {
    const auto x = __builtin_amdgcn_raw_buffer_load_b128(r, off, 0, 2);
    w[0] = x[0]; w[1] = x[1]; w[2] = x[2]; w[3] = x[3];
  }
}

// Buffer resource of `bytes` bytes from a wave-uniform address.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t rows_rsrc(const uint8_t* base, int bytes) {
  const uint64_t a = reinterpret_cast<uint64_t>(base);
  const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)a), hi = __builtin_amdgcn_readfirstlane((uint32_t)(a >> 32));
  return __builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<void*>((uint64_t)hi << 32 | lo), (short)0,
                                           __builtin_amdgcn_readfirstlane(bytes), 0x00020000);
}

// Bytes d of four words (tokens) to four words of tokens (dims).
__device__ __forceinline__ void transpose4(uint32_t a, uint32_t b, uint32_t c, uint32_t d, uint32_t (&o)[4]) {
  const uint32_t ab01 = __builtin_amdgcn_perm(b, a, 0x05010400u);   // a0 b0 a1 b1
  const uint32_t ab23 = __builtin_amdgcn_perm(b, a, 0x07030602u);   // a2 b2 a3 b3
  const uint32_t cd01 = __builtin_amdgcn_perm(d, c, 0x05010400u);
  const uint32_t cd23 = __builtin_amdgcn_perm(d, c, 0x07030602u);
  o[0] = __builtin_amdgcn_perm(cd01, ab01, 0x05040100u);
  o[1] = __builtin_amdgcn_perm(cd01, ab01, 0x07060302u);
  o[2] = __builtin_amdgcn_perm(cd23, ab23, 0x05040100u);
  o[3] = __builtin_amdgcn_perm(cd23, ab23, 0x07060302u);
}

template <int D, int NW> struct Smem {
  float o[NW][kCols][D + 4];
  float m[NW][kCols], l[NW][kCols];
};

// T: the queries' type.  UB: the block size is 16 or a larger power of two, so
// every 16-token half tile lies in one block whose id, scales and address are uniform.
template <typename T, int D, int NW, bool UB>
__global__ void __launch_bounds__(64 * NW) paged_decode_fp8_kernel(const DecodeFp8Params p) {
  using S = typename ScoreType<T>::type;
  constexpr int QP = sizeof(T) == 4 ? 3 : 1;       // parts of a query
  constexpr int WP = sizeof(T) == 4 ? 3 : 2;       // parts of a weight
  constexpr int KV = D / 64;                       // 16-byte loads of a K row a lane
  constexpr int KS = D / 32;                       // steps of the score product
  constexpr int VB = D / 16;                       // bytes of a V row a lane, and 16-dim blocks of O
  constexpr int VW = VB / 4;
  __shared__ Smem<D, NW> sm;

  int part = 0, b, ky;
  if (p.sched) {
    const int rows = p.num_kv_heads * p.head_chunks;
    b = __builtin_amdgcn_readfirstlane(p.sched[1 + blockIdx.x / rows]);
    ky = blockIdx.x % rows;
  } else {
    // Heads fastest: they lie side by side in a block.  Partitions slowest: later
    // ones are shorter or empty, and work-groups are dealt to the CU groups in turn,
    // so with partitions next to each other some of these get only the short ones
    // (256 sequences of 512..4096 tokens in partitions of 1024: 314 us).
    ky = blockIdx.x;
    b = blockIdx.y;
    part = blockIdx.z;
  }
  const int width = p.max_blocks * p.block_size;
  const int len = min(p.context_lens[b], width);
  const int group = p.num_heads / p.num_kv_heads;
  const int kh = ky / p.head_chunks;
  const int g0 = (ky % p.head_chunks) * kCols;     // first head of the work-group in the KV head's group
  const int heads = min(kCols, group - g0);
  const int h0 = kh * group + g0;
  const int tid = threadIdx.x;
  const size_t row0 = (size_t)b * p.num_heads + h0;
  if (len <= 0) {
    if (part == 0)
      for (int i = tid; i < heads * D; i += 64 * NW) store_as(p.out, row0 * D + i, 0.0f, p.out_dtype);
    return;
  }
  const int nparts = (len + p.partition_size - 1) / p.partition_size;
  if (part >= nparts) return;
  const int start = part * p.partition_size;
  const int end = min(start + p.partition_size, len);

  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lane = tid & 63;
  const int c = lane & 15, g = lane >> 4;
  const int bs = p.block_size;
  const int* bt = p.block_tables + (size_t)b * p.bt_stride;
  const size_t unit_bytes = (size_t)bs * D;        // one (block, head)

  // Q^T: column c is query head h0 + c
  u32x4 qf[QP][KS];
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) {
    const int dim = (ks >> 1) * 64 + g * 16 + (ks & 1) * 8;
    if constexpr (QP == 1) {
      qf[0][ks] = c < heads ? *reinterpret_cast<const u32x4*>(reinterpret_cast<const T*>(p.q) + (row0 + c) * D + dim)
                            : u32x4{0, 0, 0, 0};
    } else {
      f32x4 x = f32x4{0.f, 0.f, 0.f, 0.f}, y = x;
      if (c < heads) {
        const float* qp = reinterpret_cast<const float*>(p.q) + (row0 + c) * D + dim;
        x = *reinterpret_cast<const f32x4*>(qp);
        y = *reinterpret_cast<const f32x4*>(qp + 4);
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        uint32_t h, m, l;
        split2(x[2 * i], x[2 * i + 1], h, m, l);
        qf[0][ks][i] = h; qf[1][ks][i] = m; qf[2][ks][i] = l;
        split2(y[2 * i], y[2 * i + 1], h, m, l);
        qf[0][ks][2 + i] = h; qf[1][ks][2 + i] = m; qf[2][ks][2 + i] = l;
      }
    }
  }

  f32x4 acc[VB];
#pragma unroll
  for (int i = 0; i < VB; ++i) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
  float m = kNegInf, l = 0.0f;        // of query c, the same in its four lanes (m), a lane's own share (l)
  int bad = 0;
  const float sc = p.scale * kLog2e;

  struct Tile {
    u32x4 k[2][KV];
    uint32_t v[2][4][VW];
    f32x4 ks[2], vs[2];               // scales of tokens 4 g .. 4 g + 3 of each half
  };
  auto column = [&](int t) { return UB ? t >> p.bs_log2 : t / bs; };
  auto block_of = [&](int t) { return uniform_load(bt + column(min(t, end - 1))); };   // the last token's past the end

  auto load = [&](int t0, const int (&ids)[2], Tile& w) {
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const int ts = t0 + 16 * s;
      if constexpr (UB) {
        const int id = __builtin_amdgcn_readfirstlane(ids[s]);
        const int ok = (unsigned)id < (unsigned)p.num_blocks ? -1 : 0;
        const int rows = max(0, min(16, end - ts));
        bad |= rows & ~ok;
        const size_t unit = (size_t)(id & ok) * p.num_kv_heads + kh;
        const size_t at = unit * unit_bytes + (size_t)(ts & (bs - 1)) * D;
        const auto kr = rows_rsrc(p.k_cache + at, (rows & ok) * D);
        const auto vr = rows_rsrc(p.v_cache + at, (rows & ok) * D);
#pragma unroll
        for (int i = 0; i < KV; ++i)
          w.k[s][i] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(kr, c * D + 64 * i + 16 * g, 0, 2));
#pragma unroll
        for (int i = 0; i < 4; ++i) buffer_load_v<VB>(vr, (4 * g + i) * D + c * VB, w.v[s][i]);
        const float ks = uniform_load(p.k_scale + unit), vs = uniform_load(p.v_scale + unit);
        w.ks[s] = f32x4{ks, ks, ks, ks};
        w.vs[s] = f32x4{vs, vs, vs, vs};
      } else {
        // the lane's K token, then its four V tokens
        const int tk = ts + c;
        size_t at = 0;
        bool ok = tk < end;
        if (ok) {
          const int col = column(tk), id = bt[col];
          ok = (unsigned)id < (unsigned)p.num_blocks;
          bad |= ok ? 0 : 1;
          at = ((size_t)(ok ? id : 0) * p.num_kv_heads + kh) * unit_bytes + (size_t)(tk - col * bs) * D;
        }
#pragma unroll
        for (int i = 0; i < KV; ++i)
          w.k[s][i] = ok ? *reinterpret_cast<const u32x4*>(p.k_cache + at + 64 * i + 16 * g) : u32x4{0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int tv = ts + 4 * g + i;
          bool okv = tv < end;
          size_t unit = 0;
          at = 0;
          if (okv) {
            const int col = column(tv), id = bt[col];
            okv = (unsigned)id < (unsigned)p.num_blocks;
            unit = (size_t)(okv ? id : 0) * p.num_kv_heads + kh;
            at = unit * unit_bytes + (size_t)(tv - col * bs) * D;
          }
          typename VecOf<VB>::type x{};
          if (okv) x = *reinterpret_cast<const typename VecOf<VB>::type*>(p.v_cache + at + c * VB);
          if constexpr (VW == 1) {
            w.v[s][i][0] = x;
          } else {
#pragma unroll
            for (int j = 0; j < VW; ++j) w.v[s][i][j] = x[j];
          }
          w.ks[s][i] = okv ? p.k_scale[unit] : 0.0f;
          w.vs[s][i] = okv ? p.v_scale[unit] : 0.0f;
        }
      }
    }
  };

  auto compute = [&](int t0, const Tile& w) {
    f32x4 st[2];
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      st[s] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < KV; ++i)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t lo = w.k[s][i][2 * h], hi = w.k[s][i][2 * h + 1];
          const u32x4 a = u32x4{fp8_to_pair<S, false>(lo), fp8_to_pair<S, true>(lo), fp8_to_pair<S, false>(hi),
                                fp8_to_pair<S, true>(hi)};
#pragma unroll
          for (int q = QP - 1; q >= 0; --q) st[s] = mfma16x16x32<S>(a, qf[q][2 * i + h], st[s]);
        }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float x = st[s][i] * (sc * w.ks[s][i]);
        st[s][i] = t0 + 16 * s + 4 * g + i < end ? x : kNegInf;
      }
    }
    float mt = kNegInf;
#pragma unroll
    for (int s = 0; s < 2; ++s) mt = fmaxf(mt, fmaxf(fmaxf(st[s][0], st[s][1]), fmaxf(st[s][2], st[s][3])));
    if (__builtin_amdgcn_ballot_w64(mt > m + kSlack) != 0) {
      __asm__ volatile("");   // keeps this rare block a branch (no memory clobber: table and scales stay scalar loads)
      const float mm = max_over_g(mt);
      const float mn = mm > m + kSlack ? mm : m;
      const float alpha = mn == m ? 1.0f : fast_exp2(m - mn);
      m = mn;
      l *= alpha;
#pragma unroll
      for (int i = 0; i < VB; ++i) acc[i] *= alpha;
    }
    // weights, and their bf16 parts times 2^ev: word 2 s + i of a part holds tokens 4 g + 2 i, + 1 of half s
    u32x4 pf[WP];
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float x = fast_exp2(st[s][2 * i] - m), y = fast_exp2(st[s][2 * i + 1] - m);
        l += x + y;
        x *= w.vs[s][2 * i];
        y *= w.vs[s][2 * i + 1];
#pragma unroll
        for (int q = 0; q < WP; ++q) {
          const uint32_t h = pack2<__bf16>(x, y);
          pf[q][2 * s + i] = h;
          if (q + 1 < WP) {
            x -= bf16_lo(h);
            y -= bf16_hi(h);
          }
        }
      }
#pragma unroll
    for (int j = 0; j < VW; ++j) {
      uint32_t a[4], z[4];
      transpose4(w.v[0][0][j], w.v[0][1][j], w.v[0][2][j], w.v[0][3][j], a);
      transpose4(w.v[1][0][j], w.v[1][1][j], w.v[1][2][j], w.v[1][3][j], z);
#pragma unroll
      for (int d = 0; d < 4; ++d) {
        const u32x4 vf = u32x4{fp8_to_pair<__bf16, false>(a[d]), fp8_to_pair<__bf16, true>(a[d]),
                               fp8_to_pair<__bf16, false>(z[d]), fp8_to_pair<__bf16, true>(z[d])};
#pragma unroll
        for (int q = WP - 1; q >= 0; --q) acc[4 * j + d] = mfma16x16x32<__bf16>(vf, pf[q], acc[4 * j + d]);
      }
    }
  };

  const int step = NW * kTT;
  int t = start + wave * kTT;
  if (t < end) {
    Tile ta, tb;
    int ids[2] = {block_of(t), block_of(t + 16)};
    load(t, ids, ta);
    ids[0] = block_of(t + step);
    ids[1] = block_of(t + step + 16);
    // Requests past the end ask for no rows: a branch around them would have the
    // present tile wait for the next one's loads where the paths meet.
    for (;;) {
      load(t + step, ids, tb);
      ids[0] = block_of(t + 2 * step);
      ids[1] = block_of(t + 2 * step + 16);
      compute(t, ta);
      t += step;
      if (t >= end) break;
      load(t + step, ids, ta);
      ids[0] = block_of(t + 2 * step);
      ids[1] = block_of(t + 2 * step + 16);
      compute(t, tb);
      t += step;
      if (t >= end) break;
    }
  }

  // merge the waves: acc[i] row 4 g + r of query c is dim (4 g + r) D / 16 + i
  l = sum_over_g(l);
  if (c < heads) {
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int i = 0; i < VB; ++i) sm.o[wave][c][(4 * g + r) * VB + i] = acc[i][r];
    if (g == 0) {
      sm.m[wave][c] = m;
      sm.l[wave][c] = l;
    }
  }
  const bool any_bad = __syncthreads_or(bad ? 1 : 0) != 0;
  for (int idx = tid; idx < heads * D; idx += 64 * NW) {
    const int n = idx / D, d = idx % D;
    float M = kNegInf;
#pragma unroll
    for (int w = 0; w < NW; ++w) M = fmaxf(M, sm.m[w][n]);
    float L = 0.0f, O = 0.0f;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      const float f = sm.m[w][n] == kNegInf ? 0.0f : fast_exp2(sm.m[w][n] - M);
      // a wave without tokens, or one whose scores are all NaN, has no maximum
      L += sm.m[w][n] == kNegInf ? sm.l[w][n] : sm.l[w][n] * f;
      O += sm.m[w][n] == kNegInf ? sm.o[w][n][d] : sm.o[w][n][d] * f;
    }
    const size_t row = row0 + n;
    if (nparts == 1) {
      store_limited(p.out, row * D + d, any_bad ? __builtin_nanf("") : O / L, p.out_dtype);
    } else {
      const size_t slot = row * p.max_parts + part;
      p.part_o[slot * D + d] = O / L;
      if (d == 0) {
        p.part_ml[slot * 2] = any_bad ? __builtin_nanf("") : M;
        p.part_ml[slot * 2 + 1] = L;
      }
    }
  }
}

// Merges the partitions of a (query head, sequence): out = sum_p w_p o_p / sum_p
// w_p, w_p = L_p 2^(M_p - max M).  NT threads: a dim each, and NT / D groups that
// take partitions g, g + groups, ...; eight partitions a thread are on the way at
// once (a loop of single dependent reads took most of a split call's time).
template <int D, int NT>
__global__ void __launch_bounds__(NT) paged_decode_fp8_merge_kernel(const DecodeFp8Params p) {
  constexpr int CH = 1024;          // partitions whose weights are in LDS at once
  constexpr int G = NT / D;
  __shared__ float sw[CH];
  __shared__ float red[NT / 64];
  __shared__ float snum[NT], sden[NT];
  const int h = blockIdx.x, b = blockIdx.y, tid = threadIdx.x;
  const int len = min(p.context_lens[b], p.max_blocks * p.block_size);
  const int nparts = (len + p.partition_size - 1) / p.partition_size;
  if (nparts <= 1) return;
  const size_t row = (size_t)b * p.num_heads + h;
  const float* ml = p.part_ml + row * p.max_parts * 2;
  const float* po = p.part_o + row * p.max_parts * D;
  float M = kNegInf;
  bool nan = false;
  for (int i = tid; i < nparts; i += NT) {
    const float mi = ml[2 * i];
    nan |= mi != mi;
    M = fmaxf(M, mi);
  }
  M = group_max<64>(M);
  if ((tid & 63) == 0) red[tid >> 6] = M;
  nan = __syncthreads_or(nan ? 1 : 0) != 0;
#pragma unroll
  for (int i = 0; i < NT / 64; ++i) M = fmaxf(M, red[i]);
  const int d = tid % D, g = tid / D;
  float num = 0.0f, den = 0.0f;
  for (int c0 = 0; c0 < nparts; c0 += CH) {
    const int cn = min(CH, nparts - c0);
    __syncthreads();
    for (int i = tid; i < cn; i += NT) sw[i] = ml[2 * (c0 + i) + 1] * fast_exp2(ml[2 * (c0 + i)] - M);
    __syncthreads();
    int i = g;
    for (; i + 7 * G < cn; i += 8 * G) {
      float o[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) o[u] = po[(size_t)(c0 + i + u * G) * D + d];
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        den += sw[i + u * G];
        num = fmaf(sw[i + u * G], o[u], num);
      }
    }
    for (; i < cn; i += G) {
      den += sw[i];
      num = fmaf(sw[i], po[(size_t)(c0 + i) * D + d], num);
    }
  }
  if constexpr (G > 1) {
    snum[tid] = num;
    sden[tid] = den;
    __syncthreads();
    if (g != 0) return;
#pragma unroll
    for (int k = 1; k < G; ++k) {
      num += snum[tid + k * D];
      den += sden[tid + k * D];
    }
  }
  store_limited(p.out, row * D + d, nan ? __builtin_nanf("") : num / den, p.out_dtype);
}

// Few partitions want few threads (64 heads' worth of 4: 13.9 against 15.8 us for a
// whole call), many want all of them (63 partitions of 8 heads: 13.4 against 18.9).
template <int D> void launch_merge(const DecodeFp8Params& p, hipStream_t stream) {
  const dim3 grid(p.num_heads, p.num_seqs);
  if (p.max_parts <= 16) hipLaunchKernelGGL((paged_decode_fp8_merge_kernel<D, D>), grid, dim3(D), 0, stream, p);
  else hipLaunchKernelGGL((paged_decode_fp8_merge_kernel<D, 256>), grid, dim3(256), 0, stream, p);
}

template <typename T, int D, int NW>
void launch_of(const DecodeFp8Params& p, hipStream_t stream) {
  const int rows = p.num_kv_heads * p.head_chunks;
  const dim3 grid = p.sched ? dim3(p.num_seqs * rows) : dim3(rows, p.num_seqs, p.max_parts);
  if (p.bs_log2 >= 4)
    hipLaunchKernelGGL((paged_decode_fp8_kernel<T, D, NW, true>), grid, dim3(64 * NW), 0, stream, p);
  else
    hipLaunchKernelGGL((paged_decode_fp8_kernel<T, D, NW, false>), grid, dim3(64 * NW), 0, stream, p);
  if (p.max_parts > 1)
    launch_merge<D>(p, stream);
}

template <typename T>
void launch_dims(const DecodeFp8Params& p, int head_dim, bool wide, hipStream_t stream) {
  if (head_dim == 64) wide ? launch_of<T, 64, 8>(p, stream) : launch_of<T, 64, 4>(p, stream);
  else if (head_dim == 128) launch_of<T, 128, 4>(p, stream);
  else launch_of<T, 256, 4>(p, stream);
}

}  // namespace

void launch_paged_decode_fp8(const DecodeFp8Params& p, int head_dim, int dtype, bool wide, hipStream_t stream) {
  if (dtype == kF32) launch_dims<float>(p, head_dim, wide, stream);
  else if (dtype == kF16) launch_dims<_Float16>(p, head_dim, wide, stream);
  else launch_dims<__bf16>(p, head_dim, wide, stream);
}

}  // namespace tv
