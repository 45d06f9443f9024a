// The path through a draft tree that the model's logits accept
// (tv_verify_draft_tree).
//
// Greedy: the first maximum of a row.  Sampled, with m a row's maximum and e_i =
// 2^((x_i - m) log2(e) / temperature), S = sum e_i: children in the order of their indexes are
// taken while u S is not below their summed e; a path that ends draws from the other
// tokens, the first at which their e sum to more than u S - E, E the children's.
//
// Precision: whether u is below a sum needs fp32 only where u is not next to it: within
// `unsure` of a child's bound the sums are taken again in fp64.  With h = 2^-24, half a step of
// fp32, an fp32 sum of a row is off by less than a relative (107 + 11 rounds) h:
//   67 h  arguments: (x - m) c has four roundings (with those of c), so e is off by 4 ln(2) |y| h, y
//         its exponent; the maximum has e = 1, so of V terms the weighted mean of |y| is
//         below log2(V) <= 24.  Raising a maximum in several steps adds up to the same |y|.
//   40 h  sums in a vector, over lanes and over waves, with 3 h for each product by an exponential
//   11 h  a round, of which `rounds` follow each other: kStatVecs vectors of a thread, or
//         kPartsAtOnce parts of a row: eight additions and a raised maximum
// unsure is more than twice that, 2^-16 + 2^-19 rounds.  The draw is in fp64 throughout: a large
// vocabulary has a bound every 2^-17 of S, and an error of d in u S meets one with
// probability 2^17 d.
//
// A sum in fp64 is bound by one CU's fp64 units.  MI355X, us of a captured call, ordinary / with u of one sequence on a bound: 2 x 32
// nodes of 128256 logits in bf16 34 / 64, 64 x 16 of them 86 / 120, 64 x 64 of 32000 in fp32 41 / 49, 1 x 4 of 2^20 in fp32
// 41 / 337.
//
// A walk over a path is serial and reads its rows only; reading the rows that it may come to
// first is parallel (all_rows): bound by HBM, then by the latency of the walk and the draw, a work-group a sequence.
// MI355X: greedy, 64 sequences of 16 nodes, 32000 fp32 logits: chains' rows 12 us, walk 4; sampled, 2 of 32, 128256 in
// bf16: rows 8.3, walk 6.9, rest 4.5, draw 8.7.
#include "tv_draft.h"

#include <algorithm>

namespace tv {

namespace {

constexpr int kWalkThreads = 512;
constexpr int kStatThreads = 256;
constexpr int kStatVecs = 8;             // 16-byte vectors a thread of the stats kernel: 32 KiB of a row
constexpr int kPartsAtOnce = 8;          // parts of a row that a lane of the walk fetches together
constexpr int kChainRows = 8;            // work-groups a part for a chain's rows
constexpr int kDrawThreads = 256;
constexpr int kDrawPer = 8;              // elements a thread of the draw kernels
constexpr int kDrawChunk = kDrawThreads * kDrawPer;

// What is known of a row, or of a part of it: the first maximum, and sum e relative to it.
struct RowStat {
  u64 key;                               // order of the maximum, then ~index; all ones: a NaN; 0: nothing above -inf
  float m, s;
};

__device__ __forceinline__ uint32_t order_bits(float x) {
  const uint32_t u = __builtin_bit_cast(uint32_t, x);
  if (x == 0.0f) return 0x80000000u;     // -0 equals +0
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float from_order_bits(uint32_t o) { return u32_as_f32(o & 0x80000000u ? o & 0x7fffffffu : ~o); }
__device__ __forceinline__ u64 shfl_xor64(u64 x, int mask) {
  const uint32_t lo = __builtin_bit_cast(uint32_t, shfl_xor(u32_as_f32((uint32_t)x), mask));
  const uint32_t hi = __builtin_bit_cast(uint32_t, shfl_xor(u32_as_f32((uint32_t)(x >> 32)), mask));
  return (u64)hi << 32 | lo;
}
__device__ __forceinline__ double wave_sum(double x) {
#pragma unroll
  for (int d = 1; d < 64; d *= 2) x += __builtin_bit_cast(double, shfl_xor64(__builtin_bit_cast(u64, x), d));
  return x;
}
__device__ __forceinline__ double lane_value(double x, int lane) {
  const u64 u = __builtin_bit_cast(u64, x);
  const u64 lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)u, lane);
  const u64 hi = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(u >> 32), lane);
  return __builtin_bit_cast(double, hi << 32 | lo);
}
// Sum over the lanes up to and with this one.
__device__ __forceinline__ double wave_prefix(double x, int lane) {
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const u64 u = __builtin_bit_cast(u64, x);
    const int from = (lane - d) << 2;
    const uint32_t lo = __builtin_amdgcn_ds_bpermute(from, (int)(uint32_t)u);
    const uint32_t hi = __builtin_amdgcn_ds_bpermute(from, (int)(uint32_t)(u >> 32));
    if (lane >= d) x += __builtin_bit_cast(double, (u64)hi << 32 | lo);
  }
  return x;
}

// e of a logit in fp32.  -inf and what lies far below give 0.
__device__ __forceinline__ float weight(float x, float m, float c) { return fast_exp2(fmaxf((x - m) * c, -200.0f)); }

// e of a logit in fp64: 2^n and the Taylor series of exp over |x| <= ln(2) / 2, whose
// terms past the twelfth are below 2^-52.
__device__ __forceinline__ double weight64(float x, float m, double c) {
  const double y = ((double)x - m) * c;
  if (!(y >= -1000.0)) return 0.0;
  const double n = rint(y);
  const double r = (y - n) * 0.69314718055994530942;
  double e = 1.0 / 479001600.0;
  constexpr double kInv[] = {1.0 / 39916800, 1.0 / 3628800, 1.0 / 362880, 1.0 / 40320, 1.0 / 5040, 1.0 / 720,
                             1.0 / 120, 1.0 / 24, 1.0 / 6, 0.5, 1.0, 1.0};
#pragma unroll
  for (int i = 0; i < 12; ++i) e = fma(e, r, kInv[i]);
  return __builtin_bit_cast(double, __builtin_bit_cast(u64, e) + ((u64)(long long)(int)n << 52));
}

template <typename T> __device__ __forceinline__ float max_of(const u32x4& w, float m) {
  // NaN stays NaN
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (sizeof(T) == 4) {
      m = __builtin_elementwise_maximum(m, u32_as_f32(w[i]));
    } else {
      float a, b;
      unpack2<T>(w[i], a, b);
      m = __builtin_elementwise_maximum(m, __builtin_elementwise_maximum(a, b));
    }
  }
  return m;
}
template <typename T> __device__ __forceinline__ float sum_of(const u32x4& w, float m, float c) {
  float s = 0.0f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (sizeof(T) == 4) {
      s += weight(u32_as_f32(w[i]), m, c);
    } else {
      float a, b;
      unpack2<T>(w[i], a, b);
      s += weight(a, m, c) + weight(b, m, c);
    }
  }
  return s;
}

// One thread's share of x[0 .. n): 16-byte vectors tid, tid + threads, .. from the first 16-byte boundary on, and of the
// elements before and behind them one each.  Its maximum, the index of the first of that value, and sum e.
struct ThreadStat {
  float m, s;
  int idx;
};
template <typename T>
__device__ __forceinline__ ThreadStat thread_stat(const T* x, int n, int tid, int threads, float c, bool sampled) {
  constexpr int EPV = 16 / (int)sizeof(T);
  constexpr int U = kStatVecs;
  const int head = min(n, (int)((16 - ((uintptr_t)x & 15)) & 15) / (int)sizeof(T));
  const int vecs = (n - head) / EPV;
  const u32x4* body = reinterpret_cast<const u32x4*>(x + head);
  float m = kNegInf, s = 0.0f;
  int at = 0;                            // the vector, or -1 - element, that the maximum was met in first
  u32x4 held = u32x4{0, 0, 0, 0};        // that vector
  const int tail = head + vecs * EPV + tid;
  const float first = tid < head ? to_float<T>(x[tid]) : kNegInf;
  const float last = tail < n ? to_float<T>(x[tail]) : kNegInf;
  if (first != kNegInf) {
    m = first;
    at = -1 - tid;
    s = 1.0f;
  }
  for (int v0 = tid; v0 < vecs; v0 += threads * U) {
    u32x4 w[U];
#pragma unroll
    for (int u = 0; u < U; ++u) w[u] = body[min(v0 + u * threads, vecs - 1)];
    const float old = m;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const float was = m;
      m = max_of<T>(w[u], m);            // (past the end the last vector again: it raises nothing)
      const bool up = m != was;          // a NaN differs from itself: at is not looked at then
      at = up ? min(v0 + u * threads, vecs - 1) : at;
#pragma unroll
      for (int i = 0; i < 4; ++i) held[i] = up ? w[u][i] : held[i];
    }
    if (sampled && m > kNegInf) {
      if (m > old) s *= old > kNegInf ? weight(old, m, c) : 0.0f;
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (v0 + u * threads < vecs) s += sum_of<T>(w[u], m, c);
    }
  }
  const float was = m;
  m = __builtin_elementwise_maximum(m, last);
  if (m > was) {
    at = -1 - tail;
    s *= was > kNegInf ? weight(was, m, c) : 0.0f;
  }
  if (last > kNegInf && m > kNegInf) s += weight(last, m, c);
  int idx = -1 - at;
  if (at >= 0) {
#pragma unroll
    for (int e = EPV - 1; e >= 0; --e) {
      float v;
      if constexpr (sizeof(T) == 4) {
        v = u32_as_f32(held[e]);
      } else {
        float lo, hi;
        unpack2<T>(held[e / 2], lo, hi);
        v = e % 2 ? hi : lo;
      }
      if (v == m) idx = head + at * EPV + e;
    }
  }
  return ThreadStat{m, s, idx};
}

// One thread's share of the sum of e in fp64, of the same vectors and elements.  Vectors are on the way four at a time, and
// their exponentials do not wait for each other (an element at a time, with 64 threads for rows read first: 417 us where a
// call now takes 64).
template <typename T>
__device__ __forceinline__ double thread_sum64(const T* x, int n, int tid, int threads, float m, double c) {
  constexpr int EPV = 16 / (int)sizeof(T);
  constexpr int U = 4;
  const int head = min(n, (int)((16 - ((uintptr_t)x & 15)) & 15) / (int)sizeof(T));
  const int vecs = (n - head) / EPV;
  const u32x4* body = reinterpret_cast<const u32x4*>(x + head);
  const int tail = head + vecs * EPV + tid;
  double sum = tid < head ? weight64(to_float<T>(x[tid]), m, c) : 0.0;
  if (tail < n) sum += weight64(to_float<T>(x[tail]), m, c);
  for (int v0 = tid; v0 < vecs; v0 += threads * U) {
    u32x4 w[U];
#pragma unroll
    for (int u = 0; u < U; ++u) w[u] = body[min(v0 + u * threads, vecs - 1)];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (v0 + u * threads >= vecs) break;
      double e = 0.0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (sizeof(T) == 4) {
          e += weight64(u32_as_f32(w[u][i]), m, c);
        } else {
          float a, b;
          unpack2<T>(w[u][i], a, b);
          e += weight64(a, m, c) + weight64(b, m, c);
        }
      }
      sum += e;
    }
  }
  return sum;
}

// The wave's shares as one, in every lane.
__device__ __forceinline__ RowStat wave_stat(const ThreadStat& t, float c, bool sampled) {
  RowStat r{0, group_max<64>(t.m), 0.0f};                    // (of a NaN nothing is used)
  if (__builtin_amdgcn_ballot_w64(t.m != t.m)) {
    r.key = ~0ull;
    return r;
  }
  if (r.m == kNegInf) return r;
  // nearly always one lane has it; of several the lowest index
  u64 with = __builtin_amdgcn_ballot_w64(t.m == r.m);
  int idx = 0x7fffffff;
  while (with) {
    idx = min(idx, __builtin_amdgcn_readlane(t.idx, __builtin_ctzll(with)));
    with &= with - 1;
  }
  r.key = (u64)order_bits(r.m) << 32 | (uint32_t)~idx;
  if (sampled) r.s = group_sum<64>(t.m > kNegInf ? t.s * weight(t.m, r.m, c) : 0.0f);
  return r;
}

__device__ __forceinline__ float temperature_of(const VerifyParams& p, int b) {
  const float t = p.temperatures ? p.temperatures[b] : 0.0f;
  return t >= 0x1p-126f ? t : 0.0f;
}

// What the walk leaves for the draw after a sequence's last node.
struct DrawJob {
  double mass;                           // E: the children's e
  double u;
  int node;                              // -1: no draw
  float top;                             // m
  int children;
  int token[kDraftMaxNodes];             // theirs, each once
};

struct VerifyWorkspace {
  DrawJob* jobs;                         // [B]
  double* sums;                          // [B, draw chunks]
  RowStat* stats;                        // [B * nodes, stat parts]
};

__host__ __device__ inline VerifyWorkspace workspace_of(const VerifyParams& p) {
  VerifyWorkspace w;
  w.jobs = reinterpret_cast<DrawJob*>(p.workspace);
  w.sums = reinterpret_cast<double*>(w.jobs + p.num_seqs);
  w.stats = reinterpret_cast<RowStat*>(w.sums + (size_t)p.num_seqs * p.draw_chunks);
  return w;
}

// Parts of the rows of all live nodes; where all sequences are greedy, of those that a path can come to: of a node's
// children only that with the largest logit (the lowest token of equal ones, the first of equal tokens) can be the row's first
// maximum, so there is one path, a chain from node 0 on, known without its rows.  Every work-group finds it for itself;
// p.chain_rows of them share its rows.
template <typename T> __global__ void __launch_bounds__(kStatThreads) verify_stats_kernel(const VerifyParams p) {
  static_assert(kStatThreads == kDraftMaxNodes, "a thread for every node");
  __shared__ RowStat red[kStatThreads / 64];
  __shared__ u64 best[kDraftMaxNodes];                       // of a node's children: logit, token, node, by order
  const int part = blockIdx.y, tid = threadIdx.x;
  const bool chain = p.chain_rows != 0;
  const int each = chain ? p.chain_rows : p.nodes;
  // sequences innermost: the rows of a chain's end, often none, are spread over the XCDs
  const int j = blockIdx.x / p.num_seqs, b = blockIdx.x - j * p.num_seqs;
  const int len = min(p.tree_lens[b], p.nodes);
  const T* row0 = reinterpret_cast<const T*>(p.logits) + (size_t)b * p.nodes * p.row_stride;
  if (chain) {
    best[tid] = 0;
    __syncthreads();
    if (tid < len) {
      const int tok = p.tokens[(size_t)b * p.nodes + tid], up = p.parents[(size_t)b * p.nodes + tid];
      if (up >= 0 && up < tid && (unsigned)tok < (unsigned)p.vocab) {
        const float x = to_float<T>(row0[(size_t)up * p.row_stride + tok]);
        atomicMax(&best[up], (u64)order_bits(x) << 32 | (u64)(0xffffffu - tok) << 8 | (u64)(255 - tid));
      }
    }
    __syncthreads();
  }
  auto further = [&](int node, int steps) {                  // along the chain (children have higher indexes)
    for (; steps > 0 && node < len; --steps) {
      const u64 child = best[node];
      node = __builtin_amdgcn_readfirstlane(child ? 255 - (int)(child & 255u) : len);
    }
    return node;
  };
  const float temp = temperature_of(p, b);
  const bool sampled = temp > 0.0f;
  const float c = sampled ? kLog2e / temp : 0.0f;
  const int first = part * p.stat_size, n = min(p.stat_size, p.vocab - first);
  int node = chain ? further(0, j) : j;
  while (node < len) {
    RowStat r = wave_stat(thread_stat<T>(row0 + (size_t)node * p.row_stride + first, n, tid, kStatThreads, c, sampled), c, sampled);
    if ((tid & 63) == 0) red[tid >> 6] = r;
    __syncthreads();
    if (tid == 0) {
#pragma unroll
      for (int w = 1; w < kStatThreads / 64; ++w) {
        const RowStat o = red[w];
        r.key = max(r.key, o.key);
        const float top = fmaxf(r.m, o.m);
        if (top > kNegInf) r.s = r.s * weight(r.m, top, c) + o.s * weight(o.m, top, c);
        r.m = top;
      }
      if (r.key != 0 && r.key != ~0ull) r.key -= first;      // ~(index + first)
      workspace_of(p).stats[((size_t)b * p.nodes + node) * p.stat_parts + part] = r;
    }
    node = chain ? further(node, each) : len;
    if (node < len) __syncthreads();                         // red: read
  }
}

// A work-group per sequence.  STATS: the rows' parts are there (64 threads do for these, but not for a sum in fp64).  NC: nodes of a lane.
template <typename T, bool STATS, int NC>
__global__ void __launch_bounds__(kWalkThreads) verify_walk_kernel(const VerifyParams p) {
  constexpr int kThreads = kWalkThreads;
  constexpr int kWaves = kThreads / 64;
  __shared__ int tokens[kDraftMaxNodes], parents[kDraftMaxNodes];
  __shared__ float logits[kDraftMaxNodes];                   // of a node's token after its parent
  __shared__ float uniforms[kDraftMaxNodes];
  __shared__ RowStat red[kWaves];
  __shared__ u64 keys[STATS ? kDraftMaxNodes : 1];            // the nodes' joined parts
  __shared__ double totals[STATS ? kDraftMaxNodes : 1];
  __shared__ double red_d[kWaves];
  const int b = blockIdx.x, tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int len = min(max(p.tree_lens[b], 0), p.nodes);
  const int vocab = p.vocab;
  const VerifyWorkspace ws = workspace_of(p);
  const float temp = temperature_of(p, b);
  const bool sampled = temp > 0.0f;
  const float c = sampled ? kLog2e / temp : 0.0f;
  const double c64 = sampled ? 1.4426950408889634074 / (double)temp : 0.0;
  int* path = p.path + (size_t)b * p.nodes;
  const T* row0 = reinterpret_cast<const T*>(p.logits) + (size_t)b * p.nodes * p.row_stride;
  const RowStat* stats = ws.stats + (size_t)b * p.nodes * p.stat_parts;
  // what the walk may come to is fetched beforehand: its steps then wait for rows (or nothing) only
  for (int i = tid; i < p.nodes; i += kThreads) {
    const int tok = p.tokens[(size_t)b * p.nodes + i], up = p.parents[(size_t)b * p.nodes + i];
    const bool is = up >= 0 && up < i && i < len && (unsigned)tok < (unsigned)vocab;
    if (sampled) uniforms[i] = p.uniforms[(size_t)b * p.nodes + i];
    tokens[i] = tok;
    parents[i] = is ? up : -1;                               // a node that cannot be taken has no parent
    if (sampled && is) logits[i] = to_float<T>(row0[(size_t)up * p.row_stride + tok]);
  }
  if constexpr (STATS) {
    for (int i = tid; i < len; i += kThreads) {
      const RowStat* parts = stats + (size_t)i * p.stat_parts;
      u64 key = 0;
      float top = kNegInf;
      double S = 0.0;
      for (int k0 = 0; k0 < p.stat_parts; k0 += kPartsAtOnce) {
        RowStat part[kPartsAtOnce];
#pragma unroll
        for (int k = 0; k < kPartsAtOnce; ++k) part[k] = parts[min(k0 + k, p.stat_parts - 1)];
        const float old = top;
#pragma unroll
        for (int k = 0; k < kPartsAtOnce; ++k) {
          key = max(key, part[k].key);
          top = fmaxf(top, part[k].m);
        }
        if (sampled && top > kNegInf) {
          S = old > kNegInf ? S * weight(old, top, c) : 0.0;
#pragma unroll
          for (int k = 0; k < kPartsAtOnce; ++k)
            if (k0 + k < p.stat_parts && part[k].m > kNegInf) S += (double)part[k].s * weight(part[k].m, top, c);
        }
      }
      keys[i] = key;
      totals[i] = S;
    }
  }
  __syncthreads();

  int count = 0, cur = len > 0 ? 0 : -1, next = -1, draw = -1;
  float M = 0.0f;
  double mass = 0.0;
  while (cur >= 0) {
    if (tid == 0) path[count] = cur;
    ++count;
    const T* x = row0 + (size_t)cur * p.row_stride;

    u64 key = 0;
    double S = 0.0;
    if constexpr (STATS) {
      key = keys[cur];
      S = totals[cur];
      M = from_order_bits((uint32_t)(key >> 32));
    } else {
      const RowStat r = wave_stat(thread_stat<T>(x, vocab, tid, kThreads, c, sampled), c, sampled);
      if (lane == 0) red[wave] = r;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < kWaves; ++w) key = max(key, red[w].key);
      M = from_order_bits((uint32_t)(key >> 32));
      if (sampled && key != ~0ull) {
#pragma unroll
        for (int w = 0; w < kWaves; ++w)
          if (red[w].m > kNegInf) S += (double)red[w].s * weight(red[w].m, M, c);
      }
      __syncthreads();                   // red: read by all
    }
    const int best = (int)~(uint32_t)key;
    if (key == 0 || key == ~0ull || (sampled && M == __builtin_inff())) break;      // next stays -1

    // the children: every wave finds the same
    int child[NC];
#pragma unroll
    for (int n = 0; n < NC; ++n) {
      const int i = lane + 64 * n;
      child[n] = i < p.nodes && parents[i] == cur ? tokens[i] : -1;
    }
    int go = -1;
    if (!sampled) {
#pragma unroll
      for (int n = 0; n < NC; ++n) {
        const u64 hit = __builtin_amdgcn_ballot_w64(child[n] == best);
        if (hit && go < 0) go = 64 * n + __builtin_ctzll(hit);
      }
      if (go < 0) {
        next = best;
        break;
      }
    } else {
      const double u = uniforms[cur];
      double e[NC];
#pragma unroll
      for (int n = 0; n < NC; ++n) e[n] = child[n] >= 0 ? weight64(logits[lane + 64 * n], M, c64) : 0.0;
      // of equal tokens the first counts
#pragma unroll
      for (int n = 0; n < NC; ++n) {
        u64 left = __builtin_amdgcn_ballot_w64(child[n] >= 0);
        while (left) {
          const int l = __builtin_ctzll(left);
          left &= left - 1;
          const int tok = __builtin_amdgcn_readlane(child[n], l);
#pragma unroll
          for (int k = n; k < NC; ++k)
            if (child[k] == tok && (k > n || lane > l)) child[k] = -1;
          left &= __builtin_amdgcn_ballot_w64(child[n] >= 0);
        }
      }
      // sure: whether u is away from every bound that was met
      auto choose = [&](double total, double margin, bool& sure) {
        int found = -1;
        mass = 0.0;
        sure = true;
#pragma unroll
        for (int n = 0; n < NC; ++n) {
          u64 left = __builtin_amdgcn_ballot_w64(child[n] >= 0);
          while (left && found < 0) {
            const int l = __builtin_ctzll(left);
            left &= left - 1;
            mass += lane_value(e[n], l);
            sure = sure && fabs(u * total - mass) >= margin * total;
            if (u * total < mass) found = 64 * n + l;
          }
        }
        return found;
      };
      bool sure;
      go = choose(S, p.unsure, sure);
      if (!sure) {
        const double part = wave_sum(thread_sum64<T>(x, vocab, tid, kThreads, M, c64));
        if (lane == 0) red_d[wave] = part;
        __syncthreads();
        S = 0.0;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) S += red_d[w];
        go = choose(S, 0.0, sure);
        __syncthreads();                 // red_d: read by all
      }
      if (go < 0) {
        draw = cur;
        if (wave == 0) {
          DrawJob& job = ws.jobs[b];
          int before = 0;
#pragma unroll
          for (int n = 0; n < NC; ++n) {
            const u64 is = __builtin_amdgcn_ballot_w64(child[n] >= 0);
            if (child[n] >= 0) job.token[before + __popcll(is & ((1ull << lane) - 1))] = child[n];
            before += __popcll(is);
          }
          if (lane == 0) {
            job.mass = mass;
            job.u = u;
            job.top = M;
            job.children = before;
          }
        }
        break;
      }
    }
    cur = go;
  }
  for (int j = count + tid; j < p.nodes; j += kThreads) path[j] = -1;
  if (tid == 0) {
    p.counts[b] = count;
    p.next_tokens[b] = next;
    if (p.temperatures) ws.jobs[b].node = draw;
  }
}

// A draw's row, and this lane's children; all loads at once.
template <typename T> struct DrawRow {
  static constexpr int NC = kDraftMaxNodes / 64;
  const T* x;
  int node, children, vocab;
  int token[NC];
  float top;
  double c64;
  __device__ __forceinline__ DrawRow(const VerifyParams& p, const DrawJob& job, int b) {
    node = job.node;
    children = job.children;
    top = job.top;
    vocab = p.vocab;
    c64 = 1.4426950408889634074 / (double)p.temperatures[b];
#pragma unroll
    for (int n = 0; n < NC; ++n) token[n] = job.token[(threadIdx.x & 63) + 64 * n];      // (past the children: of no meaning)
    x = reinterpret_cast<const T*>(p.logits) + ((size_t)b * p.nodes + max(node, 0)) * p.row_stride;
  }
  // The thread's kDrawPer consecutive elements of a chunk as e, children's and those past the row as 0.
  __device__ __forceinline__ void elements(int chunk, double (&e)[kDrawPer]) const {
    const int first = chunk * kDrawChunk + threadIdx.x * kDrawPer, lane = threadIdx.x & 63;
    float v[kDrawPer];
#pragma unroll
    for (int k = 0; k < kDrawPer; ++k) v[k] = to_float<T>(x[min(first + k, vocab - 1)]);
#pragma unroll
    for (int k = 0; k < kDrawPer; ++k) e[k] = first + k < vocab ? weight64(v[k], top, c64) : 0.0;
#pragma unroll
    for (int n = 0; n < NC; ++n) {
      const int at = token[n] - chunk * kDrawChunk;
      u64 in = __builtin_amdgcn_ballot_w64(lane + 64 * n < children && (unsigned)at < (unsigned)kDrawChunk);
      while (in) {
        const int off = __builtin_amdgcn_readlane(at, __builtin_ctzll(in)) - (int)threadIdx.x * kDrawPer;
        in &= in - 1;
#pragma unroll
        for (int k = 0; k < kDrawPer; ++k)
          if (off == k) e[k] = 0.0;
      }
    }
  }
};

template <typename T> __global__ void __launch_bounds__(kDrawThreads) verify_rest_kernel(const VerifyParams p) {
  __shared__ double red[kDrawThreads / 64];
  const int chunk = blockIdx.x, b = blockIdx.y;
  const VerifyWorkspace ws = workspace_of(p);
  const DrawRow<T> row(p, ws.jobs[b], b);
  if (row.node < 0) return;
  double e[kDrawPer];
  row.elements(chunk, e);
  double sum = 0.0;
#pragma unroll
  for (int k = 0; k < kDrawPer; ++k) sum += e[k];
  sum = wave_sum(sum);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    sum = 0.0;
#pragma unroll
    for (int w = 0; w < kDrawThreads / 64; ++w) sum += red[w];
    ws.sums[(size_t)b * p.draw_chunks + chunk] = sum;
  }
}

template <typename T> __global__ void __launch_bounds__(kDrawThreads) verify_draw_kernel(const VerifyParams p) {
  constexpr int kWaves = kDrawThreads / 64;
  __shared__ double red[kWaves];
  __shared__ int found, lowest;
  const int b = blockIdx.x, tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const VerifyWorkspace ws = workspace_of(p);
  // the rest's chunks: every wave sums and searches them for itself
  const double* sums = ws.sums + (size_t)b * p.draw_chunks;
  const int per = (p.draw_chunks + 63) / 64;
  double mine = 0.0;                                      // (without a draw of no meaning, and not used)
  for (int k = 0; k < per; ++k) mine += lane * per + k < p.draw_chunks ? sums[lane * per + k] : 0.0;
  const double mass = ws.jobs[b].mass, u = ws.jobs[b].u;
  const DrawRow<T> row(p, ws.jobs[b], b);
  if (row.node < 0) return;
  const double upto = wave_prefix(mine, lane);
  const double rest = lane_value(upto, 63);
  const double target = u * (mass + rest) - mass;
  u64 past = __builtin_amdgcn_ballot_w64(upto > target && mine > 0.0);
  if (!past) {                                            // u of 1: the last token
    const u64 some = __builtin_amdgcn_ballot_w64(mine > 0.0);
    past = some ? 1ull << (63 - __builtin_clzll(some)) : 1ull;
  }
  const int l = __builtin_ctzll(past);
  double before = lane_value(upto - mine, l);
  int chunk = l * per;
  double chunk_before = before;
  for (int g = l * per; g < min((l + 1) * per, p.draw_chunks); ++g) {
    const double s = sums[g];
    if (s > 0.0) {
      chunk = g;
      chunk_before = before;
      if (before + s > target) break;
    }
    before += s;
  }
  double e[kDrawPer];
  row.elements(chunk, e);
  double own = 0.0;
#pragma unroll
  for (int k = 0; k < kDrawPer; ++k) own += e[k];
  const double in_wave = wave_prefix(own, lane);
  if (lane == 63) red[wave] = in_wave;
  if (tid == 0) {
    found = -1;
    lowest = 0x7fffffff;
  }
  __syncthreads();
  double sum = chunk_before + in_wave - own;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) sum += w < wave ? red[w] : 0.0;
  // the last token with a weight whose sum of those before it is not above the target
  int hit = -1, any = -1;
#pragma unroll
  for (int k = 0; k < kDrawPer; ++k) {
    if (e[k] > 0.0) {
      if (any < 0) any = k;
      if (sum <= target) hit = k;
    }
    sum += e[k];
  }
  const int first = chunk * kDrawChunk + tid * kDrawPer;
  if (hit >= 0) atomicMax(&found, first + hit);
  if (any >= 0) atomicMin(&lowest, first + any);
  __syncthreads();
  // none where the target lies below the chunk's first token by a rounding
  if (tid == 0) p.next_tokens[b] = found >= 0 ? found : lowest == 0x7fffffff ? -1 : lowest;
}

int stat_size(int dtype) { return kStatThreads * kStatVecs * 16 / (dtype == kF32 ? 4 : 2); }

// Whether rows are read first: at 5.2 GB/ms, against seven steps of a walk, each 0.9 us and 36 ns for a KiB of its row (paths
// are about so long; their lengths are known on the device only).  Sampled, all rows; greedy, chains, of about eight nodes,
// but at the worst of all.  MI355X, us, rows first / walk, trees with paths of up to 7 nodes: greedy, 32000 fp32 logits: 64 x 16
// nodes 16 / 25, 64 x 64 15 / 29, 128 x 8 25 / 21, 256 x 16 32 / 35; 128256 bf16: 8 x 64 15 / 24, 64 x 16 27 / 38, 64 x 32 26 / 37;
// sampled: 2 x 32 of 128256 bf16 27 / 74, 64 x 64 of 32000 fp32 107 / 57.
// Shorter paths make a walk shorter and leave the rows as they are.  A path without branches, us, rows first / walk, for 1, 3, 7
// and all drafted tokens accepted: greedy, 32000 fp32: 1 x 8 7 / 7, 7 / 11, 8 / 20; 16 x 32 20 / 7, 20 / 12, 21 / 21, 26 / 104;
// 1 x 64 22 / 7, 23 / 11, 24 / 20, 37 / 197; 1 x 256 83 / 7, 83 / 12, 85 / 23, 207 / 819; 64 x 16 26 / 9, 27 / 15, 27 / 30, 29 / 55;
// 128256 bf16: 1 x 32 13 / 11, 14 / 19, 15 / 37, 20 / 155; 16 x 256 235 / 11, 234 / 21, 236 / 41, 352 / 1650; sampled, 128256
// bf16: 1 x 32 21 / 35, 22 / 56, 25 / 96, 39 / 365; 64 x 16 78 / 50, 79 / 71, 81 / 116, 87 / 204.
bool all_rows(int num_seqs, int nodes, int vocab, int dtype, bool sampled) {
  const long long rows = (long long)num_seqs * nodes, row = (long long)vocab * (dtype == kF32 ? 4 : 2);
  const double walk = 7.0 * (0.9 + row / 1024.0 * 0.036);
  auto reading = [&](long long n) { return n * row / 5.2e6 + 4.0; };
  if (rows > 1 << 20) return false;
  return sampled ? reading(rows) <= walk : reading((long long)num_seqs * std::min(nodes, 8)) <= walk && reading(rows) <= 3 * walk;
}

int stat_parts(int num_seqs, int nodes, int vocab, int dtype, bool sampled) {
  return all_rows(num_seqs, nodes, vocab, dtype, sampled) ? (vocab + stat_size(dtype) - 1) / stat_size(dtype) : 0;
}

void plan(VerifyParams& p, int dtype) {
  p.draw_chunks = (p.vocab + kDrawChunk - 1) / kDrawChunk;
  p.stat_size = stat_size(dtype);
  p.stat_parts = stat_parts(p.num_seqs, p.nodes, p.vocab, dtype, p.temperatures != nullptr);
  p.chain_rows = p.stat_parts && !p.temperatures ? std::min(p.nodes, kChainRows) : 0;
  const int vecs = p.vocab / (dtype == kF32 ? 4 : 8);
  const int rounds = p.stat_parts ? 1 + (p.stat_parts + kPartsAtOnce - 1) / kPartsAtOnce
                                  : (vecs + kWalkThreads * kStatVecs - 1) / (kWalkThreads * kStatVecs);
  p.unsure = 0x1p-16 + rounds * 0x1p-19;
}

template <typename T, int NC> void launch_walk(const VerifyParams& p, hipStream_t s) {
  if (p.stat_parts) hipLaunchKernelGGL((verify_walk_kernel<T, true, NC>), dim3(p.num_seqs), dim3(kWalkThreads), 0, s, p);
  else hipLaunchKernelGGL((verify_walk_kernel<T, false, NC>), dim3(p.num_seqs), dim3(kWalkThreads), 0, s, p);
}

template <typename T> void launch_of(const VerifyParams& p, hipStream_t s) {
  if (p.stat_parts) {
    const dim3 grid(p.num_seqs * (p.chain_rows ? p.chain_rows : p.nodes), p.stat_parts);
    hipLaunchKernelGGL(verify_stats_kernel<T>, grid, dim3(kStatThreads), 0, s, p);
  }
  if (p.nodes <= 64) launch_walk<T, 1>(p, s);
  else if (p.nodes <= 128) launch_walk<T, 2>(p, s);
  else launch_walk<T, 4>(p, s);
  if (p.temperatures) {
    hipLaunchKernelGGL(verify_rest_kernel<T>, dim3(p.draw_chunks, p.num_seqs), dim3(kDrawThreads), 0, s, p);
    hipLaunchKernelGGL(verify_draw_kernel<T>, dim3(p.num_seqs), dim3(kDrawThreads), 0, s, p);
  }
}

}  // namespace

size_t verify_workspace_bytes(int num_seqs, int nodes, int vocab, int dtype) {
  VerifyParams p{};
  p.num_seqs = num_seqs;
  p.nodes = nodes;
  p.vocab = vocab;
  plan(p, dtype);
  const int parts = std::max(p.stat_parts, stat_parts(num_seqs, nodes, vocab, dtype, true));      // greedy or not
  return reinterpret_cast<uintptr_t>(workspace_of(p).stats + (size_t)num_seqs * nodes * parts);
}

void launch_verify(VerifyParams p, int dtype, hipStream_t s) {
  plan(p, dtype);
  if (dtype == kF32) launch_of<float>(p, s);
  else if (dtype == kF16) launch_of<_Float16>(p, s);
  else launch_of<__bf16>(p, s);
}

}  // namespace tv
