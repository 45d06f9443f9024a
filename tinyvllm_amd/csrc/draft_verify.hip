// The path through a draft tree that the model's logits accept
// (tv_verify_draft_tree).
//
// Greedy: the first maximum of a row.  Sampled, with m a row's maximum and e_i =
// 2^((x_i - m) log2(e) / temperature), S = sum e_i: children in the order of their indexes are
// taken while u S is not below their summed e; a path that ends draws from the other
// tokens, the first at which their e sum to more than u S - E, E the children's.
//
// Precision: whether u is below a sum needs fp32 only where u is not next to it: within
// kUnsure of a child's bound the sums are taken again in fp64.  (fp32 sums are off by a
// relative 2^-17 at most: a thread's 128 and more terms, each with the rounding of an
// argument that matters, below 2^5.)  The draw is in fp64 throughout: a large
// vocabulary has a bound every 2^-17 of S, and an error of d in u S meets one with
// probability 2^17 d.
//
// A walk over a path is serial and reads its rows only; reading the rows of all
// nodes first is parallel.  The second is taken for trees of few logits.
#include "tv_draft.h"

#include <algorithm>

namespace tv {

namespace {

constexpr int kWalkThreads = 1024;
constexpr int kStatThreads = 256;
constexpr int kStatVecs = 8;             // 16-byte vectors a thread of the stats kernel: 32 KiB of a row
constexpr int kDrawThreads = 256;
constexpr int kDrawPer = 8;              // elements a thread of the draw kernels
constexpr int kDrawChunk = kDrawThreads * kDrawPer;
constexpr int NC = kDraftMaxNodes / 64;
constexpr double kUnsure = 0x1p-13;

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
// elements before and behind them one each.
template <typename T>
__device__ __forceinline__ RowStat thread_stat(const T* x, int n, int tid, int threads, float c, bool sampled) {
  constexpr int EPV = 16 / (int)sizeof(T);
  constexpr int U = kStatVecs;
  const int head = min(n, (int)((16 - ((uintptr_t)x & 15)) & 15) / (int)sizeof(T));
  const int vecs = (n - head) / EPV;
  const u32x4* body = reinterpret_cast<const u32x4*>(x + head);
  float m = kNegInf, s = 0.0f;
  int at = 0;                            // the vector, or -1 - element, that the maximum was met in first
  if (tid < head) {
    m = to_float<T>(x[tid]);
    at = -1 - tid;
    s = m > kNegInf ? 1.0f : 0.0f;
  }
  for (int v0 = tid; v0 < vecs; v0 += threads * U) {
    u32x4 w[U];
#pragma unroll
    for (int u = 0; u < U; ++u) w[u] = body[min(v0 + u * threads, vecs - 1)];
    const float old = m;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (v0 + u * threads >= vecs) break;
      const float was = m;
      m = max_of<T>(w[u], m);
      at = m != was ? v0 + u * threads : at;   // (a NaN differs from itself: at is not looked at then)
    }
    if (sampled && m > kNegInf) {
      if (m > old) s *= old > kNegInf ? weight(old, m, c) : 0.0f;
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (v0 + u * threads < vecs) s += sum_of<T>(w[u], m, c);
    }
  }
  const int tail = head + vecs * EPV + tid;
  if (tail < n) {
    const float v = to_float<T>(x[tail]);
    const float was = m;
    m = __builtin_elementwise_maximum(m, v);
    if (m > was) {
      at = -1 - tail;
      s *= was > kNegInf ? weight(was, m, c) : 0.0f;
    }
    if (m > kNegInf) s += weight(v, m, c);
  }
  RowStat r{0, m, s};
  if (m != m) {
    r.key = ~0ull;
  } else if (m > kNegInf) {
    int idx = -1 - at;
    if (at >= 0) {
      idx = head + at * EPV;
#pragma unroll
      for (int e = EPV - 1; e >= 0; --e)
        if (to_float<T>(x[head + at * EPV + e]) == m) idx = head + at * EPV + e;
    }
    r.key = (u64)order_bits(m) << 32 | (uint32_t)~idx;
  }
  return r;
}

// The wave's shares as one, in every lane.
__device__ __forceinline__ RowStat wave_stat(RowStat r, float c, bool sampled) {
#pragma unroll
  for (int d = 1; d < 64; d *= 2) r.key = max(r.key, shfl_xor64(r.key, d));
  if (sampled) {
    const float top = group_max<64>(r.m);      // (of a NaN nothing is used)
    r.s = group_sum<64>(r.m > kNegInf ? r.s * weight(r.m, top, c) : 0.0f);
    r.m = top;
  }
  return r;
}

__device__ __forceinline__ float temperature_of(const VerifyParams& p, int b) {
  const float t = p.temperatures ? p.temperatures[b] : 0.0f;
  return t >= 0x1p-126f ? t : 0.0f;
}

struct VerifyWorkspace {
  int* node;                             // [B] the node to draw after, or -1
  float* top;                            // [B] its maximum
  double* sums;                          // [B, draw chunks]
  RowStat* stats;                        // [B * nodes, stat parts]
};

__host__ __device__ inline VerifyWorkspace workspace_of(const VerifyParams& p) {
  VerifyWorkspace w;
  w.sums = reinterpret_cast<double*>(p.workspace);
  w.stats = reinterpret_cast<RowStat*>(w.sums + (((size_t)p.num_seqs * p.draw_chunks + 1) & ~(size_t)1));
  w.node = reinterpret_cast<int*>(w.stats + (size_t)p.num_seqs * p.nodes * p.stat_parts);
  w.top = reinterpret_cast<float*>(w.node + p.num_seqs);
  return w;
}

// Parts of the rows of all live nodes.
template <typename T> __global__ void __launch_bounds__(kStatThreads) verify_stats_kernel(const VerifyParams p) {
  __shared__ RowStat red[kStatThreads / 64];
  const int row = blockIdx.x, part = blockIdx.y;
  const int b = row / p.nodes;
  if (row - b * p.nodes >= p.tree_lens[b]) return;
  const int tid = threadIdx.x;
  const float temp = temperature_of(p, b);
  const bool sampled = temp > 0.0f;
  const float c = sampled ? kLog2e / temp : 0.0f;
  const int first = part * p.stat_size, n = min(p.stat_size, p.vocab - first);
  const T* x = reinterpret_cast<const T*>(p.logits) + (size_t)row * p.row_stride + first;
  RowStat r = wave_stat(thread_stat<T>(x, n, tid, kStatThreads, c, sampled), c, sampled);
  if ((tid & 63) == 0) red[tid >> 6] = r;
  __syncthreads();
  if (tid != 0) return;
#pragma unroll
  for (int w = 1; w < kStatThreads / 64; ++w) {
    const RowStat o = red[w];
    r.key = max(r.key, o.key);
    const float top = fmaxf(r.m, o.m);
    if (top > kNegInf) r.s = r.s * weight(r.m, top, c) + o.s * weight(o.m, top, c);
    r.m = top;
  }
  if (r.key != 0 && r.key != ~0ull) r.key -= first;          // ~(index + first)
  workspace_of(p).stats[(size_t)row * p.stat_parts + part] = r;
}

// A work-group per sequence.  STATS: the rows' parts are there.
template <typename T, bool STATS>
__global__ void __launch_bounds__(STATS ? 64 : kWalkThreads) verify_walk_kernel(const VerifyParams p) {
  constexpr int kThreads = STATS ? 64 : kWalkThreads;
  constexpr int kWaves = kThreads / 64;
  __shared__ int tokens[kDraftMaxNodes], parents[kDraftMaxNodes];
  __shared__ RowStat red[kWaves];
  __shared__ double red_d[kWaves];
  const int b = blockIdx.x, tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int len = min(max(p.tree_lens[b], 0), p.nodes);
  const int vocab = p.vocab;
  const VerifyWorkspace ws = workspace_of(p);
  for (int i = tid; i < p.nodes; i += kThreads) {
    tokens[i] = p.tokens[(size_t)b * p.nodes + i];
    parents[i] = p.parents[(size_t)b * p.nodes + i];
  }
  const float temp = temperature_of(p, b);
  const bool sampled = temp > 0.0f;
  const float c = sampled ? kLog2e / temp : 0.0f;
  int* path = p.path + (size_t)b * p.nodes;
  __syncthreads();

  int count = 0, cur = len > 0 ? 0 : -1, next = -1, draw = -1;
  float M = 0.0f;
  while (cur >= 0) {
    if (tid == 0) path[count] = cur;
    ++count;
    const size_t row = (size_t)b * p.nodes + cur;
    const T* x = reinterpret_cast<const T*>(p.logits) + row * p.row_stride;

    u64 key = 0;
    double S = 0.0;
    if constexpr (STATS) {
      const RowStat* parts = ws.stats + row * p.stat_parts;
      for (int i = lane; i < p.stat_parts; i += 64) key = max(key, parts[i].key);
#pragma unroll
      for (int d = 1; d < 64; d *= 2) key = max(key, shfl_xor64(key, d));
      M = key == 0 || key == ~0ull ? 0.0f : to_float<T>(x[(int)~(uint32_t)key]);
      if (sampled) {
        for (int i = lane; i < p.stat_parts; i += 64)
          if (parts[i].m > kNegInf) S += (double)parts[i].s * weight(parts[i].m, M, c);
        S = wave_sum(S);
      }
    } else {
      const RowStat r = wave_stat(thread_stat<T>(x, vocab, tid, kThreads, c, sampled), c, sampled);
      if (lane == 0) red[wave] = r;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < kWaves; ++w) key = max(key, red[w].key);
      M = key == 0 || key == ~0ull ? 0.0f : to_float<T>(x[(int)~(uint32_t)key]);
      if (sampled) {
#pragma unroll
        for (int w = 0; w < kWaves; ++w)
          if (red[w].m > kNegInf) S += (double)red[w].s * weight(red[w].m, M, c);
      }
      __syncthreads();                   // red: read by all
    }
    const int best = (int)~(uint32_t)key;
    if (key == 0 || key == ~0ull || (sampled && M == __builtin_inff())) break;      // next stays -1

    // the children, of equal tokens the first: every wave finds the same
    int child[NC];
#pragma unroll
    for (int n = 0; n < NC; ++n) {
      const int i = lane + 64 * n;
      const bool is = i > cur && i < len && parents[i] == cur && (unsigned)tokens[i] < (unsigned)vocab;
      child[n] = is ? tokens[i] : -1;
    }
    int go = -1;
    if (!sampled) {
#pragma unroll
      for (int n = 0; n < NC; ++n) {
        const u64 hit = __builtin_amdgcn_ballot_w64(child[n] == best);
        if (hit && go < 0) go = 64 * n + __builtin_ctzll(hit);
      }
    } else {
      const double u = p.uniforms[row];
      const double c64 = 1.4426950408889634074 / (double)temp;
      double e[NC];
#pragma unroll
      for (int n = 0; n < NC; ++n) e[n] = child[n] >= 0 ? weight64(to_float<T>(x[child[n]]), M, c64) : 0.0;
      // sure: whether u is away from every bound that was met
      auto choose = [&](double total, double margin, bool& sure, double& mass, int& last) {
        int found = -1;
        mass = 0.0;
        last = -1;
        sure = true;
#pragma unroll
        for (int n = 0; n < NC; ++n) {
          u64 left = __builtin_amdgcn_ballot_w64(child[n] >= 0);
          while (left && found < 0) {
            const int l = __builtin_ctzll(left);
            left &= left - 1;
            const int tok = __builtin_amdgcn_readlane(child[n], l);
            bool before = false;
#pragma unroll
            for (int k = 0; k < NC; ++k) before |= child[k] == tok && (k < n || (k == n && lane < l));
            if (__builtin_amdgcn_ballot_w64(before)) continue;
            const double mine = lane_value(e[n], l);
            mass += mine;
            if (mine > 0.0) last = 64 * n + l;
            sure = sure && fabs(u * total - mass) >= margin * total;
            if (u * total < mass) found = 64 * n + l;
          }
        }
        return found;
      };
      bool sure;
      double mass;
      int last;
      go = choose(S, kUnsure, sure, mass, last);
      if (!sure) {
        double part = 0.0;
        for (int i = tid; i < vocab; i += kThreads) part += weight64(to_float<T>(x[i]), M, c64);
        part = wave_sum(part);
        if (lane == 0) red_d[wave] = part;
        __syncthreads();
        S = 0.0;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) S += red_d[w];
        go = choose(S, 0.0, sure, mass, last);
        // nearly all of S is the children's: whether there is anything else to draw
        if (go < 0 && S - mass <= 0x1p-40 * S) go = last;
        __syncthreads();                 // red_d: read by all
      }
      if (go < 0) draw = cur;
    }
    if (go < 0) {
      if (!sampled) next = best;
      break;
    }
    cur = go;
  }
  for (int j = count + tid; j < p.nodes; j += kThreads) path[j] = -1;
  if (tid == 0) {
    p.counts[b] = count;
    p.next_tokens[b] = next;
    if (p.temperatures) {
      ws.node[b] = draw;
      ws.top[b] = M;
    }
  }
}

// Tokens of the children of a node, and whether one lies in a range.
struct DrawChildren {
  int token[NC];
  template <typename F> __device__ __forceinline__ DrawChildren(const VerifyParams& p, int b, int node, F keep) {
    const int len = min(max(p.tree_lens[b], 0), p.nodes);
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int n = 0; n < NC; ++n) {
      const int i = lane + 64 * n;
      token[n] = -1;
      if (i > node && i < len && p.parents[(size_t)b * p.nodes + i] == node) token[n] = keep(p.tokens[(size_t)b * p.nodes + i]);
    }
  }
};

// A thread's kDrawPer consecutive elements of a chunk as e, children's and those past the row as 0.
template <typename T>
__device__ __forceinline__ void draw_elements(const VerifyParams& p, int b, int node, float M, double c64, int chunk,
                                              double (&e)[kDrawPer]) {
  const T* x = reinterpret_cast<const T*>(p.logits) + ((size_t)b * p.nodes + node) * p.row_stride;
  const int first = chunk * kDrawChunk + threadIdx.x * kDrawPer;
  float v[kDrawPer];
#pragma unroll
  for (int k = 0; k < kDrawPer; ++k) v[k] = to_float<T>(x[min(first + k, p.vocab - 1)]);
  const DrawChildren children(p, b, node, [](int t) { return t; });
#pragma unroll
  for (int k = 0; k < kDrawPer; ++k) e[k] = first + k < p.vocab ? weight64(v[k], M, c64) : 0.0;
#pragma unroll
  for (int n = 0; n < NC; ++n) {
    const int at = children.token[n] - chunk * kDrawChunk;
    u64 in = __builtin_amdgcn_ballot_w64(children.token[n] >= 0 && (unsigned)at < (unsigned)kDrawChunk);
    while (in) {
      const int off = __builtin_amdgcn_readlane(at, __builtin_ctzll(in)) - (int)threadIdx.x * kDrawPer;
      in &= in - 1;
#pragma unroll
      for (int k = 0; k < kDrawPer; ++k)
        if (off == k) e[k] = 0.0;
    }
  }
}

template <typename T> __global__ void __launch_bounds__(kDrawThreads) verify_rest_kernel(const VerifyParams p) {
  __shared__ double red[kDrawThreads / 64];
  const int chunk = blockIdx.x, b = blockIdx.y;
  const VerifyWorkspace ws = workspace_of(p);
  const int node = ws.node[b];
  if (node < 0) return;
  double e[kDrawPer];
  draw_elements<T>(p, b, node, ws.top[b], 1.4426950408889634074 / (double)temperature_of(p, b), chunk, e);
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
  const int node = ws.node[b];
  if (node < 0) return;
  const float M = ws.top[b];
  const double c64 = 1.4426950408889634074 / (double)temperature_of(p, b);
  const T* x = reinterpret_cast<const T*>(p.logits) + ((size_t)b * p.nodes + node) * p.row_stride;
  const double* sums = ws.sums + (size_t)b * p.draw_chunks;

  // the children's mass, of equal tokens once: every wave finds the same
  const int vocab = p.vocab;
  const DrawChildren children(p, b, node, [vocab](int t) { return (unsigned)t < (unsigned)vocab ? t : -1; });
  double mass = 0.0;
#pragma unroll
  for (int n = 0; n < NC; ++n) {
    const double e = children.token[n] >= 0 ? weight64(to_float<T>(x[children.token[n]]), M, c64) : 0.0;
    u64 left = __builtin_amdgcn_ballot_w64(children.token[n] >= 0);
    while (left) {
      const int l = __builtin_ctzll(left);
      left &= left - 1;
      const int tok = __builtin_amdgcn_readlane(children.token[n], l);
      bool before = false;
#pragma unroll
      for (int k = 0; k < NC; ++k) before |= children.token[k] == tok && (k < n || (k == n && lane < l));
      if (!__builtin_amdgcn_ballot_w64(before)) mass += lane_value(e, l);
    }
  }
  // the rest's chunks: every wave sums and searches them for itself
  const int per = (p.draw_chunks + 63) / 64;
  double mine = 0.0;
  for (int k = 0; k < per; ++k) mine += lane * per + k < p.draw_chunks ? sums[lane * per + k] : 0.0;
  const double upto = wave_prefix(mine, lane);
  const double rest = lane_value(upto, 63);
  const double u = p.uniforms[(size_t)b * p.nodes + node];
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
  draw_elements<T>(p, b, node, M, c64, chunk, e);
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
  if (tid == 0) p.next_tokens[b] = found >= 0 ? found : lowest;
}

int stat_size(int dtype) { return kStatThreads * kStatVecs * 16 / (dtype == kF32 ? 4 : 2); }

// Whether the rows of all nodes are read first.
bool all_rows(int num_seqs, int nodes, int vocab, int dtype) {
  const long long rows = (long long)num_seqs * nodes;
  return rows <= 1 << 20 && rows * vocab * (dtype == kF32 ? 4 : 2) <= 64LL << 20;
}

void plan(VerifyParams& p, int dtype) {
  p.draw_chunks = (p.vocab + kDrawChunk - 1) / kDrawChunk;
  p.stat_size = stat_size(dtype);
  p.stat_parts = all_rows(p.num_seqs, p.nodes, p.vocab, dtype) ? (p.vocab + p.stat_size - 1) / p.stat_size : 0;
}

template <typename T> void launch_of(const VerifyParams& p, hipStream_t s) {
  if (p.stat_parts) {
    hipLaunchKernelGGL(verify_stats_kernel<T>, dim3(p.num_seqs * p.nodes, p.stat_parts), dim3(kStatThreads), 0, s, p);
    hipLaunchKernelGGL((verify_walk_kernel<T, true>), dim3(p.num_seqs), dim3(64), 0, s, p);
  } else {
    hipLaunchKernelGGL((verify_walk_kernel<T, false>), dim3(p.num_seqs), dim3(kWalkThreads), 0, s, p);
  }
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
  return reinterpret_cast<uintptr_t>(workspace_of(p).top + num_seqs);
}

void launch_verify(VerifyParams p, int dtype, hipStream_t s) {
  plan(p, dtype);
  if (dtype == kF32) launch_of<float>(p, s);
  else if (dtype == kF16) launch_of<_Float16>(p, s);
  else launch_of<__bf16>(p, s);
}

}  // namespace tv
