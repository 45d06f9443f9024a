// Log-probabilities of given tokens under rows of logits, with the rows' entropy
// and their most likely tokens (tv_token_logprobs, include/tv_llama.h).
//
// With m the largest logit of a row and the sums over all other tokens,
//   s = sum e^(x - m),  t = sum (m - x) e^(x - m)
//   log p(token) = (x_token - m) - log(1 + s)
//   entropy      = log(1 + s) + t / (1 + s)
// Every term is positive, and the maximum's own term, which is exactly 1, stays
// out of the sums: log1p(s) keeps its digits where one token has nearly all of
// the probability, and nothing cancels.
//
// Bound: one read of the logits, and close behind it the vector unit (an
// exponential and three more operations an element).  A work-group holds kVecs
// 16-byte vectors a thread of one row in registers (32 KiB at 256 threads, 128 KiB
// at 1024: a row of 32000 fp32 logits is read once and needs no second launch), so
// the sums are taken relative to the final maximum.  Longer rows are cut into such
// segments, and a second kernel joins their (m, s, t) and lists.  MI355X: 1000 rows
// of 32000 fp32 26 us (4.9 TB/s), with 5 top tokens 33; of bf16 20 (3.2 TB/s); 2047
// of 128256 bf16 with 20 top tokens 146 (3.6 TB/s), without 110 (4.8 TB/s).
// Top tokens of a segment: from the threads' maxima, rounded down to 16 bits, a
// search over bits with ballots finds a bound that at least k elements reach and few
// others do; those that do go to a list in LDS and are ranked by (value, then lowest
// index).  Where too many reach
// it (equal logits) or there is a NaN, k passes over the segment take the largest
// remaining key each.  NaN ranks above every number.
#include "tv_logprobs.h"

namespace tv {

namespace {

constexpr int kVecs = 8;          // 16-byte vectors a thread
constexpr int kList = 512;        // candidates of a segment
// Distances from the maximum are limited to this in t: their exponentials are 0 in
// fp32, and the distance of a logit of -inf must not be infinite beside it.
constexpr float kFar = 300.0f;
constexpr float kLn2 = 0.6931471805599453f;

typedef unsigned long long u64;

// Order-preserving bits: NaN highest, -0 equal to +0.
__device__ __forceinline__ uint32_t order_bits(float x) {
  const uint32_t u = __builtin_bit_cast(uint32_t, x);
  if (x != x) return 0xffffffffu;
  if (x == 0.0f) return 0x80000000u;
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float from_order_bits(uint32_t o) {
  if (o == 0xffffffffu) return __builtin_nanf("");
  return u32_as_f32(o & 0x80000000u ? o & 0x7fffffffu : ~o);
}
// Larger key: larger value, then lower index.
__device__ __forceinline__ u64 make_key(float x, int idx) { return (u64)order_bits(x) << 32 | (uint32_t)~idx; }

__device__ __forceinline__ u64 shfl_xor64(u64 x, int mask) {
  const uint32_t lo = __builtin_bit_cast(uint32_t, shfl_xor(u32_as_f32((uint32_t)x), mask));
  const uint32_t hi = __builtin_bit_cast(uint32_t, shfl_xor(u32_as_f32((uint32_t)(x >> 32)), mask));
  return (u64)hi << 32 | lo;
}

// Element e of a vector as fp32.
template <typename T> __device__ __forceinline__ float element(const u32x4& w, int e) {
  if constexpr (sizeof(T) == 4) {
    return u32_as_f32(w[e]);
  } else {
    float a, b;
    unpack2<T>(w[e >> 1], a, b);
    return e & 1 ? b : a;
  }
}
template <typename T> constexpr uint32_t kNegInfWord = 0;
template <> constexpr uint32_t kNegInfWord<float> = 0xff800000u;
template <> constexpr uint32_t kNegInfWord<_Float16> = 0xfc00fc00u;
template <> constexpr uint32_t kNegInfWord<__bf16> = 0xff80ff80u;

// Results of a row from m, s, t; list: its first top_k keys in order.
template <typename T>
__device__ __forceinline__ void finish_row(const LogprobParams& p, int row, float m, float s, float t, const u64* list,
                                           int tid, int threads) {
  const float inf = __builtin_inff();
  const float log_total = fabsf(m) < inf ? log1pf(s) : __builtin_nanf("");
  if (tid == 0) {
    const int tok = p.tokens[row];
    const float x = (unsigned)tok < (unsigned)p.vocab
                        ? to_float<T>(reinterpret_cast<const T*>(p.logits)[(size_t)row * p.row_stride + tok])
                        : __builtin_nanf("");
    p.logprobs[row] = (x - m) - log_total;
    p.entropy[row] = log_total + t / (1.0f + s);
  }
  for (int i = tid; i < p.top_k; i += threads) {
    const u64 k = list[i];
    p.top_ids[(size_t)row * p.top_k + i] = (int)~(uint32_t)k;
    p.top_logprobs[(size_t)row * p.top_k + i] = (from_order_bits((uint32_t)(k >> 32)) - m) - log_total;
  }
}

// ALIGNED: rows start at multiples of 16 bytes.  TOP: top_k > 0 (its code costs registers: held to
// the 64 of eight waves a SIMD 2047 rows of 128256 bf16 with 20 top tokens take 153 us, at six waves 146; work-groups
// of 1024 threads need the eight for two of them per CU).
template <typename T, int NT, bool ALIGNED, bool TOP>
__global__ void __launch_bounds__(NT) __attribute__((amdgpu_waves_per_eu(TOP && NT < 1024 ? 6 : 8))) logprobs_kernel(const LogprobParams p) {
  constexpr int NW = NT / 64;
  constexpr int EPV = 16 / (int)sizeof(T);
  constexpr int SEG = NT * kVecs * EPV;
  __shared__ float red[4][NW];
  __shared__ uint32_t bound[2][NW];
  __shared__ u64 cand[kList];
  __shared__ u64 best[kLogprobTopMax];
  __shared__ u64 wave_best[NW];
  __shared__ int count;

  const int row = blockIdx.x, seg = blockIdx.y;
  const int tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lane = tid & 63;
  const T* x = reinterpret_cast<const T*>(p.logits) + (size_t)row * p.row_stride;
  const int first = seg * SEG + tid * EPV;
  auto index_of = [&](int j) { return first + j * NT * EPV; };

  // -inf past the row; the one vector that the row's end cuts goes by elements
  const u32x4 none = u32x4{kNegInfWord<T>, kNegInfWord<T>, kNegInfWord<T>, kNegInfWord<T>};
  u32x4 w[kVecs];
  auto by_elements = [&](int at) {
    u32x4 v = none;
#pragma unroll
    for (int e = 0; e < EPV; ++e) {
      if constexpr (sizeof(T) == 4) {
        const uint32_t x4 = reinterpret_cast<const uint32_t*>(x)[min(at + e, p.vocab - 1)];
        v[e] = at + e < p.vocab ? x4 : v[e];
      } else {
        const uint32_t x2 = reinterpret_cast<const uint16_t*>(x)[min(at + e, p.vocab - 1)];
        const uint32_t old = v[e >> 1];
        const uint32_t put = e & 1 ? (old & 0xffffu) | x2 << 16 : (old & 0xffff0000u) | x2;
        v[e >> 1] = at + e < p.vocab ? put : old;
      }
    }
    return v;
  };
  if constexpr (ALIGNED) {
#pragma unroll
    for (int j = 0; j < kVecs; ++j)
      w[j] = index_of(j) + EPV <= p.vocab ? *reinterpret_cast<const u32x4*>(x + index_of(j)) : none;
    const int cut = p.vocab % EPV ? p.vocab - p.vocab % EPV : -1;
    if (cut >= first && (cut - first) % (NT * EPV) == 0 && cut - first < SEG) {
      const u32x4 v = by_elements(cut);
#pragma unroll
      for (int j = 0; j < kVecs; ++j) w[j] = index_of(j) == cut ? v : w[j];
    }
  } else {
#pragma unroll
    for (int j = 0; j < kVecs; ++j) w[j] = by_elements(index_of(j));
  }
  if (tid == 0) count = 0;
  // The vectors are made opaque between the passes over them: otherwise the
  // compiler keeps every element's fp32 form from the first pass on.
  auto again = [&]() {
#pragma unroll
    for (int j = 0; j < kVecs; ++j) __asm__ volatile("" : "+v"(w[j]));
  };

  float vmax[kVecs];                // NaN is left out here and shows in the sums
  float tmax = kNegInf;
#pragma unroll
  for (int j = 0; j < kVecs; ++j) {
    __asm__ volatile("" : "+v"(tmax), "+v"(w[j]));
    vmax[j] = element<T>(w[j], 0);
#pragma unroll
    for (int e = 1; e < EPV; ++e) vmax[j] = fmaxf(vmax[j], element<T>(w[j], e));
    tmax = fmaxf(tmax, vmax[j]);
  }
  again();
  float m = group_max<64>(tmax);
  if (lane == 0) red[0][wave] = m;
  // Bounds of 16 bits: the largest b that at least `lanes` of the wave's threads reach with their maxima.
  // At least top_k elements reach every wave's bound for top_k lanes, and the lowest of the waves' bounds
  // for top_k / NW lanes each, which is the closer one where the waves have much the same.
  const int k = TOP ? p.top_k : 0;
  if constexpr (TOP) {
    const uint32_t key = order_bits(tmax);
    auto reached_by = [&](int lanes) {
      uint32_t b = 0;
#pragma unroll
      for (int bit = 31; bit >= 16; --bit) {
        const uint32_t c = b | 1u << bit;
        b = __builtin_popcountll(__builtin_amdgcn_ballot_w64(key >= c)) >= lanes ? c : b;
      }
      return b;
    };
    const uint32_t all = reached_by(k), some = reached_by((k + NW - 1) / NW);
    if (lane == 0) {
      bound[0][wave] = all;
      bound[1][wave] = some;
    }
  }
  __syncthreads();
  m = red[0][0];
#pragma unroll 4
  for (int i = 1; i < NW; ++i) m = fmaxf(m, red[0][i]);

  if constexpr (TOP) {
    // what reaches the bound, before the sums: the vectors that hold some are read again, from cache
    uint32_t b = bound[0][0], some = bound[1][0];
#pragma unroll 4
    for (int i = 1; i < NW; ++i) {
      b = max(b, bound[0][i]);
      some = min(some, bound[1][i]);
    }
    b = max(b, some);
    const float least = b > order_bits(kNegInf) ? from_order_bits(b) : kNegInf;
    uint32_t vecs = 0;
#pragma unroll
    for (int j = 0; j < kVecs; ++j) vecs |= vmax[j] >= least && index_of(j) < p.vocab ? 1u << j : 0u;
    while (vecs) {
      const int at = index_of(__builtin_ctz(vecs));
      vecs &= vecs - 1;
      const u32x4 held = ALIGNED && at + EPV <= p.vocab ? *reinterpret_cast<const u32x4*>(x + at) : by_elements(at);
#pragma unroll
      for (int e = 0; e < EPV; ++e) {
        const float v = element<T>(held, e);
        if (v >= least && at + e < p.vocab) {
          const int to = atomicAdd(&count, 1);
          if (to < kList) cand[to] = make_key(v, at + e);
        }
      }
    }
  }

  // Sums without the maximum's own term: elements equal to m count 1 each, less one
  // for the row.  In log2 units relative to mh, m log2 e rounded: one fma an element;
  // what the rounding left, ml, is a factor of the whole sums.
  // From 2^30 on (a row of the type's lowest numbers, say) another number's term is
  // below 2^-184, zero in fp32: with mh of 0 for a low m and infinity for a high one
  // every y is far below or -inf.
  const bool far = !(fabsf(m) < 0x1p30f);
  float mh = far ? (m < 0.0f ? 0.0f : __builtin_inff()) : m * kLog2e;
  const float ml = far ? 0.0f : fmaf(m, kLog2e, -mh);
  float s = 0.0f, t = 0.0f, eq = 0.0f;
  if (tmax < m) {
#pragma unroll
    for (int j = 0; j < kVecs; ++j) {
      // a vector at a time (the next one's terms depend on this): registers for two work-groups a CU
      __asm__ volatile("" : "+v"(mh), "+v"(s), "+v"(t), "+v"(w[j]));
#pragma unroll
      for (int e = 0; e < EPV; ++e) {
        const float y = fmaf(element<T>(w[j], e), kLog2e, -mh);
        const float q = fast_exp2(y);
        s += q;
        t = fmaf(fmaxf(y, -kFar), q, t);
      }
    }
  } else {
    int equal = 0;
#pragma unroll
    for (int j = 0; j < kVecs; ++j) {
      __asm__ volatile("" : "+v"(mh), "+v"(s), "+v"(t), "+v"(w[j]));
#pragma unroll
      for (int e = 0; e < EPV; ++e) {
        const float v = element<T>(w[j], e);
        const float y = fmaf(v, kLog2e, -mh);
        const float q = fast_exp2(y);
        equal += v == m ? 1 : 0;
        s += v == m ? 0.0f : q;
        t = v == m ? t : fmaf(fmaxf(y, -kFar), q, t);
      }
    }
    eq = (float)equal;
  }
  again();
  s = group_sum<64>(s);
  t = group_sum<64>(t);
  eq = group_sum<64>(eq);
  if (lane == 0) {
    red[1][wave] = s;
    red[2][wave] = t;
    red[3][wave] = eq;
  }

  __syncthreads();
  s = red[1][0];
  t = red[2][0];
  eq = red[3][0];
#pragma unroll 2
  for (int i = 1; i < NW; ++i) {
    s += red[1][i];
    t += red[2][i];
    eq += red[3][i];
  }
  // t in nats and positive: (m - x) e^(x - m) = -(y - ml) 2^(y - ml) ln 2
  const float left = fast_exp2(-ml);
  t = fmaf(ml, s, -t) * left * kLn2;
  s = fmaf(s, left, eq - 1.0f);

  if constexpr (TOP) {
    const bool slow = s != s || count > kList;      // a NaN, or too many equal logits
    if (!slow) {
      const int n = count;
      for (int i = tid; i < n; i += NT) {
        const u64 mine = cand[i];
        int rank = 0;
        for (int o = 0; o < n; ++o) rank += cand[o] > mine ? 1 : 0;
        if (rank < k) best[rank] = mine;
      }
      for (int i = n + tid; i < k; i += NT) best[i] = 0;   // a last segment of fewer than k
    } else {
      u64 last = 0;
      for (int i = 0; i < k; ++i) {
        u64 top = 0;
        for (int o = seg * SEG + tid; o < min((seg + 1) * SEG, p.vocab); o += NT) {
          const u64 c = make_key(to_float<T>(x[o]), o);
          top = (i == 0 || c < last) && c > top ? c : top;
        }
#pragma unroll
        for (int mask = 1; mask < 64; mask <<= 1) {
          const u64 o = shfl_xor64(top, mask);
          top = o > top ? o : top;
        }
        __syncthreads();            // the last round's wave_best has been read
        if (lane == 0) wave_best[wave] = top;
        __syncthreads();
        last = wave_best[0];
        for (int o = 1; o < NW; ++o) last = wave_best[o] > last ? wave_best[o] : last;
        if (tid == 0) best[i] = last;
      }
    }
    __syncthreads();
  }

  if (gridDim.y == 1) {
    finish_row<T>(p, row, m, s, t, best, tid, NT);
  } else {
    const size_t at = (size_t)row * gridDim.y + seg;
    if (tid == 0) {
      p.part[at * 3] = m;
      p.part[at * 3 + 1] = s;
      p.part[at * 3 + 2] = t;
    }
    for (int i = tid; i < k; i += NT) p.part_keys[at * k + i] = best[i];
  }
}

// Joins the segments of a row.  A segment's sums leave its own maximum out: it
// comes back, times e^(m_i - M), for every segment but the first that holds M.
// A key's rank is its place in its own list plus the keys above it in the others,
// found by bisection (the lists are in order).
template <typename T>
__global__ void __launch_bounds__(256) logprobs_merge_kernel(const LogprobParams p, int segs) {
  __shared__ u64 best[kLogprobTopMax];
  const int row = blockIdx.x, tid = threadIdx.x, k = p.top_k;
  const float* part = p.part + (size_t)row * segs * 3;
  float M = kNegInf;
  for (int i = 0; i < segs; ++i) M = fmaxf(M, part[3 * i]);
  float s = 0.0f, t = 0.0f;
  bool held = false;
  for (int i = 0; i < segs; ++i) {
    const float m = part[3 * i], si = part[3 * i + 1], ti = part[3 * i + 2];
    if (m == M && !held) {
      held = true;
      s += si;
      t += ti;
    } else {                        // a segment of nothing but -inf adds 0
      const float d = M - m;
      const float q = fast_exp2(d * -kLog2e);
      s = fmaf(q, 1.0f + si, s);
      t = fmaf(q, fmaf(fminf(d, kFar), 1.0f + si, ti), t);
    }
  }
  const u64* keys = p.part_keys + (size_t)row * segs * k;
  for (int c = tid; c < segs * k; c += 256) {
    const u64 mine = keys[c];
    const int own = c / k;
    int rank = c - own * k;
    for (int i = 0; i < segs && rank < k; ++i) {
      if (i == own) continue;
      int lo = 0, hi = k;             // keys of list i above mine
      while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (keys[i * k + mid] > mine) lo = mid + 1;
        else hi = mid;
      }
      rank += lo;
    }
    if (rank < k) best[rank] = mine;
  }
  __syncthreads();
  finish_row<T>(p, row, M, s, t, best, tid, 256);
}

template <typename T, int NT, bool ALIGNED> void launch_rows(const LogprobParams& p, int segs, hipStream_t stream) {
  const dim3 grid(p.rows, segs);
  if (p.top_k > 0) hipLaunchKernelGGL((logprobs_kernel<T, NT, ALIGNED, true>), grid, dim3(NT), 0, stream, p);
  else hipLaunchKernelGGL((logprobs_kernel<T, NT, ALIGNED, false>), grid, dim3(NT), 0, stream, p);
}

template <typename T, int NT> void launch_of(const LogprobParams& p, int segs, hipStream_t stream) {
  if (p.aligned) launch_rows<T, NT, true>(p, segs, stream);
  else launch_rows<T, NT, false>(p, segs, stream);
  if (segs > 1) hipLaunchKernelGGL(logprobs_merge_kernel<T>, dim3(p.rows), dim3(256), 0, stream, p, segs);
}

template <typename T> void launch_type(const LogprobParams& p, hipStream_t stream) {
  const int segs = logprob_segments(p.vocab, (int)sizeof(T));
  const int threads = logprob_threads(p.vocab, (int)sizeof(T));
  if (threads == 256) launch_of<T, 256>(p, segs, stream);
  else if (threads == 512) launch_of<T, 512>(p, segs, stream);
  else launch_of<T, 1024>(p, segs, stream);
}

}  // namespace

void launch_logprobs(const LogprobParams& p, int dtype, hipStream_t stream) {
  if (dtype == kF32) launch_type<float>(p, stream);
  else if (dtype == kF16) launch_type<_Float16>(p, stream);
  else launch_type<__bf16>(p, stream);
}

}  // namespace tv
