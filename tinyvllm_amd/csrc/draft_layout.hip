// What every node of a draft tree sees, its position and its cache slot
// (tv_draft_tree_layout), and the accepted rows' way to their places
// (tv_keep_draft_rows).
//
// Layout: a work-group per sequence, a thread per node.  Ancestors by doubling: with
// mask_k(i) the 2^k nearest of i and its ancestors and up_k(i) the 2^k-th ancestor,
//   mask_{k+1}(i) = mask_k(i) | mask_k(up_k(i)),  up_{k+1}(i) = up_k(up_k(i)),
// so a chain of 256 nodes takes eight rounds; the depth is the number of bits less one.
// Bound by the launch.  MI355X: 4 sequences of 8 nodes 2.4 us, 256 of 64 3.2 us.
#include "tv_draft.h"

#include <type_traits>

namespace tv {

namespace {

template <int W>
__global__ void __launch_bounds__(kDraftMaxNodes) draft_layout_kernel(const DraftLayoutParams p) {
  __shared__ u64 seen[2][kDraftMaxNodes][W];
  __shared__ int up[2][kDraftMaxNodes];
  const int b = blockIdx.x, i = threadIdx.x;
  const int len = min(max(p.tree_lens[b], 0), p.nodes);
  const int ctx = max(p.context_lens[b], 0);
  const bool live = i < len;
  int above = i < p.nodes ? p.parents[(size_t)b * p.nodes + i] : -1;
  if (above < 0 || above >= i || !live) above = -1;
  u64 mine[W];
#pragma unroll
  for (int w = 0; w < W; ++w) mine[w] = live && i / 64 == w ? 1ull << (i % 64) : 0;
  for (int reach = 1, k = 0; reach < len; reach *= 2, k ^= 1) {
#pragma unroll
    for (int w = 0; w < W; ++w) seen[k][i][w] = mine[w];
    up[k][i] = above;
    __syncthreads();
    if (above >= 0) {
#pragma unroll
      for (int w = 0; w < W; ++w) mine[w] |= seen[k][above][w];
      above = up[k][above];
    }
  }
  if (i >= p.nodes) return;
  const size_t at = (size_t)b * p.nodes + i;
  int bits = 0;
#pragma unroll
  for (int w = 0; w < W; ++w) {
    if (w < p.words) p.mask[at * p.words + w] = mine[w];
    bits += __popcll(mine[w]);
  }
  int slot = -1;
  const long long pos = (long long)ctx + i;
  if (live && pos / p.block_size < p.bt_stride) {
    const int blk = p.block_tables[(size_t)b * p.bt_stride + pos / p.block_size];
    if ((unsigned)blk < (unsigned)p.num_blocks) slot = blk * p.block_size + (int)(pos % p.block_size);
  }
  p.positions[at] = live ? (int)((unsigned)ctx + (bits - 1)) : 0;
  p.slots[at] = slot;
}

// A work-group moves 256 vectors of every row that has to, of one sequence and layer, K and V.  The rows' places are
// looked up first, one by a thread, and listed in their order.  A thread then owns a vector of every row; it reads kAhead rows
// before it writes them: row path[j] > j is read before any row past j is written, since every write up to then went to
// rows below j.  Bound by HBM after the look-ups,
// a chain of three loads.  MI355X: 64 sequences of 48 nodes, 32 layers, rows of 2 KiB in K and V each (72 MB) 24 us, 3.0 TB/s.
template <typename V>
__global__ void __launch_bounds__(256) keep_rows_kernel(const KeepParams p) {
  constexpr int kAhead = 8;
  __shared__ int from[kDraftMaxNodes], to[kDraftMaxNodes];
  __shared__ int moved[4];                 // of the nodes of a wave
  const int e = blockIdx.x * 256 + threadIdx.x, j = threadIdx.x;
  const int b = blockIdx.y, layer = blockIdx.z;
  const int count = min(max(p.counts[b], 0), p.nodes);
  const int ctx = max(p.context_lens[b], 0);
  const int* table = p.block_tables + (size_t)b * p.bt_stride;
  auto slot_of = [&](int pos) {            // -1: the table does not reach it, or its block is outside the cache
    if (pos < 0 || pos / p.block_size >= p.bt_stride) return -1;     // (below 0: past 32 bits)
    const int blk = table[pos / p.block_size];
    return (unsigned)blk < (unsigned)p.num_blocks ? blk * p.block_size + pos % p.block_size : -1;
  };
  int source = -1, place = -1;
  if (j < count) {
    const int node = p.path[(size_t)b * p.nodes + j];
    if (node > j && node < p.nodes) {      // else it is in its place, or none
      source = slot_of((int)((unsigned)ctx + node));
      place = slot_of((int)((unsigned)ctx + j));
    }
  }
  const bool moves = source >= 0 && place >= 0;
  const u64 with = __builtin_amdgcn_ballot_w64(moves);
  if ((j & 63) == 0) moved[j >> 6] = __popcll(with);
  __syncthreads();
  int at = __popcll(with & ((1ull << (j & 63)) - 1)), n = 0;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    at += w < j >> 6 ? moved[w] : 0;
    n += moved[w];
  }
  if (moves) {
    from[at] = source;
    to[at] = place;
  }
  __syncthreads();
  if (e >= 2 * p.row_vecs) return;
  const bool second = e >= p.row_vecs;
  V* rows = reinterpret_cast<V*>(second ? p.v[layer] : p.k[layer]) + (second ? e - p.row_vecs : e);
  // as many rows at a time as there are, up to kAhead (always eight, the last one again past the end: 25.5 us for 23.9)
  auto move = [&](int i0, auto count) {
    constexpr int U = decltype(count)::value;
    V held[U];
#pragma unroll
    for (int u = 0; u < U; ++u) held[u] = rows[(size_t)from[i0 + u] * p.row_vecs];
#pragma unroll
    for (int u = 0; u < U; ++u) rows[(size_t)to[i0 + u] * p.row_vecs] = held[u];
  };
  n = __builtin_amdgcn_readfirstlane(n);
  int i0 = 0;
  for (; i0 + kAhead <= n; i0 += kAhead) move(i0, std::integral_constant<int, kAhead>());
  switch (n - i0) {
    case 7: move(i0, std::integral_constant<int, 7>()); break;
    case 6: move(i0, std::integral_constant<int, 6>()); break;
    case 5: move(i0, std::integral_constant<int, 5>()); break;
    case 4: move(i0, std::integral_constant<int, 4>()); break;
    case 3: move(i0, std::integral_constant<int, 3>()); break;
    case 2: move(i0, std::integral_constant<int, 2>()); break;
    case 1: move(i0, std::integral_constant<int, 1>()); break;
  }
}

}  // namespace

void launch_draft_layout(const DraftLayoutParams& p, hipStream_t s) {
  const dim3 grid(p.num_seqs), block((p.nodes + 63) / 64 * 64);
  switch (p.words) {
    case 1: hipLaunchKernelGGL(draft_layout_kernel<1>, grid, block, 0, s, p); break;
    case 2: hipLaunchKernelGGL(draft_layout_kernel<2>, grid, block, 0, s, p); break;
    default: hipLaunchKernelGGL(draft_layout_kernel<4>, grid, block, 0, s, p); break;
  }
}

void launch_keep(const KeepParams& p, int layers, int vec_bytes, hipStream_t s) {
  const dim3 grid((2 * p.row_vecs + 255) / 256, p.num_seqs, layers);
  switch (vec_bytes) {
    case 16: hipLaunchKernelGGL(keep_rows_kernel<u32x4>, grid, dim3(256), 0, s, p); break;
    case 8: hipLaunchKernelGGL(keep_rows_kernel<u32x2>, grid, dim3(256), 0, s, p); break;
    case 4: hipLaunchKernelGGL(keep_rows_kernel<uint32_t>, grid, dim3(256), 0, s, p); break;
    default: hipLaunchKernelGGL(keep_rows_kernel<uint16_t>, grid, dim3(256), 0, s, p); break;
  }
}

}  // namespace tv
