// What every node of a draft tree sees, its position and its cache slot
// (tv_draft_tree_layout), and the accepted rows' way to their places
// (tv_keep_draft_rows).
//
// Layout: a work-group per sequence, a thread per node.  Ancestors by doubling: with
// mask_k(i) the 2^k nearest of i and its ancestors and up_k(i) the 2^k-th ancestor,
//   mask_{k+1}(i) = mask_k(i) | mask_k(up_k(i)),  up_{k+1}(i) = up_k(up_k(i)),
// so a chain of 256 nodes takes eight rounds; the depth is the number of bits less one.
#include "tv_draft.h"

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
  p.positions[at] = live ? ctx + bits - 1 : 0;
  p.slots[at] = slot;
}

// A thread owns vector e of every row of one sequence and layer, K or V.  It reads
// kAhead rows before it writes them: row path[j] >= j is read before any row past
// j is written, since every write up to then went to rows below j.
template <typename V>
__global__ void __launch_bounds__(256) keep_rows_kernel(const KeepParams p) {
  constexpr int kAhead = 8;
  const int e = blockIdx.x * 256 + threadIdx.x;
  if (e >= 2 * p.row_vecs) return;
  const int b = blockIdx.y, layer = blockIdx.z;
  const bool second = e >= p.row_vecs;
  V* rows = reinterpret_cast<V*>(second ? p.v[layer] : p.k[layer]) + (second ? e - p.row_vecs : e);
  const int count = min(max(p.counts[b], 0), p.nodes);
  const int ctx = max(p.context_lens[b], 0);
  const int* path = p.path + (size_t)b * p.nodes;
  const int* table = p.block_tables + (size_t)b * p.bt_stride;
  auto slot_of = [&](long long pos) -> long long {
    if (pos / p.block_size >= p.bt_stride) return -1;
    const int blk = table[pos / p.block_size];
    return (unsigned)blk < (unsigned)p.num_blocks ? (long long)blk * p.block_size + pos % p.block_size : -1;
  };
  for (int j0 = 0; j0 < count; j0 += kAhead) {
    V held[kAhead];
    long long to[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int j = j0 + u;
      const int node = j < count ? path[j] : -1;
      to[u] = -1;
      if (node <= j || node >= p.nodes) continue;      // in its place already, or none
      const long long from = slot_of((long long)ctx + node);
      const long long place = slot_of((long long)ctx + j);
      if (from < 0 || place < 0) continue;
      held[u] = rows[from * p.row_vecs];
      to[u] = place;
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u)
      if (to[u] >= 0) rows[to[u] * p.row_vecs] = held[u];
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
