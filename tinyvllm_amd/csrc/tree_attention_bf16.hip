#include "tree_attention.cuh"

namespace tv {

void launch_tree_bf16(const TreeParams& p, int head_dim, hipStream_t s) { tree_launch<__bf16>(p, head_dim, s); }

}  // namespace tv
