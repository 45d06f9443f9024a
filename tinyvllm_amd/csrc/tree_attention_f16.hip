#include "tree_attention.cuh"

namespace tv {

void launch_tree_f16(const TreeParams& p, int head_dim, hipStream_t s) { tree_launch<_Float16>(p, head_dim, s); }

}  // namespace tv
