#include "tree_attention.cuh"

namespace tv {

void launch_tree_f32(const TreeParams& p, int head_dim, hipStream_t s) { tree_launch<float>(p, head_dim, s); }

}  // namespace tv
