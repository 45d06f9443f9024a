// Tree attention for element type float.
#include "tree_attention.cuh"

namespace tv {

void launch_tree_f32(const TreeParams& p, int head_dim, hipStream_t s) { tree_launch<float>(p, head_dim, s); }
TreeShapeInfo tree_info_f32(long long rows, int head_dim) { return tree_info<float>(rows, head_dim); }

}  // namespace tv
