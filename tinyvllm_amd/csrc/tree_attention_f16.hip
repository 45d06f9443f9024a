// Tree attention for element type _Float16.
#include "tree_attention.cuh"

namespace tv {

void launch_tree_f16(const TreeParams& p, int head_dim, hipStream_t s) { tree_launch<_Float16>(p, head_dim, s); }
TreeShapeInfo tree_info_f16(long long rows, int head_dim) { return tree_info<_Float16>(rows, head_dim); }

}  // namespace tv
