// Tree attention for element type __bf16.
#include "tree_attention.cuh"

namespace tv {

void launch_tree_bf16(const TreeParams& p, int head_dim, hipStream_t s) { tree_launch<__bf16>(p, head_dim, s); }
TreeShapeInfo tree_info_bf16(long long rows, int head_dim) { return tree_info<__bf16>(rows, head_dim); }

}  // namespace tv
