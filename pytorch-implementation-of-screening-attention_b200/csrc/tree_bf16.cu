// Tree attention over bf16 pages (tree_mma.cuh).
#include "tree_mma.cuh"
namespace screen {
void tree_bf16(const TreeParams& p, float* part, cudaStream_t s) {
  tree::launch_tree_e<__nv_bfloat16, __nv_bfloat16>(p, part, s);
}
}  // namespace screen
