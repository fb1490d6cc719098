// Tree attention over bf16 pages (tree_mma.cuh).
#include "tree_mma.cuh"
namespace screen {
bool tree_bf16(TreeParams p, float* part, cudaStream_t s) {
  return tree::launch_tree_e<__nv_bfloat16, __nv_bfloat16>(p, part, s);
}
}  // namespace screen
