// Tree attention and single-token decode over int8 pages, bf16 activations
// (tree_mma.cuh).
#include "tree_mma.cuh"
namespace screen {
bool tree_i8(TreeParams p, float* part, cudaStream_t s) {
  return tree::launch_tree_e<signed char, __nv_bfloat16>(p, part, s);
}
}  // namespace screen
