// Tree attention and single-token decode over int8 pages, fp32 activations
// (tree_mma.cuh): the query and alpha enter the products as hi + lo halves.
#include "tree_mma.cuh"
namespace screen {
bool tree_i8_f32(TreeParams p, float* part, cudaStream_t s) {
  return tree::launch_tree_e<signed char, float>(p, part, s);
}
}  // namespace screen
