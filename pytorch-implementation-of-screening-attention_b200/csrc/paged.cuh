// Host-side declarations of the kernels of speculative serving on the paged
// cache (paged_rows.cu, tree_decode*.cu, verify.cu).
#pragma once
#include "common.cuh"

namespace screen {
void paged_append8(const screen_paged_append_args& a, cudaStream_t s);
void paged_read(const screen_paged_read_args& a, cudaStream_t s);
void commit(const screen_commit_args& a, cudaStream_t s);

// Positions are cut into tiles of kTreeTile keys.
constexpr int kTreeTile = 64;
// CTAs of a shared-out call, at most: four on each of 148 SMs.  Its segments
// (sequence, head) are fewer, or there is nobody to share with.
constexpr int kTreeMaxCtas = 148 * 4;
struct TreeParams {
  screen_tree_args a;
  int lens_off;   // added to a.lens (decode: -1, the query is the newest cached token)
  int part_off;   // floats of the workspace before the partial sums
};
// Each returns whether it shared the tiles out (num_ctas > 1 and more CTAs resident
// than segments): tree_finish has to follow.
bool tree_bf16(TreeParams p, float* part, cudaStream_t s);
bool tree_i8(TreeParams p, float* part, cudaStream_t s);
bool tree_i8_f32(TreeParams p, float* part, cudaStream_t s);
bool tree_f32(TreeParams p, float* part, cudaStream_t s);
void tree_finish(const TreeParams& p, const float* part, cudaStream_t s);

void verify(const screen_verify_args& a, cudaStream_t s);
size_t verify_workspace(const screen_verify_args& a);
}  // namespace screen
