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
// Segments (sequence, head) of a call whose tiles are shared out over CTAs.
constexpr int kTreeMaxShared = 2048;
struct TreeParams {
  screen_tree_args a;
  int lens_off;   // added to a.lens (decode: -1, the query is the newest cached token)
  int part_off;   // floats of the workspace before the partial sums
};
void tree_bf16(const TreeParams& p, float* part, cudaStream_t s);
void tree_i8(const TreeParams& p, float* part, cudaStream_t s);
void tree_i8_f32(const TreeParams& p, float* part, cudaStream_t s);
void tree_f32(const TreeParams& p, float* part, cudaStream_t s);
void tree_finish(const TreeParams& p, const float* part, cudaStream_t s);

void verify(const screen_verify_args& a, cudaStream_t s);
size_t verify_workspace(const screen_verify_args& a);
}  // namespace screen
