// Screening attention of a tree of drafted tokens over the paged cache.
//
// Node i of sequence b (n <= 64 nodes, parents[b, i] < i, -1 = child of the
// newest cached token) owns cache slot lens[b] + i and stands at position
// p_i = lens[b] + depth_i.  It sees the cached keys j with
// 0 <= p_i - j <= ceil(w) - 1 and, among the slots, its ancestors and itself at
// distance depth_i - depth_a.  Per (query, key):
//   t = 1 - r (1 - q^.k^),  alpha = max(t, 0)^2 (1 + cos(pi rel / w)) / 2,
//   o = sum alpha v^,       y = tanh(|o|) / |o| o.
// There is no softmax normaliser, so partial sums over runs of keys simply add.
//
// Work: 4 D flops per (query, key) against 2 row reads per key shared by all n
// queries of a head.  For the n here the reads of the keys are what a pass
// cannot do without (n = 64, D = 64, int8: 120 flops a byte), so the kernel is
// built around one pass over the pages: a CTA owns a run of 64-key tiles of one
// (sequence, head) and keeps every query of the tree in registers.
//
//  * tiles are copied with cp.async (16 bytes, XOR-swizzled rows, zero fill for
//    keys outside the window or the table) into a ring of shared-memory stages;
//    pages of any size work because every row has its own address, looked up a
//    stage ahead of its copies;
//  * S and alpha V run on warp-level MMAs (m16n8k16, queries on the 16 rows):
//    with one to 64 query rows a 128-row tcgen05 tile would be mostly padding,
//    and the score fragment is directly the A operand of alpha V;
//  * a group of 16 keys whose scores all fall under the trim skips the mask and
//    the alpha V product;
//  * the mask is cos(pi (c_j - d_i) / w) = cos cos + sin sin with one pair per
//    key (c_j: position minus lens, or the node's depth) and one per query.
#pragma once
#include "kv_rows.cuh"
#include "paged.cuh"

namespace screen {
namespace tree {

constexpr int kTile = kTreeTile;
constexpr int kThreads = 128;
constexpr int kMaxN = SCREEN_TREE_MAX_NODES;
constexpr int kNoKey = -2000000000;   // c of a key that nothing sees

// Tiles [t0, t1] that sequence b, head h reads, and the tiles one split owns.
struct Range {
  long long lens, first;  // first: oldest key any node sees
  int t0, nt, per, used;  // used: splits that own a tile
  int dmax;
};
__device__ __forceinline__ Range tree_range(const TreeParams& p, int b, int h) {
  Range g;
  g.lens = (long long)p.a.lens[b] + p.lens_off;
  g.dmax = window_dmax(p.a.w[h]);
  if (g.lens < 0) {  // an empty place in the batch
    g.t0 = g.nt = g.used = 0;
    g.per = 1;
    g.first = 0;
    return g;
  }
  g.first = g.lens - (g.dmax > 0 ? g.dmax : 0);
  if (g.first < 0) g.first = 0;
  g.t0 = (int)(g.first / kTile);
  g.nt = (int)((g.lens + p.a.n - 1) / kTile) - g.t0 + 1;
  // the host's tiles per split gives every CTA the same work across heads of
  // different windows; a window wider than the host was told still fits
  const int least = (g.nt + p.a.num_splits - 1) / p.a.num_splits;
  g.per = p.per > least ? p.per : least;
  g.used = (g.nt + g.per - 1) / g.per;
  return g;
}

// Ancestor masks, depths and presence of the n nodes of sequence b, by warp 0:
// pointer doubling, lane l owns nodes l and l + 32.
struct Nodes {
  unsigned long long line[kMaxN];  // ancestors and self; 0 for an absent node
  int depth[kMaxN];
  int jump[kMaxN];
};
__device__ __forceinline__ void tree_nodes(const screen_tree_args& a, int b, Nodes& s, int lane) {
  const int n = a.n;
  // jump: next ancestor to merge, -1 past the root, -2 an absent line
  for (int i = lane; i < kMaxN; i += 32) {
    int p = -2;
    if (i < n) p = a.parents ? a.parents[(long long)b * a.parents_sb + i] : i - 1;
    if (p < -1 || p >= i) p = -2;
    s.jump[i] = p;
    s.line[i] = 1ull << i;
  }
  __syncwarp();
  for (int hop = 1; hop < n; hop *= 2) {
    unsigned long long m[2];
    int j[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int i = lane + 32 * e, p = s.jump[i];
      m[e] = s.line[i];
      j[e] = p;
      if (p >= 0) {
        m[e] |= s.line[p];
        j[e] = s.jump[p];
      }
    }
    __syncwarp();
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      s.line[lane + 32 * e] = m[e];
      s.jump[lane + 32 * e] = j[e];
    }
    __syncwarp();
  }
  for (int i = lane; i < kMaxN; i += 32) {
    if (s.jump[i] == -2) s.line[i] = 0;
    s.depth[i] = s.line[i] ? __popcll(s.line[i]) - 1 : 0;
  }
  __syncwarp();
}

// Rows of the nodes whose slots lie in the tiles [c0, c1] written to the pages.
template <typename E, typename TA, int D>
__device__ __forceinline__ void append_rows(const screen_tree_args& a, const Nodes& nodes, int b,
                                            int h, long long lens, int c0, int c1) {
  constexpr int G = D / 4, RPI = kThreads / G;
  const int tid = threadIdx.x, gl = tid % G;
  long long lo = (long long)c0 * kTile - lens, hi = (long long)(c1 + 1) * kTile - 1 - lens;
  if (lo < 0) lo = 0;
  if (hi > a.n - 1) hi = a.n - 1;
  const int cnt = hi >= lo ? (int)(hi - lo + 1) : 0;
  for (int base = 0; base < 2 * cnt; base += RPI) {   // uniform over the CTA
    const int u = base + tid / G;
    const bool in = u < 2 * cnt;
    const bool isv = in && u >= cnt;
    const int i = in ? (int)lo + (isv ? u - cnt : u) : 0;
    const bool take = in && nodes.line[i] != 0;
    float x[4] = {0.f, 0.f, 0.f, 0.f};
    if (take)
      load4(reinterpret_cast<const TA*>(isv ? a.v : a.k) + (long long)b * (isv ? a.v_sb : a.k_sb) +
                (long long)i * (isv ? a.v_st : a.k_st) + (long long)h * D + gl * 4, x);
    const long long row = take ? paged_row(a.cache, b, a.H, h, lens + i) : -1;
    write_cache_row<E, D>(x, a.eps, gl, row,
                          reinterpret_cast<E*>(isv ? a.cache.v_pages : a.cache.k_pages),
                          isv ? a.v_scales : a.k_scales);
  }
  __syncthreads();
}

// y row from the sum o (D values spread over a warp, PER per lane at d = lane +
// 32 e; lanes past D hold 0).
template <typename TA, int D>
__device__ __forceinline__ void store_row(const screen_tree_args& a, int b, int i, int h, int lane,
                                          const float (&o)[D < 32 ? 1 : D / 32], bool present) {
  constexpr int PER = D < 32 ? 1 : D / 32;
  float ss = 0.f;
#pragma unroll
  for (int e = 0; e < PER; ++e) ss = fmaf(o[e], o[e], ss);
  ss = warp_sum(ss);
  // a query that sees a non-finite row has no norm: its whole output is NaN
  const float g = ss < __uint_as_float(0x7f800000u) ? tanhnorm_scale(sqrtf(ss), a.eps)
                                                    : __uint_as_float(0x7fc00000u);
  TA* y = reinterpret_cast<TA*>(a.y) + (((long long)b * a.n + i) * a.H + h) * D;
#pragma unroll
  for (int e = 0; e < PER; ++e)
    if (lane + 32 * e < D) y[lane + 32 * e] = from_f<TA>(present ? o[e] * g : 0.f);
}

}  // namespace tree
}  // namespace screen
