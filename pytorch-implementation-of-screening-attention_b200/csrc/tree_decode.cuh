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
// queries of a head.  The reads of the keys are what a pass cannot do without,
// so the kernels are built around one pass over the pages.
//
// Sharing out the keys.  Positions are cut into 64-key tiles; the tiles of all
// (sequence, head) segments, one after another, form one list that is cut into
// equal runs, a CTA each.  Heads have windows of very different lengths (2 to
// thousands of keys in one layer), so a fixed number of splits per head would
// leave most CTAs idle while the widest head's work; the list needs no host
// knowledge of lengths or windows.  A CTA that owns only a part of a segment
// leaves its sum in workspace slot (CTA + segment), which no other pair shares
// because both grow along the list, and tree_finish_kernel adds a segment's
// slots in order.  With few tiles a segment goes to one CTA and no second launch
// follows.
#pragma once
#include "kv_rows.cuh"
#include "paged.cuh"

namespace screen {
namespace tree {

constexpr int kTile = kTreeTile;
constexpr int kThreads = 128;
constexpr int kMaxN = SCREEN_TREE_MAX_NODES;
constexpr int kNoKey = -2000000000;   // c of a key that nothing sees

// Tiles [t0, t0 + nt) that sequence b, head h reads.
struct Range {
  long long lens, first;  // first: oldest key any node sees
  int t0, nt, dmax;       // nt >= 1, a dummy tile for an empty place
  bool any;
};
__device__ __forceinline__ Range tree_range(const TreeParams& p, int b, int h) {
  Range g;
  g.lens = (long long)p.a.lens[b] + p.lens_off;
  g.dmax = window_dmax(p.a.w[h]);
  g.any = g.lens >= 0;
  if (!g.any) {  // an empty place in the batch
    g.t0 = 0;
    g.nt = 1;
    g.first = 0;
    return g;
  }
  g.first = g.lens - (g.dmax > 0 ? g.dmax : 0);
  if (g.first < 0) g.first = 0;
  g.t0 = (int)(g.first / kTile);
  g.nt = (int)((g.lens + p.a.n - 1) / kTile) - g.t0 + 1;
  return g;
}

// A CTA's run of the tile list, segment by segment.
struct Share {
  long long pos, end, start;   // next tile, end of the run, first tile of `seg`
  long long total;
  int ctas;                    // CTAs that have a run
  int seg;
};
// Slots of the partial sums of each segment: CTAs first .. last, none if the
// segment's rows were written by the CTA that owned all of it.
struct SegSlots {
  int first, last;
};
constexpr int kMinTiles = 4;   // a run is at least this long
__device__ __forceinline__ long long share_begin(const Share& s, int cta) {
  return s.total * cta / s.ctas;
}
// All threads of the CTA; false if it has nothing to do.
__device__ __forceinline__ bool share_init(const TreeParams& p, Share& s) {
  const int segs = p.a.B * p.a.H;
  if (p.a.num_ctas == 1) {     // one CTA per segment
    s.seg = blockIdx.x;
    s.start = s.pos = 0;
    s.ctas = 0;
    return true;
  }
  __shared__ long long warp_s[kThreads / 32];
  __shared__ long long start_s;
  __shared__ int seg_s;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int each = (segs + kThreads - 1) / kThreads;
  long long mine = 0;
  for (int j = tid * each; j < (tid + 1) * each && j < segs; ++j)
    mine += tree_range(p, j / p.a.H, j % p.a.H).nt;
  long long inc = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long y = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += y;
  }
  if (lane == 31) warp_s[warp] = inc;
  __syncthreads();
  long long before = inc - mine;
  s.total = 0;
#pragma unroll
  for (int i = 0; i < kThreads / 32; ++i) {
    if (i < warp) before += warp_s[i];
    s.total += warp_s[i];
  }
  const long long most = (s.total + kMinTiles - 1) / kMinTiles;
  s.ctas = (long long)gridDim.x < most ? (int)gridDim.x : (int)most;
  if ((int)blockIdx.x >= s.ctas) return false;
  s.pos = share_begin(s, blockIdx.x);
  s.end = share_begin(s, blockIdx.x + 1);
  if (s.pos >= before && s.pos < before + mine) {   // this thread's segments hold it
    int j = tid * each;
    long long at = before;
    while (true) {
      const int nt = tree_range(p, j / p.a.H, j % p.a.H).nt;
      if (s.pos < at + nt) break;
      at += nt;
      ++j;
    }
    seg_s = j;
    start_s = at;
  }
  __syncthreads();
  s.seg = seg_s;
  s.start = start_s;
  return true;
}
// Next piece: tiles [c0, c1] of segment s.seg.  False at the end of the run.
__device__ __forceinline__ bool share_next(const TreeParams& p, Share& s, Range& g, int& c0,
                                           int& c1, bool& whole, SegSlots* slots) {
  if (s.ctas == 0) {
    if (s.pos) return false;
    g = tree_range(p, s.seg / p.a.H, s.seg % p.a.H);
    c0 = g.t0;
    c1 = g.t0 + g.nt - 1;
    whole = true;
    s.pos = 1;
    return true;
  }
  if (s.pos >= s.end) return false;
  if (s.pos >= s.start) {
    g = tree_range(p, s.seg / p.a.H, s.seg % p.a.H);
    while (s.pos >= s.start + g.nt) {   // the previous piece ended its segment
      s.start += g.nt;
      ++s.seg;
      g = tree_range(p, s.seg / p.a.H, s.seg % p.a.H);
    }
  }
  const long long stop = s.end < s.start + g.nt ? s.end : s.start + g.nt;
  c0 = g.t0 + (int)(s.pos - s.start);
  c1 = g.t0 + (int)(stop - s.start) - 1;
  whole = s.pos == s.start && stop == s.start + g.nt;
  if (s.pos == s.start && threadIdx.x == 0) {
    SegSlots q{0, -1};
    if (!whole) {
      q.first = blockIdx.x;
      // the last CTA whose run begins at or before the segment's last tile
      q.last = (int)(((s.start + g.nt) * s.ctas - 1) / s.total);
    }
    slots[s.seg] = q;
  }
  s.pos = stop;
  return true;
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
    write_cache_row<E, TA, D>(x, a.eps, gl, row,
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

// One CTA per segment, or at most as many as are resident at once: a run for
// each, all of one length.
constexpr int kSMs = 148;
inline dim3 tree_grid(const TreeParams& p, int per_sm) {
  if (p.a.num_ctas == 1) return dim3(p.a.B * p.a.H);
  return dim3(p.a.num_ctas < kSMs * per_sm ? p.a.num_ctas : kSMs * per_sm);
}

}  // namespace tree
}  // namespace screen
