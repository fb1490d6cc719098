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
// Sharing out the keys.  Heads have windows of very different lengths (2 to
// thousands of keys in one layer), so a fixed number of splits per (sequence,
// head) segment would leave most CTAs idle while the widest head's work.  Every
// CTA reads all lengths and windows and finds the shortest run of 64-key tiles, L,
// at which the segments, cut into ceil(tiles / L) equal runs each, fill the CTAs
// that are resident at once; it then takes its own run.  No host knowledge of
// lengths or windows is needed.  A run that is not a whole segment leaves its sum
// in the workspace slot of its CTA, and tree_finish_kernel adds a segment's slots
// in order.  Calls with as many segments as resident CTAs (444 or 592 for most forms,
// 28 or 37 sequences of 16 heads) get a CTA per segment and are not cut: there the
// longest segment sets the time.  (Cutting the list of all tiles into equal runs instead gave some
// CTAs parts of two segments, and a part costs 6 us before its first tile.)  With
// few tiles a segment goes to one CTA and no second launch follows.
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
  // no key stands past the end of the block table
  const long long rows = (long long)p.a.cache.max_blocks * p.a.cache.page_size;
  long long last = g.lens + p.a.n - 1;
  if (last > rows - 1) last = rows - 1;
  g.nt = (int)(last / kTile) - g.t0 + 1;
  if (g.nt < 1) g.nt = 1;
  return g;
}

// CTAs whose partial sums make up each segment: `count` from `first` on, 0 if the
// CTA that owned all of it wrote the rows.
struct SegSlots {
  int first, count;
};
constexpr int kMinTiles = 4;         // a run is at least this long
// This CTA's run: tiles [c0, c1] of segment seg.  False if there is none for it.
// All threads of the CTA; `tiles` is kTreeMaxCtas ints of shared memory.
__device__ __forceinline__ bool find_run(const TreeParams& p, int* tiles, SegSlots* slots, int& seg,
                                         Range& g, int& c0, int& c1, bool& whole) {
  const int segs = p.a.B * p.a.H, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (p.a.num_ctas == 1) {           // one CTA per segment
    seg = blockIdx.x;
    g = tree_range(p, seg / p.a.H, seg % p.a.H);
    c0 = g.t0;
    c1 = g.t0 + g.nt - 1;
    whole = true;
    return true;
  }
  constexpr int NW = kThreads / 32;
  __shared__ long long sum_s[NW];
  __shared__ int run_s[2];
  const int ctas = gridDim.x;
  long long sum = 0;
  // writing the nodes' rows takes the time of about a tile per 16 of them, behind a
  // segment's last (counted so, 64 nodes over 32K keys: 157 us, not counted 164)
  const int extra = p.a.k ? (p.a.n + 15) / 16 : 0;
  for (int j = tid; j < segs; j += kThreads) {
    const Range rg = tree_range(p, j / p.a.H, j % p.a.H);
    const int nt = rg.nt + (rg.any ? extra : 0);
    tiles[j] = nt;
    sum += nt;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (lane == 0) sum_s[warp] = sum;
  __syncthreads();
  sum = 0;
#pragma unroll
  for (int i = 0; i < NW; ++i) sum += sum_s[i];
  // runs of L tiles: too many at lo - 1, few enough at hi; each warp counts one
  // candidate a round
  int lo = (int)((sum + ctas - 1) / ctas);
  if (lo < kMinTiles) lo = kMinTiles;
  int hi = ctas > segs ? (int)((sum + ctas - segs - 1) / (ctas - segs)) : 0x3fffffff;
  if (hi < lo) hi = lo;
  while (lo < hi) {
    __syncthreads();
    const int cand = lo + (int)((long long)(hi - lo) * warp / NW);
    int runs = 0;
    for (int j = lane; j < segs; j += 32) runs += (tiles[j] + cand - 1) / cand;
    runs = __reduce_add_sync(0xffffffffu, runs);
    if (lane == 0) sum_s[warp] = runs;
    __syncthreads();
    int l = lo, h = hi;
#pragma unroll
    for (int i = NW - 1; i >= 0; --i) {
      const int c = lo + (int)((long long)(hi - lo) * i / NW);
      if (sum_s[i] <= ctas) h = c;
      else if (c + 1 > l) l = c + 1;
    }
    lo = l;
    hi = h;
    if (hi < lo) hi = lo;
  }
  __syncthreads();
  if (warp == 0) {                   // the segment whose runs hold this CTA
    int before = 0;
    for (int j0 = 0; j0 < segs; j0 += 32) {
      const int j = j0 + lane, n = j < segs ? (tiles[j] + hi - 1) / hi : 0;
      int inc = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += y;
      }
      const int mine = (int)blockIdx.x - (before + inc - n);
      const unsigned who = __ballot_sync(0xffffffffu, mine >= 0 && mine < n);
      if (who) {
        if (lane == __ffs(who) - 1) {
          run_s[0] = j;
          run_s[1] = mine;
        }
        break;
      }
      before += __shfl_sync(0xffffffffu, inc, 31);
      if (j0 + 32 >= segs && lane == 0) run_s[0] = -1;
    }
  }
  __syncthreads();
  seg = run_s[0];
  if (seg < 0) return false;
  const int i = run_s[1], nt = tiles[seg], n = (nt + hi - 1) / hi;
  __syncthreads();                   // `tiles` has been read
  g = tree_range(p, seg / p.a.H, seg % p.a.H);
  c0 = g.t0 + (int)((long long)nt * i / n);
  c1 = min(g.t0 + (int)((long long)nt * (i + 1) / n), g.t0 + g.nt) - 1;   // a run may be empty
  whole = n == 1;
  if (i == 0 && tid == 0) slots[seg] = SegSlots{(int)blockIdx.x, whole ? 0 : n};
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

// Rows of the nodes whose slots lie in the tiles [c0, c1] written to the pages: a
// thread per 8 elements, up to four of them in flight, the parts of a row meeting
// in `scratch` (kAppendScratch bytes of shared memory).  A whole row per lane group
// or per thread took up to 20 us for a tree of 64.  fp32 / bf16 pages: the sums of
// kv_append_kernel (four elements, then halves of the D / 4 partial sums).
constexpr int kAppendChunks = 4 * kThreads;
constexpr int kAppendScratch = kAppendChunks * 8;
template <typename E, typename TA, int D>
__device__ __forceinline__ void append_rows(const screen_tree_args& a, const Nodes& nodes, int b,
                                            int h, long long lens, int c0, int c1, void* scratch) {
  constexpr int N = 8, C = D / N, U = kAppendChunks / kThreads;
  constexpr bool kI8 = sizeof(E) == 1;
  float2* part = reinterpret_cast<float2*>(scratch);
  long long lo = (long long)c0 * kTile - lens, hi = (long long)(c1 + 1) * kTile - 1 - lens;
  if (lo < 0) lo = 0;
  if (hi > a.n - 1) hi = a.n - 1;
  const int cnt = hi >= lo ? (int)(hi - lo + 1) : 0, chunks = 2 * cnt * C;
  const int* table = a.cache.block_table + (long long)b * a.cache.max_blocks;
#pragma unroll 1
  for (int base = 0; base < chunks; base += kAppendChunks) {   // whole rows: C divides it
    float x[U][N];
    long long row[U];
    // chunk u of the batch: row (base + u) / C (K rows, then V rows), element 8 (u % C)
#pragma unroll
    for (int k = 0; k < U; ++k) {
      const int u = base + k * kThreads + threadIdx.x, r = u / C;
      const bool isv = r >= cnt;
      const int i = (int)lo + (isv ? r - cnt : r);
      row[k] = -1;
#pragma unroll
      for (int e = 0; e < N; ++e) x[k][e] = 0.f;
      if (u < chunks && nodes.line[i]) {
        load8f(reinterpret_cast<const TA*>(isv ? a.v : a.k) + (long long)b * (isv ? a.v_sb : a.k_sb) +
                   (long long)i * (isv ? a.v_st : a.k_st) + (long long)h * D + u % C * N, x[k]);
        row[k] = table_row(a.cache, table, a.H, h, lens + i);
      }
    }
#pragma unroll
    for (int k = 0; k < U; ++k) {
      float2 p;
      if constexpr (kI8) {
        uint32_t top = 0;
#pragma unroll
        for (int e = 0; e < N; ++e) top = max(top, __float_as_uint(x[k][e]) & 0x7fffffffu);
        p = make_float2(__uint_as_float(top), 0.f);
      } else {
        const float* v = x[k];
        p.x = v[0] * v[0] + v[1] * v[1] + v[2] * v[2] + v[3] * v[3];
        p.y = v[4] * v[4] + v[5] * v[5] + v[6] * v[6] + v[7] * v[7];
      }
      part[k * kThreads + threadIdx.x] = p;
    }
    __syncthreads();
    uint32_t tops[U];
    int ss[U];
#pragma unroll
    for (int k = 0; k < U; ++k) {
      const int u = k * kThreads + threadIdx.x, c = u % C;
      const float2* mine = part + (u - c);
      E* dst = reinterpret_cast<E*>((base + u) / C >= cnt ? a.cache.v_pages : a.cache.k_pages) +
               row[k] * D + c * N;
      if constexpr (kI8) {
        tops[k] = 0;
#pragma unroll
        for (int j = 0; j < C; ++j) tops[k] = max(tops[k], __float_as_uint(mine[j].x));
        uint32_t m[2];
        ss[k] = 0;
        int8_pack<N, sizeof(TA) == 2>(x[k], int8_scale<sizeof(TA) == 2>(tops[k]), m, ss[k]);
        if (row[k] >= 0) *reinterpret_cast<uint2*>(dst) = make_uint2(m[0], m[1]);
      } else {
        float p[2 * C];
#pragma unroll
        for (int j = 0; j < C; ++j) {
          p[2 * j] = mine[j].x;
          p[2 * j + 1] = mine[j].y;
        }
#pragma unroll
        for (int o = C; o > 0; o >>= 1)
#pragma unroll
          for (int j = 0; j < o; ++j) p[j] += p[j + o];
        const float nrm = fmaxf(sqrtf(p[0]), a.eps);
        if (row[k] >= 0) {
#pragma unroll
          for (int e = 0; e < N; ++e) dst[e] = from_f<E>(x[k][e] / nrm);
        }
      }
    }
    __syncthreads();
    if constexpr (kI8) {
#pragma unroll
      for (int k = 0; k < U; ++k) part[k * kThreads + threadIdx.x].y = __int_as_float(ss[k]);
      __syncthreads();
#pragma unroll
      for (int k = 0; k < U; ++k) {
        const int u = k * kThreads + threadIdx.x;
        if (u % C == 0 && row[k] >= 0) {
          int sum = 0;
#pragma unroll
          for (int j = 0; j < C; ++j) sum += __float_as_int(part[u + j].y);
          ((base + u) / C >= cnt ? a.v_scales : a.k_scales)[row[k]] =
              int8_stored_scale(tops[k], sum, a.eps);
        }
      }
      __syncthreads();
    }
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

// The whole of an SM's L1 as shared memory for `fn`: an SM whose split was made for
// another kernel's CTAs takes fewer of this one's until it has run empty.
inline void prefer_shared(const void* fn) {
  static std::mutex mu;
  static std::set<std::pair<int, const void*>> done;
  int dev = -1;
  if (cudaGetDevice(&dev) != cudaSuccess) return;
  std::lock_guard<std::mutex> lock(mu);
  if (!done.insert({dev, fn}).second) return;
  cudaFuncSetAttribute(fn, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
}

// CTAs that an SM's 228 KB of shared memory hold, `most` of them at most: a CTA takes
// its own, the static arrays (under 1.5 KB) and 1 KB more.
constexpr int fit_shared(size_t smem, int most) {
  const size_t cta = smem + 1536 + 1024, n = 228 * 1024 / cta;
  return n < (size_t)most ? (int)n : most;
}

// The grid: as many CTAs as are resident at once, num_ctas at most; one per segment,
// and num_ctas = 1, if that is no more than the segments.
inline dim3 tree_grid(TreeParams& p, int per_sm) {
  const int segs = p.a.B * p.a.H, fit = kTreeMaxCtas / 4 * per_sm;
  const int ctas = p.a.num_ctas < fit ? p.a.num_ctas : fit;
  if (ctas > segs) return dim3(ctas);
  p.a.num_ctas = 1;
  return dim3(segs);
}

}  // namespace tree
}  // namespace screen
