// Tree attention over fp32 pages, and the pass that finishes split runs.
#include "tree_decode.cuh"

namespace screen {
namespace tree {
namespace {

// fp32 pages keep the 1e-4 contract of the fp32 path with plain fp32 FMAs: 32
// keys at a time in shared memory, one (query, key) score per thread and step,
// then alpha V with the threads over (query group, d).  Bound by the FMAs and the
// shared-memory reads that feed them.
constexpr int kKeys = 32;

template <int D>
__global__ void __launch_bounds__(kThreads) tree_f32_kernel(TreeParams p, float* __restrict__ ws) {
  constexpr int LD = D + 4;                        // rows of 16-byte pieces on distinct banks
  constexpr int QG = kThreads / D < 1 ? 1 : kThreads / D;  // query groups in alpha V
  constexpr int PQ = (kMaxN + QG - 1) / QG;
  extern __shared__ __align__(16) float fsm[];
  float* qs = fsm;                                 // [n][D] unit queries
  float* kt = qs + (size_t)p.a.n * D;              // [32][LD]
  float* vt = kt + kKeys * LD;
  float* al = vt + kKeys * LD;                     // [n][33]
  static_assert(2 * kKeys * LD * 4 >= kAppendScratch, "append_rows works in the key tiles");
  __shared__ Nodes nodes;
  __shared__ int c_s[kKeys];
  __shared__ long long row_s[kKeys];
  pdl_wait();
  pdl_trigger();
  const screen_tree_args& a = p.a;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int n = a.n;
  SegSlots* slots = reinterpret_cast<SegSlots*>(ws);
  float* part = ws + p.part_off;
  Range rg;
  int seg, c0, c1;
  bool whole;
  if (!find_run(p, reinterpret_cast<int*>(fsm), slots, seg, rg, c0, c1, whole)) return;
  const int b = seg / a.H, h = seg % a.H;
  const float w = a.w[h], r = a.r[h];
  const long long lens = rg.lens;
  if (warp == 0) tree_nodes(a, b, nodes, lane);
  __syncthreads();
  if (rg.any && a.k) append_rows<float, float, D>(a, nodes, b, h, lens, c0, c1, kt);
  for (int i = warp; i < n; i += 4) {
    const float* q = reinterpret_cast<const float*>(a.q) + (long long)b * a.q_sb +
                     (long long)i * a.q_st + (long long)h * D;
    float ss = 0.f;
    for (int d = lane; d < D; d += 32) ss = fmaf(q[d], q[d], ss);
    ss = warp_sum(ss);
    const float nrm = fmaxf(sqrtf(ss), a.eps);
    for (int d = lane; d < D; d += 32) qs[i * D + d] = q[d] / nrm;
  }
  const int dd = tid % D, qg = tid / D;
  float acc[PQ];
#pragma unroll
  for (int x = 0; x < PQ; ++x) acc[x] = 0.f;
  const int k0 = c0 * (kTile / kKeys), k1 = rg.any ? (c1 + 1) * (kTile / kKeys) - 1 : k0 - 1;
  for (int tile = k0; tile <= k1; ++tile) {
    __syncthreads();
    if (tid < kKeys) {
      const long long pos = (long long)tile * kKeys + tid;
      int c = kNoKey;
      long long row = -1;
      if (pos >= rg.first && pos < lens + n) {
        const long long slot = pos - lens;
        if (slot < 0) c = (int)slot;
        else if (nodes.line[slot]) c = nodes.depth[slot];
        if (c != kNoKey) row = paged_row(a.cache, b, a.H, h, pos);
        if (row < 0) c = kNoKey;
      }
      c_s[tid] = c;
      row_s[tid] = row;
    }
    __syncthreads();
    for (int u = tid; u < kKeys * (D / 4); u += kThreads) {
      const int k = u / (D / 4), d = u % (D / 4) * 4;
      const long long row = row_s[k];
      cp_async16(smem_u32(kt + k * LD + d),
                 reinterpret_cast<const float*>(a.cache.k_pages) + (row < 0 ? 0 : row) * D + d, row >= 0);
      cp_async16(smem_u32(vt + k * LD + d),
                 reinterpret_cast<const float*>(a.cache.v_pages) + (row < 0 ? 0 : row) * D + d, row >= 0);
    }
    cp_async_commit();
    cp_async_wait<0>();
    __syncthreads();
    const int c = c_s[lane];
    const long long slot = (long long)tile * kKeys + lane - lens;
    for (int i = warp; i < n; i += 4) {
      const int dep = nodes.depth[i];
      bool see = nodes.line[i] != 0 && c != kNoKey && dep - c <= rg.dmax;
      if (slot >= 0 && slot < n) see = see && (nodes.line[i] >> slot & 1);
      float dot = 0.f;
#pragma unroll
      for (int d = 0; d < D; d += 4) {
        const float4 kk = *reinterpret_cast<const float4*>(kt + lane * LD + d);
        const float4 qq = *reinterpret_cast<const float4*>(qs + i * D + d);
        dot = fmaf(kk.x, qq.x, fmaf(kk.y, qq.y, fmaf(kk.z, qq.z, fmaf(kk.w, qq.w, dot))));
      }
      const float t = 1.0f - r * (1.0f - dot);
      float v = 0.f;
      if (see && t > 0.f) v = t * t * (0.5f * (cospif((float)(c - dep) / w) + 1.0f));
      al[i * 33 + lane] = v;
    }
    __syncthreads();
    if (qg < QG) {
#pragma unroll
      for (int x = 0; x < PQ; ++x) {
        const int i = qg + x * QG;
        if (i < n)
          for (int k = 0; k < kKeys; ++k) {
            const float v = al[i * 33 + k];
            if (v != 0.f) acc[x] = fmaf(v, vt[k * LD + dd], acc[x]);
          }
      }
    }
  }
  // rows to shared memory (over the queries), then one warp per row
  __syncthreads();
  if (qg < QG) {
#pragma unroll
    for (int x = 0; x < PQ; ++x)
      if (qg + x * QG < n) qs[(qg + x * QG) * D + dd] = acc[x];
  }
  __syncthreads();
  constexpr int PER = D < 32 ? 1 : D / 32;
  for (int i = warp; i < n; i += 4) {
    float x[PER];
#pragma unroll
    for (int e = 0; e < PER; ++e) x[e] = lane + 32 * e < D ? qs[i * D + lane + 32 * e] : 0.f;
    if (!whole) {
      float* dst = part + ((size_t)blockIdx.x * n + i) * D;
#pragma unroll
      for (int e = 0; e < PER; ++e)
        if (lane + 32 * e < D) dst[lane + 32 * e] = x[e];
    } else {
      store_row<float, D>(a, b, i, h, lane, x, rg.any && nodes.line[i] != 0);
    }
  }
}

// Sum a segment's partials in the order of its runs, TanhNorm, store; a warp per
// (segment, node).  The sum of an absent node is zero (nothing was seen).
template <typename TA, int D>
__global__ void __launch_bounds__(128) tree_finish_kernel(TreeParams p, const float* __restrict__ ws) {
  pdl_wait();
  pdl_trigger();
  constexpr int PER = D < 32 ? 1 : D / 32;
  const screen_tree_args& a = p.a;
  const int lane = threadIdx.x & 31;
  const long long row = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (row >= (long long)a.B * a.H * a.n) return;
  const int i = (int)(row % a.n), seg = (int)(row / a.n);
  const SegSlots q = reinterpret_cast<const SegSlots*>(ws)[seg];
  if (q.count == 0) return;   // written by the CTA that owned the segment
  float x[PER];
#pragma unroll
  for (int e = 0; e < PER; ++e) x[e] = 0.f;
  const float* src = ws + p.part_off + (size_t)i * D;
#pragma unroll 4
  for (int c = q.first; c < q.first + q.count; ++c)
#pragma unroll
    for (int e = 0; e < PER; ++e)
      if (lane + 32 * e < D) x[e] += src[(size_t)c * a.n * D + lane + 32 * e];
  store_row<TA, D>(a, seg / a.H, i, seg % a.H, lane, x, true);
}

template <int D>
bool launch_f32(TreeParams& p, float* part, cudaStream_t s) {
  const size_t smem = ((size_t)p.a.n * D + 2 * kKeys * (D + 4) + (size_t)p.a.n * 33) * 4;
  static_assert(2 * kKeys * (D + 4) >= kTreeMaxCtas, "find_run works in it");
  constexpr int kMost = (kMaxN * D + 2 * kKeys * (D + 4) + kMaxN * 33) * 4;
  if (ensure_smem_optin((const void*)tree_f32_kernel<D>, kMost) != cudaSuccess) return false;
  prefer_shared((const void*)tree_f32_kernel<D>);
  // three CTAs an SM where they fit (64 nodes of 128: two)
  static_assert(sizeof(Nodes) + kKeys * 12 + 64 <= 1536, "the static arrays are counted");
  const dim3 grid = tree_grid(p, fit_shared(smem, 3));
  launch_pdl(tree_f32_kernel<D>, grid, dim3(kThreads), smem, s, p, part);
  return p.a.num_ctas > 1;
}
template <typename TA, int D>
void launch_finish(const TreeParams& p, const float* part, cudaStream_t s) {
  const long long rows = (long long)p.a.B * p.a.H * p.a.n;
  prefer_shared((const void*)tree_finish_kernel<TA, D>);
  launch_pdl(tree_finish_kernel<TA, D>, dim3((unsigned)((rows + 3) / 4)), dim3(128), 0, s, p, part);
}
template <typename TA>
void finish_d(const TreeParams& p, const float* part, cudaStream_t s) {
  switch (p.a.D) {
    case 16: launch_finish<TA, 16>(p, part, s); break;
    case 32: launch_finish<TA, 32>(p, part, s); break;
    case 64: launch_finish<TA, 64>(p, part, s); break;
    case 128: launch_finish<TA, 128>(p, part, s); break;
  }
}

}  // namespace
}  // namespace tree

bool tree_f32(TreeParams p, float* part, cudaStream_t s) {
  switch (p.a.D) {
    case 16: return tree::launch_f32<16>(p, part, s);
    case 32: return tree::launch_f32<32>(p, part, s);
    case 64: return tree::launch_f32<64>(p, part, s);
    default: return tree::launch_f32<128>(p, part, s);
  }
}
void tree_finish(const TreeParams& p, const float* part, cudaStream_t s) {
  if (p.a.dtype == SCREEN_F32) tree::finish_d<float>(p, part, s);
  else tree::finish_d<__nv_bfloat16>(p, part, s);
}

}  // namespace screen
