// Verification of drafted tokens against the target's probabilities, from
// given uniform numbers (speculative sampling on a chain or a tree).
//
// Row 0 of a sequence's logits follows its newest token, row 1 + i follows
// drafted token i.  With p = softmax(target row / T) and q = softmax(drafting
// row / T) (without drafting logits: q = 1 at the token, a token that was
// picked rather than drawn) the nodes are scanned in order; a node whose parent
// is the current row is tested:
//     accept  iff  u_i q(x) Z < p(x) - c q(x)        (c = 0, Z = 1 at a new row)
//     reject:  c += Z,  Z = sum_v max(p(v) - c q(v), 0)
// which is the residual of repeated rejections in closed form: after k of them
// it is proportional to max(p - c_k q, 0).  For a picked token a rejection
// takes the token out of p, and Z = 1 - (the mass taken out).  After the scan
// one token is drawn from the residual by inverting its running sum (in index
// order) at u_n.
//
// The tests need p(x) only: rows are read once in 32 bits (maximum, sum of
// exponentials), and a test that comes within 2e-5 of equality repeats the sum
// in 64 bits.  Residual sums and the final draw are in 64 bits: with 50K
// tokens of probability 1e-5 a running sum in 32 bits would often cross u one
// token away.
#include <cooperative_groups.h>
#include "paged.cuh"

namespace screen {
namespace {
namespace cg = cooperative_groups;

constexpr int kT = 256;              // threads of a walker CTA
constexpr int kC = 8;                // CTAs of a walker cluster
constexpr int kMaxN = SCREEN_TREE_MAX_NODES;
constexpr float kLog2e = 1.4426950408889634f;

struct RowStat {
  float m, s;   // maximum, sum of exp((x - m) / T)
  int arg;      // first index of the maximum
};
__device__ __forceinline__ bool usable(const RowStat& r) {
  return r.s > 0.f && r.s < 3.0e38f;   // no finite maximum: s is NaN
}

// Elements [v, v + 8) of a row as floats, -inf past the end.
template <typename T, bool VEC>
__device__ __forceinline__ void load8(const T* row, int v, int V, float (&x)[8]) {
  if (VEC && v + 8 <= V) {
    if constexpr (sizeof(T) == 2) {
      const uint4 u = *reinterpret_cast<const uint4*>(row + v);
      const float2 a = unpack_bf16(u.x), b = unpack_bf16(u.y), c = unpack_bf16(u.z),
                   d = unpack_bf16(u.w);
      x[0] = a.x; x[1] = a.y; x[2] = b.x; x[3] = b.y;
      x[4] = c.x; x[5] = c.y; x[6] = d.x; x[7] = d.y;
    } else {
      const float4 a = *reinterpret_cast<const float4*>(row + v);
      const float4 b = *reinterpret_cast<const float4*>(row + v + 4);
      x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
      x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = v + e < V ? to_f(row[v + e]) : -INFINITY;
  }
}

// Running (maximum, sum, argmax) of a thread, then merged pairwise.
__device__ __forceinline__ void stat_add8(RowStat& r, const float (&x)[8], int v, float sc) {
  float top = x[0];
#pragma unroll
  for (int e = 1; e < 8; ++e) top = fmaxf(top, x[e]);
  if (top > r.m) {
    r.s = r.m == -INFINITY ? r.s : r.s * exp2f((r.m - top) * sc);
    r.m = top;
#pragma unroll
    for (int e = 7; e >= 0; --e)
      if (x[e] == top) r.arg = v + e;
  }
  // -inf adds nothing; a NaN stays in the sum, as does +inf - +inf
#pragma unroll
  for (int e = 0; e < 8; ++e) r.s += x[e] == -INFINITY ? 0.f : exp2f((x[e] - r.m) * sc);
}
__device__ __forceinline__ RowStat stat_merge(const RowStat& a, const RowStat& b, float sc) {
  RowStat r;
  const bool first = a.m > b.m || (a.m == b.m && a.arg <= b.arg);
  r.m = first ? a.m : b.m;
  r.arg = first ? a.arg : b.arg;
  // an empty part (m = -inf) keeps its s: 0, or NaN from NaN elements
  const float sa = a.m == -INFINITY ? a.s : a.s * exp2f((a.m - r.m) * sc);
  const float sb = b.m == -INFINITY ? b.s : b.s * exp2f((b.m - r.m) * sc);
  r.s = sa + sb;
  return r;
}
template <int NW>
__device__ RowStat stat_block(RowStat r, float sc, RowStat* sh) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    RowStat x;
    x.m = __shfl_xor_sync(0xffffffffu, r.m, o);
    x.s = __shfl_xor_sync(0xffffffffu, r.s, o);
    x.arg = __shfl_xor_sync(0xffffffffu, r.arg, o);
    // the lower lane's part first, so that every lane ends with the same bits
    r = (lane & o) ? stat_merge(x, r, sc) : stat_merge(r, x, sc);
  }
  if (lane == 0) sh[warp] = r;
  __syncthreads();
  r = sh[0];
#pragma unroll
  for (int i = 1; i < NW; ++i) r = stat_merge(r, sh[i], sc);
  __syncthreads();
  return r;
}
// exponent scale log2(e) / T in 32 bits; T not above 0 means the maximum only
// (the sum then uses T = 1: it only says whether the row is usable)
__device__ __forceinline__ float scale_of(float temp) {
  return temp > 0.f ? fminf(kLog2e / temp, 3.0e38f) : kLog2e;
}
__device__ __forceinline__ float temp_of(const screen_verify_args& a, int b) {
  return a.temperatures ? a.temperatures[b] : a.temperature;
}

template <typename T>
__device__ __forceinline__ const T* target_row(const screen_verify_args& a, int b, int row) {
  return reinterpret_cast<const T*>(a.logits) + (long long)b * a.l_sb + (long long)row * a.l_st;
}
template <typename T>
__device__ __forceinline__ const T* draft_row(const screen_verify_args& a, int b, int row) {
  return reinterpret_cast<const T*>(a.draft_logits) + (long long)b * a.d_sb + (long long)row * a.d_st;
}

// ---------------------------------------------------------------------------
// All rows' statistics at once: one CTA of 512 threads per row, rows of the
// target first, then the drafting rows.
// ---------------------------------------------------------------------------
template <typename T, bool VEC>
__global__ void __launch_bounds__(512) row_stats_kernel(screen_verify_args a, RowStat* out) {
  pdl_wait();
  pdl_trigger();
  __shared__ RowStat sh[16];
  const int targets = a.B * (a.n + 1);
  const int id = blockIdx.x;
  const bool tgt = id < targets;
  const int b = tgt ? id / (a.n + 1) : (id - targets) / a.n;
  const T* row = tgt ? target_row<T>(a, b, id % (a.n + 1)) : draft_row<T>(a, b, (id - targets) % a.n);
  const float sc = scale_of(temp_of(a, b));
  RowStat r{-INFINITY, 0.f, 0x7fffffff};
#pragma unroll 2
  for (int v = threadIdx.x * 8; v < a.V; v += 512 * 8) {
    float x[8];
    load8<T, VEC>(row, v, a.V, x);
    stat_add8(r, x, v, sc);
  }
  r = stat_block<16>(r, sc, sh);
  if (threadIdx.x == 0) out[id] = r;
}

// ---------------------------------------------------------------------------
// Walker: a cluster of 8 CTAs per sequence.  Every CTA scans the same nodes on
// the same numbers and so takes the same branches; passes over a row are split
// over the cluster and summed in rank order by everybody.
// ---------------------------------------------------------------------------
struct Exchange {
  RowStat st[2];
  double d[2];
};

template <typename T, bool VEC>
struct Walker {
  const screen_verify_args& a;
  cg::cluster_group cl;
  Exchange* ex;
  double* red;           // [kT / 32]
  RowStat* sred;
  const int* gone;       // tokens taken out of p (picked tokens)
  int phase, rank, b, v0, v1;
  float sc;              // 32-bit exponent scale
  double isc;            // 1 / T

  __device__ RowStat cluster_stat(RowStat r) {
    r = stat_block<kT / 32>(r, sc, sred);
    if (threadIdx.x == 0) ex->st[phase] = r;
    cl.sync();
    RowStat o = *cl.map_shared_rank(&ex->st[phase], 0);
#pragma unroll
    for (int i = 1; i < kC; ++i) o = stat_merge(o, *cl.map_shared_rank(&ex->st[phase], i), sc);
    phase ^= 1;
    return o;
  }
  __device__ double block_sum(double x) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
    if (lane == 0) red[warp] = x;
    __syncthreads();
    x = red[0];
#pragma unroll
    for (int i = 1; i < kT / 32; ++i) x += red[i];
    __syncthreads();
    return x;
  }
  // sum over the cluster; `before` the ranks below this one, `mine` this one's
  __device__ double cluster_sum(double x, double& before, double& mine) {
    mine = block_sum(x);
    if (threadIdx.x == 0) ex->d[phase] = mine;
    cl.sync();
    double all = 0.0;
    before = 0.0;
#pragma unroll
    for (int i = 0; i < kC; ++i) {
      if (i == rank) before = all;
      all += *cl.map_shared_rank(&ex->d[phase], i);
    }
    phase ^= 1;
    return all;
  }
  __device__ RowStat stats(const T* row) {
    RowStat r{-INFINITY, 0.f, 0x7fffffff};
    for (int v = v0 + threadIdx.x * 8; v < v1; v += kT * 8) {
      float x[8];
      load8<T, VEC>(row, v, a.V, x);
      stat_add8(r, x, v, sc);
    }
    return cluster_stat(r);
  }
  __device__ double e64(float x, float m) const {
    return x == -INFINITY ? 0.0 : exp(((double)x - (double)m) * isc);
  }
  // what a pass sums: 0 exp of the row; 1 the same without the tokens taken
  // out; 2 max(ip e_p - iq e_q, 0)
  struct Weights {
    int kind, n_gone;
    const T *p, *q;
    float mp, mq;
    double ip, iq;
  };
  __device__ void weights8(const Weights& w, int v, double (&o)[8]) const {
    float x[8];
    load8<T, VEC>(w.p, v, a.V, x);
#pragma unroll
    for (int e = 0; e < 8; ++e) o[e] = e64(x[e], w.mp);
    if (w.kind == 1) {
      for (int k = 0; k < w.n_gone; ++k) {
        const int d = gone[k] - v;
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (d == e) o[e] = 0.0;
      }
    } else if (w.kind == 2) {
      float y[8];
      load8<T, VEC>(w.q, v, a.V, y);
#pragma unroll
      for (int e = 0; e < 8; ++e) o[e] = fmax(w.ip * o[e] - w.iq * e64(y[e], w.mq), 0.0);
    }
  }
  __device__ double sum(const Weights& w, double& before, double& mine) {
    double s = 0.0;
    for (int v = v0 + threadIdx.x * 8; v < v1; v += kT * 8) {
      double o[8];
      weights8(w, v, o);
#pragma unroll
      for (int e = 0; e < 8; ++e) s += o[e];
    }
    return cluster_sum(s, before, mine);
  }
  __device__ double sum(const Weights& w) {
    double x, y;
    return sum(w, x, y);
  }
};

template <typename T, bool VEC>
__global__ void __launch_bounds__(kT) walk_kernel(screen_verify_args a, const RowStat* stats) {
  __shared__ Exchange ex;
  __shared__ double red[kT / 32];
  __shared__ RowStat sred[kT / 32];
  __shared__ unsigned long long children[kMaxN + 1];
  __shared__ long long tok[kMaxN];
  __shared__ float lp[kMaxN], lq[kMaxN], un[kMaxN];
  __shared__ int gone[kMaxN];
  __shared__ int path[kMaxN];
  __shared__ double scan_s[kT / 32];
  __shared__ int found_s, last_s;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  pdl_wait();
  pdl_trigger();
  cg::cluster_group cl = cg::this_cluster();
  const int n = a.n, V = a.V;
  const int b = blockIdx.x / kC;
  const bool drawn = a.draft_logits != nullptr;
  const float temp = temp_of(a, b);
  const bool greedy = !(temp > 0.f);
  const int rank = (int)cl.block_rank();
  const int span = ((V + 8 * kC - 1) / (8 * kC)) * 8;
  Walker<T, VEC> w{a, cl, &ex, red, sred, gone, 0, rank, b, min(V, rank * span),
                   min(V, (rank + 1) * span), scale_of(temp), greedy ? 1.0 : 1.0 / (double)temp};

  for (int i = tid; i <= kMaxN; i += kT) children[i] = 0ull;
  __syncthreads();
  if (tid < n) {
    const int i = tid;
    const int p = a.parents ? a.parents[(long long)b * a.p_sb + i] : i - 1;
    const long long x = a.tokens[(long long)b * a.t_sb + i];
    tok[i] = x;
    un[i] = a.uniforms[(long long)b * a.u_sb + i];
    if (p >= -1 && p < i && x >= 0 && x < V) {
      lp[i] = to_f(target_row<T>(a, b, p + 1)[x]);
      lq[i] = drawn ? to_f(draft_row<T>(a, b, p + 1)[x]) : 0.f;
      atomicOr(&children[p + 1], 1ull << i);
    }
  }
  __syncthreads();

  using W = typename Walker<T, VEC>::Weights;
  int cur = 0, count = 0;
  long long token = -1;
  while (true) {
    // --- a new row ------------------------------------------------------------
    const T* prow = target_row<T>(a, b, cur);
    const T* qrow = drawn && cur < n ? draft_row<T>(a, b, cur) : nullptr;
    unsigned long long left = children[cur];
    RowStat ps = stats ? stats[(long long)b * (n + 1) + cur] : w.stats(prow);
    RowStat qs{0.f, 1.f, 0};
    if (drawn && left)
      qs = stats ? stats[(long long)a.B * (n + 1) + (long long)b * n + cur] : w.stats(qrow);
    if (!usable(ps)) break;                       // no distribution: no token
    if (drawn && !usable(qs)) left = 0;           // nothing was drawn from this
    double sp = ps.s, sq = qs.s;                  // sums, exact once `exact`
    bool exact = greedy;
    double c = 0.0, z = 1.0, out_mass = 0.0;      // out_mass: exp sum taken out
    int n_gone = 0, next = -1;
    auto make_exact = [&] {
      if (exact) return;
      sp = w.sum(W{0, 0, prow, nullptr, ps.m, 0.f, 0.0, 0.0});
      if (drawn) sq = w.sum(W{0, 0, qrow, nullptr, qs.m, 0.f, 0.0, 0.0});
      exact = true;
      if (!drawn) z = 1.0 - out_mass / sp;
    };
    while (left) {
      const int i = __ffsll((long long)left) - 1;
      left &= left - 1;
      const int x = (int)tok[i];
      const double u = un[i];
      bool dup = false;
      if (!drawn)
        for (int k = 0; k < n_gone; ++k) dup = dup || gone[k] == x;
      bool accept = false;
      for (int go = 0; go < 2; ++go) {
        double px, qx;
        if (greedy) {
          px = x == ps.arg ? 1.0 : 0.0;
          qx = !drawn || x == qs.arg ? 1.0 : 0.0;
        } else {
          px = w.e64(lp[i], ps.m) / sp;
          qx = drawn ? w.e64(lq[i], qs.m) / sq : 1.0;
        }
        if (dup) px = 0.0;
        const double pr = px - c * qx, need = u * qx * z;
        accept = pr > 0.0 && need < pr;
        if (exact || fabs(need - pr) > 2e-5 * (fabs(need) + fabs(px) + c * qx + u * qx)) break;
        make_exact();
      }
      if (accept) {
        next = i;
        break;
      }
      // rejected
      if (drawn) {
        if (greedy) {
          // p and q are one point each: the residual keeps p where q is not
          c += z;
          z = fmax((ps.arg == qs.arg ? 1.0 - c : 1.0), 0.0);
        } else {
          make_exact();
          c += z;
          z = w.sum(W{2, 0, prow, qrow, ps.m, qs.m, 1.0 / sp, c / sq});
        }
      } else if (!dup) {
        __syncthreads();
        if (tid == 0) gone[n_gone] = x;
        __syncthreads();
        ++n_gone;
        if (greedy) {
          if (x == ps.arg) z = 0.0;
        } else {
          out_mass += w.e64(lp[i], ps.m);
          z = 1.0 - out_mass / sp;
          if (z < 1e-4) {                          // too little left for a difference
            make_exact();
            z = w.sum(W{1, n_gone, prow, nullptr, ps.m, 0.f, 0.0, 0.0}) / sp;
          }
        }
      }
    }
    if (next >= 0) {
      if (tid == 0) path[count] = next;
      ++count;
      cur = next + 1;
      continue;
    }
    // --- the last token: the residual at u_n ----------------------------------
    if (greedy) {
      token = ps.arg;                              // rejected nodes were not it
      break;
    }
    const double u = a.uniforms[(long long)b * a.u_sb + n];
    W wt{0, 0, prow, qrow, ps.m, qs.m, 0.0, 0.0};
    if (drawn && c > 0.0 && z > 0.0) {
      wt.kind = 2;
      wt.ip = 1.0 / sp;
      wt.iq = c / sq;
    } else if (!drawn && n_gone) {
      wt.kind = 1;
      wt.n_gone = n_gone;
    }
    double before, mine;
    double all = w.sum(wt, before, mine);
    if (!(all > 0.0)) {                            // nothing left: p itself
      wt.kind = 0;
      all = w.sum(wt, before, mine);
    }
    const double goal = fmax(u * all, 0.0);
    // the CTA whose part holds the crossing looks for it; if the rounding of
    // its sums leaves none, the largest index with weight is taken
    if (tid == 0) {
      found_s = 0x7fffffff;
      last_s = -1;
    }
    __syncthreads();
    const bool here = before <= goal && before + mine > goal;   // one rank at most
    if (before <= goal) {
      double base = before;
      for (int t0 = w.v0; t0 < w.v1; t0 += kT * 8) {
        const int v = t0 + tid * 8;
        double o[8] = {0, 0, 0, 0, 0, 0, 0, 0};
        if (v < w.v1) w.weights8(wt, v, o);
        double s = 0.0;
#pragma unroll
        for (int e = 0; e < 8; ++e) s += o[e];
        double inc = s;                            // inclusive scan over the warp
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
          const double y = __shfl_up_sync(0xffffffffu, inc, d);
          if (lane >= d) inc += y;
        }
        if (lane == 31) scan_s[warp] = inc;
        __syncthreads();
        double off = base;
        for (int k = 0; k < warp; ++k) off += scan_s[k];
        double tot = 0.0;
        for (int k = 0; k < kT / 32; ++k) tot += scan_s[k];
        double run = off + (inc - s);
        int hit = 0x7fffffff, lastw = -1;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          run += o[e];
          if (o[e] > 0.0) {
            lastw = v + e;
            if (run > goal && hit == 0x7fffffff) hit = v + e;
          }
        }
        if (here && hit != 0x7fffffff) atomicMin(&found_s, hit);
        if (lastw >= 0) atomicMax(&last_s, lastw);
        base += tot;
        __syncthreads();
        if (found_s != 0x7fffffff) break;          // uniform: read after the barrier
      }
    }
    __syncthreads();
    // the lowest crossing of the cluster, else the last weighted index
    if (tid == 0) {
      ex.st[w.phase].arg = here && found_s == 0x7fffffff && last_s >= 0 ? last_s : found_s;
      ex.d[w.phase] = (double)last_s;
    }
    cl.sync();
    int best = 0x7fffffff, lst = -1;
#pragma unroll
    for (int i = 0; i < kC; ++i) {
      best = min(best, cl.map_shared_rank(&ex.st[w.phase], i)->arg);
      lst = max(lst, (int)*cl.map_shared_rank(&ex.d[w.phase], i));
    }
    token = best != 0x7fffffff ? best : lst;
    break;
  }
  __syncthreads();
  if (rank == 0) {
    for (int i = tid; i <= n; i += kT) {
      if (i < n) a.path[(long long)b * n + i] = i < count ? path[i] : -1;
      a.out_tokens[(long long)b * (n + 1) + i] = i < count ? tok[path[i]] : i == count ? token : -1;
    }
    if (tid == 0) a.counts[b] = count;
  }
  cl.sync();   // nobody's shared memory goes away while a rank may read it
}

// All rows are read up front while that costs less than the walk's own waits
// (a row's pass by a cluster takes a few microseconds, one row after another).
bool stats_up_front(const screen_verify_args& a) {
  const size_t rows = (size_t)a.B * (a.n + 1) + (a.draft_logits ? (size_t)a.B * a.n : 0);
  return rows * a.V * (a.dtype == SCREEN_F32 ? 4 : 2) <= (48u << 20);
}

template <typename T, bool VEC>
void launch_verify(const screen_verify_args& a, cudaStream_t s) {
  RowStat* st = nullptr;
  if (stats_up_front(a)) {
    st = reinterpret_cast<RowStat*>(a.workspace);
    const int rows = a.B * (a.n + 1) + (a.draft_logits ? a.B * a.n : 0);
    launch_pdl(row_stats_kernel<T, VEC>, dim3(rows), dim3(512), 0, s, a, st);
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(a.B * kC);
  cfg.blockDim = dim3(kT);
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = kC;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  cudaLaunchKernelEx(&cfg, walk_kernel<T, VEC>, a, (const RowStat*)st);
}
template <typename T>
void verify_t(const screen_verify_args& a, cudaStream_t s) {
  const int vec = 16 / (int)sizeof(T);
  bool ok = ((uintptr_t)a.logits & 15) == 0 && a.l_sb % vec == 0 && a.l_st % vec == 0;
  if (a.draft_logits)
    ok = ok && ((uintptr_t)a.draft_logits & 15) == 0 && a.d_sb % vec == 0 && a.d_st % vec == 0;
  if (ok) launch_verify<T, true>(a, s);
  else launch_verify<T, false>(a, s);
}

}  // namespace

size_t verify_workspace(const screen_verify_args& a) {
  return ((size_t)a.B * (2 * (size_t)a.n + 1)) * sizeof(RowStat);
}
void verify(const screen_verify_args& a, cudaStream_t s) {
  if (a.dtype == SCREEN_F32) verify_t<float>(a, s);
  else verify_t<__nv_bfloat16>(a, s);
}

}  // namespace screen
