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
// A cluster of CTAs per sequence walks its tree.  Every CTA of the cluster scans
// the same nodes on the same numbers and takes the same branches; a pass over a
// row is split over the cluster, its parts are exchanged through distributed
// shared memory and added in rank order by everybody.  With few rows in all a
// first kernel sums every row over the whole GPU and the walk only adds the
// parts; a big batch of trees (33 rows each, of which a walk passes two or
// three) is read row by row as the walk gets there.
//
// Bound by the passes of a walk, one after another, each a row through the 64-bit
// units of a cluster's SMs: 4 chains of 4 with drafting logits over 50257 tokens 24
// us, 32 trees of 32 34 us; greedy, where only the sums' health is used, 14 and 28 us.
//
// Sums are in 64 bits throughout: with 50K tokens of probability 1e-5 a running
// sum in 32 bits would often cross u one token away, and an acceptance test next
// to equality would tip.  The exponentials are good to 2^-31, which moves the
// borders of the draw by about 1e-12 of the whole.
#include <cooperative_groups.h>
#include "paged.cuh"

namespace screen {
namespace {
namespace cg = cooperative_groups;

constexpr int kT = 256;              // threads of a CTA
constexpr int kMaxC = 8;             // CTAs of a cluster, at most
constexpr int kMaxN = SCREEN_TREE_MAX_NODES;
constexpr int kNone = 0x7fffffff;

// A finite float (or -inf, as -2^128) as a double by moving its bits; numbers
// below 2^-126 as 0.
__device__ __forceinline__ double wide(float x) {
  const uint32_t u = __float_as_uint(x), m = u & 0x7fffffffu;
  const uint32_t hi = m < 0x00800000u ? 0u : (m >> 3) + 0x38000000u;
  return __hiloint2double((int)((u & 0x80000000u) | hi), (int)(m << 29));
}
// 2^y for a few single y <= 0 (a little above is fine): n = rint(y), f = y - n and
// the Taylor polynomial of 2^f, |f| <= 1/2, whose first dropped term
// (f ln 2)^11 / 11! is below 2.2e-13.  Under 2^-1000 it counts as 0.
__device__ __forceinline__ double exp2_64(double y) {
  const double magic = 6755399441055744.0;   // 1.5 * 2^52
  const double t = y + magic;
  const int n = __double2loint(t);
  const double f = (y - (t - magic)) * 0.6931471805599453;
  double p = 1.0 / 3628800.0;
  p = fma(f, p, 1.0 / 362880.0);
  p = fma(f, p, 1.0 / 40320.0);
  p = fma(f, p, 1.0 / 5040.0);
  p = fma(f, p, 1.0 / 720.0);
  p = fma(f, p, 1.0 / 120.0);
  p = fma(f, p, 1.0 / 24.0);
  p = fma(f, p, 1.0 / 6.0);
  p = fma(f, p, 0.5);
  p = fma(f, p, 1.0);
  p = fma(f, p, 1.0);
  const double e = __hiloint2double(__double2hiint(p) + (n << 20), __double2loint(p));
  return y < -1000.0 ? 0.0 : e;
}

// exp((x - m) / T) of 8 elements of a row, c2 = log2(e) / T, k = c2 m, in
// three 64-bit operations each (a chain as above ran at 1.5 exponentials per
// cycle and SM: 64-bit FMAs of three registers at 28, conversions at 16; this
// at 4).
// Table-driven after P. Tang (1989): adding 1.5 * 2^12 leaves y = x c2 - k in the
// low word pair as a fixed-point number, bits 40.. its integer part n, the next 8
// an index j, the last 32 a remainder g < 2^-8; 2^y = 2^n T[j] (1 + w) with
// T[j] = 2^(j/256) and w = 2^g - 1 = u + u^2/2 + u^3/6, u = g ln 2, in 32 bits: the
// dropped u^4/24 is below 3e-12, w's rounding below 2^-24 * 2.8e-3.  Where k is
// large (a temperature near 0) x c2 - k would lose the low bits of both, so x - m is
// taken first, with one operation more.
constexpr int kTab = 256;
__device__ __forceinline__ void fill_table(double* tab) {
  for (int i = threadIdx.x; i < kTab; i += blockDim.x) tab[i] = 2.0 * exp2_64((double)i / kTab - 1.0);
}
__device__ __forceinline__ void exp8(const float (&x)[8], double c2, double m, const double* tab,
                                     double (&o)[8]) {
  // step by step over the eight, so that their chains run side by side (one
  // after another took 1170 cycles a warp, this 450)
  const double k = c2 * m, base = 6144.0 - k;
  double t[8], w[8];
  int hi[8];
  float u[8];
  if (fabs(k) <= 8192.0) {           // uniform
#pragma unroll
    for (int e = 0; e < 8; ++e) t[e] = fma(c2, wide(x[e]), base);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) t[e] = fma(c2, wide(x[e]) - m, 6144.0);
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    hi[e] = __double2hiint(t[e]);
    u[e] = __uint2float_rn((uint32_t)__double2loint(t[e])) * 6.304136882681135e-13f;   // ln(2) 2^-40
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) t[e] = tab[hi[e] & (kTab - 1)];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const uint32_t b = __float_as_uint(fmaf(u[e] * u[e], fmaf(u[e], 1.0f / 6.0f, 0.5f), u[e]));
    w[e] = __hiloint2double((int)((b >> 3) + 0x38000000u), (int)(b << 29));   // as wide()
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) t[e] = fma(t[e], w[e], t[e]);
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const int n20 = (int)(((uint32_t)hi[e] << 12) & 0xfff00000u) - (int)0x80000000u;   // n << 20
    const double r = __hiloint2double(__double2hiint(t[e]) + n20, __double2loint(t[e]));
    o[e] = hi[e] < 0x40b41800 ? 0.0 : r;   // y < -1000 (a negative sum among them)
  }
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

// A row, or a part of one: first index of the maximum, sum of
// exp((x - m) / T); s is NaN with a NaN or +inf in it, 0 if all is -inf.
struct RowSum {
  double s;
  float m;
  int arg;
};
__device__ __forceinline__ bool usable(const RowSum& r) { return r.s > 0.0; }

__device__ __forceinline__ double add8(const double (&o)[8]) {
  return ((o[0] + o[1]) + (o[2] + o[3])) + ((o[4] + o[5]) + (o[6] + o[7]));
}
__device__ __forceinline__ double warp_add(double s) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  return s;
}

// The part of a row that a CTA owns, elements [v0, v1), in at most kUnits units
// of 256 k elements; a warp takes a unit, a lane 8 elements at a time.  The sums
// of the units are kept: they lead the final draw to the unit it falls in.
constexpr int kUnits = 512;
struct Part {
  int v0, v1, k, units;
};
__device__ __forceinline__ Part part_of(int V, int rank, int C) {
  const int span = (V + 8 * C - 1) / (8 * C) * 8;
  Part t;
  t.v0 = min(V, rank * span);
  t.v1 = min(V, t.v0 + span);
  t.k = (span + kUnits * 256 - 1) / (kUnits * 256);
  t.units = (t.v1 - t.v0 + 256 * t.k - 1) / (256 * t.k);
  return t;
}

// Weights that a pass sums: exp of p's row; without the tokens taken out; or,
// with q, max(ip e_p - iq e_q, 0).
template <typename T>
struct Weights {
  const T *p, *q;
  double mp, mq, ip, iq;   // maxima; factors
  int n_gone;
  const int* gone;
};
template <typename T, bool VEC>
__device__ __forceinline__ void weights8(const Weights<T>& w, double c2, const double* tab, int v, int V,
                                         double (&o)[8]) {
  float x[8], y[8];
  load8<T, VEC>(w.p, v, V, x);
  if (w.q) load8<T, VEC>(w.q, v, V, y);
  exp8(x, c2, w.mp, tab, o);
  if (w.q) {
    double f[8];
    exp8(y, c2, w.mq, tab, f);
#pragma unroll
    for (int e = 0; e < 8; ++e) o[e] = fmax(w.ip * o[e] - w.iq * f[e], 0.0);
  }
#pragma unroll 1
  for (int k = 0; k < w.n_gone; ++k) {
    const int d = w.gone[k] - v;
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (d == e) o[e] = 0.0;
  }
}
// Sums of the units into wsum; the part's sum to warp 0's lanes.  Ends with the
// CTA in step.
template <typename T, bool VEC>
__device__ double sum_part(const Weights<T>& w, double c2, const double* tab, const Part& t, int V,
                           double* wsum) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll 1
  for (int u = warp; u < t.units; u += kT / 32) {
    double s = 0.0;
#pragma unroll 1
    for (int i = 0; i < t.k; ++i) {
      const int v = t.v0 + (u * t.k + i) * 256 + lane * 8;
      if (v < t.v1) {
        double o[8];
        weights8<T, VEC>(w, c2, tab, v, V, o);
        s += add8(o);
      }
    }
    s = warp_add(s);
    if (lane == 0) wsum[u] = s;
  }
  __syncthreads();
  double s = 0.0;
  if (warp == 0) {
    for (int u = lane; u < t.units; u += 32) s += wsum[u];
    s = warp_add(s);
  }
  return s;
}
// Maximum, its first index and health of the part of a row, to everybody.
template <typename T, bool VEC>
__device__ RowSum top_part(const T* row, const Part& t, int V, RowSum* sh) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  float top = -INFINITY;
  int arg = kNone;
  bool bad = false;
  constexpr int U = 4;               // loads in flight
#pragma unroll 1
  for (int v = t.v0 + threadIdx.x * 8; v < t.v1; v += kT * 8 * U) {
    float x[U][8];
#pragma unroll
    for (int k = 0; k < U; ++k)
      load8<T, VEC>(row, v + k * kT * 8 < t.v1 ? v + k * kT * 8 : V, V, x[k]);
    float m = -INFINITY;
#pragma unroll
    for (int k = 0; k < U; ++k)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        m = fmaxf(m, x[k][e]);
        bad = bad || !(x[k][e] < INFINITY);   // +inf or NaN
      }
    if (m > top) {
      top = m;
#pragma unroll
      for (int k = U - 1; k >= 0; --k)
#pragma unroll
        for (int e = 7; e >= 0; --e)
          if (x[k][e] == m) arg = v + k * kT * 8 + e;
    }
  }
  float m = top;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  arg = __reduce_min_sync(0xffffffffu, top == m ? arg : kNone);
  bad = __any_sync(0xffffffffu, bad);
  if (lane == 0) sh[warp] = RowSum{bad ? __longlong_as_double(0x7ff8000000000000ll) : 0.0, m, arg};
  __syncthreads();
  RowSum r{0.0, -INFINITY, kNone};
#pragma unroll
  for (int i = 0; i < kT / 32; ++i) {
    const RowSum x = sh[i];
    if (x.m > r.m || (x.m == r.m && x.arg < r.arg)) {
      r.m = x.m;
      r.arg = x.arg;
    }
    r.s += x.s;
  }
  __syncthreads();
  return r;
}
// The part of a row: its RowSum in thread 0 (m and arg everywhere).
template <typename T, bool VEC>
__device__ RowSum row_part(const T* row, const Part& t, int V, double c2, const double* tab, RowSum* sh,
                           double* wsum) {
  RowSum r = top_part<T, VEC>(row, t, V, sh);
  if (r.m != -INFINITY) {            // uniform
    const Weights<T> w{row, nullptr, wide(r.m), 0.0, 0.0, 0.0, 0, nullptr};
    r.s += sum_part<T, VEC>(w, c2, tab, t, V, wsum);
  }
  return r;
}

__device__ __forceinline__ float temp_of(const screen_verify_args& a, int b) {
  return a.temperatures ? a.temperatures[b] : a.temperature;
}
// log2(e) / T; T = 0 means the maximum only (any positive T then tells whether the row
// is usable), below 0 or NaN nothing.  T counts as 1e30 above that: -inf, held as -2^128,
// keeps the weight 0.
__device__ __forceinline__ double scale_of(float temp) {
  return 1.4426950408889634 / (temp > 0.f ? fmin((double)temp, 1e30) : 1.0);
}

// ---------------------------------------------------------------------------
// All rows at once: CTA (part, row); rows of the target first, then drafting rows.
// ---------------------------------------------------------------------------
template <typename T, bool VEC>
__global__ void __launch_bounds__(kT, 2) rows_kernel(screen_verify_args a, RowSum* out) {
  __shared__ RowSum sh[kT / 32];
  __shared__ double wsum[kUnits], tab[kTab];
  fill_table(tab);       // the first barrier of top_part comes before its use
  pdl_wait();
  pdl_trigger();
  const int C = gridDim.x, targets = a.B * (a.n + 1), id = blockIdx.y;
  const bool tgt = id < targets;
  const int b = tgt ? id / (a.n + 1) : (id - targets) / a.n;
  const T* row = tgt ? reinterpret_cast<const T*>(a.logits) + (long long)b * a.l_sb + (id % (a.n + 1)) * a.l_st
                     : reinterpret_cast<const T*>(a.draft_logits) + (long long)b * a.d_sb +
                           ((id - targets) % a.n) * a.d_st;
  const RowSum r = row_part<T, VEC>(row, part_of(a.V, blockIdx.x, C), a.V, scale_of(temp_of(a, b)), tab,
                                      sh, wsum);
  if (threadIdx.x == 0) out[(long long)id * C + blockIdx.x] = r;
}

// ---------------------------------------------------------------------------
// The walk.
// ---------------------------------------------------------------------------
struct Exchange {
  RowSum r[2][2];        // [phase][p, q]
  double d[2];
  int token;
};

template <typename T, bool VEC>
struct Walker {
  const screen_verify_args& a;
  const RowSum* given;   // all rows' parts, or NULL: read as the walk gets there
  cg::cluster_group cl;
  Exchange* ex;
  RowSum* sh;            // [kT / 32]
  double* wsum;          // [kUnits]
  const double* tab;
  int phase, rank, C, b;
  Part t;
  double c2;

  // Lane i holds rank i's part: their sum, the ranks below this one, this one,
  // added in rank order.
  __device__ __forceinline__ void ranks(double part, double& all, double& before, double& mine) const {
    double run = 0.0;
    before = mine = 0.0;
#pragma unroll
    for (int i = 0; i < kMaxC; ++i) {
      const double s = __shfl_sync(0xffffffffu, part, i);
      if (i < C) {
        if (i == rank) {
          before = run;
          mine = s;
        }
        run += s;
      }
    }
    all = run;
  }
  // The sums of row `cur` of p and, if qrow, of q.  before / mine: parts of
  // p's sum (and wsum this rank's units, not with `given` rows).
  __device__ void rows(int cur, const T* prow, const T* qrow, RowSum& P, RowSum& Q, double& before,
                       double& mine) {
    const int lane = threadIdx.x & 31, r = lane & 15;
    RowSum z{0.0, -INFINITY, kNone};
    float own = -INFINITY;         // the maximum that wsum is relative to
    if (given) {
      const long long at = lane < 16 ? (long long)b * (a.n + 1) + cur
                                     : (long long)a.B * (a.n + 1) + (long long)b * a.n + cur;
      if (r < C && (lane < 16 || qrow)) z = given[at * C + r];
    } else {
      if (qrow) {
        const RowSum q = row_part<T, VEC>(qrow, t, a.V, c2, tab, sh, wsum);
        if (threadIdx.x == 0) ex->r[phase][1] = q;
      }
      const RowSum p = row_part<T, VEC>(prow, t, a.V, c2, tab, sh, wsum);
      own = p.m;
      if (threadIdx.x == 0) ex->r[phase][0] = p;
      cl.sync();
      if (r < C && (lane < 16 || qrow)) z = cl.map_shared_rank(&ex->r[phase][0], r)[lane < 16 ? 0 : 1];
      phase ^= 1;
    }
    // every warp brings the ranks' parts to the row's maximum: lanes 0 .. C-1
    // those of p, 16 .. 16+C-1 those of q
    float m = z.m;
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    int i = z.m == m ? z.arg : kNone;
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) i = min(i, __shfl_xor_sync(0xffffffffu, i, o));
    // a part that is all -inf keeps its s: 0, or NaN
    if (z.m != -INFINITY) z.s *= exp2_64(c2 * (wide(z.m) - wide(m)));
    ranks(z.s, P.s, before, mine);
    P.m = __shfl_sync(0xffffffffu, m, 0);
    P.arg = __shfl_sync(0xffffffffu, i, 0);
    Q.m = __shfl_sync(0xffffffffu, m, 16);
    Q.arg = __shfl_sync(0xffffffffu, i, 16);
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) z.s += __shfl_xor_sync(0xffffffffu, z.s, o);
    Q.s = __shfl_sync(0xffffffffu, z.s, 16);
    // the units too, for the draw
    if (own != -INFINITY && own != P.m) {
      const double f = exp2_64(c2 * (wide(own) - wide(P.m)));
      for (int u = threadIdx.x; u < t.units; u += kT) wsum[u] *= f;
    } else if (own == -INFINITY && !given) {
      for (int u = threadIdx.x; u < t.units; u += kT) wsum[u] = 0.0;
    }
    __syncthreads();
  }
  __device__ double sum(const Weights<T>& w, double& before, double& mine) {
    const double s = sum_part<T, VEC>(w, c2, tab, t, a.V, wsum);
    if (threadIdx.x == 0) ex->d[phase] = s;
    cl.sync();
    const int lane = threadIdx.x & 31;
    double all;
    ranks(lane < C ? *cl.map_shared_rank(&ex->d[phase], lane) : 0.0, all, before, mine);
    phase ^= 1;
    return all;
  }
  // By warp 0 of the rank whose part holds the crossing: the first index whose
  // running sum (base: the ranks below) passes goal; if the rounding of the sums
  // leaves none, the last index with weight of the unit it falls in.
  __device__ int find(const Weights<T>& w, double base, double goal) const {
    const int lane = threadIdx.x & 31;
    const int each = (t.units + 31) / 32;
    double s = 0.0;
    for (int u = lane * each; u < min(t.units, (lane + 1) * each); ++u) s += wsum[u];
    double inc = s;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const double y = __shfl_up_sync(0xffffffffu, inc, d);
      if (lane >= d) inc += y;
    }
    // the first lane whose units pass goal, else the last that has any weight
    const unsigned hit = __ballot_sync(0xffffffffu, base + inc > goal && s > 0.0);
    const unsigned some = __ballot_sync(0xffffffffu, s > 0.0);
    const int who = hit ? __ffs(hit) - 1 : 31 - __clz(some);
    double run = base + (inc - s), at = run;
    int unit = -1;
    for (int u = lane * each; u < min(t.units, (lane + 1) * each); ++u) {
      if (wsum[u] > 0.0) {
        unit = u;
        at = run;
        run += wsum[u];
        if (run > goal) break;
      }
    }
    unit = __shfl_sync(0xffffffffu, unit, who);
    run = __shfl_sync(0xffffffffu, at, who);
    int last = -1;
    for (int i = 0; i < t.k; ++i) {
      const int v = t.v0 + (unit * t.k + i) * 256 + lane * 8;
      double o[8] = {0, 0, 0, 0, 0, 0, 0, 0};
      if (v < t.v1) weights8<T, VEC>(w, c2, tab, v, a.V, o);
      const double m = add8(o);
      double in = m;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const double y = __shfl_up_sync(0xffffffffu, in, d);
        if (lane >= d) in += y;
      }
      double x = run + (in - m);
      int found = kNone, mine = -1;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        x += o[e];
        if (o[e] > 0.0) {
          mine = v + e;
          if (x > goal && found == kNone) found = v + e;
        }
      }
      found = __reduce_min_sync(0xffffffffu, found);
      if (found != kNone) return found;
      last = max(last, __reduce_max_sync(0xffffffffu, mine));
      run += __shfl_sync(0xffffffffu, in, 31);
    }
    return last;
  }
};

template <typename T, bool VEC>
__global__ void __launch_bounds__(kT, 2) walk_kernel(screen_verify_args a, const RowSum* given) {
  __shared__ Exchange ex;
  __shared__ RowSum sh[kT / 32];
  __shared__ double wsum[kUnits], tab[kTab];
  __shared__ unsigned long long children[kMaxN + 1];
  __shared__ long long tok[kMaxN];
  __shared__ float lp[kMaxN], lq[kMaxN], un[kMaxN];
  __shared__ int gone[kMaxN];
  __shared__ int path[kMaxN];
  const int tid = threadIdx.x;
  cg::cluster_group cl = cg::this_cluster();
  const int C = (int)cl.num_blocks(), rank = (int)cl.block_rank();
  const int n = a.n, V = a.V, b = blockIdx.x / C;
  for (int i = tid; i <= kMaxN; i += kT) children[i] = 0ull;
  fill_table(tab);
  __syncthreads();
  pdl_wait();
  pdl_trigger();
  const bool drawn = a.draft_logits != nullptr;
  const float temp = temp_of(a, b);
  const bool greedy = !(temp > 0.f);
  const T* logits = reinterpret_cast<const T*>(a.logits) + (long long)b * a.l_sb;
  const T* drafts = reinterpret_cast<const T*>(a.draft_logits) + (long long)b * a.d_sb;
  Walker<T, VEC> w{a, given, cl, &ex, sh, wsum, tab, 0, rank, C, b, part_of(V, rank, C), scale_of(temp)};
  if (tid < n) {
    const int i = tid;
    const int p = a.parents ? a.parents[(long long)b * a.p_sb + i] : i - 1;
    const long long x = a.tokens[(long long)b * a.t_sb + i];
    tok[i] = x;
    un[i] = a.uniforms[(long long)b * a.u_sb + i];
    if (p >= -1 && p < i && x >= 0 && x < V) {
      lp[i] = to_f(logits[(p + 1) * a.l_st + x]);
      lq[i] = drawn ? to_f(drafts[(p + 1) * a.d_st + x]) : 0.f;
      atomicOr(&children[p + 1], 1ull << i);
    }
  }
  __syncthreads();

  int cur = 0, count = 0;
  long long token = -1;
  while (true) {
    // --- a new row ------------------------------------------------------------
    unsigned long long left = children[cur];
    const T* prow = logits + cur * a.l_st;
    const T* qrow = drawn && left ? drafts + cur * a.d_st : nullptr;
    RowSum P, Q;
    double before, mine;                          // parts of the last residual's sum
    w.rows(cur, prow, qrow, P, Q, before, mine);
    if (!usable(P) || !(temp >= 0.f)) break;      // no distribution: no token
    if (qrow && !usable(Q)) left = 0;             // nothing was drawn from this
    const double mp = wide(P.m), mq = wide(Q.m);
    double c = 0.0, z = 1.0, all = P.s, out_mass = 0.0;
    int n_gone = 0, next = -1;
    bool stale = given != nullptr;                // all and wsum are not the residual's
    while (left) {
      const int i = __ffsll((long long)left) - 1;
      left &= left - 1;
      const int x = (int)tok[i];
      bool dup = false;
      for (int k = 0; k < n_gone; ++k) dup = dup || gone[k] == x;
      double px, qx;
      if (greedy) {
        px = x == P.arg ? 1.0 : 0.0;
        qx = !drawn || x == Q.arg ? 1.0 : 0.0;
      } else {
        px = exp2_64(w.c2 * (wide(lp[i]) - mp)) / P.s;
        qx = drawn ? exp2_64(w.c2 * (wide(lq[i]) - mq)) / Q.s : 1.0;
      }
      if (dup) px = 0.0;
      const double rest = px - c * qx;
      if (rest > 0.0 && (double)un[i] * qx * z < rest) {
        next = i;
        break;
      }
      // rejected
      if (drawn) {
        c += z;
        if (greedy) {                             // p and q are one point each
          z = fmax(P.arg == Q.arg ? 1.0 - c : 1.0, 0.0);
        } else {
          z = all = w.sum({prow, qrow, mp, mq, 1.0 / P.s, c / Q.s, 0, gone}, before, mine);
          stale = false;
        }
      } else if (!dup) {
        __syncthreads();
        if (tid == 0) gone[n_gone] = x;
        __syncthreads();
        ++n_gone;
        stale = true;
        if (greedy) {
          if (x == P.arg) z = 0.0;
        } else {
          out_mass += px;
          z = 1.0 - out_mass;
          if (z < 1e-6) {                         // too little left for a difference
            all = w.sum({prow, nullptr, mp, 0.0, 0.0, 0.0, n_gone, gone}, before, mine);
            z = all / P.s;
            stale = false;
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
      token = P.arg;                              // rejected nodes were not it
      break;
    }
    const double u = a.uniforms[(long long)b * a.u_sb + n];
    Weights<T> wt{prow, nullptr, mp, mq, 0.0, 0.0, n_gone, gone};
    if (c > 0.0) {
      wt.q = qrow;
      wt.ip = 1.0 / P.s;
      wt.iq = c / Q.s;
    }
    if (stale) all = w.sum(wt, before, mine);
    if (!(all > 0.0)) {                           // nothing left: p itself
      wt.q = nullptr;
      wt.n_gone = 0;
      all = w.sum(wt, before, mine);
    }
    // u outside [0, 1) counts as the nearest end
    const double goal = fmin(fmax(u, 0.0), 1.0 - 0x1p-53) * all;
    const bool here = before <= goal && before + mine > goal;   // one rank
    if (here && tid < 32) {
      const int x = w.find(wt, before, goal);
      if (tid < C) *cl.map_shared_rank(&ex.token, tid) = x;
    }
    cl.sync();
    token = ex.token;
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

// CTAs per sequence: enough to fill two per SM, 8 at most (a portable cluster).
int cluster_of(const screen_verify_args& a) {
  int C = kMaxC;
  while (C > 1 && (long long)a.B * C > 2 * 148) C >>= 1;
  return C;
}
// All rows up front while that is a few microseconds of the whole GPU.
bool all_rows(const screen_verify_args& a) {
  const long long rows = (long long)a.B * (a.n + 1) + (a.draft_logits ? (long long)a.B * a.n : 0);
  return rows * a.V <= (4ll << 20) && rows <= 65535;
}

template <typename T, bool VEC>
void launch_verify(const screen_verify_args& a, cudaStream_t s) {
  const int C = cluster_of(a);
  RowSum* given = nullptr;
  if (all_rows(a)) {
    given = reinterpret_cast<RowSum*>(a.workspace);
    const int rows = a.B * (a.n + 1) + (a.draft_logits ? a.B * a.n : 0);
    launch_pdl(rows_kernel<T, VEC>, dim3(C, rows), dim3(kT), 0, s, a, given);
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(a.B * C);
  cfg.blockDim = dim3(kT);
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = C;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  cudaLaunchKernelEx(&cfg, walk_kernel<T, VEC>, a, (const RowSum*)given);
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
  const size_t rows = (size_t)a.B * (a.n + 1) + (a.draft_logits ? (size_t)a.B * a.n : 0);
  return all_rows(a) ? rows * cluster_of(a) * sizeof(RowSum) : 0;
}
void verify(const screen_verify_args& a, cudaStream_t s) {
  if (a.dtype == SCREEN_F32) verify_t<float>(a, s);
  else verify_t<__nv_bfloat16>(a, s);
}

}  // namespace screen
