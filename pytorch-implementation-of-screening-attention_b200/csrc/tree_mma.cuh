// The warp-MMA form of the tree attention: bf16 pages with bf16 activations,
// or int8 pages with bf16 / fp32 activations.
#pragma once
#include <cuda_fp16.h>
#include "tree_decode.cuh"

namespace screen {
namespace tree {

__device__ __forceinline__ void mma_f16(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
      "{%8,%9}, {%0,%1,%2,%3};\n"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
// two signed bytes, already placed as (b, 0x64, b', 0x64) with their top bit
// flipped: 1024 + 128 + value in fp16 each, so minus 1152 is exact
__device__ __forceinline__ uint32_t f16_of_biased(uint32_t u) {
  const uint32_t bias = 0x64806480u;  // 1152, 1152
  const __half2 v = __hsub2(*reinterpret_cast<const __half2*>(&u),
                            *reinterpret_cast<const __half2*>(&bias));
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src, bool pred) {
  const int n = pred ? 4 : 0;
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;\n" ::"r"(dst), "l"(src), "r"(n));
}

template <typename E_, typename TA_, int D_, int QW_, int MG_>
struct Cfg {
  using E = E_;
  using TA = TA_;
  static constexpr int D = D_;
  static constexpr int QW = QW_;                 // 16-query tiles per warp
  static constexpr int MG = MG_;                 // warps side by side over the queries
  static constexpr int WK = 4 / MG_;             // warps side by side over the keys
  static constexpr bool I8 = sizeof(E_) == 1;
  static constexpr bool HL = I8 && sizeof(TA_) == 4;  // q and alpha as hi + lo halves
  static constexpr int RB = D_ * (int)sizeof(E_);     // row bytes
  static constexpr int CH = RB / 16;                  // 16-byte chunks per row
  static constexpr int KS = D_ / 16;                  // MMA k steps of S
  static constexpr int NT = D_ / 8;                   // 8-column tiles of O
  static constexpr int TILE_B = kTile * RB;
  // about 48 KB of copies in flight per CTA
  static constexpr int S = RB >= 256 ? 3 : RB >= 128 ? 4 : 6;
  static constexpr int MS = 8;                        // meta ring, >= S + 1
  static constexpr int STAGE_B = 2 * TILE_B + (I8 ? 2 * kTile * 4 : 0);
  static constexpr int RED_B = 4 * QW_ * 16 * D_ * 4; // the warps' sums at the end
  static constexpr int SMEM = S * STAGE_B > RED_B ? S * STAGE_B : RED_B;
};

// What the compute warps need to know about each key of a tile.
struct Meta {
  long long row[kTile];        // row index in the pages, -1 none
  float2 cs[kTile];            // cos, sin of pi c / w
  int c[kTile];                // position - lens, a node's depth, or kNoKey
  int edge[2];                 // some key of this half needs a per-score test
};

// Byte offset of 16-byte chunk c of key row r inside a tile.  The XOR makes the
// fragment loads below hit distinct banks (rows of 64 or 128 bytes alias).
template <class C>
__device__ __forceinline__ uint32_t k_off(int r, int c) {
  int x = c;
  if constexpr (C::CH >= 8) x = c ^ ((r & 1) << 2);
  return (uint32_t)(r * C::RB + (x << 4));
}
template <class C>
__device__ __forceinline__ uint32_t v_off(int r, int c) {
  int x = c;
  if constexpr (C::I8) {
    if constexpr (C::CH == 8) x = c ^ (r & 6);
    else if constexpr (C::CH == 4) x = c ^ ((r & 4) >> 1);
  } else {
    if constexpr (C::CH >= 8) x = c ^ (r & 7);
    else if constexpr (C::CH == 4) x = c ^ ((r >> 1) & 3);
    else x = c ^ ((r >> 2) & 1);
  }
  return (uint32_t)(r * C::RB + (x << 4));
}
// Key of column c of an 8-key score tile.  int8: neighbouring columns (a
// thread's pair) are taken so that the four pairs a load touches start on
// different banks for both K (even / odd rows) and V.
template <class C>
__device__ __forceinline__ int key_of(int c) {
  return C::I8 ? c ^ ((c >> 1) & 1) : c;
}

// B operand of S for 8 keys: row r of K, all k steps.  Thread t = lane % 4 holds
// chunk t (+ 4 h) of the row; k step s takes 4 consecutive elements of it, and
// the query fragments use the same order of d.
template <class C>
__device__ __forceinline__ int d_of(int t, int s) {  // first of the 4 elements
  if constexpr (C::I8) {
    if constexpr (C::D == 128) return 64 * (s >> 2) + 16 * t + 4 * (s & 3);
    else if constexpr (C::D == 64) return 16 * t + 4 * s;
    else if constexpr (C::D == 32) return 8 * t + 4 * s;
    else return 4 * t;
  } else {
    if constexpr (C::D >= 32) return 32 * (s >> 1) + 8 * t + 4 * (s & 1);
    else return 4 * t;
  }
}
template <class C>
__device__ __forceinline__ void load_k(const unsigned char* kt, int r, int t,
                                       uint32_t (&kb)[C::KS][2]) {
  if constexpr (C::I8) {
    constexpr int W = C::KS;              // words: 4 bytes per k step
    uint32_t w[W];
    if constexpr (C::D >= 64) {
#pragma unroll
      for (int hh = 0; hh < C::D / 64; ++hh)
        *reinterpret_cast<uint4*>(&w[4 * hh]) =
            *reinterpret_cast<const uint4*>(kt + k_off<C>(r, t + 4 * hh));
    } else if constexpr (C::D == 32) {
      *reinterpret_cast<uint2*>(&w[0]) =
          *reinterpret_cast<const uint2*>(kt + r * C::RB + 8 * t);
    } else {
      w[0] = *reinterpret_cast<const uint32_t*>(kt + r * C::RB + 4 * t);
    }
#pragma unroll
    for (int s = 0; s < W; ++s) {
      const uint32_t u = w[s] ^ 0x80808080u;
      kb[s][0] = f16_of_biased(__byte_perm(u, 0x64646464u, 0x4140));
      kb[s][1] = f16_of_biased(__byte_perm(u, 0x64646464u, 0x4342));
    }
  } else if constexpr (C::D >= 32) {
#pragma unroll
    for (int hh = 0; hh < C::D / 32; ++hh) {
      const uint4 u = *reinterpret_cast<const uint4*>(kt + k_off<C>(r, t + 4 * hh));
      kb[2 * hh][0] = u.x; kb[2 * hh][1] = u.y;
      kb[2 * hh + 1][0] = u.z; kb[2 * hh + 1][1] = u.w;
    }
  } else {
    const uint2 u = *reinterpret_cast<const uint2*>(kt + r * C::RB + 8 * t);
    kb[0][0] = u.x; kb[0][1] = u.y;
  }
}

// Column of O that register pair (nt, e) of thread t holds: C fragments have
// n = 2 t + e; for int8 pages column n of tile nt stands for d = NT n + nt, so
// that a thread's NT columns are consecutive bytes of a V row.
template <class C>
__device__ __forceinline__ int o_col(int nt, int n) {
  return C::I8 ? C::NT * n + nt : 8 * nt + n;
}

// B operand of alpha V for 16 keys, rows base .. base + 15 of the V tile.
template <class C>
__device__ __forceinline__ void load_v(const unsigned char* vt, int base, int lane,
                                       uint32_t (&vb)[C::NT][2]) {
  const int g = lane >> 2, t = lane & 3;
  if constexpr (C::I8) {
#pragma unroll
    for (int hh = 0; hh < 2; ++hh) {      // keys 0-7 / 8-15 of the group
      const int r0 = base + 8 * hh + key_of<C>(2 * t), r1 = base + 8 * hh + key_of<C>(2 * t + 1);
      constexpr int W = C::NT >= 4 ? C::NT / 4 : 1;
      uint32_t x[W], y[W];
      if constexpr (C::D == 128) {
        *reinterpret_cast<uint4*>(&x[0]) = *reinterpret_cast<const uint4*>(vt + v_off<C>(r0, g));
        *reinterpret_cast<uint4*>(&y[0]) = *reinterpret_cast<const uint4*>(vt + v_off<C>(r1, g));
      } else if constexpr (C::D == 64) {
        *reinterpret_cast<uint2*>(&x[0]) =
            *reinterpret_cast<const uint2*>(vt + v_off<C>(r0, g >> 1) + 8 * (g & 1));
        *reinterpret_cast<uint2*>(&y[0]) =
            *reinterpret_cast<const uint2*>(vt + v_off<C>(r1, g >> 1) + 8 * (g & 1));
      } else if constexpr (C::D == 32) {
        x[0] = *reinterpret_cast<const uint32_t*>(vt + r0 * C::RB + 4 * g);
        y[0] = *reinterpret_cast<const uint32_t*>(vt + r1 * C::RB + 4 * g);
      } else {
        x[0] = *reinterpret_cast<const unsigned short*>(vt + r0 * C::RB + 2 * g);
        y[0] = *reinterpret_cast<const unsigned short*>(vt + r1 * C::RB + 2 * g);
      }
#pragma unroll
      for (int q = 0; q < W; ++q) {
        const uint32_t lo = __byte_perm(x[q], y[q], 0x5140) ^ 0x80808080u;  // x0 y0 x1 y1
        vb[4 * q + 0][hh] = f16_of_biased(__byte_perm(lo, 0x64646464u, 0x4140));
        vb[4 * q + 1][hh] = f16_of_biased(__byte_perm(lo, 0x64646464u, 0x4342));
        if constexpr (C::NT >= 4) {
          const uint32_t hi = __byte_perm(x[q], y[q], 0x7362) ^ 0x80808080u;
          vb[4 * q + 2][hh] = f16_of_biased(__byte_perm(hi, 0x64646464u, 0x4140));
          vb[4 * q + 3][hh] = f16_of_biased(__byte_perm(hi, 0x64646464u, 0x4342));
        }
      }
    }
  } else {
    // ldmatrix.trans: lanes 0-7 / 8-15 address keys 0-7 / 8-15 of chunk c, lanes
    // 16-31 those of chunk c + 1
    const int r = base + (lane & 15);
    const uint32_t at = smem_u32(vt);
#pragma unroll
    for (int c = 0; c < C::NT; c += 2)
      ldsm_x4_t(at + v_off<C>(r, c + (lane >> 4)), vb[c][0], vb[c][1], vb[c + 1][0], vb[c + 1][1]);
  }
}

template <class C>
__global__ void __launch_bounds__(kThreads) tree_mma_kernel(TreeParams p, float* __restrict__ part) {
  using E = typename C::E;
  using TA = typename C::TA;
  constexpr int D = C::D, QW = C::QW, S = C::S;
  extern __shared__ __align__(128) unsigned char dsm[];
  __shared__ Nodes nodes;
  __shared__ Meta meta[C::MS];
  pdl_wait();
  pdl_trigger();
  const screen_tree_args& a = p.a;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  const int bh = blockIdx.y, b = bh / a.H, h = bh % a.H, split = blockIdx.x;
  const Range rg = tree_range(p, b, h);
  const int c0 = rg.t0 + split * rg.per;
  int c1 = c0 + rg.per - 1;
  if (c1 > rg.t0 + rg.nt - 1) c1 = rg.t0 + rg.nt - 1;
  if (split >= (rg.used > 0 ? rg.used : 1)) return;   // uniform over the CTA
  const float w = a.w[h], r = a.r[h];
  const long long lens = rg.lens;

  if (warp == 0) tree_nodes(a, b, nodes, lane);
  __syncthreads();
  if (rg.nt > 0 && a.k) append_rows<E, TA, D>(a, nodes, b, h, lens, c0, c1);

  // --- per-key facts of a tile, two steps: addresses early, store late -------
  struct Key { long long row; int c; };
  const int krow = tid & (kTile - 1);
  auto key_early = [&](int tile) -> Key {
    Key k{-1, kNoKey};
    const long long pos = (long long)tile * kTile + krow;
    if (tile <= c1 && pos >= rg.first && pos < lens + a.n) {
      const long long slot = pos - lens;
      if (slot < 0) k.c = (int)slot;
      else if (nodes.line[slot]) k.c = nodes.depth[slot];
      if (k.c != kNoKey) k.row = paged_row(a.cache, b, a.H, h, pos);
      if (k.row < 0) k.c = kNoKey;
    }
    return k;
  };
  auto key_late = [&](int tile, const Key& k) {
    Meta& m = meta[tile & (C::MS - 1)];
    float sn = 0.f, cn = 0.f;
    if (k.c != kNoKey) sincospif((float)k.c / w, &sn, &cn);
    m.row[krow] = k.row;
    m.cs[krow] = make_float2(cn, sn);
    m.c[krow] = k.c;
    // a score needs its own window / ancestor test next to the window's old
    // end, in the nodes' own slots, and where a key is missing
    const long long pos = (long long)tile * kTile + krow;
    const bool e = k.c == kNoKey || pos >= lens || pos < lens - rg.dmax + kMaxN;
    const unsigned any = __ballot_sync(0xffffffffu, e);
    if (lane == 0) m.edge[warp & 1] = any != 0;
  };
  const uint32_t sm0 = smem_u32(dsm);
  auto load_tile = [&](int tile) {
    if (tile <= c1) {
      const Meta& m = meta[tile & (C::MS - 1)];
      const uint32_t st = sm0 + (uint32_t)((tile - c0) % S) * C::STAGE_B;
      const char* kp = reinterpret_cast<const char*>(a.cache.k_pages);
      const char* vp = reinterpret_cast<const char*>(a.cache.v_pages);
#pragma unroll
      for (int i = 0; i < (kTile * C::CH + kThreads - 1) / kThreads; ++i) {
        const int u = i * kThreads + tid;
        if (kTile * C::CH % kThreads == 0 || u < kTile * C::CH) {
          const int row = u / C::CH, c = u % C::CH;
          const long long at = m.row[row];
          const long long off = (at < 0 ? 0 : at) * C::RB + c * 16;
          cp_async16(st + k_off<C>(row, c), kp + off, at >= 0);
          cp_async16(st + C::TILE_B + v_off<C>(row, c), vp + off, at >= 0);
        }
      }
      if constexpr (C::I8) {
        const int row = tid & (kTile - 1);
        const long long at = m.row[row];
        const float* sc = tid < kTile ? a.k_scales : a.v_scales;
        cp_async4(st + 2 * C::TILE_B + tid * 4, sc + (at < 0 ? 0 : at), at >= 0);
      }
    }
    cp_async_commit();
  };

  // --- queries: fragments, per-row factors ------------------------------------
  const int mg = warp % C::MG, wk = warp / C::MG;
  uint32_t qa[QW][C::KS][4];
  uint32_t ql[C::HL ? QW : 1][C::HL ? C::KS : 1][4];
  float rq[QW][2], ci[QW][2], si[QW][2];
  int dep[QW][2], node[QW][2];
#pragma unroll
  for (int m = 0; m < QW; ++m)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int i = (mg * QW + m) * 16 + g + 8 * e;
      const bool in = i < a.n && rg.nt > 0;
      node[m][e] = in ? i : 0;
      float x[C::KS][4];
      float ss = 0.f;
      uint32_t top = 0;
#pragma unroll
      for (int s = 0; s < C::KS; ++s) {
#pragma unroll
        for (int f = 0; f < 4; ++f) x[s][f] = 0.f;
        if (in)
          load4(reinterpret_cast<const TA*>(a.q) + (long long)b * a.q_sb + (long long)i * a.q_st +
                    (long long)h * D + d_of<C>(t, s), x[s]);
#pragma unroll
        for (int f = 0; f < 4; ++f) {
          ss = fmaf(x[s][f], x[s][f], ss);
          top = max(top, __float_as_uint(x[s][f]) & 0x7fffffffu);
        }
      }
      ss += __shfl_xor_sync(0xffffffffu, ss, 1);
      ss += __shfl_xor_sync(0xffffffffu, ss, 2);
      float scale = 1.f;
      if constexpr (C::I8) {
        // bring the row's largest element into [1, 2): the bf16 row is then
        // exact in fp16 (elements under 2^-16 of the largest round at 2^-25 of
        // it), an fp32 row is held as hi + lo halves to 2^-25
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
        int ex = (int)(top >> 23);
        ex = ex < 1 ? 1 : ex > 253 ? 253 : ex;
        const float down = __uint_as_float((uint32_t)(254 - ex) << 23);
        scale = __uint_as_float((uint32_t)ex << 23);
#pragma unroll
        for (int s = 0; s < C::KS; ++s)
#pragma unroll
          for (int f = 0; f < 4; ++f) x[s][f] *= down;
      }
#pragma unroll
      for (int s = 0; s < C::KS; ++s) {
        if constexpr (C::I8) {
          qa[m][s][e] = pack_f16(x[s][0], x[s][1]);
          qa[m][s][2 + e] = pack_f16(x[s][2], x[s][3]);
          if constexpr (C::HL) {
            const float2 u = __half22float2(*reinterpret_cast<__half2*>(&qa[m][s][e]));
            const float2 v = __half22float2(*reinterpret_cast<__half2*>(&qa[m][s][2 + e]));
            ql[m][s][e] = pack_f16(x[s][0] - u.x, x[s][1] - u.y);
            ql[m][s][2 + e] = pack_f16(x[s][2] - v.x, x[s][3] - v.y);
          }
        } else {
          qa[m][s][e] = pack_bf16(x[s][0], x[s][1]);
          qa[m][s][2 + e] = pack_bf16(x[s][2], x[s][3]);
        }
      }
      // S = q.k scale / max(|q|, eps), times r; scale first: 2^ex / |q| <= 1
      rq[m][e] = r * (scale / fmaxf(sqrtf(ss), a.eps));
      const bool live = in && nodes.line[i] != 0;
      dep[m][e] = live ? nodes.depth[i] : 0;
      float sn, cn;
      sincospif((float)dep[m][e] / w, &sn, &cn);
      ci[m][e] = 0.5f * cn;
      si[m][e] = 0.5f * sn;
      if (!live) rq[m][e] = __uint_as_float(0x7fc00000u);  // t = NaN: sees nothing
    }
  const float one_r = 1.0f - r;

  float o[QW][C::NT][4];
  // pass 0 takes every V row as finite.  A row with an infinity or NaN (a
  // non-finite raw row) times alpha = 0 would spoil queries that do not see
  // it: if any sum comes out non-finite, pass 1 repeats the run with such rows
  // left out of the product and put back as NaN for the queries that see them.
  for (int pass = 0; pass < (C::I8 ? 1 : 2); ++pass) {
#pragma unroll
    for (int m = 0; m < QW; ++m)
#pragma unroll
      for (int j = 0; j < C::NT; ++j)
#pragma unroll
        for (int f = 0; f < 4; ++f) o[m][j][f] = 0.f;
    if (rg.nt > 0) {
      // the first S tiles: threads 0-63 take the even ones, 64-127 the odd ones,
      // all table lookups in flight before the first use
      Key k[(S + 1) / 2];
#pragma unroll
      for (int x = 0; x < (S + 1) / 2; ++x) k[x] = key_early(c0 + 2 * x + tid / kTile);
#pragma unroll
      for (int x = 0; x < (S + 1) / 2; ++x)
        if (2 * x + tid / kTile < S) key_late(c0 + 2 * x + tid / kTile, k[x]);
      __syncthreads();
#pragma unroll
      for (int x = 0; x < S - 1; ++x) load_tile(c0 + x);
      for (int tile = c0; tile <= c1; ++tile) {
        cp_async_wait<S - 2>();
        __syncthreads();
        load_tile(tile + S - 1);
        Key next;
        if (tid < kTile) next = key_early(tile + S);
        const Meta& m0 = meta[tile & (C::MS - 1)];
        const unsigned char* kt = dsm + (size_t)((tile - c0) % S) * C::STAGE_B;
        const unsigned char* vt = kt + C::TILE_B;
        const float* ks = reinterpret_cast<const float*>(kt + 2 * C::TILE_B);
        const float* vs = ks + kTile;
        const bool edge = (m0.edge[0] | m0.edge[1]) != 0;
        const long long slot0 = (long long)tile * kTile - lens;   // slot of the tile's first key
#pragma unroll 1
        for (int kg = wk; kg < kTile / 16; kg += C::WK) {
          float s[QW][2][4];
          float tmax = 0.f;
          int key[2][2];
#pragma unroll
          for (int nt = 0; nt < 2; ++nt) {
            const int base = kg * 16 + nt * 8;
            uint32_t kb[C::KS][2];
            load_k<C>(kt, base + key_of<C>(g), t, kb);
#pragma unroll
            for (int m = 0; m < QW; ++m) {
#pragma unroll
              for (int f = 0; f < 4; ++f) s[m][nt][f] = 0.f;
#pragma unroll
              for (int x = 0; x < C::KS; ++x) {
                if constexpr (C::I8) {
                  mma_f16(s[m][nt], qa[m][x], kb[x][0], kb[x][1]);
                  if constexpr (C::HL) mma_f16(s[m][nt], ql[m][x], kb[x][0], kb[x][1]);
                } else {
                  mma_bf16(s[m][nt], qa[m][x], kb[x][0], kb[x][1]);
                }
              }
            }
#pragma unroll
            for (int f = 0; f < 2; ++f) {
              key[nt][f] = base + key_of<C>(2 * t + f);
              const float sc = C::I8 ? ks[key[nt][f]] : 1.f;
#pragma unroll
              for (int m = 0; m < QW; ++m)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                  float& x = s[m][nt][2 * e + f];
                  // NaN (an unseen row, a non-finite key) counts as 0
                  x = fmaxf(fmaf(C::I8 ? x * sc : x, rq[m][e], one_r), 0.f);
                }
            }
          }
          if (edge) {
#pragma unroll
            for (int nt = 0; nt < 2; ++nt)
#pragma unroll
              for (int f = 0; f < 2; ++f) {
                const int c = m0.c[key[nt][f]];
                const long long slot = slot0 + key[nt][f];
#pragma unroll
                for (int m = 0; m < QW; ++m)
#pragma unroll
                  for (int e = 0; e < 2; ++e) {
                    bool see = dep[m][e] - c <= rg.dmax;
                    if (slot >= 0 && slot < a.n) see = see && (nodes.line[node[m][e]] >> slot & 1);
                    if (!see) s[m][nt][2 * e + f] = 0.f;
                  }
              }
          }
#pragma unroll
          for (int m = 0; m < QW; ++m)
#pragma unroll
            for (int nt = 0; nt < 2; ++nt)
#pragma unroll
              for (int f = 0; f < 4; ++f) tmax = fmaxf(tmax, s[m][nt][f]);
          if (!__any_sync(0xffffffffu, tmax > 0.f)) continue;
          uint32_t vb[C::NT][2];
          load_v<C>(vt, kg * 16, lane, vb);
          uint32_t bad = 0;
          if constexpr (!C::I8) {
            if (pass == 1) {
              // which of the 16 rows hold a non-finite element (lane: one row)
              bool nf = false;
              for (int c = 0; c < C::CH; ++c) {
                const uint4 u =
                    *reinterpret_cast<const uint4*>(vt + v_off<C>(kg * 16 + (lane & 15), c));
                const uint32_t ww[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
                for (int q = 0; q < 4; ++q)
                  nf = nf || (ww[q] & 0x7f80u) == 0x7f80u || (ww[q] & 0x7f800000u) == 0x7f800000u;
              }
              bad = __ballot_sync(0xffffffffu, nf) & 0xffffu;
#pragma unroll
              for (int j = 0; j < C::NT; ++j)
#pragma unroll
                for (int hh = 0; hh < 2; ++hh) {
                  if (bad >> (8 * hh + 2 * t) & 1) vb[j][hh] &= 0xffff0000u;
                  if (bad >> (8 * hh + 2 * t + 1) & 1) vb[j][hh] &= 0x0000ffffu;
                }
            }
          }
#pragma unroll
          for (int m = 0; m < QW; ++m) {
            uint32_t pa[4], pl[4];
#pragma unroll
            for (int nt = 0; nt < 2; ++nt) {
              float al[4];
#pragma unroll
              for (int f = 0; f < 2; ++f) {
                const float2 cs = m0.cs[key[nt][f]];
                // int8: the row's scale rides on alpha; alpha scale <= 1 / 127,
                // 2^20 keeps it normal in fp16 down to alpha = 2^-23
                const float sv = C::I8 ? vs[key[nt][f]] * 0x1p20f : 1.f;
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                  const float x = s[m][nt][2 * e + f];
                  const float mk = fmaf(cs.x, ci[m][e], fmaf(cs.y, si[m][e], 0.5f));
                  float v = x * x * mk;
                  if constexpr (C::I8) v = x > 0.f ? v * sv : 0.f;  // NaN scales stay out of 0
                  al[2 * e + f] = v;
                }
              }
              if constexpr (C::I8) {
                pa[2 * nt] = pack_f16(al[0], al[1]);
                pa[2 * nt + 1] = pack_f16(al[2], al[3]);
                if constexpr (C::HL) {
                  const float2 u = __half22float2(*reinterpret_cast<__half2*>(&pa[2 * nt]));
                  const float2 v = __half22float2(*reinterpret_cast<__half2*>(&pa[2 * nt + 1]));
                  pl[2 * nt] = pack_f16(al[0] - u.x, al[1] - u.y);
                  pl[2 * nt + 1] = pack_f16(al[2] - v.x, al[3] - v.y);
                }
              } else {
                // alpha to bf16 (half a step, 2^-8): the output rounds as much
                pa[2 * nt] = pack_bf16(al[0], al[1]);
                pa[2 * nt + 1] = pack_bf16(al[2], al[3]);
                if (bad) {
                  // a seen non-finite row makes the query's whole output NaN
                  const uint32_t two = bad >> (8 * nt + 2 * t);
#pragma unroll
                  for (int e = 0; e < 2; ++e)
                    if (((two & 1) && s[m][nt][2 * e] > 0.f) ||
                        ((two & 2) && s[m][nt][2 * e + 1] > 0.f))
                      o[m][0][2 * e] = __uint_as_float(0x7fc00000u);
                }
              }
            }
#pragma unroll
            for (int j = 0; j < C::NT; ++j) {
              if constexpr (C::I8) {
                mma_f16(o[m][j], pa, vb[j][0], vb[j][1]);
                if constexpr (C::HL) mma_f16(o[m][j], pl, vb[j][0], vb[j][1]);
              } else {
                mma_bf16(o[m][j], pa, vb[j][0], vb[j][1]);
              }
            }
          }
        }
        if (tid < kTile) key_late(tile + S, next);
      }
      cp_async_wait<0>();
    }
    if constexpr (!C::I8) {
      bool nf = false;
#pragma unroll
      for (int m = 0; m < QW; ++m)
#pragma unroll
        for (int j = 0; j < C::NT; ++j)
#pragma unroll
          for (int f = 0; f < 4; ++f) nf = nf || !(fabsf(o[m][j][f]) < 3.0e38f);
      if (!__syncthreads_or(nf)) break;
    }
  }
  __syncthreads();   // the stages become the reduction buffer

  // --- sum the key warps, finish or hand the partial on -----------------------
  float* red = reinterpret_cast<float*>(dsm);          // [WK][MG * QW * 16][D]
  constexpr int ROWS = C::MG * QW * 16;
#pragma unroll
  for (int m = 0; m < QW; ++m)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float* dst = red + ((size_t)wk * ROWS + (mg * QW + m) * 16 + g + 8 * e) * D;
#pragma unroll
      for (int j = 0; j < C::NT; ++j)
#pragma unroll
        for (int f = 0; f < 2; ++f)
          dst[o_col<C>(j, 2 * t + f)] = C::I8 ? o[m][j][2 * e + f] * 0x1p-20f : o[m][j][2 * e + f];
    }
  __syncthreads();
  constexpr int PER = D < 32 ? 1 : D / 32;
  for (int i = warp; i < a.n; i += 4) {
    float x[PER];
#pragma unroll
    for (int e = 0; e < PER; ++e) {
      x[e] = 0.f;
      if (lane + 32 * e < D)
#pragma unroll
        for (int k = 0; k < C::WK; ++k) x[e] += red[((size_t)k * ROWS + i) * D + lane + 32 * e];
    }
    if (a.num_splits > 1) {
      float* dst = part + (((size_t)bh * a.num_splits + split) * a.n + i) * D;
#pragma unroll
      for (int e = 0; e < PER; ++e)
        if (lane + 32 * e < D) dst[lane + 32 * e] = x[e];
    } else {
      store_row<TA, D>(a, b, i, h, lane, x, rg.nt > 0 && nodes.line[i] != 0);
    }
  }
}

template <class C>
void launch_tree(const TreeParams& p, float* part, cudaStream_t s) {
  static_assert(C::MS >= C::S + 1 && (C::MS & (C::MS - 1)) == 0, "meta ring");
  if (ensure_smem_optin((const void*)tree_mma_kernel<C>, C::SMEM) != cudaSuccess) return;
  launch_pdl(tree_mma_kernel<C>, dim3(p.a.num_splits, p.a.B * p.a.H), dim3(kThreads),
             (size_t)C::SMEM, s, p, part);
}
// Query tiles per warp: two where the registers allow it (D <= 64) and there
// are more than 16 queries, so that a K / V fragment feeds two products.
template <typename E, typename TA, int D>
void launch_tree_d(const TreeParams& p, float* part, cudaStream_t s) {
  constexpr int Q2 = D <= 64 ? 2 : 1;
  if (p.a.n <= 16) launch_tree<Cfg<E, TA, D, 1, 1>>(p, part, s);
  else if (p.a.n <= 32) launch_tree<Cfg<E, TA, D, Q2, 2 / Q2>>(p, part, s);
  else launch_tree<Cfg<E, TA, D, Q2, 4 / Q2>>(p, part, s);
}
template <typename E, typename TA>
void launch_tree_e(const TreeParams& p, float* part, cudaStream_t s) {
  switch (p.a.D) {
    case 16: launch_tree_d<E, TA, 16>(p, part, s); break;
    case 32: launch_tree_d<E, TA, 32>(p, part, s); break;
    case 64: launch_tree_d<E, TA, 64>(p, part, s); break;
    case 128: launch_tree_d<E, TA, 128>(p, part, s); break;
  }
}

}  // namespace tree
}  // namespace screen
