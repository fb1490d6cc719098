// The warp-MMA form of the tree attention: bf16 pages with bf16 activations,
// or int8 pages with bf16 / fp32 activations.
#pragma once
#include <cuda_fp16.h>
#include "tree_decode.cuh"

namespace screen {
namespace tree {

// Not volatile: a product depends on its operands only, and the compiler may
// interleave independent chains.
__device__ __forceinline__ void mma_f16(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
      "{%8,%9}, {%0,%1,%2,%3};\n"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_b16(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
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

// Packed pairs of fp32 (two keys of one query row).
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) { return __ffma2_rn(a, b, c); }
__device__ __forceinline__ float2 mul2(float2 a, float2 b) { return __fmul2_rn(a, b); }
__device__ __forceinline__ float2 both(float x) { return make_float2(x, x); }

template <typename E_, typename TA_, int D_, int QW_, int MG_, int RH_>
struct Cfg {
  using E = E_;
  using TA = TA_;
  static constexpr int D = D_;
  static constexpr int QW = QW_;                 // 16-query tiles per warp
  static constexpr int MG = MG_;                 // warps of a group, side by side over the queries
  static constexpr int RH = RH_;                 // query rows per thread and tile: 1 if n <= 8
  static constexpr int WK = 4 / MG_;             // groups side by side over the keys
  static constexpr bool I8 = sizeof(E_) == 1;
  // fp32 activations: q and alpha as hi + lo halves, fp32 sums between products.
  // bf16 pages: alpha as hi + lo (one half would round as much as the output).
  static constexpr bool QHL = I8 && sizeof(TA_) == 4;
  static constexpr bool PHL = QHL || !I8;
  static constexpr int RB = D_ * (int)sizeof(E_);     // row bytes
  static constexpr int CH = RB / 16;                  // 16-byte chunks per row
  static constexpr int KS = D_ / 16;                  // MMA k steps of S
  static constexpr int NT = D_ / 8;                   // 8-column tiles of O
  static constexpr int KT = RB <= 64 ? 32 : 16;       // keys per stage of a group
  static constexpr int TILE_B = KT * RB;
  // per key, in score-column order: cos, sin of pi c / w, K / V scale, c
  static constexpr int META_B = KT * (I8 ? 20 : 12) + 16;
  static constexpr int STAGE_B = 2 * TILE_B + META_B;
  static constexpr int S = 3;
  static constexpr int RING_B = WK * S * STAGE_B;
  static constexpr int RED_B = 4 * QW_ * 16 * D_ * 4; // the warps' sums at the end
  static constexpr int SMEM = RING_B > RED_B ? RING_B : RED_B;
  // CTAs per SM the registers are cut to: what a thread holds of O and q decides
  static constexpr int HELD = QW_ * (D_ / 2 + D_ / 4 * (QHL ? 2 : 1));
    static constexpr int MINB = HELD <= 32 ? 4 : HELD <= 64 ? 3 : 2;
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
    for (int s = 0; s < W; ++s) w[s] ^= 0x80808080u;
#pragma unroll
    for (int s = 0; s < W; ++s) {
      kb[s][0] = __byte_perm(w[s], 0x64646464u, 0x4140);
      kb[s][1] = __byte_perm(w[s], 0x64646464u, 0x4342);
    }
#pragma unroll
    for (int s = 0; s < W; ++s) {
      kb[s][0] = f16_of_biased(kb[s][0]);
      kb[s][1] = f16_of_biased(kb[s][1]);
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
    constexpr int W = C::NT >= 4 ? C::NT / 4 : 1;
    uint32_t x[2][W], y[2][W];            // rows of a thread's key pair, both halves
#pragma unroll
    for (int hh = 0; hh < 2; ++hh) {      // keys 0-7 / 8-15 of the group
      const int r0 = base + 8 * hh + key_of<C>(2 * t), r1 = base + 8 * hh + key_of<C>(2 * t + 1);
      if constexpr (C::D == 128) {
        *reinterpret_cast<uint4*>(&x[hh][0]) = *reinterpret_cast<const uint4*>(vt + v_off<C>(r0, g));
        *reinterpret_cast<uint4*>(&y[hh][0]) = *reinterpret_cast<const uint4*>(vt + v_off<C>(r1, g));
      } else if constexpr (C::D == 64) {
        *reinterpret_cast<uint2*>(&x[hh][0]) =
            *reinterpret_cast<const uint2*>(vt + v_off<C>(r0, g >> 1) + 8 * (g & 1));
        *reinterpret_cast<uint2*>(&y[hh][0]) =
            *reinterpret_cast<const uint2*>(vt + v_off<C>(r1, g >> 1) + 8 * (g & 1));
      } else if constexpr (C::D == 32) {
        x[hh][0] = *reinterpret_cast<const uint32_t*>(vt + r0 * C::RB + 4 * g);
        y[hh][0] = *reinterpret_cast<const uint32_t*>(vt + r1 * C::RB + 4 * g);
      } else {
        x[hh][0] = *reinterpret_cast<const unsigned short*>(vt + r0 * C::RB + 2 * g);
        y[hh][0] = *reinterpret_cast<const unsigned short*>(vt + r1 * C::RB + 2 * g);
      }
    }
#pragma unroll
    for (int hh = 0; hh < 2; ++hh)
#pragma unroll
      for (int q = 0; q < W; ++q) {
        const uint32_t lo = __byte_perm(x[hh][q], y[hh][q], 0x5140);   // x0 y0 x1 y1
        y[hh][q] = __byte_perm(x[hh][q], y[hh][q], 0x7362) ^ 0x80808080u;   // x2 y2 x3 y3
        x[hh][q] = lo ^ 0x80808080u;
      }
#pragma unroll
    for (int hh = 0; hh < 2; ++hh)
#pragma unroll
      for (int q = 0; q < W; ++q) {
        vb[4 * q + 0][hh] = __byte_perm(x[hh][q], 0x64646464u, 0x4140);
        vb[4 * q + 1][hh] = __byte_perm(x[hh][q], 0x64646464u, 0x4342);
        if constexpr (C::NT >= 4) {
          vb[4 * q + 2][hh] = __byte_perm(y[hh][q], 0x64646464u, 0x4140);
          vb[4 * q + 3][hh] = __byte_perm(y[hh][q], 0x64646464u, 0x4342);
        }
      }
#pragma unroll
    for (int hh = 0; hh < 2; ++hh)
#pragma unroll
      for (int j = 0; j < C::NT; ++j) vb[j][hh] = f16_of_biased(vb[j][hh]);
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

// The CTA's four warps form 4 / MG groups; a group streams its own stages of KT
// keys (no barrier across the CTA inside the loop), groups taking the stages of
// a run in turn.
template <class C>
__global__ void __launch_bounds__(kThreads, C::MINB) tree_mma_kernel(TreeParams p,
                                                                     float* __restrict__ ws) {
  using E = typename C::E;
  using TA = typename C::TA;
  constexpr int D = C::D, QW = C::QW, S = C::S, KT = C::KT, RH = C::RH;
  extern __shared__ __align__(128) unsigned char dsm[];
  __shared__ Nodes nodes;
  pdl_wait();
  pdl_trigger();
  const screen_tree_args& a = p.a;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  const int mg = warp % C::MG, wk = warp / C::MG;
  const int gt = mg * 32 + lane;                       // thread of the group
  unsigned char* ring = dsm + (size_t)wk * S * C::STAGE_B;
  SegSlots* slots = reinterpret_cast<SegSlots*>(ws);
  float* part = ws + p.part_off;
  auto group_sync = [&] {
    if constexpr (C::MG == 1) __syncwarp();
    else asm volatile("bar.sync %0, %1;" ::"r"(1 + wk), "n"(32 * C::MG) : "memory");
  };
  // page of a position without a 64-bit division
  const int ps = a.cache.page_size;
  const int ps_shift = (ps & (ps - 1)) == 0 ? 31 - __clz(ps) : -1;

  Share sh;
  if (!share_init(p, sh)) return;
  Range rg;
  int c0, c1, last_b = -1;
  bool whole;
  while (share_next(p, sh, rg, c0, c1, whole, slots)) {
    const int b = sh.seg / a.H, h = sh.seg % a.H;
    const float w = a.w[h], r = a.r[h];
    const long long lens = rg.lens;
    __syncthreads();   // the previous piece is done with the shared arrays
    if (b != last_b) {
      if (warp == 0) tree_nodes(a, b, nodes, lane);
      __syncthreads();
      last_b = b;
    }
    if (rg.any && a.k) append_rows<E, TA, D>(a, nodes, b, h, lens, c0, c1);

    // --- a stage: KT keys, their addresses and facts ---------------------------
    const int s0 = c0 * (kTile / KT), s1 = (c1 + 1) * (kTile / KT) - 1;
    const int* table = a.cache.block_table + (long long)b * a.cache.max_blocks;
    // row of this lane's key of stage x, -1 none
    auto key_row = [&](int x) -> long long {
      const long long pos = (long long)x * KT + lane;
      if (lane >= KT || x > s1 || pos < rg.first || pos >= lens + a.n) return -1;
      if (pos >= lens && !nodes.line[pos - lens]) return -1;
      const unsigned q = (unsigned)pos;                // a table holds < 2^31 positions
      const unsigned blk = ps_shift >= 0 ? q >> ps_shift : q / (unsigned)ps;
      if (blk >= (unsigned)a.cache.max_blocks) return -1;
      const int page = table[blk];
      if (page < 0 || page >= a.cache.num_pages) return -1;
      return ((long long)page * a.H + h) * ps + (q - blk * (unsigned)ps);
    };
    auto load_stage = [&](int x, int slot, long long row) {
      unsigned char* st = ring + (size_t)slot * C::STAGE_B;
      if (x <= s1) {
        const uint32_t sa = smem_u32(st);
        const char* kp = reinterpret_cast<const char*>(a.cache.k_pages);
        const char* vp = reinterpret_cast<const char*>(a.cache.v_pages);
        constexpr int GT = 32 * C::MG;
        const long long row0 = __shfl_sync(0xffffffffu, row, 0);
        const bool run = __all_sync(0xffffffffu, lane >= KT || row == row0 + lane) && row0 >= 0;
        if (run) {                                     // all keys there, one after another
#pragma unroll
          for (int i = 0; i < (KT * C::CH + GT - 1) / GT; ++i) {
            const int u = i * GT + gt;
            if (KT * C::CH % GT == 0 || u < KT * C::CH) {
              const long long off = row0 * C::RB + u * 16;
              cp_async16(sa + k_off<C>(u / C::CH, u % C::CH), kp + off, true);
              cp_async16(sa + C::TILE_B + v_off<C>(u / C::CH, u % C::CH), vp + off, true);
            }
          }
        } else {
#pragma unroll 1
          for (int i = 0; i < (KT * C::CH + GT - 1) / GT; ++i) {
            const int u = i * GT + gt, k = u / C::CH;
            const long long at = __shfl_sync(0xffffffffu, row, k & (KT - 1));
            if (k < KT) {
              const long long off = (at < 0 ? 0 : at) * C::RB + u % C::CH * 16;
              cp_async16(sa + k_off<C>(k, u % C::CH), kp + off, at >= 0);
              cp_async16(sa + C::TILE_B + v_off<C>(k, u % C::CH), vp + off, at >= 0);
            }
          }
        }
        if (mg == 0) {
          // this lane's key, stored at its score column
          const int k = lane & (KT - 1);
          const int col = (k & ~7) | key_of<C>(k & 7); // key_of is its own inverse
          float* cs = reinterpret_cast<float*>(st + 2 * C::TILE_B);
          if constexpr (C::I8) {
            // KT = 16: lanes 16-31 fetch the V scales
            const long long at = KT == 32 ? row : __shfl_sync(0xffffffffu, row, k);
            const long long off = at < 0 ? 0 : at;
            if (KT == 32 || lane < KT)
              cp_async4(smem_u32(cs + 2 * KT + col), a.k_scales + off, at >= 0);
            if (KT == 32 || lane >= KT)
              cp_async4(smem_u32(cs + 3 * KT + col), a.v_scales + off, at >= 0);
          }
          const long long pos = (long long)x * KT + lane;
          int c = kNoKey;
          if (row >= 0) c = pos < lens ? (int)(pos - lens) : nodes.depth[pos - lens];
          // a score needs its own window / ancestor test next to the window's
          // old end, in the nodes' own slots, and where a key is missing
          const bool e = lane < KT && (c == kNoKey || pos >= lens || pos < lens - rg.dmax + kMaxN);
          const unsigned edge = __ballot_sync(0xffffffffu, e);
          if (lane < KT) {
            float sn = 0.f, cn = 0.f;
            if (c != kNoKey) sincospif((float)c / w, &sn, &cn);
            cs[col] = cn;
            cs[KT + col] = sn;
            reinterpret_cast<int*>(cs)[(C::I8 ? 4 : 2) * KT + col] = c;
          }
          if (lane == 0) reinterpret_cast<int*>(cs)[(C::I8 ? 5 : 3) * KT] = edge != 0;
        }
      }
      cp_async_commit();
    };

    // --- queries: fragments, per-row factors ------------------------------------
    uint32_t qa[QW][C::KS][4];
    uint32_t ql[C::QHL ? QW : 1][C::QHL ? C::KS : 1][4];
    float rq[QW][RH], ci[QW][RH], si[QW][RH];
    int dep[QW][RH];
#pragma unroll
    for (int m = 0; m < QW; ++m)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        if (e >= RH) {
#pragma unroll
          for (int s = 0; s < C::KS; ++s) {
            qa[m][s][1] = qa[m][s][3] = 0u;
            if constexpr (C::QHL) ql[m][s][1] = ql[m][s][3] = 0u;
          }
          continue;
        }
        const int i = (mg * QW + m) * 16 + g + 8 * e;
        const bool in = i < a.n && rg.any;
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
        }
#pragma unroll
        for (int s = 0; s < C::KS; ++s)
#pragma unroll
          for (int f = 0; f < 4; ++f) {
            ss = fmaf(x[s][f], x[s][f], ss);
            top = max(top, __float_as_uint(x[s][f]) & 0x7fffffffu);
          }
        ss += __shfl_xor_sync(0xffffffffu, ss, 1);
        ss += __shfl_xor_sync(0xffffffffu, ss, 2);
        float scale = 1.f;
        if constexpr (C::I8) {
          // bring the row's largest element into [1, 2): the bf16 row is then
          // exact in fp16 (elements under 2^-16 of the largest round at 2^-25
          // of it), an fp32 row is held as hi + lo halves to 2^-25
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
            if constexpr (C::QHL) {
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
        // int8: alpha carries the V row's scale <= 1 / 127; 2^20 keeps it normal
        // in fp16 down to alpha = 2^-23
        ci[m][e] = (C::I8 ? 0x1p19f : 0.5f) * cn;
        si[m][e] = (C::I8 ? 0x1p19f : 0.5f) * sn;
        if (!live) rq[m][e] = __uint_as_float(0x7fc00000u);  // t = NaN: sees nothing
      }
    const float2 one_r = both(1.0f - r);

    float o[QW][C::NT][4];
    // pass 0 takes every V row and scale as finite.  A non-finite one times
    // alpha = 0 would spoil queries that do not see it: if any sum comes out
    // non-finite, pass 1 repeats the run with such rows left out of the product
    // and put back as NaN for the queries that see them.
#pragma unroll 1
    for (int pass = 0; pass < 2; ++pass) {
#pragma unroll
      for (int m = 0; m < QW; ++m)
#pragma unroll
        for (int j = 0; j < C::NT; ++j)
#pragma unroll
          for (int f = 0; f < 4; ++f) o[m][j][f] = 0.f;
      if (rg.any) {
        // stage x of the group sits in ring slot (its turn) % S
        long long rows[S - 1], next;
#pragma unroll
        for (int i = 0; i < S - 1; ++i) rows[i] = key_row(s0 + wk + i * C::WK);
        next = key_row(s0 + wk + (S - 1) * C::WK);
#pragma unroll
        for (int i = 0; i < S - 1; ++i) load_stage(s0 + wk + i * C::WK, i, rows[i]);
        int slot = 0, fill = S - 1;
#pragma unroll 1
        for (int x = s0 + wk; x <= s1; x += C::WK) {
          cp_async_wait<S - 2>();
          group_sync();
          load_stage(x + (S - 1) * C::WK, fill, next);
          next = key_row(x + S * C::WK);
          const unsigned char* kt = ring + (size_t)slot * C::STAGE_B;
          const unsigned char* vt = kt + C::TILE_B;
          const float* cs = reinterpret_cast<const float*>(kt + 2 * C::TILE_B);
          const int* cpos = reinterpret_cast<const int*>(cs) + (C::I8 ? 4 : 2) * KT;
          const bool edge = cpos[KT] != 0;
          slot = slot + 1 == S ? 0 : slot + 1;
          fill = fill + 1 == S ? 0 : fill + 1;
#pragma unroll
          for (int kg = 0; kg < KT / 16; ++kg) {
            float2 s[QW][2][RH];                       // keys 2t, 2t + 1 of an 8-key tile
            float tmax = 0.f;
            {
              uint32_t kb[2][C::KS][2];
              float c[2][QW][4], d[C::QHL ? 2 : 1][QW][4];
              float2 ks[2];
#pragma unroll
              for (int nt = 0; nt < 2; ++nt) {
                const int base = kg * 16 + nt * 8;
                load_k<C>(kt, base + key_of<C>(g), t, kb[nt]);
                ks[nt] = both(1.f);
                if constexpr (C::I8)
                  ks[nt] = *reinterpret_cast<const float2*>(cs + 2 * KT + base + 2 * t);
#pragma unroll
                for (int m = 0; m < QW; ++m)
#pragma unroll
                  for (int f = 0; f < 4; ++f) {
                    c[nt][m][f] = 0.f;
                    if constexpr (C::QHL) d[nt][m][f] = 0.f;
                  }
              }
              // k step outermost: 2 QW independent chains of products
              if constexpr (C::QHL) {
                // the small products first, and two chains: the tensor core's
                // sums truncate
#pragma unroll
                for (int x2 = 0; x2 < C::KS; ++x2)
#pragma unroll
                  for (int nt = 0; nt < 2; ++nt)
#pragma unroll
                    for (int m = 0; m < QW; ++m)
                      mma_f16(x2 & 1 ? d[nt][m] : c[nt][m], ql[m][x2], kb[nt][x2][0], kb[nt][x2][1]);
              }
#pragma unroll
              for (int x2 = 0; x2 < C::KS; ++x2)
#pragma unroll
                for (int nt = 0; nt < 2; ++nt)
#pragma unroll
                  for (int m = 0; m < QW; ++m) {
                    if constexpr (C::QHL)
                      mma_f16(x2 & 1 ? d[nt][m] : c[nt][m], qa[m][x2], kb[nt][x2][0], kb[nt][x2][1]);
                    else if constexpr (C::I8)
                      mma_f16(c[nt][m], qa[m][x2], kb[nt][x2][0], kb[nt][x2][1]);
                    else
                      mma_b16(c[nt][m], qa[m][x2], kb[nt][x2][0], kb[nt][x2][1]);
                  }
              // step by step over all scores: their chains run side by side
#pragma unroll
              for (int nt = 0; nt < 2; ++nt)
#pragma unroll
                for (int m = 0; m < QW; ++m)
#pragma unroll
                  for (int e = 0; e < RH; ++e) {
                    s[m][nt][e] = make_float2(c[nt][m][2 * e], c[nt][m][2 * e + 1]);
                    if constexpr (C::QHL) {
                      s[m][nt][e].x += d[nt][m][2 * e];
                      s[m][nt][e].y += d[nt][m][2 * e + 1];
                    }
                    if constexpr (C::I8) s[m][nt][e] = mul2(s[m][nt][e], ks[nt]);
                  }
#pragma unroll
              for (int nt = 0; nt < 2; ++nt)
#pragma unroll
                for (int m = 0; m < QW; ++m)
#pragma unroll
                  for (int e = 0; e < RH; ++e)
                    s[m][nt][e] = fma2(s[m][nt][e], both(rq[m][e]), one_r);
              // NaN (an unseen row, a non-finite key) counts as 0
#pragma unroll
              for (int nt = 0; nt < 2; ++nt)
#pragma unroll
                for (int m = 0; m < QW; ++m)
#pragma unroll
                  for (int e = 0; e < RH; ++e)
                    s[m][nt][e] = make_float2(fmaxf(s[m][nt][e].x, 0.f), fmaxf(s[m][nt][e].y, 0.f));
            }
            if (edge) {
#pragma unroll
              for (int nt = 0; nt < 2; ++nt)
#pragma unroll
                for (int f = 0; f < 2; ++f) {
                  const int col = kg * 16 + nt * 8 + 2 * t + f;
                  const int c = cpos[col];
                  const long long at =
                      (long long)x * KT + (col & ~7) + key_of<C>(2 * t + f) - lens;
#pragma unroll
                  for (int m = 0; m < QW; ++m)
#pragma unroll
                    for (int e = 0; e < RH; ++e) {
                      bool see = dep[m][e] - c <= rg.dmax;
                      const int i = (mg * QW + m) * 16 + g + 8 * e;
                      if (at >= 0 && at < a.n && i < a.n) see = see && (nodes.line[i] >> at & 1);
                      if (!see) (f ? s[m][nt][e].y : s[m][nt][e].x) = 0.f;
                    }
                }
            }
#pragma unroll
            for (int m = 0; m < QW; ++m)
#pragma unroll
              for (int nt = 0; nt < 2; ++nt)
#pragma unroll
                for (int e = 0; e < RH; ++e) tmax = fmaxf(tmax, fmaxf(s[m][nt][e].x, s[m][nt][e].y));
            if (!__any_sync(0xffffffffu, tmax > 0.f)) continue;
            uint32_t vb[C::NT][2];
            load_v<C>(vt, kg * 16, lane, vb);
            // which of the 16 keys' V rows are non-finite (pass 1 only)
            uint32_t bad = 0;
            if (pass == 1) {
              bool nf = false;
              if constexpr (C::I8) {
                nf = !(fabsf(cs[3 * KT + kg * 16 + (lane & 15)]) < 3.0e38f);
              } else {
                for (int c = 0; c < C::CH; ++c) {
                  const uint4 u =
                      *reinterpret_cast<const uint4*>(vt + v_off<C>(kg * 16 + (lane & 15), c));
                  const uint32_t ww[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
                  for (int q = 0; q < 4; ++q)
                    nf = nf || (ww[q] & 0x7f80u) == 0x7f80u || (ww[q] & 0x7f800000u) == 0x7f800000u;
                }
              }
              bad = __ballot_sync(0xffffffffu, nf) & 0xffffu;  // bit: score column
              if constexpr (!C::I8) {
#pragma unroll
                for (int j = 0; j < C::NT; ++j)
#pragma unroll
                  for (int hh = 0; hh < 2; ++hh) {
                    if (bad >> (8 * hh + 2 * t) & 1) vb[j][hh] &= 0xffff0000u;
                    if (bad >> (8 * hh + 2 * t + 1) & 1) vb[j][hh] &= 0x0000ffffu;
                  }
              }
            }
            // cos, sin and 1/2 of the mask, times the V row's scale
            float2 cc[2], sc[2], hc[2];
#pragma unroll
            for (int nt = 0; nt < 2; ++nt) {
              const int at = kg * 16 + nt * 8 + 2 * t;
              cc[nt] = *reinterpret_cast<const float2*>(cs + at);
              sc[nt] = *reinterpret_cast<const float2*>(cs + KT + at);
              hc[nt] = both(0.5f);
              if constexpr (C::I8) {
                const float2 vs = *reinterpret_cast<const float2*>(cs + 3 * KT + at);
                cc[nt] = mul2(cc[nt], vs);
                sc[nt] = mul2(sc[nt], vs);
                hc[nt] = mul2(vs, both(0x1p19f));
              }
            }
            float2 al[QW][2][RH];
#pragma unroll
            for (int m = 0; m < QW; ++m)
#pragma unroll
              for (int nt = 0; nt < 2; ++nt)
#pragma unroll
                for (int e = 0; e < RH; ++e) al[m][nt][e] = fma2(sc[nt], both(si[m][e]), hc[nt]);
#pragma unroll
            for (int m = 0; m < QW; ++m)
#pragma unroll
              for (int nt = 0; nt < 2; ++nt)
#pragma unroll
                for (int e = 0; e < RH; ++e) al[m][nt][e] = fma2(cc[nt], both(ci[m][e]), al[m][nt][e]);
#pragma unroll
            for (int m = 0; m < QW; ++m)
#pragma unroll
              for (int nt = 0; nt < 2; ++nt)
#pragma unroll
                for (int e = 0; e < RH; ++e)
                  al[m][nt][e] = mul2(mul2(s[m][nt][e], s[m][nt][e]), al[m][nt][e]);
            if (bad) {
#pragma unroll
              for (int m = 0; m < QW; ++m)
#pragma unroll
                for (int nt = 0; nt < 2; ++nt)
#pragma unroll
                  for (int e = 0; e < RH; ++e) {
                    const uint32_t two = bad >> (8 * nt + 2 * t);
                    const float2 x1 = s[m][nt][e];
                    if (((two & 1) && x1.x > 0.f) || ((two & 2) && x1.y > 0.f))
                      o[m][0][2 * e] = __uint_as_float(0x7fc00000u);
                    if (two & 1) al[m][nt][e].x = 0.f;
                    if (two & 2) al[m][nt][e].y = 0.f;
                  }
            }
            // a fragment's registers: row half e of 8-key tile nt
            uint32_t pa[QW][4], pl[C::PHL ? QW : 1][4];
#pragma unroll
            for (int m = 0; m < QW; ++m)
#pragma unroll
              for (int nt = 0; nt < 2; ++nt)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                  const int f = 2 * nt + e;
                  if (e >= RH) {
                    pa[m][f] = 0u;
                    if constexpr (C::PHL) pl[m][f] = 0u;
                    continue;
                  }
                  const float2 v = al[m][nt][e < RH ? e : 0];
                  pa[m][f] = C::I8 ? pack_f16(v.x, v.y) : pack_bf16(v.x, v.y);
                  if constexpr (C::PHL) {
                    const float2 u = C::I8 ? __half22float2(*reinterpret_cast<__half2*>(&pa[m][f]))
                                           : unpack_bf16(pa[m][f]);
                    pl[m][f] = C::I8 ? pack_f16(v.x - u.x, v.y - u.y) : pack_bf16(v.x - u.x, v.y - u.y);
                  }
                }
#pragma unroll
            for (int m = 0; m < QW; ++m)
#pragma unroll
              for (int j = 0; j < C::NT; ++j) {
                if constexpr (C::QHL) {
                  float d[4] = {0.f, 0.f, 0.f, 0.f};
                  mma_f16(d, pl[m], vb[j][0], vb[j][1]);
                  mma_f16(d, pa[m], vb[j][0], vb[j][1]);
#pragma unroll
                  for (int f = 0; f < 2 * RH; ++f) o[m][j][f] += d[f];
                } else if constexpr (C::I8) {
                  mma_f16(o[m][j], pa[m], vb[j][0], vb[j][1]);
                } else {
                  mma_b16(o[m][j], pl[m], vb[j][0], vb[j][1]);
                }
              }
            if constexpr (!C::I8) {
#pragma unroll
              for (int m = 0; m < QW; ++m)
#pragma unroll
                for (int j = 0; j < C::NT; ++j) mma_b16(o[m][j], pa[m], vb[j][0], vb[j][1]);
            }
          }
        }
        cp_async_wait<0>();
      }
      bool nf = false;
#pragma unroll
      for (int m = 0; m < QW; ++m)
#pragma unroll
        for (int j = 0; j < C::NT; ++j)
#pragma unroll
          for (int f = 0; f < 2 * RH; ++f) nf = nf || !(fabsf(o[m][j][f]) < 3.0e38f);
      if (!__syncthreads_or(nf)) break;
    }
    __syncthreads();   // the rings become the reduction buffer

    // --- sum the groups, finish or leave the partial ----------------------------
    float* red = reinterpret_cast<float*>(dsm);          // [WK][MG * QW * 16][D]
    constexpr int ROWS = C::MG * QW * 16;
#pragma unroll
    for (int m = 0; m < QW; ++m)
#pragma unroll
      for (int e = 0; e < RH; ++e) {
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
      if (!whole) {
        float* dst = part + ((size_t)(blockIdx.x + sh.seg) * a.n + i) * D;
#pragma unroll
        for (int e = 0; e < PER; ++e)
          if (lane + 32 * e < D) dst[lane + 32 * e] = x[e];
      } else {
        store_row<TA, D>(a, b, i, h, lane, x, rg.any && nodes.line[i] != 0);
      }
    }
  }
}

template <class C>
void launch_tree(const TreeParams& p, float* ws, cudaStream_t s) {
  if (ensure_smem_optin((const void*)tree_mma_kernel<C>, C::SMEM) != cudaSuccess) return;
  launch_pdl(tree_mma_kernel<C>, tree_grid(p, C::MINB), dim3(kThreads),
             (size_t)C::SMEM, s, p, ws);
}
// Query tiles per warp: two where the registers allow it (D <= 64) and there
// are more than 16 queries, so that a K / V fragment feeds two products; up to
// 8 queries the lower half of a tile is not computed on.
template <typename E, typename TA, int D>
void launch_tree_d(const TreeParams& p, float* ws, cudaStream_t s) {
    constexpr int Q2 = D <= 64 ? 2 : 1;
  if (p.a.n <= 8) launch_tree<Cfg<E, TA, D, 1, 1, 1>>(p, ws, s);
  else if (p.a.n <= 16) launch_tree<Cfg<E, TA, D, 1, 1, 2>>(p, ws, s);
  else if (p.a.n <= 32) launch_tree<Cfg<E, TA, D, Q2, 2 / Q2, 2>>(p, ws, s);
  else launch_tree<Cfg<E, TA, D, Q2, 4 / Q2, 2>>(p, ws, s);
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
