// The warp-MMA form of the tree attention: bf16 pages with bf16 activations,
// or int8 pages with bf16 / fp32 activations.
#pragma once
#include <cuda_fp16.h>
#include <type_traits>
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
// The first product of a chain: sums from zero, no registers cleared for it.
template <bool F16>
__device__ __forceinline__ void mma_first(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
  if constexpr (F16)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%10,%10,%10,%10};\n"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%10,%10,%10,%10};\n"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
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

template <typename E_, typename TA_, int D_, int MG_, int RH_>
struct Cfg {
  using E = E_;
  using TA = TA_;
  static constexpr int D = D_;
  static constexpr int MG = MG_;                 // warps of a group, 16 queries each
  static constexpr int RH = RH_;                 // query rows per thread: 1 if n <= 8
  static constexpr int WK = 4 / MG_;             // groups side by side over the keys
  static constexpr bool I8 = sizeof(E_) == 1;
  // A group of several warps turns its int8 stage into fp16 once, for all of
  // them; a lone warp does it on the way into the fragments.
  static constexpr bool CONV = I8 && MG_ > 1;
  static constexpr bool LDM = !I8 || CONV;       // 16-bit tiles read by ldmatrix
  // alpha enters the product whole: as two fp16 numbers over int8 pages (2^-22 of
  // it), as three bf16 numbers over bf16 pages (2^-24).  One fp16 or two bf16 numbers
  // (2^-11, 2^-16) show wherever values cancel.
  // fp32 activations: q as hi + lo too, fp32 sums between products.
  static constexpr bool QHL = I8 && sizeof(TA_) == 4;
  // up to 8 queries leave the lower rows of a tile free: alpha's second numbers go
  // there, in the same product as the first
  static constexpr bool SPARE = !QHL && RH_ == 1;
  static constexpr int RB = D_ * (int)sizeof(E_);     // row bytes
  static constexpr int CH = RB / 16;                  // 16-byte chunks per row
  static constexpr int CH16 = D_ / 8;                 // of a 16-bit row
  static constexpr int KS = D_ / 16;                  // MMA k steps of S
  static constexpr int NT = D_ / 8;                   // 8-column tiles of O
  static constexpr int KT = RB <= 128 ? 32 : 16;      // keys per stage of a group
  static constexpr int NK = KT / 16;                  // 16-key groups of it
  static constexpr int GT = 32 * MG_;                 // threads of a group
  static constexpr int TILE_B = KT * RB;
  // per key, in score-column order: cos, sin of pi c / w, K / V scale, c
  static constexpr int META_B = KT * (I8 ? 20 : 12) + 16;
  static constexpr int STAGE_B = 2 * TILE_B + META_B;
  static constexpr int S = CONV ? 4 : RB * KT <= 2048 ? 3 : 2;   // stages of a group's ring
  static constexpr int RING_B = S * STAGE_B;
  static constexpr int HALF_B = CONV ? KT * D_ * 2 : 0;   // fp16 tile; K and V, two of each
  static constexpr int PLAN_B = MG_ > 1 ? 2 * (KT + 1) * 8 + 16 : 0;   // see `plan`; two of them
  static constexpr int PLAN_AT = RING_B + 4 * HALF_B;
  static constexpr int GROUP_B = (PLAN_AT + PLAN_B + 15) / 16 * 16;
  static constexpr int RED_B = 4 * 16 * D_ * 4;       // the warps' sums at the end
  static constexpr int MAIN_B = WK * GROUP_B > RED_B ? WK * GROUP_B : RED_B;
  static constexpr int SMEM = MAIN_B > kAppendScratch ? MAIN_B : kAppendScratch;
  static_assert(SMEM >= kAppendScratch && SMEM >= kTreeMaxCtas * 4, "append_rows and find_run work in it");
  // CTAs per SM the registers are cut to: what a thread holds of O and q decides
  static constexpr int HELD = D_ / 2 + D_ / 4 * (QHL ? 2 : 1);
  // (a group of four warps on int8 pages waits at its barriers and gains by a fourth
  // CTA: 64 nodes over 32K keys 157 us, 160 with three)
  static constexpr int MINB =
      HELD <= 32 ? 4 : HELD <= 64 ? (CONV && MG_ == 4 && !QHL ? 4 : 3) : 2;
  // CTAs resident on an SM (int8 rows of 128 with 17 to 32 nodes: one; 32 nodes, 4 x 8
  // heads, 8K keys 47 us, 56 with runs cut for two; 24 nodes, 4 x 16 heads, 32K keys,
  // where two waves even out the heads, 290 and 275)
  static constexpr int PER_SM = fit_shared(SMEM, MINB);
  static_assert(PER_SM >= 1 && sizeof(Nodes) + 64 <= 1536, "a CTA fits, and its static arrays are counted");
};

// Byte offset of 16-byte chunk c of row r in a tile: the XOR makes the fragment
// loads below hit distinct banks (rows of 64 or 128 bytes alias).
template <int CH>
__device__ __forceinline__ uint32_t off16(int r, int c) {   // 16-bit rows, for ldmatrix
  const int x = CH >= 8 ? c ^ (r & 7) : CH == 4 ? c ^ ((r >> 1) & 3) : c ^ ((r >> 2) & 1);
  return (uint32_t)(r * CH * 16 + (x << 4));
}
template <class C>
__device__ __forceinline__ uint32_t k_off(int r, int c) {
  if constexpr (!C::I8) return off16<C::CH>(r, c);
  const int x = C::CH >= 8 ? c ^ ((r & 1) << 2) : c;
  return (uint32_t)(r * C::RB + (x << 4));
}
template <class C>
__device__ __forceinline__ uint32_t v_off(int r, int c) {
  if constexpr (!C::I8) return off16<C::CH>(r, c);
  const int x = C::CH == 8 ? c ^ (r & 6) : C::CH == 4 ? c ^ ((r & 4) >> 1) : c;
  return (uint32_t)(r * C::RB + (x << 4));
}
// Key of column c of an 8-key score tile.  int8 fragments: neighbouring columns
// (a thread's pair) are taken so that the four pairs a load touches start on
// different banks for both K (even / odd rows) and V.
template <class C>
__device__ __forceinline__ int key_of(int c) {
  return C::LDM ? c : c ^ ((c >> 1) & 1);
}

// d of pair e (elements 2 e, 2 e + 1 of a thread's four) of k step s.  ldmatrix
// fragments: 16 s + 2 t and 8 on.  int8 fragments: thread t = lane % 4 holds chunk t
// (+ 4 h) of a key row, k step s takes four consecutive elements of it.
template <class C>
__device__ __forceinline__ int d_of(int t, int s, int e) {
  if constexpr (C::LDM) return 16 * s + 8 * e + 2 * t;
  else if constexpr (C::D == 128) return 64 * (s >> 2) + 16 * t + 4 * (s & 3) + 2 * e;
  else if constexpr (C::D == 64) return 16 * t + 4 * s + 2 * e;
  else if constexpr (C::D == 32) return 8 * t + 4 * s + 2 * e;
  else return 4 * t + 2 * e;
}
// B operands of S for k step s of the 16 keys from row `base`, both 8-key tiles,
// from 16-bit rows: lanes 0-7 / 8-15 address keys 0-7, chunks 2 s / 2 s + 1; 16-31
// keys 8-15.
template <class C>
__device__ __forceinline__ void load_k16(const unsigned char* kt, int base, int s, int lane,
                                         uint32_t (&k0)[2], uint32_t (&k1)[2]) {
  const int r = base + (lane & 7) + ((lane >> 4) << 3), c = (lane >> 3) & 1;
  ldsm_x4(smem_u32(kt) + off16<C::CH16>(r, 2 * s + c), k0[0], k0[1], k1[0], k1[1]);
}
// The same for all k steps from int8 rows.
template <class C>
__device__ __forceinline__ void load_k8(const unsigned char* kt, int base, int lane,
                                        uint32_t (&kb)[2][C::KS][2]) {
  const int g = lane >> 2, t = lane & 3;
  constexpr int W = C::KS;              // words: 4 bytes per k step
  uint32_t w[2][W];
#pragma unroll
  for (int nt = 0; nt < 2; ++nt) {
    const int r = base + 8 * nt + key_of<C>(g);
    if constexpr (C::D >= 64) {
#pragma unroll
      for (int hh = 0; hh < C::D / 64; ++hh)
        *reinterpret_cast<uint4*>(&w[nt][4 * hh]) =
            *reinterpret_cast<const uint4*>(kt + k_off<C>(r, t + 4 * hh));
    } else if constexpr (C::D == 32) {
      *reinterpret_cast<uint2*>(&w[nt][0]) = *reinterpret_cast<const uint2*>(kt + r * C::RB + 8 * t);
    } else {
      w[nt][0] = *reinterpret_cast<const uint32_t*>(kt + r * C::RB + 4 * t);
    }
  }
#pragma unroll
  for (int nt = 0; nt < 2; ++nt)
#pragma unroll
    for (int s = 0; s < W; ++s) w[nt][s] ^= 0x80808080u;
#pragma unroll
  for (int nt = 0; nt < 2; ++nt)
#pragma unroll
    for (int s = 0; s < W; ++s) {
      kb[nt][s][0] = __byte_perm(w[nt][s], 0x64646464u, 0x4140);
      kb[nt][s][1] = __byte_perm(w[nt][s], 0x64646464u, 0x4342);
    }
#pragma unroll
  for (int nt = 0; nt < 2; ++nt)
#pragma unroll
    for (int s = 0; s < W; ++s) {
      kb[nt][s][0] = f16_of_biased(kb[nt][s][0]);
      kb[nt][s][1] = f16_of_biased(kb[nt][s][1]);
    }
}

// Column of O that column n of tile nt stands for: for int8 fragments d = NT n +
// nt, so that a thread's NT columns are consecutive bytes of a V row.
template <class C>
__device__ __forceinline__ int o_col(int nt, int n) {
  return C::LDM ? 8 * nt + n : C::NT * n + nt;
}
// B operand of alpha V for the 16 keys from row `base` of the V tile.
template <class C>
__device__ __forceinline__ void load_v(const unsigned char* vt, int base, int lane,
                                       uint32_t (&vb)[C::NT][2]) {
  const int g = lane >> 2, t = lane & 3;
  if constexpr (C::LDM) {
    // ldmatrix.trans: lanes 0-7 / 8-15 address keys 0-7 / 8-15 of chunk c, lanes
    // 16-31 those of chunk c + 1
    const int r = base + (lane & 15);
    const uint32_t at = smem_u32(vt);
#pragma unroll
    for (int c = 0; c < C::NT; c += 2)
      ldsm_x4_t(at + off16<C::CH16>(r, c + (lane >> 4)), vb[c][0], vb[c][1], vb[c + 1][0], vb[c + 1][1]);
  } else {
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
  }
}
// 16 int8 values as two chunks of fp16.
__device__ __forceinline__ void widen16(uint4 u, uint4& lo, uint4& hi) {
  uint32_t w[4] = {u.x, u.y, u.z, u.w}, h[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] ^= 0x80808080u;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    h[2 * i] = __byte_perm(w[i], 0x64646464u, 0x4140);
    h[2 * i + 1] = __byte_perm(w[i], 0x64646464u, 0x4342);
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) h[i] = f16_of_biased(h[i]);
  lo = make_uint4(h[0], h[1], h[2], h[3]);
  hi = make_uint4(h[4], h[5], h[6], h[7]);
}

// The CTA's four warps form 4 / MG groups; a group streams its own stages of KT
// keys (no barrier across the CTA inside the loop), groups taking the stages of
// a run in turn.  Work on scores goes step by step over all of a thread's scores,
// so that their dependent chains run side by side.
//
// A group of one warp (up to 16 nodes) is bound by its issue and its waits before
// HBM: one query per sequence over 100K int8 keys of 64 heads 122 us, 4.5 TB/s.  64
// nodes over 32K int8 keys 157 us, 137 TFLOP/s, half of the issue slots and 40 % of
// mma.sync used (490 instructions a warp per 32 keys x 16 nodes; 136 us and 430 with
// alpha as one fp16 number).  64 nodes over 32K bf16 keys 178 us (151 with alpha as
// two bf16 numbers).  16 nodes over windows of 4K on bf16 pages 25 us, 8.1 us for one
// token over 256 int8 keys: latency.
template <class C>
__global__ void __launch_bounds__(kThreads, C::MINB) tree_mma_kernel(TreeParams p,
                                                                     float* __restrict__ ws) {
  using E = typename C::E;
  using TA = typename C::TA;
  constexpr int D = C::D, S = C::S, KT = C::KT, RH = C::RH, GT = C::GT;
  constexpr int AHEAD = C::CONV ? 1 : 0;               // stages widened before their use
  extern __shared__ __align__(128) unsigned char dsm[];
  __shared__ Nodes nodes;
  pdl_wait();
  pdl_trigger();
  const screen_tree_args& a = p.a;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  const int mg = warp % C::MG, wk = warp / C::MG;
  const int gt = mg * 32 + lane;                       // thread of the group
  unsigned char* ring = dsm + (size_t)wk * C::GROUP_B;
  unsigned char* half = ring + C::RING_B;              // CONV: K, V tiles in fp16, twice
  SegSlots* slots = reinterpret_cast<SegSlots*>(ws);
  float* part = ws + p.part_off;
  auto group_sync = [&] {
    if constexpr (C::MG == 1) __syncwarp();
    else asm volatile("bar.sync %0, %1;" ::"r"(1 + wk), "n"(GT) : "memory");
  };
  // page of a position without a 64-bit division
  const int ps = a.cache.page_size;
  const int ps_shift = (ps & (ps - 1)) == 0 ? 31 - __clz(ps) : -1;

  Range rg;
  int seg, c0, c1;
  bool whole;
  if (!find_run(p, reinterpret_cast<int*>(dsm), slots, seg, rg, c0, c1, whole)) return;
  const int b = seg / a.H, h = seg % a.H;
  // w <= 1 sees the query's own position alone, where the mask is 1 whatever w is;
  // 0, a NaN or a tiny w would put a NaN into the factors of its cosine
  const float w = fmaxf(a.w[h], 1.f), r = a.r[h];
  // r < 0 turns alpha up to (1 + 2 |r|)^2: t is held down by a power of two, so
  // that alpha stays below 4 (fp16 holds alpha * 2^20 / 127 up to alpha = 7.9)
  const float up = r < 0.f ? __uint_as_float(__float_as_uint(1.f - 2.f * r) & 0x7f800000u) : 1.f;
  const long long lens = rg.lens;
  if (warp == 0) tree_nodes(a, b, nodes, lane);
  __syncthreads();
  if (rg.any && a.k) append_rows<E, TA, D>(a, nodes, b, h, lens, c0, c1, dsm);

  // --- a stage: KT keys, their addresses and facts ---------------------------
  const int s0 = c0 * (kTile / KT), s1 = (c1 + 1) * (kTile / KT) - 1;
  const int* table = a.cache.block_table + (long long)b * a.cache.max_blocks;
  // page of this lane's key of stage x (-1 none) and the key's place in it; the row,
  // -1 none, is made of them as late as it is needed, so that nothing waits for
  // the table
  struct Key {
    int page;
    unsigned at;
  };
  auto key_page = [&](int x) -> Key {
    const long long pos = (long long)x * KT + lane;
    if (lane >= KT || x > s1 || pos < rg.first || pos >= lens + a.n) return Key{-1, 0};
    if (pos >= lens && !nodes.line[pos - lens]) return Key{-1, 0};
    const unsigned q = (unsigned)pos;                // a table holds < 2^31 positions
    const unsigned blk = ps_shift >= 0 ? q >> ps_shift : q / (unsigned)ps;
    if (blk >= (unsigned)a.cache.max_blocks) return Key{-1, 0};
    return Key{table[blk], q - blk * (unsigned)ps};
  };
  auto key_row = [&](Key k) -> long long {
    return (unsigned)k.page < (unsigned)a.cache.num_pages ? ((long long)k.page * a.H + h) * ps + k.at : -1;
  };
  // In a group of several warps they take turns in looking a stage's rows up: its
  // warp leaves them in a plan (rows, then the first row if all follow it, else
  // -1) that the group reads after its next barrier.
  auto plan = [&](int turn) {
    return reinterpret_cast<long long*>(ring + C::PLAN_AT) + (turn & 1) * (KT + 1);
  };
  auto first_of_run = [&](long long row) -> long long {
    const long long row0 = __shfl_sync(0xffffffffu, row, 0);
    const bool run = __all_sync(0xffffffffu, lane >= KT || row == row0 + lane) && row0 >= 0;
    return run ? row0 : -1;
  };
  auto make_plan = [&](int turn, long long row) {
    const long long row0 = first_of_run(row);
    long long* pl = plan(turn);
    if (lane < KT) pl[lane] = row;
    if (lane == 0) pl[KT] = row0;
  };
  // `row`: this lane's key, of the warp whose turn it is
  auto load_stage = [&](int turn, int slot, long long row, bool planned) {
    const int x = s0 + wk + turn * C::WK;
    unsigned char* st = ring + (size_t)slot * C::STAGE_B;
    if (x <= s1) {
      const uint32_t sa = smem_u32(st);
      const char* kp = reinterpret_cast<const char*>(a.cache.k_pages);
      const char* vp = reinterpret_cast<const char*>(a.cache.v_pages);
      const long long* pl = plan(turn);
      const long long row0 = C::MG > 1 && planned ? pl[KT] : first_of_run(row);
      if (row0 >= 0) {                               // all keys there, one after another
        const long long off = row0 * C::RB + gt * 16;
#pragma unroll
        for (int i = 0; i < (KT * C::CH + GT - 1) / GT; ++i) {
          const int u = i * GT + gt;
          if (KT * C::CH % GT == 0 || u < KT * C::CH) {
            cp_async16(sa + k_off<C>(u / C::CH, u % C::CH), kp + off + i * GT * 16, true);
            cp_async16(sa + C::TILE_B + v_off<C>(u / C::CH, u % C::CH), vp + off + i * GT * 16, true);
          }
        }
      } else {
#pragma unroll 1
        for (int i = 0; i < (KT * C::CH + GT - 1) / GT; ++i) {
          const int u = i * GT + gt, k = u / C::CH;
          long long at = __shfl_sync(0xffffffffu, row, k & (KT - 1));
          if (C::MG > 1 && planned) at = pl[k & (KT - 1)];
          if (k < KT) {
            const long long off = (at < 0 ? 0 : at) * C::RB + u % C::CH * 16;
            cp_async16(sa + k_off<C>(k, u % C::CH), kp + off, at >= 0);
            cp_async16(sa + C::TILE_B + v_off<C>(k, u % C::CH), vp + off, at >= 0);
          }
        }
      }
      if (mg == turn % C::MG) {
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
  // CONV: a landed int8 stage as fp16 tiles for ldmatrix
  auto widen_stage = [&](int slot, int buf) {
    const unsigned char* kt = ring + (size_t)slot * C::STAGE_B;
    unsigned char* kh = half + (size_t)buf * 2 * C::HALF_B;
#pragma unroll
    for (int i = 0; i < (KT * C::CH + GT - 1) / GT; ++i) {
      const int u = i * GT + gt;
      if (KT * C::CH % GT == 0 || u < KT * C::CH) {
        const int k = u / C::CH, c = u % C::CH;
        const uint4 x = *reinterpret_cast<const uint4*>(kt + k_off<C>(k, c));
        const uint4 y = *reinterpret_cast<const uint4*>(kt + C::TILE_B + v_off<C>(k, c));
        uint4 x0, x1, y0, y1;
        widen16(x, x0, x1);
        widen16(y, y0, y1);
        *reinterpret_cast<uint4*>(kh + off16<C::CH16>(k, 2 * c)) = x0;
        *reinterpret_cast<uint4*>(kh + off16<C::CH16>(k, 2 * c + 1)) = x1;
        *reinterpret_cast<uint4*>(kh + C::HALF_B + off16<C::CH16>(k, 2 * c)) = y0;
        *reinterpret_cast<uint4*>(kh + C::HALF_B + off16<C::CH16>(k, 2 * c + 1)) = y1;
      }
    }
    // the mask's factors with the V row's scale in them, once for all warps
    if (gt < KT) {
      float* cs = reinterpret_cast<float*>(ring + (size_t)slot * C::STAGE_B + 2 * C::TILE_B) + gt;
      const float vs = cs[3 * KT];
      cs[0] *= vs;
      cs[KT] *= vs;
      cs[3 * KT] = vs * 0x1p19f;
    }
  };

  // --- the first stages, under way while the queries are brought in ------------
  auto start = [&]() -> Key {
    // the group's stage number `turn` sits in ring slot turn % S
    Key keys[S];
#pragma unroll
    for (int i = 0; i < S; ++i) keys[i] = key_page(s0 + wk + i * C::WK);
#pragma unroll
    for (int i = 0; i < S - 1; ++i) load_stage(i, i, key_row(keys[i]), false);
    if (C::MG > 1 && mg == (S - 1) % C::MG) make_plan(S - 1, key_row(keys[S - 1]));
    return keys[S - 1];
  };
  Key next{-1, 0};
  if (rg.any) next = start();

  // --- queries: fragments, per-row factors ------------------------------------
  uint32_t qa[C::KS][4];
  uint32_t ql[C::QHL ? C::KS : 1][4];
  float rq[RH], ci[RH], si[RH];
  int dep[RH];
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    if (e >= RH) {
#pragma unroll
      for (int s = 0; s < C::KS; ++s) {
        qa[s][1] = qa[s][3] = 0u;
        if constexpr (C::QHL) ql[s][1] = ql[s][3] = 0u;
      }
      continue;
    }
    const int i = mg * 16 + g + 8 * e;
    const bool in = i < a.n && rg.any;
    const TA* q = reinterpret_cast<const TA*>(a.q) + (long long)b * a.q_sb + (long long)i * a.q_st +
                  (long long)h * D;
    float x[C::KS][4];
    // QHL: an error of |q| is one of every score, r / t times over in alpha: 64 bits
    using Sum = typename std::conditional<C::QHL, double, float>::type;
    Sum ss = 0;
    uint32_t top = 0;
#pragma unroll
    for (int s = 0; s < C::KS; ++s)
#pragma unroll
      for (int f = 0; f < 2; ++f) {
        x[s][2 * f] = x[s][2 * f + 1] = 0.f;
        if (in) {
          if constexpr (sizeof(TA) == 2) {
            const float2 v = unpack_bf16(*reinterpret_cast<const uint32_t*>(q + d_of<C>(t, s, f)));
            x[s][2 * f] = v.x;
            x[s][2 * f + 1] = v.y;
          } else {
            const float2 v = *reinterpret_cast<const float2*>(q + d_of<C>(t, s, f));
            x[s][2 * f] = v.x;
            x[s][2 * f + 1] = v.y;
          }
        }
      }
#pragma unroll
    for (int s = 0; s < C::KS; ++s)
#pragma unroll
      for (int f = 0; f < 4; ++f) {
        ss = fma((Sum)x[s][f], (Sum)x[s][f], ss);
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
    for (int s = 0; s < C::KS; ++s)
#pragma unroll
      for (int f = 0; f < 2; ++f) {
        if constexpr (C::I8) {
          qa[s][2 * f + e] = pack_f16(x[s][2 * f], x[s][2 * f + 1]);
          if constexpr (C::QHL) {
            const float2 u = __half22float2(*reinterpret_cast<__half2*>(&qa[s][2 * f + e]));
            ql[s][2 * f + e] = pack_f16(x[s][2 * f] - u.x, x[s][2 * f + 1] - u.y);
          }
        } else {
          qa[s][2 * f + e] = pack_bf16(x[s][2 * f], x[s][2 * f + 1]);
        }
      }
    // S = q.k scale / max(|q|, eps), times r; scale first: 2^ex / |q| <= 1.  QHL: -S
    if constexpr (C::QHL) rq[e] = (float)(-(double)scale / fmax(sqrt(ss), (double)a.eps));
    else rq[e] = r / up * (scale / fmaxf(sqrtf(ss), a.eps));
    const bool live = in && nodes.line[i] != 0;
    dep[e] = live ? nodes.depth[i] : 0;
    float sn, cn;
    sincospif((float)dep[e] / w, &sn, &cn);
    // int8: alpha carries the V row's scale <= 1 / 127; 2^20 keeps it normal
    // in fp16 down to alpha = 2^-23
    ci[e] = (C::I8 ? 0x1p19f : 0.5f) * cn;
    si[e] = (C::I8 ? 0x1p19f : 0.5f) * sn;
    if (!live) rq[e] = __uint_as_float(0x7fc00000u);  // t = NaN: sees nothing
  }
  // t = r S + (1 - r); QHL: 1 - r (1 - S), whose roundings do not grow with r
  const float2 one_r = both((1.0f - r) / up), nr = both(-r / up), one = both(1.0f / up);

  float o[C::NT][4];
  // pass 0 takes every V row and scale as finite.  A non-finite one times
  // alpha = 0 would spoil queries that do not see it: if any sum comes out
  // non-finite, pass 1 repeats the run with such rows left out of the product
  // and put back as NaN for the queries that see them.
#pragma unroll 1
  for (int pass = 0; pass < 2; ++pass) {
#pragma unroll
    for (int j = 0; j < C::NT; ++j)
#pragma unroll
      for (int f = 0; f < 4; ++f) o[j][f] = 0.f;
    if (rg.any) {
      if (pass == 1) next = start();
      int slot = 0, fill = S - 1, buf = 0;
      if constexpr (C::CONV) {
        cp_async_wait<S - 2>();
        group_sync();
        if (s0 + wk <= s1) widen_stage(0, 0);
      }
#pragma unroll 1
      for (int x = s0 + wk, turn = 0; x <= s1; x += C::WK, ++turn) {
        cp_async_wait<S - 2 - AHEAD>();
        group_sync();
        load_stage(turn + S - 1, fill, key_row(next), true);
        if (C::MG == 1 || mg == (turn + S) % C::MG) {
          next = key_page(x + S * C::WK);
          if constexpr (C::MG > 1) make_plan(turn + S, key_row(next));
        }
        const unsigned char* st = ring + (size_t)slot * C::STAGE_B;
        const float* cs = reinterpret_cast<const float*>(st + 2 * C::TILE_B);
        const int* cpos = reinterpret_cast<const int*>(cs) + (C::I8 ? 4 : 2) * KT;
        const bool edge = cpos[KT] != 0;
        slot = slot + 1 == S ? 0 : slot + 1;
        fill = fill + 1 == S ? 0 : fill + 1;
        const unsigned char *kt = st, *vt = st + C::TILE_B;
        if constexpr (C::CONV) {
          if (x + C::WK <= s1) widen_stage(slot, buf ^ 1);
          kt = half + (size_t)buf * 2 * C::HALF_B;
          vt = kt + C::HALF_B;
          buf ^= 1;
        }
        // --- scores of the stage: 2 NK tiles of 8 keys, each its own chain ------
        constexpr int N8 = 2 * C::NK;
        float2 s[N8][RH];                            // keys 2t, 2t + 1 of an 8-key tile
        {
          float c[N8][4];
          // QHL: the tensor core's sums truncate, so a k step's products are summed
          // from zero, the small ones first, and the steps in fp32 (y over 11K keys is
          // 0.7e-6 off; 1.0e-6 with one chain, |q| in 32 bits and t = r S + (1 - r))
          auto score_hl = [&](float (&c)[N8][4], int x2, const uint32_t (&k2)[N8][2]) {
            float d[N8][4];
#pragma unroll
            for (int nt = 0; nt < N8; ++nt) mma_first<true>(d[nt], ql[x2], k2[nt][0], k2[nt][1]);
#pragma unroll
            for (int nt = 0; nt < N8; ++nt) mma_f16(d[nt], qa[x2], k2[nt][0], k2[nt][1]);
#pragma unroll
            for (int nt = 0; nt < N8; ++nt)
#pragma unroll
              for (int f = 0; f < 2 * RH; ++f) c[nt][f] = x2 == 0 ? d[nt][f] : c[nt][f] + d[nt][f];
          };
          if constexpr (C::LDM) {
#pragma unroll
            for (int x2 = 0; x2 < C::KS; ++x2) {
              uint32_t kb[N8][2];
#pragma unroll
              for (int kg = 0; kg < C::NK; ++kg) load_k16<C>(kt, kg * 16, x2, lane, kb[2 * kg], kb[2 * kg + 1]);
              if constexpr (C::QHL) {
                score_hl(c, x2, kb);
              } else {
#pragma unroll
                for (int nt = 0; nt < N8; ++nt) {
                  if (x2 == 0) mma_first<C::I8>(c[nt], qa[x2], kb[nt][0], kb[nt][1]);
                  else if constexpr (C::I8) mma_f16(c[nt], qa[x2], kb[nt][0], kb[nt][1]);
                  else mma_b16(c[nt], qa[x2], kb[nt][0], kb[nt][1]);
                }
              }
            }
          } else {
            uint32_t kb[C::NK][2][C::KS][2];
#pragma unroll
            for (int kg = 0; kg < C::NK; ++kg) load_k8<C>(kt, kg * 16, lane, kb[kg]);
#pragma unroll
            for (int x2 = 0; x2 < C::KS; ++x2) {
              if constexpr (C::QHL) {
                uint32_t k2[N8][2];
#pragma unroll
                for (int nt = 0; nt < N8; ++nt) {
                  k2[nt][0] = kb[nt >> 1][nt & 1][x2][0];
                  k2[nt][1] = kb[nt >> 1][nt & 1][x2][1];
                }
                score_hl(c, x2, k2);
              } else {
#pragma unroll
                for (int nt = 0; nt < N8; ++nt) {
                  const uint32_t* k2 = kb[nt >> 1][nt & 1][x2];
                  if (x2 == 0) mma_first<true>(c[nt], qa[x2], k2[0], k2[1]);
                  else mma_f16(c[nt], qa[x2], k2[0], k2[1]);
                }
              }
            }
          }
#pragma unroll
          for (int nt = 0; nt < N8; ++nt) {
            float2 ks = both(1.f);
            if constexpr (C::I8) ks = *reinterpret_cast<const float2*>(cs + 2 * KT + nt * 8 + 2 * t);
#pragma unroll
            for (int e = 0; e < RH; ++e) {
              s[nt][e] = make_float2(c[nt][2 * e], c[nt][2 * e + 1]);
              if constexpr (C::I8) s[nt][e] = mul2(s[nt][e], ks);
            }
          }
#pragma unroll
          for (int nt = 0; nt < N8; ++nt)
#pragma unroll
            for (int e = 0; e < RH; ++e) {
              if constexpr (C::QHL) s[nt][e] = fma2(fma2(s[nt][e], both(rq[e]), both(1.f)), nr, one);
              else s[nt][e] = fma2(s[nt][e], both(rq[e]), one_r);
            }
          // NaN (an unseen row, a non-finite key) counts as 0
#pragma unroll
          for (int nt = 0; nt < N8; ++nt)
#pragma unroll
            for (int e = 0; e < RH; ++e)
              s[nt][e] = make_float2(fmaxf(s[nt][e].x, 0.f), fmaxf(s[nt][e].y, 0.f));
        }
        if (edge) {
#pragma unroll
          for (int nt = 0; nt < N8; ++nt)
#pragma unroll
            for (int f = 0; f < 2; ++f) {
              const int c = cpos[nt * 8 + 2 * t + f];
              const long long at = (long long)x * KT + nt * 8 + key_of<C>(2 * t + f) - lens;
#pragma unroll
              for (int e = 0; e < RH; ++e) {
                bool see = dep[e] - c <= rg.dmax;
                const int i = mg * 16 + g + 8 * e;
                if (at >= 0 && at < a.n && i < a.n) see = see && (nodes.line[i] >> at & 1);
                if (!see) (f ? s[nt][e].y : s[nt][e].x) = 0.f;
              }
            }
        }
        // a lone warp skips the alpha V of 16 keys that are all under the trim; of
        // several warps' queries some nearly always see one
        bool live[C::NK];
#pragma unroll
        for (int kg = 0; kg < C::NK; ++kg) {
          float tmax = 0.f;
#pragma unroll
          for (int nt = 2 * kg; nt < 2 * kg + 2; ++nt)
#pragma unroll
            for (int e = 0; e < RH; ++e) tmax = fmaxf(tmax, fmaxf(s[nt][e].x, s[nt][e].y));
          live[kg] = C::MG > 1 || __any_sync(0xffffffffu, tmax > 0.f);
        }
        // --- alpha = t^2 (1 + cos) / 2, times the V row's scale -------------------
        float2 al[N8][RH];
#pragma unroll
        for (int nt = 0; nt < N8; ++nt) {
          float2 cc = *reinterpret_cast<const float2*>(cs + nt * 8 + 2 * t);
          float2 sc = *reinterpret_cast<const float2*>(cs + KT + nt * 8 + 2 * t);
          float2 hc = both(0.5f);
          if constexpr (C::I8) {
            const float2 vs = *reinterpret_cast<const float2*>(cs + 3 * KT + nt * 8 + 2 * t);
            if constexpr (C::CONV) {
              hc = vs;
            } else {
              cc = mul2(cc, vs);
              sc = mul2(sc, vs);
              hc = mul2(vs, both(0x1p19f));
            }
          }
#pragma unroll
          for (int e = 0; e < RH; ++e) al[nt][e] = fma2(sc, both(si[e]), hc);
#pragma unroll
          for (int e = 0; e < RH; ++e) al[nt][e] = fma2(cc, both(ci[e]), al[nt][e]);
        }
#pragma unroll
        for (int nt = 0; nt < N8; ++nt)
#pragma unroll
          for (int e = 0; e < RH; ++e) al[nt][e] = mul2(mul2(s[nt][e], s[nt][e]), al[nt][e]);
        // pass 1: V rows with a non-finite value (bit: score column) leave the
        // product; a query that sees one gets NaN
        uint32_t bad = 0;
        if (pass == 1) {
          bool nf = false;
          if (lane < KT) {
            if constexpr (C::I8) {
              nf = !(fabsf(cs[3 * KT + lane]) < 3.0e38f);
            } else {
              for (int c = 0; c < C::CH; ++c) {
                const uint4 u = *reinterpret_cast<const uint4*>(vt + v_off<C>(lane, c));
                const uint32_t ww[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
                for (int q = 0; q < 4; ++q)
                  nf = nf || (ww[q] & 0x7f80u) == 0x7f80u || (ww[q] & 0x7f800000u) == 0x7f800000u;
              }
            }
          }
          bad = __ballot_sync(0xffffffffu, nf);
          if (bad) {
#pragma unroll
            for (int nt = 0; nt < N8; ++nt)
#pragma unroll
              for (int e = 0; e < RH; ++e) {
                const uint32_t two = bad >> (8 * nt + 2 * t);
                const float2 x1 = s[nt][e];
                if (((two & 1) && x1.x > 0.f) || ((two & 2) && x1.y > 0.f))
                  o[0][2 * e] = __uint_as_float(0x7fc00000u);
                if (two & 1) al[nt][e].x = 0.f;
                if (two & 2) al[nt][e].y = 0.f;
              }
          }
        }
        // --- alpha V, 16 keys at a time -------------------------------------------
#pragma unroll
        for (int kg = 0; kg < C::NK; ++kg) {
          if (!live[kg]) continue;
          // a fragment's registers: row half e of 8-key tile nt; SPARE: pl's in row half 1
          uint32_t pa[4] = {0u, 0u, 0u, 0u}, pl[4] = {0u, 0u, 0u, 0u}, pm[4] = {0u, 0u, 0u, 0u};
#pragma unroll
          for (int nt = 0; nt < 2; ++nt)
#pragma unroll
            for (int e = 0; e < RH; ++e) {
              const int f = 2 * nt + e;
              const float2 v = al[2 * kg + nt][e];
              uint32_t& second = C::SPARE ? pa[f | 1] : pl[f];
              if constexpr (C::I8) {
                pa[f] = pack_f16(v.x, v.y);
                const float2 u = __half22float2(*reinterpret_cast<__half2*>(&pa[f]));
                second = pack_f16(v.x - u.x, v.y - u.y);
              } else {
                pa[f] = pack_bf16(v.x, v.y);
                float2 u = unpack_bf16(pa[f]);
                const float2 d = make_float2(v.x - u.x, v.y - u.y);
                second = pack_bf16(d.x, d.y);
                u = unpack_bf16(second);
                pm[f] = pack_bf16(d.x - u.x, d.y - u.y);
              }
            }
          uint32_t vb[C::NT][2];
          load_v<C>(vt, kg * 16, lane, vb);
          if constexpr (!C::I8) {
            if (bad) {
#pragma unroll
              for (int j = 0; j < C::NT; ++j)
#pragma unroll
                for (int hh = 0; hh < 2; ++hh) {
                  const uint32_t two = bad >> (16 * kg + 8 * hh + 2 * t);
                  if (two & 1) vb[j][hh] &= 0xffff0000u;
                  if (two & 2) vb[j][hh] &= 0x0000ffffu;
                }
            }
          }
          if constexpr (C::QHL) {
#pragma unroll
            for (int j = 0; j < C::NT; ++j) {
              float d[4];
              mma_first<true>(d, pl, vb[j][0], vb[j][1]);
              mma_f16(d, pa, vb[j][0], vb[j][1]);
#pragma unroll
              for (int f = 0; f < 2 * RH; ++f) o[j][f] += d[f];
            }
          } else if constexpr (C::I8) {
            if constexpr (!C::SPARE) {
#pragma unroll
              for (int j = 0; j < C::NT; ++j) mma_f16(o[j], pl, vb[j][0], vb[j][1]);
            }
#pragma unroll
            for (int j = 0; j < C::NT; ++j) mma_f16(o[j], pa, vb[j][0], vb[j][1]);
          } else {
#pragma unroll
            for (int j = 0; j < C::NT; ++j) mma_b16(o[j], pm, vb[j][0], vb[j][1]);
            if constexpr (!C::SPARE) {
#pragma unroll
              for (int j = 0; j < C::NT; ++j) mma_b16(o[j], pl, vb[j][0], vb[j][1]);
            }
#pragma unroll
            for (int j = 0; j < C::NT; ++j) mma_b16(o[j], pa, vb[j][0], vb[j][1]);
          }
        }
      }
      cp_async_wait<0>();
    }
    bool nf = false;
#pragma unroll
    for (int j = 0; j < C::NT; ++j)
#pragma unroll
      for (int f = 0; f < 2 * RH; ++f) nf = nf || !(fabsf(o[j][f]) < 3.0e38f);
    if (!__syncthreads_or(nf)) break;
  }
  __syncthreads();   // the rings become the reduction buffer

  // --- sum the groups, finish or leave the partial ----------------------------
  float* red = reinterpret_cast<float*>(dsm);          // [WK][MG * 16][D]
  constexpr int ROWS = C::MG * 16;
  const float back = (C::I8 ? 0x1p-20f : 1.f) * up * up;
#pragma unroll
  for (int e = 0; e < RH; ++e) {
    float* dst = red + ((size_t)wk * ROWS + mg * 16 + g + 8 * e) * D;
#pragma unroll
    for (int j = 0; j < C::NT; ++j)
#pragma unroll
      for (int f = 0; f < 2; ++f)
        dst[o_col<C>(j, 2 * t + f)] = (C::SPARE ? o[j][f] + o[j][2 + f] : o[j][2 * e + f]) * back;
  }
  __syncthreads();
  if (!whole) {
    float4* dst = reinterpret_cast<float4*>(part + (size_t)blockIdx.x * a.n * D);
    for (int u = tid; u < a.n * (D / 4); u += kThreads) {
      float4 x = reinterpret_cast<const float4*>(red)[u];
#pragma unroll
      for (int k = 1; k < C::WK; ++k) {
        const float4 y = reinterpret_cast<const float4*>(red + (size_t)k * ROWS * D)[u];
        x.x += y.x;
        x.y += y.y;
        x.z += y.z;
        x.w += y.w;
      }
      dst[u] = x;
    }
    return;
  }
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
    store_row<TA, D>(a, b, i, h, lane, x, rg.any && nodes.line[i] != 0);
  }
}

template <class C>
bool launch_tree(TreeParams& p, float* ws, cudaStream_t s) {
  if (ensure_smem_optin((const void*)tree_mma_kernel<C>, C::SMEM) != cudaSuccess) return false;
  prefer_shared((const void*)tree_mma_kernel<C>);
  const dim3 grid = tree_grid(p, C::PER_SM);
  launch_pdl(tree_mma_kernel<C>, grid, dim3(kThreads), (size_t)C::SMEM, s, p, ws);
  return p.a.num_ctas > 1;
}
// A warp for every 16 queries; up to 8 queries the lower half of a tile is not
// computed on.
template <typename E, typename TA, int D>
bool launch_tree_d(TreeParams& p, float* ws, cudaStream_t s) {
  if (p.a.n <= 8) return launch_tree<Cfg<E, TA, D, 1, 1>>(p, ws, s);
  if (p.a.n <= 16) return launch_tree<Cfg<E, TA, D, 1, 2>>(p, ws, s);
  if (p.a.n <= 32) return launch_tree<Cfg<E, TA, D, 2, 2>>(p, ws, s);
  return launch_tree<Cfg<E, TA, D, 4, 2>>(p, ws, s);
}
template <typename E, typename TA>
bool launch_tree_e(TreeParams& p, float* ws, cudaStream_t s) {
  switch (p.a.D) {
    case 16: return launch_tree_d<E, TA, 16>(p, ws, s);
    case 32: return launch_tree_d<E, TA, 32>(p, ws, s);
    case 64: return launch_tree_d<E, TA, 64>(p, ws, s);
    default: return launch_tree_d<E, TA, 128>(p, ws, s);
  }
}

}  // namespace tree
}  // namespace screen
