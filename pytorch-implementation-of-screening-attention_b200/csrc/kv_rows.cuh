// Rows of the paged cache: addressing, and the unit / int8 form of a raw row.
#pragma once
#include "common.cuh"

namespace screen {

// Row index (in rows of D elements) of position `pos` of sequence b, head h:
// pages are [num_pages, H, page_size, D].  -1 outside the table or for a page
// id outside the cache.
__device__ __forceinline__ long long paged_row(const screen_kv_cache& c, int b, int H, int h,
                                               long long pos) {
  if (pos < 0) return -1;
  const long long blk = pos / c.page_size;
  if (blk >= c.max_blocks) return -1;
  const int page = c.block_table[(long long)b * c.max_blocks + blk];
  if (page < 0 || page >= c.num_pages) return -1;
  return ((long long)page * H + h) * c.page_size + (pos - blk * c.page_size);
}

// The same from a sequence's table row, in 32 bits; a shift where the page size
// is a power of two.
__device__ __forceinline__ long long table_row(const screen_kv_cache& c, const int* table, int H,
                                               int h, long long pos) {
  if (pos < 0 || pos > 0x7fffffff) return -1;
  const unsigned p = (unsigned)pos, ps = (unsigned)c.page_size;
  const unsigned blk = (ps & (ps - 1)) == 0 ? p >> (31 - __clz(ps)) : p / ps;
  if (blk >= (unsigned)c.max_blocks) return -1;
  const int page = table[blk];
  if (page < 0 || page >= c.num_pages) return -1;
  return ((long long)page * H + h) * ps + (p - blk * ps);
}

template <typename T>
__device__ __forceinline__ void load4(const T* p, float (&x)[4]);
template <>
__device__ __forceinline__ void load4<float>(const float* p, float (&x)[4]) {
  const float4 v = *reinterpret_cast<const float4*>(p);
  x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w;
}
template <>
__device__ __forceinline__ void load4<__nv_bfloat16>(const __nv_bfloat16* p, float (&x)[4]) {
  const uint2 u = *reinterpret_cast<const uint2*>(p);
  const float2 a = unpack_bf16(u.x), b = unpack_bf16(u.y);
  x[0] = a.x; x[1] = a.y; x[2] = b.x; x[3] = b.y;
}

template <typename T>
__device__ __forceinline__ void load8f(const T* p, float (&x)[8]) {
  float a[4], b[4];
  load4(p, a);
  load4(p + 4, b);
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    x[e] = a[e];
    x[4 + e] = b[e];
  }
}

// The int8 form of a raw row x:
//   m = round_half_even(127 x / max|x|),  scale = 1 / max(|m|, 127 eps / max|x|),
// so scale * m is the unit form of the rounded raw row.  The integers do not
// depend on any order of summation: max|x| is exact, and |m|^2 <= 128 * 127^2 is
// summed in integers.  For bf16 values (BF) 127 x is exact in 32 bits, and a product
// with the approximate reciprocal and one remainder step leave the quotient right
// to 2^-24 (its nearest float, but for 2^-44 of it): a half comes out exactly, and
// no other quotient of 8-bit significands lies within 2^-17 of one; for fp32 a quotient so near a half
// that 32 bits cannot tell is decided by an exact comparison in 64 bits: three roundings
// of 2^-24 of up to 127 move it by 2.3e-5, and what lies within 2^-15 = 3.1e-5 of a
// half (one in 16,000) is compared.  A row with an infinity or NaN becomes m = 0, scale
// NaN.
struct Int8Scale {
  float up, am, inv;     // x is scaled by up (0: a row of zeros); am = max|up x|
};
// of a row whose largest magnitude has the bits `top`
template <bool BF>
__device__ __forceinline__ Int8Scale int8_scale(uint32_t top) {
  const bool finite = top < 0x7f800000u;
  const float amax = __uint_as_float(top);
  Int8Scale s{1.0f, amax, 0.f};
  if (!(amax > 1.0e-30f && amax < 1.0e30f)) {
    // outside the reciprocal's range: scaled by a power of two; a row of zeros
    // or with a non-finite value becomes zeros
    s.up = finite && top ? (amax < 1.0f ? 0x1p100f : 0x1p-100f) : 0.f;
    s.am = s.up != 0.f ? amax * s.up : 1.0f;
  }
  if constexpr (BF) asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(s.inv) : "f"(s.am));
  else s.inv = 1.0f / s.am;
  return s;
}
// E elements as int8, four to a word, and the sum of their squares added to ss.
template <int E, bool BF>
__device__ __forceinline__ void int8_pack(float (&x)[E], const Int8Scale& s, uint32_t (&m)[E / 4], int& ss) {
  if (s.up != 1.0f) {
#pragma unroll
    for (int e = 0; e < E; ++e) x[e] = s.up != 0.f ? x[e] * s.up : 0.f;
  }
  const float magic = 12582912.0f;   // 1.5 * 2^23: rounds to an integer in the low byte
  float f[E];
  if constexpr (BF) {
    // two elements an instruction, step by step over the row's part
    const float2 c127 = make_float2(127.0f, 127.0f), inv = make_float2(s.inv, s.inv);
    const float2 neg = make_float2(-s.am, -s.am), mg = make_float2(magic, magic);
    float2 d[E / 2], q[E / 2];
#pragma unroll
    for (int e = 0; e < E / 2; ++e) d[e] = __fmul2_rn(make_float2(x[2 * e], x[2 * e + 1]), c127);
#pragma unroll
    for (int e = 0; e < E / 2; ++e) q[e] = __fmul2_rn(d[e], inv);
#pragma unroll
    for (int e = 0; e < E / 2; ++e) d[e] = __ffma2_rn(q[e], neg, d[e]);
#pragma unroll
    for (int e = 0; e < E / 2; ++e) q[e] = __ffma2_rn(d[e], inv, q[e]);
#pragma unroll
    for (int e = 0; e < E / 2; ++e) {
      q[e] = __fadd2_rn(q[e], mg);
      f[2 * e] = q[e].x;
      f[2 * e + 1] = q[e].y;
    }
  } else {
    bool near = false;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const float t = 127.0f * x[e] * s.inv;
      f[e] = t + magic;
      near = near || fabsf(t - (f[e] - magic)) > 0.5f - 0x1p-15f;
    }
    if (near) {
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const float t = fabsf(127.0f * x[e] * s.inv), k = floorf(t);
        if (fabsf(t - k - 0.5f) < 0x1p-15f) {
          const double num = 127.0 * (double)fabsf(x[e]), half = ((double)k + 0.5) * (double)s.am;
          const bool odd = (int)k & 1;
          f[e] = copysignf(num > half || (num == half && odd) ? k + 1.0f : k, x[e]) + magic;
        }
      }
    }
  }
#pragma unroll
  for (int w = 0; w < E / 4; ++w) {
    const uint32_t a = __float_as_uint(f[4 * w]), b = __float_as_uint(f[4 * w + 1]);
    const uint32_t c = __float_as_uint(f[4 * w + 2]), d = __float_as_uint(f[4 * w + 3]);
    m[w] = __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
    ss = __dp4a((int)m[w], (int)m[w], ss);
  }
}
// The stored scale of a row, ss = |m|^2.
__device__ __forceinline__ float int8_stored_scale(uint32_t top, int ss, float eps) {
  // 1 / |m| by one Newton step from the approximate reciprocal root, the product
  // n2 y with its rounding error, so that only the last sum rounds
  const float amax = __uint_as_float(top), n2 = (float)ss, y = rsqrtf(n2);
  const float p = n2 * y, low = fmaf(n2, y, -p);
  float scale = fmaf(0.5f * y, fmaf(-low, y, fmaf(-p, y, 1.0f)), y);
  // |m| >= 127: only a row below eps can meet the other bound, 1 / max(a, b) as
  // min(1 / a, 1 / b)
  if (!(amax >= eps)) scale = top ? fminf(scale, amax / (127.0f * eps)) : 0.f;
  return top < 0x7f800000u ? scale : __uint_as_float(0x7fc00000u);
}
}  // namespace screen
