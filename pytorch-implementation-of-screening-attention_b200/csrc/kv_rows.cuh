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

// The int8 form of a raw row x held by a group of G lanes, 4 elements a lane:
//   m = round_half_even(127 x / max|x|),  scale = 1 / max(|m|, 127 eps / max|x|),
// so scale * m is the unit form of the rounded raw row.  The integers do not
// depend on any order of summation: max|x| is exact, a product that lands
// within 2^-10 of a half is decided in 64 bits (127 x is exact there and a
// correctly rounded quotient cannot cross a half), and |m|^2 <= 128 * 127^2 is
// summed in integers.  A row with an infinity or NaN becomes m = 0, scale NaN.
// All 32 lanes of the warp must call it.
template <int G>
__device__ __forceinline__ void int8_row(const float (&x)[4], float eps, char4& m, float& scale) {
  uint32_t top = 0;
#pragma unroll
  for (int e = 0; e < 4; ++e) top = max(top, __float_as_uint(x[e]) & 0x7fffffffu);
#pragma unroll
  for (int o = G / 2; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o, G));
  const bool finite = top < 0x7f800000u;
  const float amax = __uint_as_float(top);
  // 127 / amax overflows for the smallest rows: those take the 64-bit path
  const bool tiny = amax < 1.0e-30f;
  const float inv = tiny ? 0.f : 127.0f / amax;
  int q[4];
  int ss = 0;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float t = x[e] * inv;
    float f = rintf(t);
    if (tiny || !(fabsf(t - f) < 0.5f - 0x1p-10f))
      f = top && finite ? (float)rint((double)x[e] * 127.0 / (double)amax) : 0.f;
    q[e] = finite ? (int)f : 0;
    ss += q[e] * q[e];
  }
#pragma unroll
  for (int o = G / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o, G);
  // 1 / max(a, b) as min(1 / a, 1 / b): 127 eps / amax overflows for tiny rows
  scale = finite ? fminf(1.0f / sqrtf((float)ss), amax / (127.0f * eps)) : __uint_as_float(0x7fc00000u);
  m = make_char4((signed char)q[0], (signed char)q[1], (signed char)q[2], (signed char)q[3]);
}

// Write the cache form of one raw row (G = D / 4 lanes, 4 elements a lane) at
// row index `row` (< 0: nothing is written; the lanes still take part in the
// shuffles).  E = signed char: int8 row and scale; else the unit row in E with
// the arithmetic of kv_append_kernel.
template <typename E, int D>
__device__ __forceinline__ void write_cache_row(const float (&x)[4], float eps, int gl,
                                                long long row, E* pages, float* scales) {
  constexpr int G = D / 4;
  if constexpr (sizeof(E) == 1) {
    char4 m;
    float sc;
    int8_row<G>(x, eps, m, sc);
    if (row >= 0) {
      *reinterpret_cast<char4*>(pages + row * D + gl * 4) = m;
      if (gl == 0) scales[row] = sc;
    }
  } else {
    float ss = x[0] * x[0] + x[1] * x[1] + x[2] * x[2] + x[3] * x[3];
#pragma unroll
    for (int o = G / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o, G);
    const float nrm = fmaxf(sqrtf(ss), eps);
    if (row >= 0) {
#pragma unroll
      for (int e = 0; e < 4; ++e) pages[row * D + gl * 4 + e] = from_f<E>(x[e] / nrm);
    }
  }
}

}  // namespace screen
