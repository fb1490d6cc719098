// Rows of an int8 paged cache written and read back, and the accepted path of
// a tree of drafts moved to the positions it keeps.
#include "paged.cuh"
#include "kv_rows.cuh"

namespace screen {
namespace {

// ---------------------------------------------------------------------------
// Append to int8 pages: D / 4 lanes per raw row, blockIdx.y selects K / V.
// Bound by HBM: D * sizeof(T) bytes in, D + 4 out per row.  Consecutive row
// groups walk n (the token) first: the int8 rows and scales of one head are
// contiguous along a page, a raw row is a whole 128-byte line (bf16, D = 64)
// wherever it lies.
// ---------------------------------------------------------------------------
template <typename T, int D>
__global__ void __launch_bounds__(256) append8_kernel(screen_paged_append_args a) {
  pdl_wait();
  pdl_trigger();
  constexpr int G = D / 4;
  constexpr int RPB = 256 / G;
  const long long row = (long long)blockIdx.x * RPB + threadIdx.x / G;
  const int gl = threadIdx.x % G;
  const long long rows = (long long)a.B * a.n_new * a.H;
  const bool valid = row < rows;  // no early exit: the group shuffles need every lane
  const long long rr = valid ? row : 0;
  const long long n = rr % a.n_new;
  const int h = (int)(rr / a.n_new % a.H);
  const int b = (int)(rr / ((long long)a.H * a.n_new));
  const bool isv = blockIdx.y == 1;
  float x[4] = {0.f, 0.f, 0.f, 0.f};
  if (valid)
    load4(reinterpret_cast<const T*>(isv ? a.v : a.k) + (long long)b * (isv ? a.v_sb : a.k_sb) +
              n * (isv ? a.v_st : a.k_st) + (long long)h * D + gl * 4, x);
  const long long dst = valid ? paged_row(a.cache, b, a.H, h, (long long)a.positions[b] + n) : -1;
  write_cache_row<signed char, D>(x, a.eps, gl, dst,
                                  reinterpret_cast<signed char*>(isv ? a.cache.v_pages : a.cache.k_pages),
                                  isv ? a.v_scales : a.k_scales);
}

// ---------------------------------------------------------------------------
// Read back: out (B, n, H, D) contiguous, 4 elements a lane.
// ---------------------------------------------------------------------------
template <typename E>
__device__ __forceinline__ void row4(const E* p, float (&x)[4]) {
  if constexpr (sizeof(E) == 1) {
    const char4 c = *reinterpret_cast<const char4*>(p);
    x[0] = c.x; x[1] = c.y; x[2] = c.z; x[3] = c.w;
  } else {
    load4(p, x);
  }
}
template <typename E, typename T, int D>
__global__ void __launch_bounds__(256) paged_read_kernel(screen_paged_read_args a) {
  pdl_wait();
  pdl_trigger();
  constexpr int G = D / 4;
  constexpr int RPB = 256 / G;
  const long long row = (long long)blockIdx.x * RPB + threadIdx.x / G;
  const int gl = threadIdx.x % G;
  if (row >= (long long)a.B * a.n * a.H) return;
  const long long n = row % a.n;
  const int h = (int)(row / a.n % a.H);
  const int b = (int)(row / ((long long)a.H * a.n));
  const bool isv = blockIdx.y == 1;
  const long long src = paged_row(a.cache, b, a.H, h, (long long)a.positions[b] + n);
  float x[4] = {0.f, 0.f, 0.f, 0.f};
  if (src >= 0) {
    row4(reinterpret_cast<const E*>(isv ? a.cache.v_pages : a.cache.k_pages) + src * D + gl * 4, x);
    if constexpr (sizeof(E) == 1) {
      const float sc = (isv ? a.v_scales : a.k_scales)[src];
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] *= sc;
    }
  }
  T* out = reinterpret_cast<T*>(isv ? a.v : a.k) + (((long long)b * a.n + n) * a.H + h) * D + gl * 4;
  if constexpr (sizeof(T) == 4)
    *reinterpret_cast<float4*>(out) = make_float4(x[0], x[1], x[2], x[3]);
  else
    *reinterpret_cast<uint2*>(out) = make_uint2(pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]));
}

// ---------------------------------------------------------------------------
// Commit: row lens[b] + path[b, i] -> lens[b] + i for i < counts[b], one CTA
// per (layer, K / V, sequence, head).  All source rows are staged in shared
// memory before the first write, so any path is right, and rows that stay
// where they are (a chain's) are not touched.
// ---------------------------------------------------------------------------
__global__ void __launch_bounds__(128) commit_kernel(screen_commit_args a, int row_bytes) {
  pdl_wait();
  pdl_trigger();
  extern __shared__ __align__(16) unsigned char rows_s[];
  __shared__ long long from_s[SCREEN_TREE_MAX_NODES], to_s[SCREEN_TREE_MAX_NODES];
  __shared__ float sc_s[SCREEN_TREE_MAX_NODES];
  const int tid = threadIdx.x;
  const int b = blockIdx.x / a.H, h = blockIdx.x % a.H, layer = blockIdx.y;
  const bool isv = blockIdx.z == 1;
  const long long lens = a.lens[b];
  int count = a.counts[b];
  if (count > a.n) count = a.n;
  if (lens < 0 || count <= 0) return;
  for (int i = tid; i < count; i += 128) {
    const int p = a.path[(long long)b * a.path_sb + i];
    long long from = -1, to = -1;
    if (p >= 0 && p < a.n && p != i) {
      from = paged_row(a.cache, b, a.H, h, lens + p);
      to = paged_row(a.cache, b, a.H, h, lens + i);
      if (from < 0) to = -1;
    }
    from_s[i] = from;
    to_s[i] = to;
  }
  __syncthreads();
  unsigned char* pages = reinterpret_cast<unsigned char*>(isv ? a.cache.v_pages : a.cache.k_pages) +
                         (size_t)layer * a.layer_stride * row_bytes;
  float* scales = isv ? a.v_scales : a.k_scales;
  if (scales) scales += (size_t)layer * a.layer_stride;
  const int chunks = row_bytes / 16;
  for (int c = tid; c < count * chunks; c += 128) {
    const int i = c / chunks;
    if (to_s[i] >= 0)
      reinterpret_cast<uint4*>(rows_s)[c] =
          reinterpret_cast<const uint4*>(pages + from_s[i] * row_bytes)[c - i * chunks];
  }
  if (scales)
    for (int i = tid; i < count; i += 128)
      if (to_s[i] >= 0) sc_s[i] = scales[from_s[i]];
  __syncthreads();
  for (int c = tid; c < count * chunks; c += 128) {
    const int i = c / chunks;
    if (to_s[i] >= 0)
      reinterpret_cast<uint4*>(pages + to_s[i] * row_bytes)[c - i * chunks] =
          reinterpret_cast<uint4*>(rows_s)[c];
  }
  if (scales)
    for (int i = tid; i < count; i += 128)
      if (to_s[i] >= 0) scales[to_s[i]] = sc_s[i];
}

template <typename T, int D>
void launch_append8(const screen_paged_append_args& a, cudaStream_t s) {
  constexpr int RPB = 256 / (D / 4);
  const long long rows = (long long)a.B * a.n_new * a.H;
  launch_pdl(append8_kernel<T, D>, dim3((unsigned)((rows + RPB - 1) / RPB), 2), dim3(256), 0, s, a);
}
template <typename E, typename T, int D>
void launch_read(const screen_paged_read_args& a, cudaStream_t s) {
  constexpr int RPB = 256 / (D / 4);
  const long long rows = (long long)a.B * a.n * a.H;
  launch_pdl(paged_read_kernel<E, T, D>, dim3((unsigned)((rows + RPB - 1) / RPB), 2), dim3(256), 0,
             s, a);
}
template <int D>
void append8_d(const screen_paged_append_args& a, cudaStream_t s) {
  if (a.dtype == SCREEN_F32) launch_append8<float, D>(a, s);
  else launch_append8<__nv_bfloat16, D>(a, s);
}
template <int D>
void read_d(const screen_paged_read_args& a, cudaStream_t s) {
  const bool f32 = a.dtype == SCREEN_F32;
  if (a.cache_dtype == SCREEN_I8) {
    if (f32) launch_read<signed char, float, D>(a, s);
    else launch_read<signed char, __nv_bfloat16, D>(a, s);
  } else if (a.cache_dtype == SCREEN_F32) {
    if (f32) launch_read<float, float, D>(a, s);
    else launch_read<float, __nv_bfloat16, D>(a, s);
  } else {
    if (f32) launch_read<__nv_bfloat16, float, D>(a, s);
    else launch_read<__nv_bfloat16, __nv_bfloat16, D>(a, s);
  }
}

}  // namespace

void paged_append8(const screen_paged_append_args& a, cudaStream_t s) {
  switch (a.D) {
    case 16: append8_d<16>(a, s); break;
    case 32: append8_d<32>(a, s); break;
    case 64: append8_d<64>(a, s); break;
    case 128: append8_d<128>(a, s); break;
  }
}
void paged_read(const screen_paged_read_args& a, cudaStream_t s) {
  switch (a.D) {
    case 16: read_d<16>(a, s); break;
    case 32: read_d<32>(a, s); break;
    case 64: read_d<64>(a, s); break;
    case 128: read_d<128>(a, s); break;
  }
}
void commit(const screen_commit_args& a, cudaStream_t s) {
  const int row_bytes = a.D * (a.cache_dtype == SCREEN_I8 ? 1 : a.cache_dtype == SCREEN_BF16 ? 2 : 4);
  launch_pdl(commit_kernel, dim3(a.B * a.H, a.L, 2), dim3(128), (size_t)a.n * row_bytes, s, a,
             row_bytes);
}

}  // namespace screen
