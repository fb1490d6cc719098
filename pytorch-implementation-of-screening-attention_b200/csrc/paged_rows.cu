// Rows of an int8 paged cache written and read back, and the accepted path of
// a tree of drafts moved to the positions it keeps.
#include "paged.cuh"
#include "kv_rows.cuh"

namespace screen {
namespace {

// A block moves `tokens` consecutive tokens of one sequence, all heads, K in the
// lower half of the grid, V in the upper.  Heads run fastest through its rows:
// a token's raw rows are one contiguous run of H * D elements, and a few tokens
// make a run of each head's page (walking the tokens of one head first, 128-byte
// rows 6 KB apart, read the packed QKV projection at 0.7 TB/s).  A group of G
// lanes moves a row 16 bytes a lane (of the wider side), R rows of a group with
// all loads in flight before the first use.
constexpr int kThreads = 256;
struct RowBlock {
  int b, n0, rows;       // rows of the block, row r: token n0 + r / H, head r % H
  bool isv;
};
// r / H for r, H < 65536: inv = ceil(2^32 / H)
__device__ __forceinline__ int div_heads(int r, int H, unsigned inv) {
  return H == 1 ? r : (int)__umulhi((unsigned)r, inv);
}
__device__ __forceinline__ RowBlock row_block(int B, int H, int n, int tokens) {
  const unsigned tiles = ((unsigned)n + tokens - 1) / tokens;
  unsigned id = blockIdx.x;
  RowBlock r;
  r.isv = id >= tiles * (unsigned)B;
  if (r.isv) id -= tiles * (unsigned)B;
  r.b = (int)(id / tiles);
  r.n0 = (int)((id - r.b * tiles) * tokens);
  r.rows = min(tokens, n - r.n0) * H;
  return r;
}
// ---------------------------------------------------------------------------
// Append to int8 pages.  D * sizeof(T) bytes in, D + 4 out per row; bound by issue
// before HBM, so two elements go through an instruction where one takes pairs,
// and a token's place in the pages is looked up once for all its heads: 4 x 4097
// tokens of 16 x 64 in bf16 take 29 us (16 us of traffic), 44 without either.
// ---------------------------------------------------------------------------
// The bits of the largest magnitude among the row whose 16-byte parts G lanes hold.
template <typename T, int G>
__device__ __forceinline__ uint32_t row_top(const uint4& u) {
  uint32_t top;
  if constexpr (sizeof(T) == 2) {
    const uint32_t abs = 0x7fff7fffu;
    top = __vmaxu2(__vmaxu2(u.x & abs, u.y & abs), __vmaxu2(u.z & abs, u.w & abs));
#pragma unroll
    for (int o = G / 2; o > 0; o >>= 1) top = __vmaxu2(top, __shfl_xor_sync(0xffffffffu, top, o, G));
    return max(top & 0xffff0000u, top << 16);
  } else {
    const uint32_t abs = 0x7fffffffu;
    top = max(max(u.x & abs, u.y & abs), max(u.z & abs, u.w & abs));
#pragma unroll
    for (int o = G / 2; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o, G));
    return top;
  }
}
template <typename T>
__device__ __forceinline__ void widen(const uint4& u, float (&x)[16 / sizeof(T)]) {
  if constexpr (sizeof(T) == 2) {
    const float2 a = unpack_bf16(u.x), b = unpack_bf16(u.y), c = unpack_bf16(u.z), d = unpack_bf16(u.w);
    x[0] = a.x; x[1] = a.y; x[2] = b.x; x[3] = b.y;
    x[4] = c.x; x[5] = c.y; x[6] = d.x; x[7] = d.y;
  } else {
    x[0] = __uint_as_float(u.x); x[1] = __uint_as_float(u.y);
    x[2] = __uint_as_float(u.z); x[3] = __uint_as_float(u.w);
  }
}
template <typename T, int D, int R>
__global__ void __launch_bounds__(kThreads) append8_kernel(screen_paged_append_args a, int tokens,
                                                                unsigned inv_heads) {
  constexpr int E = 16 / (int)sizeof(T), G = D / E, GROUPS = kThreads / G;
  __shared__ long long base[R * GROUPS];   // row of head 0 per token of the block, -1 none
  pdl_wait();
  pdl_trigger();
  const RowBlock rb = row_block(a.B, a.H, a.n_new, tokens);
  const int gl = threadIdx.x % G, grp = threadIdx.x / G;
  const long long sb = rb.isv ? a.v_sb : a.k_sb, st = rb.isv ? a.v_st : a.k_st;
  const T* src = reinterpret_cast<const T*>(rb.isv ? a.v : a.k) + (long long)rb.b * sb + rb.n0 * st + gl * E;
  const int* table = a.cache.block_table + (long long)rb.b * a.cache.max_blocks;
  const long long pos0 = (long long)a.positions[rb.b] + rb.n0;
  signed char* pages = reinterpret_cast<signed char*>(rb.isv ? a.cache.v_pages : a.cache.k_pages) + gl * E;
  float* scales = rb.isv ? a.v_scales : a.k_scales;
  for (int t = threadIdx.x; t < tokens; t += kThreads) base[t] = table_row(a.cache, table, a.H, 0, pos0 + t);
#pragma unroll 1
  for (int r0 = 0; r0 < rb.rows; r0 += R * GROUPS) {   // uniform: the shuffles need every lane
    uint4 u[R];
    int t[R], h[R];
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const int r = r0 + i * GROUPS + grp;
      u[i] = make_uint4(0u, 0u, 0u, 0u);
      t[i] = -1;
      if (r < rb.rows) {
        t[i] = div_heads(r, a.H, inv_heads);
        h[i] = r - t[i] * a.H;
        u[i] = *reinterpret_cast<const uint4*>(src + t[i] * st + h[i] * D);
      }
    }
    if (r0 == 0) __syncthreads();
#pragma unroll
    for (int i = 0; i < R; ++i) {
      float x[E];
      uint32_t m[E / 4];
      const uint32_t top = row_top<T, G>(u[i]);
      widen<T>(u[i], x);
      int ss = 0;
      int8_pack<E, sizeof(T) == 2>(x, int8_scale<sizeof(T) == 2>(top), m, ss);
#pragma unroll
      for (int o = G / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o, G);
      long long row = t[i] < 0 ? -1 : base[t[i]];
      if (row >= 0) {
        row += (long long)h[i] * a.cache.page_size;
        signed char* dst = pages + row * D;
        if constexpr (E == 8) *reinterpret_cast<uint2*>(dst) = make_uint2(m[0], m[1]);
        else *reinterpret_cast<uint32_t*>(dst) = m[0];
        if (gl == 0) scales[row] = int8_stored_scale(top, ss, a.eps);
      }
    }
  }
}

// ---------------------------------------------------------------------------
// Read back: out (B, n, H, D) contiguous, 16 bytes of it a lane.  Bound by HBM: 4 x
// 4097 tokens of 16 x 64 in fp32 take 30 us (26 us of traffic).
// ---------------------------------------------------------------------------
template <typename E, int N>
__device__ __forceinline__ void row_n(const E* p, float (&x)[N]) {
  if constexpr (sizeof(E) == 1) {
#pragma unroll
    for (int w = 0; w < N / 4; ++w) {
      const char4 c = *reinterpret_cast<const char4*>(p + 4 * w);
      x[4 * w] = c.x; x[4 * w + 1] = c.y; x[4 * w + 2] = c.z; x[4 * w + 3] = c.w;
    }
  } else {
#pragma unroll
    for (int w = 0; w < N / 4; ++w) {
      float y[4];
      load4(p + 4 * w, y);
#pragma unroll
      for (int e = 0; e < 4; ++e) x[4 * w + e] = y[e];
    }
  }
}
template <typename E, typename T, int D, int R>
__global__ void __launch_bounds__(kThreads) paged_read_kernel(screen_paged_read_args a, int tokens,
                                                                   unsigned inv_heads) {
  pdl_wait();
  pdl_trigger();
  constexpr int N = 16 / (int)sizeof(T), G = D / N, GROUPS = kThreads / G;
  const RowBlock rb = row_block(a.B, a.H, a.n, tokens);
  const int gl = threadIdx.x % G, grp = threadIdx.x / G;
  const int* table = a.cache.block_table + (long long)rb.b * a.cache.max_blocks;
  const long long pos0 = a.positions[rb.b];
  const E* pages = reinterpret_cast<const E*>(rb.isv ? a.cache.v_pages : a.cache.k_pages);
  const float* scales = rb.isv ? a.v_scales : a.k_scales;
  T* out = reinterpret_cast<T*>(rb.isv ? a.v : a.k) + ((long long)rb.b * a.n + rb.n0) * a.H * D + gl * N;
#pragma unroll 1
  for (int r0 = grp; r0 < rb.rows; r0 += R * GROUPS) {
    float x[R][N], sc[R];
    long long row[R];
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const int r = r0 + i * GROUPS;
      row[i] = -1;
      if (r < rb.rows) {
        const int t = div_heads(r, a.H, inv_heads);
        row[i] = table_row(a.cache, table, a.H, r - t * a.H, pos0 + rb.n0 + t);
      }
    }
#pragma unroll
    for (int i = 0; i < R; ++i) {
#pragma unroll
      for (int e = 0; e < N; ++e) x[i][e] = 0.f;
      sc[i] = 1.f;
      if (row[i] >= 0) {
        row_n(pages + row[i] * D + gl * N, x[i]);
        if constexpr (sizeof(E) == 1) sc[i] = scales[row[i]];
      }
    }
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const int r = r0 + i * GROUPS;
      if (r >= rb.rows) continue;
      if constexpr (sizeof(E) == 1)
#pragma unroll
        for (int e = 0; e < N; ++e) x[i][e] *= sc[i];
      T* dst = out + (long long)r * D;
      if constexpr (sizeof(T) == 4)
        *reinterpret_cast<float4*>(dst) = make_float4(x[i][0], x[i][1], x[i][2], x[i][3]);
      else
        *reinterpret_cast<uint4*>(dst) = make_uint4(pack_bf16(x[i][0], x[i][1]), pack_bf16(x[i][2], x[i][3]),
                                                    pack_bf16(x[i][4], x[i][5]), pack_bf16(x[i][6], x[i][7]));
    }
  }
}

// ---------------------------------------------------------------------------
// Commit: row lens[b] + path[b, i] -> lens[b] + i for i < counts[b], one CTA
// per (layer, K / V, sequence, head).  All source rows are staged in shared
// memory before the first write, so any path is right, and rows that stay
// where they are (a chain's) are not touched.  Bound by latency: lengths, path, table
// and rows one after another, 3.6 us for 12 layers of a tree of 16 on bf16 pages, 8.1
// us for 64 rows of 8 x 16 heads on int8 pages (2 us of traffic; 1.7 times as many
// CTAs as are resident at once).
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

// Tokens of a block: as many as its groups hold at R rows each.
struct RowGrid {
  int tokens;
  unsigned blocks, inv_heads;
};
RowGrid row_grid(int B, int H, int n, int rows) {
  RowGrid g;
  g.tokens = rows > H ? rows / H : 1;
  g.inv_heads = (unsigned)(((1ull << 32) + H - 1) / H);
  g.blocks = 2u * B * (unsigned)((n + g.tokens - 1) / g.tokens);
  return g;
}
template <typename T, int D>
void launch_append8(const screen_paged_append_args& a, cudaStream_t s) {
  constexpr int R = 4, GROUPS = kThreads / (D * (int)sizeof(T) / 16);
  const RowGrid g = row_grid(a.B, a.H, a.n_new, R * GROUPS);
  launch_pdl(append8_kernel<T, D, R>, dim3(g.blocks), dim3(kThreads), 0, s, a, g.tokens,
             g.inv_heads);
}
template <typename E, typename T, int D>
void launch_read(const screen_paged_read_args& a, cudaStream_t s) {
  constexpr int R = 4, GROUPS = kThreads / (D * (int)sizeof(T) / 16);
  const RowGrid g = row_grid(a.B, a.H, a.n, R * GROUPS);
  launch_pdl(paged_read_kernel<E, T, D, R>, dim3(g.blocks), dim3(kThreads), 0, s, a, g.tokens,
             g.inv_heads);
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
