// extern "C" entry points of speculative serving on the paged cache:
// validation and dispatch; no allocation, no exceptions across the boundary.
#include "paged.cuh"

using namespace screen;

namespace {

bool dim_ok(int D) { return D == 16 || D == 32 || D == 64 || D == 128; }
bool act_ok(int t) { return t == SCREEN_F32 || t == SCREEN_BF16; }
bool al16(const void* p) { return ((uintptr_t)p & 15u) == 0; }
bool al4(const void* p) { return ((uintptr_t)p & 3u) == 0; }
bool raw_ok(const void* p, int64_t sb, int64_t st, int vec = 4) {
  return al16(p) && sb % vec == 0 && st % vec == 0;
}
// 2 B blocks of tokens in one grid dimension, a token a block at least; a block's
// rows in 32 bits
bool blocks_ok(long long B, long long H, long long n) {
  return H < 65536 && 2 * B * n < (1ll << 31);
}
size_t round_up(size_t x) { return (x + 255) & ~(size_t)255; }

int cache_ok(const screen_kv_cache& c, int cache_dtype, const float* ks, const float* vs) {
  if (!c.k_pages || !c.v_pages || !c.block_table || c.page_size <= 0 || c.max_blocks <= 0 ||
      c.num_pages < 0)
    return SCREEN_ERR_INVALID_ARG;
  if (cache_dtype == SCREEN_I8 && (!ks || !vs)) return SCREEN_ERR_INVALID_ARG;
  if (!al16(c.k_pages) || !al16(c.v_pages) || !al4(ks) || !al4(vs)) return SCREEN_ERR_ALIGNMENT;
  return SCREEN_OK;
}
// floats of the tree workspace before the partial sums: two ints per segment
long long part_off(const screen_tree_args* a) { return ((long long)a->B * a->H * 2 + 3) & ~3ll; }

int tree_checks(const screen_tree_args* a) {
  if (!act_ok(a->dtype)) return SCREEN_ERR_DTYPE;
  if (a->cache_dtype != a->dtype && a->cache_dtype != SCREEN_I8) return SCREEN_ERR_DTYPE;
  if (!dim_ok(a->D)) return SCREEN_ERR_HEAD_DIM;
  if (a->B < 0 || a->H < 0 || a->n < 0 || a->n > SCREEN_TREE_MAX_NODES || a->num_ctas < 1 ||
      a->num_ctas > 65535)
    return SCREEN_ERR_INVALID_ARG;
  return SCREEN_OK;
}
int tree_run(const screen_tree_args* a, int lens_off, cudaStream_t s) {
  if ((long long)a->B * a->H * a->n == 0) return SCREEN_OK;
  if (!a->q || !a->lens || !a->r || !a->w || !a->y || (!a->k) != (!a->v))
    return SCREEN_ERR_INVALID_ARG;
  if ((long long)a->B * a->H > (1 << 28)) return SCREEN_ERR_UNSUPPORTED;
  int st = cache_ok(a->cache, a->cache_dtype, a->k_scales, a->v_scales);
  if (st) return st;
  if (!raw_ok(a->q, a->q_sb, a->q_st) || !al16(a->y)) return SCREEN_ERR_ALIGNMENT;
  if (a->k && (!raw_ok(a->k, a->k_sb, a->k_st) || !raw_ok(a->v, a->v_sb, a->v_st)))
    return SCREEN_ERR_ALIGNMENT;
  const size_t need = screen_tree_workspace_size(a);
  if (need && (!a->workspace || a->workspace_bytes < need)) return SCREEN_ERR_WORKSPACE;
  if (need && !al16(a->workspace)) return SCREEN_ERR_ALIGNMENT;
  TreeParams p{*a, lens_off, (int)part_off(a)};
  if (!need) p.a.num_ctas = 1;   // nobody to share with
  bool shared;
  float* part = reinterpret_cast<float*>(a->workspace);
  if (a->cache_dtype == SCREEN_I8) {
    shared = a->dtype == SCREEN_F32 ? tree_i8_f32(p, part, s) : tree_i8(p, part, s);
  } else {
    shared = a->dtype == SCREEN_F32 ? tree_f32(p, part, s) : tree_bf16(p, part, s);
  }
  st = check_launch();
  if (st || !shared) return st;
  tree_finish(p, part, s);
  return check_launch();
}

}  // namespace

extern "C" {

int screen_paged_append_i8(const screen_paged_append_args* a, screen_stream_t stream) {
  if (!a) return SCREEN_ERR_INVALID_ARG;
  if (!act_ok(a->dtype)) return SCREEN_ERR_DTYPE;
  if (!dim_ok(a->D)) return SCREEN_ERR_HEAD_DIM;
  if (a->B < 0 || a->H < 0 || a->n_new < 0) return SCREEN_ERR_INVALID_ARG;
  if ((long long)a->B * a->H * a->n_new == 0) return SCREEN_OK;
  if (!a->k || !a->v || !a->positions) return SCREEN_ERR_INVALID_ARG;
  int st = cache_ok(a->cache, SCREEN_I8, a->k_scales, a->v_scales);
  if (st) return st;
  const int vec = a->dtype == SCREEN_BF16 ? 8 : 4;
  if (!raw_ok(a->k, a->k_sb, a->k_st, vec) || !raw_ok(a->v, a->v_sb, a->v_st, vec))
    return SCREEN_ERR_ALIGNMENT;
  if (!blocks_ok(a->B, a->H, a->n_new)) return SCREEN_ERR_UNSUPPORTED;
  paged_append8(*a, (cudaStream_t)stream);
  return check_launch();
}

int screen_paged_read(const screen_paged_read_args* a, screen_stream_t stream) {
  if (!a) return SCREEN_ERR_INVALID_ARG;
  if (!act_ok(a->dtype) || (!act_ok(a->cache_dtype) && a->cache_dtype != SCREEN_I8))
    return SCREEN_ERR_DTYPE;
  if (!dim_ok(a->D)) return SCREEN_ERR_HEAD_DIM;
  if (a->B < 0 || a->H < 0 || a->n < 0) return SCREEN_ERR_INVALID_ARG;
  if ((long long)a->B * a->H * a->n == 0) return SCREEN_OK;
  if (!a->k || !a->v || !a->positions) return SCREEN_ERR_INVALID_ARG;
  int st = cache_ok(a->cache, a->cache_dtype, a->k_scales, a->v_scales);
  if (st) return st;
  if (!al16(a->k) || !al16(a->v)) return SCREEN_ERR_ALIGNMENT;
  if (!blocks_ok(a->B, a->H, a->n)) return SCREEN_ERR_UNSUPPORTED;
  paged_read(*a, (cudaStream_t)stream);
  return check_launch();
}

size_t screen_tree_workspace_size(const screen_tree_args* a) {
  if (!a || tree_checks(a)) return 0;
  // as many segments as CTAs: one each, and no sums to join
  const long long segs = (long long)a->B * a->H;
  if (segs >= a->num_ctas || segs >= kTreeMaxCtas) return 0;
  return round_up((part_off(a) + (size_t)a->num_ctas * a->n * a->D) * sizeof(float));
}

int screen_tree_decode(const screen_tree_args* a, screen_stream_t stream) {
  if (!a) return SCREEN_ERR_INVALID_ARG;
  int st = tree_checks(a);
  if (st) return st;
  return tree_run(a, 0, (cudaStream_t)stream);
}

int screen_paged_decode_i8(const screen_tree_args* a, screen_stream_t stream) {
  if (!a) return SCREEN_ERR_INVALID_ARG;
  int st = tree_checks(a);
  if (st) return st;
  if (a->cache_dtype != SCREEN_I8) return SCREEN_ERR_DTYPE;
  if (a->n != 1 || a->k || a->v || a->parents) return SCREEN_ERR_INVALID_ARG;
  return tree_run(a, -1, (cudaStream_t)stream);
}

int screen_paged_commit(const screen_commit_args* a, screen_stream_t stream) {
  if (!a) return SCREEN_ERR_INVALID_ARG;
  if (!act_ok(a->cache_dtype) && a->cache_dtype != SCREEN_I8) return SCREEN_ERR_DTYPE;
  if (!dim_ok(a->D)) return SCREEN_ERR_HEAD_DIM;
  if (a->L < 0 || a->B < 0 || a->H < 0 || a->n < 0 || a->n > SCREEN_TREE_MAX_NODES ||
      a->layer_stride < 0)
    return SCREEN_ERR_INVALID_ARG;
  if ((long long)a->L * a->B * a->H * a->n == 0) return SCREEN_OK;
  if (!a->lens || !a->path || !a->counts) return SCREEN_ERR_INVALID_ARG;
  if (a->L > 65535 || (long long)a->B * a->H > (1 << 28)) return SCREEN_ERR_UNSUPPORTED;
  int st = cache_ok(a->cache, a->cache_dtype, a->k_scales, a->v_scales);
  if (st) return st;
  commit(*a, (cudaStream_t)stream);
  return check_launch();
}

size_t screen_verify_workspace_size(const screen_verify_args* a) {
  if (!a || a->B <= 0 || a->n < 0 || a->V < 1) return 0;
  return round_up(verify_workspace(*a));
}

int screen_verify_drafts(const screen_verify_args* a, screen_stream_t stream) {
  if (!a) return SCREEN_ERR_INVALID_ARG;
  if (!act_ok(a->dtype)) return SCREEN_ERR_DTYPE;
  if (a->B < 0 || a->n < 0 || a->n > SCREEN_TREE_MAX_NODES || a->V < 1 || a->V > (1 << 30) ||
      !(a->temperature >= 0.f) || a->temperature > 3.0e38f)
    return SCREEN_ERR_INVALID_ARG;
  if (a->B == 0) return SCREEN_OK;
  if (!a->logits || !a->uniforms || !a->out_tokens || !a->counts ||
      (a->n > 0 && (!a->tokens || !a->path)))
    return SCREEN_ERR_INVALID_ARG;
  if (a->B > (1 << 24)) return SCREEN_ERR_UNSUPPORTED;
  const size_t need = screen_verify_workspace_size(a);
  if (need && (!a->workspace || a->workspace_bytes < need)) return SCREEN_ERR_WORKSPACE;
  if (need && !al16(a->workspace)) return SCREEN_ERR_ALIGNMENT;
  verify(*a, (cudaStream_t)stream);
  return check_launch();
}

}  // extern "C"
