"""Speculative serving on the paged cache: int8 rows, attention for a tree of
drafted tokens, the accepted path kept, and the drafts' verification.

The calls take the cache as tensors -- pages [num_pages, H, page_size, D] of
unit rows, a block table [B, max_blocks] int32, and for int8 pages fp32 scales
[num_pages, H, page_size]; PagedKVCache keeps such tensors per layer and has a
method for each call.  They serve generation and have no backward; every launch
goes to the current stream of the tensors' device and allocates what it needs
from torch, so calls on several streams, or captured into several CUDA graphs,
share nothing.  The reference has no counterpart: its generate() recomputes the
prefix for every token (multiscreen/model.py:131-133).
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib

_PAGE_DTYPES = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16, torch.int8: _lib.I8}
MAX_NODES = _lib.TREE_MAX_NODES


def _same_device(dev, *ts):
    for t in ts:
        if t is not None and t.device != dev:
            raise RuntimeError(f"expected every tensor on {dev}, got one on {t.device}")


def _run(fn, args, dev):
    stream = torch.cuda.current_stream(dev).cuda_stream
    if torch.cuda.current_device() == dev.index:
        _lib._check(fn(ctypes.byref(args), stream))
    else:
        with torch.cuda.device(dev):
            _lib._check(fn(ctypes.byref(args), stream))


def _pages(k_pages, v_pages, block_table, k_scales, v_scales, ndim=4):
    """Checks a cache; returns (descriptor, dtype code, H, D, block table)."""
    _lib._require_cuda(k_pages, v_pages, block_table, k_scales, v_scales)
    _same_device(k_pages.device, v_pages, block_table, k_scales, v_scales)
    code = _PAGE_DTYPES.get(k_pages.dtype)
    if code is None or v_pages.dtype != k_pages.dtype:
        raise TypeError(f"pages are float32, bfloat16 or int8, both alike; got {k_pages.dtype} "
                        f"and {v_pages.dtype}")
    if k_pages.dim() != ndim or v_pages.shape != k_pages.shape:
        raise ValueError(f"k_pages {tuple(k_pages.shape)} and v_pages {tuple(v_pages.shape)}: "
                         "expected two of [num_pages, H, page_size, D]")
    if not (k_pages.is_contiguous() and v_pages.is_contiguous()):
        raise ValueError("pages must be contiguous")
    if (code == _lib.I8) != (k_scales is not None) or (k_scales is None) != (v_scales is None):
        raise ValueError("int8 pages come with k_scales and v_scales, other pages with neither")
    for s in (k_scales, v_scales):
        if s is not None and (s.dtype != torch.float32 or s.shape != k_pages.shape[:-1]
                              or not s.is_contiguous()):
            raise ValueError("scales must be contiguous float32 of the pages' shape without D")
    if block_table.dtype != torch.int32 or block_table.dim() != 2 or not block_table.is_contiguous():
        raise ValueError("block_table must be a contiguous int32 [B, max_blocks]")
    P, H, ps, D = k_pages.shape[-4:]
    desc = _lib.KVCacheDesc(k_pages=k_pages.data_ptr(), v_pages=v_pages.data_ptr(),
                            block_table=block_table.data_ptr(), num_pages=P, page_size=ps,
                            max_blocks=block_table.shape[1])
    return desc, code, H, D


def _per_seq(t, B, dev, name):
    _lib._require_cuda(t)
    _same_device(dev, t)
    if t.dtype != torch.int32 or t.shape != (B,):
        raise ValueError(f"{name} must be int32 of shape ({B},), got {t.dtype} {tuple(t.shape)}")
    return t.contiguous()


def _node_ints(t, B, n, dev, name):
    """An int32 (B, n) tensor with unit stride over n, or None."""
    if t is None:
        return None
    _lib._require_cuda(t)
    _same_device(dev, t)
    if t.dtype != torch.int32 or t.shape != (B, n):
        raise ValueError(f"{name} must be int32 of shape ({B}, {n}), got {t.dtype} {tuple(t.shape)}")
    return t if n == 0 or t.stride(1) == 1 else t.contiguous()


def _head_params(r, w, H, dev):
    _lib._require_cuda(r, w)
    _same_device(dev, r, w)
    if r.shape != (H,) or w.shape != (H,):
        raise ValueError(f"r and w must have shape ({H},)")
    return r.detach().float().contiguous(), w.detach().float().contiguous()


def _rows(x, B, n, H, D, dev, name):
    _lib._require_cuda(x)
    _same_device(dev, x)
    if x.shape != (B, n, H, D):
        raise ValueError(f"{name} must have shape {(B, n, H, D)}, got {tuple(x.shape)}")
    return _lib._bthd(x.detach())


def _table_batch(block_table, B):
    if block_table.shape[0] != B:
        raise ValueError(f"block_table has {block_table.shape[0]} rows for a batch of {B}")


def paged_append(k, v, positions, k_pages, v_pages, block_table, k_scales=None, v_scales=None,
                 eps: float = 1e-8) -> None:
    """Write the unit rows of raw k, v (B, n, H, D) at positions[b] + (0 .. n-1)
    (int32).  int8 pages hold m = round_half_even(127 x / max|x|) and the scale
    1 / max(|m|, 127 eps / max|x|) per row, so that scale * m is a unit row; k, v
    are then float32 or bfloat16, otherwise of the pages' dtype.  Positions
    outside the block table are skipped."""
    desc, code, H, D = _pages(k_pages, v_pages, block_table, k_scales, v_scales)
    dev = k_pages.device
    if k.dim() != 4 or v.dtype != k.dtype:
        raise ValueError("k and v must be (B, n, H, D) of one dtype")
    B, n = k.shape[:2]
    k, v = _rows(k, B, n, H, D, dev, "k"), _rows(v, B, n, H, D, dev, "v")
    positions = _per_seq(positions, B, dev, "positions")
    _table_batch(block_table, B)
    if code != _lib.I8:
        if k.dtype != k_pages.dtype:
            raise TypeError("cache dtype must match k/v")
        a = _lib.KVAppendArgs(dtype=code, B=B, H=H, D=D, n_new=n, eps=float(eps),
                              k=k.data_ptr(), k_sb=k.stride(0), k_st=k.stride(1),
                              v=v.data_ptr(), v_sb=v.stride(0), v_st=v.stride(1),
                              positions=positions.data_ptr(), cache=desc)
        return _run(_lib.load().screen_kv_append, a, dev)
    a = _lib.PagedAppendArgs(dtype=_lib._dtype_code(k), B=B, H=H, D=D, n_new=n, eps=float(eps),
                             k=k.data_ptr(), k_sb=k.stride(0), k_st=k.stride(1),
                             v=v.data_ptr(), v_sb=v.stride(0), v_st=v.stride(1),
                             positions=positions.data_ptr(), cache=desc,
                             k_scales=k_scales.data_ptr(), v_scales=v_scales.data_ptr())
    return _run(_lib.load().screen_paged_append_i8, a, dev)


def paged_read(positions, n: int, k_pages, v_pages, block_table, k_scales=None, v_scales=None,
               dtype: torch.dtype | None = None):
    """(k, v) (B, n, H, D): the values of the cached rows at positions[b] +
    (0 .. n-1), in `dtype` (float32 or bfloat16; default the pages' own, float32
    for int8).  Rows outside the block table are zero."""
    desc, code, H, D = _pages(k_pages, v_pages, block_table, k_scales, v_scales)
    dev = k_pages.device
    B = block_table.shape[0]
    positions = _per_seq(positions, B, dev, "positions")
    if n < 0:
        raise ValueError("n must not be negative")
    if dtype is None:
        dtype = torch.float32 if code == _lib.I8 else k_pages.dtype
    if dtype not in _lib._DTYPES:
        raise TypeError(f"rows are read as float32 or bfloat16, got {dtype}")
    k = torch.empty((B, n, H, D), dtype=dtype, device=dev)
    v = torch.empty_like(k)
    a = _lib.PagedReadArgs(dtype=_lib._DTYPES[dtype], cache_dtype=code, B=B, H=H, D=D, n=int(n),
                           k=k.data_ptr(), v=v.data_ptr(), positions=positions.data_ptr(),
                           cache=desc, k_scales=_lib._ptr(k_scales), v_scales=_lib._ptr(v_scales))
    _run(_lib.load().screen_paged_read, a, dev)
    return k, v


def _tree_ctas(bh: int, keys: int) -> int:
    """CTAs that the 64-key tiles of a call are shared out over, at most (the
    library takes as many as run at once); 1: one for each of the bh (sequence,
    head) pairs, and no second launch."""
    if keys // 64 + 2 <= 8 or bh > 2048:
        return 1
    return 148 * 4


def _tree(fn, q, k, v, lens, parents, r, w, k_pages, v_pages, block_table, k_scales, v_scales,
          max_window, num_ctas, eps):
    desc, code, H, D = _pages(k_pages, v_pages, block_table, k_scales, v_scales)
    dev = k_pages.device
    if q.dim() != 4:
        raise ValueError("q must be (B, n, H, D)")
    B, n = q.shape[:2]
    q = _rows(q, B, n, H, D, dev, "q")
    if code != _lib.I8 and q.dtype != k_pages.dtype:
        raise TypeError(f"q is {q.dtype}, the cache {k_pages.dtype}")
    if n > MAX_NODES:
        raise ValueError(f"a tree has at most {MAX_NODES} nodes, got {n}")
    _table_batch(block_table, B)
    lens = _per_seq(lens, B, dev, "lens")
    parents = _node_ints(parents, B, n, dev, "parents")
    r, w = _head_params(r, w, H, dev)
    if (k is None) != (v is None):
        raise ValueError("k and v are given together")
    y = torch.empty((B, n, H, D), dtype=q.dtype, device=dev)
    if y.numel() == 0:
        return y
    table = block_table.shape[1] * k_pages.shape[2]
    keys = table if not max_window or max_window <= 0 else min(int(-(-max_window // 1)), table)
    ctas = _tree_ctas(B * H, keys + n) if num_ctas is None else int(num_ctas)
    a = _lib.TreeArgs(dtype=_lib._dtype_code(q), cache_dtype=code, B=B, H=H, D=D, n=n,
                      num_ctas=ctas, eps=float(eps),
                      q=q.data_ptr(), q_sb=q.stride(0), q_st=q.stride(1), lens=lens.data_ptr(),
                      r=r.data_ptr(), w=w.data_ptr(), cache=desc, k_scales=_lib._ptr(k_scales),
                      v_scales=_lib._ptr(v_scales), y=y.data_ptr())
    if k is not None:
        k, v = _rows(k, B, n, H, D, dev, "k"), _rows(v, B, n, H, D, dev, "v")
        if k.dtype != q.dtype or v.dtype != q.dtype:
            raise TypeError("q, k, v must share a dtype")
        a.k, a.k_sb, a.k_st = k.data_ptr(), k.stride(0), k.stride(1)
        a.v, a.v_sb, a.v_st = v.data_ptr(), v.stride(0), v.stride(1)
    if parents is not None:
        a.parents, a.parents_sb = parents.data_ptr(), parents.stride(0)
    lib = _lib.load()
    if ctas > 1:
        need = lib.screen_tree_workspace_size(ctypes.byref(a))
        ws = torch.empty(need, dtype=torch.uint8, device=dev)
        a.workspace, a.workspace_bytes = ws.data_ptr(), need
    _run(getattr(lib, fn), a, dev)
    return y


def paged_decode(q, seq_lens, r, w, k_pages, v_pages, block_table, k_scales=None, v_scales=None,
                 max_window=None, num_ctas: int | None = None, eps: float = 1e-8):
    """y (B, H, D) of raw q (B, H, D), the newest cached token of each sequence
    (position seq_lens[b] - 1, int32), over the window's cached keys.
    `max_window` (the largest w) and num_ctas only set how the work is shared out."""
    if q.dim() != 3:
        raise ValueError("q must be (B, H, D)")
    if k_pages.dtype != torch.int8:
        desc, code, H, D = _pages(k_pages, v_pages, block_table, k_scales, v_scales)
        B, dev = q.shape[0], k_pages.device
        if q.shape[1:] != (H, D):
            raise ValueError(f"q must have shape {(B, H, D)}, got {tuple(q.shape)}")
        if q.dtype != k_pages.dtype:
            raise TypeError(f"q is {q.dtype}, the cache {k_pages.dtype}")
        _table_batch(block_table, B)
        _same_device(dev, q)
        seq_lens = _per_seq(seq_lens, B, dev, "seq_lens")
        r, w = _head_params(r, w, H, dev)
        table = block_table.shape[1] * k_pages.shape[2]
        keys = table if not max_window or max_window <= 0 else min(int(-(-max_window // 1)), table)
        if num_ctas is None:
            num_ctas = _tree_ctas(B * H, keys)
        # splits of every (sequence, head), at least a page each
        num_splits = max(1, min(-(-num_ctas // max(1, B * H)), -(-keys // k_pages.shape[2])))
        with torch.cuda.device(dev):
            return _lib.screen_decode(q.detach(), seq_lens, r, w, k_pages, v_pages, block_table,
                                      eps, num_splits)[0]
    return _tree("screen_paged_decode_i8", q.unsqueeze(1), None, None, seq_lens, None, r, w, k_pages,
                 v_pages, block_table, k_scales, v_scales, max_window, num_ctas, eps).squeeze(1)


def paged_tree_decode(q, k, v, lens, parents, r, w, k_pages, v_pages, block_table, k_scales=None,
                      v_scales=None, max_window=None, num_ctas: int | None = None,
                      eps: float = 1e-8):
    """y (B, n, H, D) of a tree of n <= 64 drafted tokens per sequence, from raw
    q, k, v (B, n, H, D).

    lens (B,) int32: cached tokens before the tree (negative: an empty place in
    the batch).  parents (B, n) int32: -1 for a child of the newest cached token,
    else an earlier node; any other value makes the node and its descendants
    absent (y = 0, their cache rows left alone).  None: a chain.  Node i owns
    cache position lens[b] + i, where its unit row is written before it is read
    (k, v None: the rows are there already), and stands at position lens[b] +
    depth: it sees the cached tokens of its window, its ancestors and itself.
    Every path of the tree gives what decoding its tokens one by one gives.  A
    ring table must hold ceil(max w) - 1 + n rows per sequence; nodes whose row
    falls outside the table are not seen.  `max_window` and num_ctas as in
    paged_decode."""
    return _tree("screen_tree_decode", q, k, v, lens, parents, r, w, k_pages, v_pages, block_table,
                 k_scales, v_scales, max_window, num_ctas, eps)


def paged_commit(lens, path, counts, k_pages, v_pages, block_table, k_scales=None,
                 v_scales=None) -> None:
    """Keep an accepted path: row lens[b] + path[b, i] moves to lens[b] + i for
    i < counts[b] (all int32; path (B, n), n <= 64, entries outside [0, n) leave
    their row).  Pages (and scales) may carry a leading layer dimension: all
    layers move in one launch."""
    ndim = k_pages.dim()
    if ndim not in (4, 5):
        raise ValueError("pages must be [num_pages, H, page_size, D], or that per layer")
    desc, code, H, D = _pages(k_pages, v_pages, block_table, k_scales, v_scales, ndim)
    dev = k_pages.device
    B = block_table.shape[0]
    if path.dim() != 2 or path.shape[1] > MAX_NODES:
        raise ValueError(f"path must be (B, n) with n <= {MAX_NODES}")
    n = path.shape[1]
    path = _node_ints(path, B, n, dev, "path")
    lens, counts = _per_seq(lens, B, dev, "lens"), _per_seq(counts, B, dev, "counts")
    L = k_pages.shape[0] if ndim == 5 else 1
    if k_pages.numel() == 0 or n == 0:
        return
    a = _lib.CommitArgs(cache_dtype=code, L=L, B=B, H=H, D=D, n=n, lens=lens.data_ptr(),
                        path=path.data_ptr(), path_sb=path.stride(0), counts=counts.data_ptr(),
                        cache=desc, k_scales=_lib._ptr(k_scales), v_scales=_lib._ptr(v_scales),
                        layer_stride=k_pages.numel() // (L * D))
    _run(_lib.load().screen_paged_commit, a, dev)


def _logit_rows(x, B, n, V, dev, name):
    _lib._require_cuda(x)
    _same_device(dev, x)
    if x.shape != (B, n, V):
        raise ValueError(f"{name} must have shape {(B, n, V)}, got {tuple(x.shape)}")
    x = x.detach()
    if x.dtype == torch.float16:
        x = x.float()
    return x if x.stride(2) == 1 or x.numel() == 0 else x.contiguous()


def verify_drafts(logits, tokens, parents, uniforms, draft_logits=None, temperature=1.0):
    """Speculative sampling: which drafted tokens the target keeps, and one more.

    logits (B, n + 1, V): row 0 follows each sequence's newest token, row 1 + i
    drafted token i.  tokens (B, n) int64, parents (B, n) int32 as in
    paged_tree_decode (None: a chain), uniforms (B, n + 1) float32 in [0, 1).
    draft_logits (B, n, V): row j is the distribution the children of row j were
    drawn from; None: the tokens were picked, not drawn.  temperature: a float,
    or a float32 (B,) tensor; 0 is greedy (the first maximum).

    Nodes are scanned in order, starting at row 0 with c = 0 and Z = 1.  A node
    whose parent is the current row is accepted iff u q(x) Z < p(x) - c q(x), p
    and q the softmaxes of the two rows over the temperature (q(x) = 1 without
    draft_logits), and its row becomes the current one; otherwise c += Z and
    Z = sum max(p - c q, 0) (without draft_logits x leaves p).  Then one token is
    drawn from the residual, the first index whose running sum passes
    uniforms[:, n] Z.  Each returned token is so distributed as the target's.

    Returns (tokens (B, n + 1) int64: accepted, the drawn one, then -1; path
    (B, n) int32: accepted nodes, then -1; counts (B,) int32).  A logits row
    without a finite maximum, or with a NaN, accepts nothing and gives -1; -inf
    entries have probability 0.  float16 logits are read as float32."""
    if logits.dim() != 3 or logits.shape[1] < 1 or logits.shape[2] < 1:
        raise ValueError("logits must be (B, n + 1, V)")
    B, n, V = logits.shape[0], logits.shape[1] - 1, logits.shape[2]
    if n > MAX_NODES:
        raise ValueError(f"a tree has at most {MAX_NODES} nodes, got {n}")
    _lib._require_cuda(logits, tokens, uniforms)
    dev = logits.device
    logits = _logit_rows(logits, B, n + 1, V, dev, "logits")
    if tokens.dtype != torch.int64 or tokens.shape != (B, n):
        raise ValueError(f"tokens must be int64 of shape ({B}, {n})")
    if uniforms.dtype != torch.float32 or uniforms.shape != (B, n + 1):
        raise ValueError(f"uniforms must be float32 of shape ({B}, {n + 1})")
    _same_device(dev, tokens, uniforms)
    parents = _node_ints(parents, B, n, dev, "parents")
    if n and tokens.stride(1) != 1:
        tokens = tokens.contiguous()
    if uniforms.stride(1) != 1:
        uniforms = uniforms.contiguous()
    a = _lib.VerifyArgs(dtype=_lib._dtype_code(logits), B=B, n=n, V=V, logits=logits.data_ptr(),
                        l_sb=logits.stride(0), l_st=logits.stride(1), tokens=tokens.data_ptr(),
                        t_sb=tokens.stride(0), uniforms=uniforms.data_ptr(),
                        u_sb=uniforms.stride(0))
    if isinstance(temperature, torch.Tensor):
        _lib._require_cuda(temperature)
        _same_device(dev, temperature)
        if temperature.dtype != torch.float32 or temperature.shape != (B,):
            raise ValueError(f"temperature must be a float or float32 of shape ({B},)")
        temperature = temperature.contiguous()
        a.temperatures = temperature.data_ptr()
    else:
        temperature = float(temperature)
        if not 0.0 <= temperature < 3.0e38:
            raise ValueError(f"temperature must be finite and not negative, got {temperature}")
        a.temperature = temperature
    if draft_logits is not None and n:
        draft_logits = _logit_rows(draft_logits, B, n, V, dev, "draft_logits")
        if draft_logits.dtype != logits.dtype:
            raise TypeError("logits and draft_logits must share a dtype")
        a.draft_logits, a.d_sb, a.d_st = (draft_logits.data_ptr(), draft_logits.stride(0),
                                          draft_logits.stride(1))
    if parents is not None:
        a.parents, a.p_sb = parents.data_ptr(), parents.stride(0)
    out = torch.empty((B, n + 1), dtype=torch.int64, device=dev)
    path = torch.empty((B, n), dtype=torch.int32, device=dev)
    counts = torch.empty((B,), dtype=torch.int32, device=dev)
    if B == 0:
        return out, path, counts
    a.out_tokens, a.path, a.counts = out.data_ptr(), path.data_ptr(), counts.data_ptr()
    lib = _lib.load()
    need = lib.screen_verify_workspace_size(ctypes.byref(a))
    if need:
        ws = torch.empty(need, dtype=torch.uint8, device=dev)
        a.workspace, a.workspace_bytes = ws.data_ptr(), need
    _run(lib.screen_verify_drafts, a, dev)
    return out, path, counts
