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
import math
import struct

import torch

from . import _lib

_PAGE_DTYPES = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16, torch.int8: _lib.I8}
MAX_NODES = _lib.TREE_MAX_NODES

# A call's arguments are packed straight into the bytes of its C struct
# (include/screening_b200.h; native alignment) in the order of the struct's ctypes
# mirror: building the mirror field by field cost as much as the shortest of these
# kernels runs.
_STRUCTS = {
    "screen_kv_append": _lib.KVAppendArgs,
    "screen_paged_append_i8": _lib.PagedAppendArgs,
    "screen_paged_read": _lib.PagedReadArgs,
    "screen_tree_decode": _lib.TreeArgs,
    "screen_paged_decode_i8": _lib.TreeArgs,
    "screen_paged_commit": _lib.CommitArgs,
    "screen_verify_drafts": _lib.VerifyArgs,
}
_CODES = {ctypes.c_int32: "i", ctypes.c_int64: "q", ctypes.c_float: "f", ctypes.c_void_p: "P",
          ctypes.c_size_t: "N"}
_entries = {}


def _layout(mirror) -> str:
    """The fields of a ctypes struct as struct codes, those of nested structs in line."""
    return "".join(_layout(t) if issubclass(t, ctypes.Structure) else _CODES[t]
                   for _, t in mirror._fields_)


def _entry(name):
    """(pack, call) of a C entry point."""
    e = _entries.get(name)
    if e is None:
        lib = _lib.load()
        mirror = _STRUCTS[name]
        st = struct.Struct(_layout(mirror) + "0q")
        if st.size != ctypes.sizeof(mirror):
            raise RuntimeError(f"{name}: packed arguments differ from {mirror.__name__}")
        proto = ctypes.CFUNCTYPE(ctypes.c_int, ctypes.c_char_p, ctypes.c_void_p)
        e = _entries[name] = (st.pack, proto(ctypes.cast(getattr(lib, name), ctypes.c_void_p).value))
    return e


def _size_query(name):
    """A workspace size query on packed arguments."""
    q = _entries.get(name)
    if q is None:
        proto = ctypes.CFUNCTYPE(ctypes.c_size_t, ctypes.c_char_p)
        q = _entries[name] = proto(ctypes.cast(getattr(_lib.load(), name), ctypes.c_void_p).value)
    return q


_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda index: torch.cuda.current_stream(index).cuda_stream)


def _run(call, args, index):
    """The call on the current stream of CUDA device `index`."""
    if torch.cuda.current_device() == index:
        status = call(args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            status = call(args, _raw_stream(index))
    if status:
        _lib._check(status)


def _same_device(index, *ts):
    for t in ts:
        if t is not None and t.get_device() != index:
            _lib._require_cuda(t)
            raise RuntimeError(f"expected every tensor on cuda:{index}, got one on {t.device}")


def _pages(k_pages, v_pages, block_table, k_scales, v_scales, ndim=4):
    """Checks a cache; returns (device index, dtype code, shape, its packed
    arguments (pages, table, sizes), the scales' pointers)."""
    index = k_pages.get_device()
    if index < 0:
        _lib._require_cuda(k_pages)
    _same_device(index, v_pages, block_table, k_scales, v_scales)
    dtype, shape = k_pages.dtype, k_pages.shape
    code = _PAGE_DTYPES.get(dtype)
    if code is None or v_pages.dtype is not dtype:
        raise TypeError(f"pages are float32, bfloat16 or int8, both alike; got {k_pages.dtype} "
                        f"and {v_pages.dtype}")
    if len(shape) != ndim or v_pages.shape != shape:
        raise ValueError(f"k_pages {tuple(k_pages.shape)} and v_pages {tuple(v_pages.shape)}: "
                         "expected two of [num_pages, H, page_size, D]")
    if not (k_pages.is_contiguous() and v_pages.is_contiguous()):
        raise ValueError("pages must be contiguous")
    if (code == _lib.I8) != (k_scales is not None) or (k_scales is None) != (v_scales is None):
        raise ValueError("int8 pages come with k_scales and v_scales, other pages with neither")
    scales = (0, 0)
    if k_scales is not None:
        for s in (k_scales, v_scales):
            if s.dtype is not torch.float32 or s.shape != shape[:-1] or not s.is_contiguous():
                raise ValueError("scales must be contiguous float32 of the pages' shape without D")
        scales = (k_scales.data_ptr(), v_scales.data_ptr())
    if block_table.dtype is not torch.int32 or block_table.dim() != 2 or not block_table.is_contiguous():
        raise ValueError("block_table must be a contiguous int32 [B, max_blocks]")
    P, H, ps, D = shape[-4:]
    return index, code, shape, (k_pages.data_ptr(), v_pages.data_ptr(), block_table.data_ptr(), P, ps,
                                block_table.shape[1], 0), scales


def _per_seq(t, B, index, name):
    if t.get_device() != index:
        _same_device(index, t)
    if t.dtype is not torch.int32 or t.shape != (B,):
        raise ValueError(f"{name} must be int32 of shape ({B},), got {t.dtype} {tuple(t.shape)}")
    return t if t.is_contiguous() else t.contiguous()


def _node_ints(t, B, n, index, name):
    """An int32 (B, n) tensor with unit stride over n, or None."""
    if t is None:
        return None
    if t.get_device() != index:
        _same_device(index, t)
    if t.dtype is not torch.int32 or t.shape != (B, n):
        raise ValueError(f"{name} must be int32 of shape ({B}, {n}), got {t.dtype} {tuple(t.shape)}")
    return t if n == 0 or t.stride(1) == 1 else t.contiguous()


def _head_params(r, w, H, index):
    _same_device(index, r, w)
    if r.shape != (H,) or w.shape != (H,):
        raise ValueError(f"r and w must have shape ({H},)")
    if r.dtype is not torch.float32 or not r.is_contiguous():
        r = r.detach().float().contiguous()
    if w.dtype is not torch.float32 or not w.is_contiguous():
        w = w.detach().float().contiguous()
    return r, w


def _rows(x, shape, index, name):
    """(tensor to keep, pointer, batch stride, row stride) of raw rows the
    kernels read in place where their layout allows it."""
    if x.get_device() != index:
        _same_device(index, x)
    if x.shape != shape:
        raise ValueError(f"{name} must have shape {tuple(shape)}, got {tuple(x.shape)}")
    sb, st, sh, sd = x.stride()
    vec = 8 if x.dtype is torch.bfloat16 else 4
    p = x.data_ptr()
    if sd != 1 or sh != shape[3] or sb % vec or st % vec or p % 16:
        # a copy even where torch counts x as contiguous: it may start anywhere
        x = x.detach().clone(memory_format=torch.contiguous_format)
        sb, st, _, _ = x.stride()
        p = x.data_ptr()
    return x, p, sb, st


def _like(x, shape):
    """A contiguous tensor of `shape`, which is x's (empty_like keeps x's order of
    strides; it is the cheapest allocation there is)."""
    y = torch.empty_like(x)
    return y if y.is_contiguous() else x.new_empty(shape)


def _table_batch(block_table, B):
    if block_table.shape[0] != B:
        raise ValueError(f"block_table has {block_table.shape[0]} rows for a batch of {B}")


def paged_append(k, v, positions, k_pages, v_pages, block_table, k_scales=None, v_scales=None,
                 eps: float = 1e-8) -> None:
    """Write the unit rows of raw k, v (B, n, H, D) at positions[b] + (0 .. n-1)
    (int32).  int8 pages hold m = round_half_even(127 x / max|x|) and the scale
    1 / max(|m|, 127 eps / max|x|) per row, so that scale * m is a unit row; k, v
    are then float32 or bfloat16, otherwise of the pages' dtype.  Positions
    outside the block table are skipped.  The rows of one call have to lie on
    different rows of the pages: of a ring table, n is at most the ring's rows."""
    index, code, shape, cache, scales = _pages(k_pages, v_pages, block_table, k_scales, v_scales)
    if k.dim() != 4 or v.dtype is not k.dtype:
        raise ValueError("k and v must be (B, n, H, D) of one dtype")
    B, n = k.shape[:2]
    H, D = shape[1], shape[3]
    k, kp, k_sb, k_st = _rows(k, (B, n, H, D), index, "k")
    v, vp, v_sb, v_st = _rows(v, (B, n, H, D), index, "v")
    positions = _per_seq(positions, B, index, "positions")
    _table_batch(block_table, B)
    if code == _lib.I8:
        pack, call = _entry("screen_paged_append_i8")
        _run(call, pack(_lib._dtype_code(k), B, H, D, n, eps, kp, k_sb, k_st, vp, v_sb, v_st,
                        positions.data_ptr(), *cache, *scales), index)
        return
    if k.dtype is not k_pages.dtype:
        raise TypeError("cache dtype must match k/v")
    pack, call = _entry("screen_kv_append")
    _run(call, pack(code, B, H, D, n, eps, kp, k_sb, k_st, vp, v_sb, v_st, positions.data_ptr(),
                    *cache), index)


def paged_read(positions, n: int, k_pages, v_pages, block_table, k_scales=None, v_scales=None,
               dtype: torch.dtype | None = None):
    """(k, v) (B, n, H, D): the values of the cached rows at positions[b] +
    (0 .. n-1), in `dtype` (float32 or bfloat16; default the pages' own, float32
    for int8).  Rows outside the block table are zero."""
    index, code, shape, cache, scales = _pages(k_pages, v_pages, block_table, k_scales, v_scales)
    B, H, D = block_table.shape[0], shape[1], shape[3]
    positions = _per_seq(positions, B, index, "positions")
    if n < 0:
        raise ValueError("n must not be negative")
    if dtype is None:
        dtype = torch.float32 if code == _lib.I8 else k_pages.dtype
    if dtype not in _lib._DTYPES:
        raise TypeError(f"rows are read as float32 or bfloat16, got {dtype}")
    k = torch.empty((B, n, H, D), dtype=dtype, device=k_pages.device)
    v = torch.empty_like(k)
    pack, call = _entry("screen_paged_read")
    _run(call, pack(_lib._DTYPES[dtype], code, B, H, D, int(n), k.data_ptr(), v.data_ptr(),
                    positions.data_ptr(), *cache, *scales), index)
    return k, v


_MAX_CTAS = 148 * 4          # of a tree call that are resident at once, at most


def _tree_ctas(bh: int, keys: int) -> int:
    """CTAs that the 64-key tiles of a call are shared out over, at most (the
    library takes as many as run at once); 1: one for each of the bh (sequence,
    head) pairs, and no second launch.  From as many pairs as resident CTAs on the
    library takes one each in any case."""
    if keys // 64 + 2 <= 8 or bh >= _MAX_CTAS:
        return 1
    return _MAX_CTAS


def _keys_seen(max_window, block_table, page_size):
    table = block_table.shape[1] * page_size
    return math.ceil(max_window) if max_window and 0 < max_window < table else table


def decode_splits(pairs: int, keys: int, page_size: int) -> int:
    """Splits per (sequence, head) of a decode over fp32 / bf16 pages: runs of whole
    pages, at least one wave of CTAs (148 SMs x 3 resident decode CTAs), and about
    sqrt(pages) for long windows -- measured at 32K and 100K keys per window, fewer
    leave a wave tail, more pay the per-CTA pipeline fill (4 x 16 heads of 64 over 100K
    bf16 keys, windows from a quarter on: 185 us with 43 splits, 262 with 10).  Windows of up to 512 keys
    (the w <= 256 of a model at init) take one, which applies TanhNorm itself: a
    finishing launch costs more than the few pages it would spread."""
    if keys <= 512:
        return 1
    pages = math.ceil(keys / page_size)
    fill = math.ceil(148 * 3 / max(1, pairs))
    return max(1, min(256, pages, max(fill, round(1.1 * math.sqrt(pages)))))


def _tree(name, q, k, v, lens, parents, r, w, k_pages, v_pages, block_table, k_scales, v_scales,
          max_window, num_ctas, eps):
    """q, k, v (B, n, H, D); or q (B, H, D), one query per sequence."""
    index, code, shape, cache, scales = _pages(k_pages, v_pages, block_table, k_scales, v_scales)
    H, D = shape[1], shape[3]
    if q.dim() == 3:
        B, n = q.shape[0], 1
        full = (B, H, D)
        if q.get_device() != index:
            _same_device(index, q)
        if q.shape != full:
            raise ValueError(f"q must have shape {full}, got {tuple(q.shape)}")
        q_sb, sh, sd = q.stride()
        if sd != 1 or sh != D or q_sb % (8 if q.dtype is torch.bfloat16 else 4) or q.data_ptr() % 16:
            q = q.detach().clone(memory_format=torch.contiguous_format)
            q_sb = H * D
        qp, q_st = q.data_ptr(), 0
    else:
        B, n = q.shape[:2]
        full = (B, n, H, D)
        q, qp, q_sb, q_st = _rows(q, full, index, "q")
    dtype = q.dtype
    if code != _lib.I8 and dtype is not k_pages.dtype:
        raise TypeError(f"q is {q.dtype}, the cache {k_pages.dtype}")
    if n > MAX_NODES:
        raise ValueError(f"a tree has at most {MAX_NODES} nodes, got {n}")
    _table_batch(block_table, B)
    lens = _per_seq(lens, B, index, "lens")
    parents = _node_ints(parents, B, n, index, "parents")
    r, w = _head_params(r, w, H, index)
    kp = k_sb = k_st = vp = v_sb = v_st = 0
    if (k is None) != (v is None):
        raise ValueError("k and v are given together")
    if k is not None:
        if k.dtype is not dtype or v.dtype is not dtype:
            raise TypeError("q, k, v must share a dtype")
        k, kp, k_sb, k_st = _rows(k, full, index, "k")
        v, vp, v_sb, v_st = _rows(v, full, index, "v")
    y = _like(q, full)
    dcode = _lib._dtype_code(q)
    if B * n * H == 0:
        return y
    if num_ctas is None:
        num_ctas = _tree_ctas(B * H, _keys_seen(max_window, block_table, shape[2]) + n)
    pack, call = _entry(name)
    pp, p_sb = (0, 0) if parents is None else (parents.data_ptr(), parents.stride(0))
    args = (dcode, code, B, H, D, n, int(num_ctas), eps, qp, q_sb, q_st, kp, k_sb, k_st, vp, v_sb,
            v_st, lens.data_ptr(), pp, p_sb, r.data_ptr(), w.data_ptr(), *cache, *scales,
            y.data_ptr())
    if num_ctas > 1:
        need = _size_query("screen_tree_workspace_size")(pack(*args, 0, 0))
        ws = torch.UntypedStorage(need, device=q.device) if need else None
        _run(call, pack(*args, ws.data_ptr() if need else 0, need), index)
    else:
        _run(call, pack(*args, 0, 0), index)
    return y


def paged_decode(q, seq_lens, r, w, k_pages, v_pages, block_table, k_scales=None, v_scales=None,
                 max_window=None, num_ctas: int | None = None, eps: float = 1e-8):
    """y (B, H, D) of raw q (B, H, D), the newest cached token of each sequence
    (position seq_lens[b] - 1, int32), over the window's cached keys.
    `max_window` (the largest w) and num_ctas only set how the work is shared out."""
    if q.dim() != 3:
        raise ValueError("q must be (B, H, D)")
    if k_pages.dtype is not torch.int8:
        index, code, shape, _, _ = _pages(k_pages, v_pages, block_table, k_scales, v_scales)
        B, H, D = q.shape[0], shape[1], shape[3]
        if q.shape[1:] != (H, D):
            raise ValueError(f"q must have shape {(B, H, D)}, got {tuple(q.shape)}")
        if q.dtype is not k_pages.dtype:
            raise TypeError(f"q is {q.dtype}, the cache {k_pages.dtype}")
        _table_batch(block_table, B)
        _same_device(index, q)
        seq_lens = _per_seq(seq_lens, B, index, "seq_lens")
        r, w = _head_params(r, w, H, index)
        keys = _keys_seen(max_window, block_table, shape[2])
        if num_ctas is None:
            num_splits = decode_splits(B * H, keys, shape[2])
        else:                    # of every (sequence, head), at least a page each
            num_splits = max(1, min(-(-num_ctas // max(1, B * H)), -(-keys // shape[2])))
        with torch.cuda.device(index):
            return _lib.screen_decode(q.detach(), seq_lens, r, w, k_pages, v_pages, block_table,
                                      eps, num_splits)[0]
    return _tree("screen_paged_decode_i8", q, None, None, seq_lens, None, r, w, k_pages, v_pages,
                 block_table, k_scales, v_scales, max_window, num_ctas, eps)


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
    if q.dim() != 4:
        raise ValueError("q must be (B, n, H, D)")
    return _tree("screen_tree_decode", q, k, v, lens, parents, r, w, k_pages, v_pages, block_table,
                 k_scales, v_scales, max_window, num_ctas, eps)


def tree_depths(parents):
    """Depth (B, n) int64 of every node of parents (B, n): 0 below the newest cached
    token.  Absent nodes have a depth without meaning."""
    p = parents.long()
    B, n = p.shape
    p = torch.where((p >= 0) & (p < torch.arange(n, device=p.device)), p, -1)
    depth = (p >= 0).long()
    hop = 1
    while hop < n:                        # pointer doubling
        at = p.clamp_min(0)
        inner = p >= 0
        depth = depth + torch.where(inner, depth.gather(1, at), 0)
        p = torch.where(inner, p.gather(1, at), -1)
        hop *= 2
    return depth


def paged_commit(lens, path, counts, k_pages, v_pages, block_table, k_scales=None,
                 v_scales=None) -> None:
    """Keep an accepted path: row lens[b] + path[b, i] moves to lens[b] + i for
    i < counts[b] (all int32; path (B, n), n <= 64, entries outside [0, n) leave
    their row).  Pages (and scales) may carry a leading layer dimension: all
    layers move in one launch."""
    ndim = k_pages.dim()
    if ndim not in (4, 5):
        raise ValueError("pages must be [num_pages, H, page_size, D], or that per layer")
    index, code, shape, cache, scales = _pages(k_pages, v_pages, block_table, k_scales, v_scales, ndim)
    B = block_table.shape[0]
    if path.dim() != 2 or path.shape[1] > MAX_NODES:
        raise ValueError(f"path must be (B, n) with n <= {MAX_NODES}")
    n = path.shape[1]
    path = _node_ints(path, B, n, index, "path")
    lens, counts = _per_seq(lens, B, index, "lens"), _per_seq(counts, B, index, "counts")
    P, H, ps, D = shape[-4:]
    L = shape[0] if ndim == 5 else 1
    if L * P * H * ps * D == 0 or n == 0:
        return
    pack, call = _entry("screen_paged_commit")
    _run(call, pack(code, L, B, H, D, n, lens.data_ptr(), path.data_ptr(), path.stride(0),
                    counts.data_ptr(), *cache, *scales, P * H * ps), index)


def _logit_rows(x, shape, index, name):
    _same_device(index, x)
    if x.shape != shape:
        raise ValueError(f"{name} must have shape {tuple(shape)}, got {tuple(x.shape)}")
    if x.dtype is torch.float16:
        x = x.detach().float()
    return x if x.stride(2) == 1 or x.numel() == 0 else x.detach().contiguous()


def verify_drafts(logits, tokens, parents, uniforms, draft_logits=None, temperature=1.0):
    """Speculative sampling: which drafted tokens the target keeps, and one more.

    logits (B, n + 1, V): row 0 follows each sequence's newest token, row 1 + i
    drafted token i.  tokens (B, n) int64, parents (B, n) int32 as in
    paged_tree_decode (None: a chain), uniforms (B, n + 1) float32 in [0, 1).
    draft_logits (B, n, V): row j is the distribution the children of row j were
    drawn from; None: the tokens were picked, not drawn.  temperature: a finite
    float that is not negative, or a float32 (B,) tensor; 0 is greedy (the first
    maximum), above 1e30 counts as 1e30.  A sequence whose entry is negative or NaN
    has no distribution.

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
    B, rows, V = logits.shape
    n = rows - 1
    if n > MAX_NODES:
        raise ValueError(f"a tree has at most {MAX_NODES} nodes, got {n}")
    index = logits.get_device()
    if index < 0:
        _lib._require_cuda(logits)
    logits = _logit_rows(logits, (B, rows, V), index, "logits")
    if tokens.dtype is not torch.int64 or tokens.shape != (B, n):
        raise ValueError(f"tokens must be int64 of shape ({B}, {n})")
    if uniforms.dtype is not torch.float32 or uniforms.shape != (B, rows):
        raise ValueError(f"uniforms must be float32 of shape ({B}, {rows})")
    _same_device(index, tokens, uniforms)
    parents = _node_ints(parents, B, n, index, "parents")
    if n and tokens.stride(1) != 1:
        tokens = tokens.contiguous()
    if uniforms.stride(1) != 1:
        uniforms = uniforms.contiguous()
    tp = 0
    if isinstance(temperature, torch.Tensor):
        _same_device(index, temperature)
        if temperature.dtype is not torch.float32 or temperature.shape != (B,):
            raise ValueError(f"temperature must be a float or float32 of shape ({B},)")
        temps = temperature.contiguous()
        tp, temperature = temps.data_ptr(), 1.0
    else:
        temperature = float(temperature)
        if not 0.0 <= temperature < 3.0e38:
            raise ValueError(f"temperature must be finite and not negative, got {temperature}")
    dp = d_sb = d_st = 0
    if draft_logits is not None and n:
        draft_logits = _logit_rows(draft_logits, (B, n, V), index, "draft_logits")
        if draft_logits.dtype is not logits.dtype:
            raise TypeError("logits and draft_logits must share a dtype")
        dp, (d_sb, d_st, _) = draft_logits.data_ptr(), draft_logits.stride()
    dcode = _lib._dtype_code(logits)
    out = torch.empty_like(uniforms, dtype=torch.int64)
    if not out.is_contiguous():
        out = uniforms.new_empty((B, rows), dtype=torch.int64)
    path = torch.empty((B, n), dtype=torch.int32, device=logits.device)
    counts = torch.empty(B, dtype=torch.int32, device=logits.device)
    if B == 0:
        return out, path, counts
    pack, call = _entry("screen_verify_drafts")
    l_sb, l_st, _ = logits.stride()
    pp, p_sb = (0, 0) if parents is None else (parents.data_ptr(), parents.stride(0))
    args = (dcode, B, n, V, temperature, 0, tp, logits.data_ptr(), l_sb, l_st, dp, d_sb, d_st,
            tokens.data_ptr() if n else 0, tokens.stride(0), pp, p_sb, uniforms.data_ptr(),
            uniforms.stride(0), out.data_ptr(), path.data_ptr(), counts.data_ptr())
    need = _size_query("screen_verify_workspace_size")(pack(*args, 0, 0))
    ws = torch.UntypedStorage(need, device=logits.device) if need else None
    _run(call, pack(*args, ws.data_ptr() if need else 0, need), index)
    return out, path, counts
