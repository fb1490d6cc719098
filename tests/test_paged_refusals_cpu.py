"""Refusals of the speculative-serving calls: status codes of the C entry
points before anything touches the device, and the Python checks that need no
GPU."""
import ctypes

import pytest
import torch


def desc(L, **kw):
    base = dict(k_pages=256, v_pages=512, block_table=1024, num_pages=4, page_size=16, max_blocks=2)
    base.update(kw)
    return L.KVCacheDesc(**base)


def call(L, name, a):
    return getattr(L.load(), name)(ctypes.byref(a), None)


def test_struct_sizes(ms):
    L = ms._lib
    lib = L.load()
    for i, st in enumerate((L.PagedAppendArgs, L.PagedReadArgs, L.TreeArgs, L.CommitArgs, L.VerifyArgs), 16):
        assert lib.screen_sizeof_args(i) == ctypes.sizeof(st), st.__name__
    assert lib.screen_sizeof_args(15) == -1 and lib.screen_sizeof_args(21) == -1
    for f in ("screen_paged_append_i8", "screen_paged_read", "screen_tree_decode", "screen_paged_decode_i8",
              "screen_paged_commit", "screen_verify_drafts"):
        assert getattr(lib, f)(None, None) == -1
    assert lib.screen_tree_workspace_size(None) == 0


def test_append_and_read_codes(ms):
    L = ms._lib
    ok = dict(dtype=L.BF16, B=1, H=1, D=64, n_new=1, eps=1e-8, k=16, k_sb=64, k_st=64, v=32, v_sb=64, v_st=64,
              positions=64, k_scales=128, v_scales=128)
    for bad, code in ((dict(dtype=2), -3), (dict(D=48), -2), (dict(B=-1), -1), (dict(n_new=-1), -1), (dict(k=None), -1),
                      (dict(positions=None), -1), (dict(k_scales=None), -1), (dict(k=8), -4), (dict(v_st=3), -4),
                      (dict(cache=desc(L, page_size=0)), -1), (dict(cache=desc(L, k_pages=None)), -1),
                      (dict(cache=desc(L, v_pages=520)), -4), (dict(n_new=0), 0), (dict(B=0), 0)):
        assert call(L, "screen_paged_append_i8", L.PagedAppendArgs(**{**ok, "cache": desc(L), **bad})) == code, bad
    ok = dict(dtype=L.F32, cache_dtype=L.I8, B=1, H=1, D=64, n=1, k=16, v=32, positions=64, k_scales=128, v_scales=128)
    for bad, code in ((dict(dtype=2), -3), (dict(cache_dtype=3), -3), (dict(D=24), -2), (dict(n=-1), -1),
                      (dict(v=None), -1), (dict(v_scales=None), -1), (dict(k=4), -4), (dict(n=0), 0)):
        assert call(L, "screen_paged_read", L.PagedReadArgs(**{**ok, "cache": desc(L), **bad})) == code, bad


def test_tree_codes(ms):
    L = ms._lib
    ok = dict(dtype=L.BF16, cache_dtype=L.BF16, B=1, H=1, D=64, n=2, num_ctas=1, eps=1e-8, q=16, q_sb=64, q_st=64,
              k=16, k_sb=64, k_st=64, v=32, v_sb=64, v_st=64, lens=64, r=64, w=64, y=128)
    for bad, code in ((dict(dtype=2), -3), (dict(cache_dtype=L.F32), -3), (dict(D=20), -2), (dict(n=65), -1),
                      (dict(n=-1), -1), (dict(num_ctas=0), -1), (dict(lens=None), -1), (dict(v=None), -1),
                      (dict(cache_dtype=L.I8), -1), (dict(q=24), -4), (dict(k_st=2), -4), (dict(y=136), -4),
                      (dict(num_ctas=2), -5), (dict(num_ctas=2, workspace=256, workspace_bytes=16), -5),
                      (dict(num_ctas=70000), -1), (dict(n=0), 0), (dict(B=0), 0)):
        assert call(L, "screen_tree_decode", L.TreeArgs(**{**ok, "cache": desc(L), **bad})) == code, bad
    one = {**ok, "cache": desc(L), "n": 1, "k": None, "v": None, "cache_dtype": L.I8, "k_scales": 64, "v_scales": 64}
    for bad, code in ((dict(cache_dtype=L.BF16), -3), (dict(n=2), -1), (dict(k=16, v=16), -1), (dict(parents=64), -1),
                      (dict(B=0), 0)):
        assert call(L, "screen_paged_decode_i8", L.TreeArgs(**{**one, **bad})) == code, bad
    a = L.TreeArgs(**{**ok, "cache": desc(L), "num_ctas": 3})
    assert L.load().screen_tree_workspace_size(ctypes.byref(a)) >= 3 * 2 * 64 * 4


def test_commit_and_verify_codes(ms):
    L = ms._lib
    ok = dict(cache_dtype=L.BF16, L=1, B=1, H=1, D=64, n=4, lens=64, path=64, path_sb=4, counts=64, layer_stride=64)
    for bad, code in ((dict(cache_dtype=5), -3), (dict(D=63), -2), (dict(n=65), -1), (dict(L=-1), -1),
                      (dict(path=None), -1), (dict(layer_stride=-1), -1), (dict(cache_dtype=L.I8), -1),
                      (dict(L=70000), -9), (dict(L=0), 0), (dict(n=0), 0)):
        assert call(L, "screen_paged_commit", L.CommitArgs(**{**ok, "cache": desc(L), **bad})) == code, bad
    ok = dict(dtype=L.F32, B=1, n=2, V=10, temperature=1.0, logits=16, l_sb=30, l_st=10, tokens=64, t_sb=2, uniforms=64,
              u_sb=3, out_tokens=64, path=64, counts=64, workspace=256, workspace_bytes=4096)
    for bad, code in ((dict(dtype=2), -3), (dict(n=65), -1), (dict(n=-1), -1), (dict(V=0), -1),
                      (dict(temperature=-1.0), -1), (dict(temperature=float("nan")), -1),
                      (dict(temperature=float("inf")), -1), (dict(logits=None), -1), (dict(tokens=None), -1),
                      (dict(path=None), -1), (dict(workspace=None), -5), (dict(workspace_bytes=1), -5),
                      (dict(workspace=264), -4), (dict(B=0), 0)):
        assert call(L, "screen_verify_drafts", L.VerifyArgs(**{**ok, **bad})) == code, bad


def test_cpu_tensors_are_refused(ms):
    kp = torch.zeros(2, 1, 16, 64)
    table = torch.zeros(1, 2, dtype=torch.int32)
    i1, q = torch.zeros(1, dtype=torch.int32), torch.zeros(1, 2, 1, 64)
    r = torch.ones(1)
    for f in (lambda: ms.paged_append(q, q, i1, kp, kp, table), lambda: ms.paged_read(i1, 1, kp, kp, table),
              lambda: ms.paged_decode(q[:, 0], i1, r, r, kp, kp, table),
              lambda: ms.paged_tree_decode(q, q, q, i1, None, r, r, kp, kp, table),
              lambda: ms.paged_commit(i1, torch.zeros(1, 2, dtype=torch.int32), i1, kp, kp, table),
              lambda: ms.verify_drafts(torch.zeros(1, 2, 5), torch.zeros(1, 1, dtype=torch.long), None,
                                       torch.zeros(1, 2))):
        with pytest.raises(RuntimeError, match="CUDA"):
            f()
    with pytest.raises(ValueError):
        ms.verify_drafts(torch.zeros(2, 5), None, None, None)
    with pytest.raises(ValueError):
        ms.verify_drafts(torch.zeros(1, 66, 5), None, None, None)
    with pytest.raises(ValueError):
        ms.paged_decode(q, i1, r, r, kp, kp, table)
    with pytest.raises(ValueError):
        ms.paged_commit(i1, i1, i1, kp[0], kp[0], table)
