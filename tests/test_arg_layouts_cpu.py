"""The argument structs: the C header's fields against the ctypes mirrors, one by one,
and the bytes that the serving calls pack against the mirrors' fields."""
import ctypes
import re
from pathlib import Path

import pytest
import torch

HEADER = Path(__file__).resolve().parent.parent / "include" / "screening_b200.h"
MIRRORS = {
    "screen_fwd_args": "FwdArgs", "screen_bwd_args": "BwdArgs", "screen_kv_cache": "KVCacheDesc",
    "screen_kv_append_args": "KVAppendArgs", "screen_decode_args": "DecodeArgs",
    "screen_rows_linear_args": "RowsLinearArgs", "screen_xent_args": "XentArgs", "screen_rmsnorm_args": "RmsNormArgs",
    "screen_paged_append_args": "PagedAppendArgs", "screen_paged_read_args": "PagedReadArgs",
    "screen_tree_args": "TreeArgs", "screen_commit_args": "CommitArgs", "screen_verify_args": "VerifyArgs",
}
KINDS = {"int32_t": ctypes.c_int32, "uint32_t": ctypes.c_uint32, "int64_t": ctypes.c_int64, "uint64_t": ctypes.c_uint64,
         "float": ctypes.c_float, "size_t": ctypes.c_size_t}


def fields(text, name):
    """[(field, C type, pointer?)] of a struct of the header."""
    body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (name, name), text, re.S).group(1)
    out = []
    for decl in re.sub(r"/\*.*?\*/", "", body, flags=re.S).split(";"):
        decl = " ".join(decl.split())
        if not decl:
            continue
        kind, names = re.match(r"(?:const )?(\w+)\s?(.*)", decl).groups()
        for n in names.split(","):
            out.append((n.strip(" *"), kind, "*" in n or "* " in n))
    return out


@pytest.mark.parametrize("name", sorted(MIRRORS))
def test_header_and_mirror(ms, name):
    L = ms._lib
    want = []
    for field, kind, pointer in fields(HEADER.read_text(), name):
        want.append((field, ctypes.c_void_p if pointer else getattr(L, MIRRORS[kind]) if kind in MIRRORS else KINDS[kind]))
    assert [(n, t) for n, t in getattr(L, MIRRORS[name])._fields_] == want


def leaves(mirror, base=0):
    for n, t in mirror._fields_:
        at = base + getattr(mirror, n).offset
        if issubclass(t, ctypes.Structure):
            yield from leaves(t, at)
        else:
            yield n, t, at


@pytest.mark.parametrize("name", ["screen_kv_append", "screen_paged_append_i8", "screen_paged_read", "screen_tree_decode",
                                  "screen_paged_decode_i8", "screen_paged_commit", "screen_verify_drafts"])
def test_packed_bytes(ms, name):
    """A value of its own in every argument comes out of the mirror's field."""
    pack, _ = ms.paged._entry(name)
    mirror = ms.paged._STRUCTS[name]
    flat = list(leaves(mirror))
    raw = pack(*[float(i + 1) if t is ctypes.c_float else i + 1 for i, (_, t, _) in enumerate(flat)])
    assert len(raw) == ctypes.sizeof(mirror)
    for i, (n, t, at) in enumerate(flat):
        assert t.from_buffer_copy(raw, at).value == i + 1, n


class Fake(torch.Tensor):
    """A CPU tensor that says it is on a GPU."""

    def get_device(self):
        return 0


def fake(*shape, dtype=torch.float32):
    return torch.zeros(*shape, dtype=dtype).as_subclass(Fake)


@pytest.fixture
def packed(ms, monkeypatch):
    """Calls f() without the launch; its arguments as the mirror `name`."""
    seen = []
    monkeypatch.setattr(ms.paged, "_run", lambda call, args, index: seen.append(args))

    def run(f, name):
        out = f()
        return getattr(ms._lib, name).from_buffer_copy(seen.pop()), out

    return run


B, n, H, D, ps, PAGES, BLOCKS = 2, 3, 4, 16, 8, 5, 6


def cache():
    return [*(fake(PAGES, H, ps, D, dtype=torch.int8) for _ in range(2)), fake(B, BLOCKS, dtype=torch.int32),
            *(fake(PAGES, H, ps) for _ in range(2))]


def check_cache(a, c):
    d = a.cache
    assert [d.k_pages, d.v_pages, d.block_table, a.k_scales, a.v_scales] == [t.data_ptr() for t in c]
    assert (d.num_pages, d.page_size, d.max_blocks) == (PAGES, ps, BLOCKS)


def ints(*shape):
    return fake(*shape, dtype=torch.int32)


def test_tree_and_decode_by_name(ms, packed):
    c = cache()
    q, k, v = (fake(B, n, H, D, dtype=torch.bfloat16) for _ in range(3))
    lens, par, r, w = ints(B), ints(B, n), fake(H), fake(H)
    a, y = packed(lambda: ms.paged_tree_decode(q, k, v, lens, par, r, w, *c, num_ctas=1, eps=0.5), "TreeArgs")
    assert (a.dtype, a.cache_dtype, a.B, a.H, a.D, a.n, a.num_ctas, a.eps) == (ms._lib.BF16, ms._lib.I8, B, H, D, n, 1, 0.5)
    for got, t in ((a.q, q), (a.k, k), (a.v, v), (a.lens, lens), (a.parents, par), (a.r, r), (a.w, w), (a.y, y)):
        assert got == t.data_ptr()
    assert a.q_sb == a.k_sb == a.v_sb == n * H * D and a.q_st == a.k_st == a.v_st == H * D and a.parents_sb == n
    check_cache(a, c)
    one = fake(B, H, D)
    a, y = packed(lambda: ms.paged_decode(one, lens, r, w, *c, num_ctas=1), "TreeArgs")
    assert (a.dtype, a.n, a.q, a.q_sb, a.y, a.k, a.v, a.parents) == (ms._lib.F32, 1, one.data_ptr(), H * D, y.data_ptr(),
                                                                     None, None, None)
    check_cache(a, c)


def test_append_read_and_commit_by_name(ms, packed):
    c = cache()
    k, v, pos = fake(B, n, H, D), fake(B, n, H, D), ints(B)
    a, _ = packed(lambda: ms.paged_append(k, v, pos, *c, eps=0.25), "PagedAppendArgs")
    assert (a.dtype, a.B, a.H, a.D, a.n_new, a.eps) == (ms._lib.F32, B, H, D, n, 0.25)
    assert (a.k, a.v, a.positions) == (k.data_ptr(), v.data_ptr(), pos.data_ptr())
    assert a.k_sb == a.v_sb == n * H * D and a.k_st == a.v_st == H * D
    check_cache(a, c)
    a, (k2, v2) = packed(lambda: ms.paged_read(pos, n, *c, dtype=torch.bfloat16), "PagedReadArgs")
    assert (a.dtype, a.cache_dtype, a.B, a.H, a.D, a.n) == (ms._lib.BF16, ms._lib.I8, B, H, D, n)
    assert (a.k, a.v, a.positions) == (k2.data_ptr(), v2.data_ptr(), pos.data_ptr())
    check_cache(a, c)
    path, counts = ints(B, n), ints(B)
    a, _ = packed(lambda: ms.paged_commit(pos, path, counts, *c), "CommitArgs")
    assert (a.cache_dtype, a.L, a.B, a.H, a.D, a.n, a.path_sb, a.layer_stride) == (ms._lib.I8, 1, B, H, D, n, n, PAGES * H * ps)
    assert (a.lens, a.path, a.counts) == (pos.data_ptr(), path.data_ptr(), counts.data_ptr())
    check_cache(a, c)


def test_verify_by_name(ms, packed):
    # so many rows that none are summed up front: a workspace would need a GPU
    N, V = 40, 20000
    lg, dl, tok = fake(N, n + 1, V), fake(N, n, V), fake(N, n, dtype=torch.int64)
    par, u, temp = ints(N, n), fake(N, n + 1), fake(N)
    a, (out, path, counts) = packed(lambda: ms.verify_drafts(lg, tok, par, u, draft_logits=dl, temperature=temp), "VerifyArgs")
    assert (a.dtype, a.B, a.n, a.V, a.temperature) == (ms._lib.F32, N, n, V, 1.0)
    for got, t in ((a.logits, lg), (a.draft_logits, dl), (a.tokens, tok), (a.parents, par), (a.uniforms, u),
                   (a.temperatures, temp), (a.out_tokens, out), (a.path, path), (a.counts, counts)):
        assert got == t.data_ptr()
    assert (a.l_sb, a.l_st, a.d_sb, a.d_st, a.t_sb, a.p_sb, a.u_sb) == ((n + 1) * V, V, n * V, V, n, n, n + 1)
    assert a.workspace is None
    a, _ = packed(lambda: ms.verify_drafts(lg, tok, None, u, temperature=0.5), "VerifyArgs")
    assert (a.temperature, a.temperatures, a.parents, a.draft_logits) == (0.5, None, None, None)
