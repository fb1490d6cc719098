"""Attention for a tree of drafted tokens over the paged cache, and the commit
of its accepted path, against the 64-bit restatement."""
import math

import pytest
import torch

from oracle import paged_oracle as po
from tests.test_paged_int8_gpu import bound

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


def make(ms, B, H, D, ps, T, n, dtype, q8, seed, blocks=None, ring=None):
    g = torch.Generator().manual_seed(seed)
    blocks = blocks or (T + n) // ps + 1
    per = ring or blocks
    table = torch.randperm(B * per, generator=g).view(B, per)[:, torch.arange(blocks) % per]
    table = table.to(torch.int32).contiguous().to(DEV)
    pd = torch.int8 if q8 else dtype
    kp = torch.zeros(B * per, H, ps, D, dtype=pd, device=DEV)
    vp = torch.zeros_like(kp)
    ks = torch.zeros(B * per, H, ps, device=DEV) if q8 else None
    vs = torch.zeros_like(ks) if q8 else None
    mean = 0.7 * torch.randn(H, D, generator=g)
    k = (torch.randn(B, T + n, H, D, generator=g) + mean).to(dtype)
    v = torch.randn(B, T + n, H, D, generator=g).to(dtype)
    if T:
        keep = min(T, per * ps)
        ms.paged_append(k[:, T - keep:T].to(DEV), v[:, T - keep:T].to(DEV),
                        torch.full((B,), T - keep, dtype=torch.int32, device=DEV), kp, vp, table, ks, vs)
    q = (k[:, T - 1:T] if T else k[:, :1]) + 0.8 * torch.randn(B, n, H, D, generator=g)
    return dict(kp=kp, vp=vp, ks=ks, vs=vs, table=table, q=q.to(dtype), k=k[:, T:], v=v[:, T:], g=g)


def tree_parents(B, n, kind, g):
    if kind == "chain":
        return None
    if kind == "star":
        return torch.full((B, n), -1, dtype=torch.int32)
    p = torch.stack([torch.stack([torch.randint(-1, max(i, 1), (), generator=g) if i else torch.tensor(-1)
                                  for i in range(n)]) for _ in range(B)]).to(torch.int32)
    if kind == "ragged":            # absent nodes, and with them their descendants
        p[0, n // 2:] = -2
        if n > 3:
            p[-1, 2] = 5
            p[-1, 1] = -9
    return p


def check(ms, c, lens, parents, r, w, dtype, q8, **kw):
    B, n, H, D = c["q"].shape
    dev = [None if x is None else x.to(DEV) for x in (c["q"], c["k"], c["v"], lens, parents, r, w)]
    prefix = [None if x is None else x.cpu().clone() for x in (c["kp"], c["vp"], c["ks"], c["vs"], c["table"])]
    y = ms.paged_tree_decode(*dev, c["kp"], c["vp"], c["table"], c["ks"], c["vs"], **kw)
    for b in range(B):
        lines = po.ancestors(None if parents is None else parents[b], n)
        here = [i for i in range(n) if lines[i] and lens[b] >= 0]
        # the nodes' rows as the cache holds them now, each within its rounding
        held = [po.cache_values(c[x + "p"], c[x + "s"], c["table"], b, [int(lens[b]) + i for i in range(n)])
                for x in "kv"]
        for x, got in zip("kv", held):
            if q8:
                m, sc = po.int8_rows(c[x][b])
                row, tol = m.double() * sc[..., None], 2.0**-21
            else:
                row, tol = po.unit_rows(c[x][b]), 2.0**-21 + (2.0**-8 if dtype == torch.bfloat16 else 0.0)
            assert ((got - row)[here].abs() <= tol * row[here].abs() + 1e-12).all()
        want, sums = po.tree(c["q"][b], held[0], held[1], int(lens[b]), parents, r, w, tuple(prefix), b)
        err = (y[b].double().cpu() - want).norm(dim=-1)
        lim = bound(want, sums, r, dtype, q8)
        assert (err <= lim).all(), (b, float((err - lim).max()))
        for i in range(n):
            if not lines[i]:
                assert (y[b, i] == 0).all()
    return y


SHAPES = [(1, 1, 64, 64, 0, 1), (2, 2, 64, 64, 5, 1), (2, 2, 64, 64, 130, 5), (3, 2, 64, 16, 200, 16),
          (2, 3, 16, 8, 61, 17), (2, 2, 32, 24, 150, 33), (1, 2, 128, 100, 260, 64), (2, 2, 64, 64, 300, 64),
          (1, 2, 128, 64, 90, 20), (1, 2, 64, 64, 64, 31), (1, 1, 32, 16, 1, 64), (1, 2, 16, 64, 90, 40)]


@pytest.mark.parametrize("kind", ["chain", "random", "ragged"])
@pytest.mark.parametrize("dtype,q8", [(torch.bfloat16, False), (torch.bfloat16, True),
                                      (torch.float32, False), (torch.float32, True)])
@pytest.mark.parametrize("B,H,D,ps,T,n", SHAPES)
def test_tree(ms, B, H, D, ps, T, n, dtype, q8, kind):
    c = make(ms, B, H, D, ps, T, n, dtype, q8, 31 * n + T)
    lens = torch.tensor([max(0, T - 3 * b) for b in range(B)], dtype=torch.int32)
    r, w = torch.linspace(1.05, 1.8, H), torch.linspace(T + 30.0, max(3.5, T / 5), H)
    check(ms, c, lens, tree_parents(B, n, kind, c["g"]), r, w, dtype, q8)


@pytest.mark.parametrize("dtype,q8", [(torch.bfloat16, False), (torch.bfloat16, True),
                                      (torch.float32, False), (torch.float32, True)])
@pytest.mark.parametrize("ctas", [1, 2, 7, 40])
def test_ctas_agree(ms, dtype, q8, ctas):
    """Any number of CTAs, and any hint of the window, gives the same rows to
    the order of the sums; twice the same call gives the same bits."""
    c = make(ms, 2, 2, 64, 16, 500, 9, dtype, q8, 5)
    lens = torch.tensor([500, 444], dtype=torch.int32)
    parents = tree_parents(2, 9, "random", c["g"])
    r, w = torch.tensor([1.1, 1.4]), torch.tensor([600.0, 90.0])
    y = check(ms, c, lens, parents, r, w, dtype, q8, num_ctas=ctas, max_window=3)
    z = check(ms, c, lens, parents, r, w, dtype, q8, num_ctas=ctas, max_window=3)
    assert torch.equal(y, z)


@pytest.mark.parametrize("dtype,q8", [(torch.bfloat16, False), (torch.bfloat16, True), (torch.float32, False)])
def test_paths_equal_tokens_one_by_one(ms, dtype, q8):
    """A chain of drafts gives what single-token steps give, and leaves the same
    cache behind, over a ring that wraps."""
    B, H, D, ps, T, n = 2, 2, 64, 16, 90, 7
    w = torch.tensor([40.0, 12.5])
    per = math.ceil((40 + n) / ps) + 1
    r = torch.tensor([1.1, 1.5])
    a = make(ms, B, H, D, ps, T, n, dtype, q8, 9, ring=per)
    b = make(ms, B, H, D, ps, T, n, dtype, q8, 9, ring=per)
    lens = torch.full((B,), T, dtype=torch.int32, device=DEV)
    args = (r.to(DEV), w.to(DEV))
    y = ms.paged_tree_decode(a["q"].to(DEV), a["k"].to(DEV), a["v"].to(DEV), lens, None, *args,
                             a["kp"], a["vp"], a["table"], a["ks"], a["vs"])
    for i in range(n):
        ms.paged_append(b["k"][:, i:i + 1].to(DEV), b["v"][:, i:i + 1].to(DEV), lens + i, b["kp"], b["vp"],
                        b["table"], b["ks"], b["vs"])
        z = ms.paged_decode(b["q"][:, i].to(DEV), lens + i + 1, *args, b["kp"], b["vp"], b["table"],
                            b["ks"], b["vs"])
        # bf16: both sides round the output (2^-8 each); the tree also rounds alpha
        # (2^-8 of sums with little cancellation here)
        tol = 2.0**-6 if dtype == torch.bfloat16 else 2.0**-17
        assert ((y[:, i] - z).float().norm(dim=-1) <= tol * z.float().norm(dim=-1) + 1e-6).all(), i
    for x in ("kp", "vp", "ks", "vs"):
        if a[x] is not None:
            assert torch.equal(a[x], b[x])


@pytest.mark.parametrize("dtype,q8", [(torch.bfloat16, False), (torch.bfloat16, True), (torch.float32, False)])
def test_non_finite_rows_stay_where_they_are_seen(ms, dtype, q8):
    B, H, D, ps, T, n = 1, 2, 64, 16, 70, 6
    c = make(ms, B, H, D, ps, T, n, dtype, q8, 12)
    parents = torch.tensor([[-1, 0, 0, 1, 2, -1]], dtype=torch.int32, device=DEV)
    lens = torch.full((1,), T, dtype=torch.int32, device=DEV)
    r, w = torch.full((H,), 1.01, device=DEV), torch.full((H,), 60.0, device=DEV)
    q, k, v = (c[x].to(DEV) for x in "qkv")
    q, k = q.abs() + 0.1, k.abs() + 0.1             # every pair is over the trim

    def run(v, k=k, q=q):
        return ms.paged_tree_decode(q, k, v, lens, parents, r, w, c["kp"], c["vp"], c["table"], c["ks"], c["vs"])

    good = run(v)
    assert good.isfinite().all()
    for bad in (math.nan, math.inf, -math.inf):
        vv = v.clone()
        vv[0, 1, 0, 3] = bad                         # node 1, head 0: seen by nodes 1 and 3
        y = run(vv)
        assert y[0, [1, 3], 0].isnan().all()
        keep = torch.ones(n, H, dtype=torch.bool)
        keep[[1, 3], 0] = False
        assert torch.equal(y[0][keep], good[0][keep])
    kk = k.clone()
    kk[0, 2, 1, 0] = math.nan                        # a key that is not seen by anyone
    y = run(v, k=kk)
    assert y.isfinite().all() and torch.equal(y[0, :, 0], good[0, :, 0])
    assert torch.equal(y[0, [0, 1, 3, 5], 1], good[0, [0, 1, 3, 5], 1])
    qq = q.clone()
    qq[0, 4] = math.nan                              # a query that sees nothing
    y = run(v, q=qq)
    assert (y[0, 4] == 0).all() and torch.equal(y[0, :4], good[0, :4])


@pytest.mark.parametrize("dtype,q8", [(torch.bfloat16, False), (torch.bfloat16, True), (torch.float32, False)])
def test_absent_nodes_and_empty_places_write_nothing(ms, dtype, q8):
    B, H, D, ps, T, n = 3, 2, 64, 16, 40, 8
    c = make(ms, B, H, D, ps, T, n, dtype, q8, 21)
    parents = torch.tensor([[-1, 0, -2, 2, 1, -1, 9, 6]] * B, dtype=torch.int32, device=DEV)
    lens = torch.tensor([T, -1, T - 7], dtype=torch.int32, device=DEV)
    k = c["k"].to(DEV)
    k[:, 2] = math.nan
    before = [None if c[x] is None else c[x].clone() for x in ("kp", "vp", "ks", "vs")]
    r, w = torch.full((H,), 1.2, device=DEV), torch.full((H,), 30.0, device=DEV)
    y = ms.paged_tree_decode(c["q"].to(DEV), k, c["v"].to(DEV), lens, parents, r, w, c["kp"], c["vp"], c["table"],
                             c["ks"], c["vs"])
    assert (y[1] == 0).all() and (y[:, [2, 3, 6, 7]] == 0).all() and y.isfinite().all()
    wrote = {(b, i) for b, l in ((0, T), (2, T - 7)) for i in (0, 1, 4, 5)}
    allowed = torch.zeros(c["kp"].shape[0], ps, dtype=torch.bool)
    for b, i in wrote:
        p = int(lens[b]) + i
        allowed[int(c["table"][b, p // ps]), p % ps] = True
    for x, old in zip(("kp", "vp"), before):
        diff = (c[x] != old).any(-1).any(1).cpu()
        assert not (diff & ~allowed).any() and diff.any()


def test_nodes_past_the_table_are_not_seen(ms):
    c = make(ms, 1, 2, 64, 16, 30, 6, torch.bfloat16, False, 2, blocks=2)
    lens = torch.full((1,), 30, dtype=torch.int32, device=DEV)       # rows 32 .. 35 have no place
    r, w = torch.full((2,), 1.05, device=DEV), torch.full((2,), 64.0, device=DEV)
    y = ms.paged_tree_decode(c["q"].to(DEV), c["k"].to(DEV), c["v"].to(DEV), lens, None, r, w, c["kp"], c["vp"],
                             c["table"])
    assert y.isfinite().all() and (y[0, :2] != 0).any()


@pytest.mark.parametrize("dtype,q8", [(torch.bfloat16, False), (torch.bfloat16, True),
                                      (torch.float32, False), (torch.float32, True)])
@pytest.mark.parametrize("n", [3, 13, 20, 40])
def test_windows_of_nothing_or_of_one_token(ms, n, dtype, q8):
    """w <= 0 or NaN: nothing is seen, y = 0; 0 < w <= 1: the node alone."""
    c = make(ms, 2, 6, 64, 16, 100, n, dtype, q8, n)
    w = torch.tensor([0.0, -5.0, math.nan, 1e-40, 0.3, 1.0])
    r = torch.full((6,), 1.2)
    lens = torch.tensor([100, 70], dtype=torch.int32)
    y = check(ms, c, lens, tree_parents(2, n, "random", c["g"]), r, w, dtype, q8)
    assert (y[:, :, :3] == 0).all()


@pytest.mark.parametrize("dtype,q8", [(torch.bfloat16, False), (torch.bfloat16, True),
                                      (torch.float32, False), (torch.float32, True)])
@pytest.mark.parametrize("n,ctas", [(2, 1), (12, 6), (30, 1)])
def test_negative_acceptance(ms, n, ctas, dtype, q8):
    """r < 0 prefers unlike keys, alpha up to (1 + 2 |r|)^2; one-hot V rows, whose
    int8 scale 1 / 127 is the largest there is."""
    c = make(ms, 2, 3, 64, 16, 150, n, dtype, q8, 3 * n)
    if q8:
        c["vp"].zero_()
        c["vp"][..., 5] = 127
        c["vs"].fill_(1.0 / 127.0)
    lens = torch.tensor([150, 90], dtype=torch.int32)
    check(ms, c, lens, None, torch.tensor([-1.0, -7.5, -0.2]), torch.tensor([200.0, 70.0, 33.0]), dtype, q8,
          num_ctas=ctas)


@pytest.mark.parametrize("q8", [False, True])
def test_rows_that_start_anywhere(ms, q8):
    """Contiguous q, k, v that do not start on 16 bytes, and size-1 dimensions of any
    stride, are read as any other."""
    c = make(ms, 1, 1, 64, 16, 40, 4, torch.bfloat16, q8, 8)
    r, w = torch.full((1,), 1.2, device=DEV), torch.full((1,), 30.0, device=DEV)
    lens = torch.full((1,), 40, dtype=torch.int32, device=DEV)

    def shifted(x):
        flat = torch.empty(x.numel() + 1, dtype=x.dtype, device=DEV)
        flat[1:] = x.flatten().to(DEV)
        return flat.as_strided(x.shape, (7, 64, 3, 1), 1)

    rest = (lens, None, r, w, c["kp"], c["vp"], c["table"], c["ks"], c["vs"])
    want = ms.paged_tree_decode(*(c[x].to(DEV) for x in "qkv"), *rest)
    assert torch.equal(ms.paged_tree_decode(*(shifted(c[x]) for x in "qkv"), *rest), want)
    held = c["kp"].clone()
    ms.paged_append(shifted(c["k"]), shifted(c["v"]), lens, c["kp"], c["vp"], c["table"], c["ks"], c["vs"])
    assert torch.equal(c["kp"], held)
    if q8:
        one = c["q"][:, 0].to(DEV)
        moved = shifted(c["q"])[:, 0]
        seq = lens + 1
        tail = (seq, r, w, c["kp"], c["vp"], c["table"], c["ks"], c["vs"])
        assert torch.equal(ms.paged_decode(one, *tail), ms.paged_decode(moved, *tail))


@pytest.mark.parametrize("dtype,q8", [(torch.bfloat16, False), (torch.float32, True), (torch.float32, False)])
def test_lengths_past_the_table(ms, dtype, q8):
    """A length far past the block table reads what the table holds."""
    c = make(ms, 2, 2, 64, 16, 60, 3, dtype, q8, 12)
    rows = c["table"].shape[1] * 16
    lens = torch.tensor([60, 900_000_000], dtype=torch.int32)
    r, w = torch.full((2,), 1.2), torch.tensor([50.0, math.inf])
    for ctas in (1, 8):
        dev = [x.to(DEV) for x in (c["q"], c["k"], c["v"], lens)]
        y = ms.paged_tree_decode(*dev, None, r.to(DEV), w.to(DEV), c["kp"], c["vp"], c["table"], c["ks"], c["vs"],
                                 num_ctas=ctas)
        assert y.isfinite().all() and (y[1, :, 0] == 0).all()    # the window lies past the table
    prefix = tuple(None if x is None else x.cpu() for x in (c["kp"], c["vp"], c["ks"], c["vs"], c["table"]))
    # w = inf sees every cached row (weight 1); the nodes have no rows
    pos = list(range(rows))
    k, v = po.cache_values(prefix[0], prefix[2], prefix[4], 1, pos), po.cache_values(prefix[1], prefix[3], prefix[4], 1, pos)
    for i in range(3):
        want, s = po.query(c["q"][1, i, 1], k[:, 1], v[:, 1], torch.zeros(rows), 1.2, 1.0)
        lim = bound(want[None, None], torch.tensor(s)[None, None], r[1:], dtype, q8)
        assert float((y[1, i, 1].double().cpu() - want).norm()) <= float(lim.max())


@pytest.mark.parametrize("dtype,q8", [(torch.bfloat16, False), (torch.float32, False), (torch.bfloat16, True)])
@pytest.mark.parametrize("L,B,n,H,D,ps", [(1, 1, 1, 1, 16, 8), (3, 2, 5, 2, 64, 16), (2, 3, 64, 2, 128, 24)])
def test_commit(ms, L, B, n, H, D, ps, dtype, q8):
    g = torch.Generator().manual_seed(n)
    T = 20
    blocks = (T + n) // ps + 2
    table = torch.randperm(B * blocks, generator=g).view(B, blocks).to(torch.int32)
    shape = (L, B * blocks, H, ps, D)
    kp = torch.randint(-127, 128, shape, generator=g).to(torch.int8) if q8 else torch.randn(shape, generator=g).to(dtype)
    vp = kp.flip(0).clone().contiguous()
    ks = torch.rand(shape[:-1], generator=g) if q8 else None
    vs = torch.rand(shape[:-1], generator=g) if q8 else None
    lens = torch.tensor([T - b for b in range(B)], dtype=torch.int32)
    counts = torch.randint(0, n + 1, (B,), generator=g).to(torch.int32)
    counts[0] = n
    path = torch.stack([torch.randperm(n, generator=g).sort().values if b == 0 else torch.randperm(n, generator=g)
                        for b in range(B)]).to(torch.int32)          # any order is allowed
    if n > 4:
        path[-1, 1] = -1
        path[-1, 3] = n + 4
        counts[-1] = n + 9                                            # read as n
    lens[-1] = -1 if B > 2 else lens[-1]
    want = [None if x is None else x.clone() for x in (kp, vp, ks, vs)]
    for b in range(B):
        if lens[b] < 0:
            continue
        for x, old in zip(want, (kp, vp, ks, vs)):
            if x is None:
                continue
            for i in range(min(int(counts[b]), n)):
                p = int(path[b, i])
                if not 0 <= p < n:
                    continue
                f, t = int(lens[b]) + p, int(lens[b]) + i
                x[:, table[b, t // ps], :, t % ps] = old[:, table[b, f // ps], :, f % ps]
    dev = [None if x is None else x.to(DEV) for x in (kp, vp, table, ks, vs)]
    ms.paged_commit(lens.to(DEV), path.to(DEV), counts.to(DEV), *dev)
    for x, y in zip((dev[0], dev[1], dev[3], dev[4]), want):
        assert x is None or torch.equal(x.cpu(), y)
    if L == 1:                                                        # without the layer dimension
        dev2 = [None if x is None else (x[0] if x.dim() > 2 else x).to(DEV).contiguous() for x in (kp, vp, table, ks, vs)]
        ms.paged_commit(lens.to(DEV), path.to(DEV), counts.to(DEV), *dev2)
        assert torch.equal(dev2[0].cpu(), want[0][0])


@pytest.mark.parametrize("q8", [False, True])
def test_captured_and_on_two_streams(ms, q8):
    """Two captured graphs replayed on two streams, and an eager call between
    them, share nothing."""
    cs = [make(ms, 2, 2, 64, 16, 400, 9, torch.bfloat16, q8, s) for s in (3, 4)]
    lens = torch.tensor([400, 380], dtype=torch.int32, device=DEV)
    r, w = torch.tensor([1.1, 1.4], device=DEV), torch.tensor([600.0, 90.0], device=DEV)

    def run(c):
        return ms.paged_tree_decode(c["dq"], c["dk"], c["dv"], lens, None, r, w, c["kp"], c["vp"], c["table"], c["ks"],
                                    c["vs"], num_ctas=4)

    for c in cs:
        c["dq"], c["dk"], c["dv"] = (c[x].to(DEV) for x in "qkv")
    want = [run(c).clone() for c in cs]
    graphs, outs, streams = [], [], [torch.cuda.Stream(), torch.cuda.Stream()]
    for c in cs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(run(c))
        graphs.append(g)
    torch.cuda.synchronize()
    for _ in range(20):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    eager = run(cs[0])
    torch.cuda.synchronize()
    for o, x in zip(outs, want):
        assert torch.equal(o, x)
    assert torch.equal(eager, want[0])


@pytest.mark.parametrize("dtype,q8", [(torch.bfloat16, False), (torch.bfloat16, True), (torch.float32, False)])
@pytest.mark.parametrize("n", [1, 33, 64])
@pytest.mark.parametrize("T", [0, 3, 63, 250])
def test_runs_shorter_than_a_tree(ms, dtype, q8, n, T):
    """More CTAs than tiles: runs of one tile, of the nodes' rows alone, of nothing."""
    c = make(ms, 2, 2, 64, 16, T, n, dtype, q8, n + T)
    lens = torch.tensor([T, max(0, T - 9)], dtype=torch.int32)
    r, w = torch.tensor([1.1, 1.4]), torch.tensor([400.0, 20.0])
    check(ms, c, lens, tree_parents(2, n, "random", c["g"]), r, w, dtype, q8, num_ctas=592)


@pytest.mark.parametrize("dtype,q8", [(torch.bfloat16, True), (torch.bfloat16, False), (torch.float32, True)])
@pytest.mark.parametrize("D", [16, 64, 128])
@pytest.mark.parametrize("n", [0, 1, 5, 12, 20, 40])
def test_values_that_cancel(ms, n, D, dtype, q8):
    """Pairs of nearly equal keys with opposite values: what is left of the sum is
    far below its terms, so that the output's rounding hides nothing of alpha's.
    alpha is held to 2^-21 (two fp16 halves, 2^-11 each, the rest sums in 32 bits),
    to 2^-17 over bf16 pages (two bf16 halves, 2^-9 each).  n = 0: one query."""
    B, H, T, ps = 2, 8, 16, 16
    g = torch.Generator().manual_seed(100 * n + D)
    k = torch.randn(B, T // 2, H, D, generator=g).repeat_interleave(2, 1)
    k = k + 0.003 * torch.randn(B, T, H, D, generator=g)
    v = torch.randn(B, T // 2, H, D, generator=g).repeat_interleave(2, 1)
    v[:, 1::2] *= -1
    mean = 2.0 * torch.randn(H, D, generator=g)
    k = (k + mean).to(dtype)
    q = (mean + torch.randn(B, max(n, 1), H, D, generator=g)).to(dtype)
    blocks = (T + n) // ps + 1
    table = torch.randperm(B * blocks, generator=g).view(B, blocks).to(torch.int32).to(DEV)
    kp = torch.zeros(B * blocks, H, ps, D, dtype=torch.int8 if q8 else dtype, device=DEV)
    vp = torch.zeros_like(kp)
    ks, vs = [torch.zeros(B * blocks, H, ps, device=DEV) if q8 else None for _ in range(2)]
    ms.paged_append(k.to(DEV), v.to(dtype).to(DEV), torch.zeros(B, dtype=torch.int32, device=DEV), kp, vp, table, ks, vs)
    prefix = [None if x is None else x.cpu().clone() for x in (kp, vp, ks, vs, table)]
    r, w = torch.full((H,), 1.05), torch.full((H,), 4000.0)
    lens = torch.full((B,), T, dtype=torch.int32, device=DEV)
    if n:
        # a node's own key is the opposite of what the queries lean on: trimmed
        own = (-mean).expand(B, n, H, D).to(dtype)
        y = ms.paged_tree_decode(q.to(DEV), own.to(DEV), own.to(DEV), lens, None, r.to(DEV), w.to(DEV), kp, vp, table, ks, vs)
    else:
        y = ms.paged_decode(q[:, 0].to(DEV), lens, r.to(DEV), w.to(DEV), kp, vp, table, ks, vs)[:, None]
    al = 2.0**-21 if q8 else 2.0**-17
    out = 2.0**-8 if dtype == torch.bfloat16 else 2.0**-22
    for b in range(B):
        pk, pv = (po.cache_values(prefix[i], prefix[i + 2], prefix[4], b, list(range(T))) for i in (0, 1))
        for i in range(max(n, 1)):
            back = torch.arange(T - 1, -1, -1) + (i + 1 if n else 0)
            for h in range(H):
                want, s = po.query(q[b, i, h], pk[:, h], pv[:, h], back, float(r[h]), float(w[h]))
                lim = out * want.norm() + al * s[0] + 2.0**-18 * 1.05 * s[1] + 2.0**-21 * s[2] + 1e-9
                err = (y[b, i, h].double().cpu() - want).norm()
                assert err <= lim, (b, i, h, float(err), float(lim))
                if D == 64:
                    assert s[0] > 20 * want.norm()          # the terms do cancel


@pytest.mark.parametrize("dtype,q8", [(torch.bfloat16, True), (torch.bfloat16, False), (torch.float32, True),
                                      (torch.float32, False)])
@pytest.mark.parametrize("D", [16, 64])
@pytest.mark.parametrize("n", [1, 5, 12, 20, 40])
def test_alpha_is_held_whole(ms, n, D, dtype, q8):
    """Two equal keys, one place apart, with opposite values: their scores are the
    same number, so what is left is the difference of the masks (2^-17 of either) and
    the roundings of alpha after the score.  Those are at most, in half steps 2^-24:
    the cosine and sine (2 each, weight 1/2), their products with the V row's scale and
    the node's factors (3), two sums, the product with t^2 (1), and 4 for two fp16
    numbers (three bf16 numbers: 1): 12 an alpha, held to 16."""
    B, H, T, ps = 2, 16, 2, 16
    g = torch.Generator().manual_seed(10 * n + D)
    lead = torch.zeros(H, D)
    lead[:, 0] = 1.0
    k = lead + 0.6 * torch.rand(B, 1, H, D, generator=g) / math.sqrt(D)
    k = k.expand(B, T, H, D).contiguous()
    v = torch.randn(B, 1, H, D, generator=g)
    v = torch.cat([v, -v], 1)
    q = lead.expand(B, n, H, D)
    own = -q
    blocks = (T + n) // ps + 1
    table = torch.randperm(B * blocks, generator=g).view(B, blocks).to(torch.int32).to(DEV)
    kp = torch.zeros(B * blocks, H, ps, D, dtype=torch.int8 if q8 else dtype, device=DEV)
    vp = torch.zeros_like(kp)
    ks, vs = [torch.zeros(B * blocks, H, ps, device=DEV) if q8 else None for _ in range(2)]
    k, v, q, own = (x.to(dtype).to(DEV) for x in (k, v, q, own))
    ms.paged_append(k, v, torch.zeros(B, dtype=torch.int32, device=DEV), kp, vp, table, ks, vs)
    prefix = [None if x is None else x.cpu().clone() for x in (kp, vp, ks, vs, table)]
    r, w = torch.full((H,), 1.0625), torch.full((H,), 4000.0)
    lens = torch.full((B,), T, dtype=torch.int32, device=DEV)
    y = ms.paged_tree_decode(q, own, own, lens, None, r.to(DEV), w.to(DEV), kp, vp, table, ks, vs)
    out = 2.0**-8 if dtype == torch.bfloat16 else 2.0**-22
    for b in range(B):
        pk, pv = (po.cache_values(prefix[i], prefix[i + 2], prefix[4], b, list(range(T))) for i in (0, 1))
        for i in range(n):
            for h in range(H):
                want, s = po.query(q[b, i, h], pk[:, h], pv[:, h], torch.tensor([i + 2, i + 1]), float(r[h]), float(w[h]))
                err = (y[b, i, h].double().cpu() - want).norm()
                assert s[0] > 1.0 and err <= out * want.norm() + 2.0**-20 * s[0], (b, i, h, float(err), s[0])


@pytest.mark.parametrize("hint", [math.inf, math.nan, -1.0])
@pytest.mark.parametrize("dtype,q8", [(torch.bfloat16, False), (torch.bfloat16, True), (torch.float32, False)])
def test_hints_of_any_window(ms, dtype, q8, hint):
    """max_window only sets how the work is shared out: inf (a head that sees all) is
    one."""
    c = make(ms, 2, 2, 64, 16, 70, 4, dtype, q8, 6)
    lens = torch.tensor([70, 50], dtype=torch.int32)
    r, w = torch.tensor([1.1, 1.4]), torch.tensor([1e9, 20.0])
    check(ms, c, lens, None, r, w, dtype, q8, max_window=hint)
    args = (c["q"][:, 0].to(DEV), (lens + 1).to(DEV), r.to(DEV), w.to(DEV), c["kp"], c["vp"], c["table"], c["ks"], c["vs"])
    assert torch.equal(ms.paged_decode(*args, max_window=hint), ms.paged_decode(*args))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T", [400, 12000])
def test_decode_is_the_cache_s_decode(ms, dtype, T):
    """paged_decode over a PagedKVCache's pages shares out its work as the cache's own
    decode does: the same bits."""
    B, H, D = 4, 16, 64
    g = torch.Generator().manual_seed(T)
    cache = ms.PagedKVCache(1, B, H, D, T + 10, float(T), dtype, DEV)
    k, v = ((torch.randn(B, T, H, D, generator=g) + 0.5).to(dtype).to(DEV) for _ in range(2))
    cache.append(0, k, v, torch.zeros(B, dtype=torch.int32, device=DEV))
    q = (k[:, -1].cpu() + 0.5 * torch.randn(B, H, D, generator=g)).to(dtype).to(DEV)
    lens = torch.tensor([T, T - 37, T // 2, 1], dtype=torch.int32, device=DEV)
    r, w = torch.full((H,), 1.1, device=DEV), torch.linspace(float(T), 50.0, H).to(DEV)
    want, _ = cache.decode(0, q, lens, r, w)
    got = ms.paged_decode(q, lens, r, w, cache.k_pages[0], cache.v_pages[0], cache.block_table, max_window=float(T))
    assert torch.equal(got, want)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_decode_queries_that_start_anywhere(ms, dtype):
    """A contiguous q that does not start on 16 bytes, and a batch of one with any
    batch stride, are read as any other over fp32 / bf16 pages too."""
    c = make(ms, 1, 3, 64, 16, 60, 1, dtype, False, 3)
    r, w = torch.full((3,), 1.2, device=DEV), torch.full((3,), 40.0, device=DEV)
    tail = (torch.full((1,), 60, dtype=torch.int32, device=DEV), r, w, c["kp"], c["vp"], c["table"])
    q = c["q"][:, 0].to(DEV)
    flat = torch.empty(q.numel() + 1, dtype=dtype, device=DEV)
    flat[1:] = q.flatten()
    want = ms.paged_decode(q, *tail)
    assert torch.equal(ms.paged_decode(flat[1:].view(1, 3, 64), *tail), want)
    assert torch.equal(ms.paged_decode(q.as_strided((1, 3, 64), (7, 64, 1)), *tail), want)


@pytest.mark.parametrize("dtype,q8", [(torch.bfloat16, False), (torch.bfloat16, True), (torch.float32, False)])
@pytest.mark.parametrize("B,H", [(31, 16), (41, 17), (70, 30)])
def test_more_pairs_than_resident_ctas(ms, B, H, dtype, q8):
    """Around and beyond one (sequence, head) pair per resident CTA, uneven lengths:
    any num_ctas gives each pair to one CTA, the bits of num_ctas = 1, which are
    those of its sequence alone."""
    D, ps, T, n = 16, 16, 300, 3
    c = make(ms, B, H, D, ps, T, n, dtype, q8, B)
    g = torch.Generator().manual_seed(B)
    lens = torch.randint(0, T, (B,), generator=g).to(torch.int32)
    lens[3] = T
    lens[5] = -1
    r, w = torch.full((H,), 1.1), torch.linspace(T + 5.0, 9.0, H)
    dev = [x.to(DEV) for x in (c["q"], c["k"], c["v"], lens)]
    rw = (r.to(DEV), w.to(DEV))

    def run(lo=0, hi=B, **kw):
        part = [x[lo:hi] for x in dev]
        return ms.paged_tree_decode(*part, None, *rw, c["kp"], c["vp"], c["table"][lo:hi], c["ks"], c["vs"], **kw)

    want = run(num_ctas=1)
    assert (want[5] == 0).all() and want.isfinite().all()
    for kw in (dict(), dict(num_ctas=B * H), dict(num_ctas=60000)):
        got = run(**kw)
        if B * H >= 592 or kw.get("num_ctas") == B * H:
            assert torch.equal(got, want), kw
        else:                                    # 496 pairs: four CTAs an SM share out, three do not
            tol = 2.0**-6 if dtype == torch.bfloat16 else 2.0**-17
            assert ((got - want).float().norm(dim=-1) <= tol * want.float().norm(dim=-1) + 1e-6).all()
    assert torch.equal(run(2, 6, num_ctas=1), want[2:6])


@pytest.mark.parametrize("dtype,q8", [(torch.bfloat16, False), (torch.bfloat16, True), (torch.float32, False),
                                      (torch.float32, True)])
@pytest.mark.parametrize("n,ctas", [(1, 1), (7, 40), (20, 1), (40, 592)])
def test_rows_that_are_there_already(ms, n, ctas, dtype, q8):
    """k, v = None: the nodes' rows were appended before.  The same bits, and nothing is
    written."""
    c = make(ms, 2, 2, 64, 24, 150, n, dtype, q8, 60 + n)
    lens = torch.tensor([150, 90], dtype=torch.int32, device=DEV)
    parents = tree_parents(2, n, "random", c["g"]).to(DEV)
    r, w = torch.tensor([1.1, 1.4], device=DEV), torch.tensor([120.0, 33.0], device=DEV)
    q, k, v = (c[x].to(DEV) for x in "qkv")
    rest = (lens, parents, r, w, c["kp"], c["vp"], c["table"], c["ks"], c["vs"])
    want = ms.paged_tree_decode(q, k, v, *rest, num_ctas=1)
    held = [None if c[x] is None else c[x].clone() for x in ("kp", "vp", "ks", "vs")]
    ms.paged_append(k, v, lens, c["kp"], c["vp"], c["table"], c["ks"], c["vs"])
    assert all(x is None or torch.equal(x, c[y]) for x, y in zip(held, ("kp", "vp", "ks", "vs")))
    got = ms.paged_tree_decode(q, None, None, *rest, num_ctas=ctas)
    if ctas == 1:
        assert torch.equal(got, want)
    else:
        tol = 2.0**-7 if dtype == torch.bfloat16 else 2.0**-18
        assert ((got - want).float().norm(dim=-1) <= tol * want.float().norm(dim=-1) + 1e-6).all()
    assert all(x is None or torch.equal(x, c[y]) for x, y in zip(held, ("kp", "vp", "ks", "vs")))


@pytest.mark.parametrize("eps", [1e-8, 0.5, 30.0])
@pytest.mark.parametrize("dtype,q8", [(torch.bfloat16, False), (torch.bfloat16, True), (torch.float32, False),
                                      (torch.float32, True)])
def test_rows_and_queries_below_eps(ms, dtype, q8, eps):
    """Raw rows of norm about 8 and 0: eps holds short rows, queries and sums down."""
    B, H, D, ps, T, n = 2, 2, 64, 16, 40, 5
    c = make(ms, B, H, D, ps, T, n, dtype, q8, 5)
    c["q"][0, 1] = 0
    c["k"][0, 2] = 0
    c["v"][1, 0] = 0
    lens = torch.tensor([T, 20], dtype=torch.int32)
    r, w = torch.tensor([0.9, 0.6]), torch.tensor([30.0, 12.0])
    dev = [c[x].to(DEV) for x in "qkv"] + [lens.to(DEV), None, r.to(DEV), w.to(DEV)]
    prefix = tuple(None if x is None else x.cpu().clone() for x in (c["kp"], c["vp"], c["ks"], c["vs"], c["table"]))
    y = ms.paged_tree_decode(*dev, c["kp"], c["vp"], c["table"], c["ks"], c["vs"], eps=eps)
    for b in range(B):
        held = []
        for x in "kv":
            got = po.cache_values(c[x + "p"], c[x + "s"], c["table"], b, [int(lens[b]) + i for i in range(n)])
            if q8:
                m, sc = po.int8_rows(c[x][b], eps)
                row, tol = m.double() * sc[..., None], 2.0**-21
            else:
                row, tol = po.unit_rows(c[x][b], eps), 2.0**-21 + (2.0**-8 if dtype == torch.bfloat16 else 0.0)
            assert ((got - row).abs() <= tol * row.abs() + 1e-12).all()
            held.append(got)
        want, sums = po.tree(c["q"][b], held[0], held[1], int(lens[b]), None, r, w, prefix, b, eps)
        err = (y[b].double().cpu() - want).norm(dim=-1)
        assert (err <= bound(want, sums, r, dtype, q8)).all(), (b, err)
