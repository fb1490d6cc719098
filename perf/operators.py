"""Workloads of speculative serving on the paged screening cache.

Five operators, each with a plain form in elementary torch operations and the
library's call beside it (`own`):

  append8  raw k / v rows written to an int8 paged cache and read back
  decode8  one query per sequence over the int8 cache
  tree     a tree of drafted tokens: its k / v rows written behind the cached
           prefix, every node attending over the prefix and its ancestors
  commit   the rows of the accepted path moved to the positions they keep
  verify   drafted tokens accepted or rejected against the target's
           probabilities from given random numbers

Definitions.  A cache row is the unit row x / max(|x|, eps) of a raw row x.
An int8 row holds the integers m = round_half_even(127 x / max|x|) and the
scale 1 / max(|m|, 127 eps / max|x|), so that scale * m is the unit form of the
rounded raw row; a row with an infinity or NaN has scale NaN and m = 0.
Query i at position p sees cached key j iff 0 <= p - j <= ceil(w) - 1, with
alpha = relu(1 - r (1 - q^.k^))^2 (1 + cos(pi (j - p) / w)) / 2, and
y = tanh(|o|) / |o| o with o = sum alpha v^.  Node i of a tree has
parents[i] < i (-1: child of the newest cached token; any other value: absent),
stands at position lens + depth and sees the window's cached keys, its
ancestors and itself.
"""
import math

import torch

own = False

EPS = 1e-8
VOCAB = 50257          # the LM benchmark's vocabulary; its logits rows are padded to 64


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def listed():
    return [
        # the rows of one generated token for a batch of four, the smallest write
        dict(name="append8-token", op="append8", B=4, n=1, H=16, D=64, ps=64, dtype="bf16"),
        # the last window of a prompt after its prefill (w = 4096)
        dict(name="append8-window", op="append8", B=4, n=4097, H=16, D=64, ps=64, dtype="bf16"),
        # a token step of a model at its initial windows (w <= 256): latency
        dict(name="decode8-w256", op="decode8", B=4, H=16, D=64, ps=64, T=700, w=256, dtype="bf16"),
        # fp32 activations, wide heads, odd batch and length, small pages
        dict(name="decode8-fp32-d128", op="decode8", B=3, H=5, D=128, ps=16, T=5003, w=4999, dtype="fp32"),
        # a token step whose windows cover a 100K-token prompt: bandwidth
        dict(name="decode8-100k", op="decode8", B=4, H=16, D=64, ps=64, T=100001, w=100002, dtype="bf16"),
        # a short chain of drafts behind the initial windows: latency
        dict(name="tree-chain5", op="tree", B=4, n=5, H=16, D=64, ps=64, T=700, w=256, dtype="bf16", q8=False, shape="chain"),
        # a tree of 16 drafts over windows of 4096, bf16 cache, ragged lengths
        dict(name="tree-16-4k", op="tree", B=4, n=16, H=16, D=64, ps=64, T=6001, w=4096, dtype="bf16", q8=False, shape="tree"),
        # the widest tree over 32K keys of an int8 cache
        dict(name="tree-64-32k", op="tree", B=4, n=64, H=16, D=64, ps=64, T=32768, w=32768, dtype="bf16", q8=True, shape="tree"),
        # an accepted path of a small tree, every layer of a 12-layer model
        dict(name="commit-16", op="commit", L=12, B=4, n=16, H=16, D=64, ps=64, q8=False),
        # the widest tree, int8 rows
        dict(name="commit-64", op="commit", L=12, B=8, n=64, H=16, D=64, ps=64, q8=True),
        # a chain of four sampled drafts with the drafting model's logits
        dict(name="verify-chain4", op="verify", B=4, n=4, V=VOCAB, dtype="bf16", shape="chain", draft=True, temperature=0.8),
        # a serving batch of 32-node trees of likely tokens
        dict(name="verify-tree32", op="verify", B=32, n=32, V=VOCAB, dtype="bf16", shape="tree", draft=False, temperature=1.0),
    ]


def _span(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append8", "decode8", "decode8", "tree", "tree", "commit", "verify", "verify"])
    D = rng.choice([16, 32, 64, 64, 128])
    H = rng.randint(1, 16)
    ps = rng.choice([8, 16, 24, 64, 100])
    dtype = rng.choice(["bf16", "bf16", "fp32"])
    if op == "append8":
        n = _span(rng, 1, 4000)
        return dict(op=op, B=rng.randint(1, 4), n=n, H=H, D=min(D, 64) if dtype == "bf16" else min(D, 32), ps=ps, dtype=dtype)
    if op == "decode8":
        T = _span(rng, 1, 60000)
        return dict(op=op, B=rng.randint(1, 4), H=H, D=D, ps=ps, T=T, w=max(2, int(T * rng.uniform(0.1, 1.2))), dtype=dtype)
    if op == "tree":
        n, T = _span(rng, 1, 64), _span(rng, 1, 16000)
        if dtype == "fp32":
            n, T = min(n, 24), min(T, 6000)
        return dict(op=op, B=rng.randint(1, 4), n=n, H=H, D=min(D, 64), ps=ps, T=T, w=max(2, int(T * rng.uniform(0.1, 1.2))),
                    dtype=dtype, q8=rng.random() < 0.5, shape=rng.choice(["chain", "tree", "padded"]))
    if op == "commit":
        return dict(op=op, L=rng.randint(1, 12), B=rng.randint(1, 8), n=_span(rng, 1, 64), H=H, D=min(D, 64), ps=ps, q8=rng.random() < 0.5)
    chain = rng.random() < 0.5
    return dict(op=op, B=rng.randint(1, 16), n=_span(rng, 1, 16), V=_span(rng, 500, 60000), dtype=dtype, shape="chain" if chain else "tree",
                draft=rng.random() < 0.6, temperature=rng.choice([0.0, 0.7, 1.0, 1.3]))


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _dt(case):
    return torch.bfloat16 if case["dtype"] == "bf16" else torch.float32


def _unit(x):
    return x / x.norm(dim=-1, keepdim=True).clamp_min(EPS)


def _int8_rows(x):
    """(m int8, scale fp32) of raw rows x: the rounding in 64 bits, where a
    product next to a half would tip either way in 32."""
    x = x.double()
    top = x.abs().amax(-1, keepdim=True)
    m = torch.where(top > 0, (127.0 * x / top.clamp_min(1e-300)).round(), 0.0)
    scale = 1.0 / torch.maximum(m.norm(dim=-1), 127.0 * EPS / top[..., 0])
    finite = x.isfinite().all(-1)
    return torch.where(finite[..., None], m, 0.0).to(torch.int8), torch.where(finite, scale, math.nan).float()


def _parents(B, n, shape, g, dev):
    """A chain; a tree whose nodes hang below a random earlier one (a few roots);
    or trees of different sizes, the missing nodes marked absent (-2)."""
    i = torch.arange(n, device=dev)
    if shape == "chain":
        return (i - 1).expand(B, n).to(torch.int32).contiguous()
    up = (torch.rand(B, n, device=dev, generator=g) ** 0.7 * (i + 1)).long() - 1
    p = torch.minimum(up, i - 1)
    if shape == "padded":
        have = torch.randint(0, n + 1, (B, 1), device=dev, generator=g)
        p = torch.where(i < have, p, -2)
    return p.to(torch.int32).contiguous()


def _pages(case, g, dev, layers=None):
    """Filled pages of a ring cache per sequence under a shuffled table, at the
    lengths `lens` (ragged, the longest first)."""
    B, H, D, ps, n = case["B"], case["H"], case["D"], case["ps"], case.get("n", 1)
    T, w = case.get("T", 64), case.get("w", 64)
    keep = min(T, w) + n
    per = -(-keep // ps) + 1
    blocks = -(-(T + n) // ps)
    per = min(per, blocks)
    order = torch.randperm(B * per, device=dev, generator=g).view(B, per)
    table = order[:, torch.arange(blocks, device=dev) % per].to(torch.int32).contiguous()
    lead = () if layers is None else (layers,)
    raw = torch.empty(lead + (B * per, H, ps, D), device=dev, dtype=torch.bfloat16).normal_(generator=g)
    val = torch.empty_like(raw).normal_(generator=g)
    # a direction common to a head's keys, as trained keys have
    raw += 0.6 * torch.randn((H, 1, D), device=dev, generator=g).to(raw.dtype)
    st = dict(case=case, block_table=table)
    # drafts and length: the tree's rows come behind lens
    st["lens"] = (T - (T // 8) * torch.arange(B, device=dev) // max(1, B - 1)).to(torch.int32)
    q8 = case.get("q8", case["op"] in ("append8", "decode8"))
    for name, x in (("k", raw), ("v", val)):
        if q8:
            flat = x.view(-1, ps, D)
            m = torch.empty(flat.shape, device=dev, dtype=torch.int8)
            s = torch.empty(flat.shape[:-1], device=dev)
            step = max(1, (1 << 25) // (ps * D))
            for a in range(0, flat.shape[0], step):
                m[a:a + step], s[a:a + step] = _int8_rows(flat[a:a + step])
            st[name + "_pages"], st[name + "_scales"] = m.view(x.shape), s.view(x.shape[:-1])
        else:
            dt = torch.bfloat16 if "dtype" not in case else _dt(case)
            st[name + "_pages"], st[name + "_scales"] = _unit(x.float()).to(dt), None
    # sharpness in [1, 2], windows up to w (the widest head sees all of it)
    st["r"] = 1.0 + torch.rand(H, device=dev, generator=g)
    st["w"] = torch.linspace(1.0, 0.25, H, device=dev) * w
    return st


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    op = case["op"]
    if op == "append8":
        B, n, H, D, ps = case["B"], case["n"], case["H"], case["D"], case["ps"]
        blocks = -(-(n + 3) // ps)
        table = torch.randperm(B * blocks, device=dev, generator=g).view(B, blocks).to(torch.int32)
        qkv = torch.randn(B, n, 3, H, D, device=dev, generator=g) * 2.0
        qkv = qkv.to(_dt(case))
        return dict(case=case, k=qkv[:, :, 1], v=qkv[:, :, 2], positions=torch.randint(0, 4, (B,), device=dev, generator=g).to(torch.int32),
                    k_pages=torch.zeros(B * blocks, H, ps, D, dtype=torch.int8, device=dev), v_pages=torch.zeros(B * blocks, H, ps, D, dtype=torch.int8, device=dev),
                    k_scales=torch.zeros(B * blocks, H, ps, device=dev), v_scales=torch.zeros(B * blocks, H, ps, device=dev), block_table=table)
    if op in ("decode8", "tree"):
        n = case.get("n", 1)
        st = _pages(case, g, dev)
        B, H, D, ps = case["B"], case["H"], case["D"], case["ps"]
        # every query leans on a cached key it can see
        back = torch.randint(0, 64, (B, n), device=dev, generator=g).clamp_max(min(case["T"], case["w"]) // 2)
        at = (st["lens"][:, None] - 1 - back).clamp_min(0).long()
        page = st["block_table"].long().gather(1, at // ps)
        lean = st["k_pages"][page, :, at % ps].float()
        noise = torch.randn(B, n, H, D, device=dev, generator=g)
        st["q"] = (_unit(lean) * math.sqrt(D) + noise).to(_dt(case))
        if op == "decode8":
            st["q"] = st["q"][:, 0].contiguous()
            return st
        kv = torch.randn(2, B, n, H, D, device=dev, generator=g)
        st["k"] = (kv[0] + 0.5 * st["q"].float()).to(_dt(case))
        st["v"] = kv[1].to(_dt(case))
        st["parents"] = _parents(B, n, case["shape"], g, dev)
        return st
    if op == "commit":
        L, B, n = case["L"], case["B"], case["n"]
        st = _pages(dict(case, T=200), g, dev, layers=L)
        counts = torch.randint(0, n + 1, (B,), device=dev, generator=g)
        counts[0] = n // 2
        pick = torch.rand(B, n, device=dev, generator=g).argsort(1)
        kept = torch.where(torch.arange(n, device=dev) < counts[:, None], pick, n).sort(1).values
        st["path"] = torch.where(kept < n, kept, -1).to(torch.int32)
        st["counts"] = counts.to(torch.int32)
        return st
    # verify: logits rows of the newest token and of each drafted one, as views
    # of rows padded to 64; drafts are samples of the drafting model, or (no
    # drafting distribution) likely tokens of the target
    B, n, V = case["B"], case["n"], case["V"]
    width = -(-V // 64) * 64
    logits = torch.randn(B, n + 1, width, device=dev, generator=g) * 3.0
    parents = _parents(B, n, case["shape"], g, dev)
    row = (parents.long() + 1).clamp(0, n - 1)
    st = dict(case=case, parents=parents, uniforms=torch.rand(B, n + 1, device=dev, generator=g), temperature=float(case["temperature"]), draft_logits=None)
    if case["draft"]:
        dl = logits[:, :n] + torch.randn(B, n, width, device=dev, generator=g)
        dl = dl.to(_dt(case))[..., :V]
        gumbel = -torch.log(-torch.log(torch.rand(B, n, V, device=dev, generator=g).clamp(1e-7, 1 - 1e-7)))
        tau = max(st["temperature"], 1e-3)
        st["tokens"] = (dl.float().gather(1, row[..., None].expand(B, n, V)) / tau + gumbel).argmax(-1)
        st["draft_logits"] = dl
    else:
        likely = logits[..., :V].topk(min(4, V), dim=-1).indices
        st["tokens"] = likely.gather(1, row[..., None].expand(B, n, likely.shape[-1]))[
            torch.arange(B, device=dev)[:, None], torch.arange(n, device=dev)[None], torch.randint(0, likely.shape[-1], (B, n), device=dev, generator=g)]
        # a peaked target, so that some of them are accepted
        logits[..., :V].scatter_add_(2, likely, torch.full(likely.shape, 4.0, device=dev))
    st["logits"] = logits.to(_dt(case))[..., :V]
    return st


# ---------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------
def _slots(block_table, pos, ps):
    """(page, row, inside) of positions pos (B, n)."""
    inside = (pos >= 0) & (pos < block_table.shape[1] * ps)
    at = torch.where(inside, pos, 0)
    return block_table.long().gather(1, at // ps), at % ps, inside


def _write(s, k, v, pos, take):
    """Unit rows of raw k, v (B, n, H, D) into the pages at pos where `take`."""
    page, row, inside = _slots(s["block_table"], pos, s["k_pages"].shape[-2])
    take = take & inside
    page, row = page[take], row[take]
    for x, name in ((k, "k"), (v, "v")):
        x = x[take].float()
        if s[name + "_scales"] is None:
            s[name + "_pages"][page, :, row] = _unit(x).to(s[name + "_pages"].dtype)
        else:
            m, sc = _int8_rows(x)
            s[name + "_pages"][page, :, row] = m
            s[name + "_scales"][page, :, row] = sc


def _read(s, name, pos):
    """fp32 rows (B, n, H, D) of the pages at pos; rows outside the table 0."""
    page, row, inside = _slots(s["block_table"], pos, s["k_pages"].shape[-2])
    x = s[name + "_pages"][page, :, row].float()
    if s[name + "_scales"] is not None:
        x = x * s[name + "_scales"][page, :, row][..., None]
    return torch.where(inside[..., None, None], x, 0.0)


def _attend(s, q, lens, n_slots, depth, sees):
    """y (B, n, H, D) of queries at lens + depth over the window's cached keys
    and the n_slots rows behind them (`sees` (B, n, n_slots))."""
    case, r, w = s["case"], s["r"], s["w"]
    span = min(case["T"], math.ceil(case["w"]) - 1)
    first = lens.long()[:, None] - span
    pos = first + torch.arange(span + n_slots, device=q.device)          # (B, K)
    k, v = _read(s, "k", pos), _read(s, "v", pos)
    qf = q.float()
    qf = qf / qf.norm(dim=-1, keepdim=True).clamp_min(EPS)
    scores = torch.matmul(qf.transpose(1, 2), k.permute(0, 2, 3, 1))      # (B, H, n, K)
    at = lens.long()[:, None] + depth                                     # (B, n)
    # a node's place on its own path: cached keys by position, drafts by depth
    kd = torch.cat([pos[:, :span], lens.long()[:, None] + depth[:, :n_slots]], 1) if n_slots else pos
    rel = kd[:, None, :] - at[..., None]                                  # (B, n, K)
    dmax = torch.ceil(w) - 1
    see = torch.cat([(pos[:, :span] >= 0)[:, None, :].expand(-1, q.shape[1], -1), sees], 2)
    live = see[:, None] & (rel[:, None] >= -dmax[None, :, None, None]) & (rel[:, None] <= 0)
    mask = 0.5 * (1.0 + torch.cos(math.pi * rel[:, None] / w[None, :, None, None]))
    alpha = torch.relu(1.0 - r[None, :, None, None] * (1.0 - scores)) ** 2 * mask
    alpha = torch.where(live, alpha, 0.0)
    o = torch.matmul(alpha, v.transpose(1, 2)).transpose(1, 2)            # (B, n, H, D)
    size = o.norm(dim=-1, keepdim=True).clamp_min(EPS)
    return (torch.tanh(size) / size * o).to(q.dtype)


def _ancestors(parents):
    """(sees (B, n, n) ancestors and self, depth (B, n), present (B, n))."""
    B, n = parents.shape
    i = torch.arange(n, device=parents.device)
    p = parents.long()
    ok = (p >= -1) & (p < i)
    up = ((p[..., None] == i) & ok[..., None]).float()                    # parent's column
    line = up + torch.eye(n, device=parents.device)
    for _ in range(6):                                                    # 64 generations
        line = (line @ line).clamp_max(1.0)
    present = (line @ (~ok).float()[..., None])[..., 0] == 0
    sees = (line > 0) & present[..., None]
    return sees, (sees.sum(-1) - 1).clamp_min(0), present


def _plain_verify(s):
    """The acceptance scan, in 64 bits: a token is drawn where u crosses the sum
    of the probabilities, and 32 bits move that border."""
    logits, tokens, u, tau = s["logits"], s["tokens"], s["uniforms"].double(), s["temperature"]
    B, rows, V = logits.shape
    n = rows - 1
    dev = logits.device
    ar = torch.arange(B, device=dev)

    def dist(x):
        x = x.double()
        if tau > 0:
            return torch.softmax(x / tau, -1)
        top = (x == x.amax(-1, keepdim=True))
        first = top & (top.cumsum(-1) == 1)
        return first.double()

    parent_row = s["parents"].long() + 1
    cur = torch.zeros(B, dtype=torch.long, device=dev)
    p = dist(logits[:, 0])
    q = None if s["draft_logits"] is None else dist(s["draft_logits"][:, 0])
    rest, c, z = p, torch.zeros(B, device=dev, dtype=torch.float64), torch.ones(B, device=dev, dtype=torch.float64)
    counts = torch.zeros(B, dtype=torch.int32, device=dev)
    path = torch.full((B, n), -1, dtype=torch.int32, device=dev)
    out = torch.full((B, n + 1), -1, dtype=torch.int64, device=dev)
    for i in range(n):
        x = tokens[:, i]
        test = (parent_row[:, i] == cur) & (s["parents"][:, i] < i) & (s["parents"][:, i] >= -1)
        px = rest[ar, x]
        qx = 1.0 if q is None else q[ar, x]
        accept = test & (px > 0) & (u[:, i] * qx * z < px)
        reject = test & ~accept
        # a rejected child leaves max(p - c q, 0), c growing by the mass left
        if q is None:
            left = rest.clone()
            left[ar, x] = 0.0
            zn = left.sum(-1)
            rest = torch.where(reject[:, None], left, rest)
        else:
            c = torch.where(reject, c + z, c)
            left = (p - c[:, None] * q).clamp_min(0.0)
            zn = left.sum(-1)
            rest = torch.where(reject[:, None], left, rest)
        z = torch.where(reject, zn, z)
        slot = counts.long()
        path[ar[:, None], slot[:, None].clamp_max(n - 1)] = torch.where(accept, i, path[ar, slot.clamp_max(n - 1)])[:, None].to(torch.int32)
        out[ar, slot] = torch.where(accept, x, out[ar, slot])
        counts = counts + accept.to(torch.int32)
        cur = torch.where(accept, i + 1, cur)
        p = torch.where(accept[:, None], dist(logits[:, i + 1]), p)
        rest = torch.where(accept[:, None], p, rest)
        if q is not None:
            q = torch.where(accept[:, None], dist(s["draft_logits"][:, min(i + 1, n - 1)]), q)
        c = torch.where(accept, 0.0, c)
        z = torch.where(accept, 1.0, z)
    rest = torch.where((z > 0)[:, None], rest, p)
    run_sum = rest.cumsum(-1)
    over = (run_sum > u[:, n:] * run_sum[:, -1:]) & (rest > 0)
    last = torch.where(over.any(-1), over.int().argmax(-1), V - 1 - (rest > 0).int().flip(-1).argmax(-1))
    out[ar, counts.long()] = last
    return out, path, counts


def _plain(s):
    op = s["case"]["op"]
    if op == "append8":
        n = s["k"].shape[1]
        pos = s["positions"].long()[:, None] + torch.arange(n, device=s["k"].device)
        _write(s, s["k"], s["v"], pos, torch.ones_like(pos, dtype=torch.bool))
        return _read(s, "k", pos), _read(s, "v", pos)
    if op == "decode8":
        B = s["q"].shape[0]
        none = torch.zeros(B, 1, 0, dtype=torch.bool, device=s["q"].device)
        zero = torch.zeros(B, 1, dtype=torch.long, device=s["q"].device)
        # the query of the newest cached token sees that token itself
        return _attend_newest(s, none, zero)
    if op == "tree":
        n = s["q"].shape[1]
        sees, depth, present = _ancestors(s["parents"])
        pos = s["lens"].long()[:, None] + torch.arange(n, device=s["q"].device)
        _write(s, s["k"], s["v"], pos, present)
        y = _attend(s, s["q"], s["lens"], n, depth, sees)
        y = torch.where(present[..., None, None], y, torch.zeros((), dtype=y.dtype, device=y.device))
        out = {"y": y, "k_pages": s["k_pages"], "v_pages": s["v_pages"]}
        if s["k_scales"] is not None:
            out |= {"k_scales": s["k_scales"], "v_scales": s["v_scales"]}
        return out
    if op == "commit":
        n = s["path"].shape[1]
        i = torch.arange(n, device=s["path"].device)
        take = i < s["counts"][:, None]
        fp, fr, _ = _slots(s["block_table"], s["lens"].long()[:, None] + torch.where(take, s["path"].long(), 0), s["case"]["ps"])
        tp, tr, _ = _slots(s["block_table"], s["lens"].long()[:, None] + i, s["case"]["ps"])
        fp, fr, tp, tr = fp[take], fr[take], tp[take], tr[take]
        out = {}
        for name in ("k_pages", "v_pages", "k_scales", "v_scales"):
            if s[name] is not None:
                s[name][:, tp, :, tr] = s[name][:, fp, :, fr]
                out[name] = s[name]
        return out
    return _plain_verify(s)


def _attend_newest(s, none, zero):
    """decode: the query stands at lens - 1 over the keys up to itself."""
    case = s["case"]
    q, lens = s["q"][:, None], s["lens"] - 1
    one = dict(s, case=dict(case, T=case["T"]))
    sees = torch.ones(q.shape[0], 1, 1, dtype=torch.bool, device=q.device)
    return _attend(one, q, lens, 1, zero, sees)[:, 0]


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(state):
    if not own:
        return _plain(state)
    s, op = state, state["case"]["op"]
    ms = _package()
    if op == "append8":
        n = s["k"].shape[1]
        ms.paged_append(s["k"], s["v"], s["positions"], s["k_pages"], s["v_pages"], s["block_table"], s["k_scales"], s["v_scales"])
        return ms.paged_read(s["positions"], n, s["k_pages"], s["v_pages"], s["block_table"], s["k_scales"], s["v_scales"], dtype=torch.float32)
    if op == "decode8":
        return ms.paged_decode(s["q"], s["lens"], s["r"], s["w"], s["k_pages"], s["v_pages"], s["block_table"], s["k_scales"], s["v_scales"],
                               max_window=s["case"]["w"])
    if op == "tree":
        y = ms.paged_tree_decode(s["q"], s["k"], s["v"], s["lens"], s["parents"], s["r"], s["w"], s["k_pages"], s["v_pages"], s["block_table"],
                                 s["k_scales"], s["v_scales"], max_window=s["case"]["w"])
        out = {"y": y, "k_pages": s["k_pages"], "v_pages": s["v_pages"]}
        if s["k_scales"] is not None:
            out |= {"k_scales": s["k_scales"], "v_scales": s["v_scales"]}
        return out
    if op == "commit":
        ms.paged_commit(s["lens"], s["path"], s["counts"], s["k_pages"], s["v_pages"], s["block_table"], s["k_scales"], s["v_scales"])
        return {k: s[k] for k in ("k_pages", "v_pages", "k_scales", "v_scales") if s[k] is not None}
    return ms.verify_drafts(s["logits"], s["tokens"], s["parents"], s["uniforms"], draft_logits=s["draft_logits"], temperature=s["temperature"])


def _package():
    import importlib
    return importlib.import_module("pytorch-implementation-of-screening-attention_b200")


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    op, B = case["op"], case["B"]
    es = 2 if case.get("dtype", "bf16") == "bf16" else 4
    if op == "append8":
        rows = 2 * B * case["n"] * case["H"]
        D = case["D"]
        # raw rows in, int8 rows and scales out and in again, fp32 rows out
        return {"bytes": rows * (D * es + 2 * (D + 4) + 4 * D), "flops": rows * D * 5}
    if op in ("decode8", "tree"):
        H, D, n = case["H"], case["D"], case.get("n", 1)
        q8 = case.get("q8", True)
        row = D + 4 if q8 else D * es
        # the head windows are spread over [w / 4, w], the lengths over [7 T / 8, T]
        keys = min(0.94 * case["T"], 0.625 * case["w"])
        rows = B * H * n * D * es
        extra = 2 * rows + 2 * B * H * n * row if op == "tree" else 0
        return {"bytes": B * H * keys * 2 * row + 2 * rows + extra, "flops": B * H * n * (keys + n / 2) * 4 * D}
    if op == "commit":
        rows = case["L"] * B * case["H"] * 2 * case["n"] / 2
        return {"bytes": 2 * rows * (case["D"] + 4 if case["q8"] else case["D"] * 2), "flops": 0}
    rows = B * (case["n"] + 1) + (B * case["n"] if case["draft"] else 0)
    return {"bytes": rows * case["V"] * es, "flops": rows * case["V"] * 4}


# ---------------------------------------------------------------------------
# the definitions in 64 bits, sequence by sequence
# ---------------------------------------------------------------------------
def _exact_row(x, q8):
    x = x.double()
    if not q8:
        return x / max(float(x.norm()), EPS)
    top = float(x.abs().max())
    if top == 0.0:
        return torch.zeros_like(x)
    m = torch.round(x * 127.0 / top)
    return m / max(float(m.norm()), 127.0 * EPS / top)


def _exact_rows(x, q8):
    """_exact_row of every row of x, at once."""
    x = x.double()
    if not q8:
        return x / x.pow(2).sum(-1, keepdim=True).sqrt().clamp(min=EPS)
    top = x.abs().max(-1, keepdim=True)[0]
    m = torch.round(x * 127.0 / top)
    size = m.pow(2).sum(-1, keepdim=True).sqrt()
    return torch.nan_to_num(m / torch.max(size, 127.0 * EPS / top))


def _exact_cache(s, b, name, hi):
    """Rows 0 .. hi-1 (those the table still holds) of sequence b, (hi, H, D)."""
    ps = s["k_pages"].shape[-2]
    t = torch.arange(hi, device=s["block_table"].device)
    pages = s["block_table"][b].long()[t // ps]
    x = s[name + "_pages"][pages, :, t % ps].double()
    if s[name + "_scales"] is not None:
        x = x * s[name + "_scales"][pages, :, t % ps].double()[..., None]
    return x


def _exact_query(q, k, v, back, r, w):
    """y (H, D) of one query over rows k, v (K, H, D) that stand `back` >= 0 (K,)
    positions before it."""
    q = q.double()
    q = q / q.norm(dim=-1, keepdim=True).clamp(min=EPS)
    r, w = r.double(), w.double()
    sim = (k * q).sum(-1)                                                 # (K, H)
    a = (1 - r * (1 - sim)).clamp(min=0).pow(2)
    m = (1 + torch.cos(math.pi * back.double()[:, None] / w)) / 2
    m = torch.where(back[:, None] < w, m, torch.zeros_like(m))            # -w < rel
    o = ((a * m)[..., None] * v).sum(0)
    size = o.norm(dim=-1, keepdim=True).clamp(min=EPS)
    return torch.tanh(size) * o / size


def exact(case, seed):
    op = case["op"]
    if op == "verify":
        return None                                   # whole numbers
    s = prepare(case, seed)
    if op == "append8":
        return _exact_rows(s["k"], True), _exact_rows(s["v"], True)
    if op == "commit":
        out = {}
        for name in ("k_pages", "v_pages", "k_scales", "v_scales"):
            if s[name] is None:
                continue
            if s[name].dtype == torch.int8:
                out[name] = None
                continue
            new = s[name].double()
            old = new.clone()
            lens, counts, path, tab = (s[x].tolist() for x in ("lens", "counts", "path", "block_table"))
            for b in range(case["B"]):
                for i in range(counts[b]):
                    a, z = lens[b] + path[b][i], lens[b] + i
                    new[:, tab[b][z // case["ps"]], :, z % case["ps"]] = old[:, tab[b][a // case["ps"]], :, a % case["ps"]]
            out[name] = new
        return out
    B, H, D = case["B"], case["H"], case["D"]
    lens = s["lens"].tolist()
    span = math.ceil(case["w"])
    if op == "decode8":
        rows = []
        for b in range(B):
            first = max(0, lens[b] - span)
            k, v = (_exact_cache(s, b, x, lens[b])[first:] for x in ("k", "v"))
            back = lens[b] - 1 - torch.arange(first, lens[b], device=k.device)
            rows.append(_exact_query(s["q"][b], k, v, back, s["r"], s["w"]))
        return torch.stack(rows)
    n, q8 = case["n"], s["k_scales"] is not None
    if B * n * min(case["T"], case["w"]) * H * D > 1.2e11:
        return None
    y = torch.zeros(B, n, H, D, dtype=torch.float64, device=s["q"].device)
    held = torch.bfloat16 if case["dtype"] == "bf16" else torch.float32
    parents = s["parents"].tolist()
    for b in range(B):
        first = max(0, lens[b] - span)
        k, v = (_exact_cache(s, b, x, lens[b])[first:] for x in ("k", "v"))
        new = [_exact_rows(s[x][b], q8) for x in ("k", "v")]
        if not q8:                                    # as the pages hold them
            new = [x.to(held).double() for x in new]
        lines = []
        for i in range(n):
            up = parents[b][i]
            line = [i] if up == -1 else lines[up] + [i] if 0 <= up < i and lines[up] else []
            lines.append(line)
            if not line:
                continue
            p = lens[b] + len(line) - 1
            back = torch.cat([p - torch.arange(first, lens[b], device=k.device), torch.arange(len(line) - 1, -1, -1, device=k.device)])
            y[b, i] = _exact_query(s["q"][b, i], torch.cat([k, new[0][line]]), torch.cat([v, new[1][line]]), back, s["r"], s["w"])
    return {"y": y, "k_pages": None, "v_pages": None} | ({"k_scales": None, "v_scales": None} if q8 else {})
