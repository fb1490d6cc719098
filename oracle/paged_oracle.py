"""The paged-cache operators of speculative serving restated in 64 bits, one
sequence, head, node or token at a time: int8 rows, a tree of drafted tokens
over the cached prefix, and the acceptance of drafted tokens."""
from __future__ import annotations

import math

import numpy as np
import torch


def int8_rows(x: torch.Tensor, eps: float = 1e-8):
    """(m int8, scale float64) of raw rows x (.., D)."""
    x = x.detach().double().cpu()
    finite = x.isfinite().all(-1, keepdim=True)
    x = torch.where(finite, x, torch.zeros_like(x))
    top = x.abs().amax(-1, keepdim=True)
    m = torch.where(top > 0, torch.round(127.0 * x / torch.where(top > 0, top, torch.ones_like(top))),
                    torch.zeros_like(x))
    floor = torch.where(top > 0, 127.0 * eps / torch.where(top > 0, top, torch.ones_like(top)),
                        torch.full_like(top, math.inf))
    scale = 1.0 / torch.maximum(m.norm(dim=-1, keepdim=True), floor)
    scale = torch.where(finite, scale, torch.full_like(scale, math.nan))
    return m.to(torch.int8), scale[..., 0]


def unit_rows(x: torch.Tensor, eps: float = 1e-8) -> torch.Tensor:
    x = x.detach().double().cpu()
    return x / x.norm(dim=-1, keepdim=True).clamp_min(eps)


def cache_values(pages, scales, block_table, b: int, positions):
    """float64 rows (len(positions), H, D) of sequence b, NaN where there is none."""
    P, H, ps, D = pages.shape
    out = torch.full((len(positions), H, D), math.nan, dtype=torch.float64)
    for i, p in enumerate(positions):
        blk = p // ps
        if p < 0 or blk >= block_table.shape[1]:
            continue
        page = int(block_table[b, blk])
        if not 0 <= page < P:
            continue
        row = pages[page, :, p % ps].double().cpu()
        if scales is not None:
            row = row * scales[page, :, p % ps].double().cpu()[:, None]
        out[i] = row
    return out


def ancestors(parents, n: int):
    """Per node its line (ancestors and itself, root first), [] when absent."""
    lines = []
    for i in range(n):
        p = i - 1 if parents is None else int(parents[i])
        if p == -1:
            lines.append([i])
        elif 0 <= p < i and lines[p]:
            lines.append(lines[p] + [i])
        else:
            lines.append([])
    return lines


def query(q, k, v, back, r: float, w: float, eps: float = 1e-8):
    """One query q (D,) over rows k, v (K, D) standing `back` (K,) positions
    before it.  Returns y (D,) and the sums its rounding bounds are made of:
    norms of sum alpha |v|, sum 2 t m |v| and sum t^2 |v|.  Rows that are not
    seen (outside the window, no row, trimmed) contribute nothing."""
    q = q.detach().double().cpu()
    q = q / max(float(q.norm()), eps)
    t = 1.0 - r * (1.0 - k @ q)
    dmax = math.ceil(w) - 1 if w == w else -1
    seen = (back >= 0) & (back <= dmax) & (t > 0)
    k, v, t, back = k[seen], v[seen], t[seen], back[seen].double()
    m = 0.5 * (1.0 + torch.cos(math.pi * back / w))
    a = t * t * m
    o = (a[:, None] * v).sum(0)
    size = max(float(o.norm()), eps) if o.isfinite().all() else math.nan
    y = math.tanh(size) / size * o
    va = v.abs()
    sums = [float((c[:, None] * va).sum(0).norm()) for c in (a, 2 * t * m, t * t)]
    return y, sums


def tree(q, new_k, new_v, lens: int, parents, r, w, cache, b: int, eps: float = 1e-8):
    """y (n, H, D) float64 and bounds (n, H, 3) of sequence b.  new_k / new_v
    (n, H, D): the nodes' rows as the cache holds them.  cache: (k_pages,
    v_pages, k_scales, v_scales, block_table) holding the prefix."""
    n, H, D = q.shape
    y = torch.zeros(n, H, D, dtype=torch.float64)
    sums = torch.zeros(n, H, 3, dtype=torch.float64)
    if lens < 0:
        return y, sums
    kp, vp, ks, vs, table = cache
    reach = max([math.ceil(float(x)) for x in w.tolist() if x == x and x > 0] + [0])
    first = max(0, lens - reach)
    pos = list(range(first, lens))
    pk, pv = cache_values(kp, ks, table, b, pos), cache_values(vp, vs, table, b, pos)
    lines = ancestors(None if parents is None else parents[b], n)
    for i in range(n):
        if not lines[i]:
            continue
        at = lens + len(lines[i]) - 1
        back = torch.tensor([at - p for p in pos] + list(range(len(lines[i]) - 1, -1, -1)))
        k = torch.cat([pk, new_k[lines[i]]])
        v = torch.cat([pv, new_v[lines[i]]])
        for h in range(H):
            y[i, h], s = query(q[i, h], k[:, h], v[:, h], back, float(r[h]), float(w[h]), eps)
            sums[i, h] = torch.tensor(s)
    return y, sums


def verify(logits, tokens, parents, uniforms, draft_logits=None, temperature=1.0):
    """(tokens, path, counts) as lists for one sequence: logits (n + 1, V),
    tokens (n,), parents (n,) or None, uniforms (n + 1,)."""
    lg = logits.detach().double().cpu().numpy()
    dl = None if draft_logits is None else draft_logits.detach().double().cpu().numpy()
    u = uniforms.detach().double().cpu().numpy()
    n, V = lg.shape[0] - 1, lg.shape[1]

    def dist(x):
        top = x.max()
        if not np.isfinite(top) or np.isnan(x).any():
            return None
        if not temperature > 0:
            p = np.zeros(V)
            p[int(np.argmax(x))] = 1.0
            return p
        with np.errstate(under="ignore"):
            e = np.exp((x - top) / temperature)
        return e / e.sum()

    lines = ancestors(parents, n)
    cur, path, out = 0, [], []
    while True:
        p = dist(lg[cur])
        if p is None:
            return out + [-1], path, len(path)
        q = None if dl is None or cur >= n else dist(dl[cur])
        c, z, rest, nxt = 0.0, 1.0, p.copy(), None
        for i in range(n):
            parent = i - 1 if parents is None else int(parents[i])
            x = int(tokens[i])
            if parent + 1 != cur or not -1 <= parent < i or not 0 <= x < V:
                continue
            if dl is not None and q is None:
                continue
            qx = 1.0 if q is None else q[x]
            if rest[x] > 0 and u[i] * qx * z < rest[x]:
                nxt = i
                break
            if q is None:
                rest[x] = 0.0
            else:
                c += z
                rest = np.maximum(p - c * q, 0.0)
            z = rest.sum()
        if nxt is not None:
            path.append(nxt)
            out.append(int(tokens[nxt]))
            cur = nxt + 1
            continue
        if not z > 0:
            rest = p
        run = np.cumsum(rest)
        over = np.nonzero((run > u[n] * run[-1]) & (rest > 0))[0]
        x = int(over[0]) if len(over) else int(np.nonzero(rest > 0)[0][-1])
        return out + [x], path, len(path)
