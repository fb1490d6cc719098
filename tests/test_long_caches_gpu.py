"""Decode and trees over caches of 20K to 100K keys, against the restatement in 64
bits.  All keys but some thirty are trimmed: those few, at the ends of the cache, of
pages and of tiles and anywhere else, make up the output, so that one of them missed,
or one other seen, shows."""
import math

import pytest
import torch

from oracle import paged_oracle as po

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


def rows_of(pages, scales, table, b, h, first, end):
    """float64 rows of positions [first, end) of head h."""
    ps = pages.shape[2]
    pos = torch.arange(first, end, device=DEV)
    page = table[b].long()[pos // ps]
    x = pages[page, h, pos % ps].double()
    return x if scales is None else x * scales[page, h, pos % ps].double()[:, None]


CASES = [(100_003, 0, torch.bfloat16, True, 64, 64), (100_003, 0, torch.bfloat16, True, 24, 64),
         (60_001, 0, torch.float32, True, 64, 128), (60_001, 0, torch.bfloat16, False, 64, 64),
         (100_003, 5, torch.bfloat16, True, 64, 64), (32_771, 5, torch.bfloat16, False, 24, 64),
         (32_771, 16, torch.bfloat16, False, 64, 64), (32_771, 20, torch.bfloat16, True, 64, 128),
         (32_771, 24, torch.float32, True, 100, 64), (32_771, 64, torch.bfloat16, True, 64, 64),
         (32_771, 64, torch.bfloat16, True, 16, 32), (20_001, 40, torch.bfloat16, False, 64, 64),
         (20_001, 24, torch.float32, False, 64, 64)]


@pytest.mark.parametrize("T,n,dtype,q8,ps,D", CASES)
def test_long(ms, T, n, dtype, q8, ps, D):
    B, H = 2, 3
    g = torch.Generator().manual_seed(T + n + ps)
    dev = torch.Generator(device=DEV).manual_seed(T + n + ps)
    lens = torch.tensor([T, T - 4097], dtype=torch.int32)
    lead = torch.randn(B, 1, H, D, generator=g)
    # the leading direction for a few, its opposite for all others
    sign = torch.full((B, T, H, 1), -1.0)
    for b in range(B):
        L = int(lens[b])
        at = torch.cat([torch.randint(0, L, (20,), generator=g),
                        torch.tensor([0, 31, 32, 63, 64, ps - 1, ps, L - 1, L - 2, L - ps, L // 2 // 64 * 64, L // 2 // 64 * 64 - 1])])
        sign[b, at] = 1.0
    k = torch.randn(B, T, H, D, device=DEV, generator=dev) * 0.4 + (lead * sign).to(DEV)
    v = torch.randn(B, T, H, D, device=DEV, generator=dev)
    blocks = (T + n) // ps + 1
    table = torch.randperm(B * blocks, generator=g).view(B, blocks).to(torch.int32).to(DEV)
    kp = torch.zeros(B * blocks, H, ps, D, dtype=torch.int8 if q8 else dtype, device=DEV)
    vp = torch.zeros_like(kp)
    ks, vs = [torch.zeros(B * blocks, H, ps, device=DEV) if q8 else None for _ in range(2)]
    ms.paged_append(k.to(dtype), v.to(dtype), torch.zeros(B, dtype=torch.int32, device=DEV), kp, vp, table, ks, vs)
    del k, v
    q = (lead + 0.3 * torch.randn(B, max(n, 1), H, D, generator=g)).to(dtype)
    own = (-lead).expand(B, n, H, D).to(dtype)                   # trimmed: nodes see the cache alone
    r, w = torch.full((H,), 1.3), torch.tensor([3.0 * T, T / 2 + 0.5, 1000.0])
    rest = (r.to(DEV), w.to(DEV), kp, vp, table, ks, vs)
    if n:
        parents = torch.stack([torch.randint(-1, i, (), generator=g) if i else torch.tensor(-1) for i in range(n)])
        parents = parents.to(torch.int32).expand(B, n).contiguous()
        y = ms.paged_tree_decode(q.to(DEV), own.to(DEV), own.to(DEV), lens.to(DEV), parents.to(DEV), *rest, max_window=3.0 * T)
        depth = [len(x) - 1 for x in po.ancestors(parents[0], n)]
    else:
        y = ms.paged_decode(q[:, 0].to(DEV), lens.to(DEV), *rest, max_window=3.0 * T)[:, None]
        depth = [-1]
    for b in range(B):
        L = int(lens[b])
        for h in range(H):
            K, V = (rows_of(p, s, table, b, h, 0, L) for p, s in ((kp, ks), (vp, vs)))
            qq = q[b, :, h].to(DEV).double()
            qq = qq / qq.norm(dim=-1, keepdim=True)
            t = 1 - float(r[h]) * (1 - qq @ K.T)                                      # (n, L)
            back = L + torch.tensor(depth, device=DEV)[:, None] - torch.arange(L, device=DEV)
            seen = (back >= 0) & (back <= math.ceil(float(w[h])) - 1) & (t > 0)
            m = 0.5 * (1 + torch.cos(math.pi * back.double() / float(w[h])))
            a = torch.where(seen, t * t * m, 0.0)
            o = a @ V
            size = o.norm(dim=-1, keepdim=True)
            want = torch.tanh(size) / size.clamp_min(1e-8) * o
            # the output's half step; 2^-18 of a score's terms (32-bit sums), r / t times over
            # in alpha; 2^-20 of alpha (12 half steps) and 2^-23 for each of the sums of a few
            # dozen live terms; all over max(1, |o|), which TanhNorm divides by
            va = V.abs()
            s0, s1 = (a @ va).norm(dim=-1), (torch.where(seen, 2 * t * m, 0.0) @ va).norm(dim=-1)
            out = 2.0**-8 if dtype == torch.bfloat16 else 2.0**-22
            lim = out * want.norm(dim=-1) + (2.0**-18 * float(r[h]) * s1 + (2.0**-20 + 32 * 2.0**-23) * s0) / size[:, 0].clamp_min(1) + 1e-9
            err = (y[b, :, h].double() - want).norm(dim=-1)
            assert (err <= lim).all(), (b, h, float((err / lim).max()))
            if h == 0:
                live = (a > 0).sum(-1)
                assert 20 < int(live.min()) and int(live.max()) < 200
