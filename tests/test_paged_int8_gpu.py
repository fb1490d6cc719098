"""int8 rows of the paged cache: written, read back and decoded over, against
the 64-bit restatement."""
import math

import pytest
import torch

from oracle import paged_oracle as po

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


def empty_cache(B, H, D, ps, blocks, seed=0, fill=7):
    g = torch.Generator().manual_seed(seed)
    P = B * blocks
    table = torch.randperm(P, generator=g).view(B, blocks).to(torch.int32).to(DEV)
    kp = torch.full((P, H, ps, D), fill, dtype=torch.int8, device=DEV)
    vp = kp.clone()
    ks = torch.full((P, H, ps), 0.5, device=DEV)
    return kp, vp, table, ks, ks.clone()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("B,n,H,D,ps", [(1, 1, 1, 64, 64), (3, 5, 2, 16, 8), (2, 67, 3, 32, 24),
                                        (2, 130, 2, 128, 100), (4, 33, 16, 64, 16)])
def test_append_and_read(ms, dtype, B, n, H, D, ps):
    g = torch.Generator().manual_seed(n * D + ps)
    qkv = (torch.randn(B, n, 3, H, D, generator=g) * 3).to(dtype).to(DEV)
    k, v = qkv[:, :, 1], qkv[:, :, 2]            # strided views
    pos = torch.arange(B, dtype=torch.int32) * 2
    blocks = (n + 2 * B) // ps + 2
    kp, vp, table, ks, vs = empty_cache(B, H, D, ps, blocks)
    ms.paged_append(k, v, pos.to(DEV), kp, vp, table, ks, vs)
    got = ms.paged_read(pos.to(DEV), n, kp, vp, table, ks, vs)
    half = ms.paged_read(pos.to(DEV), n, kp, vp, table, ks, vs, dtype=torch.bfloat16)
    for raw, pages, scales, val, val16 in ((k, kp, ks, got[0], half[0]), (v, vp, vs, got[1], half[1])):
        m, sc = po.int8_rows(raw)
        for b in range(B):
            p = torch.arange(n) + int(pos[b])
            page = table[b].cpu().long()[p // ps]
            assert torch.equal(pages[page.to(DEV), :, (p % ps).to(DEV)].cpu(), m[b])
            # sqrt, maximum, reciprocal: three roundings of half a step each
            s = scales[page.to(DEV), :, (p % ps).to(DEV)].double().cpu()
            assert ((s - sc[b]).abs() <= 3 * 2.0**-24 * sc[b]).all()
        want = m.double() * sc[..., None]
        assert ((val.double().cpu() - want).abs() <= 4 * 2.0**-24 * want.abs()).all()
        assert ((val16.double().cpu() - want).abs() <= (2.0**-8 + 2.0**-21) * want.abs()).all()
    # everything else was left alone
    touched = sum(int((x != 7).any(-1).sum()) for x in (kp, vp))
    assert touched <= 2 * B * n * H


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_append_extreme_rows(ms, dtype):
    """zero, tiny (subnormal), huge rows, ties of the rounding, rows below eps,
    and rows with an infinity or NaN."""
    D = 64
    rows = torch.randn(12, D, generator=torch.Generator().manual_seed(1))
    rows[0] = 0.0
    rows[1] *= 1e-39
    rows[2] = rows[2].clamp(-1, 1) * 3e38
    rows[3] = 0.0
    rows[3, :5] = torch.tensor([254.0, 1.0, 3.0, -5.0, 127.0])   # halves: 0.5, 1.5, -2.5, 63.5
    rows[4] *= 1e-10                                              # norm below eps = 1e-8
    rows[5, 7] = math.inf
    rows[6, 9] = math.nan
    rows[7] = 0.0
    rows[7, 63] = -1e-45
    rows[8] *= 1e-33
    rows[9, 0] = -math.inf
    x = rows.to(dtype).view(1, 12, 1, D)
    kp, vp, table, ks, vs = empty_cache(1, 1, D, 16, 1)
    pos = torch.zeros(1, dtype=torch.int32, device=DEV)
    ms.paged_append(x.to(DEV), x.to(DEV), pos, kp, vp, table, ks, vs)
    m, sc = po.int8_rows(x[0, :, 0])
    page = int(table[0, 0])
    assert torch.equal(kp[page, 0, :12].cpu(), m) and torch.equal(vp[page, 0, :12].cpu(), m)
    got = ks[page, 0, :12].double().cpu()
    assert torch.equal(got.isnan(), sc.isnan()) and int(sc.isnan().sum()) == 3
    ok = ~sc.isnan()
    # below the smallest normal number a step is 2^-149
    assert ((got - sc)[ok].abs() <= 5 * 2.0**-24 * sc[ok] + 2.0**-149).all()
    val = ms.paged_read(pos, 12, kp, vp, table, ks, vs)[0][0, :, 0]
    assert val[5].isnan().all() and val[6].isnan().all() and (val[0] == 0).all()


def test_positions_outside_the_table_are_skipped(ms):
    B, H, D, ps, blocks = 3, 2, 64, 16, 2
    kp, vp, table, ks, vs = empty_cache(B, H, D, ps, blocks)
    table[2, 1] = -1                                   # a page that is not there
    table[1, 0] = 10_000
    before = [t.clone() for t in (kp, vp, ks, vs)]
    k = torch.randn(B, 4, H, D, device=DEV)
    pos = torch.tensor([-2, 14, 30], dtype=torch.int32, device=DEV)
    ms.paged_append(k, k, pos, kp, vp, table, ks, vs)
    val = ms.paged_read(pos, 4, kp, vp, table, ks, vs)[0]
    there = torch.tensor([[0, 0, 1, 1], [0, 0, 1, 1], [0, 0, 0, 0]], dtype=torch.bool, device=DEV)
    assert torch.equal((val != 0).any(-1).any(-1), there)
    assert int((kp != before[0]).any(-1).sum()) <= int(there.sum()) * H
    ms.paged_append(k[:0], k[:0], pos[:0], kp, vp, table[:0], ks, vs)      # nothing to do
    ms.paged_append(k[:, :0], k[:, :0], pos, kp, vp, table, ks, vs)


def _filled(ms, B, H, D, ps, T, dtype, seed, extra=0):
    """An int8 cache of T rows per sequence written by paged_append."""
    g = torch.Generator().manual_seed(seed)
    k = torch.randn(B, max(T, 1), H, D, generator=g)
    k += 0.7 * torch.randn(H, D, generator=g)
    v = torch.randn(B, max(T, 1), H, D, generator=g)
    blocks = (T + extra) // ps + 1
    c = empty_cache(B, H, D, ps, blocks, seed, fill=0)
    kp, vp, table, ks, vs = c
    ms.paged_append(k[:, :T].to(dtype).to(DEV), v[:, :T].to(dtype).to(DEV),
                    torch.zeros(B, dtype=torch.int32, device=DEV), kp, vp, table, ks, vs)
    return c, k.to(dtype), g


def bound(y, sums, r, dtype, i8):
    """The row norm that the kernel's roundings may move: the output's half
    step (bf16 2^-8), alpha's (fp16 2^-11, bf16 2^-8; hi + lo 2^-21), the scores' 32-bit sums
    (2^-18 of |q||k|, through t) and the mask's (2^-21)."""
    out = 2.0**-8 if dtype == torch.bfloat16 else 2.0**-22
    al = 2.0**-21 if dtype == torch.float32 else 2.0**-11 if i8 else 2.0**-8
    return (out * y.norm(dim=-1) + al * sums[..., 0] + 2.0**-18 * r.abs() * sums[..., 1]
            + 2.0**-21 * sums[..., 2] + 1e-9)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("B,H,D,ps,T,w", [(1, 1, 64, 64, 1, 2.0), (3, 2, 64, 64, 300, 130.5),
                                          (2, 3, 16, 8, 77, 500.0), (2, 2, 32, 24, 129, 64.0),
                                          (2, 2, 128, 100, 333, 1000.0), (1, 2, 64, 16, 1500, 1500.0)])
@pytest.mark.parametrize("ctas", [None, 1, 5])
def test_decode(ms, dtype, B, H, D, ps, T, w, ctas):
    (kp, vp, table, ks, vs), k, g = _filled(ms, B, H, D, ps, T, dtype, T + D)
    lens = torch.tensor([max(1, T - 11 * b) for b in range(B)], dtype=torch.int32)
    q = (k[:, -1] + 0.6 * torch.randn(B, H, D, generator=g)).to(dtype)
    r = torch.linspace(1.02, 1.9, H)
    ww = torch.linspace(w, max(1.5, w / 7), H)
    y = ms.paged_decode(q.to(DEV), lens.to(DEV), r.to(DEV), ww.to(DEV), kp, vp, table, ks, vs,
                        max_window=w, num_ctas=ctas)
    cache = (kp.cpu(), vp.cpu(), ks.cpu(), vs.cpu(), table.cpu())
    for b in range(B):
        t = int(lens[b])
        row = [po.cache_values(cache[0], cache[2], table, b, [t - 1]),
               po.cache_values(cache[1], cache[3], table, b, [t - 1])]
        want, sums = po.tree(q[b:b + 1].expand(1, H, D), row[0], row[1], t - 1, None, r, ww, cache, b)
        err = (y[b].double().cpu() - want[0]).norm(dim=-1)
        assert (err <= bound(want, sums, r, dtype, True)[0]).all(), (b, err)


def test_decode_empty_places(ms):
    """An empty sequence, windows that hold nothing, non-finite parameters and
    query, and a key row with NaN: all give what the keys that are left give."""
    B, H, D = 4, 5, 64
    (kp, vp, table, ks, vs), k, g = _filled(ms, B, H, D, 16, 40, torch.bfloat16, 3)
    lens = torch.tensor([0, 40, -3, 40], dtype=torch.int32, device=DEV)
    q = k[:, 38].clone()
    q[3, 1, 5] = math.nan
    r = torch.tensor([1.2, 1.2, 1.2, math.nan, 1.2], device=DEV)
    w = torch.tensor([20.0, 64.0, 0.0, 20.0, math.nan], device=DEV)
    y = ms.paged_decode(q.to(DEV), lens, r, w, kp, vp, table, ks, vs)
    assert y.isfinite().all()
    assert (y[0] == 0).all() and (y[2] == 0).all() and (y[:, 2:] == 0).all()
    assert (y[3, 1] == 0).all() and (y[1, :2] != 0).any(-1).all()
    # a NaN row in K is not seen; in V it shows only where it is seen
    page, row = int(table[1, 36 // 16]), 36 % 16
    ks[page, 0, row] = math.nan
    vs[page, 1, row] = math.nan
    y2 = ms.paged_decode(q.to(DEV), lens, r, w, kp, vp, table, ks, vs)
    assert y2[1, 0].isfinite().all() and torch.equal(y2[3], y[3])
    near = ms.paged_decode(q.to(DEV), lens, r, torch.full((H,), 3.0, device=DEV), kp, vp, table, ks, vs)
    assert near[1, 1].isfinite().all()            # the window ends before it


def test_every_bf16_quotient(ms):
    """All pairs of 8-bit significands, eight binades down: the integers are those
    of the exact quotient, halves to even."""
    A = torch.arange(128, 256).repeat_interleave(8)                     # a row's largest value
    X = torch.arange(128, 256)
    shift = torch.arange(8).repeat(128)
    rows = (X[None] * 2.0 ** -shift[:, None].float()).clamp(max=A[:, None].float())
    rows[:, 5] = A.float()
    rows[:, ::3] *= -1
    k = rows.view(1, 1024, 1, 128).to(torch.bfloat16)
    assert torch.equal(k.float().view(1024, 128), rows)
    kp, vp, table, ks, vs = empty_cache(1, 1, 128, 64, 16)
    ms.paged_append(k.to(DEV), (k * 2.0**-60).to(DEV), torch.zeros(1, dtype=torch.int32, device=DEV), kp, vp, table, ks, vs)
    # 127 |x| / A = n / A' in integers, rounded half to even
    num, den = (127 * rows.abs() * 2.0**shift[:, None].float()).long(), (A << shift)[:, None]
    q, rest = num // den, num % den
    want = (q + ((2 * rest > den) | ((2 * rest == den) & (q % 2 == 1))).long()) * rows.sign().long()
    for pages in (kp, vp):
        assert torch.equal(pages[table[0].long()].cpu().view(1024, 128).long(), want)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("D", [16, 64, 128])
def test_scales_are_rounded_once(ms, dtype, D):
    """|m|^2 is a whole number below 2^21, exact in 32 bits; 1 / |m| is off by one
    rounding (2^-24) and 2^-44, the square of the approximate root's error."""
    n, H = 500, 8
    x = torch.randn(1, n, H, D, generator=torch.Generator().manual_seed(D)).to(dtype)
    kp, vp, table, ks, vs = empty_cache(1, H, D, 64, n // 64 + 1)
    ms.paged_append(x.to(DEV), x.flip(1).to(DEV), torch.zeros(1, dtype=torch.int32, device=DEV), kp, vp, table, ks, vs)
    for scales, rows in ((ks, x), (vs, x.flip(1))):
        _, want = po.int8_rows(rows[0])                                          # (n, H)
        got = scales[table[0].long()].transpose(1, 2).reshape(-1, H)[:n].double().cpu()
        assert ((got - want).abs() <= (1 + 2.0**-16) * 2.0**-24 * want).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("H", [40, 150])
def test_more_heads_than_a_block_moves_at_once(ms, dtype, H):
    """A token's heads go through a block in several turns."""
    B, n, D, ps = 2, 3, 128, 16
    g = torch.Generator().manual_seed(H)
    k, v = (torch.randn(B, n, H, D, generator=g).to(dtype) for _ in range(2))
    pos = torch.tensor([14, 3], dtype=torch.int32)
    kp, vp, table, ks, vs = empty_cache(B, H, D, ps, 2)
    ms.paged_append(k.to(DEV), v.to(DEV), pos.to(DEV), kp, vp, table, ks, vs)
    got = ms.paged_read(pos.to(DEV), n, kp, vp, table, ks, vs)
    for raw, pages, scales, val in ((k, kp, ks, got[0]), (v, vp, vs, got[1])):
        m, sc = po.int8_rows(raw)
        for b in range(B):
            p = torch.arange(n) + int(pos[b])
            page = table[b].cpu().long()[p // ps]
            assert torch.equal(pages[page.to(DEV), :, (p % ps).to(DEV)].cpu(), m[b])
        want = m.double() * sc[..., None]
        assert ((val.double().cpu() - want).abs() <= 4 * 2.0**-24 * want.abs()).all()
    assert int((kp != 7).any(-1).sum()) <= B * n * H


@pytest.mark.parametrize("page,out", [(torch.float32, torch.bfloat16), (torch.bfloat16, torch.float32),
                                      (torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16)])
@pytest.mark.parametrize("H,D,ps", [(3, 16, 8), (5, 128, 24), (70, 64, 16)])
def test_read_of_other_pages(ms, H, D, ps, page, out):
    B, n = 2, 37
    g = torch.Generator().manual_seed(H)
    P = B * 4
    table = torch.randperm(P, generator=g).view(B, 4).to(torch.int32)
    table[1, 2] = -1
    kp, vp = (torch.randn(P, H, ps, D, generator=g).to(page) for _ in range(2))
    pos = torch.tensor([-3, ps - 1], dtype=torch.int32)
    got = ms.paged_read(pos.to(DEV), n, kp.to(DEV), vp.to(DEV), table.to(DEV), dtype=out)
    for pages, x in zip((kp, vp), got):
        assert x.dtype == out and x.shape == (B, n, H, D)
        for b in range(B):
            want = po.cache_values(pages, None, table, b, [int(pos[b]) + i for i in range(n)]).nan_to_num(0.0)
            assert torch.equal(x[b].cpu(), want.float().to(out))
