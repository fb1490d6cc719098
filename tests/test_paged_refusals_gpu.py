"""Python-side refusals of the speculative-serving calls on CUDA tensors: a
request that is refused launches nothing."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


def test_refusals(ms):
    B, n, H, D, ps = 2, 3, 2, 64, 16
    kp = torch.zeros(4, H, ps, D, dtype=torch.bfloat16, device=DEV)
    k8 = kp.to(torch.int8)
    sc = torch.zeros(4, H, ps, device=DEV)
    table = torch.arange(4, dtype=torch.int32, device=DEV).view(2, 2)
    q = torch.randn(B, n, H, D, device=DEV, dtype=torch.bfloat16)
    lens = torch.zeros(B, dtype=torch.int32, device=DEV)
    r = torch.ones(H, device=DEV)
    par = torch.full((B, n), -1, dtype=torch.int32, device=DEV)

    def tree(q=q, k=q, v=q, lens=lens, par=par, r=r, w=r, kp=kp, vp=kp, table=table, ks=None, vs=None, **kw):
        return ms.paged_tree_decode(q, k, v, lens, par, r, w, kp, vp, table, ks, vs, **kw)

    tree()
    bad = [dict(kp=k8, vp=k8), dict(ks=sc, vs=sc), dict(kp=k8, vp=k8, ks=sc), dict(kp=k8, vp=k8, ks=sc, vs=sc.half()),
           dict(kp=kp[..., :32], vp=kp[..., :32]), dict(vp=kp[:2]), dict(lens=lens.long()), dict(lens=lens[:1]),
           dict(par=par.long()), dict(par=par[:, :2]), dict(r=r[:1]), dict(k=None), dict(k=q[:, :2]),
           dict(q=q[..., :32]), dict(table=table.long()), dict(table=table[:1]), dict(table=table.t()),
           dict(q=torch.randn(B, 65, H, D, device=DEV, dtype=torch.bfloat16))]
    for kw in bad:
        with pytest.raises(ValueError):
            tree(**kw)
    for kw in (dict(kp=kp.half(), vp=kp.half()), dict(vp=kp.float()), dict(q=q.float()), dict(q=q.half()),
               dict(k=q.float()), dict(q=q.half(), k=q.half(), v=q.half(), kp=k8, vp=k8, ks=sc, vs=sc)):
        with pytest.raises(TypeError):
            tree(**kw)
    for kw in (dict(q=q.cpu()), dict(lens=lens.cpu()), dict(k=q.cpu()), dict(table=table.cpu()), dict(num_ctas=0)):
        with pytest.raises(RuntimeError):
            tree(**kw)
    with pytest.raises(TypeError):
        ms.paged_append(q.float(), q.float(), lens, kp, kp, table)
    with pytest.raises(ValueError):
        ms.paged_append(q, q.float(), lens, k8, k8, table, sc, sc)
    with pytest.raises(TypeError):
        ms.paged_read(lens, 2, kp, kp, table, dtype=torch.float16)
    with pytest.raises(ValueError):
        ms.paged_read(lens, -1, kp, kp, table)
    with pytest.raises(ValueError):
        ms.paged_decode(q[:, 0, :1], lens, r, r, k8, k8, table, sc, sc)
    with pytest.raises(TypeError):
        ms.paged_decode(q[:, 0].float(), lens, r, r, kp, kp, table)
    with pytest.raises(ValueError):
        ms.paged_commit(lens, torch.zeros(B, 65, dtype=torch.int32, device=DEV), lens, kp, kp, table)
    with pytest.raises(ValueError):
        ms.paged_commit(lens, par.long(), lens, kp, kp, table)


def test_verify_refusals(ms):
    B, n, V = 2, 3, 11
    lg = torch.randn(B, n + 1, V, device=DEV)
    tok = torch.zeros(B, n, dtype=torch.long, device=DEV)
    u = torch.rand(B, n + 1, device=DEV)
    ms.verify_drafts(lg, tok, None, u)
    ms.verify_drafts(lg.half(), tok, None, u)
    assert ms.verify_drafts(lg[:0], tok[:0], None, u[:0])[0].shape == (0, n + 1)
    for a in ((lg, tok.int(), None, u), (lg, tok[:, :2], None, u), (lg, tok, tok, u), (lg, tok, None, u[:, :n]),
              (lg, tok, None, u.double())):
        with pytest.raises(ValueError):
            ms.verify_drafts(*a)
    for kw in (dict(draft_logits=lg), dict(temperature=-0.5), dict(temperature=float("nan")),
               dict(temperature=torch.ones(B + 1, device=DEV)), dict(temperature=torch.ones(B, device=DEV).double())):
        with pytest.raises(ValueError):
            ms.verify_drafts(lg, tok, None, u, **kw)
    with pytest.raises(TypeError):
        ms.verify_drafts(lg, tok, None, u, draft_logits=lg[:, :n].bfloat16())
    with pytest.raises(TypeError):
        ms.verify_drafts(lg.double(), tok, None, u)
    with pytest.raises(RuntimeError):
        ms.verify_drafts(lg, tok.cpu(), None, u)
