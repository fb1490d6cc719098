"""The speculative-serving operators together, as generation uses them: tree
steps over the cache, verification, the accepted path kept, int8 caches."""
import pytest
import torch

from oracle import paged_oracle as po
from tests.conftest import rel_err

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


def lm(ms, dtype, layers=2, d=64, heads=2, vocab=97, seed=0, max_len=160):
    torch.manual_seed(seed)
    m = ms.MultiscreenLM(vocab, d_model=d, num_heads=heads, num_layers=layers, max_seq_len=max_len).to(DEV)
    with torch.no_grad():
        for p in m.token_emb.parameters():
            p.mul_(20.0)                       # tied head: logits of order one
        for blk in m.blocks:
            blk.attn.s_r.fill_(-2.0)           # r = 1.14: most of a window is seen
    return m.to(dtype).eval()


# fp32: the 1e-4 contract of the fp32 path; bf16: 2e-2 of the largest logit, as
# the other model tests hold decode against recompute
TOL = {torch.float32: 1e-4, torch.bfloat16: 2e-2}


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("quantize", [None, "int8"])
@pytest.mark.parametrize("B,n", [(2, 3), (3, 7)])
def test_chain_step_equals_single_steps(ms, dtype, quantize, B, n):
    m = lm(ms, dtype)
    ids = torch.randint(0, 97, (B, 40), device=DEV)
    caches = [m.make_cache(B, 80, quantize=quantize, max_draft=n) for _ in range(2)]
    for c in caches:
        m.prefill(ids[:, :30], c)
    chain = ids[:, 30:30 + n]
    lens = torch.full((B,), 30, dtype=torch.int32, device=DEV)
    a = m.tree_step(chain, lens, caches[0])
    b = torch.stack([m.decode_step(chain[:, i:i + 1], lens + i, caches[1]) for i in range(n)], 1)
    assert a.shape == b.shape == (B, n, 97)
    assert rel_err(a.float(), b.float()) <= TOL[dtype]
    if quantize is None:
        whole = m(ids[:, :30 + n])["logits"][:, 30:]
        assert rel_err(a.float(), whole.float()) <= TOL[dtype]


@pytest.mark.parametrize("quantize", [None, "int8"])
def test_tree_verify_commit_round(ms, quantize):
    """A tree's nodes have the logits of their own paths; after the accepted path
    is committed the next step gives what a cache of its tokens gives."""
    m = lm(ms, torch.float32)
    B, n, T = 3, 9, 24
    g = torch.Generator(device=DEV).manual_seed(3)
    ids = torch.randint(0, 97, (B, T), device=DEV, generator=g)
    parents = torch.tensor([[-1, 0, 0, 1, 1, 2, 4, 6, -2]] * B, dtype=torch.int32, device=DEV)
    parents[1] = torch.tensor([-1, 0, 1, 2, 3, 4, 5, 6, 7])
    tokens = torch.randint(0, 97, (B, n), device=DEV, generator=g)
    cache = m.make_cache(B, 64, quantize=quantize, max_draft=n - 1)
    m.prefill(ids, cache)
    lens = torch.full((B,), T, dtype=torch.int32, device=DEV)
    logits = m.tree_step(tokens, lens, cache, parents=parents)
    for b in range(B):
        for i, line in enumerate(po.ancestors(parents[b], n)):
            if not line:
                continue
            solo = m.make_cache(1, 64, quantize=quantize)
            m.prefill(ids[b:b + 1], solo)
            path = tokens[b, line]
            for k, t in enumerate(path):
                one = m.decode_step(t.view(1, 1), T + k, solo)
            assert rel_err(logits[b, i].float(), one[0].float()) <= TOL[torch.float32], (b, i)
    # keep a path per sequence, as verification would return it
    path = torch.tensor([[0, 1, 4, 6, 7, -1, -1, -1, -1], [0, 1, 2, -1, -1, -1, -1, -1, -1],
                         [0, 2, 5, -1, -1, -1, -1, -1, -1]], dtype=torch.int32, device=DEV)
    counts = torch.tensor([5, 3, 3], dtype=torch.int32, device=DEV)
    cache.commit(lens, path, counts)
    nxt = torch.randint(0, 97, (B, 1), device=DEV, generator=g)
    got = m.decode_step(nxt, lens + counts, cache)
    for b in range(B):
        solo = m.make_cache(1, 64, quantize=quantize)
        m.prefill(ids[b:b + 1], solo)
        for k, t in enumerate(tokens[b, path[b, :int(counts[b])].long()]):
            m.decode_step(t.view(1, 1), T + k, solo)
        want = m.decode_step(nxt[b:b + 1], T + int(counts[b]), solo)
        assert rel_err(got[b].float(), want[0].float()) <= TOL[torch.float32]


def test_cache_tree_needs_room(ms):
    m = lm(ms, torch.float32)
    cache = m.make_cache(1, 40, max_draft=2)
    with pytest.raises(ValueError):
        m.tree_step(torch.zeros(1, 4, dtype=torch.long, device=DEV),
                    torch.zeros(1, dtype=torch.int32, device=DEV), cache)
    with pytest.raises(ValueError):
        m.make_cache(1, 40, quantize="int4")
    with pytest.raises(ValueError):
        m.make_cache(1, 40, max_draft=-1)


def test_int8_cache_is_smaller_and_reads_back(ms):
    m = lm(ms, torch.bfloat16)
    ids = torch.randint(0, 97, (2, 50), device=DEV)
    plain, small = m.make_cache(2, 60), m.make_cache(2, 60, quantize="int8")
    assert small.nbytes() * 32 == plain.nbytes() * 18      # (32 + 4) of 64 bytes a row, D = 32
    m.prefill(ids, plain)
    m.prefill(ids, small)
    pos = torch.full((2,), 45, dtype=torch.int32, device=DEV)
    for a, b in zip(plain.read(0, pos, 5), small.read(0, pos, 5)):
        assert a.dtype == b.dtype == torch.bfloat16 and a.shape == (2, 5, 2, 32)
        # int8: half a step of max|x| / 127 <= |x| / 127 an element, then to unit
        # length (twice that at most); bf16: 2^-8 of an element on either side
        assert float((a.float() - b.float()).abs().max()) <= 2 * 0.5 / 127 + 2 * 2.0**-8


@pytest.mark.parametrize("quantize", [None, "int8"])
def test_generate_on_an_int8_cache_graph_equals_eager(ms, quantize):
    m = lm(ms, torch.bfloat16)
    ids = torch.randint(0, 97, (2, 20), device=DEV)
    out = [m.generate(ids, 12, top_k=1, cuda_graph=g, cache_quantize=quantize) for g in (True, False)]
    assert out[0].shape == (2, 32) and torch.equal(out[0], out[1])


@pytest.mark.parametrize("quantize", [None, "int8"])
@pytest.mark.parametrize("graph", [True, False])
@pytest.mark.parametrize("num_draft", [1, 4, 9])
def test_greedy_speculation_equals_greedy_generation(ms, quantize, graph, num_draft):
    m, d = lm(ms, torch.float32), lm(ms, torch.float32, layers=1, seed=0)
    ids = torch.randint(0, 97, (3, 17), device=DEV, generator=torch.Generator(device=DEV).manual_seed(1))
    want = m.generate(ids, 25, top_k=1, cache_quantize=quantize)
    got = m.generate_speculative(ids, d, 25, num_draft=num_draft, temperature=0.0, cuda_graph=graph,
                                 cache_quantize=quantize)
    assert torch.equal(got, want)
    # the model drafting for itself
    assert torch.equal(m.generate_speculative(ids, m, 25, num_draft=num_draft, temperature=0.0,
                                              cuda_graph=graph, cache_quantize=quantize), want)


def test_sampled_speculation_graph_equals_eager(ms):
    m, d = lm(ms, torch.bfloat16), lm(ms, torch.bfloat16, layers=1)
    ids = torch.randint(0, 97, (2, 30), device=DEV)
    runs = [m.generate_speculative(ids, d, 30, num_draft=3, temperature=0.9, top_k=20, cuda_graph=g,
                                   generator=torch.Generator(device=DEV).manual_seed(5))
            for g in (True, False)]
    assert runs[0].shape == (2, 60) and torch.equal(runs[0], runs[1])
    assert torch.equal(runs[0][:, :30], ids) and int(runs[0].max()) < 97 and int(runs[0].min()) >= 0


def test_to_the_last_position(ms):
    """Drafts past max_seq_len are made and dropped."""
    m, d = lm(ms, torch.float32, max_len=40), lm(ms, torch.float32, layers=1, max_len=40)
    ids = torch.randint(0, 97, (2, 21), device=DEV)
    want = m.generate(ids, 20, top_k=1)
    assert torch.equal(m.generate_speculative(ids, d, 20, num_draft=6, temperature=0.0), want)
    with pytest.raises(IndexError):
        m.generate_speculative(ids, d, 21, num_draft=2)
    with pytest.raises(ValueError):
        m.generate_speculative(ids, d, 5, num_draft=0)


def test_speculative_samples_follow_the_model(ms):
    """The second generated token of 6000 copies of a prompt, drafted by another
    model: distributed as the model's own (chi-square over the 8 tokens that
    top_k leaves, 7 degrees: 24.3 is exceeded once in 1000)."""
    m, d = lm(ms, torch.float32, vocab=24), lm(ms, torch.float32, layers=1, vocab=24, seed=9)
    ids = torch.randint(0, 24, (1, 6), device=DEV, generator=torch.Generator(device=DEV).manual_seed(2))
    N = 6000
    out = m.generate_speculative(ids.expand(N, 6).contiguous(), d, 2, num_draft=2, top_k=8, cuda_graph=False,
                                 generator=torch.Generator(device=DEV).manual_seed(4))
    first, second = out[:, 6], out[:, 7]
    seen = torch.zeros(24, dtype=torch.double)
    want = torch.zeros(24, dtype=torch.double)
    for t in first.unique().tolist():
        here = second[first == t]
        lg = m(torch.cat([ids, torch.tensor([[t]], device=DEV)], 1))["logits"][0, -1].detach().double()
        lg = lg.masked_fill(lg < lg.topk(8).values[-1], float("-inf"))
        if t == first.mode().values.item():
            want = lg.softmax(-1).cpu() * len(here)
            seen = torch.bincount(here.cpu(), minlength=24).double()
    ok = want > 0
    assert seen[~ok].sum() == 0
    assert float(((seen - want)[ok] ** 2 / want[ok]).sum()) < 24.3


@pytest.mark.parametrize("graph", [True, False])
def test_rows_without_a_distribution_yield_minus_one(ms, graph):
    """A model whose logits are NaN: the tokens say so, nothing is looked up with
    them; with a drafting model of that kind the tokens are the model's own."""
    m, d = lm(ms, torch.float32), lm(ms, torch.float32, layers=1)
    ids = torch.randint(0, 97, (2, 17), device=DEV)
    want = m.generate(ids, 9, top_k=1)
    with torch.no_grad():
        d.norm.weight.fill_(float("nan"))
    assert torch.equal(m.generate_speculative(ids, d, 9, num_draft=3, temperature=0.0, cuda_graph=graph), want)
    out = d.generate_speculative(ids, m, 9, num_draft=3, cuda_graph=graph)
    assert torch.equal(out[:, :17], ids) and (out[:, 17:] == -1).all()


def test_drafts_are_verified_against_the_rows_they_were_drawn_from(ms, monkeypatch):
    """An fp32 drafting model under a bf16 model: its rows are not rounded."""
    m, d = lm(ms, torch.bfloat16), lm(ms, torch.float32, layers=1)
    ids = torch.randint(0, 97, (2, 17), device=DEV)
    seen = []
    import sys
    mod = sys.modules[type(m).__module__]
    real = mod.verify_drafts

    def spy(logits, *args, **kw):
        seen.append((logits, kw.get("draft_logits")))
        return real(logits, *args, **kw)

    monkeypatch.setattr(mod, "verify_drafts", spy)
    out = m.generate_speculative(ids, d, 4, num_draft=2, cuda_graph=False)
    assert out.shape == (2, 21) and int(out.min()) >= 0
    drawn = [x for x, rows in seen[1:] if rows is None][:2]
    logits, rows = next((x, r) for x, r in seen if r is not None)
    assert logits.dtype == rows.dtype == torch.float32
    assert torch.equal(torch.cat(drawn, 1), rows)


@pytest.mark.parametrize("quantize", [None, "int8"])
def test_serving_loop_of_trees_equals_greedy_generation(ms, quantize):
    """Trees step, are verified and committed round after round, three sequences of
    different progress in one batch, one of them an empty place."""
    m = lm(ms, torch.float32)
    B, T, new, n = 3, 19, 30, 8
    g = torch.Generator(device=DEV).manual_seed(6)
    ids = torch.randint(0, 97, (B, T), device=DEV, generator=g)
    want = m.generate(ids, new + n, top_k=1, cache_quantize=quantize)
    cache = m.make_cache(B, T + new + 2 * n, quantize=quantize, max_draft=n - 1)
    lens = torch.full((B,), T, dtype=torch.int32, device=DEV)
    last = m.prefill(ids, cache).argmax(-1)
    lens[2] = -1                                        # nobody sits there
    got = [[int(last[b])] for b in range(B)]
    parents = torch.tensor([[-1, 0, 0, 1, 1, 4, 5, 2]] * B, dtype=torch.int32, device=DEV)
    parents[1, 5:] = -2                                 # a smaller tree
    good = [[0, 1, 4, 5, 6], [0, 2, 7]]                 # the true tokens sit on one of these paths
    counted = 0
    for turn in range(2 * new):
        if min(len(got[b]) for b in range(2)) >= new:
            break
        tokens = torch.randint(0, 97, (B, n), device=DEV, generator=g)
        tokens[:, 0] = last
        for b in range(2):
            for k, node in enumerate(good[(turn + b) % 2][:1 + turn % 5]):
                tokens[b, node] = int(want[b, T + len(got[b]) - 1 + k]) if T + len(got[b]) - 1 + k < want.shape[1] else 0
        logits = m.tree_step(tokens, lens, cache, parents=parents)
        u = torch.rand(B, n, device=DEV, generator=g)
        out, path, counts = ms.verify_drafts(logits, tokens[:, 1:], parents[:, 1:] - 1, u, temperature=0.0)
        kept = torch.cat([torch.zeros_like(path[:, :1]), path + 1], 1)
        cache.commit(lens, kept, counts + 1)
        counted += int(counts[:2].sum())
        for b in range(2):
            if len(got[b]) < new:
                a = int(counts[b])
                got[b] += out[b, :a + 1].tolist()
                last[b] = out[b, a]
                lens[b] += a + 1
    for b in range(2):
        assert got[b][:new] == want[b, T:T + new].tolist()
    assert counted > new // 2                           # drafts were accepted


@pytest.mark.parametrize("graph", [True, False])
def test_int32_prompts(ms, graph):
    """A prompt may be int32, as for generate()."""
    m, d = lm(ms, torch.float32), lm(ms, torch.float32, layers=1)
    ids = torch.randint(0, 97, (2, 17), device=DEV)
    want = m.generate(ids.int(), 9, top_k=1)
    got = m.generate_speculative(ids.int(), d, 9, num_draft=3, temperature=0.0, cuda_graph=graph)
    assert got.dtype == want.dtype and torch.equal(got, want)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_tree_step_near_the_end(ms, dtype):
    """Nodes past max_seq_len and absent nodes with negative tokens leave the others'
    logits alone."""
    m = lm(ms, dtype, max_len=24)
    ids = torch.randint(0, 97, (2, 22), device=DEV, generator=torch.Generator(device=DEV).manual_seed(8))
    lens = torch.full((2,), 22, dtype=torch.int32, device=DEV)
    tokens = torch.tensor([[5, 6, 7, -1], [8, 9, 10, -1]], device=DEV)
    parents = torch.tensor([[-1, 0, 1, -2]] * 2, dtype=torch.int32, device=DEV)
    caches = [m.make_cache(2, 30, max_draft=3) for _ in range(2)]
    for c in caches:
        m.prefill(ids, c)
    a = m.tree_step(tokens, lens, caches[0], parents=parents)
    b = torch.stack([m.decode_step(tokens[:, i:i + 1], lens + i, caches[1]) for i in range(2)], 1)
    assert a.isfinite().all() and rel_err(a[:, :2].float(), b.float()) <= TOL[dtype]
