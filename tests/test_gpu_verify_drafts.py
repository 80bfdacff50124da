"""Verification of drafted tokens on the GPU against a walk in float64 on the host.

Outputs are whole numbers and have to be equal; the uniforms of the random cases are drawn, not
chosen, so that a comparison lies within float64 rounding of its border with a probability below 10^-9.
"""

import pytest
import torch

from turboquant_pytorch import verify_drafts

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _walk(tokens, target, uniforms, parents=None, draft=None):
    B, T, V = target.shape
    p_all, u = target.double().cpu(), uniforms.double().cpu()
    q_all = draft.double().cpu() if draft is not None else None
    tok = tokens.cpu().tolist()
    paths, counts, nexts = [], [], []
    for b in range(B):
        par = [i - 1 for i in range(T)] if parents is None else \
            (parents if parents.dim() == 1 else parents[b]).cpu().tolist()
        at, path, w = 0, [0], None
        while w is None:
            p = p_all[b, at]
            w, left, spent, hop = p.clone(), 1.0, set(), None
            for i in range(at + 1, T):
                if par[i] != at:
                    continue
                x = tok[b][i]
                px = float(p[x]) if 0 <= x < V else 0.0
                if q_all is not None:
                    qx = float(q_all[b, at, x]) if 0 <= x < V else 0.0
                    if float(u[b, i]) * qx < px:
                        hop = i
                        break
                    w = (p - q_all[b, at]).clamp(min=0)
                    continue
                if x in spent:
                    continue
                if float(u[b, i]) * left < px:
                    hop = i
                    break
                left -= px
                spent.add(x)
                if 0 <= x < V:
                    w[x] = 0.0
            if hop is not None:
                path.append(hop)
                at, w = hop, None
        w = torch.where(w > 0, w, torch.zeros_like(w))
        if not float(w.sum()) > 0:
            w = torch.where(p_all[b, at] > 0, p_all[b, at], torch.zeros_like(w))
        c = w.cumsum(0)
        over = torch.nonzero((c > float(u[b, 0]) * float(c[-1])) & (w > 0))
        pos = torch.nonzero(w > 0)
        nexts.append(int(over[0]) if len(over) else (int(pos[-1]) if len(pos) else -1))
        paths.append(path + [-1] * (T - len(path)))
        counts.append(len(path))
    return (torch.tensor(paths, dtype=torch.int32), torch.tensor(counts, dtype=torch.int32), torch.tensor(nexts))


def _inputs(B, T, V, dtype, seed, tree, sharp=2.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    logits = sharp * torch.randn(B, T, V, device=DEV, generator=g)
    target = torch.softmax(logits, -1).to(dtype)
    near = torch.softmax(logits[:, :T - 1] + 0.7 * torch.randn(B, T - 1, V, device=DEV, generator=g), -1)
    u = torch.rand(B, T, device=DEV, generator=g)
    tokens = torch.randint(0, V, (B, T), device=DEV, generator=g)
    if not tree:
        if T > 1:
            tokens[:, 1:] = torch.multinomial(near.reshape(-1, V), 1, generator=g).reshape(B, T - 1)
        return tokens, target, u, None, near.to(dtype)
    par = torch.empty(B, T, dtype=torch.int32)
    hg = torch.Generator().manual_seed(seed)
    for b in range(B):
        for i in range(T):
            par[b, i] = int(torch.randint(max(0, i - 6), i, (1,), generator=hg)) if i else -1
    best = target.float().topk(min(8, V), -1).indices
    for b in range(B):
        for i in range(1, T):
            rank = int((par[b, :i] == par[b, i]).sum())
            tokens[b, i] = best[b, par[b, i], min(rank, best.shape[-1] - 1)]
    return tokens, target, u, par.to(DEV), None


def _equal(got, want):
    for a, w, name in zip(got, want, ("path", "count", "next")):
        assert a.dtype == w.dtype and torch.equal(a.cpu(), w), (name, a.cpu(), w)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("B,T,V", [(1, 1, 1), (3, 1, 1000), (5, 2, 7), (4, 5, 2047), (2, 9, 50257), (3, 64, 4099),
                                   (130, 4, 515), (1, 3, 151936)])
@pytest.mark.parametrize("kind", ["tree", "chain", "chosen"])
def test_random_cases(dtype, B, T, V, kind):
    print("case:", dtype, B, T, V, kind, flush=True)
    tokens, target, u, par, draft = _inputs(B, T, V, dtype, T + V, kind == "tree")
    if kind == "chosen":
        draft = None
    _equal(verify_drafts(tokens, target, u, parents=par, draft_probs=draft), _walk(tokens, target, u, par, draft))


def test_distribution_of_the_emitted_token():
    """Whatever was drafted, the first emitted token is distributed as the target's: 200 000 sequences
    over 6 tokens; each frequency within 5 standard deviations."""
    n, V = 200000, 6
    g = torch.Generator(device=DEV).manual_seed(1)
    p = torch.tensor([0.05, 0.3, 0.2, 0.0, 0.35, 0.1], device=DEV)
    q = torch.tensor([0.3, 0.1, 0.1, 0.2, 0.25, 0.05], device=DEV)
    batch = 50000
    for kind in ("chain", "tree"):
        seen = torch.zeros(V, dtype=torch.float64)
        for _ in range(n // batch):
            if kind == "chain":
                x = torch.multinomial(q.expand(batch, V), 1, generator=g)
                par, draft, T = None, q.expand(batch, 1, V).contiguous(), 2
                tokens = torch.cat([torch.zeros_like(x), x], 1)
            else:
                T = 4
                tokens = torch.tensor([0, 4, 3, 1], device=DEV).expand(batch, T).contiguous()
                par, draft = torch.tensor([-1, 0, 0, 0], dtype=torch.int32, device=DEV), None
            u = torch.rand(batch, T, device=DEV, generator=g)
            path, count, nxt = verify_drafts(tokens, p.expand(batch, T, V).contiguous(), u, parents=par, draft_probs=draft)
            first = torch.where(count > 1, tokens.gather(1, path[:, 1:2].clamp(min=0).long())[:, 0], nxt)
            seen += torch.bincount(first, minlength=V).double().cpu()
        f, pt = seen / n, p.double().cpu()
        assert ((f - pt).abs() <= 5 * (pt * (1 - pt) / n).sqrt()).all(), (kind, f)


def test_borders_and_odd_inputs():
    V = 3000
    one = torch.zeros(1, 3, V, device=DEV)
    one[:, :, 1234] = 1.0
    tok = torch.tensor([[0, 1234, 1234]], device=DEV)
    u0 = torch.zeros(1, 3, device=DEV)
    # certain tokens are accepted at u = 0 and just below 1
    for u in (u0, u0 + (1 - 2.0 ** -24)):
        path, count, nxt = verify_drafts(tok, one, u)
        assert path.tolist() == [[0, 1, 2]] and count.tolist() == [3] and nxt.tolist() == [1234]
    # a token of probability 0 is rejected at u = 0 too; what is left is drawn
    path, count, nxt = verify_drafts(torch.tensor([[0, 7, 1234]], device=DEV), one, u0)
    assert path.tolist() == [[0, -1, -1]] and nxt.tolist() == [1234]
    # tokens outside the vocabulary, repeated candidates, parents that are no earlier node
    tok = torch.tensor([[0, -5, V, 1234, 1234, 9]], device=DEV)
    six = one[:, :1].expand(1, 6, V).contiguous()
    par = torch.tensor([[-1, 0, 0, 7, -9, 5]], dtype=torch.int32, device=DEV)
    path, count, nxt = verify_drafts(tok, six, torch.zeros(1, 6, device=DEV), parents=par)
    assert path.tolist() == [[0, -1, -1, -1, -1, -1]] and nxt.tolist() == [1234]
    # p equal to q, rejected by an odd uniform: nothing is left of (p - q)+, so p itself is drawn
    p = torch.full((1, 2, 4), 0.25, device=DEV)
    path, count, nxt = verify_drafts(torch.tensor([[0, 2]], device=DEV), p, torch.tensor([[0.6, 1.5]], device=DEV),
                                     draft_probs=p[:, :1].contiguous())
    assert count.tolist() == [1] and nxt.tolist() == [2]
    # rows without a positive probability
    for bad in (0.0, float("nan"), -1.0):
        _, count, nxt = verify_drafts(torch.zeros(2, 1, dtype=torch.long, device=DEV),
                                      torch.full((2, 1, 5000), bad, device=DEV), torch.rand(2, 1, device=DEV))
        assert count.tolist() == [1, 1] and nxt.tolist() == [-1, -1]
    # uniforms at and beyond their ends still give a token of positive probability
    p = torch.zeros(4, 1, 9000, device=DEV)
    p[:, :, 100] = 0.5
    p[:, :, 8000] = 0.5
    _, _, nxt = verify_drafts(torch.zeros(4, 1, dtype=torch.long, device=DEV), p,
                              torch.tensor([[0.0], [1.0], [-1.0], [0.5]], device=DEV))
    assert nxt.tolist() == [100, 8000, 100, 8000]
    # no sequences
    path, count, nxt = verify_drafts(torch.zeros(0, 3, dtype=torch.long, device=DEV), torch.zeros(0, 3, 10, device=DEV),
                                     torch.zeros(0, 3, device=DEV))
    assert path.shape == (0, 3) and count.shape == (0,) and nxt.shape == (0,)


def test_strided_probabilities():
    """Rows of a larger logits buffer: any stride between nodes and sequences, odd row starts."""
    tokens, target, u, _, draft = _inputs(3, 4, 1001, torch.float32, 5, False)
    big = torch.zeros(3, 6, 1003, device=DEV)
    big[:, 1:5, 1:1002] = target
    low = torch.zeros(3, 4, 1005, device=DEV)
    low[:, :3, 3:1004] = draft
    got = verify_drafts(tokens, big[:, 1:5, 1:1002], u, draft_probs=low[:, :3, 3:1004])
    _equal(got, _walk(tokens, target, u, None, draft))


def test_graph_replays():
    tokens, target, u, par, _ = _inputs(4, 8, 5003, torch.bfloat16, 3, True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        verify_drafts(tokens, target, u, parents=par)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = verify_drafts(tokens, target, u, parents=par)
    for rep in range(4):
        t, p, v, a, _ = _inputs(4, 8, 5003, torch.bfloat16, 30 + rep, True)
        tokens.copy_(t), target.copy_(p), u.copy_(v), par.copy_(a)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        _equal(got, _walk(tokens, target, u, par, None))


def test_nodes_without_a_place_spoil_no_sibling():
    """A node whose parent is no earlier node is nobody's earlier sibling, whatever its token is."""
    V = 40
    ones = torch.ones(1, 4, V, device=DEV)
    tok, u = torch.tensor([[0, 7, 5, 7]], device=DEV), torch.zeros(1, 4, device=DEV)
    for first in (2, -2, 1, 99, -1):
        par = torch.tensor([[-1, first, 0, 2]], dtype=torch.int32, device=DEV)
        path, count, nxt = verify_drafts(tok, ones, u, parents=par)
        assert path.tolist() == [[0, 2, 3, -1]] and count.tolist() == [3], first
        _equal((path, count, nxt), _walk(tok, ones, u, par))
    # many such nodes in random trees, few distinct tokens
    for seed in range(20):
        tokens, target, uni, par, _ = _inputs(16, 24, 6, torch.float32, 100 + seed, True)
        g = torch.Generator(device=DEV).manual_seed(seed)
        i = torch.arange(24, device=DEV)
        far = torch.randint(0, 24, (16, 24), device=DEV, generator=g).maximum(i).to(torch.int32)
        par = torch.where((torch.rand(16, 24, device=DEV, generator=g) < 0.4) & (i > 0), far, par)
        _equal(verify_drafts(tokens, target, uni, parents=par), _walk(tokens, target, uni, par))
