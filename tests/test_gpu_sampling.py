"""Sampling by temperature, top-k, top-p and min-p against float64.

The oracle sorts a row (stable, so equal logits stand by index) and applies the filters one after another in float64.  What
is kept and which token is drawn have to be the same; probabilities are off by the one rounding to float32
(2^-24 of the value) and by 2^-40 for the float64 weights of both sides (series 2 10^-13, sums of 10^5 terms).
Where the border of a draw is itself within 2^-40 of the total, both tokens beside it are right.
"""

import math

import pytest
import torch

from turboquant_pytorch import filter_probs, sample_tokens

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _oracle(row, t, k, p, m):
    """Weights (float64, not normalised) of the kept tokens of one row."""
    l = row.double().cpu()
    l = torch.where(l.isnan(), -math.inf, l)
    V = l.numel()
    if not t > 0:
        t, k = 1.0, 1
    top = l.max()
    out = torch.zeros(V, dtype=torch.float64)
    if top == -math.inf:
        return out
    w = torch.exp((l - top) / t) if top < math.inf else (l == top).double()
    w[l == top] = 1.0
    order = torch.sort(l, descending=True, stable=True).indices
    s = w[order]
    keep = torch.ones(V, dtype=torch.bool)
    if 0 < k < V:
        keep[k:] = False
    s = torch.where(keep, s, 0.0)
    if p < 1:
        c = s.cumsum(0)
        first = keep.clone()
        keep &= c - s < p * c[-1]
        keep[0] = first[0]
    keep &= s >= min(m, 1.0)
    out[order] = torch.where(keep, s, 0.0)
    return out


def _value(x, i):
    return x[i].item() if isinstance(x, torch.Tensor) else x


def _check(logits, u, t=1.0, k=0, p=1.0, m=0.0):
    probs = filter_probs(logits, t, k, p, m)
    tokens = sample_tokens(logits, u, t, k, p, m)
    assert probs.dtype == torch.float32 and probs.shape == logits.shape
    assert tokens.dtype == torch.int64 and tokens.shape == logits.shape[:-1]
    for i in range(logits.shape[0]):
        w = _oracle(logits[i], *(_value(x, i) for x in (t, k, p, m)))
        got = probs[i].double().cpu()
        if not (w > 0).any():
            assert tokens[i] == -1 and (got == 0).all(), i
            continue
        ref = w / w.sum()
        assert ((got - ref).abs() <= ref * (2.0 ** -24 + 2.0 ** -40) + 2.0 ** -149).all(), (i, (got - ref).abs().max())
        tiny = 2.0 ** -140  # what float32 holds
        assert ((got > 0) == (ref > 0))[(ref > tiny) | (ref == 0)].all(), i
        c = w.cumsum(0)
        goal, x = float(u[i]) * c[-1], int(tokens[i])
        want = int(torch.nonzero((c > goal) & (w > 0))[0])
        # a border that u hits to within the rounding of both sides' sums (half of the tokens, u = 1/2) is nobody's
        near = 2.0 ** -40 * float(c[-1]) if u[i] > 0 else 0.0
        assert x == want or (w[x] > 0 and c[x] > goal - near and c[x] - w[x] <= goal + near), (i, x, want)
    return probs, tokens


def _logits(N, V, dtype, seed, scale=2.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    l = scale * torch.randn(N, V, device=DEV, generator=g)
    l.scatter_add_(1, torch.randint(0, V, (N, min(V, 20)), device=DEV, generator=g), 8 * torch.rand(N, min(V, 20), device=DEV, generator=g))
    return l.to(dtype), torch.rand(N, device=DEV, generator=g)


SETTINGS = [dict(), dict(t=0.0), dict(t=0.7), dict(k=1), dict(k=50), dict(t=0.3, p=0.9), dict(p=0.5), dict(t=1.5, p=0.99), dict(m=0.1),
            dict(t=2.0, m=0.001), dict(t=0.8, k=40, p=0.95), dict(k=200, p=0.9, m=0.02), dict(p=0.97, m=0.05), dict(p=0.3, m=0.01),
            dict(p=0.0), dict(k=30, p=0.0, m=1.0), dict(m=1.0), dict(k=3000, p=0.999), dict(t=0.02, k=7), dict(t=50.0, p=0.2)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("N,V", [(1, 1), (5, 7), (3, 1000), (2, 8191), (4, 8200), (2, 50257), (3, 40001)])
def test_settings(dtype, N, V):
    for i, kw in enumerate(SETTINGS):
        print("case:", dtype, N, V, kw, flush=True)
        _check(*_logits(N, V, dtype, 100 * i + V), **kw)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_settings_of_the_rows(dtype):
    """Every row its own; the mixed batch gives what each row gives alone."""
    N, V = 3 * len(SETTINGS), 5003
    logits, u = _logits(N, V, dtype, 5)
    rows = [dict(dict(t=1.0, k=0, p=1.0, m=0.0), **SETTINGS[i % len(SETTINGS)]) for i in range(N)]
    t, p, m = (torch.tensor([r[n] for r in rows], device=DEV) for n in "tpm")
    k = torch.tensor([r["k"] for r in rows], dtype=torch.int32, device=DEV)
    _check(logits, u, t, k, p, m)
    _check(logits, u, 0.9, k, 0.8, m)
    out = torch.tensor([float("nan"), -1.0, 1.0, 1.0], device=DEV)  # values that no row should have
    q = torch.tensor([1.0, 1.0, float("nan"), 2.0], device=DEV)
    got = filter_probs(logits[:4], out, torch.tensor([-5, 0, 0, V + 9], dtype=torch.int32, device=DEV), q, q.flip(0) - 3)
    want = [filter_probs(logits[:1], 0.0), filter_probs(logits[1:2], 0.0), filter_probs(logits[2:3]), filter_probs(logits[3:4])]
    assert torch.equal(got, torch.cat(want))


def test_many_rows_and_large_vocabularies():
    for N, V, dtype in ((700, 20011, torch.bfloat16), (300, 100003, torch.bfloat16), (70, 60000, torch.float32), (3000, 300, torch.float16),
                        (1, 3_000_001, torch.float32)):
        logits, u = _logits(N, V, dtype, V)
        for kw in (dict(t=0.8, p=0.9), dict(k=50), dict(m=0.05), dict()):
            print("case:", N, V, dtype, kw, flush=True)
            probs, tokens = filter_probs(logits, *(kw.get(n, d) for n, d in zip("tkpm", (1.0, 0, 1.0, 0.0)))), sample_tokens(
                logits, u, *(kw.get(n, d) for n, d in zip("tkpm", (1.0, 0, 1.0, 0.0))))
            some = sorted({0, 1 % N, N // 2, N - 1})
            p2, t2 = _check(logits[some], u[some], **kw)
            # another batch is cut into other chunks: each side is within 2^-24 + 2^-40 of the exact value
            assert ((probs[some] - p2).abs() <= p2 * (2.0 ** -23 + 2.0 ** -38)).all() and torch.equal(tokens[some], t2)


def test_equal_logits():
    """The border lies among equal logits: by index, whatever their number."""
    for V in (10, 1000, 8192, 70000):
        logits = torch.full((3, V), 1.25, device=DEV)
        logits[1, ::2] = 3.0
        logits[2, V // 3:] = -math.inf
        u = torch.tensor([0.0, 0.5, 0.999], device=DEV)
        for kw in (dict(k=3), dict(k=V // 2), dict(p=0.5), dict(p=0.25, t=0.5), dict(k=V // 2 + 1, p=0.5), dict(m=0.5), dict(t=0.0),
                   dict(p=0.75, m=0.3), dict()):
            print("case:", V, kw, flush=True)
            _check(logits, u, **kw)


def test_long_borders():
    """Borders among thousands of tokens that lie together."""
    g = torch.Generator(device=DEV).manual_seed(1)
    V = 60000
    flat = 0.05 * torch.randn(3, V, device=DEV, generator=g)
    far = torch.cat([torch.full((3, 1), 60.0, device=DEV), flat[:, 1:] * 20], 1)  # the rest lies below every bin
    u = torch.rand(3, device=DEV, generator=g)
    for kw in (dict(p=0.6), dict(k=20000), dict(k=30000, p=0.5), dict(t=0.1, p=0.3, m=0.1), dict(k=5000, t=5.0, p=0.9), dict(t=30.0, p=0.9),
               dict(t=100.0, k=1000, p=0.7), dict(t=8.0, p=0.98, m=1e-4)):
        print("case:", kw, flush=True)
        _check(flat, u, **kw)
        _check(far, u, **kw)


def test_values_at_the_ends():
    V = 3001
    base, _ = _logits(8, V, torch.float32, 3)
    l = base.clone()
    l[0] = -math.inf
    l[1] = float("nan")
    l[2, ::3] = float("nan")
    l[3, [5, 77, 2000]] = math.inf
    l[4] = -math.inf
    l[4, 1234] = -1e30
    l[5] *= 1e30
    l[6] = 1e-40 * base[6]
    l[7, :] = -3.4e38
    l[7, ::7] = 3.4e38
    u = torch.tensor([0.3, 0.3, 0.9, 0.5, 0.1, 0.7, 0.2, 0.6], device=DEV)
    for kw in (dict(), dict(k=2), dict(k=400), dict(p=0.4), dict(m=0.2), dict(t=0.0), dict(t=1e-30, p=0.5), dict(t=1e30, p=0.5, m=0.5),
               dict(k=600, p=0.9, m=1e-3)):
        print("case:", kw, flush=True)
        _check(l, u, **kw)
    for dtype in (torch.bfloat16, torch.float16):
        _check(l.to(dtype), u, k=10, p=0.8)


def test_uniforms_at_the_ends():
    logits, _ = _logits(4, 9001, torch.float32, 8, scale=10.0)
    logits[:, :50] = -math.inf
    for u in (0.0, 2.0 ** -24, 1 - 2.0 ** -24):
        uu = torch.full((4,), u, device=DEV)
        for kw in (dict(), dict(t=0.1), dict(p=0.9), dict(k=5), dict(m=0.01), dict(t=0.05, p=0.9999), dict(t=3.0, k=2000, p=0.99)):
            print("case:", u, kw, flush=True)
            _check(logits, uu, **kw)


def test_shapes_and_strides():
    g = torch.Generator(device=DEV).manual_seed(2)
    x = torch.randn(3, 4, 1003, device=DEV, generator=g)
    u = torch.rand(3, 4, device=DEV, generator=g)
    probs, tok = filter_probs(x, top_k=9), sample_tokens(x, u, top_k=9)
    assert probs.shape == x.shape and tok.shape == (3, 4)
    _check(x.reshape(12, -1), u.reshape(-1), k=9)
    assert torch.equal(sample_tokens(x[:, -1], u[:, -1], top_k=9), tok[:, -1])  # rows apart from one another
    assert torch.equal(filter_probs(x[:, 1, 1:901], top_p=0.5), filter_probs(x[:, 1, 1:901].contiguous(), top_p=0.5))
    wide = x[0, 0].expand(5, -1)  # one row for all
    assert torch.equal(sample_tokens(wide, u.reshape(-1)[:5], top_p=0.9), sample_tokens(wide.contiguous(), u.reshape(-1)[:5], top_p=0.9))
    k = torch.full((3, 4), 9, dtype=torch.int32, device=DEV)
    assert torch.equal(sample_tokens(x, u, top_k=k), tok)
    one = sample_tokens(x[0, 0], u[0, 0], top_k=9)
    assert one.shape == () and one == tok[0, 0]
    assert sample_tokens(x[:0], u[:0]).shape == (0, 4) and filter_probs(x[:, :0]).shape == (3, 0, 1003)


def test_the_same_every_time_and_on_other_streams():
    logits, u = _logits(40, 50257, torch.bfloat16, 9)
    for kw in (dict(temperature=0.8, top_p=0.95), dict(top_k=100, top_p=0.9), dict(min_p=0.01)):
        want, probs = sample_tokens(logits, u, **kw), filter_probs(logits, **kw)
        torch.cuda.synchronize()
        streams, got = [torch.cuda.Stream() for _ in range(2)], []
        for i in range(6):
            with torch.cuda.stream(streams[i % 2]):
                got.append((sample_tokens(logits, u, **kw), filter_probs(logits, **kw)))
        torch.cuda.synchronize()
        for a, b in got:
            assert torch.equal(a, want) and torch.equal(b, probs)


def test_graph_replays():
    """Captured once with settings of the rows; logits, uniforms and settings change between the replays."""
    N, V = 6, 12001
    logits, u = _logits(N, V, torch.float32, 11)
    t, p, m = (torch.full((N,), x, device=DEV) for x in (0.8, 0.9, 0.0))
    k = torch.zeros(N, dtype=torch.int32, device=DEV)

    def call():
        return sample_tokens(logits, u, t, k, p, m), filter_probs(logits, t, k, p, m)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for rep in range(5):
        new, nu = _logits(N, V, torch.float32, 20 + rep)
        logits.copy_(new)
        u.copy_(nu)
        k.fill_((0, 40, 1, 0, 300)[rep])
        p.fill_((0.9, 0.9, 1.0, 1.0, 0.5)[rep])
        m.fill_((0.0, 0.01, 0.0, 0.1, 0.0)[rep])
        torch.cuda.synchronize()
        want = [x.clone() for x in call()]
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1]), rep
        _check(logits, u, t, k, p, m)


def test_probabilities_of_more_rows_than_a_step_of_their_writing():
    """Rows that keep many among rows that keep few, over more than 2048 of them."""
    N, V = 4500, 2100
    logits, u = _logits(N, V, torch.bfloat16, 31)
    g = torch.Generator(device=DEV).manual_seed(32)
    k = torch.where(torch.rand(N, device=DEV, generator=g) < 0.7, 5, 0).to(torch.int32)  # without a k: all tokens
    probs = filter_probs(logits, top_k=k)
    some = torch.tensor([0, 1, 255, 256, 2046, 2047, 2048, 2049, 4095, 4096, 4097, N - 2, N - 1], device=DEV)
    some = torch.cat([some, torch.randint(0, N, (40,), device=DEV, generator=g)])
    p2, _ = _check(logits[some], u[some], 1.0, k[some])
    assert (k[some] > 0).any() and (k[some] == 0).any()
    assert ((probs[some] - p2).abs() <= p2 * (2.0 ** -23 + 2.0 ** -38)).all()  # one rounding each
    assert (((probs > 0).sum(1) == 5) == (k == 5)).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_min_p_above_and_below_the_border_of_top_p(dtype):
    """The one that keeps less decides; with equal logits at either border."""
    V = 30000
    g = torch.Generator(device=DEV).manual_seed(41)
    l = 1.5 * torch.randn(4, V, device=DEV, generator=g)
    l[1] = (l[1] * 8).round() / 8
    l[2, :3000] = 6.0
    l[3] = (l[3] * 2).round() / 2 + 50
    l, u = l.to(dtype), torch.rand(4, device=DEV, generator=g)
    top = l.double().max(1, keepdim=True).values
    for t in (0.5, 1.0, 2.5):
        w = torch.exp((l.double() - top) / t)
        for p in (0.05, 0.5, 0.9, 0.999):
            for q in (0.2, 0.5, 0.8):  # a weight that some token has, so that min-p's border is one's own
                m = w.flatten()[torch.argsort(w.flatten())[int(q * 4 * V)]].item()
                for mm in (m * (1 - 1e-9), m * (1 + 1e-9)):
                    print("case:", dtype, t, p, mm, flush=True)
                    _check(l, u, t=t, p=p, m=mm)


def test_top_p_keeps_no_more_of_equal_logits_than_top_k():
    """top_k ends among many equal logits and top_p behind them, or just in front of the last."""
    g = torch.Generator(device=DEV).manual_seed(51)
    for V, step in ((2747, 0.25), (9000, 0.5), (40001, 0.125)):
        l = ((0.5 * torch.randn(3, V, device=DEV, generator=g)) / step).round() * step
        u = torch.rand(3, device=DEV, generator=g)
        for k in (100, 300, 1200, V - 5):
            for p in (0.5, 0.99, 1 - 1e-4, 1 - 1e-9):
                print("case:", V, step, k, p, flush=True)
                _check(l, u, t=20.0, k=k, p=p)
                _check(l.half(), u, t=3.0, k=k, p=p, m=1e-4)


def test_logits_that_are_strided_along_the_vocabulary():
    g = torch.Generator(device=DEV).manual_seed(71)
    u = torch.rand(6, device=DEV, generator=g)
    x = torch.randn(2006, 6, device=DEV, generator=g).to(torch.bfloat16)
    for l in (x.t(), x.reshape(6, -1)[:, ::2], x.t().reshape(6, 1, -1)[..., ::3], x.reshape(1003, 2, 6).permute(2, 1, 0)):
        v = u[:, None].expand(l.shape[:-1]) if l.dim() == 3 else u
        assert l.stride(-1) != 1
        for kw in (dict(top_k=9), dict(top_p=0.7)):
            assert torch.equal(sample_tokens(l, v, **kw), sample_tokens(l.contiguous(), v, **kw))
            assert torch.equal(filter_probs(l, **kw), filter_probs(l.contiguous(), **kw))
