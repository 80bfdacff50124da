"""TurboQuantPagedCache(shared_prefix=True) without a GPU: which active sequences it takes for a group, and what
speculative_step refuses and passes on."""

import random
import types

import pytest
import torch

import turboquant_pytorch
from test_paged_cache_cpu import check, make, step, text
from transformers_turboquant import TurboQuantPagedCache, speculative_step
from transformers_turboquant.paged_cache import _best_runs


def sharing(**kw):
    cache = make(**kw)
    cache.shared_prefix = True
    return cache


def runs(cache):
    """(sequences, shared positions) of each run of the step under way."""
    if cache._groups is None:
        return [(1, 0)] * len(cache.active)
    out = []
    for row in cache._groups.tolist():
        if out and out[-1][0] == row:
            out[-1][1] += 1
        else:
            out.append([row, 1])
    return [(n, row[1]) for row, n in out]


def test_forks_share_whole_pages():
    cache = sharing(pages=40)
    assert TurboQuantPagedCache(4, 1).shared_prefix is False and TurboQuantPagedCache(4, 1, shared_prefix=True).shared_prefix
    step(cache, [list(range(70))])
    (a,) = cache.active
    b, c = cache.fork(a, 2)
    cache.use([a, b, c])
    step(cache, [[1], [2], [3]])
    assert runs(cache) == [(3, 64)]  # the third page, which is written, is each one's own
    step(cache, [[1], [2], [3]])
    assert runs(cache) == [(3, 64)]
    (d,) = cache.fork(b)
    cache.use([c, b, d, a])
    step(cache, [[5] * 40] * 4)
    assert runs(cache) == [(4, 64)]
    cache.crop(-30)
    (e,) = cache.fork(d)
    cache.use([e, d, c])
    step(cache, [[6]] * 3)
    assert runs(cache) == [(3, 64)]
    plain = cache.add(1)
    cache.use([a, *plain, b])
    step(cache, [[7]] * 3)
    assert cache._groups is None
    check(cache)


def test_nested_forks_are_cut_where_it_saves_most():
    cache = sharing(pages=90)
    step(cache, [list(range(64))])
    (a,) = cache.active
    b = cache.fork(a)[0]
    cache.use([b])
    step(cache, [list(range(320))])
    b2 = cache.fork(b)[0]
    a2 = cache.fork(a)[0]
    cache.use([a, a2, b, b2])
    step(cache, [[1]] * 4)
    assert runs(cache) == [(2, 64), (2, 384)]
    cache.use([b, b2, a])
    step(cache, [[1]] * 3)
    assert runs(cache) == [(2, 384), (1, 0)]
    assert (cache._device_state[0][:2, :12] == cache._device_state[0][:1, :12]).all()


def test_little_in_common_is_read_apart():
    """A group is read as one while it saves a fifth of the pages."""
    cache = sharing(pages=90)
    step(cache, [list(range(64))])  # 2 pages
    (a,) = cache.active
    b = cache.fork(a)[0]
    cache.use([a, b])
    seen = []
    for _ in range(8):
        step(cache, [[1] * 32] * 2)  # a page more of each one's own
        pages = sum(len(s) for s in (row[row >= 0] for row in cache._device_state[0]))
        seen.append((5 * 2 >= pages, cache._groups is not None))
    assert all(want == got for want, got in seen) and seen[0][1] and not seen[-1][1]
    check(cache)


def test_best_runs_against_every_cut():
    rng = random.Random(1)
    for n in list(range(1, 9)) * 12:
        common = [rng.choice([0, 1, 2, 5, 9]) for _ in range(n - 1)]
        got = _best_runs(common)
        best = 0
        for cuts in range(1 << (n - 1)):
            at, total = 0, 0
            for i in range(n):
                if i == n - 1 or cuts >> i & 1:
                    total += (i - at) * min(common[at:i], default=0)
                    at = i + 1
            best = max(best, total)
        at, total = 0, 0
        for size, shared in got:
            assert shared == 0 and size == 1 or shared == min(common[at:at + size - 1]) > 0
            total, at = total + (size - 1) * shared, at + size
        assert at == n and total == best, (common, got)
    assert _best_runs([3] * 500) == [(501, 3)]
    assert sum(size for size, _ in _best_runs([3, 4] * 100)) == 201 and max(size for size, _ in _best_runs([3, 4] * 100)) <= 64


@pytest.mark.parametrize("seed", range(4))
def test_random_histories_group_equal_pages_only(seed):
    rng = random.Random(seed)
    cache, n = sharing(pages=80, layers=2), 0
    seen = set()
    for _ in range(150):
        live = list(cache._seqs)
        op = rng.choice(["add", "fork", "fork", "free", "use", "step", "step", "step", "crop", "reorder"])
        if op == "add":
            cache.add()
        elif op == "fork" and live:
            cache.fork(rng.choice(live), rng.randint(1, 3))
        elif op == "free" and len(live) > 3:
            cache.free(rng.choice(live))
        elif op == "use" and live:
            cache.use(rng.sample(live, rng.randint(1, len(live))))
        elif op == "crop":
            cache.crop(-rng.randint(1, 40))
        elif op == "reorder" and cache.active:
            cache.reorder_cache(torch.tensor([rng.randrange(len(cache.active)) for _ in cache.active]))
        elif op == "step" and cache.active:
            before = {i: text(cache, i) for i in cache._seqs}
            rows = [[n := n + 1 for _ in range(rng.choice([1, 30]))] for _ in [0]] * len(cache.active)
            lengths = cache.lengths()
            try:
                step(cache, rows)
            except RuntimeError:
                cache.free(rng.choice(cache.active))
                continue
            table, at = cache._device_state[0], 0
            for size, shared in runs(cache):
                seen.add(size > 1)
                assert shared % cache.page_size == 0 and (size > 1) == (shared > 0)
                pages = shared // cache.page_size
                assert (table[at:at + size, :pages] == table[at, :pages]).all() and (table[at, :pages] >= 0).all()
                assert all(k >= shared for k in lengths[at:at + size])
                at += size
            assert all(text(cache, i)[:len(before[i])] == before[i] for i in before)
        check(cache)
    assert seen == {True, False}


def test_filters_of_a_speculative_step(monkeypatch):
    cache = make()
    step(cache, [[1] * 9])
    tokens = torch.tensor([[5, 6, 7]])
    for kw in (dict(top_k=-1), dict(top_p=1.5), dict(top_p=-0.1), dict(min_p=2.0), dict(min_p=float("nan"))):
        with pytest.raises(ValueError, match="lie in"):
            speculative_step(None, cache, tokens, **kw)

    def model(input_ids, position_ids, past_key_values, use_cache):
        step(past_key_values, input_ids.tolist())
        return types.SimpleNamespace(logits=torch.arange(30.0).reshape(1, 3, 10))

    asked, verified = [], []

    def filters(*args):
        asked.append(args[1:])
        return torch.full((1, 3, 10), 0.25)

    def verify(tokens, probs, uniforms, **kw):
        verified.append(probs)
        return torch.tensor([[0, 1, -1]], dtype=torch.int32), torch.tensor([2], dtype=torch.int32), torch.tensor([4])

    monkeypatch.setattr(turboquant_pytorch, "filter_probs", filters)
    monkeypatch.setattr(turboquant_pytorch, "verify_drafts", verify)
    cache.pool.keep = lambda table, lengths, path, count: lengths + count
    for kw, want in ((dict(top_k=3), (1.0, 3, 1.0, 0.0)), (dict(temperature=0.5, top_p=0.9), (0.5, 0, 0.9, 0.0)), (dict(min_p=0.1), (1.0, 0, 1.0, 0.1))):
        assert speculative_step(model, cache, tokens, **kw) == [[6, 4]]
        assert asked.pop() == want and (verified.pop() == 0.25).all()
    for kw in (dict(), dict(temperature=0.7), dict(temperature=0, top_k=3)):  # as before
        speculative_step(model, cache, tokens, **kw)
        assert not asked and float(verified.pop().sum()) == pytest.approx(3.0)
