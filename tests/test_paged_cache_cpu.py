"""TurboQuantPagedCache without a GPU: which pages sequences get, share, copy and give back, what the
cache tells transformers, and what it refuses.  The rows themselves are covered on the GPU."""

import random
import types

import pytest
import torch

from transformers_turboquant import TurboQuantPagedCache, apply_turboquant, speculative_step
from transformers_turboquant.speculative import _depths


class FakePool:
    """Records page copies; pages hold the text they would, so that sharing mistakes show."""

    device = torch.device("cpu")
    num_kv_heads, head_dim, bits = 2, 64, 3

    def __init__(self, pages, size):
        self.rows = [[None] * size for _ in range(pages)]

    def copy(self, src, dst):
        assert not set(src.tolist()) & set(dst.tolist()) and len(set(dst.tolist())) == len(dst)
        for s, d in zip(src.tolist(), dst.tolist()):
            self.rows[d] = list(self.rows[s])

    def nbytes(self):
        return 1000 * len(self.rows)


def make(pages=12, layers=2, size=32):
    cache = TurboQuantPagedCache(pages, layers, size)
    cache.pool = FakePool(pages, size)
    return cache


def step(cache, tokens):
    """Append tokens (a list per active sequence, equally long), as the layers of a forward would."""
    k = torch.zeros(len(tokens), 2, len(tokens[0]), 64)
    for layer in range(cache.num_layers):
        cache._begin(layer, k, 3)
        table, lengths = cache._device_state
        if layer == 0:
            for b, row in enumerate(tokens):
                for i, t in enumerate(row):
                    j = int(lengths[b]) + i
                    cache.pool.rows[int(table[b, j // cache.page_size])][j % cache.page_size] = t
        cache._finish(layer)


def text(cache, i):
    s = cache._seqs[i]
    return [cache.pool.rows[s.pages[j // cache.page_size]][j % cache.page_size] for j in range(s.length)]


def check(cache):
    used = [p for s in cache._seqs.values() for p in s.pages]
    for p in range(cache.num_pages):
        assert cache._refs[p] == used.count(p)
        assert (p in cache._free) == (p not in used)
    assert len(set(cache._free)) == len(cache._free)


def test_sequences_grow_and_are_freed():
    cache = make()
    step(cache, [[1, 2, 3], [4, 5, 6]])  # the first forward makes its sequences
    a, b = cache.active
    assert cache.lengths() == [3, 3] and cache.get_seq_length() == 3 and cache.free_pages == 10
    assert cache.nbytes() == 2000
    (c,) = cache.add()
    cache.use([c])
    step(cache, [list(range(100, 170))])
    assert cache.lengths([a, b, c]) == [3, 3, 70] and cache.free_pages == 7
    cache.use([c, a])
    step(cache, [[7], [8]])
    assert text(cache, a) == [1, 2, 3, 8] and text(cache, c) == [*range(100, 170), 7] and text(cache, b) == [4, 5, 6]
    check(cache)
    cache.free(c, c)
    assert cache.active == [a] and cache.free_pages == 10
    cache.reset()
    assert cache.free_pages == 12 and cache.active == []
    step(cache, [[1]])
    assert cache.lengths() == [1]


def test_fork_copies_a_shared_page_before_it_is_written():
    cache = make()
    step(cache, [list(range(40))])
    (a,) = cache.active
    b, c = cache.fork(a, 2)
    assert cache.free_pages == 10  # all shared
    check(cache)
    cache.use([a, b, c])
    step(cache, [[-1], [-2], [-3]])
    assert cache.free_pages == 8  # the second page twice more; the last holder keeps the original
    for i, t in ((a, -1), (b, -2), (c, -3)):
        assert text(cache, i) == [*range(40), t]
    check(cache)
    cache.free(a)
    check(cache)
    assert text(cache, b) == [*range(40), -2]


def test_a_full_page_stays_shared():
    cache = make()
    step(cache, [list(range(64))])
    (a,) = cache.active
    (b,) = cache.fork(a)
    cache.use([a, b])
    step(cache, [[-1], [-2]])
    assert cache._seqs[a].pages[:2] == cache._seqs[b].pages[:2] and cache.free_pages == 8
    assert text(cache, a)[-2:] == [63, -1] and text(cache, b)[-2:] == [63, -2]


def test_a_forked_sequence_that_is_not_active_is_not_written():
    cache = make()
    step(cache, [[1, 2]])
    (a,) = cache.active
    (b,) = cache.fork(a)
    step(cache, [[3]])
    assert text(cache, b) == [1, 2] and text(cache, a) == [1, 2, 3]
    cache.use([b])
    step(cache, [[4]])
    assert text(cache, a) == [1, 2, 3] and text(cache, b) == [1, 2, 4]
    check(cache)


def test_beams_and_crop():
    cache = make(pages=40)
    step(cache, [list(range(33)), list(range(50, 83)), list(range(90, 123))])
    cache.reorder_cache(torch.tensor([2, 2, 0]))
    step(cache, [[-1], [-2], [-3]])
    got = [text(cache, i) for i in cache.active]
    assert got == [[*range(90, 123), -1], [*range(90, 123), -2], [*range(33), -3]]
    check(cache)
    cache.crop(-4)
    assert cache.lengths() == [30, 30, 30]
    check(cache)
    step(cache, [[-5], [-6], [-7]])
    assert [text(cache, i) for i in cache.active] == [[*range(90, 120), -5], [*range(90, 120), -6], [*range(30), -7]]
    cache.batch_repeat_interleave(2)
    assert len(cache.active) == 6
    cache.batch_select_indices(torch.tensor([5, 0]))
    assert [text(cache, i) for i in cache.active] == [[*range(30), -7], [*range(90, 120), -5]]
    cache.crop(10)
    assert cache.lengths() == [10, 10]
    cache.crop(-100)
    assert cache.lengths() == [0, 0] and cache.free_pages == 40
    check(cache)


@pytest.mark.parametrize("seed", range(6))
def test_random_histories_keep_every_text(seed):
    rng = random.Random(seed)
    cache, texts, n = make(pages=60, layers=rng.choice([1, 3])), {}, 0
    for _ in range(120):
        op = rng.choice(["add", "fork", "free", "use", "step", "step", "step", "crop", "reorder"])
        live = list(texts)
        if op == "add":
            (i,) = cache.add()
            texts[i] = []
        elif op == "fork" and live:
            i = rng.choice(live)
            (j,) = cache.fork(i)
            texts[j] = list(texts[i])
        elif op == "free" and len(live) > 3:
            i = rng.choice(live)
            cache.free(i)
            del texts[i]
        elif op == "use" and live:
            cache.use(rng.sample(live, rng.randint(1, len(live))))
        elif op == "crop":
            k = rng.randint(1, 40)
            cache.crop(-k)
            for i in cache.active:
                texts[i] = texts[i][:max(0, len(texts[i]) - k)]
        elif op == "reorder" and cache.active:
            rows = [rng.randrange(len(cache.active)) for _ in cache.active]
            old = [texts[i] for i in cache.active]
            cache.reorder_cache(torch.tensor(rows))
            for i, r in zip(cache.active, rows):
                texts[i] = list(old[r])
        elif op == "step" and cache.active:
            T = rng.choice([1, 2, 30, 70])
            rows = [[n := n + 1 for _ in range(T)] for _ in cache.active]
            try:
                step(cache, rows)
            except RuntimeError as e:
                assert "full" in str(e)
                i = rng.choice(cache.active)
                cache.free(i)
                del texts[i]
            else:
                for i, row in zip(cache.active, rows):
                    texts[i] += row
        check(cache)
        assert {i: text(cache, i) for i in cache._seqs} == texts


def test_a_full_cache_changes_nothing():
    cache = make(pages=3)
    step(cache, [[1] * 20, [2] * 20])
    a, b = cache.active
    cache.use([a])
    step(cache, [[1] * 20])
    cache.use([a, b])
    before = [list(s.pages) for s in cache._seqs.values()]
    with pytest.raises(RuntimeError, match="full: 1 more pages of 32 positions wanted, 0 of 3 free"):
        step(cache, [[3] * 13, [4] * 13])
    assert [list(s.pages) for s in cache._seqs.values()] == before and cache.lengths() == [40, 20]
    step(cache, [[3] * 12, [4] * 12])
    check(cache)


def test_steps_that_do_not_fit_or_do_not_finish():
    cache = make(layers=3)
    step(cache, [[1, 2]])
    with pytest.raises(ValueError, match="a batch of 2 for 1 active"):
        cache._begin(0, torch.zeros(2, 2, 1, 64), 3)
    k = torch.zeros(1, 2, 40, 64)
    cache._begin(0, k, 3)
    cache._finish(0)
    with pytest.raises(ValueError, match="layer 1 appends 2 tokens in a step of 40"):
        cache._begin(1, k[:, :, :2], 3)
    with pytest.raises(RuntimeError, match="wrote 1 of the cache's 3 layers"):
        cache._begin(0, k, 3)
    assert cache.lengths() == [2] and cache.free_pages == 11
    step(cache, [[3]])
    assert text(cache, cache.active[0]) == [1, 2, 3]
    for bad, heads, dim, bits in (("heads", 3, 64, 3), ("dim", 2, 128, 3), ("bits", 2, 64, 4)):
        with pytest.raises(ValueError, match="the cache's pages hold 2 heads of 64 at 3 bits"):
            cache._begin(0, torch.zeros(1, heads, 1, dim), bits)


def test_drafts_are_dropped_unless_accepted():
    cache = make()
    step(cache, [[1, 2], [3, 4]])
    with pytest.raises(RuntimeError, match="accept"):
        cache.accept(torch.zeros(2, 3, dtype=torch.int32), torch.ones(2, dtype=torch.int32))
    with cache.draft():
        step(cache, [list(range(40)), list(range(40))])
    assert cache.lengths() == [2, 2] and cache.free_pages == 8
    with pytest.raises(ValueError, match=r"path must be \[2, 40\]"):
        cache.accept(torch.zeros(2, 3, dtype=torch.int32), torch.ones(2, dtype=torch.int32))
    moved = []

    def keep(table, lengths, path, count):
        moved.append((table.shape, lengths.tolist(), path[:, 0].tolist()))
        return lengths + count
    cache.pool.keep = keep
    assert cache.accept(torch.zeros(2, 40, dtype=torch.int32), torch.tensor([1, 35], dtype=torch.int32)) == [3, 37]
    assert moved == [((2, 2), [2, 2], [0, 0])]
    assert cache.lengths() == [3, 37] and cache.free_pages == 9
    with pytest.raises(RuntimeError, match="accept"):
        cache.accept(torch.zeros(2, 40, dtype=torch.int32), torch.ones(2, dtype=torch.int32))
    with cache.draft():  # not accepted: the next step goes over it
        step(cache, [[9] * 40] * 2)
    step(cache, [[5], [6]])
    assert cache.lengths() == [4, 38]
    assert text(cache, cache.active[0])[-1] == 5
    with pytest.raises(ZeroDivisionError):
        with cache.draft():
            step(cache, [[9] * 40] * 2)
            raise ZeroDivisionError
    with pytest.raises(RuntimeError, match="inside"):
        with cache.draft():
            with cache.draft():
                pass
    with cache.draft():  # no forward inside
        pass
    with pytest.raises(RuntimeError, match="accept"):
        cache.accept(torch.zeros(2, 40, dtype=torch.int32), torch.ones(2, dtype=torch.int32))
    with pytest.raises(ValueError, match="parents"):
        with cache.draft(torch.zeros(3)):
            pass
    with pytest.raises(ValueError, match=r"parents \(3,\) for 2 sequences of 4"):
        with cache.draft(torch.zeros(3, dtype=torch.int32)):
            step(cache, [[9] * 4] * 2)
    assert cache.lengths() == [4, 38]
    check(cache)


def test_refusals():
    for args in ((0, 2), (4, 0), (4, 2, 16), (4, 2, 48)):
        with pytest.raises(ValueError):
            TurboQuantPagedCache(*args)
    cache = make()
    (a,) = cache.add()
    for call in (lambda: cache.use([a, a]), lambda: cache.use([99]), lambda: cache.free(99), lambda: cache.fork(99),
                 lambda: cache.lengths([99]), lambda: cache.reorder_cache(torch.tensor([0]))):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(NotImplementedError):
        cache.update(torch.zeros(1), torch.zeros(1), 0)
    with pytest.raises(ValueError, match="GPU"):
        cache.append_attend(0, None, None, torch.zeros(1, 2, 1, 64), torch.zeros(1, 2, 1, 64), torch.zeros(1, 2, 1, 64))
    comp = [types.SimpleNamespace(bits=3, mse_bits=2, seed=s) for s in (1, 2, 3)]
    cache._check_codec(0, comp[0], comp[1])
    cache.use([a])
    step(cache, [[1]])
    with pytest.raises(ValueError, match="other settings"):
        cache._check_codec(0, comp[0], comp[2])
    with pytest.raises(ValueError, match="one bit width"):
        cache._check_codec(0, types.SimpleNamespace(bits=3, mse_bits=3, seed=1), comp[1])


def test_models_build_no_mask_and_the_cpu_is_refused():
    from transformers import LlamaConfig, LlamaForCausalLM
    from transformers.masking_utils import create_causal_mask

    cfg = LlamaConfig(vocab_size=128, hidden_size=128, intermediate_size=256, num_hidden_layers=2, num_attention_heads=2,
                      num_key_value_heads=2)
    cfg._attn_implementation = "sdpa"
    cache = make()
    step(cache, [[1] * 37])
    for T in (1, 5, 80):  # decoding, a tree, a chunk; ones are what generate() passes
        for mask in (None, torch.ones(1, 37 + T, dtype=torch.long)):
            pos = torch.full((1, T), 37)  # siblings of a tree share a position
            got = create_causal_mask(config=cfg, inputs_embeds=torch.zeros(1, T, 128), attention_mask=mask,
                                     past_key_values=cache, position_ids=pos)
            assert got is None, (T, mask is None)
    model = apply_turboquant(LlamaForCausalLM(cfg).eval(), bits=3, causal="auto")
    with pytest.raises(ValueError, match="GPU"):
        model(input_ids=torch.zeros(1, 1, dtype=torch.long), past_key_values=TurboQuantPagedCache(4, 2), use_cache=True)


def test_tree_depths_and_their_refusals():
    tree, depth = _depths(None, 2, 4)
    assert tree is None and depth.tolist() == [[0, 1, 2, 3]]
    tree, depth = _depths([-1, 0, 0, 1, 3, -2], 2, 6)
    assert tree.dtype == torch.int32 and depth.tolist() == [[0, 1, 1, 2, 3, 0]]
    tree, depth = _depths(torch.tensor([[-1, 0, 1], [-1, 0, -2]]), 2, 3)
    assert depth.tolist() == [[0, 1, 2], [0, 1, 0]]
    for bad in ([0, 0], [-1, -1], [-1, 1], [-1, 2], [-1, -3], [-2, 0]):
        with pytest.raises(ValueError, match="node"):
            _depths(bad, 1, 2)
    with pytest.raises(ValueError, match="parents must be"):
        _depths([-1, 0, 1], 1, 2)
    cache = make()
    for tokens, kw in ((torch.zeros(2, 65, dtype=torch.long), {}), (torch.zeros(2, dtype=torch.long), {}),
                       (torch.zeros(1, 2, dtype=torch.long), {"temperature": -1.0}),
                       (torch.zeros(1, 2, dtype=torch.long), {}),
                       (torch.zeros(1, 2, dtype=torch.long), {"parents": [-1, 0], "draft_probs": torch.ones(1, 1, 4)})):
        with pytest.raises(ValueError):
            speculative_step(None, cache, tokens, **kw)


def _tiny(kind, **kw):
    import transformers as tr

    cfg = getattr(tr, kind + "Config")(vocab_size=128, hidden_size=128, intermediate_size=128, num_hidden_layers=2,
                                       num_attention_heads=2, num_key_value_heads=2, **kw)
    cfg._attn_implementation = "sdpa"
    return apply_turboquant(getattr(tr, kind + "ForCausalLM")(cfg).eval(), bits=3, causal="auto")


def _ids(B, T):
    return torch.zeros(B, T, dtype=torch.long)


@pytest.mark.parametrize("kind,kw", [("Mistral", dict(sliding_window=24)),
                                     ("Qwen2", dict(use_sliding_window=True, sliding_window=24, max_window_layers=1)),
                                     ("Qwen2", dict(use_sliding_window=True, sliding_window=24, max_window_layers=0))])
def test_sliding_windows_are_refused_once_a_token_is_past_them(kind, kw):
    model = _tiny(kind, **kw)
    for n, T, past in ((0, 24, False), (20, 4, False), (23, 1, False), (0, 25, True), (20, 5, True), (24, 1, True), (300, 1, True)):
        for call in (model, model.model):  # the decoder may be called by itself
            cache = make(pages=40)
            if n:
                step(cache, [[1] * n])
            free = cache.free_pages
            with pytest.raises(ValueError, match="sliding window of 24" if past else "GPU"):
                call(input_ids=_ids(1, T), past_key_values=cache, use_cache=True)
            assert cache.free_pages == free and cache.get_seq_length() == n
            with pytest.raises(ValueError, match="sliding window of 24" if past else "GPU"):
                call(_ids(1, T), None, None, cache)
    # other caches keep their masks
    from transformers_turboquant import TurboQuantCache

    assert model(input_ids=_ids(1, 30), past_key_values=TurboQuantCache(), use_cache=True).logits.shape == (1, 30, 128)


def test_windows_of_attention_modules():
    for kind, kw, want in (("Llama", {}, [None, None]), ("Qwen2", dict(sliding_window=8), [None, None]),
                           ("Mistral", dict(sliding_window=None), [None, None]), ("Mistral", dict(sliding_window=8), [8, 8]),
                           ("Qwen2", dict(use_sliding_window=True, sliding_window=8, max_window_layers=1), [None, 8])):
        model = _tiny(kind, **kw)
        assert [layer.self_attn.sliding_window for layer in model.model.layers] == want
        with pytest.raises(ValueError, match="GPU" if want[1] is None else "window"):
            model(input_ids=_ids(1, 100), past_key_values=make(), use_cache=True)
    # patched a second time: still one check
    assert len(apply_turboquant(model, bits=3).model._forward_pre_hooks) == 1


@pytest.mark.parametrize("kind", ["Llama", "GPT2"])
def test_padding_over_a_cache_is_refused(kind):
    """A zero anywhere in the 2-D mask, over cached positions or new ones."""
    if kind == "GPT2":
        from transformers import GPT2Config, GPT2LMHeadModel

        model = apply_turboquant(GPT2LMHeadModel(GPT2Config(n_layer=2, n_embd=128, n_head=2, vocab_size=128)).eval(), bits=3,
                                 causal="auto")
    else:
        model = _tiny(kind)
    cache = make()
    step(cache, [[1] * 20, [2] * 20])
    for T in (1, 10):
        for where in (None, 0, 7, 19, 20 + T // 2, 19 + T):
            for dtype in (torch.long, torch.bool, torch.float32):
                mask = torch.ones(2, 20 + T, dtype=dtype)
                if where is not None:
                    mask[1, where] = 0
                for call in (model, model.base_model):
                    with pytest.raises(ValueError, match="GPU" if where is None else "padding"):
                        call(input_ids=_ids(2, T), attention_mask=mask, past_key_values=cache, use_cache=True)
    assert cache.lengths() == [20, 20] and cache.free_pages == 10
    with pytest.raises(ValueError, match="padding"):
        model(input_ids=_ids(2, 3), attention_mask=torch.tensor([[1, 1, 1], [0, 1, 1]]), past_key_values=make(), use_cache=True)


def _positions(call, layer, **kw):
    """The position_ids that the decoder's layers get (the CPU is refused behind them)."""
    seen = []
    hook = layer.register_forward_pre_hook(lambda m, a, k: seen.append(k.get("position_ids")), with_kwargs=True)
    with pytest.raises(ValueError, match="GPU"):
        call(**kw, use_cache=True)
    hook.remove()
    return seen[0].tolist()


def test_tokens_stand_behind_their_own_sequence():
    model = _tiny("Llama")
    layer = model.model.layers[0]
    cache = make()
    a, b = cache.add(2)
    for i, n in ((a, 20), (b, 33)):
        cache.use([i])
        step(cache, [[1] * n])
    cache.use([b])
    assert _positions(model, layer, input_ids=_ids(1, 2), past_key_values=cache) == [[33, 34]]
    cache.use([a, b])
    for call in (model, model.model):
        got = _positions(call, layer, input_ids=_ids(2, 3), past_key_values=cache)
        assert got == [[20, 21, 22], [33, 34, 35]]
        given = torch.tensor([[5, 6], [7, 8]])
        assert _positions(call, layer, input_ids=_ids(2, 2), past_key_values=cache, position_ids=given) == given.tolist()
        ones = torch.ones(2, 2, dtype=torch.long)
        assert _positions(call, layer, input_ids=_ids(2, 2), past_key_values=cache, attention_mask=ones) == [[20, 21], [33, 34]]
        with pytest.raises(ValueError, match="position_ids"):
            call(input_ids=_ids(2, 2), past_key_values=cache, position_ids=torch.tensor([[33, 34]]), use_cache=True)
        with pytest.raises(ValueError, match="a mask of 35 positions"):
            call(input_ids=_ids(2, 2), past_key_values=cache, attention_mask=torch.ones(2, 35, dtype=torch.long), use_cache=True)
    seen = []
    hook = layer.register_forward_pre_hook(lambda m, a, k: seen.append(k["position_ids"]), with_kwargs=True)
    with pytest.raises(ValueError, match="GPU"):  # None in its place
        model.model(_ids(2, 1), None, None, cache)
    hook.remove()
    assert seen[0].tolist() == [[20], [33]]
    # generate() counts every row from the longest sequence
    with pytest.raises(ValueError, match="a mask of 34 positions"):
        model.generate(_ids(2, 34), past_key_values=cache, use_cache=True, max_new_tokens=2, pad_token_id=5)
    assert cache.lengths() == [20, 33]


def test_drafted_nodes_stand_at_their_depth():
    model = _tiny("Llama")
    layer = model.model.layers[0]
    cache = make()
    step(cache, [[1] * 20] * 2)
    tree = torch.tensor([-1, 0, 0, 1, 3, -2, 5, -1, 7], dtype=torch.int32)
    want = [0, 1, 1, 2, 3, 0, 1, 0, 1]
    with cache.draft(tree):
        assert _positions(model, layer, input_ids=_ids(2, 9), past_key_values=cache) == [[20 + d for d in want]] * 2
    both = torch.stack([tree, torch.arange(-1, 8, dtype=torch.int32)])
    with cache.draft(both):
        assert _positions(model, layer, input_ids=_ids(2, 9), past_key_values=cache) == [
            [20 + d for d in want], list(range(20, 29))]
    with cache.draft():
        assert _positions(model, layer, input_ids=_ids(2, 3), past_key_values=cache)[0] == [20, 21, 22]
    fresh = TurboQuantPagedCache(8, 2, 32)
    with fresh.draft(tree):
        assert _positions(model, layer, input_ids=_ids(1, 9), past_key_values=fresh) == [want]


def test_a_speculative_step_that_fails_keeps_nothing(monkeypatch):
    import turboquant_pytorch

    cache = make()
    step(cache, [[1] * 9, [2] * 9])
    cache.use(cache.active[:1])
    step(cache, [[1] * 21])
    cache.use([0, 1])
    free, tokens = cache.free_pages, torch.tensor([[5, 6, 7, 8], [9, 10, 11, 12]])

    def model(input_ids, position_ids, past_key_values, use_cache):
        step(past_key_values, input_ids.tolist())
        return types.SimpleNamespace(logits=torch.zeros(2, 4, 16))

    path = torch.tensor([[0, 1, 2, -1], [0, 3, -1, -1]], dtype=torch.int32)
    count = torch.tensor([3, 2], dtype=torch.int32)
    kept = []
    cache.pool.keep = lambda table, lengths, path, count: kept.append(1) or lengths + count
    for bad in ([3, -1], [-1, 4]):
        monkeypatch.setattr(turboquant_pytorch, "verify_drafts", lambda *a, **k: (path, count, torch.tensor(bad)))
        with pytest.raises(RuntimeError, match="no positive probability"):
            speculative_step(model, cache, tokens)
        assert cache.lengths() == [30, 9] and cache.free_pages == free and not kept
        with pytest.raises(RuntimeError, match="accept"):
            cache.accept(path, count)
        check(cache)
    monkeypatch.setattr(turboquant_pytorch, "verify_drafts", lambda *a, **k: (path, count, torch.tensor([3, 4])))
    assert speculative_step(model, cache, tokens) == [[6, 7, 3], [12, 4]]
    assert cache.lengths() == [33, 11] and kept == [1]
    check(cache)


def test_a_refused_first_forward_leaves_an_empty_cache():
    cache = TurboQuantPagedCache(3, 2, 32)

    def empty():
        assert (cache.active, cache.free_pages, cache.pool, cache._seqs) == ([], 3, None, {}) and not cache.is_initialized
        check(cache)

    with pytest.raises(RuntimeError, match="full: 4 more pages"):
        cache._begin(0, torch.zeros(1, 2, 100, 64), 3)
    empty()
    with pytest.raises(RuntimeError, match="full: 4 more pages"):  # another batch, another geometry
        cache._begin(0, torch.zeros(4, 3, 10, 128), 4)
    empty()
    with pytest.raises(ValueError, match="parents"):
        with cache.draft(torch.zeros(3, dtype=torch.int32)):
            cache._begin(0, torch.zeros(2, 2, 4, 64), 3)
    empty()
    # a forward that ends between its layers
    cache._begin(0, torch.zeros(1, 2, 5, 64), 3)
    cache._finish(0)
    with pytest.raises(RuntimeError, match="wrote 1 of the cache's 2 layers"):
        cache._begin(0, torch.zeros(1, 2, 5, 64), 3)
    empty()
    cache._begin(0, torch.zeros(1, 2, 5, 64), 3)
    cache._finish(0)
    with pytest.raises(RuntimeError, match="wrote 1 of the cache's 2 layers"):  # found by another batch
        cache._begin(0, torch.zeros(2, 2, 5, 64), 3)
    empty()
    cache.pool = FakePool(3, 32)
    step(cache, [[1], [2]])
    assert cache.lengths() == [1, 1] and cache.free_pages == 1
    # sequences that were there stay, whatever fails on them
    with pytest.raises(RuntimeError, match="full"):
        step(cache, [[1] * 40, [2] * 40])
    assert cache.lengths() == [1, 1] and cache.free_pages == 1 and cache.pool is not None
    check(cache)
