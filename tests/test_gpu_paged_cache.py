"""TurboQuantPagedCache and speculative_step on the GPU: page writes, tree attention, page copies, kept paths
and verification run together under a model, against recomputation without a cache."""

import pytest
import torch

from oracle import tq_oracle as O
from transformers_turboquant import TurboQuantCache, TurboQuantPagedCache, apply_turboquant, speculative_step

pytestmark = pytest.mark.gpu

V = 1000


def llama(dtype=torch.float32, heads=8, kv=2, hidden=1024, bits=3):
    from transformers import LlamaConfig, LlamaForCausalLM

    torch.manual_seed(0)
    cfg = LlamaConfig(vocab_size=V, hidden_size=hidden, intermediate_size=hidden, num_hidden_layers=2,
                      num_attention_heads=heads, num_key_value_heads=kv)
    return apply_turboquant(LlamaForCausalLM(cfg).eval(), bits=bits, causal="auto").to("cuda", dtype)


def ids(B, T, seed=5):
    return torch.randint(0, V, (B, T), generator=torch.Generator().manual_seed(seed)).cuda()


def run(model, cache, tokens):
    """Logits of every token, appended to the cache's active sequences."""
    pos = torch.tensor(cache.lengths() or [0] * len(tokens), device="cuda")[:, None]
    pos = pos + torch.arange(tokens.shape[1], device="cuda")
    with torch.no_grad():
        return model(input_ids=tokens, position_ids=pos, past_key_values=cache, use_cache=True).logits.float()


def recompute(model, tokens):
    with torch.no_grad():
        return model(input_ids=tokens, use_cache=False).logits.float()


def close(a, b, dtype=torch.float32):
    """The bound that cached decoding is held to: the same estimator through other kernels, which round the
    weights of a softmax to f16 at other places."""
    cos = [O.cosine(x.cpu().numpy(), y.cpu().numpy()) for x, y in zip(a.reshape(-1, V), b.reshape(-1, V))]
    assert min(cos) > (0.9999 if dtype == torch.float32 else 0.999), min(cos)


@pytest.mark.parametrize("dtype,heads,kv,hidden,bits", [
    (torch.float32, 8, 2, 1024, 3),
    (torch.bfloat16, 8, 2, 1024, 2),
    (torch.float16, 4, 4, 256, 4),  # head_dim 64
    (torch.float32, 4, 2, 128, 3),  # head_dim 32: attention over gathered rows
])
def test_generate_matches_recompute(dtype, heads, kv, hidden, bits):
    print("case: paged generate", dtype, heads, kv, hidden, bits, flush=True)
    model, prompt = llama(dtype, heads, kv, hidden, bits), ids(2, 37)
    kw = dict(max_new_tokens=8, min_new_tokens=8, do_sample=False, output_logits=True, return_dict_in_generate=True,
              attention_mask=torch.ones_like(prompt))
    cache = TurboQuantPagedCache(16, 2, 32)
    with torch.no_grad():
        ref = model.generate(prompt, use_cache=False, **kw)
        got = model.generate(prompt, use_cache=True, past_key_values=cache, **kw)
    assert cache.lengths() == [44, 44] and cache.free_pages == 12
    close(torch.stack(got.logits), torch.stack(ref.logits), dtype)
    assert (got.sequences == ref.sequences).float().mean() > 0.95


def test_gpt2_generates_from_pages():
    print("case: paged gpt2", flush=True)
    from transformers import GPT2Config, GPT2LMHeadModel

    torch.manual_seed(0)
    model = apply_turboquant(GPT2LMHeadModel(GPT2Config(n_layer=2, n_embd=128, n_head=2, vocab_size=V)), bits=3,
                             causal="auto").cuda().eval()  # the new modules too: no dropout
    prompt = ids(2, 11)
    kw = dict(max_new_tokens=6, min_new_tokens=6, do_sample=False, output_logits=True, return_dict_in_generate=True,
              attention_mask=torch.ones_like(prompt))
    with torch.no_grad():
        ref = model.generate(prompt, use_cache=False, **kw)
        got = model.generate(prompt, use_cache=True, past_key_values=TurboQuantPagedCache(8, 2), **kw)
    close(torch.stack(got.logits), torch.stack(ref.logits))


def test_beam_search_matches_the_contiguous_cache():
    print("case: paged beams", flush=True)
    model, prompt = llama(), ids(2, 40)
    kw = dict(max_new_tokens=12, min_new_tokens=12, do_sample=False, num_beams=3, output_scores=True,
              return_dict_in_generate=True, attention_mask=torch.ones_like(prompt))
    cache = TurboQuantPagedCache(64, 2, 32)
    with torch.no_grad():
        ref = model.generate(prompt, use_cache=True, past_key_values=TurboQuantCache(), **kw)
        got = model.generate(prompt, use_cache=True, past_key_values=cache, **kw)
    assert len(cache.active) == 6
    # the same text, or one that scores as well
    same = (got.sequences == ref.sequences).all(-1)
    gap = (got.sequences_scores - ref.sequences_scores).abs() / ref.sequences_scores.abs()
    assert bool((same | (gap < 1e-3)).all()), (same, gap)


def test_chunks_and_unequal_lengths_match_recompute():
    print("case: paged chunks", flush=True)
    model, cache = llama(), TurboQuantPagedCache(40, 2, 32)
    text = ids(3, 330)
    a, b, c = cache.add(3)
    cache.use([a, b])
    got = [run(model, cache, text[:2, :100])]  # a fresh prompt
    got.append(run(model, cache, text[:2, 100:107]))  # few tokens
    got.append(run(model, cache, text[:2, 107:207]))  # a long chunk over a prefix
    close(torch.cat(got, 1), recompute(model, text[:2, :207]))
    cache.use([c])
    last = run(model, cache, text[2:, :33])
    close(last, recompute(model, text[2:, :33]))
    cache.use([c, a])  # lengths 33 and 207
    for n in (1, 5, 70):
        n0, n1 = cache.lengths()
        got = run(model, cache, torch.stack([text[2, n0:n0 + n], text[0, n1:n1 + n]]))
        close(got[0], recompute(model, text[2:, :n0 + n])[0, n0:])
        close(got[1], recompute(model, text[:1, :n1 + n])[0, n1:])
    assert cache.lengths([a, b, c]) == [283, 207, 109]


def test_forks_equal_sequences_run_apart():
    print("case: paged forks", flush=True)
    model = llama(torch.bfloat16)
    prompt, more = ids(1, 45), ids(3, 30, seed=6)
    fork, apart = TurboQuantPagedCache(16, 2, 32), TurboQuantPagedCache(16, 2, 32)
    (a,) = fork.add()
    fork.use([a])
    run(model, fork, prompt)
    fork.use([a, *fork.fork(a, 2)])
    seqs = apart.add(3)
    for i in seqs:
        apart.use([i])
        run(model, apart, prompt)
    apart.use(seqs)
    assert fork.free_pages == 14 and apart.free_pages == 10
    for lo, hi in ((0, 1), (1, 4), (4, 30)):
        assert torch.equal(run(model, fork, more[:, lo:hi]), run(model, apart, more[:, lo:hi]))
    assert fork.free_pages == 16 - (1 + 3 * 2) and apart.free_pages == 16 - 9


def greedy(model, cache, root, steps):
    out = []
    for _ in range(steps):
        root = run(model, cache, root)[:, -1:].argmax(-1)
        out.append(root)
    return torch.cat(out, 1)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_speculative_steps_follow_greedy_decoding(dtype):
    """Chains and trees that hold the right tokens at various depths, over sequences of unequal
    length: what is emitted are likeliest tokens of a recomputation, and right drafts are kept."""
    print("case: speculative steps", dtype, flush=True)
    model, cache = llama(dtype), TurboQuantPagedCache(64, 2, 32)
    prompts = [ids(1, 29, 1), ids(1, 75, 2)]
    seqs = cache.add(2)
    for i, p in zip(seqs, prompts):
        cache.use([i])
        run(model, cache, p[:, :-1])
    cache.use(seqs)
    truth_cache = cache.fork(seqs[0]) + cache.fork(seqs[1])
    cache.use(truth_cache)
    root = torch.cat([p[:, -1:] for p in prompts])
    truth = greedy(model, cache, root, 60)
    cache.use(seqs)
    free = cache.free_pages
    done, texts, accepted = [0, 0], [list(p[0].tolist()) for p in prompts], 0
    g = torch.Generator().manual_seed(3)
    for step in range(8):
        T, right = [(4, 3), (1, 0), (6, 2), (5, 0), (8, 7), (3, 1), (7, 3), (2, 1)][step]
        # the right continuation first `right` deep; other nodes are wrong
        parents, rows = [-1], [[t[-1]] for t in texts]
        spine = 0
        for i in range(1, T):
            on = i % 2 == 1 if step % 2 else i <= right  # odd steps: wrong siblings between the right nodes
            depth = sum(1 for _ in _up(parents, spine))
            for b in range(2):
                want = truth[b, min(done[b] + depth - 1, 59)].item()
                wrong = (want + 1 + int(torch.randint(0, 900, (1,), generator=g))) % V
                rows[b].append(want if on and depth <= right else wrong)
            parents.append(spine)
            if on and depth <= right:
                spine = i
        out = speculative_step(model, cache, torch.tensor(rows, device="cuda"), parents if step % 2 else None, temperature=0)
        for b in range(2):
            accepted += len(out[b]) - 1
            done[b] += len(out[b])
            texts[b] += out[b]
        assert cache.lengths() == [len(t) - 1 for t in texts]
    total = same = 0
    for b, p in enumerate(prompts):
        n = p.shape[1]
        logits = recompute(model, torch.tensor([texts[b]], device="cuda"))[0, n - 1:-1]
        new = torch.tensor(texts[b][n:], device="cuda")
        best = logits.max(-1).values - logits.gather(1, new[:, None])[:, 0]
        # logits apart by less than the cosine bound allows: an error of relative norm sqrt(2 (1 - cos)),
        # spread over V entries, five of them
        tol = (2 * (1e-4 if dtype == torch.float32 else 1e-3)) ** 0.5 * logits.norm(dim=-1) / V ** 0.5 * 5
        assert bool((best <= tol).all()), (best / tol).max()
        same += int((new == truth[b, :len(new)]).sum())
        total += len(new)
    if same == total:  # no near-tie: every right draft was kept
        assert accepted == 2 * (3 + 0 + 2 + 0 + 7 + 1 + 3 + 1)
    last = run(model, cache, torch.tensor([[t[-1]] for t in texts], device="cuda"))
    for b in range(2):  # the kept rows are those of the text
        close(last[b], recompute(model, torch.tensor([texts[b]], device="cuda"))[0, -1:], dtype)
    cache.free(*truth_cache)
    assert cache.free_pages >= free


def _up(parents, i):
    while i >= 0:
        yield i
        i = parents[i]


def test_drawn_drafts():
    """Tokens drawn from a draft distribution: u = 0 keeps every token of positive probability, u near 1
    none where the draft is surer than the model; the length follows."""
    print("case: drawn drafts", flush=True)
    model, cache = llama(), TurboQuantPagedCache(16, 2, 32)
    run(model, cache, ids(2, 20))
    tokens = ids(2, 5, 9)
    q = torch.zeros(2, 4, V, device="cuda").scatter_(-1, tokens[:, 1:, None], 1.0)
    out = speculative_step(model, cache, tokens, draft_probs=q, uniforms=torch.zeros(2, 5, device="cuda"))
    assert [o[:-1] for o in out] == tokens[:, 1:].tolist() and cache.lengths() == [25, 25]
    root = torch.tensor([[o[-1]] for o in out], device="cuda")
    tokens = torch.cat([root, ids(2, 4, 10)], 1)
    q = torch.zeros(2, 4, V, device="cuda").scatter_(-1, tokens[:, 1:, None], 1.0)
    out = speculative_step(model, cache, tokens, draft_probs=q, uniforms=torch.full((2, 5), 0.999, device="cuda"))
    assert [len(o) for o in out] == [1, 1] and cache.lengths() == [26, 26]
    # a tree of one node draws the next token only; -2 pads
    out = speculative_step(model, cache, torch.tensor([[out[0][0], 0], [out[1][0], 0]], device="cuda"), [-1, -2])
    assert [len(o) for o in out] == [1, 1] and cache.lengths() == [27, 27]


def test_refusals_under_a_model():
    print("case: paged refusals", flush=True)
    model, cache = llama(), TurboQuantPagedCache(16, 2, 32)
    run(model, cache, ids(2, 20))
    with pytest.raises(ValueError, match="mask"):  # left padding
        mask = torch.ones(2, 22, dtype=torch.long, device="cuda")
        mask[0, 0] = 0
        model(input_ids=ids(2, 22), attention_mask=mask, past_key_values=TurboQuantPagedCache(16, 2, 32), use_cache=True)
    with pytest.raises(ValueError, match="at most 64"):
        with cache.draft():
            run(model, cache, ids(2, 65))
    with pytest.raises(RuntimeError, match="full"):
        run(model, cache, ids(2, 300))
    assert cache.lengths() == [20, 20]
    for m in model.modules():
        if hasattr(m, "causal_mode"):
            m.causal_mode = False
    with pytest.raises(ValueError, match="causal"):
        run(model, cache, ids(2, 3))
    for m in model.modules():
        if hasattr(m, "causal_mode"):
            m.causal_mode = "auto"
    close(run(model, cache, ids(2, 3, 4)), recompute(model, torch.cat([ids(2, 20), ids(2, 3, 4)], 1))[:, 20:])
    short = TurboQuantPagedCache(16, 3, 32)  # more layers than the model has
    run(model, short, ids(1, 4))
    with pytest.raises(RuntimeError, match="wrote 2 of the cache's 3 layers"):
        run(model, short, ids(1, 4))


def test_positions_of_unequal_sequences_and_trees():
    """Without position_ids: sequences of unequal length, and a drafted tree, against recomputation."""
    print("case: paged positions", flush=True)
    model, cache = llama(), TurboQuantPagedCache(40, 2, 32)
    text = ids(2, 120)
    a, b = cache.add(2)
    for i, n in ((a, 90), (b, 33)):
        cache.use([i])
        with torch.no_grad():
            model(input_ids=text[[a, b].index(i)][None, :n], past_key_values=cache, use_cache=True)
    cache.use([a, b])
    with torch.no_grad():
        got = model(input_ids=torch.stack([text[0, 90:95], text[1, 33:38]]), past_key_values=cache, use_cache=True).logits.float()
    close(got[0], recompute(model, text[:1, :95])[0, 90:])
    close(got[1], recompute(model, text[1:, :38])[0, 33:])
    tree = torch.tensor([-1, 0, 0, 1], dtype=torch.int32, device="cuda")
    drafted = torch.stack([text[0, [95, 96, 7, 97]], text[1, [38, 39, 7, 40]]])
    with cache.draft(tree), torch.no_grad():
        got = model(input_ids=drafted, past_key_values=cache, use_cache=True).logits.float()
    for row, (n, t) in enumerate(((95, text[0]), (38, text[1]))):
        close(got[row, [0, 1, 3]], recompute(model, t[None, :n + 3])[0, n:])
        close(got[row, 2], recompute(model, torch.cat([t[:n + 1], t[7:8]])[None])[0, -1])
    assert cache.lengths() == [95, 38]


def test_a_step_that_fails_leaves_the_cache_as_it_was(monkeypatch):
    print("case: paged failures", flush=True)
    from transformers_turboquant import paged_cache

    model, cache = llama(), TurboQuantPagedCache(6, 2, 32)
    with pytest.raises(RuntimeError, match="full"):
        run(model, cache, ids(4, 70))
    assert cache.active == [] and cache.free_pages == 6 and cache.pool is None
    real = paged_cache.append_tree_attention

    def fail(*a, **k):
        raise ValueError("refused by the operator")

    monkeypatch.setattr(paged_cache, "append_tree_attention", fail)
    with pytest.raises(ValueError, match="refused by the operator"):
        run(model, cache, ids(3, 40))
    assert cache.active == [] and cache.free_pages == 6
    monkeypatch.setattr(paged_cache, "append_tree_attention", real)
    plain = TurboQuantPagedCache(6, 2, 32)  # where nothing failed
    # another batch; bit for bit
    assert torch.equal(run(model, cache, ids(2, 40)), run(model, plain, ids(2, 40)))
    monkeypatch.setattr(paged_cache, "append_tree_attention", fail)
    with pytest.raises(ValueError, match="refused by the operator"):
        run(model, cache, ids(2, 30, 6))
    assert cache.lengths() == [40, 40] and cache.free_pages == 2
    monkeypatch.setattr(paged_cache, "append_tree_attention", real)
    assert torch.equal(run(model, cache, ids(2, 3, 4)), run(model, plain, ids(2, 3, 4)))
    assert cache.lengths() == plain.lengths() and cache.free_pages == plain.free_pages
