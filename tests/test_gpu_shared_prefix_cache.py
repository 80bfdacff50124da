"""Several continuations of one prompt under a model: forks of a paged cache whose shared pages are read once, tokens
drawn by sample_tokens, drafted tokens verified against filter_probs; against the same without sharing."""

import pytest
import torch

from test_gpu_paged_cache import V, close, ids, llama, recompute, run
from transformers_turboquant import TurboQuantPagedCache, paged_cache, speculative_step
from turboquant_pytorch import filter_probs, sample_tokens, verify_drafts

pytestmark = pytest.mark.gpu


def forked(model, prompt, n, **kw):
    cache = TurboQuantPagedCache(64, 2, 32, **kw)
    (a,) = cache.add()
    cache.use([a])
    run(model, cache, prompt)
    cache.use([a, *cache.fork(a, n - 1)])
    return cache


@pytest.mark.parametrize("dtype,heads,kv,hidden,bits", [(torch.float32, 8, 2, 1024, 3), (torch.bfloat16, 8, 2, 1024, 2),
                                                        (torch.float16, 4, 4, 256, 4)])
def test_forks_match_recomputation(dtype, heads, kv, hidden, bits, monkeypatch):
    print("case: shared forks", dtype, heads, bits, flush=True)
    calls = []
    real = paged_cache.append_prefix_attention
    monkeypatch.setattr(paged_cache, "append_prefix_attention", lambda *a: calls.append(a[9].tolist()) or real(*a))
    model = llama(dtype, heads, kv, hidden, bits)
    prompt, more = ids(1, 205), ids(5, 40, seed=6)
    cache = forked(model, prompt, 5, shared_prefix=True)
    got = torch.cat([run(model, cache, more[:, lo:hi]) for lo, hi in ((0, 1), (1, 2), (2, 9), (9, 40))], 1)
    assert len(calls) == 8 and calls[0] == [[0, 192]] * 5
    for b in range(5):
        close(got[b], recompute(model, torch.cat([prompt, more[b:b + 1]], 1))[0, 205:], dtype)
    # what is cached is the same as without sharing
    plain = forked(model, prompt, 5)
    want = run(model, plain, more)
    close(got, want, dtype)
    assert cache.lengths() == plain.lengths() and cache.free_pages == plain.free_pages
    # sequences that share nothing run as they always did
    (new,) = cache.add()
    cache.use([new])
    (other,) = plain.add()
    plain.use([other])
    for part in (more[:1, :3], more[:1, 3:4]):
        assert torch.equal(run(model, cache, part), run(model, plain, part))
    assert len(calls) == 8


def test_beam_search():
    model, prompt = llama(), ids(2, 130)
    kw = dict(max_new_tokens=10, min_new_tokens=10, do_sample=False, num_beams=3, output_scores=True,
              return_dict_in_generate=True, attention_mask=torch.ones_like(prompt))
    with torch.no_grad():
        ref = model.generate(prompt, use_cache=True, past_key_values=TurboQuantPagedCache(128, 2, 32), **kw)
        got = model.generate(prompt, use_cache=True, past_key_values=TurboQuantPagedCache(128, 2, 32, shared_prefix=True), **kw)
    same = (got.sequences == ref.sequences).all(-1)
    gap = (got.sequences_scores - ref.sequences_scores).abs() / ref.sequences_scores.abs()
    assert bool((same | (gap < 1e-3)).all()), (same, gap)


def test_samples_of_one_prompt():
    """A decoding loop: attention over shared pages and sampling, every token checked against the logits it came from."""
    model, prompt = llama(torch.bfloat16), ids(1, 300)
    n, g = 6, torch.Generator(device="cuda").manual_seed(3)
    cache = forked(model, prompt[:, :-1], n, shared_prefix=True)
    tokens, texts = prompt[:, -1:].expand(n, 1).contiguous(), [[] for _ in range(n)]
    setting = dict(temperature=torch.linspace(0.0, 1.5, n, device="cuda"), top_k=50, top_p=0.95)
    for step in range(12):
        logits = run(model, cache, tokens)[:, -1]
        u = torch.rand(n, device="cuda", generator=g)
        nxt = sample_tokens(logits, u, **setting)
        probs = filter_probs(logits, **setting)
        assert (probs.gather(1, nxt[:, None]) > 0).all() and ((probs > 0).sum(1) <= 50).all()
        assert nxt[0] == logits[0].argmax()
        # a sequence without drafts: verification of the root alone draws from the same distribution
        _, count, same = verify_drafts(tokens, probs[:, None], u[:, None])
        assert (count == 1).all()
        c = probs.double().cumsum(1)
        goal = u.double() * c[:, -1]
        near = ((c.gather(1, nxt[:, None])[:, 0] - goal).abs() < 1e-6) | ((c.gather(1, same[:, None])[:, 0] - goal).abs() < 1e-6)
        assert ((nxt == same) | near).all()
        for b in range(n):
            texts[b].append(int(nxt[b]))
        tokens = nxt[:, None]
    assert cache.lengths() == [299 + 12] * n and len({tuple(t) for t in texts}) > 1
    for b in (0, n - 1):
        whole = torch.cat([prompt, torch.tensor([texts[b]], device="cuda")], 1)
        last = recompute(model, whole[:, :-1])[0, -1]
        close(logits[b][None], last[None], torch.bfloat16)


def test_speculation_in_forks_with_filters():
    """Trees and chains in sequences that share pages, verified against filtered distributions: an accepted or
    emitted token is one that the filter keeps."""
    model, prompt = llama(), ids(1, 170)
    cache, plain = forked(model, prompt[:, :-1], 4, shared_prefix=True), forked(model, prompt[:, :-1], 4)
    texts = [prompt[0].tolist() for _ in range(4)]
    g = torch.Generator().manual_seed(2)
    for parents in (None, [-1, 0, 0, 1, 2, -2], [-1]):
        T = 4 if parents is None else len(parents)
        drafted = torch.randint(0, V, (4, T), generator=g)
        drafted[:, 0] = torch.tensor([t[-1] for t in texts])
        u = torch.rand(4, T, generator=g).cuda()
        out = speculative_step(model, cache, drafted.cuda(), parents, uniforms=u, temperature=0.8, top_k=20, top_p=0.9)
        ref = speculative_step(model, plain, drafted.cuda(), parents, uniforms=u, temperature=0.8, top_k=20, top_p=0.9)
        assert [len(o) for o in out] == [len(o) for o in ref]
        assert cache.lengths() == plain.lengths()
        for b, new in enumerate(out):
            # the likeliest 20 of a recomputation, and 5 more for what other kernels round
            best = recompute(model, torch.tensor([texts[b]], device="cuda"))[0, -1].topk(25).indices
            assert new[0] in best.tolist()
            texts[b] += new
        if out != ref:  # a draw next to a border: the texts differ from here on
            break
