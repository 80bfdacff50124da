"""TurboQuantPagedCache(shared_prefix=True) with batches large enough that shared pages are read once for a group.

prefix_attention works a small batch sequence by sequence, whatever the groups say; here every step's operands are checked
to be past that rule.  At each layer of each step the groups that the cache hands over are compared with the pages of its
table, and the output with tree attention of every sequence over its own pages (16 2^-10 of the norm, as
tests/test_gpu_tree_attention.py derives it for one output; both sides may be off by that, and are rounded to their type)."""

import pytest
import torch

from test_gpu_paged_cache import V, close, ids, llama, recompute, run
from transformers_turboquant import TurboQuantPagedCache, paged_cache, speculative_step
from turboquant_pytorch import _native, tree_attention

pytestmark = pytest.mark.gpu


def claims_hold(table, lengths, groups, page):
    """Sequences that follow one another with equal (id, shared) have the pages of their first `shared` positions in common, and
    are no shorter."""
    for b, (i, shared) in enumerate(groups):
        if i < 0 or not shared:
            continue
        if shared % page or lengths[b] < shared:
            return False
        if b and groups[b - 1] == [i, shared] and table[b][:shared // page] != table[b - 1][:shared // page]:
            return False
    return True


class Checked:
    """append_prefix_attention as the cache calls it, every call checked."""

    def __init__(self, monkeypatch):
        self.calls, self.detected, self.real = [], 0, paged_cache.append_prefix_attention
        monkeypatch.setattr(paged_cache, "append_prefix_attention", self)

    def __call__(self, k, v, q, kc, vc, pool, layer, table, lengths, groups, parents, scale, out_dtype):
        out = self.real(k, v, q, kc, vc, pool, layer, table, lengths, groups, parents, scale, out_dtype)
        B, Hq, T, D = q.shape
        H, P, W = pool.num_kv_heads, pool.page_size, table.shape[1]
        columns = Hq // H * T
        # more rounds of 128 keys than any number of resident blocks, columns that do not fill two tiles of 16
        rounds = B * -(-W * P // 128) * H * -(-columns // 32)
        assert rounds > 4 * torch.cuda.get_device_properties(0).multi_processor_count and columns % 32
        shape = (B, Hq, H, T, W, P, D, pool.bits)
        assert _native.lib().tq_prefix_workspace_size(*shape) != _native.lib().tq_tree_workspace_size(*shape)
        rows = table.tolist(), lengths.tolist(), groups.tolist()
        assert claims_hold(*rows, P)
        alone = tree_attention(q, kc, vc, pool, layer, table, lengths, parents, scale, torch.float32)
        bound = (2 * 16 * 2.0 ** -10 + torch.finfo(out.dtype).eps / 2) * alone.norm()
        assert (out.float() - alone).norm() <= bound
        self.calls.append((B, T, [g[1] for g in rows[2]]))
        # an oracle that takes one page more for shared, where it is not, fails both checks
        wrong = [[i, n + P] if n else [i, n] for i, n in rows[2]]
        for b in range(1, B):
            shared = rows[2][b][1]
            if shared and rows[2][b] == rows[2][b - 1] and rows[0][b][shared // P] != rows[0][b - 1][shared // P] and \
                    rows[1][b] >= shared + P <= rows[1][b - 1]:
                assert not claims_hold(rows[0], rows[1], wrong, P)
                theirs = table.clone()
                theirs[b, shared // P] = table[b - 1, shared // P]
                other = tree_attention(q, kc, vc, pool, layer, theirs, lengths, parents, scale, torch.float32)
                assert (out[b].float() - other[b]).norm() > 4 * (out[b].float() - alone[b]).norm()
                self.detected += 1
                break
        return out


@pytest.mark.parametrize("dtype,heads,kv,n,bits", [(torch.float32, 16, 8, 20, 3), (torch.bfloat16, 8, 8, 24, 2), (torch.float16, 16, 4, 40, 4)])
def test_steps_over_shared_pages(dtype, heads, kv, n, bits, monkeypatch):
    print("case: shared pages", dtype, heads, kv, n, bits, flush=True)
    checked = Checked(monkeypatch)
    model = llama(dtype, heads, kv, 1024, bits)
    prompt = ids(1, 1000)
    cache = TurboQuantPagedCache(600, 2, 32, shared_prefix=True)
    (a,) = cache.add()
    cache.use([a])
    run(model, cache, prompt)
    seqs = [a, *cache.fork(a, n - 1)]
    cache.use(seqs)
    texts = {s: prompt[0].tolist() for s in seqs}

    def step(tokens):
        tokens = tokens.cuda()
        got = run(model, cache, tokens)
        for s, row in zip(cache.active, tokens.tolist()):
            texts[s] += row
        return got

    def compare(got, some):
        for b in some:
            whole = torch.tensor([texts[cache.active[b]]], device="cuda")
            close(got[b], recompute(model, whole)[0, -got.shape[1]:], dtype)

    g = torch.Generator().manual_seed(4)
    draw = lambda B, T: torch.randint(0, V, (B, T), generator=g)
    for T in (1, 1, 7):  # single tokens, then some at once
        compare(step(draw(n, T)), (0, 1, n - 1))
    assert len(checked.calls) == 6 and all(c[2] == [992] * n for c in checked.calls)

    # drafted trees: what is kept differs from sequence to sequence
    tokens = draw(n, 5)
    before = cache.lengths()
    out = speculative_step(model, cache, tokens.cuda(), [-1, 0, 0, 1, 2], uniforms=torch.rand(n, 5, generator=g).cuda())
    for s, t, new, was, now in zip(cache.active, tokens.tolist(), out, before, cache.lengths()):
        texts[s] += t[:1] + new[:-1]
        assert now == was + len(new) == len(texts[s])
    compare(step(draw(n, 1)), (0, n // 2))

    # pages of their own behind the prompt, and copies on writing: the youngest forks share more than the prompt
    compare(step(draw(n, 15 if heads == kv else 13 if heads == 2 * kv else 7)), (1,))
    for _ in range(4):
        step(draw(n, 7))
    assert checked.detected
    cache.use([seqs[1]])
    step(draw(1, 400))
    young = cache.fork(seqs[1], 3)
    for s in young:
        texts[s] = list(texts[seqs[1]])
    order = [*young, seqs[1], *seqs[4:], seqs[0]]
    cache.use(order)
    compare(step(draw(len(order), 1)), (0, 3, 4, len(order) - 1))
    shared = checked.calls[-1][2]
    assert shared[:4] == [len(texts[young[0]]) // 32 * 32] * 4 and shared[4:] == [992] * (len(order) - 4)
    cache.crop(-70)  # the shortest end in the prompt again, whose last page they write
    for s in order:
        texts[s] = texts[s][:-70]
    compare(step(draw(len(order), 2)), (0, 5, len(order) - 1))
    cache.free(*order[5:8])
    rest = order[:5] + order[8:]
    cache.use(rest[::-1])
    compare(step(draw(len(rest), 1)), (0, len(rest) - 1))
    assert cache.lengths() == [len(texts[s]) for s in cache.active]
