"""Argument checks of sampling, on the CPU: meta tensors, and C entry points that refuse before any launch."""

import pytest
import torch

from turboquant_pytorch import _native, filter_probs, sample_tokens
from turboquant_pytorch._ops import ops

M = "meta"
N, V = 5, 1000


def _e(*shape, dtype=torch.float32, device=M):
    return torch.empty(*shape, dtype=dtype, device=device)


def _args(draw):
    a = dict(logits=_e(N, V, dtype=torch.bfloat16), u=_e(N), ts=None, t=0.7, ks=None, k=5, ps=None, p=0.9, ms=None, m=0.1)
    if not draw:
        del a["u"]
    return a


@pytest.mark.parametrize("draw", [True, False])
@pytest.mark.parametrize("bad,match", [
    (dict(logits=_e(N, V, dtype=torch.float64)), "logits must be"),
    (dict(logits=_e(N * V)), "logits must be"),
    (dict(logits=_e(V, N).t()), "contiguous along"),
    (dict(logits=_e(N, 0)), "1 to 2\\^24"),
    (dict(logits=_e(1, (1 << 24) + 1)), "1 to 2\\^24"),
    (dict(ts=_e(N, dtype=torch.float64)), "temperature must be"),
    (dict(ts=_e(N + 1)), "temperature must be"),
    (dict(ts=_e(2 * N)[::2]), "contiguous"),
    (dict(ks=_e(N)), "top_k must be"),
    (dict(ks=_e(N, dtype=torch.int64)), "top_k must be"),
    (dict(ps=_e(N, 1)), "top_p must be"),
    (dict(ms=_e(N, device="cpu")), "expected meta"),
    (dict(t=-0.1), "must not be negative"),
    (dict(t=float("nan")), "must not be negative"),
    (dict(k=-1), "must not be negative"),
    (dict(k=1 << 31), "must not be negative"),
    (dict(p=1.1), "lie in"),
    (dict(p=-0.1), "lie in"),
    (dict(m=1.5), "lie in"),
    (dict(m=float("nan")), "lie in"),
])
def test_refuses(draw, bad, match):
    fn = ops().sample_tokens if draw else ops().filter_probs
    for ks in (None, _e(N, dtype=torch.int32)):
        out = fn(*dict(_args(draw), ks=ks).values())
        assert (out.shape, out.dtype) == (((N,), torch.int64) if draw else ((N, V), torch.float32))
    with pytest.raises(RuntimeError, match=match):
        fn(*dict(_args(draw), **bad).values())


@pytest.mark.parametrize("u,match", [(_e(N, dtype=torch.float64), "uniforms must be"), (_e(N - 1), "uniforms must be"),
                                     (_e(N, device="cpu"), "expected meta"), (_e(2 * N)[::2], "uniforms must be")])
def test_refuses_uniforms(u, match):
    with pytest.raises(RuntimeError, match=match):
        ops().sample_tokens(*dict(_args(True), u=u).values())


def test_python_checks():
    assert sample_tokens(_e(2, 3, V), _e(2, 3), top_k=_e(2, 3, dtype=torch.int32)).shape == (2, 3)
    assert filter_probs(_e(2, 3, V), temperature=_e(2, 3)).shape == (2, 3, V)
    with pytest.raises(ValueError, match="uniforms must be"):
        sample_tokens(_e(2, 3, V), _e(6))
    with pytest.raises(ValueError, match="top_p must be a number"):
        filter_probs(_e(2, 3, V), top_p=_e(2))
    with pytest.raises((RuntimeError, NotImplementedError)):
        sample_tokens(torch.zeros(1, 4), torch.zeros(1))


def test_c_entries_refuse():
    lib = _native.lib()
    none = None

    def call(logits=16, dt=0, ld=10, n=1, v=10, t=1.0, k=0, p=1.0, m=0.0, u=16, ws=none, b=0):
        return lib.tq_sample_tokens(logits, dt, ld, n, v, u, none, t, none, k, none, p, none, m, 16, ws, b, none)

    for kw, msg in ((dict(dt=7), b"dtype"), (dict(v=0), b"bad shape"), (dict(ld=-1), b"bad shape"), (dict(n=-1), b"bad shape"),
                    (dict(v=(1 << 24) + 1), b"2^24"), (dict(t=-1.0), b"negative"), (dict(k=-1), b"negative"), (dict(p=float("nan")), b"negative"),
                    (dict(logits=none), b"null"), (dict(u=none), b"null"), (dict(), b"workspace"), (dict(ws=8, b=1 << 30), b"workspace"),
                    (dict(ws=16, b=16), b"workspace")):
        assert call(**kw) == -1 and msg in lib.tq_last_error(), (kw, lib.tq_last_error())
    assert call(n=0, logits=none) == 0
    assert lib.tq_filter_probs(16, 0, 10, 1, 10, none, 1.0, none, 0, none, 1.0, none, 0.0, none, 16, 1 << 30, none) == -1
    assert lib.tq_sample_workspace_size(0, 10) == 0 and lib.tq_sample_workspace_size(1, (1 << 24) + 1) == 0
    assert lib.tq_sample_workspace_size(1, 1) > 0


@pytest.mark.parametrize("n,v,taken", [((1 << 22) - 1, 10, True), (1 << 22, 10, False), ((1 << 22) - 1, 1 << 15, True),
                                       ((1 << 22) - 1, (1 << 15) + 1, True), ((1 << 22) - 1, (1 << 16) + 1, False),
                                       (1 << 14, 1 << 24, False), ((1 << 14) - 1, 1 << 24, True), ((1 << 31) - 1, 1, False)])
def test_no_more_rows_and_chunks_than_a_launch_has_threads_for(n, v, taken):
    """A grid of HIP has fewer than 2^32 threads along x: 1024 work on a row, 512 on a chunk of 2^15 tokens."""
    lib, none = _native.lib(), None
    assert (lib.tq_sample_workspace_size(n, v) > 0) == taken
    args = [dict(_args(True), logits=_e(n, v, dtype=torch.bfloat16), u=_e(n)), dict(_args(False), logits=_e(n, v, dtype=torch.bfloat16))]
    for fn, a in zip((ops().sample_tokens, ops().filter_probs), args):
        if taken:
            assert fn(*a.values()).shape[0] == n
        else:
            with pytest.raises(RuntimeError, match="fewer than 2\\^22 rows"):
                fn(*a.values())
    if not taken:
        for call in (lambda: lib.tq_sample_tokens(16, 0, v, n, v, 16, none, 1.0, none, 0, none, 1.0, none, 0.0, 16, 16, 1 << 50, none),
                     lambda: lib.tq_filter_probs(16, 0, v, n, v, none, 1.0, none, 0, none, 1.0, none, 0.0, 16, 16, 1 << 50, none)):
            assert call() == -1 and b"fewer than 2^22 rows" in lib.tq_last_error()


def test_logits_that_are_strided_along_the_vocabulary():
    for x in (_e(V, N).t(), _e(N, 2 * V)[:, ::2], _e(N, 1, 3 * V)[..., ::3], _e(V, 2, N).permute(2, 1, 0)):
        assert sample_tokens(x, _e(*x.shape[:-1]), top_k=3).shape == x.shape[:-1]
        assert filter_probs(x, top_p=0.5).shape == x.shape
