"""Argument checks of attention over shared prefixes, on the CPU: meta tensors, and C entry points that refuse before any
launch.  No GPU is touched."""

import pytest
import torch

from test_draft_ops_cpu import B, D, F16, H, I32, I64, P, POOL, T, W, _append_args, _e, _refuses, _tree_args
from turboquant_pytorch import _native, prefix_groups
from turboquant_pytorch._ops import ops


def _with_groups(args):
    out = {}
    for k, v in args.items():
        out[k] = v
        if k == "lengths":
            out["groups"] = _e(B, 2, dtype=I32)
    return out


@pytest.mark.parametrize("bad,match", POOL + [
    (dict(groups=_e(B, 2, dtype=I64)), "int32"),
    (dict(groups=_e(B, 3, dtype=I32)), "groups must be"),
    (dict(groups=_e(B + 1, 2, dtype=I32)), "groups must be"),
    (dict(groups=_e(2 * B, dtype=I32)), "groups must be"),
    (dict(groups=_e(2, B, dtype=I32).t()), "contiguous"),
    (dict(groups=_e(B, 2, dtype=I32, device="cpu")), "expected meta"),
    (dict(lengths=_e(B, 1, dtype=I32)), "lengths must be"),
    (dict(parents=_e(T + 1, dtype=I32)), "parents must be"),
    (dict(table=_e(B + 1, W, dtype=I32)), "block_table has"),
    (dict(bits=4), "the pool holds"),
    (dict(out=torch.int32), "out_dtype"),
    (dict(vpit=_e(D, D, dtype=F16)), "Pi_v"),
])
def test_prefix_attention_refuses(bad, match):
    for fn, args in ((ops().prefix_attend, _tree_args(True)), (ops().prefix_page_attend, _append_args())):
        args = _with_groups(args)
        for par in (None, _e(T, dtype=I32), _e(B, T, dtype=I32)):
            out = fn(*dict(args, parents=par).values())
            assert out.shape == (B, T, 8, D) and out.dtype == torch.bfloat16
        _refuses(fn, args, bad, match)


def test_more_work_than_an_index_counts_is_refused_before_a_row_is_written():
    n = 65535
    big = dict(table=_e(n, (1 << 24) // P, dtype=I32), lengths=_e(n, dtype=I32), groups=_e(n, 2, dtype=I32))
    for args, fn in ((_append_args(), ops().prefix_page_attend), (_tree_args(True), ops().prefix_attend)):
        new = {k: _e(n, *args[k].shape[1:], dtype=args[k].dtype) for k in ("k", "v", "q") if k in args}
        _refuses(fn, _with_groups(args), {**new, **big}, "blocks of work")


@pytest.mark.parametrize("positions", [1 << 16, 1 << 18, 1 << 22])
def test_the_operators_refuse_what_the_library_does(positions):
    n, args = 65535, _tree_args(True)
    q = args["q"]
    wide = dict(q=_e(n, *q.shape[1:], dtype=q.dtype), table=_e(n, positions // P, dtype=I32), lengths=_e(n, dtype=I32),
                groups=_e(n, 2, dtype=I32))
    size = _native.lib().tq_prefix_workspace_size(n, q.shape[1], H, q.shape[2], positions // P, P, D, args["bits"])
    if size:
        assert ops().prefix_attend(*dict(_with_groups(args), **wide).values()).shape[0] == n
    else:
        _refuses(ops().prefix_attend, _with_groups(args), wide, "blocks of work")
    assert (size > 0) == (positions == 1 << 16)


def test_groups():
    assert prefix_groups([2, 1, 3], [64, 0, 100], device="cpu").tolist() == [[0, 64]] * 2 + [[1, 0]] + [[2, 100]] * 3
    assert prefix_groups([], [], device="cpu").shape == (0, 2)
    for sizes, shared in (([1], [1, 2]), ([0], [4]), ([2], [-1]), ([1], [2 ** 31])):
        with pytest.raises(ValueError):
            prefix_groups(sizes, shared, device="cpu")


def test_c_entry_refuses():
    lib = _native.lib()
    none = None

    def call(B=1, T=2, d=64, bits=3, P=64, W=2, Hq=4, groups=16, ws=none, q=16, n=0):
        return lib.tq_prefix_attention(q, *[16] * 6, bits, *[16] * 4, 5, P, 16, W, W, 16, groups, none, 0, B, Hq, 2, T, d, 0.1, 0.1,
                                       16, 0, 0, 0, 0, ws, n, none)

    assert call(d=96) == -2 and call(bits=5) == -2
    for kw, msg in ((dict(T=65), b"at most 64"), (dict(T=0), b"bad shape"), (dict(Hq=5), b"bad shape"), (dict(P=16), b"power of two"),
                    (dict(P=96), b"power of two"), (dict(W=0), b"does not hold"), (dict(W=1 << 20), b"2^24"),
                    (dict(B=65536), b"65535"), (dict(B=65535, T=64, W=1 << 18), b"2^31"), (dict(groups=none), b"null"),
                    (dict(q=8), b"16-byte"), (dict(), b"workspace"), (dict(ws=8, n=1 << 40), b"workspace"),
                    (dict(ws=16, n=16), b"workspace")):
        assert call(**kw) == -1 and msg in lib.tq_last_error(), (kw, lib.tq_last_error())
    assert call(B=0, groups=none) == 0
    assert lib.tq_prefix_workspace_size(1, 4, 2, 65, 2, 64, 64, 3) == 0
    assert lib.tq_prefix_workspace_size(1, 4, 2, 1, 2, 64, 96, 3) == 0
