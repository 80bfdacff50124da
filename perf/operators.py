"""Performance cases of the operators that serve drafted tokens over a paged compressed KV cache.

  attend   attention of T drafted tokens (a tree; T = 1 is a decoding step) of every sequence over
           its pages of compressed keys and values and over their ancestors among the drafted ones
  write    compressed rows of new tokens into the pages of a layer
  read     a layer's cached rows out of its pages, contiguous again
  copy     pages of every layer copied (a sequence forked: its last page is its own from then on)
  keep     the rows of an accepted path moved down behind the cached ones, in every layer
  verify   drafted tokens against the target's probabilities, and the next token, from given uniforms

``run`` computes each in elementary torch operations, or with ``own`` through the framework.
``exact`` restates it in float64.
"""

from __future__ import annotations

import functools
import math
import os
import sys

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_SEED = 42  # the default seed of apply_turboquant
_PLANES = ("kcodes", "ksigns", "krn", "kvn", "vcodes", "vvn")


# ------------------------------------------------------------------ cases
def listed() -> list[dict]:
    return [
        # one interactive sequence of a GPT-2-shaped layer, a page of text cached, one token
        _attend("attend_d64_b1_t1_1k", 1, 12, 12, 64, 1, 1000, 3, 64),
        # serving 16 sequences of unequal length with a Llama-3-8B-shaped layer, one token each
        _attend("attend_d128_b16_t1_32k", 16, 32, 8, 128, 1, 32700, 3, 64),
        # speculation for one sequence: a tree of 16 drafted tokens
        _attend("attend_d128_b1_t16_4k", 1, 32, 8, 128, 16, 4000, 3, 64),
        # the same for a batch of unequal sequences at long context
        _attend("attend_d128_b16_t16_32k", 16, 32, 8, 128, 16, 32700, 3, 64),
        # a wide tree under 8 query heads per kv head (Qwen2.5-3B shape), padded trees, float16
        _attend("attend_d128_b4_t61_gqa8", 4, 16, 2, 128, 61, 8191, 4, 128, dtype="f16"),
        # a prompt chunk of four sequences goes into a layer's pages
        dict(name="write_b4_s2000", kind="write", B=4, Hkv=8, D=128, S=2000, len=1000, bits=3, page=64),
        # cached prefixes laid out contiguously for the prompt kernels
        dict(name="read_b4_9000", kind="read", B=4, Hkv=8, D=128, S=9000, len=9000, bits=3, page=64),
        # 16 sequences forked: their last pages copied in 32 layers
        dict(name="copy_16_pages_32_layers", kind="copy", B=16, Hkv=8, D=128, bits=3, page=64, layers=32),
        # accepted paths of 16 sequences compacted in 32 layers
        dict(name="keep_b16_t16_32_layers", kind="keep", B=16, Hkv=8, D=128, T=16, bits=3, page=64, layers=32),
        # speculation for one sequence: a chain of 4 drafted tokens, GPT-2's vocabulary
        dict(name="verify_chain_b1", kind="verify", B=1, T=5, V=50257, dtype="f32", tree=False),
        # chains of a served batch, a Llama-3-sized vocabulary
        dict(name="verify_chain_b64", kind="verify", B=64, T=8, V=128256, dtype="f32", tree=False),
        # trees of chosen candidates, a Qwen2.5-sized vocabulary
        dict(name="verify_tree_b16", kind="verify", B=16, T=32, V=151936, dtype="bf16", tree=True),
    ]


def _attend(name, B, Hq, Hkv, D, T, n, bits, page, dtype="bf16"):
    case = dict(name=name, kind="attend", B=B, Hq=Hq, Hkv=Hkv, D=D, T=T, len=n, bits=bits, page=page, dtype=dtype)
    return case if name else {k: v for k, v in case.items() if k != "name"}


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng) -> dict:
    kind = rng.choice(["attend"] * 5 + ["write", "read", "copy", "keep", "verify", "verify"])
    bits, page = rng.choice([2, 3, 3, 4]), rng.choice([32, 64, 64, 128, 256])
    D = rng.choice([64, 128, 128])
    if kind == "attend":
        Hq, Hkv = rng.choice([(12, 12), (32, 8), (16, 2), (32, 32), (14, 2), (28, 4), (64, 8)])
        B, n = _log_int(rng, 1, 16), _log_int(rng, 17, 32700)
        T = rng.choice([1, 1, 2, 4, 7, 16, 25, 33, 64])
        while B * n * Hkv * D > 16 * 32700 * 8 * 128 or B * n * Hq * T * D > 16 * 32700 * 32 * 16 * 128:
            n = (n + 1) // 2
        return _attend(None, B, Hq, Hkv, D, T, n, bits, page, rng.choice(["bf16", "bf16", "f16"]))
    if kind == "verify":
        B, T, V = _log_int(rng, 1, 64), _log_int(rng, 1, 33), _log_int(rng, 1000, 151936)
        while B * T * V > 64 * 8 * 128256:
            V = (V + 1) // 2
        return dict(kind="verify", B=B, T=T, V=V, dtype=rng.choice(["f32", "bf16", "f16"]), tree=rng.random() < 0.5)
    Hkv, B = rng.choice([2, 4, 8, 12, 32]), _log_int(rng, 1, 16)
    case = dict(kind=kind, B=B, Hkv=Hkv, D=D, bits=bits, page=page)
    if kind in ("write", "read"):
        S = _log_int(rng, 1, 9000)
        while B * S * Hkv * D > 4 * 9000 * 8 * 128:
            S = (S + 1) // 2
        return dict(case, S=S, len=S if kind == "read" else rng.randrange(0, 2000))
    layers = rng.choice([12, 24, 32, 36])
    while B * Hkv * D * page * layers > 16 * 8 * 128 * 64 * 32 and B > 1:
        B = (B + 1) // 2
    case = dict(case, B=B, layers=layers)
    return case if kind == "copy" else dict(case, T=rng.choice([2, 5, 8, 16, 33, 64]))


def _lengths(case) -> list[int]:
    """Cached positions of each sequence: the last one has them all, the others a share down to a quarter."""
    n, B = case["len"], case["B"]
    return [n] if B == 1 else [n - (3 * n * (B - 1 - b)) // (4 * (B - 1)) for b in range(B)]


def _record(case) -> tuple[dict, int]:
    """Bytes of a row in each plane, and in all."""
    D, bits = case["D"], case["bits"]
    w = {"kcodes": (D * (bits - 1) + 7) // 8, "ksigns": D // 8, "krn": 2, "kvn": 2, "vcodes": D * bits // 8, "vvn": 2}
    return w, sum(w.values())


# ------------------------------------------------------------------ inputs
@functools.lru_cache(maxsize=None)
def _codebook(D, bits):
    """Lloyd-Max centroids of N(0, 1/D): the centre of mass of each cell, iterated."""
    c = torch.linspace(-2.0, 2.0, 2 ** bits, dtype=torch.float64)
    for _ in range(400):
        e = torch.cat([torch.tensor([-40.0], dtype=torch.float64), (c[1:] + c[:-1]) / 2,
                       torch.tensor([40.0], dtype=torch.float64)])
        pdf = torch.exp(-e * e / 2) / math.sqrt(2 * math.pi)
        cdf = 0.5 * (1 + torch.erf(e / math.sqrt(2)))
        c = (pdf[:-1] - pdf[1:]) / (cdf[1:] - cdf[:-1])
    return (c / math.sqrt(D)).float()


def _pack(codes, b):
    """uint8 codes [..., D] as rows of D * b bits, the first code in the lowest bits."""
    D = codes.shape[-1]
    group = codes.reshape(*codes.shape[:-1], D // 8, 8).to(torch.int32)
    word = (group << (b * torch.arange(8, device=codes.device, dtype=torch.int32))).sum(-1, dtype=torch.int32)
    out = (word.unsqueeze(-1) >> (8 * torch.arange(b, device=codes.device, dtype=torch.int32))) & 255
    return out.to(torch.uint8).reshape(*codes.shape[:-1], D // 8 * b)


def _codes(g, shape, D, b, cent):
    """Packed codes of Gaussian coordinates, 2^18 rows at a time."""
    rows = math.prod(shape)
    bounds = ((cent[1:] + cent[:-1]) / 2).to(g.device)
    parts = []
    for at in range(0, rows, 1 << 18):
        y = torch.randn(min(1 << 18, rows - at), D, device=g.device, generator=g) / math.sqrt(D)
        parts.append(_pack(torch.bucketize(y, bounds).to(torch.uint8), b))
    return torch.cat(parts).reshape(*shape, -1)


def _bytes(g, *shape):
    return torch.randint(0, 256, shape, device=g.device, generator=g, dtype=torch.uint8)


def _norms(g, shape, mean, spread):
    return (mean * torch.exp(spread * torch.randn(shape, device=g.device, generator=g))).half()


def _rows(g, shape, case, cent):
    """The six planes of random compressed rows."""
    D, bits = case["D"], case["bits"]
    kvn = _norms(g, shape, math.sqrt(D), 0.25)
    return {"kcodes": _codes(g, shape, D, bits - 1, cent["key"]), "ksigns": _bytes(g, *shape, D // 8),
            "krn": (kvn.float() * (0.6, 0.34, 0.19)[bits - 2]).half(), "kvn": kvn,
            "vcodes": _codes(g, shape, D, bits, cent["value"]), "vvn": _norms(g, shape, math.sqrt(D), 0.1)}


def _parents(g, B, T, pads):
    """Trees in index order: a node's parent is one of the 7 nodes before it.  With pads, every
    other sequence drafted a quarter fewer tokens; the nodes behind have no place in its tree (-2)."""
    i = torch.arange(T, device=g.device)
    back = torch.randint(1, 8, (B, T), device=g.device, generator=g)
    par = (i - back).clamp(min=0)
    par[:, 0] = -1
    if pads:
        par[1::2, T - T // 4:] = -2
    return par.to(torch.int32)


def _table(g, case, lens, extra):
    """Each sequence's pages, scattered over the pool; entries behind its last page are -1."""
    P = case["page"]
    need = [(n + extra + P - 1) // P for n in lens]
    order = torch.randperm(sum(need) + 3, device=g.device, generator=g).to(torch.int32)
    table = torch.full((len(lens), max(need)), -1, dtype=torch.int32, device=g.device)
    at = 0
    for b, k in enumerate(need):
        table[b, :k] = order[at:at + k]
        at += k
    return table, sum(need) + 3


def prepare(case: dict, seed: int) -> dict:
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dev, kind, B = g.device, case["kind"], case["B"]
    st = {"case": case, "kind": kind}
    if kind == "verify":
        _prepare_verify(case, g, st)
    else:
        D, bits, H, P = case["D"], case["bits"], case["Hkv"], case["page"]
        cent = {"key": _codebook(D, bits - 1), "value": _codebook(D, bits)}
        layers = case.get("layers", 1)
        if kind == "copy":
            pages = 4 * B
            order = torch.randperm(pages, device=dev, generator=g).to(torch.int32)
            st["src"], st["dst"] = order[:B].clone(), order[B:2 * B].clone()
        elif kind == "keep":
            T = case["T"]
            # from the first pages on; two pages of room, for rows that cross a page's end
            lens = torch.randint(0, P, (B,), device=dev, generator=g)
            st["table"], pages = _table(g, case, [P] * B, max(P, T))
            st["lengths"] = lens.to(torch.int32)
            # an accepted path: the root, then nodes in rising order; those that move come from
            # behind every place that is written, so that a pass over the same rows can be repeated
            count = torch.randint(1, 1 + (T + 1) // 2, (B, 1), device=dev, generator=g)
            i = torch.arange(T, device=dev)
            pick = torch.where(i < count, 2.0, torch.rand(B, T, device=dev, generator=g)).argsort(1)
            path = torch.where(i < count - 1, pick, T).sort(1).values.roll(1, 1)
            path[:, 0] = 0
            st["count"] = count[:, 0].to(torch.int32)
            st["path"] = torch.where(i < count, path, -1).to(torch.int32)
        else:
            lens = _lengths(case)
            extra = case["T"] if kind == "attend" else case["S"] if kind == "write" else 0
            st["table"], pages = _table(g, case, lens, extra)
            st["lengths"] = torch.tensor(lens, dtype=torch.int32, device=dev)
        st["planes"] = {n: t.reshape(layers, pages, H, P, *t.shape[1:])
                        for n, t in _rows(g, (layers * pages * H * P,), case, cent).items()}
        if kind == "write":
            st["new"] = {n: t.reshape(B, H, case["S"], *t.shape[1:])
                         for n, t in _rows(g, (B * H * case["S"],), case, cent).items()}
        if kind == "attend":
            _prepare_attend(case, g, st, cent)
    if own:
        _handles(st)
    return st


def _prepare_attend(case, g, st, cent):
    """Queries, trees, and the matrices of a layer's compressors, drawn as the framework draws them."""
    B, Hq, D, T, dev = case["B"], case["Hq"], case["D"], case["T"], g.device
    w = {}
    for n, seed in (("pi", _SEED), ("pi_v", _SEED + 10000)):
        q, r = torch.linalg.qr(torch.randn(D, D, generator=torch.Generator().manual_seed(seed)))
        s = torch.where(torch.diagonal(r) < 0, -1.0, 1.0)
        w[n] = (q * s).to(dev)
    w["s"] = torch.randn(D, D, generator=torch.Generator().manual_seed(_SEED + 10000)).to(dev)
    w["key_cent"], w["value_cent"] = cent["key"].to(dev), cent["value"].to(dev)
    st["weights"] = w
    st["q"] = torch.randn(B, T, Hq, D, device=dev, generator=g).to(_DTYPES[case["dtype"]]).transpose(1, 2)
    st["parents"] = _parents(g, B, T, pads=T > 32)


def _prepare_verify(case, g, st):
    """Peaked target distributions over the vocabulary, a draft model near them, drafted tokens."""
    B, T, V, dev = case["B"], case["T"], case["V"], g.device
    dt = _DTYPES[case["dtype"]]
    logits = 2.5 * torch.randn(B, T, V, device=dev, generator=g)
    near = logits[:, :max(1, T - 1)] + 0.7 * torch.randn(B, max(1, T - 1), V, device=dev, generator=g)
    st["target"] = torch.softmax(logits, -1).to(dt)
    st["uniforms"] = torch.rand(B, T, device=dev, generator=g)
    tokens = torch.randint(0, V, (B, T), device=dev, generator=g)
    if case["tree"]:
        # candidates: the draft model's best tokens behind the parent, siblings in falling order
        st["parents"] = par = _parents(g, B, T, pads=T > 8)
        best = near.topk(min(8, V), -1).indices
        i = torch.arange(T, device=dev)
        rank = ((par[:, :, None] == par[:, None, :]) & (i[None, None, :] < i[None, :, None])).sum(-1).clamp(max=7)
        row = par.clamp(min=0, max=max(0, T - 2)).long()
        tokens[:, 1:] = best[torch.arange(B, device=dev)[:, None], row, rank][:, 1:]
        st["draft"] = None
    else:
        q = torch.softmax(near, -1)
        if T > 1:
            tokens[:, 1:] = torch.multinomial(q.reshape(B * (T - 1), V), 1, generator=g).reshape(B, T - 1)
        st["parents"], st["draft"] = None, q[:, :T - 1].to(dt).contiguous()
    st["tokens"] = tokens


def _handles(st):
    """What a program that serves with the framework holds: a pool of pages, a layer's compressors."""
    _import()
    from turboquant_pytorch import PagePool
    from turboquant_pytorch.compressors import TurboQuantCompressorMSE, TurboQuantCompressorV2

    if "planes" in st:
        st["pool"] = PagePool.over(**st["planes"])
    if "weights" in st:
        w, D, bits = st["weights"], st["case"]["D"], st["case"]["bits"]
        kc = TurboQuantCompressorV2(D, bits, seed=_SEED, device="cuda")
        vc = TurboQuantCompressorMSE(D, bits, seed=_SEED + 10000, device="cuda")
        kc.Pi, kc.S, kc.centroids = w["pi"], w["s"], w["key_cent"]
        vc.Pi, vc.centroids = w["pi_v"], w["value_cent"]
        st["kc"], st["vc"] = kc, vc


def _import():
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    pkg = os.path.join(root, "transformers-turboquant_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)


# ------------------------------------------------------------------ one pass
def run(st: dict):
    if own:
        return _run_own(st)
    return {"attend": _plain_attend, "write": _plain_write, "read": _plain_read, "copy": _plain_copy,
            "keep": _plain_keep, "verify": _plain_verify}[st["kind"]](st)


def _run_own(st):
    from turboquant_pytorch import tree_attention, verify_drafts

    kind, case = st["kind"], st["case"]
    if kind == "attend":
        return {"out": tree_attention(st["q"], st["kc"], st["vc"], st["pool"], 0, st["table"], st["lengths"],
                                      st["parents"])}
    if kind == "verify":
        path, count, token = verify_drafts(st["tokens"], st["target"], st["uniforms"], parents=st["parents"],
                                           draft_probs=st["draft"])
        return {"path": path, "count": count, "next": token}
    pool = st["pool"]
    if kind == "write":
        n, shape = st["new"], (case["B"], case["Hkv"], case["S"], case["D"])
        pool.write(0, {"packed_key_indices": n["kcodes"], "packed_qjl_signs": n["ksigns"], "residual_norm": n["krn"],
                       "vec_norms": n["kvn"], "shape": shape},
                   {"packed_indices": n["vcodes"], "vec_norms": n["vvn"], "shape": shape}, st["table"], st["lengths"])
        return dict(st["planes"])
    if kind == "read":
        k, v = pool.read(0, st["table"], st["lengths"], case["S"])
        return {"kcodes": k["packed_key_indices"], "ksigns": k["packed_qjl_signs"], "krn": k["residual_norm"],
                "kvn": k["vec_norms"], "vcodes": v["packed_indices"], "vvn": v["vec_norms"]}
    if kind == "copy":
        pool.copy(st["src"], st["dst"])
        return dict(st["planes"])
    lengths = pool.keep(st["table"], st["lengths"], st["path"], st["count"])
    return {**st["planes"], "lengths": lengths}


def _unpack(rows, D, b):
    at = b * torch.arange(D, device=rows.device)
    byte, off = at // 8, (at % 8).to(torch.int32)
    wide = torch.nn.functional.pad(rows, (0, 1)).to(torch.int32)
    both = wide[..., byte] | (wide[..., byte + 1] << 8)
    return (both >> off) & ((1 << b) - 1)


def _paged(plane, table):
    """A plane's rows [pages, H, P, ...] in the order of each sequence's positions: [B, H, W P, ...]."""
    x = plane[table.clamp(min=0).long()].transpose(1, 2)
    return x.reshape(*x.shape[:2], x.shape[2] * x.shape[3], *x.shape[4:])


def _ancestors(par):
    """[B, T, T]: column t is row i's ancestor, or i itself; rows of nodes without a place are empty."""
    B, T = par.shape
    i = torch.arange(T, device=par.device)
    placed = (par >= -1) & (par < i)
    step = (placed & (par >= 0))[:, :, None] & (par[:, :, None] == i)
    eye = torch.eye(T, device=par.device, dtype=torch.float64)
    return (torch.matrix_power(eye + step.double(), max(1, T)) > 0) & placed[:, :, None] & placed[:, None, :]


def _plain_attend(st):
    case, w, pl = st["case"], st["weights"], {n: t[0] for n, t in st["planes"].items()}
    B, Hq, H, D, T, bits = (case[k] for k in ("B", "Hq", "Hkv", "D", "T", "bits"))
    dev, table, n = st["q"].device, st["table"], st["lengths"].long()
    rot = (st["q"].float() @ w["pi"].T).half().float()
    proj = rot @ (w["s"] @ w["pi"].T).half().float().T
    rot, proj = rot.reshape(B, H, -1, D), proj.reshape(B, H, -1, D)
    N = table.shape[1] * case["page"]
    pos = torch.arange(N, device=dev)
    keys = w["key_cent"].half().float()[_unpack(_paged(pl["kcodes"], table), D, bits - 1)]
    s = (rot @ keys.transpose(2, 3)) * _paged(pl["kvn"], table).float()[:, :, None]
    del keys
    signs = 2.0 * _unpack(_paged(pl["ksigns"], table), D, 1).float() - 1.0
    coeff = math.sqrt(math.pi / 2) / D
    s = s + coeff * (proj @ signs.transpose(2, 3)) * _paged(pl["krn"], table).float()[:, :, None]
    del signs
    anc = _ancestors(st["parents"])
    t = pos[None, :] - n[:, None]  # [B, N]: which drafted token a position holds
    drafted = anc.gather(2, t.clamp(0, T - 1)[:, None, :].expand(B, T, N))
    seen = torch.where((t < 0)[:, None], anc.any(2, keepdim=True), drafted & (t < T)[:, None])  # [B, T, N]
    seen = seen[:, None, None].expand(B, H, Hq // H, T, N).reshape(B, H, -1, N)
    s = torch.where(seen, s / math.sqrt(D), -math.inf)
    top = s.amax(-1, keepdim=True)
    e = torch.where(seen, torch.exp(s - torch.where(top == -math.inf, 0.0, top)), 0.0)
    total = e.sum(-1, keepdim=True)
    p = e / torch.where(total == 0, 1.0, total)
    live = (t < T)[:, None, :, None]
    vals = w["value_cent"][_unpack(_paged(pl["vcodes"], table), D, bits)]
    vals = torch.where(live, vals * _paged(pl["vvn"], table).float()[..., None], 0.0)
    out = (p @ vals) @ w["pi_v"]
    return {"out": out.reshape(B, Hq, T, D).transpose(1, 2).to(st["q"].dtype).contiguous()}


def _plain_write(st):
    case, P = st["case"], st["case"]["page"]
    pos = st["lengths"].long()[:, None] + torch.arange(case["S"], device=st["table"].device)
    page, row = st["table"].long().gather(1, pos // P), pos % P
    return {n: _put(t, page, row, st["new"][n]) for n, t in st["planes"].items()}


def _put(plane, page, row, new):
    plane[0][page, :, row] = new.transpose(1, 2)
    return plane


def _plain_read(st):
    case, table = st["case"], st["table"]
    kept = torch.arange(case["S"], device=table.device)[None, :] < st["lengths"][:, None]
    return {n: _cut(_paged(t[0], table)[:, :, :case["S"]], kept) for n, t in st["planes"].items()}


def _cut(rows, kept):
    kept = kept[:, None] if rows.dim() == 3 else kept[:, None, :, None]
    return torch.where(kept, rows, torch.zeros((), dtype=rows.dtype, device=rows.device))


def _plain_copy(st):
    src, dst = st["src"].long(), st["dst"].long()
    return {n: t.index_copy_(1, dst, t.index_select(1, src)) for n, t in st["planes"].items()}


def _plain_keep(st):
    P, table, n = st["case"]["page"], st["table"].long(), st["lengths"].long()[:, None]
    i = torch.arange(st["case"]["T"], device=table.device)
    old = n + torch.where(i < st["count"][:, None], st["path"].long(), i)
    new = (n + i).expand_as(old)
    where = [x for pos in (old, new) for x in (table.gather(1, pos // P), pos % P)]
    out = {name: _move(t, *where) for name, t in st["planes"].items()}
    return {**out, "lengths": st["lengths"] + st["count"]}


def _move(plane, page, row, to_page, to_row):
    plane[:, to_page, :, to_row] = plane[:, page, :, row]
    return plane


def _plain_verify(st):
    case = st["case"]
    B, T, V = case["B"], case["T"], case["V"]
    tok, u = st["tokens"], st["uniforms"].double()
    dev = tok.device
    i = torch.arange(T, device=dev)
    par = st["parents"] if case["tree"] else (i - 1).to(torch.int32).expand(B, T)
    b = torch.arange(B, device=dev)
    above = par.clamp(min=0).long()
    p = st["target"][b[:, None], above, tok].double()
    inner = (par >= 0) & (par < i)
    if case["tree"]:
        earlier = (par[:, :, None] == par[:, None, :]) & (i[None, None, :] < i[None, :, None])
        bar = u * (1.0 - (earlier * p[:, None, :]).sum(-1))
    else:
        earlier = torch.zeros(B, T, T, dtype=torch.bool, device=dev)
        q = st["draft"][b[:, None], i[:T - 1], tok[:, 1:]].double()
        bar = torch.cat([u[:, :1], u[:, 1:] * q], 1)
    good = inner & (bar < p)
    first = good & ~(earlier & good[:, None, :]).any(-1)
    first[:, 0] = True
    anc = _ancestors(torch.where(i == 0, -1, par))
    rooted = anc[:, :, 0]
    taken = rooted & (~anc | first[:, None, :]).all(-1)
    count = taken.sum(1).to(torch.int32)
    path = torch.where(taken, i, T).sort(1).values
    stop = path.gather(1, (count.long() - 1)[:, None])[:, 0]
    path = torch.where(path < T, path, -1).to(torch.int32)
    wt = st["target"][b, stop].double()
    if case["tree"]:
        child = inner & (par == stop[:, None])
        wt = wt.scatter(1, torch.where(child, tok, tok[:, :1]),
                        torch.where(child, 0.0, wt.gather(1, tok[:, :1]).expand(B, T)))
        spoken = (child & (tok == tok[:, :1])).any(1)  # the stand-in is itself a rejected token
        wt[b, tok[:, 0]] = torch.where(spoken, 0.0, wt[b, tok[:, 0]])
    elif T > 1:
        low = st["draft"][b, stop.clamp(max=T - 2)].double()
        wt = torch.where((stop < T - 1)[:, None], (wt - low).clamp(min=0), wt)
    total = wt.cumsum(1)
    over = (total > u[:, :1] * total[:, -1:]) & (wt > 0)
    return {"path": path, "count": count, "next": over.to(torch.int8).argmax(1)}


# ------------------------------------------------------------------ the same in 64 bits
def exact(case: dict, seed: int):
    st = prepare(case, seed)
    if case["kind"] == "attend":
        return {"out": _exact_attend(st)}
    if case["kind"] == "verify":
        return _exact_verify(st)
    return None  # bytes that move: nothing is computed


def _exact_attend(st):
    """One sequence and kv head at a time: gather its rows, decode them, attend in float64."""
    case, w, pl = st["case"], st["weights"], st["planes"]
    B, Hq, H, D, T, bits, P = (case[k] for k in ("B", "Hq", "Hkv", "D", "T", "bits", "page"))
    G, dev = Hq // H, st["q"].device
    pi, pi_v = w["pi"].double(), w["pi_v"].double()
    s_eff = (w["s"] @ w["pi"].T).half().double()
    ck, cv = w["key_cent"].half().double(), w["value_cent"].double()
    out = torch.zeros(B, T, Hq, D, dtype=torch.float64, device=dev)
    par, table, lens = st["parents"].tolist(), st["table"].tolist(), st["lengths"].tolist()
    bit = lambda rows, b: ((rows[..., None] >> torch.arange(8, device=dev)) & 1).flatten(-2).reshape(  # noqa: E731
        *rows.shape[:-1], D, b)

    def code(rows, b):
        return (bit(rows, b) * (2 ** torch.arange(b, device=dev))).sum(-1)

    for b in range(B):
        N = lens[b] + T
        pages = torch.tensor(table[b][:(N + P - 1) // P], device=dev)
        sees = torch.zeros(T, N, dtype=torch.bool, device=dev)
        for i in range(T):
            if -1 <= par[b][i] < i:
                sees[i, :lens[b]] = True
                if par[b][i] >= 0:
                    sees[i, lens[b]:] = sees[par[b][i], lens[b]:]
                sees[i, lens[b] + i] = True
        for h in range(H):
            row = {n: t[0, pages, h].flatten(0, 1)[:N] for n, t in pl.items()}
            q = (st["q"][b, h * G:(h + 1) * G].double() @ pi.T).half().double()
            mse = ck[code(row["kcodes"], bits - 1).long()] * row["kvn"].double()[:, None]
            sgn = (2.0 * code(row["ksigns"], 1).double() - 1.0) * row["krn"].double()[:, None]
            s = q @ mse.T + math.sqrt(math.pi / 2) / D * ((q @ s_eff.T) @ sgn.T)
            s = (s / math.sqrt(D)).masked_fill(~sees, -math.inf)
            p = torch.nan_to_num(torch.softmax(s, -1))
            val = cv[code(row["vcodes"], bits).long()] * row["vvn"].double()[:, None]
            out[b, :, h * G:(h + 1) * G] = ((p @ val) @ pi_v).transpose(0, 1)
    return out


def _exact_verify(st):
    """Walked node by node."""
    case = st["case"]
    B, T, tree = case["B"], case["T"], case["tree"]
    tok, u = st["tokens"].tolist(), st["uniforms"].double().tolist()
    par = st["parents"].tolist() if tree else [[i - 1 for i in range(T)]] * B
    paths, counts, nexts = [], [], []
    for b in range(B):
        at, path, go = 0, [0], True
        while go:
            go, left = False, 1.0
            p = st["target"][b, at].double()
            w = p.clone()
            for i in range(at + 1, T):
                if par[b][i] != at:
                    continue
                x = tok[b][i]
                if tree:
                    if u[b][i] * left < p[x].item():
                        at, go = i, True
                        break
                    left -= p[x].item()
                    w[x] = 0.0
                else:
                    q = st["draft"][b, at].double()
                    if u[b][i] * q[x].item() < p[x].item():
                        at, go = i, True
                        break
                    w = (p - q).clamp(min=0)
            if go:
                path.append(at)
        c = w.cumsum(0)
        paths.append(path + [-1] * (T - len(path)))
        counts.append(len(path))
        nexts.append(int(torch.nonzero((c > u[b][0] * c[-1]) & (w > 0))[0]))
    dev = st["tokens"].device
    return {"path": torch.tensor(paths, dtype=torch.int32, device=dev),
            "count": torch.tensor(counts, dtype=torch.int32, device=dev),
            "next": torch.tensor(nexts, dtype=torch.int64, device=dev)}


# ------------------------------------------------------------------ what a pass cannot do without
def work(case: dict) -> dict:
    kind, B = case["kind"], case["B"]
    if kind == "verify":
        # tokens, uniforms and their probabilities; one row of the target's, one of the draft's, per sequence
        es, T, V = (4 if case["dtype"] == "f32" else 2), case["T"], case["V"]
        rows = 1 if case["tree"] or T == 1 else 2
        return {"bytes": B * (rows * V * es + T * (12 + 2 * es)), "flops": 3 * B * V}
    H, D = case["Hkv"], case["D"]
    rec = _record(case)[1]
    if kind == "attend":
        Hq, T = case["Hq"], case["T"]
        n = sum(_lengths(case))
        q = B * Hq * T * D
        flops = 3 * 2 * D * Hq * T * (n + B * T) + 3 * 2 * D * q
        return {"bytes": 2 * 2 * q + H * (n + B * T) * rec, "flops": flops}
    if kind in ("write", "read"):
        return {"bytes": 2 * H * rec * (B * case["S"] if kind == "write" else sum(_lengths(case))), "flops": 0}
    if kind == "copy":
        return {"bytes": 2 * B * H * case["page"] * rec * case["layers"], "flops": 0}
    # keep: on average a quarter of a tree's nodes is on its accepted path
    return {"bytes": 2 * B * H * max(1, case["T"] // 4) * rec * case["layers"], "flops": 0}
