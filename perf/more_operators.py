"""Performance cases of the operators that continue one prompt several times over a paged compressed KV cache.

  attend   attention of the new tokens (T of them, a tree; T = 1 is a decoding step) of sequences that were forked from
           a few prompts: the pages of a prompt are the same for all of its continuations, each has pages of its own behind
  sample   the next token of every sequence from its logits and a given uniform, by temperature, top-k, top-p and min-p
  probs    the distribution that such a draw has, written out, for the verification of drafted tokens

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


# ------------------------------------------------------------------ cases
def listed() -> list[dict]:
    return [
        # four answers to one short prompt, a GPT-2-shaped layer
        _attend("attend_d64_4_of_1k", "4", "960", 200, 12, 12, 64, 1, 3, 64),
        # sixteen samples of a long document's summary, a Llama-3-8B-shaped layer
        _attend("attend_d128_16_of_32k", "16", "32000", 700, 32, 8, 128, 1, 3, 64),
        # speculation in eight continuations of one context: trees of 8 drafted tokens
        _attend("attend_d128_8x8_of_16k", "8", "16384", 500, 32, 8, 128, 8, 3, 128),
        # 64 samples under 8 query heads per kv head (Qwen2.5-3B shape), float16
        _attend("attend_d128_64_of_8k_gqa8", "64", "8192", 1000, 16, 2, 128, 1, 4, 64, dtype="f16"),
        # a served batch: two prompts, continued 5 and 11 times, long answers, one sequence for itself
        _attend("attend_d128_three_groups", "5 11 1", "4096 12032 0", 4000, 32, 8, 128, 1, 3, 64),
        # one sequence, GPT-2's vocabulary
        _sample("sample_b1_50257", 1, 50257, "f32", t=0.8, k=50, p=1.0, m=0.0),
        # a batch under nucleus sampling, a Llama-3-sized vocabulary
        _sample("sample_b64_128256", 64, 128256, "f32", t=0.7, k=0, p=0.9, m=0.0),
        # requests with settings of their own, some of them under a grammar that bans most tokens
        _sample("sample_b16_151936_mixed", 16, 151936, "bf16", t=1.0, k=40, p=0.95, m=0.02, rows=True, banned=0.9),
        # many sequences, no order of the tokens needed
        _sample("sample_b256_128256_min_p", 256, 128256, "bf16", t=1.2, k=0, p=1.0, m=0.05),
        # the distributions that verify one sequence's chain of 4 drafted tokens
        _probs("probs_b1_t5_50257", 5, 50257, "f32", t=0.8, k=50, p=0.95, m=0.0),
        # the same for 16 trees of 32, a Qwen2.5-sized vocabulary
        _probs("probs_b16_t32_151936", 512, 151936, "bf16", t=0.7, k=0, p=0.9, m=0.0),
    ]


def _named(case):
    return case if case["name"] else {k: v for k, v in case.items() if k != "name"}


def _attend(name, sizes, shared, new, Hq, Hkv, D, T, bits, page, dtype="bf16"):
    return _named(dict(name=name, kind="attend", sizes=sizes, shared=shared, new=new, Hq=Hq, Hkv=Hkv, D=D, T=T, bits=bits,
                       page=page, dtype=dtype))


def _draw_case(name, kind, N, V, dtype, t, k, p, m, rows, banned):
    return _named(dict(name=name, kind=kind, N=N, V=V, dtype=dtype, t=t, k=k, p=p, m=m, rows=rows, banned=banned))


def _sample(name, N, V, dtype, t, k, p, m, rows=False, banned=0.0):
    return _draw_case(name, "sample", N, V, dtype, t, k, p, m, rows, banned)


def _probs(name, N, V, dtype, t, k, p, m, rows=False, banned=0.0):
    return _draw_case(name, "probs", N, V, dtype, t, k, p, m, rows, banned)


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng) -> dict:
    kind = rng.choice(["attend", "attend", "sample", "probs"])
    if kind == "attend":
        Hq, Hkv = rng.choice([(12, 12), (32, 8), (16, 2), (32, 32), (14, 2), (28, 4), (64, 8)])
        D, bits, page = rng.choice([64, 128, 128]), rng.choice([2, 3, 3, 4]), rng.choice([32, 64, 64, 128, 256])
        T, new = rng.choice([1, 1, 1, 2, 5, 8, 16]), _log_int(rng, 1, 4000)
        sizes = [_log_int(rng, 1, 32) for _ in range(rng.choice([1, 1, 2, 3]))]
        shared = [rng.randrange(1, max(2, _log_int(rng, page, 32000) // page)) * page for _ in sizes]
        while sum(s * (n + new) for s, n in zip(sizes, shared)) * Hkv * D * max(1, Hq * T // (8 * Hkv)) > 16 * 32700 * 8 * 128:
            new = (new + 1) // 2
            shared = [max(page, n // page // 2 * page) for n in shared]
            sizes = [(s + 1) // 2 for s in sizes] if max(shared) == page else sizes
        sizes, shared = (" ".join(map(str, x)) for x in (sizes, shared))
        return _attend(None, sizes, shared, new, Hq, Hkv, D, T, bits, page, rng.choice(["bf16", "bf16", "f16"]))
    N, V = _log_int(rng, 1, 256 if kind == "sample" else 512), _log_int(rng, 1000, 151936)
    dtype = rng.choice(["f32", "bf16", "f16"])
    while N * V * (4 if dtype == "f32" else 2) > 256 * 128256 * 2:
        N = (N + 1) // 2
    return _draw_case(None, kind, N, V, dtype, t=round(rng.uniform(0.4, 1.5), 2), k=rng.choice([0, 0, 1, 20, 50, 1000]),
                      p=rng.choice([1.0, 0.5, 0.9, 0.99]), m=rng.choice([0.0, 0.0, 0.01, 0.1]), rows=rng.random() < 0.4,
                      banned=rng.choice([0.0, 0.0, 0.5, 0.99]))


def _groups_of(case) -> tuple[list[int], list[int]]:
    """Sequences of each group, and how many positions they share."""
    return tuple([int(x) for x in case[k].split()] for k in ("sizes", "shared"))


def _rows_of(case) -> list[tuple[int, int]]:
    """(shared, cached) positions of every sequence; the last one has `new` behind the shared ones, the others a
    share of them down to a quarter."""
    shared = [n for s, n in zip(*_groups_of(case)) for _ in range(s)]
    B, new = len(shared), case["new"]
    return [(n, n + (new if B == 1 else new - 3 * new * (B - 1 - b) // (4 * (B - 1)))) for b, n in enumerate(shared)]


# ------------------------------------------------------------------ inputs
def prepare(case: dict, seed: int) -> dict:
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    st = {"case": case, "kind": case["kind"]}
    if case["kind"] == "attend":
        _prepare_attend(case, g, st)
    else:
        _prepare_logits(case, g, st)
    return st


@functools.lru_cache(maxsize=None)
def _codebook(D, bits):
    """Lloyd-Max centroids of N(0, 1/D): the centre of mass of each cell, iterated."""
    c = torch.linspace(-2.0, 2.0, 2 ** bits, dtype=torch.float64)
    edge = torch.tensor([40.0], dtype=torch.float64)
    for _ in range(400):
        e = torch.cat([-edge, (c[1:] + c[:-1]) / 2, edge])
        pdf, cdf = torch.exp(-e * e / 2) / math.sqrt(2 * math.pi), 0.5 * (1 + torch.erf(e / math.sqrt(2)))
        c = (pdf[:-1] - pdf[1:]) / (cdf[1:] - cdf[:-1])
    return (c / math.sqrt(D)).float()


def _codes(g, rows, D, b, cent):
    """Packed codes of Gaussian coordinates, the first code in a row's lowest bits, 2^18 rows at a time."""
    dev, parts = g.device, []
    bounds = ((cent[1:] + cent[:-1]) / 2).to(dev)
    for at in range(0, rows, 1 << 18):
        y = torch.randn(min(1 << 18, rows - at), D, device=dev, generator=g) / math.sqrt(D)
        code = torch.bucketize(y, bounds).reshape(-1, D // 8, 8).to(torch.int32)
        word = (code << (b * torch.arange(8, device=dev, dtype=torch.int32))).sum(-1, dtype=torch.int32)
        byte = (word.unsqueeze(-1) >> (8 * torch.arange(b, device=dev, dtype=torch.int32))) & 255
        parts.append(byte.to(torch.uint8).reshape(-1, D // 8 * b))
    return torch.cat(parts)


def _prepare_attend(case, g, st):
    """Pages of compressed rows in a pool, tables in which a prompt's pages stand in every row of its group, queries, trees."""
    D, H, Hq, T, P, bits, dev = (*(case[k] for k in ("D", "Hkv", "Hq", "T", "page", "bits")), g.device)
    rows = _rows_of(case)
    B = len(rows)
    need = [(n + T + P - 1) // P for _, n in rows]
    sizes, shared = _groups_of(case)
    heads = [n // P for n in shared]  # pages of each prompt
    pages = sum(heads) + sum(k - s // P for k, (s, _) in zip(need, rows)) + 2
    order = torch.randperm(pages, device=dev, generator=g).to(torch.int32)
    table = torch.full((B, max(need)), -1, dtype=torch.int32, device=dev)
    at = b0 = 0
    for size, head in zip(sizes, heads):
        prompt, at = order[at:at + head], at + head
        for b in range(b0, b0 + size):
            table[b, :head] = prompt
            table[b, head:need[b]] = order[at:at + need[b] - head]
            at += need[b] - head
        b0 += size
    st["table"], st["lengths"] = table, torch.tensor([n for _, n in rows], dtype=torch.int32, device=dev)

    cent, n = {"key": _codebook(D, bits - 1), "value": _codebook(D, bits)}, pages * H * P
    norms = math.sqrt(D) * torch.exp(0.25 * torch.randn(n, device=dev, generator=g))
    planes = {"kcodes": _codes(g, n, D, bits - 1, cent["key"]),
              "ksigns": torch.randint(0, 256, (n, D // 8), device=dev, generator=g, dtype=torch.uint8),
              "krn": ((0.6, 0.34, 0.19)[bits - 2] * norms).half(), "kvn": norms.half(),
              "vcodes": _codes(g, n, D, bits, cent["value"]),
              "vvn": (math.sqrt(D) * torch.exp(0.1 * torch.randn(n, device=dev, generator=g))).half()}
    st["planes"] = {name: t.reshape(1, pages, H, P, *t.shape[1:]) for name, t in planes.items()}

    w = {"key_cent": cent["key"].to(dev), "value_cent": cent["value"].to(dev)}
    for name, seed in (("pi", _SEED), ("pi_v", _SEED + 10000)):
        q, r = torch.linalg.qr(torch.randn(D, D, generator=torch.Generator().manual_seed(seed)))
        w[name] = (q * torch.where(torch.diagonal(r) < 0, -1.0, 1.0)).to(dev)
    w["s"] = torch.randn(D, D, generator=torch.Generator().manual_seed(_SEED + 10000)).to(dev)
    st["weights"] = w
    st["q"] = torch.randn(B, T, Hq, D, device=dev, generator=g).to(_DTYPES[case["dtype"]]).transpose(1, 2)
    # trees in index order: a node's parent is one of the 7 nodes before it
    back = torch.randint(1, 8, (B, T), device=dev, generator=g)
    parents = (torch.arange(T, device=dev) - back).clamp(min=0)
    parents[:, 0] = -1
    st["parents"] = parents.to(torch.int32)
    if own:
        _handles(st)


def _prepare_logits(case, g, st):
    """Logits with a bulk and a few tokens that the text asks for, some banned (-inf); uniforms; settings."""
    N, V, dev = case["N"], case["V"], g.device
    logits = 2.0 * torch.randn(N, V, device=dev, generator=g)
    asked = torch.randint(0, V, (N, min(V, 30)), device=dev, generator=g)
    logits.scatter_add_(1, asked, 6.0 + 5.0 * torch.rand(asked.shape, device=dev, generator=g))
    if case["banned"]:
        ban = torch.rand(N, V, device=dev, generator=g) < case["banned"]
        ban[:, 7] = False
        logits.masked_fill_(ban, -math.inf)
    st["logits"] = logits.to(_DTYPES[case["dtype"]])
    if case["kind"] == "sample":
        st["uniforms"] = torch.rand(N, device=dev, generator=g)
    st["set"] = (case["t"], case["k"], case["p"], case["m"])
    if case["rows"]:  # requests' own: some greedy, some without a filter
        r = torch.rand(4, N, device=dev, generator=g)
        t = torch.where(r[0] < 0.15, 0.0, case["t"] * (0.5 + r[0]))
        k = torch.where(r[1] < 0.3, 0.0, case["k"] * 2 * r[1]).to(torch.int32)
        p = torch.where(r[2] < 0.3, 1.0, case["p"] * (0.5 + 0.5 * r[2]))
        m = torch.where(r[3] < 0.3, 0.0, case["m"] * 2 * r[3])
        st["set"] = (t, k, p, m)


def _handles(st):
    """What a program that serves with the framework holds: a pool of pages, a layer's compressors, the groups."""
    _import()
    from turboquant_pytorch import PagePool, prefix_groups
    from turboquant_pytorch.compressors import TurboQuantCompressorMSE, TurboQuantCompressorV2

    case, w = st["case"], st["weights"]
    st["pool"] = PagePool.over(**st["planes"])
    kc = TurboQuantCompressorV2(case["D"], case["bits"], seed=_SEED, device="cuda")
    vc = TurboQuantCompressorMSE(case["D"], case["bits"], seed=_SEED + 10000, device="cuda")
    kc.Pi, kc.S, kc.centroids = w["pi"], w["s"], w["key_cent"]
    vc.Pi, vc.centroids = w["pi_v"], w["value_cent"]
    st["kc"], st["vc"] = kc, vc
    st["groups"] = prefix_groups(*_groups_of(case), device="cuda")


def _import():
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    pkg = os.path.join(root, "transformers-turboquant_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)


# ------------------------------------------------------------------ one pass
def run(st: dict):
    if own:
        return _run_own(st)
    if st["kind"] == "attend":
        return {"out": _plain_attend(st)}
    probs = _plain_probs(st)
    return {"token": _plain_pick(probs, st["uniforms"])} if st["kind"] == "sample" else {"probs": probs.float()}


def _run_own(st):
    _import()
    from turboquant_pytorch import filter_probs, prefix_attention, sample_tokens

    if st["kind"] == "attend":
        return {"out": prefix_attention(st["q"], st["kc"], st["vc"], st["pool"], 0, st["table"], st["lengths"], st["groups"],
                                        st["parents"])}
    t, k, p, m = st["set"]
    if st["kind"] == "sample":
        return {"token": sample_tokens(st["logits"], st["uniforms"], temperature=t, top_k=k, top_p=p, min_p=m)}
    return {"probs": filter_probs(st["logits"], temperature=t, top_k=k, top_p=p, min_p=m)}


def _unpack(rows, D, b):
    at = b * torch.arange(D, device=rows.device)
    byte, off = at // 8, (at % 8).to(torch.int32)
    wide = torch.nn.functional.pad(rows, (0, 1)).to(torch.int32)
    return ((wide[..., byte] | (wide[..., byte + 1] << 8)) >> off) & ((1 << b) - 1)


def _paged(plane, table):
    """A plane's rows [pages, H, P, ...] in the order of each sequence's positions: [B, H, W P, ...]."""
    x = plane[table.clamp(min=0).long()].transpose(1, 2)
    return x.reshape(*x.shape[:2], x.shape[2] * x.shape[3], *x.shape[4:])


def _plain_attend(st):
    """Every sequence over its whole table; the mask decides what a node sees."""
    case, w, pl = st["case"], st["weights"], {n: t[0] for n, t in st["planes"].items()}
    Hq, H, D, T, bits = (case[k] for k in ("Hq", "Hkv", "D", "T", "bits"))
    dev, table, n, par = st["q"].device, st["table"], st["lengths"].long(), st["parents"]
    B = table.shape[0]
    rot = (st["q"].float() @ w["pi"].T).half().float()
    proj = (rot @ (w["s"] @ w["pi"].T).half().float().T).reshape(B, H, -1, D)
    rot = rot.reshape(B, H, -1, D)
    keys = w["key_cent"].half().float()[_unpack(_paged(pl["kcodes"], table), D, bits - 1)]
    s = (rot @ keys.transpose(2, 3)) * _paged(pl["kvn"], table).float()[:, :, None]
    signs = 2.0 * _unpack(_paged(pl["ksigns"], table), D, 1).float() - 1.0
    keys = None
    s = s + math.sqrt(math.pi / 2) / D * (proj @ signs.transpose(2, 3)) * _paged(pl["krn"], table).float()[:, :, None]
    signs = None
    i = torch.arange(T, device=dev)
    up = ((par[:, :, None] == i) & (par >= 0)[:, :, None]).double() + torch.eye(T, dtype=torch.float64, device=dev)
    anc = torch.matrix_power(up, max(1, T)) > 0  # [B, T, T]: row i's ancestors, and i itself
    N = s.shape[-1]
    t = torch.arange(N, device=dev)[None, :] - n[:, None]  # which new token a position holds
    seen = anc.gather(2, t.clamp(0, T - 1)[:, None, :].expand(B, T, N)) & (t < T)[:, None] | (t < 0)[:, None]
    seen = seen[:, None, None].expand(B, H, Hq // H, T, N).reshape(B, H, -1, N)
    s = torch.where(seen, s / math.sqrt(D), -math.inf)
    e = torch.exp(s - s.amax(-1, keepdim=True))
    vals = w["value_cent"][_unpack(_paged(pl["vcodes"], table), D, bits)] * _paged(pl["vvn"], table).float()[..., None]
    out = ((e / e.sum(-1, keepdim=True)) @ vals) @ w["pi_v"]
    return out.reshape(B, Hq, T, D).transpose(1, 2).to(st["q"].dtype).contiguous()


def _column(x, N, dev):
    return x.double()[:, None] if isinstance(x, torch.Tensor) else torch.full((N, 1), float(x), dtype=torch.float64, device=dev)


def _plain_probs(st):
    """The filtered distributions: in 64 bits, since what is kept and drawn lies next to a border."""
    N, V, dev = st["case"]["N"], st["case"]["V"], st["logits"].device
    t, k, p, m = (_column(x, N, dev) for x in st["set"])
    t, k = torch.where(t == 0, 1.0, t), torch.where(t == 0, 1.0, torch.where(k <= 0, float(V), k))
    rank, order = torch.sort(st["logits"].float(), dim=-1, descending=True, stable=True)
    w = torch.exp((rank.double() - rank[:, :1].double()) / t)
    rank = None
    kept = torch.arange(V, device=dev)[None] < k
    w = torch.where(kept, w, 0.0)
    upto = w.cumsum(-1)
    kept &= (upto - w < p * upto[:, -1:]) | (p >= 1.0)
    kept[:, 0] = True
    upto = None
    w = torch.where(kept & (w >= m), w, 0.0)
    return torch.zeros_like(w).scatter_(1, order, w / w.sum(-1, keepdim=True))


def _plain_pick(probs, uniforms):
    upto = probs.cumsum(-1)
    return ((upto > uniforms.double()[:, None] * upto[:, -1:]) & (probs > 0)).to(torch.int8).argmax(-1)


# ------------------------------------------------------------------ the same in 64 bits
def exact(case: dict, seed: int):
    st = prepare(case, seed)
    if case["kind"] == "attend":
        return {"out": _exact_attend(st)}
    rows = [_exact_row(st, i) for i in range(case["N"])]
    if case["kind"] == "probs":
        return {"probs": torch.stack(rows)}
    u = st["uniforms"].double().tolist()
    tokens = []
    for i, q in enumerate(rows):
        at = torch.nonzero(q)[:, 0]  # the kept tokens, in index order
        c = q[at].cumsum(0)
        tokens.append(int(at[torch.nonzero(c > u[i] * c[-1])[0, 0]]))
    return {"token": torch.tensor(tokens, dtype=torch.int64, device=st["logits"].device)}


def _exact_row(st, i):
    """One row, value by value: the distinct logits in falling order, how often each occurs, and of the last one that is
    kept, how many."""
    t, k, p, m = (x[i].item() if isinstance(x, torch.Tensor) else x for x in st["set"])
    row = st["logits"][i].double()
    if t == 0:
        t, k = 1.0, 1
    values, counts = torch.unique(row, return_counts=True)
    values, counts = values.flip(0), counts.flip(0)
    weight = torch.exp((values - values[0]) / t)
    if k > 0:
        counts = counts.minimum((k - (counts.cumsum(0) - counts)).clamp(min=0))
    if p < 1:
        mass = weight * counts
        upto = mass.cumsum(0)
        goal = p * upto[-1]
        room = torch.ceil((goal - (upto - mass)) / weight.clamp(min=5e-324)).clamp(min=0)
        room[0] = room[0].clamp(min=1)
        counts = torch.where(weight > 0, counts.double().minimum(room), 0.0).long()
    counts = torch.where(weight >= m, counts, 0)
    out = torch.zeros_like(row)
    last = int(torch.nonzero(counts)[-1, 0])
    keep = row > values[last]
    tied = row == values[last]
    keep |= tied & (tied.long().cumsum(0) <= counts[last])
    out[keep] = torch.exp((row[keep] - values[0]) / t)
    return out / out.sum()


def _exact_attend(st):
    """One sequence and kv head at a time: gather its rows, decode them, attend in float64."""
    case, w, pl = st["case"], st["weights"], st["planes"]
    Hq, H, D, T, bits, P = (case[k] for k in ("Hq", "Hkv", "D", "T", "bits", "page"))
    G, dev = Hq // H, st["q"].device
    pi, pi_v = w["pi"].double(), w["pi_v"].double()
    s_eff = (w["s"] @ w["pi"].T).half().double()
    ck, cv = w["key_cent"].half().double(), w["value_cent"].double()
    par, lens = st["parents"].tolist(), st["lengths"].tolist()
    B = len(lens)
    out = torch.zeros(B, T, Hq, D, dtype=torch.float64, device=dev)

    def code(rows, b):
        bit = ((rows[..., None] >> torch.arange(8, device=dev)) & 1).flatten(-2).reshape(*rows.shape[:-1], D, b)
        return (bit * (2 ** torch.arange(b, device=dev))).sum(-1)

    for b in range(B):
        N = lens[b] + T
        pages = st["table"][b, :(N + P - 1) // P].long()
        sees = torch.zeros(T, N, dtype=torch.bool, device=dev)
        for i in range(T):
            sees[i, :lens[b]] = True
            if par[b][i] >= 0:
                sees[i, lens[b]:] = sees[par[b][i], lens[b]:]
            sees[i, lens[b] + i] = True
        for h in range(H):
            row = {name: x[0, pages, h].flatten(0, 1)[:N] for name, x in pl.items()}
            q = (st["q"][b, h * G:(h + 1) * G].double() @ pi.T).half().double()
            mse = ck[code(row["kcodes"], bits - 1).long()] * row["kvn"].double()[:, None]
            sgn = (2.0 * code(row["ksigns"], 1).double() - 1.0) * row["krn"].double()[:, None]
            s = q @ mse.T + math.sqrt(math.pi / 2) / D * ((q @ s_eff.T) @ sgn.T)
            prob = torch.softmax((s / math.sqrt(D)).masked_fill(~sees, -math.inf), -1)
            val = cv[code(row["vcodes"], bits).long()] * row["vvn"].double()[:, None]
            out[b, :, h * G:(h + 1) * G] = ((prob @ val) @ pi_v).transpose(0, 1)
    return out


# ------------------------------------------------------------------ what a pass cannot do without
def work(case: dict) -> dict:
    if case["kind"] != "attend":
        N, V, es = case["N"], case["V"], 4 if case["dtype"] == "f32" else 2
        return {"bytes": N * (V * (es + (4 if case["kind"] == "probs" else 0)) + 12), "flops": 3 * N * V}
    H, D, Hq, T, bits = (case[k] for k in ("Hkv", "D", "Hq", "T", "bits"))
    rows = _rows_of(case)
    record = D * (bits - 1) // 8 + D // 8 + D * bits // 8 + 6
    q = len(rows) * Hq * T * D
    alone = sum(n - s + T for s, n in rows)
    keys = sum(n + T for _, n in rows)
    return {"bytes": 2 * 2 * q + H * record * (sum(_groups_of(case)[1]) + alone), "flops": 3 * 2 * D * Hq * T * keys + 3 * 2 * D * q}
