"""The operators of decoding with drafted tokens, as cases that can be timed and compared.

A model's step may run a tree of tokens that something cheaper has drafted for each request, keep the path that the model
agrees with, and throw the rest away.  A case is a dictionary of plain values; its ``kind`` names the operator:

tree    attention of a tree of drafted tokens over the paged cache (``kernels.paged_attention_tree``): a row sees the
        context (all of it or a window) and, of the drafted tokens, those that its mask names: itself and its ancestors
keep    the drafted tokens that are kept move to neighbouring places of the cache (``kernels.keep_tokens``), in all layers;
        the same call thins out a long context
copy    pages of the cache are copied to other pages (``kernels.copy_pages``), in all layers: a request is forked
score   log probabilities of given tokens, the distribution's entropy and its most likely tokens
        (``kernels.token_log_probs``)

Drafted token i of request r has its keys and values at place context[r] + i of the request.  ``seen`` [rows, words] has a
bit for every drafted token of the row's request: bit j % 32 of word j / 32.

The plain forms work in 32 bits and round once at the end.  The model sizes are those of the benchmark.
"""
from __future__ import annotations

import math
import random
from typing import Dict, List

import torch

own = False

DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
MOST_TREE = 16 * 64 * 32 * 128 * 8242          # multiply-adds of the largest listed attention, half of them
MOST_CACHE = 16 * 8242 * 8 * 128               # numbers of keys of the largest listed cache
MOST_MOVED = 72 * 512 * 16 * 8 * 128           # numbers that the largest listed copy reads
MOST_LOGITS = 2048 * 151936


def listed() -> List[dict]:
    return [
        # one chat on a small model, a short context, eight drafted tokens: the smallest call
        dict(name="tree 1x8 of 300", kind="tree", requests=1, tree=8, shortest=300, longest=300, heads=16, kv_heads=8, dim=128,
             page=16, window=0, chain=False, dtype="bf16"),
        # the benchmark's decode step of eight requests, a tree of 16 for each
        dict(name="tree 8x16 of 2048", kind="tree", requests=8, tree=16, shortest=2048, longest=2048, heads=32, kv_heads=8,
             dim=128, page=16, window=0, chain=False, dtype="bf16"),
        # sixteen requests of every age with long contexts and large trees
        dict(name="tree 16x64 of 16384", kind="tree", requests=16, tree=64, shortest=100, longest=16384, heads=32, kv_heads=8,
             dim=128, page=16, window=0, chain=False, dtype="bf16"),
        # a model of smaller heads with a window, runs of drafted tokens without branches, odd sizes
        dict(name="tree 5x37 of 5003, window", kind="tree", requests=5, tree=37, shortest=700, longest=5003, heads=20, kv_heads=4,
             dim=64, page=32, window=1500, chain=True, dtype="bf16"),
        # the true 32-bit path
        dict(name="tree 2x13 of 777, f32", kind="tree", requests=2, tree=13, shortest=301, longest=777, heads=16, kv_heads=8,
             dim=128, page=16, window=0, chain=False, dtype="f32"),
        # the benchmark's step of eight requests: the path that the model agrees with stays
        dict(name="keep 8x5 of 16", kind="keep", requests=8, kept=5, among=16, first=2048, layers=36, kv_heads=8, dim=128, page=16,
             dtype="bf16"),
        # four long contexts are thinned out
        dict(name="keep 4x1000 of 2000", kind="keep", requests=4, kept=1000, among=2000, first=5, layers=36, kv_heads=8, dim=128,
             page=16, dtype="bf16"),
        # one request of a small model is forked: the copy of its last page
        dict(name="copy 1 page", kind="copy", pairs=1, sources=1, layers=28, kv_heads=8, dim=128, page=16, dtype="bf16"),
        # prompts of 2,048 tokens are copied for four requests
        dict(name="copy 512 pages", kind="copy", pairs=512, sources=512, layers=36, kv_heads=8, dim=128, page=16, dtype="bf16"),
        # one chat that asks for its tokens' log probabilities and five alternatives
        dict(name="score 1x151936 top 5", kind="score", rows=1, vocab=151936, given=1, top=5, unused=0, dtype="f32"),
        # the drafted tokens of the benchmark's step, each with the twenty most likely ones
        dict(name="score 128x151936 top 20", kind="score", rows=128, vocab=151936, given=1, top=20, unused=267, dtype="f32"),
        # the benchmark's prompt of 2,048 tokens is scored
        dict(name="score 2048x151936 top 1", kind="score", rows=2048, vocab=151936, given=1, top=1, unused=267, dtype="f32"),
    ]


def _spread(rng: random.Random, low: int, high: int) -> int:
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(max(low, high))))))))


def draw(rng: random.Random) -> dict:
    kind = rng.choice(["tree", "tree", "tree", "keep", "copy", "score", "score"])
    if kind == "score":
        vocab = _spread(rng, 200, 262144)
        dtype = rng.choice(["f32", "f32", "bf16"])
        return dict(kind=kind, rows=_spread(rng, 1, min(4096, MOST_LOGITS // vocab)), vocab=vocab, given=rng.choice([1, 1, 1, 4]),
                    top=rng.choice([0, 1, 5, 20, 32]), unused=rng.choice([0, 0, rng.randrange(0, vocab // 2)]), dtype=dtype)
    dtype = rng.choice(["bf16", "bf16", "bf16", "f32"])
    heads, kv_heads = rng.choice([(16, 8), (32, 8), (64, 8), (8, 8), (20, 4), (32, 2)])
    dim, page = rng.choice([64, 128, 128, 128]), rng.choice([16, 16, 32, 64])
    if kind == "tree":
        requests, tree = _spread(rng, 1, 64), _spread(rng, 1, 128)
        less = 16 if dtype == "f32" else 1
        most = min(MOST_CACHE // (requests * kv_heads * dim), MOST_TREE // (requests * tree * heads * dim * less))
        longest = _spread(rng, 1, max(1, min(32768, most) - tree))
        return dict(kind=kind, requests=requests, tree=tree, shortest=rng.randrange(0, longest + 1), longest=longest, heads=heads,
                    kv_heads=kv_heads, dim=dim, page=page, window=rng.choice([0, 0, 0, rng.randrange(1, longest + 200)]),
                    chain=rng.random() < 0.3, dtype=dtype)
    layers = _spread(rng, 2, 64)
    vectors = MOST_MOVED // (2 * layers * kv_heads * dim) // (2 if dtype == "f32" else 1)
    if kind == "keep":
        requests, among = _spread(rng, 1, 64), _spread(rng, 1, 4096)
        among = max(1, min(among, vectors // (2 * requests)))
        first = rng.randrange(0, max(1, min(2000, vectors // requests - among)))
        return dict(kind=kind, requests=requests, kept=_spread(rng, 1, among), among=among, first=first, layers=layers,
                    kv_heads=kv_heads, dim=dim, page=page, dtype=dtype)
    pairs = _spread(rng, 1, min(512, vectors // page))
    return dict(kind=kind, pairs=pairs, sources=rng.choice([pairs, max(1, pairs // 4)]), layers=layers, kv_heads=kv_heads, dim=dim,
                page=page, dtype=dtype)


# ---- sizes ------------------------------------------------------------------------------------------------------------
def _contexts(case: dict) -> List[int]:
    """The contexts of an attention case: evenly from the shortest to the longest."""
    n = case["requests"]
    return [case["shortest"] + (case["longest"] - case["shortest"]) * (i + 1) // n if i + 1 < n else case["longest"]
            for i in range(n)]


def _trees(case: dict) -> List[int]:
    """The drafted tokens of each request: as many as ``tree`` says, or some fewer."""
    t = case["tree"]
    return [t - (i * 5) % (t // 4 + 1) for i in range(case["requests"])]


def _kept(case: dict) -> List[int]:
    k = case["kept"]
    return [k - (i * 3) % (k // 4 + 1) for i in range(case["requests"])]


def work(case: dict) -> Dict[str, float]:
    kind = case["kind"]
    size = {"bf16": 2, "f32": 4}[case["dtype"]]
    if kind == "score":
        n, v = case["rows"], case["vocab"]
        return {"bytes": n * (size * v + 8 * case["given"] + 4 + 8 * case["top"]), "flops": 6.0 * n * v}
    kv, d = case["kv_heads"], case["dim"]
    if kind == "tree":
        h, w = case["heads"], case["window"]
        seen = [min(c, w) if w else c for c in _contexts(case)]
        trees = _trees(case)
        return {"bytes": size * (sum(c + t for c, t in zip(seen, trees)) * kv * 2 * d + 2 * sum(trees) * h * d),
                "flops": 4.0 * h * d * sum((c + 1) * t for c, t in zip(seen, trees))}
    planes = 2 * case["layers"]
    if kind == "keep":
        return {"bytes": 2.0 * size * planes * kv * d * sum(_kept(case)), "flops": 0.0}
    return {"bytes": 1.0 * size * planes * kv * d * case["page"] * (case["pairs"] + case["sources"]), "flops": 0.0}


# ---- what a program has in hand before the call ------------------------------------------------------------------------
def _table(g, needed: List[int], page: int):
    """Every request's pages, somewhere in a pool, and the table that says where: (pages in the pool, table)."""
    counts = [-(-n // page) for n in needed]
    order = torch.randperm(sum(counts), generator=g, device=DEV).to(torch.int32)
    table = torch.full((len(needed), max(counts)), -1, dtype=torch.int32, device=DEV)
    at = 0
    for i, c in enumerate(counts):
        table[i, :c] = order[at:at + c]
        at += c
    return sum(counts), table


def _ints(numbers) -> torch.Tensor:
    return torch.tensor(numbers, dtype=torch.int32, device=DEV)


def prepare(case: dict, seed: int) -> dict:
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    rng = random.Random(seed)
    kind, dtype = case["kind"], TYPES[case["dtype"]]
    s = {"case": case}
    if kind == "score":
        n, v = case["rows"], case["vocab"]
        x = 2.5 * torch.randn((n, v), generator=g, device=DEV)
        used = v - case["unused"]
        for _ in range(4):       # a few tokens that fit the text
            x.scatter_(1, torch.randint(0, used, (n, 1), generator=g, device=DEV), 8 + 6 * torch.rand((n, 1), generator=g, device=DEV))
        x[:, used:] = float("-inf")         # places of the vocabulary that stand for no token
        s["logits"] = x.to(dtype)
        given = torch.randint(0, used, (n, case["given"]), generator=g, device=DEV)
        given[:, 0] = torch.where(torch.rand((n,), generator=g, device=DEV) < 0.7, x.argmax(1), given[:, 0])
        s["tokens"] = given.to(torch.int32)
        return s
    kv, d, page = case["kv_heads"], case["dim"], case["page"]
    if kind == "tree":
        contexts, trees = _contexts(case), _trees(case)
        rng.shuffle(contexts)
        words = -(-max(trees) // 32)
        seen, positions = [], []
        for c, t in zip(contexts, trees):
            masks = []
            for i in range(t):
                parent = i - 1 if case["chain"] else rng.randrange(max(-1, i - 12), i)
                masks.append((masks[parent] if parent >= 0 else 0) | 1 << i)
            seen += [[(m >> 32 * w & 0xFFFFFFFF) - (m >> 32 * w + 31 & 1) * 2 ** 32 for w in range(words)] for m in masks]
            positions += [c + bin(m).count("1") - 1 for m in masks]
        starts = [sum(trees[:i]) for i in range(len(trees) + 1)]
        n_pages, s["block_table"] = _table(g, [c + t for c, t in zip(contexts, trees)], page)
        s["q_start"], s["context"] = _ints(starts), _ints(contexts)
        s["positions"], s["seen"] = _ints(positions), _ints(seen)
        s["q"] = (2 * torch.randn((starts[-1], case["heads"], d), generator=g, device=DEV)).to(dtype)
        s["k"] = torch.randn((n_pages, kv, page, d), generator=g, device=DEV).to(dtype)
        s["v"] = torch.randn((n_pages, kv, page, d), generator=g, device=DEV).to(dtype)
        return s
    if kind == "keep":
        kept = _kept(case)
        places = [sorted(rng.sample(range(case["among"]), k)) for k in kept]
        n_pages, s["block_table"] = _table(g, [case["first"] + case["among"]] * len(kept), page)
        s["kept"] = _ints([p + [0] * (max(kept) - len(p)) for p in places])
        s["n_kept"], s["context"] = _ints(kept), _ints([case["first"]] * len(kept))
    else:
        pairs, sources = case["pairs"], case["sources"]
        n_pages = pairs + sources + 3
        order = torch.randperm(n_pages, generator=g, device=DEV).to(torch.int32)
        s["source"], s["target"] = order[:sources].repeat(-(-pairs // sources))[:pairs].contiguous(), order[sources:sources + pairs].contiguous()
    shape = (case["layers"], 2, n_pages, kv, page, d)
    s["pages"] = torch.empty(shape, dtype=dtype, device=DEV)
    for layer in s["pages"]:
        layer.copy_(torch.randn(shape[1:], generator=g, device=DEV))
    return s


# ---- a pass ------------------------------------------------------------------------------------------------------------
def run(s: dict):
    return (_run_own if own else _run_plain)(s)


def _run_own(s: dict):
    from inferrs_b200 import kernels

    case = s["case"]
    kind = case["kind"]
    if kind == "tree":
        out = torch.empty((s["q"].shape[0], case["heads"] * case["dim"]), dtype=s["q"].dtype, device=s["q"].device)
        kernels.paged_attention_tree(s["q"], s["k"], s["v"], s["block_table"], s["q_start"], s["context"], s["positions"], s["seen"],
                                     case["dim"] ** -0.5, case["window"] or None, out, max_tree=case["tree"],
                                     max_kv_len=case["longest"] + case["tree"])
        return out
    if kind == "keep":
        kernels.keep_tokens(s["pages"], 2, s["block_table"], s["context"], s["kept"], s["n_kept"])
        return s["pages"]
    if kind == "copy":
        kernels.copy_pages(s["pages"], 2, s["source"], s["target"])
        return s["pages"]
    n, dev = case["rows"], s["logits"].device
    out = {"log_probs": torch.empty((n, case["given"]), dtype=torch.float32, device=dev),
           "entropy": torch.empty((n,), dtype=torch.float32, device=dev)}
    if case["top"]:
        out["top_ids"] = torch.empty((n, case["top"]), dtype=torch.int32, device=dev)
        out["top_log_probs"] = torch.empty((n, case["top"]), dtype=torch.float32, device=dev)
    kernels.token_log_probs(s["logits"], s["tokens"], out["log_probs"], out["entropy"], out.get("top_ids"), out.get("top_log_probs"))
    return out


def _run_plain(s: dict):
    case = s["case"]
    kind = case["kind"]
    if kind == "score":
        x = s["logits"].float()
        z = x - x.amax(1, keepdim=True)
        e = torch.exp(z)
        total = e.sum(1, keepdim=True)
        log_total = torch.log(total)
        out = {"log_probs": z.gather(1, s["tokens"].long()) - log_total,
               "entropy": log_total[:, 0] - (e * torch.where(e > 0, z, 0.0)).sum(1) / total[:, 0]}
        if case["top"]:
            best, ids = torch.sort(z, dim=1, descending=True, stable=True)
            out["top_ids"] = ids[:, :case["top"]].to(torch.int32)
            out["top_log_probs"] = best[:, :case["top"]] - log_total
        return out
    if kind == "copy":
        pages = s["pages"]
        pages[:, :, s["target"].long()] = pages[:, :, s["source"].long()]
        return pages
    page = case["page"]
    if kind == "keep":
        pages = s["pages"]
        i = torch.arange(s["kept"].shape[1], device=pages.device)
        r, i = torch.nonzero(i[None] < s["n_kept"][:, None], as_tuple=True)
        table, first = s["block_table"].long(), s["context"].long()
        old, new = first[r] + s["kept"][r, i].long(), first[r] + i
        moved = pages[:, :, table[r, old // page], :, old % page]
        pages[:, :, table[r, new // page], :, new % page] = moved
        return pages
    n, h, kv, d = s["q"].shape[0], case["heads"], case["kv_heads"], case["dim"]
    dev, t = s["q"].device, case["tree"]
    start, context = s["q_start"].long(), s["context"].long()
    requests = context.shape[0]
    table = s["block_table"].long().clamp(min=0)
    k, v = (s[name][table].float().transpose(1, 2).reshape(requests, kv, -1, d) for name in ("k", "v"))
    length = k.shape[2]
    # a request's rows, as many as the largest tree has, and whether they are its own
    i = torch.arange(t, device=dev)
    row = (start[:-1, None] + i).clamp(max=n - 1)
    mine = i < (start[1:] - start[:-1])[:, None]
    j = torch.arange(length, device=dev)
    lo = s["positions"].long()[row] - case["window"] + 1 if case["window"] else torch.zeros_like(row)
    seen = (j < context[:, None])[:, None] & (j >= lo[..., None])
    drafted = (s["seen"].long()[:, i // 32] >> (i % 32) & 1).bool()[row] & mine[:, None]
    off = j - context[:, None]
    inside = (off >= 0) & (off < t)
    seen = seen | inside[:, None] & drafted.gather(2, off.clamp(0, t - 1)[:, None].expand(-1, t, -1))
    q = s["q"].float()[row].view(requests, t, kv, h // kv, d).permute(0, 2, 3, 1, 4).reshape(requests, kv, -1, d)
    score = ((q @ k.transpose(-1, -2)) * d ** -0.5).view(requests, kv, h // kv, t, length)
    score.masked_fill_(~seen[:, None, None], float("-inf"))
    top = score.amax(-1, keepdim=True)
    p = torch.exp_(score.sub_(torch.where(top > float("-inf"), top, 0.0)))
    total = p.sum(-1, keepdim=True)
    p = p.view(requests, kv, -1, length) @ v
    o = p.view(requests, kv, h // kv, t, d) / torch.where(total > 0, total, 1.0)
    return o.permute(0, 3, 1, 2, 4).reshape(requests, t, h * d)[mine].to(s["q"].dtype)


# ---- the same in 64 bits, from the definitions --------------------------------------------------------------------------
def exact(case: dict, seed: int):
    kind = case["kind"]
    if kind in ("copy", "keep"):      # numbers that are moved and not computed
        return None
    s = prepare(case, seed)
    if kind == "score":
        out = {"log_probs": torch.empty((case["rows"], case["given"]), dtype=torch.float64, device=DEV),
               "entropy": torch.empty((case["rows"],), dtype=torch.float64, device=DEV)}
        k = case["top"]
        if k:
            out["top_ids"] = torch.empty((case["rows"], k), dtype=torch.int64, device=DEV)
            out["top_log_probs"] = torch.empty((case["rows"], k), dtype=torch.float64, device=DEV)
        for r0 in range(0, case["rows"], 128):
            x = s["logits"][r0:r0 + 128].double()
            lp = torch.log_softmax(x, dim=1)
            rows = torch.arange(x.shape[0], device=DEV)
            out["log_probs"][r0:r0 + 128] = lp[rows[:, None], s["tokens"][r0:r0 + 128].long()]
            out["entropy"][r0:r0 + 128] = -torch.nan_to_num(lp.exp() * lp, nan=0.0).sum(1)
            for c in range(k):        # the lowest place of the largest logit, then without it
                best = x.max(dim=1).values
                place = torch.arange(x.shape[1], device=DEV).expand_as(x)
                at = torch.where(x == best[:, None], place, torch.full_like(place, x.shape[1])).min(dim=1).values
                out["top_ids"][r0:r0 + 128, c] = at
                out["top_log_probs"][r0:r0 + 128, c] = lp[rows, at]
                x[rows, at] = float("-inf")
        return out
    h, kv, d, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    start, context = s["q_start"].tolist(), s["context"].tolist()
    words, positions = s["seen"].tolist(), s["positions"].tolist()
    out = torch.zeros((start[-1], h, d), dtype=torch.float64, device=DEV)
    for r, c in enumerate(context):
        n = start[r + 1] - start[r]
        place = torch.arange(c + n, device=DEV)
        at = s["block_table"][r].long()[place // page]
        k, v = s["k"][at, :, place % page].double(), s["v"][at, :, place % page].double()       # [places, kv, d]
        mask = torch.zeros((n, c + n), dtype=torch.bool)
        for i in range(n):
            lo = max(0, positions[start[r] + i] - case["window"] + 1) if case["window"] else 0
            mask[i, lo:c] = True
            for j in range(n):
                mask[i, c + j] = bool(words[start[r] + i][j // 32] >> j % 32 & 1)
        some = mask.any(1).to(DEV)
        mask = mask.to(DEV)
        for head in range(h):
            q = s["q"][start[r]:start[r + 1], head].double()
            x = (q @ k[:, head // (h // kv)].t()) / math.sqrt(d)
            x[~mask] = float("-inf")
            o = torch.softmax(x, dim=1) @ v[:, head // (h // kv)]
            out[start[r]:start[r + 1], head] = torch.where(some[:, None], o, torch.zeros_like(o))
    return out.view(start[-1], h * d)
