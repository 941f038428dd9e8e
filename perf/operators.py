"""The operators of a model in few bits, as cases that can be timed and compared.

A case is a dictionary of plain values.  Its ``kind`` names the operator:

quantize   rows to 4-bit numbers with a scale per 32 of them (``kernels.quantize_mx4``) and back to the values that they
           stand for (``kernels.dequantize_mx4``)
linear     y = x W^T with W in 4 bits and bfloat16 rows x that keep their precision (``kernels.linear_mx4``)
linear4    the same with the rows of x brought to 4 bits on the way (``quantize_mx4``, then ``linear_mx4``)
append     the step's queries, keys and values from the fused projection: norm per head, rotation by position, keys and
           values in 8 bits into their pages (``kernels.qk_norm_rope_store_kv8``)
attention  one new token per request over the pages of 8-bit keys and values (``kernels.paged_attention_kv8``)

4-bit numbers (sign, two bits of exponent, one of mantissa: 0, 0.5, 1, 1.5, 2, 3, 4, 6) share a power of two per 32
along a row: with a the block's largest magnitude, e = floor(log2 a) - 2, one more where a > 7 * 2^e, and a number is
its quotient by 2^e rounded to the nearest (ties to even).  Two numbers are in a byte, the earlier one in its low half;
a row is padded with zeros to a multiple of 128.  Scales (e + 127) stand in tiles of 128 rows and 128 numbers of a row,
byte [tile of rows, tile of columns, row % 32, row / 32 % 4, block % 4], an even number of tiles of columns.

Keys and values in 8 bits (four bits of exponent, three of mantissa) share a float32 scale per vector of a head, a / 448
with a its largest magnitude; a number is x * (448 / a) rounded to the nearest.

The plain forms work in 32 bits and round once at the end.  The model sizes are those of the benchmark.
"""
from __future__ import annotations

import math
import random
from typing import Dict, List

import torch

own = False

DEV = "cuda"
BF16_ROUND = {"bf16": torch.bfloat16, "f32": torch.float32}
MOST_PRODUCT = 2048 * 12288 * 4096          # multiply-adds of the largest listed product
MOST_WEIGHTS = 24576 * 4096
MOST_CACHE = 16 * 8192 * 8 * 128            # numbers of keys of the largest listed cache


def listed() -> List[dict]:
    return [
        # a decode step's rows on their way into a 4-bit product: the smallest call, an odd number of rows
        dict(name="quantize 13x5120", kind="quantize", rows=13, width=5120, dtype="bf16"),
        # a checkpoint's largest matrix when it is loaded
        dict(name="quantize 24576x4096", kind="quantize", rows=24576, width=4096, dtype="bf16"),
        # one chat on a small model: a projection's latency
        dict(name="linear 1x1024x4096", kind="linear", rows=1, width=1024, features=4096),
        # the benchmark's decode step of eight requests: gate and up
        dict(name="linear 8x4096x24576", kind="linear", rows=8, width=4096, features=24576),
        # a short prompt on a model of unusual sizes
        dict(name="linear 77x2080x5003", kind="linear", rows=77, width=2080, features=5003),
        # the benchmark's prompt of 2,048 tokens: the down projection
        dict(name="linear 2048x12288x4096", kind="linear", rows=2048, width=12288, features=4096),
        # a busy server's decode step with rows in 4 bits too
        dict(name="linear4 48x4096x24576", kind="linear4", rows=48, width=4096, features=24576),
        # a prompt with rows in 4 bits too
        dict(name="linear4 2048x4096x24576", kind="linear4", rows=2048, width=4096, features=24576),
        # the benchmark's decode step of eight requests: one token each joins its cache
        dict(name="append 8 tokens", kind="append", requests=8, tokens=8, cached=2048, heads=32, kv_heads=8, dim=128,
             page=16),
        # the benchmark's prompt goes into its cache
        dict(name="append 2048 tokens", kind="append", requests=1, tokens=2048, cached=0, heads=32, kv_heads=8, dim=128,
             page=16),
        # one chat on a small model, a short context
        dict(name="attention 1x300", kind="attention", requests=1, shortest=300, longest=300, heads=16, kv_heads=8, dim=128,
             page=16, window=0),
        # a server's decode step: sixteen requests of every age with long contexts
        dict(name="attention 16x16384", kind="attention", requests=16, shortest=100, longest=16384, heads=32, kv_heads=8,
             dim=128, page=16, window=0),
    ]


def _spread(rng: random.Random, low: int, high: int) -> int:
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng: random.Random) -> dict:
    kind = rng.choice(["quantize", "linear", "linear", "linear4", "append", "attention", "attention"])
    if kind == "quantize":
        width = _spread(rng, 32, 16384)
        rows = _spread(rng, 1, min(32768, MOST_WEIGHTS // width))
        return dict(kind=kind, rows=rows, width=width, dtype=rng.choice(["bf16", "f32"]) if rows * width <= MOST_WEIGHTS // 2
                    else "bf16")
    if kind in ("linear", "linear4"):
        rows = _spread(rng, 1, 2048)
        width = _spread(rng, 16, 1024) * 16 if rng.random() < 0.7 else _spread(rng, 100, 12288)
        features = _spread(rng, 64, 32768)
        features = min(features, MOST_WEIGHTS // width, max(64, MOST_PRODUCT // (rows * width)))
        return dict(kind=kind, rows=rows, width=width, features=features)
    heads, kv_heads = rng.choice([(16, 8), (32, 8), (64, 8), (8, 8), (20, 4), (32, 2)])
    dim, page = rng.choice([64, 128, 128]), rng.choice([16, 16, 32, 64])
    if kind == "append":
        tokens = _spread(rng, 1, 2048)
        requests = _spread(rng, 1, min(tokens, 256))
        return dict(kind=kind, requests=requests, tokens=tokens, cached=rng.randrange(0, 1500 if requests < 64 else 300),
                    heads=heads, kv_heads=kv_heads, dim=dim, page=page)
    requests = _spread(rng, 1, 256)
    longest = min(_spread(rng, 1, 32768), max(1, MOST_CACHE // (requests * kv_heads * dim)))
    return dict(kind=kind, requests=requests, shortest=rng.randrange(1, longest + 1), longest=longest, heads=heads,
                kv_heads=kv_heads, dim=dim, page=page, window=rng.choice([0, 0, 0, rng.randrange(1, longest + 200)]))


# ---- sizes ------------------------------------------------------------------------------------------------------------
def _up(n: int, m: int) -> int:
    return -(-n // m) * m


def _lengths(case: dict) -> List[int]:
    """The contexts of an attention case, the new token with them: evenly from the shortest to the longest."""
    n = case["requests"]
    return [case["shortest"] + (case["longest"] - case["shortest"]) * i // max(1, n - 1) for i in range(n)]


def _portions(case: dict) -> List[int]:
    """The tokens that each request of an append case brings."""
    n, r = case["tokens"], case["requests"]
    return [n // r + (1 if i < n % r else 0) for i in range(r)]


def work(case: dict) -> Dict[str, float]:
    kind = case["kind"]
    if kind == "quantize":
        n = case["rows"] * case["width"]
        size = 2 if case["dtype"] == "bf16" else 4
        return {"bytes": n * (2 * size + 2 * 17 / 32), "flops": 4 * n}
    if kind in ("linear", "linear4"):
        n, k, m = case["rows"], case["width"], case["features"]
        return {"bytes": m * k * 17 / 32 + 2 * n * (k + m), "flops": 2.0 * n * k * m}
    h, kv, d = case["heads"], case["kv_heads"], case["dim"]
    if kind == "append":
        n = case["tokens"]
        return {"bytes": n * (2 * d * (2 * h + 2 * kv) + 2 * kv * (d + 4) + 4 * d), "flops": 10 * n * (h + 2 * kv) * d}
    seen = sum(min(n, case["window"]) if case["window"] else n for n in _lengths(case))
    return {"bytes": seen * kv * 2 * (d + 4) + 4 * case["requests"] * h * d, "flops": 4.0 * seen * h * d}


# ---- what a program has in hand before the call ------------------------------------------------------------------------
def _activations(g, n: int, k: int) -> torch.Tensor:
    """Rows as a norm leaves them: every channel with a size of its own, a few of them large."""
    size = torch.exp(0.5 * torch.randn((k,), generator=g, device=DEV))
    loud = torch.rand((k,), generator=g, device=DEV) < 0.002
    return torch.randn((n, k), generator=g, device=DEV) * torch.where(loud, 30 * size, size)


def _encode(x: torch.Tensor):
    """x [rows, width] as 4-bit codes and tiles of scales (see the head of this file), to have weights to start from."""
    rows, width = x.shape
    k = _up(width, 128)
    tiles = 2 * (_up(width, 256) // 256)
    blocks = torch.nn.functional.pad(x, (0, k - width)).view(rows, k // 32, 32)
    a = blocks.abs().amax(-1)
    e = torch.frexp(a)[1] - 3
    e = e + (a > torch.ldexp(torch.full_like(a, 7.0), e)).to(e.dtype)
    e = torch.where(a > 0, e.clamp(-127, 127), torch.full_like(e, -127))
    q = torch.ldexp(blocks, -e.unsqueeze(-1))
    m = q.abs()
    m = torch.where(m < 2, torch.round(m * 2) / 2, torch.where(m < 4, torch.round(m), torch.round(m / 2) * 2)).clamp(max=6)
    code = torch.where(m < 2, m * 2, torch.where(m < 4, m + 2, m / 2 + 4)).to(torch.uint8)
    code = (code | (torch.signbit(q).to(torch.uint8) << 3)).view(rows, k // 2, 2)
    codes = (code[..., 0] | (code[..., 1] << 4)).contiguous()
    scales = torch.zeros((_up(rows, 128), tiles * 4), dtype=torch.uint8, device=x.device)
    scales[:rows, :k // 32] = (e + 127).to(torch.uint8)
    scales = scales.view(-1, 4, 32, tiles, 4).permute(0, 3, 2, 1, 4).contiguous()
    return codes, scales


def _pages(case: dict, g, needed: List[int]):
    """A pool of pages with every request's pages somewhere in it, and the table that says where."""
    page, kv, d = case["page"], case["kv_heads"], case["dim"]
    counts = [-(-n // page) for n in needed]
    total = sum(counts)
    order = torch.randperm(total, generator=g, device=DEV).to(torch.int32)
    table = torch.zeros((len(needed), max(counts)), dtype=torch.int32, device=DEV)
    at = 0
    for i, c in enumerate(counts):
        table[i, :c] = order[at:at + c]
        at += c
    pool = {"block_table": table}
    for name, loud in (("k", 4.0), ("v", 1.0)):
        x = torch.randn((total, kv, page, d), generator=g, device=DEV)
        a = x.abs().amax(-1)
        pool[name] = (x * (448 / a).unsqueeze(-1)).clamp(-448, 448).to(torch.float8_e4m3fn)
        pool[name + "_scale"] = a / 448 * loud * torch.exp(0.3 * torch.randn(a.shape, generator=g, device=DEV))
    return pool


def prepare(case: dict, seed: int) -> dict:
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    kind = case["kind"]
    s = {"case": case}
    if kind == "quantize":
        if case["rows"] > 4096:              # a weight matrix
            x = 0.02 * torch.randn((case["rows"], case["width"]), generator=g, device=DEV)
        else:
            x = _activations(g, case["rows"], case["width"])
        s["x"] = x.to(BF16_ROUND[case["dtype"]])
    elif kind in ("linear", "linear4"):
        s["x"] = _activations(g, case["rows"], case["width"]).to(torch.bfloat16)
        s["codes"], s["scales"] = _encode(0.02 * torch.randn((case["features"], case["width"]), generator=g, device=DEV))
    elif kind == "append":
        h, kv, d = case["heads"], case["kv_heads"], case["dim"]
        n, cached = case["tokens"], case["cached"]
        portions = _portions(case)
        s["qkv"] = torch.randn((n, (h + 2 * kv) * d), generator=g, device=DEV).to(torch.bfloat16)
        s["q_weight"] = (1 + 0.2 * torch.rand((d,), generator=g, device=DEV)).to(torch.bfloat16)
        s["k_weight"] = (1 + 0.2 * torch.rand((d,), generator=g, device=DEV)).to(torch.bfloat16)
        angle = torch.arange(cached + max(portions), dtype=torch.float64, device=DEV)[:, None] * \
            1e6 ** (-torch.arange(0, d, 2, dtype=torch.float64, device=DEV) / d)
        s["cos"], s["sin"] = torch.cos(angle).float(), torch.sin(angle).float()
        s["row_request"] = torch.cat([torch.full((c,), i, dtype=torch.int32) for i, c in enumerate(portions)]).to(DEV)
        s["positions"] = torch.cat([torch.arange(cached, cached + c, dtype=torch.int32) for c in portions]).to(DEV)
        s.update(_pages(case, g, [cached + c for c in portions]))
    else:
        h, d = case["heads"], case["dim"]
        lengths = _lengths(case)
        order = torch.randperm(len(lengths), generator=g, device=DEV).tolist()
        lengths = [lengths[i] for i in order]
        s["q"] = (2 * torch.randn((len(lengths), h, d), generator=g, device=DEV)).to(torch.bfloat16)
        s["row_request"] = torch.arange(len(lengths), dtype=torch.int32, device=DEV)
        s["positions"] = torch.tensor([n - 1 for n in lengths], dtype=torch.int32, device=DEV)
        s.update(_pages(case, g, lengths))
    return s


# ---- a pass ------------------------------------------------------------------------------------------------------------
def run(s: dict):
    return (_run_own if own else _run_plain)(s)


def _run_own(s: dict):
    from inferrs_b200 import kernels

    case = s["case"]
    kind = case["kind"]
    if kind == "quantize":
        y = torch.empty_like(s["x"])
        kernels.dequantize_mx4(kernels.quantize_mx4(s["x"]), y)
        return y
    if kind in ("linear", "linear4"):
        w = kernels.Mx4Matrix(s["codes"], s["scales"], case["features"], case["width"])
        y = torch.empty((case["rows"], case["features"]), dtype=torch.bfloat16, device=s["x"].device)
        kernels.linear_mx4(s["x"] if kind == "linear" else kernels.quantize_mx4(s["x"]), w, y)
        return y
    pages = kernels.Kv8Pages(s["k"], s["v"], s["k_scale"], s["v_scale"])
    h, kv, d = case["heads"], case["kv_heads"], case["dim"]
    if kind == "append":
        q = torch.empty((case["tokens"], h, d), dtype=torch.bfloat16, device=s["qkv"].device)
        kernels.qk_norm_rope_store_kv8(s["qkv"], h, kv, d, s["q_weight"], s["k_weight"], 1e-6, s["cos"], s["sin"], d,
                                       s["positions"], s["row_request"], s["block_table"], pages, q)
        return {"q": q, "k": s["k"], "v": s["v"], "k_scale": s["k_scale"], "v_scale": s["v_scale"]}
    out = torch.empty((case["requests"], h * d), dtype=torch.bfloat16, device=s["q"].device)
    kernels.paged_attention_kv8(s["q"], pages, s["block_table"], s["row_request"], s["positions"], d ** -0.5,
                                case["window"] or None, out, case["longest"])
    return out


def _values4(x: torch.Tensor) -> torch.Tensor:
    """The values that the rows of x stand for in 4 bits, as float32."""
    rows, width = x.shape
    blocks = torch.nn.functional.pad(x.float(), (0, _up(width, 32) - width)).view(rows, -1, 32)
    a = blocks.abs().amax(-1, keepdim=True)
    e = torch.frexp(a)[1] - 3
    e = e + (a > torch.ldexp(torch.full_like(a, 7.0), e)).to(e.dtype)
    e = e.clamp(-127, 127)
    q = torch.ldexp(blocks, -e)
    m = q.abs()
    m = torch.where(m < 2, torch.round(m * 2) / 2, torch.where(m < 4, torch.round(m), torch.round(m / 2) * 2)).clamp(max=6)
    return torch.ldexp(torch.copysign(m, q), e).view(rows, -1)[:, :width]


def _decode(codes: torch.Tensor, scales: torch.Tensor, rows: int, width: int) -> torch.Tensor:
    """The float32 matrix that codes and tiles of scales stand for."""
    table = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, 0, -0.5, -1, -1.5, -2, -3, -4, -6], device=codes.device)
    v = table[torch.stack((codes & 15, codes >> 4), dim=-1).view(rows, -1).int()]
    byte = scales.permute(0, 3, 2, 1, 4).reshape(scales.shape[0] * 128, -1)[:rows, :v.shape[1] // 32]
    return torch.ldexp(v.view(rows, -1, 32), byte.int().unsqueeze(-1) - 127).view(rows, -1)[:, :width]


def _rotated(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor) -> torch.Tensor:
    half = x.shape[-1] // 2
    a, b = x[..., :half], x[..., half:]
    return torch.cat((a * cos - b * sin, b * cos + a * sin), dim=-1)


def _to8(x: torch.Tensor):
    """Vectors (the last axis) as 8-bit numbers and their scales."""
    a = x.abs().amax(-1)
    some = a >= 2.0 ** -100
    q = (x * torch.where(some, 448 / a, torch.zeros_like(a)).unsqueeze(-1)).clamp(-448, 448)
    return q.to(torch.float8_e4m3fn), torch.where(some, a / 448, torch.zeros_like(a))


def _run_plain(s: dict):
    case = s["case"]
    kind = case["kind"]
    if kind == "quantize":
        return _values4(s["x"]).to(s["x"].dtype)
    if kind in ("linear", "linear4"):
        x = s["x"].float() if kind == "linear" else _values4(s["x"])
        return (x @ _decode(s["codes"], s["scales"], case["features"], case["width"]).t()).to(torch.bfloat16)
    h, kv, d, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    req, pos = s["row_request"].long(), s["positions"].long()
    if kind == "append":
        n = case["tokens"]
        x = s["qkv"].float().view(n, h + 2 * kv, d)
        q, k, v = x[:, :h], x[:, h:h + kv], x[:, h + kv:]
        q = q * (1.0 / torch.sqrt((q * q).mean(-1, keepdim=True) + 1e-6)) * s["q_weight"].float()
        k = k * (1.0 / torch.sqrt((k * k).mean(-1, keepdim=True) + 1e-6)) * s["k_weight"].float()
        cos, sin = s["cos"][pos].unsqueeze(1), s["sin"][pos].unsqueeze(1)
        q, k = _rotated(q, cos, sin), _rotated(k, cos, sin)
        at = s["block_table"][req, pos // page].long()
        for name, vectors in (("k", k), ("v", v)):
            codes, scale = _to8(vectors)
            s[name].view(torch.uint8)[at, :, pos % page] = codes.view(torch.uint8)
            s[name + "_scale"][at, :, pos % page] = scale
        return {"q": q.to(torch.bfloat16), "k": s["k"], "v": s["v"], "k_scale": s["k_scale"], "v_scale": s["v_scale"]}
    n = case["requests"]
    table = s["block_table"][req].long()
    k, v = ((s[name].view(torch.uint8)[table].view(torch.float8_e4m3fn).float() * s[name + "_scale"][table].unsqueeze(-1))
            .transpose(1, 2).reshape(n, kv, -1, d) for name in ("k", "v"))
    q = s["q"].float().view(n, kv, h // kv, d)
    score = (q @ k.transpose(-1, -2)) * d ** -0.5
    j = torch.arange(score.shape[-1], device=score.device)
    lo = (pos - case["window"] + 1 if case["window"] else torch.zeros_like(pos))[:, None]
    seen = ((j <= pos[:, None]) & (j >= lo))[:, None, None]
    score = score.masked_fill(~seen, float("-inf"))
    p = torch.exp(score - score.amax(-1, keepdim=True))
    out = (p @ v) / p.sum(-1, keepdim=True)
    return out.reshape(n, h * d).to(torch.bfloat16)


# ---- the same in 64 bits, from the definitions --------------------------------------------------------------------------
_E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _exact_values4(x: torch.Tensor) -> torch.Tensor:
    rows, width = x.shape
    out = torch.empty((rows, width), dtype=torch.float64, device=x.device)
    edges = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], dtype=torch.float64, device=x.device)
    grid = torch.tensor(_E2M1, dtype=torch.float64, device=x.device)
    odd = torch.tensor([False, True, False, True, False, True, False], device=x.device)   # a tie goes up to an even code
    for r0 in range(0, rows, 2048):
        part = x[r0:r0 + 2048].double()
        k = _up(width, 32)
        b = torch.zeros((part.shape[0], k), dtype=torch.float64, device=x.device)
        b[:, :width] = part
        b = b.view(part.shape[0], k // 32, 32)
        a = b.abs().max(dim=-1).values
        e = torch.where(a > 0, torch.floor(torch.log2(a.clamp(min=1e-300))), torch.zeros_like(a))
        e = torch.where(2.0 ** e > a, e - 1, torch.where(2.0 ** (e + 1) <= a, e + 1, e)) - 2     # log2 rounds
        e = torch.where(a > 7 * 2.0 ** e, e + 1, e).clamp(-127, 127)
        unit = (2.0 ** e).unsqueeze(-1)
        t = b.abs() / unit
        i = torch.bucketize(t, edges)                     # edges below t
        tie = torch.zeros_like(i)
        at = i.clamp(max=6)
        tie[(t == edges[at]) & odd[at] & (i < 7)] = 1     # a number on an edge whose lower code is odd
        v = grid[(i + tie).clamp(max=7)] * unit * torch.sign(b)
        out[r0:r0 + 2048] = v.view(part.shape[0], k)[:, :width]
    return out


def _exact_matrix(codes: torch.Tensor, scales: torch.Tensor, rows: int, width: int) -> torch.Tensor:
    k = codes.shape[1] * 2
    c = torch.empty((rows, k), dtype=torch.int64, device=codes.device)
    c[:, 0::2] = codes.long() % 16
    c[:, 1::2] = codes.long() // 16
    grid = torch.tensor(_E2M1, dtype=torch.float64, device=codes.device)
    v = grid[c % 8] * (1.0 - 2.0 * (c // 8))
    r = torch.arange(rows, device=codes.device)[:, None]
    b = torch.arange(k // 32, device=codes.device)[None, :]
    byte = scales[r // 128, b // 4, r % 32, r // 32 % 4, b % 4].double()
    return (v * (2.0 ** (byte - 127)).repeat_interleave(32, dim=1))[:, :width]


def _exact8(x: torch.Tensor):
    """Nearest 8-bit numbers (ties to even) of vectors, as the values of their codes, and the scales."""
    a = x.abs().max(dim=-1).values
    t = x * (448 / a).unsqueeze(-1)
    e = torch.floor(torch.log2(t.abs().clamp(min=2.0 ** -6))).clamp(min=-6)
    step = 2.0 ** (e - 3)
    return (torch.round(t / step) * step).clamp(-448, 448), a / 448


def exact(case: dict, seed: int):
    kind = case["kind"]
    s = prepare(case, seed)
    if kind == "quantize":
        return _exact_values4(s["x"])
    if kind in ("linear", "linear4"):
        x = s["x"].double() if kind == "linear" else _exact_values4(s["x"])
        w = _exact_matrix(s["codes"], s["scales"], case["features"], case["width"])
        return torch.mm(x, w.t())
    h, kv, d, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    if kind == "append":
        n = case["tokens"]
        x = s["qkv"].double().view(n, h + 2 * kv, d)
        pos = s["positions"].long()

        def turned(y, weight):
            y = y / (y.pow(2).mean(dim=-1, keepdim=True) + 1e-6).sqrt() * weight.double()
            z = torch.complex(y[..., :d // 2].contiguous(), y[..., d // 2:].contiguous())
            z = z * torch.complex(s["cos"].double(), s["sin"].double())[pos][:, None]
            return torch.cat((z.real, z.imag), dim=-1)

        k8, ks = _exact8(turned(x[:, h:h + kv], s["k_weight"]))
        v8, vs = _exact8(x[:, h + kv:])
        out = {"q": turned(x[:, :h], s["q_weight"]), "k": s["k"].double(), "v": s["v"].double(),
               "k_scale": s["k_scale"].double(), "v_scale": s["v_scale"].double()}
        page_of = s["block_table"][s["row_request"].long(), torch.div(pos, page, rounding_mode="floor")].long()
        for name, codes, scale in (("k", k8, ks), ("v", v8, vs)):
            out[name][page_of, :, pos % page] = codes
            out[name + "_scale"][page_of, :, pos % page] = scale
        return out
    out = torch.empty((case["requests"], h, d), dtype=torch.float64, device=s["q"].device)
    for r in range(case["requests"]):
        last = int(s["positions"][r])
        first = max(0, last - case["window"] + 1) if case["window"] else 0
        j = torch.arange(first, last + 1, device=out.device)
        page_of, place = s["block_table"][r].long()[j // page], j % page
        k = s["k"].view(torch.uint8)[page_of, :, place].view(torch.float8_e4m3fn).double() * \
            s["k_scale"][page_of, :, place, None].double()
        v = s["v"].view(torch.uint8)[page_of, :, place].view(torch.float8_e4m3fn).double() * \
            s["v_scale"][page_of, :, place, None].double()
        for g in range(kv):
            q = s["q"][r, g * (h // kv):(g + 1) * (h // kv)].double()
            out[r, g * (h // kv):(g + 1) * (h // kv)] = torch.softmax(q @ k[:, g].t() / math.sqrt(d), dim=-1) @ v[:, g]
    return out.view(case["requests"], h * d)
