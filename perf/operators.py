"""The operators of a token decoder, in plain form and by the framework's entry points, and the cases they are timed on.

Kinds of case:

* `rotary`: rotary positions of one tensor of heads (`rotary`), forward, or forward and gradient;
* `norm`: the root-mean-square norm of each head of q and k and their rotary positions in one pass (`qk_norm_rotary`), forward, or
  forward and the gradients of q, k and both weights;
* `append`: new keys and values, rotated on the way, into a paged cache held in 4 bits (`kv4_append_`, which rotates q too), and what
  the cache then holds for them (`kv4_read`);
* `attend`: causal attention of the last queries of each sequence over that cache (`kv4_attention`).

The cache is a uint8 tensor `[pages, kv heads, page / 16, 16 (head dim + 8)]`. A block of sixteen tokens of one head holds first the codes
of K, head dim / 2 bytes a token, dimension 2 i in the low and 2 i + 1 in the high half of byte i; then for each two tokens a row of head
dim + 16 bytes: the codes of V in 16-bit words (word i: four dimensions from 4 i on, the lowest in the lowest bits), the words of the
even and the odd token in turn, and behind them for either token four bfloat16: step and least value of K, step and least value of V. A
value is `least + step * code`; a head's vector of one token is a group of its own, `step = (max - min) / 15`, both rounded to bfloat16
before the codes are taken (a step below 2^-126 counts as zero; a group whose range is not finite is held as NaN).
"""

from __future__ import annotations

import math

import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
BYTES = {"fp16": 2, "bf16": 2, "fp32": 4}
EPS = 1e-6
BLOCK = 16
LEAST_STEP = 2.0**-126


def listed() -> list[dict]:
    return [
        # Rotary positions of the queries of eight sequences, one new token each: latency.
        {"name": "rotary-8x1", "kind": "rotary", "batch": 8, "tokens": 1, "heads": 32, "dim": 128, "rot": 128, "interleaved": False, "grad": False, "prefix": 0, "packed": False, "dtype": "bf16"},
        # An encoder's batch of 512 px images, q inside the packed qkv tensor, class token and registers left alone, neighbouring pairs.
        {"name": "rotary-32x1029", "kind": "rotary", "batch": 32, "tokens": 1029, "heads": 16, "dim": 64, "rot": 64, "interleaved": True, "grad": False, "prefix": 5, "packed": True, "dtype": "fp16"},
        # A training step on long sequences, half of each head rotated.
        {"name": "rotary-train-4x4096", "kind": "rotary", "batch": 4, "tokens": 4096, "heads": 32, "dim": 128, "rot": 64, "interleaved": False, "grad": True, "prefix": 0, "packed": False, "dtype": "bf16"},
        # Norm and rotation of sixteen sequences' new tokens: latency.
        {"name": "norm-16x1", "kind": "norm", "batch": 16, "tokens": 1, "q_heads": 32, "kv_heads": 8, "dim": 128, "rot": 128, "interleaved": False, "grad": False, "prefix": 0, "packed": False, "dtype": "bf16"},
        # An encoder block with normed q and k on eight 518 px images: a ragged token count, views of the packed qkv tensor.
        {"name": "norm-8x1370", "kind": "norm", "batch": 8, "tokens": 1370, "q_heads": 24, "kv_heads": 24, "dim": 64, "rot": 64, "interleaved": True, "grad": False, "prefix": 1, "packed": True, "dtype": "fp16"},
        # A training step of a decoder with shared key heads.
        {"name": "norm-train-2x4096", "kind": "norm", "batch": 2, "tokens": 4096, "q_heads": 32, "kv_heads": 8, "dim": 128, "rot": 128, "interleaved": False, "grad": True, "prefix": 0, "packed": False, "dtype": "bf16"},
        # Sixty-four sequences each get their next token.
        {"name": "append-64x1", "kind": "append", "batch": 64, "tokens": 1, "q_heads": 32, "kv_heads": 8, "dim": 128, "rot": 128, "interleaved": False, "page": 64, "context": 4096, "dtype": "bf16"},
        # Prompts of four sequences, padded on the left to the longest.
        {"name": "append-4x2047", "kind": "append", "batch": 4, "tokens": 2047, "q_heads": 32, "kv_heads": 8, "dim": 128, "rot": 64, "interleaved": True, "page": 16, "context": 2047, "dtype": "bf16"},
        # One user waits for the next token behind a moderate text.
        {"name": "attend-1x1x4000", "kind": "attend", "batch": 1, "queries": 1, "q_heads": 32, "kv_heads": 8, "dim": 128, "page": 64, "context": 4000, "ragged": False, "dtype": "bf16"},
        # A server's batch, contexts of all lengths, one sequence just begun and one place unused.
        {"name": "attend-64x1x8192", "kind": "attend", "batch": 64, "queries": 1, "q_heads": 32, "kv_heads": 8, "dim": 128, "page": 64, "context": 8192, "ragged": True, "dtype": "bf16"},
        # Five drafted tokens are checked at once, each head with keys of its own, twelve heads of 64.
        {"name": "attend-16x5x1370", "kind": "attend", "batch": 16, "queries": 5, "q_heads": 12, "kv_heads": 12, "dim": 64, "page": 16, "context": 1370, "ragged": True, "dtype": "fp16"},
        # A piece of a long prompt behind what is in the cache already.
        {"name": "attend-2x500x9000", "kind": "attend", "batch": 2, "queries": 500, "q_heads": 32, "kv_heads": 8, "dim": 128, "page": 128, "context": 9000, "ragged": False, "dtype": "bf16"},
    ]


def _log_int(rng, low: int, high: int) -> int:
    n = min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(max(low, high)))))))
    return n - 1 if n == 3 * 1024 else n


def draw(rng) -> dict:
    kind = rng.choice(["rotary", "norm", "append", "attend", "attend"])
    dtype = rng.choice(["fp16", "bf16"])
    dim = rng.choice([64, 128])
    if kind in ("rotary", "norm"):
        dim = rng.choice([64, 64, 128, 128, 80, 96, 72, 256])
        rot = rng.choice([dim, dim, dim // 2, 2 * rng.randint(1, dim // 2)])
        dtype = rng.choice(["fp16", "bf16", "fp32"])
        kv = rng.choice([1, 2, 3, 4, 6, 8, 12])
        heads = rng.choice([3, 6, 12, 16, 24, 32]) if kind == "rotary" else kv * rng.choice([1, 2, 4, 5])
        heads += heads * dim == 3 * 1024 and kind == "rotary"
        grad = rng.random() < 0.5
        values = heads * dim + (kv * dim if kind == "norm" else 0)
        tokens = 1 if rng.random() < 0.25 else _log_int(rng, 2, 8192)
        batch = _log_int(rng, 1, max(1, min(128, int(4e7 / (values * tokens)))))
        packed = rng.random() < 0.5 and (kind == "rotary" or heads == kv)
        case = {"kind": kind, "batch": batch, "tokens": tokens}
        case |= {"heads": heads} if kind == "rotary" else {"q_heads": heads, "kv_heads": kv}
        return case | {"dim": dim, "rot": rot, "interleaved": rng.random() < 0.5, "grad": grad, "prefix": rng.choice([0, 0, 1, 5]) if tokens > 5 else 0, "packed": packed, "dtype": dtype}
    kv, group = rng.choice([1, 2, 3, 4, 6, 8, 12]), rng.choice([1, 2, 3, 4, 5, 7, 8])
    page = rng.choice([16, 32, 64, 128])
    if kind == "append":
        tokens = 1 if rng.random() < 0.4 else _log_int(rng, 2, 4096)
        batch = _log_int(rng, 1, max(1, min(128, int(4 * 2047 * 40 / (tokens * kv * (group + 1))))))
        context = _log_int(rng, max(16, tokens // 2), 16384)
        context = min(context, max(16, int(64 * 4096 * 8 / (batch * kv))))
        rot = rng.choice([0, dim, dim, dim // 2, 2 * rng.randint(1, dim // 2)])
        return {"kind": kind, "batch": batch, "tokens": tokens, "q_heads": kv * group, "kv_heads": kv, "dim": dim, "rot": rot, "interleaved": rng.random() < 0.5, "page": page, "context": context, "dtype": dtype}
    which = rng.random()
    queries = 1 if which < 0.5 else _log_int(rng, 2, 16) if which < 0.75 else _log_int(rng, 17, 500)
    context = _log_int(rng, 1, 32768)
    most = min(64 * 8192 * 8 * 128 / (context * kv * dim), 2 * 500 * 9000 * 32 * 128 / (queries * max(context, 64) * kv * group * dim), 4096 / queries)
    batch = _log_int(rng, 1, max(1, min(128, int(most))))
    return {"kind": kind, "batch": batch, "queries": queries, "q_heads": kv * group, "kv_heads": kv, "dim": dim, "page": page, "context": context, "ragged": rng.random() < 0.6, "dtype": dtype}


def _lengths(case: dict) -> list[int]:
    """Tokens of each sequence, the new ones among them: a fixed set of a case, spread down from the longest; in larger batches one
    sequence has a single token and one place is unused."""
    b, most = case["batch"], case["context"]
    if not case.get("ragged", True):
        return [most] * b
    got = [max(1, most * (b - i) // b) for i in range(b)]
    if b >= 4:
        got[-1], got[-2] = 0, 1
    return got


def _seen(case: dict) -> int:
    """Keys that all queries of one head see, over the batch."""
    lq = case["queries"]
    return sum(sum(max(0, n - lq + i + 1) for i in range(lq)) for n in _lengths(case))


def work(case: dict) -> dict:
    e, d = BYTES[case["dtype"]], case["dim"]
    rows = case["batch"] * case.get("tokens", case.get("queries", 1))
    if case["kind"] == "rotary":
        n = rows * case["heads"] * d
        table = 8 * (case["rot"] // 2) * min(case["tokens"] if case["tokens"] > 1 else case["batch"], 4096)
        passes = 2 if case["grad"] else 1
        return {"bytes": passes * (2 * n * e + 4 * rows) + table, "flops": passes * 3 * rows * case["heads"] * case["rot"]}
    if case["kind"] == "norm":
        n = rows * (case["q_heads"] + case["kv_heads"]) * d
        table = 8 * (case["rot"] // 2) * min(case["tokens"] if case["tokens"] > 1 else case["batch"], 4096)
        return {"bytes": (5 if case["grad"] else 2) * n * e + 4 * rows + table, "flops": (20 if case["grad"] else 7) * n}
    groups = case["kv_heads"] * (d + 8)
    if case["kind"] == "append":
        new = sum(min(case["tokens"], n) for n in _lengths(case))
        table = 8 * (case["rot"] // 2) * min(case["context"], new)
        return {"bytes": 2 * rows * case["q_heads"] * d * e + new * (2 * case["kv_heads"] * d * e + 2 * groups) + 2 * rows * case["kv_heads"] * d * e + table, "flops": 16 * rows * (case["q_heads"] + case["kv_heads"]) * d}
    return {"bytes": sum(_lengths(case)) * groups + 2 * rows * case["q_heads"] * d * e, "flops": 4 * _seen(case) * case["q_heads"] * d}


# ---- inputs ----------------------------------------------------------------------------------------------------------------------


def _table(length: int, rot: int, device: str) -> torch.Tensor:
    """Cosines and sines of a context stretched fourfold: fp32 `[length, 2, rot / 2]`."""
    inv = 10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64, device=device) / max(rot, 1)) / 4
    angle = torch.arange(length, dtype=torch.float64, device=device)[:, None] * inv
    return torch.stack((angle.cos(), angle.sin()), 1).float()


def _pages(case: dict, g: torch.Generator) -> tuple[int, torch.Tensor]:
    """How many pages the cache has, and each sequence's, in any order; places that no sequence uses point at the last page."""
    per = -(-case["context"] // case["page"])
    used = case["batch"] * per
    return used + 1, torch.randperm(used, generator=g, device="cuda").view(case["batch"], per).int()


def _views(cache: torch.Tensor, dim: int) -> tuple[torch.Tensor, ...]:
    """The parts of the cache as views of it: codes of K [.., 16, dim / 2], codes of V [.., 8, dim / 4, 2 tokens, 2 bytes], the pairs
    (step, least value) of K and of V [.., 8, 2 tokens, 4 bytes]."""
    k, rows = cache.split((8 * dim, 8 * dim + 128), -1)
    v, pairs = rows.unflatten(-1, (8, dim + 16)).split((dim, 16), -1)
    pairs = pairs.unflatten(-1, (2, 2, 4))
    return k.unflatten(-1, (BLOCK, dim // 2)), v.unflatten(-1, (dim // 4, 2, 2)), pairs[..., 0, :], pairs[..., 1, :]


def _quantised(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Codes (uint8 in 0..15) and the pair (step, least value) of the last axis."""
    low, high = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    span = high - low
    fine = span.isfinite()
    nan = torch.full_like(span, math.nan)
    pair = torch.cat((torch.where(fine, span * (1.0 / 15.0), nan), torch.where(fine, low, nan)), -1).bfloat16()
    step, least = pair.to(x.dtype).split(1, -1)
    inverse = torch.where(step >= LEAST_STEP, step.reciprocal(), torch.zeros_like(step))
    codes = ((x - least) * inverse).round().clamp(0, 15).nan_to_num(0.0).to(torch.uint8)
    pair = torch.where((pair[..., :1] < LEAST_STEP) & (torch.arange(2, device=x.device) == 0), torch.zeros_like(pair), pair)
    return codes, pair


def _filled(pages: int, case: dict, g: torch.Generator) -> torch.Tensor:
    """A cache whose blocks hold keys with a few large dimensions and values, both as rotation and projection leave them."""
    h, d, nb = case["kv_heads"], case["dim"], case["page"] // BLOCK
    cache = torch.empty(pages, h, nb, BLOCK * (d + 8), dtype=torch.uint8, device="cuda")
    large = 1.0 + 3.0 * (torch.rand(h, 1, 1, d, generator=g, device="cuda") < 0.05)
    piece = max(1, int(5e7 / (h * nb * BLOCK * d)))
    for at in range(0, pages, piece):
        ck, cv, pk, pv = _views(cache[at : at + piece], d)
        n = ck.shape[0]
        codes, pair = _quantised(torch.randn(n, h, nb, BLOCK, d, generator=g, device="cuda") * large)
        ck.copy_(codes[..., 0::2] | codes[..., 1::2] << 4)
        pk.copy_(pair.view(torch.uint8).unflatten(-2, (8, 2)))
        size = torch.exp(0.5 * torch.randn(n, h, nb, BLOCK, 1, generator=g, device="cuda"))
        codes, pair = _quantised(torch.randn(n, h, nb, BLOCK, d, generator=g, device="cuda") * size)
        byte = codes[..., 0::2] | codes[..., 1::2] << 4
        cv.copy_(byte.unflatten(-1, (d // 4, 2)).unflatten(-3, (8, 2)).transpose(-3, -2))
        pv.copy_(pair.view(torch.uint8).unflatten(-2, (8, 2)))
    return cache


def prepare(case: dict, seed: int) -> dict:
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype, b, d = DTYPES[case["dtype"]], case["batch"], case["dim"]

    def normal(*shape: int) -> torch.Tensor:
        return torch.randn(*shape, generator=g, device="cuda").to(dtype)

    s: dict = {"case": dict(case)}
    if case["kind"] in ("rotary", "norm"):
        n = case["tokens"]
        if n == 1:
            s["positions"] = torch.randint(0, 4096, (b, 1), generator=g, device="cuda").int()
            s["table"] = _table(4096, case["rot"], "cuda")
        else:
            at = torch.arange(n, device="cuda").int() - case["prefix"]
            s["positions"] = at.clamp(min=-1).expand(b, n).contiguous()
            s["table"] = _table(n - case["prefix"], case["rot"], "cuda")
        if case["kind"] == "rotary":
            s["x"] = normal(b, n, 3, case["heads"], d)[:, :, 0] if case["packed"] else normal(b, n, case["heads"], d)
            if case["grad"]:
                s["x"].requires_grad_(True)
                s["dy"] = normal(b, n, case["heads"], d)
            return s
        hq, hk = case["q_heads"], case["kv_heads"]
        if case["packed"]:
            s["q"], s["k"], _ = normal(b, n, 3, hq, d).unbind(2)
        else:
            s["q"], s["k"] = normal(b, n, hq, d), normal(b, n, hk, d)
        s["wq"], s["wk"] = ((1 + 0.2 * torch.randn(d, generator=g, device="cuda")).to(dtype) for _ in range(2))
        if case["grad"]:
            for name in ("q", "k", "wq", "wk"):
                s[name] = s[name].detach().requires_grad_(True)
            s["dq"], s["dk"] = normal(b, n, hq, d), normal(b, n, hk, d)
        return s
    s["lengths"] = torch.tensor(_lengths(case), dtype=torch.int32, device="cuda")[torch.randperm(b, generator=g, device="cuda")]
    pages, s["pages"] = _pages(case, g)
    if case["kind"] == "append":
        n, hq, hk = case["tokens"], case["q_heads"], case["kv_heads"]
        s["cache"] = torch.randint(0, 256, (pages, hk, case["page"] // BLOCK, BLOCK * (d + 8)), generator=g, device="cuda", dtype=torch.uint8)
        s["q"], s["k"], s["v"] = normal(b, n, (hq + 2 * hk), d).split((hq, hk, hk), 2)
        s["table"] = _table(case["context"], case["rot"], "cuda") if case["rot"] else None
        return s
    s["cache"] = _filled(pages, case, g)
    s["q"] = (1.5 * torch.randn(b, case["queries"], case["q_heads"], d, generator=g, device="cuda")).to(dtype)
    return s


# ---- plain form ------------------------------------------------------------------------------------------------------------------


def _turn(positions: torch.Tensor, table: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Cosine and sine for each token `[batch, tokens, 1, rot / 2]`; a token at a negative position is not turned."""
    cs = table[positions.clamp(min=0).long()]
    still = (positions < 0)[:, :, None]
    return torch.where(still, 1.0, cs[:, :, 0])[:, :, None], torch.where(still, 0.0, cs[:, :, 1])[:, :, None]


def _rotated(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, interleaved: bool) -> torch.Tensor:
    half = cos.shape[-1]
    if interleaved:
        a, b = x[..., 0 : 2 * half : 2], x[..., 1 : 2 * half : 2]
        y = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = x[..., :half], x[..., half : 2 * half]
        y = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((y, x[..., 2 * half :]), -1)


def _plain_rotary(s: dict) -> dict:
    x, inter = s["x"], s["case"]["interleaved"]
    with torch.no_grad():
        cos, sin = _turn(s["positions"], s["table"])
        got = {"y": _rotated(x.float(), cos, sin, inter).to(x.dtype)}
        if "dy" in s:
            got["dx"] = _rotated(s["dy"].float(), cos, -sin, inter).to(x.dtype)
    return got


def _plain_norm(s: dict) -> dict:
    inter, got = s["case"]["interleaved"], {}
    with torch.no_grad():
        cos, sin = _turn(s["positions"], s["table"])
        for name in ("q", "k"):
            x, w = s[name].float(), s["w" + name].float()
            r = (x.square().mean(-1, keepdim=True) + EPS).rsqrt()
            hat = x * r
            got[name] = _rotated(hat * w, cos, sin, inter).to(s[name].dtype)
            if "d" + name in s:
                t = _rotated(s["d" + name].float(), cos, -sin, inter)
                got["dw" + name] = (t * hat).sum((0, 1, 2)).to(s[name].dtype)
                t = t * w
                got["d" + name] = (r * (t - hat * (t * hat).mean(-1, keepdim=True))).to(s[name].dtype)
    return got


def _nibbles(byte: torch.Tensor) -> torch.Tensor:
    return torch.stack((byte & 15, byte >> 4), -1).flatten(-2)


def _values(codes: torch.Tensor, pair: torch.Tensor) -> torch.Tensor:
    step, least = pair.contiguous().view(torch.bfloat16).float().split(1, -1)
    return least + step * codes.float()


def _places(s: dict) -> tuple[torch.Tensor, ...]:
    """For the new tokens: position, page (the last one, which nothing reads, before a sequence's start), block, token in the block."""
    n, page = s["case"]["tokens"], s["case"]["page"]
    at = s["lengths"][:, None].long() - n + torch.arange(n, device="cuda")
    p = at.clamp(min=0)
    pages = torch.where(at < 0, s["cache"].shape[0] - 1, s["pages"].long().gather(1, p // page))
    return at, pages, p % page // BLOCK, p % BLOCK


def _plain_append(s: dict) -> dict:
    q, k, v, d = s["q"], s["k"], s["v"], s["case"]["dim"]
    at, page, block, token = _places(s)
    qr, kr = q.float(), k.float()
    if s["table"] is not None:
        cos, sin = _turn(at, s["table"])
        qr, kr = (_rotated(x, cos, sin, s["case"]["interleaved"]) for x in (qr, kr))
    ck, cv, pk, pv = _views(s["cache"], d)
    codes, pair = _quantised(kr)
    ck[page, :, block, token] = codes[..., 0::2] | codes[..., 1::2] << 4
    pk[page, :, block, token // 2, token % 2] = pair.view(torch.uint8)
    codes, pair = _quantised(v.float())
    cv[page, :, block, token // 2, :, token % 2] = (codes[..., 0::2] | codes[..., 1::2] << 4).unflatten(-1, (d // 4, 2))
    pv[page, :, block, token // 2, token % 2] = pair.view(torch.uint8)
    got = {"q": qr.to(q.dtype)}
    none = (at < 0)[:, :, None, None]
    held = _values(_nibbles(ck[page, :, block, token]), pk[page, :, block, token // 2, token % 2])
    got["k"] = torch.where(none, 0.0, held).to(q.dtype)
    held = _values(_nibbles(cv[page, :, block, token // 2, :, token % 2].flatten(-2)), pv[page, :, block, token // 2, token % 2])
    got["v"] = torch.where(none, 0.0, held).to(q.dtype)
    return got


def _held(cache: torch.Tensor, d: int) -> tuple[torch.Tensor, torch.Tensor]:
    """K and V of blocks `[.., blocks, heads, bytes]` as `[.., heads, 16 blocks, dim]`."""
    ck, cv, pk, pv = _views(cache, d)
    k = _values(_nibbles(ck), pk.flatten(-3, -2))
    v = _values(_nibbles(cv.transpose(-3, -2).flatten(-2)).flatten(-3, -2), pv.flatten(-3, -2))
    return tuple(x.transpose(-4, -3).flatten(-3, -2) for x in (k, v))


def _plain_attend(s: dict) -> dict:
    q, d, page = s["q"], s["case"]["dim"], s["case"]["page"]
    b, n, hq, _ = q.shape
    hk = s["case"]["kv_heads"]
    held = s["cache"][s["pages"].long()].transpose(2, 3).flatten(1, 2)  # [batch, blocks, heads, bytes]
    k, v = _held(held, d)  # [batch, heads, tokens, dim]
    del held
    there = torch.arange(k.shape[2], device="cuda") < s["lengths"][:, None]
    k, v = (torch.where(there[:, None, :, None], x, 0.0) for x in (k, v))
    rows = q.float().unflatten(2, (hk, hq // hk)).permute(0, 2, 1, 3, 4).flatten(2, 3)  # [batch, kv heads, queries x group, dim]
    logits = rows @ k.transpose(-1, -2) * d**-0.5
    last = s["lengths"][:, None] - n + torch.arange(n, device="cuda")
    sees = (torch.arange(k.shape[2], device="cuda") <= last[:, :, None]).repeat_interleave(hq // hk, 1)[:, None]
    logits = torch.where(sees, logits, -math.inf)
    most = logits.amax(-1, keepdim=True)
    p = torch.exp(logits - torch.where(most == -math.inf, 0.0, most))
    total = p.sum(-1, keepdim=True)
    o = p @ v / torch.where(total > 0, total, 1.0)
    return {"o": o.unflatten(2, (n, hq // hk)).permute(0, 2, 1, 3, 4).flatten(2, 3).to(q.dtype)}


# ---- one pass --------------------------------------------------------------------------------------------------------------------


def _own_run(s: dict) -> dict:
    import fastforks_b200 as ff  # noqa: PLC0415

    case = s["case"]
    if case["kind"] == "rotary":
        y = ff.rotary(s["x"], s["table"], s["positions"], interleaved=case["interleaved"])
        if "dy" not in s:
            return {"y": y}
        (dx,) = torch.autograd.grad(y, s["x"], s["dy"])
        return {"y": y, "dx": dx}
    if case["kind"] == "norm":
        q, k = ff.qk_norm_rotary(s["q"], s["k"], s["wq"], s["wk"], s["table"], s["positions"], eps=EPS, interleaved=case["interleaved"])
        if "dq" not in s:
            return {"q": q, "k": k}
        dq, dk, dwq, dwk = torch.autograd.grad((q, k), (s["q"], s["k"], s["wq"], s["wk"]), (s["dq"], s["dk"]))
        return {"q": q, "k": k, "dq": dq, "dk": dk, "dwq": dwq, "dwk": dwk}
    if case["kind"] == "append":
        q = ff.kv4_append_(s["cache"], s["k"], s["v"], s["pages"], s["lengths"], table=s["table"], interleaved=case["interleaved"], q=s["q"])
        k, v = ff.kv4_read(s["cache"], s["pages"], s["lengths"], case["tokens"], s["q"].dtype)
        return {"q": q, "k": k, "v": v}
    return {"o": ff.kv4_attention(s["q"], s["cache"], s["pages"], s["lengths"])}


def run(state: dict) -> dict:
    if own:
        return _own_run(state)
    return {"rotary": _plain_rotary, "norm": _plain_norm, "append": _plain_append, "attend": _plain_attend}[state["case"]["kind"]](state)


# ---- in 64 bits ------------------------------------------------------------------------------------------------------------------


def _rotation64(x: torch.Tensor, positions: torch.Tensor, table: torch.Tensor, interleaved: bool, back: bool = False) -> torch.Tensor:
    """As products of complex numbers."""
    turn = torch.complex(table[:, 0].double(), table[:, 1].double() * (-1 if back else 1))
    turn = torch.cat((turn, torch.ones_like(turn[:1])))[torch.where(positions < 0, table.shape[0], positions.long())][:, :, None]
    half = turn.shape[-1]
    head = x[..., : 2 * half].unflatten(-1, (half, 2) if interleaved else (2, half))
    z = torch.view_as_complex((head if interleaved else head.transpose(-1, -2)).contiguous()) * turn
    z = torch.view_as_real(z)
    return torch.cat(((z if interleaved else z.transpose(-1, -2)).flatten(-2), x[..., 2 * half :]), -1)


def _decoded64(blocks: torch.Tensor, d: int) -> tuple[torch.Tensor, torch.Tensor]:
    """K and V `[heads, tokens, dim]` of blocks `[blocks, heads, bytes]`, each code fetched by the place of its byte."""
    t, x = torch.arange(BLOCK, device="cuda")[:, None], torch.arange(d, device="cuda")
    got = []
    row = 8 * d + t // 2 * (d + 16)
    for byte, pair in ((t * (d // 2) + x // 2, 0), (row + x // 4 * 4 + t % 2 * 2 + x % 4 // 2, 4)):
        code = (blocks[..., byte] >> (4 * (x % 2))) & 15
        word = blocks[..., row + d + t % 2 * 8 + pair + torch.arange(4, device="cuda")].to(torch.int32)
        step, least = ((word[..., i] << 16 | word[..., i + 1] << 24).view(torch.float32).double()[..., None] for i in (0, 2))
        got.append((code.double() * step + least).transpose(0, 1).flatten(1, 2))
    return got[0], got[1]


def _exact_attend(s: dict) -> dict:
    q, d, page, hk = s["q"], s["case"]["dim"], s["case"]["page"], s["case"]["kv_heads"]
    n, group = q.shape[1], q.shape[2] // hk
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    for b, length in enumerate(s["lengths"].tolist()):
        if not length:
            continue
        blocks = s["cache"][s["pages"][b, : -(-length // page)].long()].transpose(1, 2).flatten(0, 1)
        k, v = (x[:, :length] for x in _decoded64(blocks, d))
        for at in range(0, n, 64):  # a few queries at a time: the logits of all would not fit beside the rest
            x = q[b, at : at + 64].double().unflatten(1, (hk, group))
            logits = torch.einsum("nhgd,htd->nhgt", x, k) / math.sqrt(d)
            last = length - n + torch.arange(at, at + x.shape[0], device="cuda")
            hidden = torch.arange(length, device="cuda") > last[:, None, None, None]
            o = torch.einsum("nhgt,htd->nhgd", torch.softmax(logits.masked_fill(hidden, -math.inf), -1), v)
            out[b, at : at + 64] = torch.where(last[:, None, None, None] < 0, 0.0, o).flatten(1, 2)
    return {"o": out}


def exact(case: dict, seed: int) -> dict | None:
    s = prepare(case, seed)
    inter = case["interleaved"] if "interleaved" in case else False
    with torch.no_grad():
        if case["kind"] == "rotary":
            got = {"y": _rotation64(s["x"].double(), s["positions"], s["table"], inter)}
            if "dy" in s:
                got["dx"] = _rotation64(s["dy"].double(), s["positions"], s["table"], inter, back=True)
            return got
        if case["kind"] == "norm":
            got = {}
            for name in ("q", "k"):
                x, w = s[name].double(), s["w" + name].double()
                size = torch.sqrt(x.pow(2).sum(-1, keepdim=True) / x.shape[-1] + EPS)
                got[name] = _rotation64(x / size * w, s["positions"], s["table"], inter)
                if "d" + name in s:
                    t = _rotation64(s["d" + name].double(), s["positions"], s["table"], inter, back=True)
                    got["dw" + name] = torch.einsum("bnhd,bnhd->d", t, x / size)
                    along = torch.einsum("bnhd,bnhd->bnh", t * w, x)[..., None]
                    got["d" + name] = t * w / size - x * along / (x.shape[-1] * size**3)
            return got
        if case["kind"] == "append":
            n = case["tokens"]
            at = s["lengths"][:, None].long() - n + torch.arange(n, device="cuda")
            q, k, v = (s[name].double() for name in ("q", "k", "v"))
            if s["table"] is not None:
                q, k = (_rotation64(x, at.clamp(min=-1), s["table"], inter) for x in (q, k))
            none = (at < 0)[:, :, None, None]
            held = {}
            for name, x in (("k", k), ("v", v)):
                low, high = x.min(-1, keepdim=True).values, x.max(-1, keepdim=True).values
                least, step = low.bfloat16().double(), ((high - low) / 15).bfloat16().double()
                code = torch.clamp(torch.round((x - least) / step), 0, 15)
                held[name] = torch.where(none, 0.0, torch.where(step > 0, least + step * code, least))
            return {"q": q, **held}
        return _exact_attend(s)
