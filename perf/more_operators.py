"""What stands between a model's last block and its gradients, in plain form and by the framework's entry points, and the cases it is timed on.

Kinds of case:

* `norm`: layer norm of rows (`layer_norm`), forward, or forward and the gradients of the rows, the weight and the bias;
* `ce`: softmax cross entropy of an output layer, from hidden states and the layer's weight (`linear_cross_entropy`), forward, or forward
  and the gradients of hidden states and weight;
* `kd`: the divergence of that output layer's distribution from a teacher's, of which the largest logits of each token are known
  (`linear_distillation`), forward, or forward and the same gradients.

Rows of `ce` whose target is -100 and entries of `kd` whose token is -1 do not count; a row without an entry is as one without a target. `mean`
is over the rows that count (0 where none does); `none` gives a loss per row, and its gradient comes with a weight of each row.
"""

from __future__ import annotations

import math

import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
BYTES = {"fp16": 2, "bf16": 2, "fp32": 4}
EPS = 1e-5
IGNORED = -100


def listed() -> list[dict]:
    return [
        # One 224 px image's tokens in an encoder of twelve heads: latency.
        {"name": "norm-197x768", "kind": "norm", "rows": 197, "dim": 768, "grad": False, "affine": True, "dtype": "fp16"},
        # Sixteen 518 px images in a large encoder: every block does this twice.
        {"name": "norm-21920x1024", "kind": "norm", "rows": 21920, "dim": 1024, "grad": False, "affine": True, "dtype": "bf16"},
        # A training step of a decoder, two sequences of 4096 tokens.
        {"name": "norm-train-8192x4096", "kind": "norm", "rows": 8192, "dim": 4096, "grad": True, "affine": True, "dtype": "bf16"},
        # Fine-tuning of a small encoder in 32 bits, ragged token count.
        {"name": "norm-train-5480x384", "kind": "norm", "rows": 5480, "dim": 384, "grad": True, "affine": True, "dtype": "fp32"},
        # A classifier's head behind an image encoder, 256 images a step: the smallest training call.
        {"name": "ce-train-256x1000x768", "kind": "ce", "rows": 256, "vocab": 1000, "dim": 768, "grad": True, "reduction": "mean", "ignored": 0.0, "dtype": "fp16"},
        # A server scores sixty-four tokens: no gradient, the weight is what is read.
        {"name": "ce-64x32000x4096", "kind": "ce", "rows": 64, "vocab": 32000, "dim": 4096, "grad": False, "reduction": "none", "ignored": 0.0, "dtype": "bf16"},
        # Odd counts of rows and of tokens in the vocabulary, weights of each row (advantages of a policy), a tenth of the rows padding.
        {"name": "ce-train-2047x50001x1024", "kind": "ce", "rows": 2047, "vocab": 50001, "dim": 1024, "grad": True, "reduction": "none", "ignored": 0.1, "dtype": "fp16"},
        # A training step on 4096 tokens over a large vocabulary.
        {"name": "ce-train-4096x128000x4096", "kind": "ce", "rows": 4096, "vocab": 128000, "dim": 4096, "grad": True, "reduction": "mean", "ignored": 0.02, "dtype": "bf16"},
        # A short validation batch of a distilled model: divergence alone, twenty logits a token.
        {"name": "kd-130x32000x1024", "kind": "kd", "rows": 130, "vocab": 32000, "dim": 1024, "top": 20, "temperature": 1.0, "grad": False, "reduction": "none", "ignored": 0.0, "dtype": "fp16"},
        # A step of distillation of a small model, few tokens.
        {"name": "kd-train-500x16001x512", "kind": "kd", "rows": 500, "vocab": 16001, "dim": 512, "top": 7, "temperature": 1.0, "grad": True, "reduction": "mean", "ignored": 0.1, "dtype": "bf16"},
        # A step of distillation over 64 logits a token, softened, prompts masked.
        {"name": "kd-train-4096x64000x2048", "kind": "kd", "rows": 4096, "vocab": 64000, "dim": 2048, "top": 64, "temperature": 2.0, "grad": True, "reduction": "mean", "ignored": 0.25, "dtype": "bf16"},
    ]


def _log_int(rng, low: int, high: int) -> int:
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(max(low, high)))))))


def draw(rng) -> dict:
    kind = rng.choice(["norm", "ce", "ce", "kd"])
    if kind == "norm":
        dim = rng.choice([64, 192, 384, 768, 1024, 1280, 2048, 4096, 8192, _log_int(rng, 1, 10000), 8 * _log_int(rng, 8, 1250)])
        rows = 1 if rng.random() < 0.1 else _log_int(rng, 1, max(1, min(65536, 2**25 // dim)))
        return {"kind": kind, "rows": rows, "dim": dim, "grad": rng.random() < 0.6, "affine": rng.random() < 0.85, "dtype": rng.choice(["fp16", "bf16", "bf16", "fp32"])}
    dim = rng.choice([64, 128, 384, 512, 768, 1024, 2048, 4096, 8 * _log_int(rng, 4, 512)])
    vocab = _log_int(rng, 10, 128000)
    rows = 1 if rng.random() < 0.1 else _log_int(rng, 2, max(2, min(8192, int(4096 * 128000 * 4096 / (vocab * max(dim, 512)) / 2))))
    case = {"kind": kind, "rows": rows, "vocab": vocab, "dim": dim}
    if kind == "kd":
        case |= {"top": min(_log_int(rng, 1, 128), max(1, vocab // 4)), "temperature": rng.choice([1.0, 1.0, 2.0, 0.7, 4.0])}
    return case | {"grad": rng.random() < 0.6, "reduction": rng.choice(["mean", "none"]), "ignored": rng.choice([0.0, 0.0, 0.1, 0.5]), "dtype": rng.choice(["fp16", "bf16"])}


def work(case: dict) -> dict:
    e, t, d = BYTES[case["dtype"]], case["rows"], case["dim"]
    if case["kind"] == "norm":
        ends = (2 if case["affine"] else 0) * d * e
        return {"bytes": (4 if case["grad"] else 2) * t * d * e + (2 if case["grad"] else 1) * ends, "flops": (20 if case["grad"] else 8) * t * d}
    v = case["vocab"]
    entries = 8 * t if case["kind"] == "ce" else 12 * t * case["top"]
    # forward: the logits' product; gradients: the two products that logits' gradients go into
    return {"bytes": (2 if case["grad"] else 1) * (t + v) * d * e + entries + 4 * t, "flops": (6 if case["grad"] else 2) * t * d * v}


# ---- inputs ----------------------------------------------------------------------------------------------------------------------


def prepare(case: dict, seed: int) -> dict:
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype, t, d = DTYPES[case["dtype"]], case["rows"], case["dim"]

    def normal(*shape: int) -> torch.Tensor:
        return torch.randn(*shape, generator=g, device="cuda")

    s: dict = {"case": dict(case)}
    if case["kind"] == "norm":
        # a residual stream: a few large channels, rows of different sizes
        large = 1.0 + 8.0 * (torch.rand(d, generator=g, device="cuda") < 0.01)
        s["x"] = ((normal(t, d) + 0.3 * normal(d)) * large * torch.exp(0.4 * normal(t, 1))).to(dtype)
        s["w"] = (1 + 0.2 * normal(d)).to(dtype) if case["affine"] else None
        s["b"] = (0.1 * normal(d)).to(dtype) if case["affine"] else None
        if case["grad"]:
            s["dy"] = normal(t, d).to(dtype)
    else:
        v = case["vocab"]
        s["w"] = (normal(v, d) * (1.6 / math.sqrt(d))).to(dtype)
        targets = torch.randint(0, v, (t,), generator=g, device="cuda")
        # normed hidden states that know their target, some better than others
        lean = 9.0 * torch.rand(t, 1, generator=g, device="cuda") / 1.6**2
        s["x"] = (normal(t, d) + lean * s["w"][targets].float()).to(dtype)
        out = torch.rand(t, generator=g, device="cuda") < case["ignored"]
        if case["kind"] == "ce":
            s["targets"] = torch.where(out, IGNORED, targets)
        else:
            k = case["top"]
            # tokens apart by gaps of all sizes, in any order, the target first; logits fall with the rank; some rows know fewer
            gaps = torch.exp(1.5 * normal(t, k)) * (v / (8 * k))
            step = (1 + gaps.long()).clamp(max=max(1, (v - 1) // k))
            ids = (targets[:, None] + torch.cat((torch.zeros_like(step[:, :1]), step[:, 1:].cumsum(1)), 1)) % v
            order = torch.cat((torch.full((t, 1), -1.0, device="cuda"), torch.rand(t, k - 1, generator=g, device="cuda")), 1).argsort(1)
            known = (k * (0.5 + torch.rand(t, 1, generator=g, device="cuda"))).ceil()
            gone = (torch.arange(k, device="cuda") >= known) | out[:, None]
            s["ids"] = torch.where(gone, -1, ids.gather(1, order))
            s["teacher"] = (12.0 + 2.5 * normal(t, k)).sort(1, descending=True).values
        if case["grad"] and case["reduction"] == "none":
            s["dloss"] = normal(t)
    if case["grad"]:
        for name in ("x", "w", "b"):
            if s.get(name) is not None:
                s[name].requires_grad_(True)
    return s


# ---- plain form ------------------------------------------------------------------------------------------------------------------


def _plain_norm(s: dict) -> dict:
    x, w, b = s["x"], s["w"], s["b"]
    xf = x.float()
    centred = xf - xf.mean(-1, keepdim=True)
    r = (centred.square().mean(-1, keepdim=True) + EPS).rsqrt()
    hat = centred * r
    y = hat if w is None else hat * w.float() + b.float()
    got = {"y": y.to(x.dtype)}
    if "dy" in s:
        t = s["dy"].float()
        if w is not None:
            got["dw"], got["db"] = (t * hat).sum(0).to(w.dtype), t.sum(0).to(b.dtype)
            t = t * w.float()
        got["dx"] = (r * (t - t.mean(-1, keepdim=True) - hat * (t * hat).mean(-1, keepdim=True))).to(x.dtype)
    return got


def _plain_loss(s: dict) -> dict:
    case, x, w = s["case"], s["x"], s["w"]
    xf, wf = x.float(), w.float()
    logits = xf @ wf.t()
    if case["kind"] == "ce":
        tau, counts = 1.0, s["targets"] != IGNORED
        ids, p = torch.where(counts, s["targets"], 0)[:, None], counts.float()[:, None]
        entropy = torch.zeros_like(p)
    else:
        tau, there = case["temperature"], s["ids"] >= 0
        ids, counts = s["ids"].clamp(min=0), there.any(1)
        z = torch.where(there, s["teacher"] / tau, -math.inf)
        p = torch.exp(z - torch.where(counts[:, None], z.amax(1, keepdim=True), 0.0))
        p = p / torch.where(counts[:, None], p.sum(1, keepdim=True), 1.0)
        entropy = torch.where(p > 0, p * torch.log(torch.where(p > 0, p, 1.0)), 0.0)
    logits = logits / tau
    most = logits.amax(1, keepdim=True)
    q = torch.exp(logits - most)
    total = q.sum(1, keepdim=True)
    lse = most + torch.log(total)
    loss = tau * tau * (entropy - p * (logits.gather(1, ids) - lse)).sum(1)
    del logits
    n = counts.sum().clamp(min=1)
    got = {"loss": loss if case["reduction"] == "none" else loss.sum() / n}
    if case["grad"]:
        size = tau * (s["dloss"] if case["reduction"] == "none" else (1.0 / n).expand(loss.shape)) * counts
        q *= (size[:, None] * p.sum(1, keepdim=True)) / total
        q.scatter_add_(1, ids, -size[:, None] * p)
        got |= {"dx": (q @ wf).to(x.dtype), "dw": (q.t() @ xf).to(w.dtype)}
    return got


# ---- one pass --------------------------------------------------------------------------------------------------------------------


def _own_run(s: dict) -> dict:
    import fastforks_b200 as ff  # noqa: PLC0415

    case = s["case"]
    if case["kind"] == "norm":
        y = ff.layer_norm(s["x"], s["w"], s["b"], eps=EPS)
        if "dy" not in s:
            return {"y": y}
        if s["w"] is None:
            (dx,) = torch.autograd.grad(y, s["x"], s["dy"])
            return {"y": y, "dx": dx}
        dx, dw, db = torch.autograd.grad(y, (s["x"], s["w"], s["b"]), s["dy"])
        return {"y": y, "dx": dx, "dw": dw, "db": db}
    if case["kind"] == "ce":
        loss = ff.linear_cross_entropy(s["x"], s["w"], s["targets"], ignore_index=IGNORED, reduction=case["reduction"])
    else:
        loss = ff.linear_distillation(s["x"], s["w"], s["ids"], s["teacher"], temperature=case["temperature"], reduction=case["reduction"])
    if not case["grad"]:
        return {"loss": loss}
    dx, dw = torch.autograd.grad(loss, (s["x"], s["w"]), s.get("dloss"))
    return {"loss": loss, "dx": dx, "dw": dw}


def run(state: dict) -> dict:
    if own:
        return _own_run(state)
    with torch.no_grad():
        return _plain_norm(state) if state["case"]["kind"] == "norm" else _plain_loss(state)


# ---- in 64 bits ------------------------------------------------------------------------------------------------------------------


def _exact_norm(s: dict) -> dict:
    x = s["x"].double()
    w, b = (None if s[k] is None else s[k].double() for k in ("w", "b"))
    n = x.shape[-1]
    mean = x.sum(-1, keepdim=True) / n
    deviation = torch.sqrt(((x - mean) ** 2).sum(-1, keepdim=True) / n + EPS)
    hat = (x - mean) / deviation
    got = {"y": hat if w is None else torch.addcmul(b, hat, w)}
    if "dy" in s:
        dy = s["dy"].double()
        if w is not None:
            got["dw"], got["db"] = torch.einsum("td,td->d", dy, hat), torch.einsum("td->d", dy)
        dhat = dy if w is None else dy * w
        # through the deviation and through the mean, one after the other
        ddeviation = -torch.einsum("td,td->t", dhat, hat)[:, None] / deviation
        dcentred = dhat / deviation + ddeviation * (x - mean) / (n * deviation)
        got["dx"] = dcentred - dcentred.sum(-1, keepdim=True) / n
    return got


def _exact_loss(s: dict) -> dict:
    case = s["case"]
    x, w = s["x"].double(), s["w"].double()
    t, v = x.shape[0], w.shape[0]
    tau = case.get("temperature", 1.0)
    logq = torch.log_softmax(torch.einsum("td,vd->tv", x, w) / tau, 1)
    rows = torch.arange(t, device=x.device)
    if case["kind"] == "ce":
        counts = s["targets"] >= 0
        loss = torch.where(counts, -logq[rows, s["targets"].clamp(min=0)], 0.0)
    else:
        counts = (s["ids"] >= 0).sum(1) > 0
        logp = torch.log_softmax((s["teacher"].double() / tau).masked_fill(s["ids"] < 0, -1e300), 1)
        p = torch.where((s["ids"] >= 0) & counts[:, None], logp.exp(), 0.0)
        loss = tau**2 * torch.einsum("tk,tk->t", p, logp.clamp(min=-1e30) - logq.gather(1, s["ids"].clamp(min=0)))
    n = max(1, int(counts.sum()))
    got = {"loss": loss if case["reduction"] == "none" else loss.sum() / n}
    if case["grad"]:
        size = torch.where(counts, s["dloss"].double() if case["reduction"] == "none" else torch.full((t,), 1.0 / n, device=x.device, dtype=torch.float64), 0.0) * tau
        dl = logq.exp_()
        if case["kind"] == "ce":
            dl[rows[counts], s["targets"][counts]] -= 1.0
        else:
            at = rows[:, None].expand_as(s["ids"])
            dl.view(-1).index_add_(0, (at * v + s["ids"].clamp(min=0)).reshape(-1), -p.reshape(-1))
        dl *= size[:, None]
        got |= {"dx": torch.einsum("tv,vd->td", dl, w), "dw": torch.einsum("tv,td->vd", dl, x)}
    return got


def exact(case: dict, seed: int) -> dict | None:
    s = prepare(case, seed)
    with torch.no_grad():
        return _exact_norm(s) if case["kind"] == "norm" else _exact_loss(s)
