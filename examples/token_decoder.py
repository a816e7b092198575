"""A small token decoder on the framework's operators: a prompt in pieces, then token by token from a captured graph, and gradient steps.

    python examples/token_decoder.py [--layers 2] [--batch 4] [--prompt 100] [--steps 16]

Each layer is `gemm` (qkv), positions, the 4-bit cache, attention over it and `gemm` again; its queries and keys are normed
(`qk_norm_rotary`) in every other layer and only turned on their way into the cache (`kv4_append_`) in the rest. Weights are random: what
is shown is how the calls go together, and that pieces, single tokens and a replayed graph agree. The last parts take a step of gradient descent on
the norms' weights through `qk_norm_rotary` and `rotary`, and one on the last norm and the output layer (`layer_norm`, `linear_cross_entropy`,
`linear_distillation`).
"""

from __future__ import annotations

import argparse
import dataclasses
import math
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))

import fastforks_b200 as ff


@dataclasses.dataclass
class Config:
    layers: int = 2
    dim: int = 512
    q_heads: int = 8
    kv_heads: int = 2
    head_dim: int = 64
    hidden: int = 1024
    context: int = 256
    page: int = 32
    dtype: torch.dtype = torch.bfloat16


class Decoder:
    """Layers with a 4-bit cache; sequences get their pages when they are made."""

    def __init__(self, cfg: Config, batch: int, *, seed: int = 0) -> None:
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.cfg, self.batch = cfg, batch

        def weight(n: int, k: int) -> torch.Tensor:
            return (torch.randn(n, k, generator=g, device="cuda") / math.sqrt(k)).to(cfg.dtype)

        heads = cfg.q_heads + 2 * cfg.kv_heads
        self.layers = [
            {
                "qkv": weight(heads * cfg.head_dim, cfg.dim),
                "proj": weight(cfg.dim, cfg.q_heads * cfg.head_dim),
                "up": weight(cfg.hidden, cfg.dim),
                "down": weight(cfg.dim, cfg.hidden),
                "norms": [torch.ones(cfg.head_dim, device="cuda", dtype=cfg.dtype) for _ in range(2)] if i % 2 == 0 else None,
            }
            for i in range(cfg.layers)
        ]
        columns = -(-cfg.context // cfg.page)
        self.pages = torch.randperm(batch * columns, generator=g, device="cuda").view(batch, columns).int()
        self.caches = [ff.kv4_cache(batch * columns, cfg.kv_heads, cfg.head_dim, page=cfg.page) for _ in range(cfg.layers)]
        # positions stretched to twice the length that the frequencies were made for
        self.table = ff.rotary_table(cfg.context, cfg.head_dim, scaling="yarn", factor=2.0, original_length=cfg.context // 2, device="cuda")
        self.lengths = torch.zeros(batch, dtype=torch.int32, device="cuda")

    @torch.no_grad()
    def __call__(self, x: torch.Tensor) -> torch.Tensor:
        """The next tokens `[batch, tokens, dim]`; `lengths` counts them already."""
        c = self.cfg
        b, n, _ = x.shape
        at = self.lengths[:, None] - n + torch.arange(n, device="cuda", dtype=torch.int32)
        for layer, cache in zip(self.layers, self.caches, strict=True):
            qkv = ff.gemm(x, layer["qkv"]).view(b, n, -1, c.head_dim)
            q, k, v = qkv.split((c.q_heads, c.kv_heads, c.kv_heads), 2)
            if layer["norms"] is not None:
                q, k = ff.qk_norm_rotary(q, k, *layer["norms"], self.table, at)
                ff.kv4_append_(cache, k, v, self.pages, self.lengths)
            else:
                q = ff.kv4_append_(cache, k, v, self.pages, self.lengths, table=self.table, q=q)
            o = ff.kv4_attention(q, cache, self.pages, self.lengths)
            x = ff.gemm(o.view(b, n, -1), layer["proj"], res=x)
            x = ff.gemm(ff.gemm(x, layer["up"], act=ff.ACT_GELU), layer["down"], res=x)
        return x

    def extend(self, x: torch.Tensor) -> torch.Tensor:
        self.lengths += x.shape[1]
        return self(x)


def decode(cfg: Config, batch: int, prompt: int, steps: int) -> float:
    """The largest relative difference between tokens one at a time from a graph and all of them at once."""
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(batch, prompt + steps, cfg.dim, generator=g, device="cuda").to(cfg.dtype)
    whole = Decoder(cfg, batch).extend(x)[:, prompt:]

    model = Decoder(cfg, batch)
    half = prompt // 2
    model.extend(x[:, :half].contiguous())  # the prompt in two pieces
    model.extend(x[:, half:prompt].contiguous())
    token = x[:, prompt : prompt + 1].clone()
    model.lengths += 1
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        model(token)  # warm; writes the first token, as its replay will
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        out = model(token)
    got = []
    for i in range(steps):  # a replay follows the lengths, which are on the device
        token.copy_(x[:, prompt + i : prompt + i + 1])
        graph.replay()
        got.append(out.clone())
        model.lengths += 1
    diff = torch.cat(got, 1).float() - whole.float()
    return float(diff.norm() / whole.float().norm())


def learn(cfg: Config) -> tuple[float, float]:
    """One step of gradient descent on the norms' weights: the loss before and after."""
    g = torch.Generator(device="cuda").manual_seed(2)
    b, n = 2, 48
    q, k, v = (torch.randn(b, n, h, cfg.head_dim, generator=g, device="cuda") for h in (cfg.q_heads, cfg.kv_heads, cfg.kv_heads))
    target = torch.randn(b, n, cfg.q_heads, cfg.head_dim, generator=g, device="cuda")
    weights = [torch.ones(cfg.head_dim, device="cuda", requires_grad=True) for _ in range(2)]
    table = ff.rotary_table(n, cfg.head_dim, device="cuda")

    def loss() -> torch.Tensor:
        nq, nk = ff.qk_norm_rotary(q, k, *weights, table)
        keys, values = (t.repeat_interleave(cfg.q_heads // cfg.kv_heads, 2) for t in (nk, ff.rotary(v, table)))
        logits = torch.einsum("bnhd,bmhd->bhnm", nq, keys) / math.sqrt(cfg.head_dim)
        logits = logits.masked_fill(torch.ones(n, n, dtype=torch.bool, device="cuda").triu(1), -math.inf)
        o = torch.einsum("bhnm,bmhd->bnhd", logits.softmax(-1), values)
        return (o - target).square().mean()

    before = loss()
    grads = torch.autograd.grad(before, weights)
    with torch.no_grad():
        size = sum(float(d.square().sum()) for d in grads)
        for w, d in zip(weights, grads, strict=True):
            w -= 1e-3 / size * d  # the loss falls by 1e-3, to first order
    return float(before.detach()), float(loss().detach())


def output_layer(cfg: Config, batch: int, tokens: int, vocabulary: int) -> dict[str, torch.Tensor]:
    """The decoder's last states normed and scored against the next tokens and, half as much, against a teacher's eight largest logits: the loss and
    its gradients for the norm and the output layer. The first tokens of each sequence are a prompt, which does not count."""
    g = torch.Generator(device="cuda").manual_seed(3)
    with torch.no_grad():
        states = Decoder(cfg, batch).extend(torch.randn(batch, tokens, cfg.dim, generator=g, device="cuda").to(cfg.dtype))
    weights = {
        "norm": torch.ones(cfg.dim, device="cuda", dtype=cfg.dtype),
        "shift": torch.zeros(cfg.dim, device="cuda", dtype=cfg.dtype),
        "head": (torch.randn(vocabulary, cfg.dim, generator=g, device="cuda") / math.sqrt(cfg.dim)).to(cfg.dtype),
    }
    targets = torch.randint(0, vocabulary, (batch, tokens), generator=g, device="cuda")
    teacher_ids = torch.randint(0, vocabulary, (batch, tokens, 8), generator=g, device="cuda")
    teacher_ids[..., 0] = targets
    teacher_logits = torch.randn(batch, tokens, 8, generator=g, device="cuda").sort(-1, descending=True).values
    targets[:, : tokens // 3], teacher_ids[:, : tokens // 3] = -100, -1
    leaves = {name: w.requires_grad_(True) for name, w in weights.items()}
    x = ff.layer_norm(states, leaves["norm"], leaves["shift"])
    loss = ff.linear_cross_entropy(x, leaves["head"], targets) + 0.5 * ff.linear_distillation(x, leaves["head"], teacher_ids, teacher_logits, temperature=2.0)
    grads = torch.autograd.grad(loss, list(leaves.values()))
    return {"loss": loss.detach(), "states": states, "targets": targets, "teacher_ids": teacher_ids, "teacher_logits": teacher_logits,
            **weights, **{f"d{name}": d for name, d in zip(leaves, grads, strict=True)}}  # fmt: skip


def main() -> None:
    p = argparse.ArgumentParser()
    for name, default in (("layers", 2), ("batch", 4), ("prompt", 100), ("steps", 16)):
        p.add_argument(f"--{name}", type=int, default=default)
    a = p.parse_args()
    cfg = Config(layers=a.layers, context=max(256, 2 * (a.prompt + a.steps)))
    print(f"tokens from a replayed graph against all at once: relative difference {decode(cfg, a.batch, a.prompt, a.steps):.2e}")
    before, after = learn(cfg)
    print(f"a gradient step on the norms' weights: loss {before:.6f} -> {after:.6f}")
    step = output_layer(cfg, a.batch, a.prompt, 1000)
    sizes = ", ".join(f"{name} {float(step['d' + name].float().norm()):.3f}" for name in ("norm", "shift", "head"))
    print(f"the output layer's loss {float(step['loss']):.4f}, gradients' norms: {sizes}")
    status = ff.device_status()
    if status:
        sys.exit(f"device status {status}")


if __name__ == "__main__":
    main()
