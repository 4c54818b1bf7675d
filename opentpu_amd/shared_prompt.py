"""Decoding a batch of sequences that share a prompt: a stack of decoder layers whose linears are `mxu.dot`'s,
with `mxu.norm_quantize` in front of them, `attention.shared` between them and `attention.evict` on the
sequences' caches.

    python -m opentpu_amd.shared_prompt --batch 64 --prompt 4096 --tokens 96 --slots 64 --budget 48

runs random weights of Qwen3-0.6B's shape and prints the time of a step.  The prompt goes through the layers
once; its keys and values are every sequence's prefix.  A sequence's own tokens have `slots` places a layer:
when they are full, each head keeps the `budget` tokens that drew the most attention (the `recent` newest
among them)."""
from __future__ import annotations

from dataclasses import dataclass

import numpy as np

from . import _lib as X
from . import attention, mxu
from .chain import down_chunk


@dataclass
class Shape:
    """A decoder's sizes (the default: Qwen3-0.6B's, with fewer layers)."""
    hidden: int = 1024
    heads: int = 16
    kv_heads: int = 8
    head: int = 128
    F: int = 3072
    layers: int = 4
    theta: float = 1e6
    eps: float = 1e-6


@dataclass
class Layer:
    """A layer's norm weights (float32 [hidden], [hidden], [head], [head]) and its linears."""
    norm: object
    norm_mlp: object
    norm_q: object
    norm_k: object
    qkv: mxu.QWeight
    o: mxu.QWeight
    gu: mxu.QWeight
    down: mxu.QWeight


def random_layers(shape: Shape, fmt: str = "int4", seed: int = 0) -> list:
    T, s = X.torch(), shape
    g = T.Generator("cuda").manual_seed(seed)

    def w(n, k):
        return mxu.QWeight.from_float(T.randn((n, k), generator=g, device="cuda") * k ** -0.5, fmt)

    def ones(n):
        return 1 + 0.1 * T.randn((n,), generator=g, device="cuda")

    q, kv = s.heads * s.head, s.kv_heads * s.head
    return [Layer(ones(s.hidden), ones(s.hidden), ones(s.head), ones(s.head), w(q + 2 * kv, s.hidden), w(s.hidden, q),
                  w(2 * s.F, s.hidden), w(s.hidden, s.F)) for _ in range(s.layers)]


class Cache:
    """A layer's own tokens: keys, values, accumulated attention weights and positions in `slots` places."""

    def __init__(self, B: int, slots: int, shape: Shape, dtype):
        T, h = X.torch(), shape.kv_heads
        self.k = T.empty((B, slots, h, shape.head), dtype=dtype, device="cuda")
        self.v = T.empty_like(self.k)
        self.weights = T.zeros((B, h, slots), dtype=T.float32, device="cuda")
        self.pos = T.full((B, h, slots), -1, dtype=T.int32, device="cuda")


class Batch:
    """B sequences after a shared prompt [P, hidden] (float32 embeddings; P may be 0)."""

    def __init__(self, layers: list, shape: Shape, prompt, B: int, slots: int, budget: int, recent: int = 0, dtype=None):
        if not 0 <= recent <= budget < slots:
            raise ValueError(f"Batch: budget {budget} of {slots} slots, the {recent} newest kept")
        T = X.torch()
        self.layers, self.shape, self.dtype = layers, shape, dtype or T.bfloat16
        self.B, self.slots, self.budget, self.recent = B, slots, budget, recent
        self.chunks = [down_chunk(shape.F, layer.down.fmt) for layer in layers]
        self.caches = [Cache(B, slots, shape, self.dtype) for _ in layers]
        self.lens = T.zeros((B,), dtype=T.int32, device="cuda")
        self.used = 0                                      # what lens holds
        self.P = self.position = prompt.shape[0]           # the prompt's tokens, the next token's position
        self.prefix = [(None, None)] * len(layers)
        if self.P:
            n = T.full((1,), self.P, dtype=T.int32, device="cuda")
            own = []

            def attend(i, q, k, v):                        # the prompt is its own sequence
                own.append((k[0], v[0]))
                return attention.shared(q, None, None, k, v, n)

            self.prompt_out = self._run(prompt.view(1, self.P, -1), 0, attend)[0]
            self.prefix = own

    def _rope(self, x, at: int):
        """x [B, L, heads, head] float32 of tokens at positions at, at + 1, .. turned by them."""
        T = X.torch()
        half = x.shape[-1] // 2
        turn = T.arange(at, at + x.shape[1], device="cuda", dtype=T.float32)[:, None, None] * \
            self.shape.theta ** (-T.arange(half, device="cuda", dtype=T.float32) / half)
        c, s = turn.cos(), turn.sin()
        a, b = x[..., :half], x[..., half:]
        return T.cat([a * c - b * s, b * c + a * s], -1)

    def _norm_head(self, x, gamma):
        return x * X.torch().rsqrt((x * x).mean(-1, keepdim=True) + self.shape.eps) * gamma

    def _run(self, x, at: int, attend):
        """x [B, L, hidden] through the layers; attend(layer, q, k, v) -> the attention's output."""
        T, s = X.torch(), self.shape
        B, L, _ = x.shape
        nq, nkv = s.heads * s.head, s.kv_heads * s.head
        h, y = None, x.reshape(B * L, s.hidden)
        for i, layer in enumerate(self.layers):
            op, h = mxu.norm_quantize(y, layer.norm, h, eps=s.eps)
            q, k, v = mxu.dot(op, layer.qkv).view(B, L, -1).split([nq, nkv, nkv], -1)
            q = self._rope(self._norm_head(q.reshape(B, L, s.heads, s.head), layer.norm_q), at).to(self.dtype)
            k = self._rope(self._norm_head(k.reshape(B, L, s.kv_heads, s.head), layer.norm_k), at).to(self.dtype)
            a = attend(i, q, k, v.reshape(B, L, s.kv_heads, s.head).to(self.dtype))
            y = mxu.dot(a.view(B * L, nq).float(), layer.o)
            op, h = mxu.norm_quantize(y, layer.norm_mlp, h, eps=s.eps)
            g, u = mxu.dot(op, layer.gu).split([s.F, s.F], -1)
            c = self.chunks[i]
            y = mxu.dot(T.nn.functional.silu(g) * u, layer.down, ranges=[c] * (s.F // c))
        return (y + h).view(B, L, s.hidden)

    def step(self, x):
        """The next L tokens of every sequence, x [B, L, hidden] float32 -> [B, L, hidden].  L is at most the slots
        over the budget, or those that are free."""
        if x.dim() != 3 or x.shape[0] != self.B or x.shape[2] != self.shape.hidden:
            raise ValueError(f"step: x is {list(x.shape)}, needs [{self.B}, L, {self.shape.hidden}]")
        L = x.shape[1]
        if self.used + L > self.slots:
            kept = min(self.used, self.budget)
            if kept + L > self.slots:                      # (refused before anything is evicted)
                raise ValueError(f"step: {L} tokens after {kept} in {self.slots} slots")
            self.evict()
        n, at = self.used, self.position
        self.lens.fill_(n + L)
        T = X.torch()
        positions = T.arange(at, at + L, device="cuda", dtype=T.int32)

        def attend(i, q, k, v):
            c = self.caches[i]
            c.k[:, n:n + L], c.v[:, n:n + L], c.pos[:, :, n:n + L] = k, v, positions
            return attention.shared(q, *self.prefix[i], c.k, c.v, self.lens, weights=c.weights)

        y = self._run(x, at, attend)
        self.used, self.position = n + L, at + L
        return y

    def evict(self):
        """Every layer's caches down to `budget` tokens a head."""
        lens = self.lens
        for c in self.caches:
            _, _, lens = attention.evict(c.k, c.v, c.weights, c.pos, self.lens, self.budget, self.recent,
                                         out=(c.weights, c.pos, X.torch().empty_like(self.lens)))
        self.lens.copy_(lens)
        self.used = min(self.used, self.budget)


def main(argv=None) -> None:
    import argparse
    ap = argparse.ArgumentParser(description=__doc__.split("\n\n")[0])
    ap.add_argument("--batch", type=int, default=64)
    ap.add_argument("--prompt", type=int, default=4096)
    ap.add_argument("--tokens", type=int, default=96)
    ap.add_argument("--slots", type=int, default=64)
    ap.add_argument("--budget", type=int, default=48)
    ap.add_argument("--recent", type=int, default=8)
    ap.add_argument("--layers", type=int, default=4)
    ap.add_argument("--fmt", default="int4", choices=("int8", "int4", "fp4", "nvfp4"))
    a = ap.parse_args(argv)
    T = X.torch()
    shape = Shape(layers=a.layers)
    rng = np.random.default_rng(0)

    def rows(*n):
        return X.dev(rng.standard_normal((*n, shape.hidden)).astype(np.float32), np.float32)

    batch = Batch(random_layers(shape, a.fmt), shape, rows(a.prompt), a.batch, a.slots, a.budget, a.recent)
    x = rows(a.batch, 1)
    x = batch.step(x)
    T.cuda.synchronize()
    begin, end = T.cuda.Event(True), T.cuda.Event(True)
    begin.record()
    for _ in range(a.tokens):
        x = batch.step(x / x.square().mean(-1, keepdim=True).sqrt())
    end.record()
    T.cuda.synchronize()
    ms = begin.elapsed_time(end) / a.tokens
    print(f"{a.batch} sequences on {a.prompt} shared tokens, {a.layers} layers of {a.fmt}: {ms:.3f} ms a step, "
          f"{a.batch / ms * 1e3:.0f} tokens/s, {batch.used} of {a.slots} slots in use", flush=True)


if __name__ == "__main__":
    main()
