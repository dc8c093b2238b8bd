"""Live streams through a small text decoder on the paged 8-bit cache.

A decoder of a few layers (Q8_0 projections through ``Q8Mat``, attention through
``KvCache8``) serves many streams at once: prompts of uneven lengths, single
tokens over a sliding window with a few first tokens that stay visible,
hypotheses that fork from a stream, streams that end, and a compaction of the
pool.  Random weights; it shows the calls and what they cost.

    python examples/live_decoder.py [--streams 64] [--layers 4] [--steps 200]
"""
from __future__ import annotations

import argparse
import os
import sys

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import numpy as np  # noqa: E402
import torch  # noqa: E402

from stealcode_b200 import KvCache8, Q8Mat, synth  # noqa: E402


def ids(x) -> torch.Tensor:
    return torch.tensor(list(x), dtype=torch.int32, device="cuda")


class Decoder:
    """Pre-norm decoder layers: x += Wo attention(Wqkv x), x += W2 silu(W1 x)."""

    def __init__(self, layers=4, d_model=1024, heads=8, kv_heads=2, d_ff=2048, streams=64, pages=4096, max_pages=256,
                 window=1024, sinks=4, page=64, block=32, seed=7):
        self.heads, self.kv, self.hd = heads, kv_heads, d_model // heads
        self.window, self.sinks = window, sinks
        rows = (heads + 2 * kv_heads) * self.hd

        def mat(i, n, k):
            return Q8Mat(synth.q8_weights(seed + i, n, k), n, k)

        self.layers = [(mat(4 * i, rows, d_model), mat(4 * i + 1, d_model, d_model), mat(4 * i + 2, d_ff, d_model),
                        mat(4 * i + 3, d_model, d_ff)) for i in range(layers)]
        self.cache = KvCache8(layers, pages, kv_heads, self.hd, streams, max_pages, page=page, block=block)

    def step(self, x: torch.Tensor, counts: torch.Tensor, n: int, *, seqs=None, cu=None) -> torch.Tensor:
        """x [rows, d_model] f32: the new tokens of the sequences (counts[i] each, at most n), one sequence
        after the other; returns the last layer's output rows."""
        c = self.cache
        c.reserve(counts, seqs=seqs)
        for i, (wqkv, wo, w1, w2) in enumerate(self.layers):
            qkv = wqkv.gemm(norm(x)).view(len(x), self.heads + 2 * self.kv, self.hd)
            q, k, v = qkv.split((self.heads, self.kv, self.kv), 1)
            c.append(i, k, v, seqs=seqs, cu=cu, n=n)
            a = c.attend(i, q, seqs=seqs, cu=cu, n=n, window=self.window, sinks=self.sinks)
            x = x + wo.gemm(a.view(len(x), -1))
            x = x + w2.gemm(torch.nn.functional.silu(w1.gemm(norm(x))))
        return x

    def tidy(self) -> None:
        """Pages that left the window go back to the pool."""
        self.cache.slide(self.window, self.sinks)


def norm(x: torch.Tensor) -> torch.Tensor:
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6)


def run(streams=64, layers=4, steps=200, d_model=1024, heads=8, kv_heads=2, d_ff=2048, window=1024, sinks=4, pages=4096,
        prompt=(20, 1500), quiet=False):
    """The example; returns the decoder and the last rows of the streams."""
    beams = streams // 4  # the last quarter of the sequences are hypotheses
    live = streams - beams
    dec = Decoder(layers, d_model, heads, kv_heads, d_ff, streams, pages, window=window, sinks=sinks)
    g = torch.Generator(device="cuda").manual_seed(1)
    lengths = np.random.default_rng(1).integers(prompt[0], prompt[1] + 1, live)
    emb = torch.randn(int(lengths.sum()), d_model, generator=g, device="cuda")
    t = [torch.cuda.Event(enable_timing=True) for _ in range(4)]
    t[0].record()
    cu = ids(np.concatenate([[0], np.cumsum(lengths)]))
    x = dec.step(emb, ids(lengths), int(lengths.max()), seqs=ids(range(live)), cu=cu)
    x = x[cu[1:].long() - 1]
    dec.tidy()
    t[1].record()
    one, seqs = ids([1] * live), ids(range(live))
    for s in range(steps):
        x = dec.step(norm(x), one, 1, seqs=seqs)
        if s % 64 == 63:
            dec.tidy()
    t[2].record()
    # every fourth stream goes on as two hypotheses; then it ends and the pool is compacted
    parents, children = ids(range(0, 4 * beams, 4)[:beams] if live >= 4 * beams - 3 else [0] * beams), ids(range(live, streams))
    dec.cache.fork(parents, children)
    y = dec.step(norm(x[parents.long()]), ids([1] * beams), 1, seqs=children)
    dec.cache.release(parents)
    dec.cache.compact()
    t[3].record()
    dec.cache.check()
    if not quiet:
        used = int((dec.cache.refs > 0).sum())
        print(f"prompts: {int(lengths.sum())} tokens of {live} streams in {t[0].elapsed_time(t[1]):.1f} ms")
        print(f"steps: {steps} x {live} tokens, {t[1].elapsed_time(t[2]) / max(1, steps):.3f} ms a step")
        print(f"fork, step, release, compact: {t[2].elapsed_time(t[3]):.2f} ms; {used} of {dec.cache.n_pages} pages in use")
    return dec, x, y


def main():
    a = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    a.add_argument("--streams", type=int, default=64)
    a.add_argument("--layers", type=int, default=4)
    a.add_argument("--steps", type=int, default=200)
    o = a.parse_args()
    run(o.streams, o.layers, o.steps)


if __name__ == "__main__":
    main()
