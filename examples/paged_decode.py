"""Serves a small quantized decoder from a paged key/value cache.

    python examples/paged_decode.py [--layers 4] [--hidden 1024] [--steps 32] [--bits 4]

Random weights.  A block is norm, packed q/k/v projections, cache_append (which rotates queries and keys and
writes the pages), paged_attention, the packed output projection, and a packed SwiGLU MLP.  The run prefills
prompts of different lengths in one step, decodes a token a step for all of them, drafts tokens and drops
the rejected ones, branches a sequence, ends one, compacts the pool and goes on; then it compares the last logits of each
sequence with a pass over its whole text without a cache, whose queries and keys `rotary` turns.
"""
import argparse
import os
import sys
import time

import torch
import torch.nn.functional as F

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "mlx-gen_amd"))
import mlxq  # noqa: E402

GROUP = 64


class Decoder:
    def __init__(self, layers=4, hidden=1024, heads=8, kv_heads=2, head_dim=128, inner=2816, vocab=4096, bits=4,
                 context=4096, seed=0, device="cuda"):
        g = torch.Generator(device).manual_seed(seed)

        def packed(n, k):
            w = torch.randn(n, k, generator=g, device=device) / k ** 0.5
            return mlxq.quantize(w.bfloat16(), GROUP, bits)

        self.heads, self.kv_heads, self.head_dim, self.bits = heads, kv_heads, head_dim, bits
        self.tokens = mlxq.TokenEmbedding.from_quantized_parts(*packed(vocab, hidden), GROUP, bits)
        self.head = packed(vocab, hidden)
        self.blocks = [{"qkv": packed((heads + 2 * kv_heads) * head_dim, hidden), "o": packed(hidden, heads * head_dim),
                        "gate": packed(inner, hidden), "up": packed(inner, hidden), "down": packed(hidden, inner)}
                       for _ in range(layers)]
        inv_freq, magnitude = mlxq.rotary_frequencies(head_dim, base=1e6)
        self.table = mlxq.rotary_table(context, inv_freq, magnitude, device=device)

    def _proj(self, x, w):
        return mlxq.quantized_matmul(x, *w, group_size=GROUP, bits=self.bits)

    def _norm(self, x):
        return F.rms_norm(x, x.shape[-1:])

    def _mlp(self, x, w):
        if x.shape[0] <= 8:
            return self._proj(mlxq.swiglu(x, w["gate"], w["up"], GROUP, self.bits), w["down"])
        return self._proj(F.silu(self._proj(x, w["gate"])) * self._proj(x, w["up"]), w["down"])

    def _run(self, ids, attend):
        """Logits of every token; attend(layer, q, k, v) is a block's attention."""
        x = self.tokens.forward(ids).to(torch.bfloat16)
        for i, w in enumerate(self.blocks):
            q, k, v = self._proj(self._norm(x), w["qkv"]).view(len(ids), -1, self.head_dim).split(
                [self.heads, self.kv_heads, self.kv_heads], dim=1)
            x = x + self._proj(attend(i, q, k, v).reshape(len(ids), -1), w["o"])
            x = x + self._mlp(self._norm(x), w)
        return self._proj(self._norm(x), self.head)

    def step(self, ids, cache, batch):
        """A step of several sequences: their new tokens one after the other, as batch.q_starts says."""
        def attend(i, q, k, v):
            keys, values = cache.layer(i)
            q = mlxq.cache_append(k, v, keys, values, batch, q=q, table=self.table)
            return mlxq.paged_attention(q, keys, values, batch)
        return self._run(ids, attend)

    def whole(self, ids):
        """One sequence without a cache, its attention in plain operations."""
        n = len(ids)
        at = torch.arange(n, dtype=torch.int32, device=ids.device)
        hidden = torch.ones(n, n, dtype=torch.bool, device=ids.device).triu(1)

        def attend(i, q, k, v):
            q, k = mlxq.rotary(q, at, self.table), mlxq.rotary(k, at, self.table)
            q, k, v = (t.float().transpose(0, 1).repeat_interleave(self.heads // t.shape[1], 0) for t in (q, k, v))
            z = (q @ k.transpose(1, 2).contiguous()) / self.head_dim ** 0.5
            return (z.masked_fill(hidden, float("-inf")).softmax(-1) @ v).transpose(0, 1).to(torch.bfloat16)
        return self._run(ids, attend)


class Server:
    """Sequences with their texts; `feed` runs one step for some of them."""

    def __init__(self, model, cache):
        self.model, self.cache, self.text, self.logits = model, cache, {}, {}

    def open(self):
        s = self.cache.new()
        self.text[s] = []
        return s

    def feed(self, new):
        """new: {sequence: its new tokens}.  Keeps the logits after each sequence's last token."""
        seqs, counts = list(new), [len(t) for t in new.values()]
        batch = self.cache.batch(seqs, counts)
        ids = torch.tensor([t for ts in new.values() for t in ts], device=self.cache.pool.device)
        out = self.model.step(ids, self.cache, batch)
        end = 0
        for s, n in zip(seqs, counts):
            end += n
            self.text[s] = self.text[s] + new[s]
            self.logits[s] = out[end - 1]
        return out

    def decode(self, steps):
        for _ in range(steps):
            best = torch.stack(list(self.logits.values())).argmax(-1).tolist()
            self.feed({s: [t] for s, t in zip(self.logits, best)})

    def fork(self, seq):
        new, = self.cache.fork([seq])
        self.text[new], self.logits[new] = list(self.text[seq]), self.logits[seq]
        return new

    def close(self, seq):
        self.cache.free(seq)
        del self.text[seq], self.logits[seq]


def run(layers=4, hidden=1024, steps=32, bits=4, prompts=(300, 17, 64, 1), seed=0, say=print):
    """The whole run; returns the largest relative error of the compared logits."""
    model = Decoder(layers=layers, hidden=hidden, inner=hidden * 11 // 4, bits=bits, seed=seed)
    vocab = model.head[0].shape[0]
    g = torch.Generator().manual_seed(seed + 1)
    draw = lambda n: torch.randint(vocab, (n,), generator=g).tolist()  # noqa: E731
    page = 16
    cache = mlxq.PagedCache(layers, sum(-(-(n + 2 * steps + 8) // page) for n in prompts) + 64, model.kv_heads,
                            model.head_dim, page)
    server = Server(model, cache)
    server.feed({server.open(): draw(n) for n in prompts})
    first, *others = server.text
    torch.cuda.synchronize()
    t = time.perf_counter()
    server.decode(steps)
    torch.cuda.synchronize()
    say(f"{len(prompts)} sequences: {(time.perf_counter() - t) / max(steps, 1) * 1e3:.3f} ms a step of one token each")

    # Six drafted tokens in one step; the first two are kept.
    drafts, had = draw(6), len(server.text[first])
    out = server.feed({first: drafts})
    cache.truncate(first, had + 2)
    server.text[first], server.logits[first] = server.text[first][:had + 2], out[1]

    # Two branches that share the full pages of their common text; a sequence ends; the pool is packed.
    branch = server.fork(first)
    server.feed({first: draw(1), branch: draw(3)})
    server.close(others[0])
    used = cache.compact()
    say(f"{used} of {cache.pages} pages held after compaction")
    server.decode(steps)

    worst = 0.0
    for s, text in server.text.items():
        want = model.whole(torch.tensor(text, device="cuda"))[-1].double()
        err = ((server.logits[s].double() - want).norm() / want.norm()).item()
        worst = max(worst, err)
        say(f"sequence {s}: {len(text)} tokens, logits differ from the pass without a cache by {err:.1e}")
    return worst


if __name__ == "__main__":
    p = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    p.add_argument("--layers", type=int, default=4)
    p.add_argument("--hidden", type=int, default=1024)
    p.add_argument("--steps", type=int, default=32)
    p.add_argument("--bits", type=int, default=4, choices=(4, 8))
    a = p.parse_args()
    run(a.layers, a.hidden, a.steps, a.bits)
