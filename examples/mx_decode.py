"""Serves and trains a small mixture-of-experts decoder in microscaled types.

    python examples/mx_decode.py [--layers 2] [--hidden 512] [--experts 8] [--steps 16]

Random weights.  A block is rms_norm of the residual's sum to 8 bits, a 4-bit packed qkv projection, cache_append and
paged_attention, the packed output projection, rms_norm again, a router, the chosen experts' packed SwiGLU MLPs and
their weighted sum; `train` fits a router and the norm before it through their gradients, the experts' packed weights and inputs
held (products of microscaled operands have no gradient).  The run
prefills prompts of different lengths, captures a decode step in a HIP graph and replays it for every token.
"""
import argparse
import os
import sys
import time

import torch
import torch.nn.functional as F

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "mlx-gen_amd"))
import mlxq  # noqa: E402


class Decoder:
    def __init__(self, layers=2, hidden=512, heads=8, kv_heads=2, head_dim=64, experts=8, top_k=2, inner=256, vocab=1024, context=1024,
                 seed=0, device="cuda"):
        g = torch.Generator(device).manual_seed(seed)
        rnd = lambda *s: torch.randn(s, generator=g, device=device)  # noqa: E731
        packed = lambda *s: mlxq.mx_quantize(rnd(*s) / s[-1] ** 0.5)  # noqa: E731
        norm = lambda: (1 + 0.1 * rnd(hidden)).bfloat16()  # noqa: E731
        self.heads, self.kv_heads, self.head_dim, self.top_k = heads, kv_heads, head_dim, top_k
        self.tokens = rnd(vocab, hidden).bfloat16()
        self.head, self.last = packed(vocab, hidden), norm()
        self.blocks = [{"norm": norm(), "qkv": packed((heads + 2 * kv_heads) * head_dim, hidden), "o": packed(hidden, heads * head_dim),
                        "moe_norm": norm(), "router": packed(experts, hidden), "gate_up": packed(experts, 2 * inner, hidden),
                        "down": packed(experts, hidden, inner)} for _ in range(layers)]
        self.table = mlxq.rotary_table(context, *mlxq.rotary_frequencies(head_dim, base=1e6), device=device)

    def moe(self, x, w):
        """The chosen experts' SwiGLU MLPs of 8-bit rows x, summed with the routing weights."""
        routing = mlxq.route_experts(mlxq.mx_matmul(x, w["router"], out_dtype=torch.float32), self.top_k)
        gate, up = mlxq.mx_experts(x, w["gate_up"], routing).chunk(2, -1)
        return mlxq.mx_experts(mlxq.mx_quantize(F.silu(gate) * up, "e4m3"), w["down"], routing, combine=True)

    def step(self, ids, cache, batch):
        """Logits of every new token of several sequences, one after the other as batch.q_starts says."""
        h, delta = self.tokens[ids], None
        for i, w in enumerate(self.blocks):
            if delta is None:
                x = mlxq.rms_norm(h, w["norm"], mx=True)
            else:
                x, h = mlxq.rms_norm(delta, w["norm"], residual=h, mx=True)
            q, k, v = mlxq.mx_matmul(x, w["qkv"]).view(len(ids), -1, self.head_dim).split([self.heads, self.kv_heads, self.kv_heads], dim=1)
            keys, values = cache.layer(i)
            q = mlxq.cache_append(k, v, keys, values, batch, q=q, table=self.table)
            a = mlxq.paged_attention(q, keys, values, batch).view(len(ids), -1)
            x, h = mlxq.rms_norm(mlxq.mx_matmul(mlxq.mx_quantize(a, "e4m3"), w["o"]), w["moe_norm"], residual=h, mx=True)
            delta = self.moe(x, w)
        x, _ = mlxq.rms_norm(delta, self.last, residual=h, mx=True)
        return mlxq.mx_matmul(x, self.head, out_dtype=torch.float32)


class Norm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight):
        ctx.save_for_backward(x, weight)
        return mlxq.rms_norm(x, weight)

    @staticmethod
    def backward(ctx, dy):
        return mlxq.rms_norm_backward(dy.contiguous(), *ctx.saved_tensors)


class Route(torch.autograd.Function):
    """The routing weights of given logits; the choice itself has no gradient."""

    @staticmethod
    def forward(ctx, logits, top_k):
        r = mlxq.route_experts(logits, top_k)
        ctx.save_for_backward(logits, r.ids)
        ctx.mark_non_differentiable(r.ids, r.starts, r.rows)
        return r.weights, r.ids, r.starts, r.rows

    @staticmethod
    def backward(ctx, dweights, *_):
        return mlxq.route_experts_backward(dweights.contiguous(), *ctx.saved_tensors), None


def moe_loss(x, norm, router, experts, top_k, target):
    """Mean squared error of a routed layer: norm [D] and router [E, D] learn, experts (Mx [E, N, D]) are packed and held, and
    no gradient passes through their 8-bit inputs."""
    n = Norm.apply(x, norm)
    weights, ids, starts, rows = Route.apply(n @ router.t(), top_k)
    routing = mlxq.Routing(ids, weights.detach(), starts, rows)
    y = mlxq.mx_experts(mlxq.mx_quantize(n.detach(), "e4m3"), experts, routing, out_dtype=torch.float32)
    return ((weights[..., None] * y).sum(1) - target).square().mean()


def train(hidden=256, experts=8, top_k=2, out=128, tokens=512, steps=30, seed=0, say=print):
    """Fits a router and a norm to outputs of others; returns the losses."""
    g = torch.Generator("cuda").manual_seed(seed)
    rnd = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
    w = mlxq.mx_quantize(rnd(experts, out, hidden) / hidden ** 0.5)
    x, target = rnd(tokens, hidden), rnd(tokens, out) * 0.5
    norm, router = torch.ones(hidden, device="cuda", requires_grad=True), (rnd(experts, hidden) / hidden ** 0.5).requires_grad_(True)
    opt, losses = torch.optim.Adam([norm, router], lr=0.02), []
    for _ in range(steps):
        opt.zero_grad()
        loss = moe_loss(x, norm, router, w, top_k, target)
        loss.backward()
        opt.step()
        losses.append(loss.item())
    say(f"training: loss {losses[0]:.4f} -> {losses[-1]:.4f} in {steps} steps")
    return losses


def serve(layers=2, hidden=512, experts=8, steps=16, prompts=(37, 5, 1), seed=0, say=print):
    """Prefill, then decode steps: one by one and, from the same cache, replayed from a graph.  Returns whether the two gave the
    same tokens."""
    model = Decoder(layers=layers, hidden=hidden, experts=experts, seed=seed)
    vocab, B = len(model.tokens), len(prompts)
    g = torch.Generator().manual_seed(seed + 1)
    cache = mlxq.PagedCache(layers, sum(n + steps for n in prompts) // 16 + 2 * B, model.kv_heads, model.head_dim)
    seqs = [cache.new() for _ in prompts]
    batch = cache.batch(seqs, prompts)
    logits = model.step(torch.randint(vocab, (sum(prompts),), generator=g).cuda(), cache, batch)
    first = logits[batch.q_starts[1:].long() - 1].argmax(-1)
    # Room for every step at once; a step's lengths are written in place.
    last = cache.batch(seqs, [steps] * B)
    lens = torch.tensor(prompts, dtype=torch.int32, device="cuda")
    starts = torch.arange(B + 1, dtype=torch.int32, device="cuda")
    now = mlxq.CacheBatch(last.block_tables, starts, lens.clone(), 1, max(prompts) + steps)
    ids = first.clone()

    def decode():
        now.kv_lens.add_(1)
        ids.copy_(model.step(ids, cache, now).argmax(-1))

    def run(step):
        now.kv_lens.copy_(lens)
        ids.copy_(first)
        tokens = []
        for _ in range(steps):
            step()
            tokens.append(ids.clone())
        return torch.stack(tokens)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        one_by_one = run(decode)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            decode()
        torch.cuda.synchronize()
        t = time.perf_counter()
        replayed = run(graph.replay)
        torch.cuda.synchronize()
    say(f"{B} sequences: {(time.perf_counter() - t) / steps * 1e3:.3f} ms a replayed step of one token each")
    return bool(torch.equal(one_by_one, replayed))


if __name__ == "__main__":
    p = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    p.add_argument("--layers", type=int, default=2)
    p.add_argument("--hidden", type=int, default=512)
    p.add_argument("--experts", type=int, default=8)
    p.add_argument("--steps", type=int, default=16)
    a = p.parse_args()
    print("replayed tokens are those of steps one by one:", serve(a.layers, a.hidden, a.experts, a.steps))
    train()
