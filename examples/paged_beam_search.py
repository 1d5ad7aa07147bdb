"""Beam search over an uncompressed paged cache whose prompt was cut to a budget.

    python examples/paged_beam_search.py [--prompt 200] [--budget 96] [--beams 4] [--steps 24]

A small random decoder (the point is the cache, not the text) runs the loop of
a serving program: the prompt's tokens are appended and attended to with
their attention weights accumulated (append, attn_weights); the cache is cut
to the heaviest tokens (evict); the beams share the prompt's pages (reorder
with every parent 0); then each step appends, attends (attn), selects over
beams and vocabulary (BeamSearch.select) and moves the pages with the beams
(reorder). Nothing is read back to the host until the end.
"""
import argparse
import importlib
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))


class TinyDecoder:
    """Random weights: embedding, layers of attention with rotary positions, output."""

    def __init__(self, vocab=512, width=256, layers=2, q_heads=8, kv_heads=2, head_dim=64, seed=0, device="cuda"):
        g = torch.Generator().manual_seed(seed)

        def rand(*shape):
            return (torch.randn(shape, generator=g) / shape[-1] ** 0.5).to(device)

        self.vocab, self.layers, self.q_heads, self.kv_heads, self.head_dim = vocab, layers, q_heads, kv_heads, head_dim
        self.embed = torch.randn((vocab, width), generator=g).to(device)
        self.wq = [rand(q_heads * head_dim, width) * 2.0 for _ in range(layers)]
        self.wk = [rand(kv_heads * head_dim, width) * 2.0 for _ in range(layers)]
        self.wv = [rand(kv_heads * head_dim, width) for _ in range(layers)]
        self.wo = [rand(width, q_heads * head_dim) * 2.0 for _ in range(layers)]
        self.out = rand(vocab, width) * 2.0
        self.freq = (10000.0 ** (-torch.arange(0, head_dim, 2, dtype=torch.float64) / head_dim)).to(device)

    def rotate(self, x, pos):
        """Rotary positions on [rows, heads, head_dim]; pos a number."""
        a = (pos * self.freq).to(x.dtype)
        lo, hi = x.chunk(2, dim=-1)
        return torch.cat([lo * a.cos() - hi * a.sin(), hi * a.cos() + lo * a.sin()], dim=-1)

    def step(self, tokens, pos, attend):
        """Logits [rows, vocab] of one token a row at position `pos`; attend(layer, q, k, v) adds the
        new key and value [rows, heads, head_dim] to the layer's cache and returns q's attention."""
        x = self.embed[tokens]
        rows = x.shape[0]
        for i in range(self.layers):
            h = x / x.norm(dim=-1, keepdim=True) * x.shape[-1] ** 0.5
            q = self.rotate((h @ self.wq[i].T).view(rows, self.q_heads, self.head_dim), pos)
            k = self.rotate((h @ self.wk[i].T).view(rows, self.kv_heads, self.head_dim), pos)
            v = (h @ self.wv[i].T).view(rows, self.kv_heads, self.head_dim)
            x = x + attend(i, q, k, v).reshape(rows, -1).to(x.dtype) @ self.wo[i].T
        return (x / x.norm(dim=-1, keepdim=True) * x.shape[-1] ** 0.5) @ self.out.T


def generate(model, prompt, *, budget, beams, steps, page=16, n_sink=4, n_recent=16, eos=1, dtype=torch.bfloat16):
    """The `beams` best continuations of `prompt` (a list of tokens): (tokens [beams, steps], scores [beams])."""
    lc = importlib.import_module("lumen-rs_b200")
    dev = model.embed.device
    heads, dim, scale = model.kv_heads, model.head_dim, model.head_dim ** -0.5
    n = len(prompt)
    width = -(-max(n, min(n, budget) + steps) // page)
    pools = [torch.zeros((model.layers, beams * width, heads, page, dim), dtype=dtype, device=dev) for _ in range(2)]
    cache = lc.PagedKvCache(*pools, max_seqs=beams, max_pages_per_seq=width, max_q_heads=model.q_heads)
    # every row has pages of its own; what the beams come to share is simply not used
    tables = torch.arange(beams * width, dtype=torch.int32, device=dev).view(beams, width)
    acc = torch.zeros((model.layers, 1, heads, width * page), device=dev)
    pos = torch.zeros((model.layers, 1, heads, width * page), dtype=torch.int32, device=dev)

    def attend(rows, lens, kind):
        def f(layer, q, k, v):
            at = pos[layer] if kind == "prompt" else None
            cache.append(layer, rows, lens, k.unsqueeze(2).contiguous(), v.unsqueeze(2).contiguous(), at,
                         lens if at is not None else None)
            q = q.to(dtype).contiguous()
            if kind == "prompt":
                return cache.attn_weights(layer, rows, lens + 1, q, scale, acc[layer])
            return cache.attn(layer, rows, lens + 1, q, scale)
        return f

    lens = torch.zeros(1, dtype=torch.int32, device=dev)
    first = tables[:1].contiguous()
    for t, token in enumerate(prompt):
        logits = model.step(torch.tensor([token], device=dev), t, attend(first, lens, "prompt"))
        lens = lens + 1
    for layer in range(model.layers):
        cache.evict(layer, first, lens, budget, acc[layer], pos[layer], n_sink=n_sink, n_recent=n_recent)
    lens = lens.clamp(max=budget)

    # one beam holds the prompt: all rows continue it
    tables = cache.reorder(tables, lens, torch.zeros((1, beams), dtype=torch.int32, device=dev))
    search = lc.BeamSearch(1, beams, model.vocab)
    scores = torch.full((1, beams), float("-inf"), device=dev)
    scores[0, 0] = 0.0
    finished = None
    logits = logits.expand(beams, -1)
    parents, tokens = [], []
    for s in range(steps):
        scores, parent, token, finished = search.select(logits.view(1, beams, -1).contiguous(), scores, finished, eos_id=eos,
                                                        pad_id=eos)
        parents.append(parent[0])
        tokens.append(token[0])
        tables = cache.reorder(tables, lens, parent)
        if s + 1 < steps:
            logits = model.step(token[0].long(), n + s, attend(tables, lens.expand(beams).contiguous(), "beams"))
            lens = lens + 1
    # back along the parents
    out = torch.empty((beams, steps), dtype=torch.int64, device=dev)
    at = torch.arange(beams, device=dev)
    for s in reversed(range(steps)):
        out[:, s] = tokens[s][at].long()
        at = parents[s][at].long()
    if cache.status() != lc.LC_OK:
        raise RuntimeError("the cache met a length or a page out of range")
    return out.cpu(), scores[0].cpu()


def main():
    ap = argparse.ArgumentParser()
    ap.add_argument("--prompt", type=int, default=200)
    ap.add_argument("--budget", type=int, default=96)
    ap.add_argument("--beams", type=int, default=4)
    ap.add_argument("--steps", type=int, default=24)
    a = ap.parse_args()
    model = TinyDecoder()
    prompt = torch.randint(2, model.vocab, (a.prompt,), generator=torch.Generator().manual_seed(1)).tolist()
    tokens, scores = generate(model, prompt, budget=a.budget, beams=a.beams, steps=a.steps)
    for row, score in zip(tokens.tolist(), scores.tolist()):
        print("%9.4f  %s" % (score, " ".join(map(str, row))))


if __name__ == "__main__":
    main()
