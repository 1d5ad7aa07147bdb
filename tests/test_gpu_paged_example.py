"""The beam search example against the same search over plain caches: every
beam's keys and values in a list of its own, copied whole when beams change
places, with the attention, the eviction and the selection of paged_ref."""
import importlib.util
import os

import numpy as np
import pytest
import torch

import paged_ref as ref
from conftest import ROOT

pytestmark = pytest.mark.gpu


def example():
    spec = importlib.util.spec_from_file_location("paged_beam_search", os.path.join(ROOT, "examples", "paged_beam_search.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


def plain(model, prompt, budget, beams, steps, n_sink=4, n_recent=16, eos=1):
    scale = model.head_dim ** -0.5
    # per beam, layer: [kv heads][slot] rows
    kv = [[[[] for _ in range(model.kv_heads)] for _ in range(model.layers)] for _ in range(beams)]
    acc = [[[] for _ in range(model.kv_heads)] for _ in range(model.layers)]

    def attend(rows, weigh):
        def f(layer, q, k, v):
            out = torch.zeros(q.shape, dtype=torch.float64)
            share = model.q_heads // model.kv_heads
            for r, beam in enumerate(rows):
                for h in range(model.kv_heads):
                    held = kv[beam][layer][h]
                    held.append((k[r, h].cpu().double(), v[r, h].cpu().double()))
                    kk, vv = torch.stack([x[0] for x in held]), torch.stack([x[1] for x in held])
                    w = torch.softmax(q[r, h * share:(h + 1) * share].cpu().double() @ kk.T * scale, 1)
                    out[r, h * share:(h + 1) * share] = w @ vv
                    if weigh:
                        a = acc[layer][h]
                        a.append(0.0)
                        acc[layer][h] = [x + y for x, y in zip(a, w.sum(0).tolist())]
            return out.to(q.device)
        return f

    n = len(prompt)
    for t, token in enumerate(prompt):
        logits = model.step(torch.tensor([token], device="cuda"), t, attend([0], True))
    for layer in range(model.layers):
        for h in range(model.kv_heads):
            _, _, pairs = ref.evict_row(acc[layer][h], list(range(n)), budget, n_sink, n_recent)
            held = kv[0][layer][h]
            for at, to in pairs:
                held[to] = held[at]
            del held[budget:]
    copy = lambda b: [[list(h) for h in layer] for layer in b]  # noqa: E731
    kv = [copy(kv[0]) for _ in range(beams)]
    scores, finished = np.full(beams, -np.inf), None
    scores[0] = 0.0
    logits = logits.expand(beams, -1)
    history = [[] for _ in range(beams)]
    for s in range(steps):
        picked = ref.select(logits.double().cpu().numpy(), scores, finished, beams, eos, eos)
        scores = np.array([p[0] for p in picked])
        finished = [p[3] for p in picked]
        kv = [copy(kv[p[1]]) for p in picked]
        history = [history[p[1]] + [p[2]] for p in picked]
        if s + 1 < steps:
            logits = model.step(torch.tensor([p[2] for p in picked], device="cuda"), n + s, attend(range(beams), False))
    return history, scores


@pytest.mark.parametrize("prompt,budget,beams,steps", [(50, 30, 4, 12), (20, 64, 3, 20), (33, 32, 1, 5), (64, 48, 6, 9)])
def test_example_matches_plain_search(lc, gpu, prompt, budget, beams, steps):
    """With 32-bit pools the two differ by sums' roundings (1e-5 of a logit), which decide between
    no two candidates here: beams are the same, scores within steps * 1e-4."""
    mod = example()
    model = mod.TinyDecoder(vocab=300, width=128, q_heads=4, kv_heads=2, head_dim=64, seed=prompt)
    tokens = torch.randint(2, 300, (prompt,), generator=torch.Generator().manual_seed(prompt)).tolist()
    got, scores = mod.generate(model, tokens, budget=budget, beams=beams, steps=steps, dtype=torch.float32)
    want, want_scores = plain(model, tokens, budget, beams, steps)
    assert got.tolist() == want
    assert np.abs(scores.numpy() - want_scores).max() <= steps * 1e-4


def test_example_bf16_runs(lc, gpu):
    mod = example()
    model = mod.TinyDecoder()
    got, scores = mod.generate(model, list(range(2, 102)), budget=40, beams=5, steps=10)
    assert got.shape == (5, 10) and torch.isfinite(scores).all() and (scores[:-1] >= scores[1:]).all()
