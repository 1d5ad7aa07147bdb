"""Beam search's selection against its plain 64-bit form."""
import numpy as np
import pytest
import torch

import paged_ref as ref

pytestmark = pytest.mark.gpu


def check(lc, logits, scores, finished, n_out, eos=2, pad=0, rtol=0.0):
    """logits [groups, beams, vocab] on the GPU. Totals in f32 are off by about
    four roundings of values below 100: 3e-5 (larger ones: rtol, of three roundings to 24 bits)."""
    g, beams, vocab = logits.shape
    beam = lc.BeamSearch(g, beams, vocab, n_out)
    fin = None if finished is None else torch.from_numpy(finished).cuda()
    s, p, t, f = beam.select(logits, torch.from_numpy(scores).cuda(), fin, eos_id=eos, pad_id=pad)
    s, p, t, f = s.cpu().numpy(), p.cpu().numpy(), t.cpu().numpy(), f.cpu().numpy()
    x = logits.double().cpu().numpy()
    for i in range(g):
        want = ref.select(x[i], scores[i], None if finished is None else finished[i], n_out, eos, pad)
        assert [int(v) for v in p[i]] == [w[1] for w in want]
        assert [int(v) for v in t[i]] == [w[2] for w in want]
        assert [int(v) for v in f[i]] == [w[3] for w in want]
        a, b = s[i].astype(np.float64), np.array([w[0] for w in want])
        assert np.array_equal(np.isinf(a), np.isinf(b))
        assert np.allclose(a[np.isfinite(a)], b[np.isfinite(b)], rtol=rtol, atol=3e-5)


def inputs(groups, beams, vocab, dtype, seed, spread=3.0):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn((groups, beams, vocab), generator=g) * spread).to(ref.DTYPES[dtype]).cuda()
    r = np.random.default_rng(seed)
    return x, (-10 * r.random((groups, beams))).astype(np.float32), r


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("groups,beams,vocab,n_out", [(1, 1, 1, 1), (1, 1, 1, 3), (2, 4, 7, 8), (1, 3, 500, 3), (3, 4, 8191, 4),
                                                      (2, 5, 8193, 10), (1, 8, 50021, 16), (2, 2, 100003, 17),
                                                      (1, 64, 1000, 64), (4, 16, 20000, 33), (1, 2, 262144, 64)])
def test_select_matches_plain(lc, gpu, dtype, groups, beams, vocab, n_out):
    x, scores, r = inputs(groups, beams, vocab, dtype, groups * 7 + vocab)
    pad = 0 if vocab < 3 else 1
    check(lc, x, scores, None, n_out, eos=2, pad=pad)
    check(lc, x, scores, (r.random((groups, beams)) < 0.4).astype(np.uint8), n_out, eos=2, pad=pad)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_select_ties(lc, gpu, dtype):
    """Equal logits: the lower token; equal beams: the lower beam. Whole rows equal take the list's
    long way."""
    x = torch.zeros((3, 4, 30011), dtype=ref.DTYPES[dtype], device="cuda")
    x[1, :, ::5] = 1.0
    x[2, :, 17::4099] = 2.0
    x[2, 1, 3] = -0.0
    check(lc, x, np.zeros((3, 4), np.float32), None, 9)


def test_select_first_step_and_dead_beams(lc, gpu):
    """One live beam (the others at -inf), then none, then NaN scores."""
    x, _, _ = inputs(3, 4, 1000, "f32", 5)
    scores = np.full((3, 4), -np.inf, np.float32)
    scores[0, 0] = 0.0
    scores[2] = [np.nan, -1.0, np.nan, -2.0]
    check(lc, x, scores, None, 4)


def test_select_masked_rows(lc, gpu):
    """Rows with few or no candidates left, NaN and infinite logits."""
    x, scores, _ = inputs(5, 3, 20000, "f32", 6)
    x[0, 0] = -float("inf")
    x[1] = -float("inf")
    x[1, 2, 19999] = 1.0
    x[2, 1, 7] = float("nan")
    x[3, 0, 9] = float("inf")
    x[4, :, 100:] = -float("inf")
    check(lc, x, scores, None, 8)
    check(lc, x, scores, np.array([[0, 1, 0]] * 5, np.uint8), 8)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_select_strided_rows_and_fewer_groups(lc, gpu, dtype):
    wide = torch.randn((3, 4, 1100), device="cuda").to(ref.DTYPES[dtype])
    scores = -torch.rand((3, 4), device="cuda")
    beam = lc.BeamSearch(5, 4, 1003)
    got = beam.select(wide[:, :, 5:1008], scores)
    same = beam.select(wide[:, :, 5:1008].contiguous(), scores)
    for a, b in zip(got, same):
        assert torch.equal(a, b)


def test_select_repeats(lc, gpu):
    x, scores, _ = inputs(4, 8, 70001, "bf16", 9)
    beam = lc.BeamSearch(4, 8, 70001, 16)
    s = torch.from_numpy(scores).cuda()
    first = beam.select(x, s)
    for _ in range(5):
        for a, b in zip(beam.select(x, s), first):
            assert torch.equal(a, b)


def test_select_refusals(lc, gpu):
    for args in ((0, 4, 100), (1, 65, 100), (1, 4, 0), (1, 4, 100, 65), (1, 4, 1 << 26), (70000, 1, 10)):
        with pytest.raises(lc.LumenError) as e:
            lc.BeamSearch(*args)
        assert e.value.code == lc.LC_ERR_INVALID
    beam = lc.BeamSearch(2, 4, 100)
    x = torch.zeros((2, 4, 100), device="cuda")
    s = torch.zeros((2, 4), device="cuda")
    with pytest.raises(lc.LumenError):
        beam.select(torch.zeros((3, 4, 100), device="cuda"), torch.zeros((3, 4), device="cuda"))
    with pytest.raises(lc.LumenError):
        beam.select(x, s, pad_id=100)
    for bad in (x.cpu(), x.double(), x[:, :3], torch.zeros((2, 100, 4), device="cuda").transpose(1, 2)):
        with pytest.raises((ValueError, TypeError)):
            beam.select(bad, s)
    with pytest.raises((ValueError, TypeError)):
        beam.select(x, s.double())
    with pytest.raises((ValueError, TypeError)):
        beam.select(x, s, s)


@pytest.mark.parametrize("beams,n_out,vocab", [(64, 64, 5000), (16, 32, 700), (12, 12, 700), (33, 40, 9001)])
def test_select_many_candidates(lc, gpu, beams, n_out, vocab):
    """Merges of many candidates: all totals equal, all but the last beam's equal, one beam far ahead,
    every beam alike up to its score."""
    x = torch.zeros((4, beams, vocab), device="cuda")
    x[1, -1] = torch.linspace(-3, 3, vocab, device="cuda")
    x[2] = torch.randn((beams, vocab), generator=torch.Generator().manual_seed(1)).cuda()
    x[3] = torch.linspace(0, 40, vocab, device="cuda").flip(0)
    scores = np.zeros((4, beams), np.float32)
    scores[2] = -30
    scores[2, beams // 2] = 0
    scores[3] = -np.arange(beams, dtype=np.float32) * np.float32(0.37)
    check(lc, x, scores, None, n_out)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("mask", ["-inf", "lowest"])
@pytest.mark.parametrize("vocab,kept", [(30011, 5), (30011, 40), (70000, 3000), (9000, 0)])
def test_select_masked_vocabulary(lc, gpu, dtype, mask, vocab, kept):
    """All tokens but a few at -inf or at the type's lowest value: spread, in one run at the end, and in
    rows of their own; ties of the lowest go to the lowest tokens."""
    x, scores, r = inputs(3, 4, vocab, dtype, vocab + kept)
    fill = -float("inf") if mask == "-inf" else torch.finfo(x.dtype).min
    y = torch.full_like(x, fill)
    spread = torch.from_numpy(r.permutation(vocab)[:kept]).cuda()
    y[0][:, spread] = x[0][:, spread]
    y[1][:, vocab - kept:] = x[1][:, vocab - kept:]
    y[2, 1] = x[2, 1]
    if kept == 0:  # a maximum of the lowest value: log of a count
        scores[:] = np.float32(-1.5)
    check(lc, y, scores, None, 8, rtol=2.0 ** -22)
    check(lc, y, scores, None, 24, rtol=2.0 ** -22)


def test_select_captured(lc, gpu):
    """A graph's replay after larger and smaller calls of its handle, with other logits in place."""
    x, scores, _ = inputs(4, 4, 30011, "f32", 3)
    beam = lc.BeamSearch(4, 4, 30011, 6)
    s = torch.from_numpy(scores).cuda()
    a, b = x[:2].clone(), x[2:].clone()
    wants = [[t.clone() for t in beam.select(y, s[:2])] for y in (a, b)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = beam.select(a, s[:2])
    for y, want in ((a.clone(), wants[0]), (b, wants[1])):
        beam.select(x, s)
        beam.select(x[:1], s[:1])
        a.copy_(y)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(got, want))


def check_f32(lc, x, scores, n_out, pad=0):
    """Against the definition in f32, whose totals the kernel's are equal to where the sums' logarithms are: rows
    whose other logits are 150 and more below one (its sum is 1), or totals whose steps are far above the logarithm."""
    g, beams, vocab = x.shape
    got = [t.cpu().numpy() for t in lc.BeamSearch(g, beams, vocab, n_out).select(x, torch.from_numpy(scores).cuda(), pad_id=pad)]
    xs = x.float().cpu().numpy()
    for i in range(g):
        d = xs[i] - xs[i].max(1, keepdims=True)
        z = scores[i][:, None] + (d - np.log(np.exp(d.astype(np.float64)).sum(1, keepdims=True)).astype(np.float32))
        assert z.dtype == np.float32
        z = z.reshape(-1)
        order = np.argsort(-z, kind="stable")[:n_out]
        m = len(order)
        np.testing.assert_array_equal(got[0][i, :m], z[order])
        np.testing.assert_array_equal(got[1][i, :m], order // vocab)
        np.testing.assert_array_equal(got[2][i, :m], order % vocab)
        assert np.isinf(got[0][i, m:]).all() and (got[3][i, m:] == 1).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("score", [-0.5, -300.0, -1e4, -1e9])
@pytest.mark.parametrize("groups,beams,vocab,n_out", [(1, 1, 30011, 1), (1, 1, 30011, 2), (2, 4, 30011, 9), (3, 8, 9001, 64),
                                                      (60, 4, 20001, 5), (300, 1, 9000, 7), (2, 2, 3, 5)])
def test_select_equal_totals_of_different_logits(lc, gpu, dtype, score, groups, beams, vocab, n_out):
    """Logits that differ by less than a step of their totals: the lower token goes first."""
    g = torch.Generator().manual_seed(vocab + n_out)
    x = (-200 - torch.rand((groups, beams, vocab), generator=g)).cuda()
    x.scatter_(2, torch.randint(0, vocab, (groups, beams, 1), generator=g).cuda(), 0.0)
    # all beams alike, or one far ahead, or steps apart that are a few of a total's
    scores = np.full((groups, beams), score, np.float32)
    scores[1::3] = np.float32(-1e9)
    scores[1::3, beams // 2] = np.float32(score)
    scores[2::3] = score * (1 + 2.0 ** -20 * np.arange(beams, dtype=np.float32))
    check_f32(lc, x.to(ref.DTYPES[dtype]), scores, n_out)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_select_equal_logits_beside_equal_totals(lc, gpu, dtype):
    """More equal logits than places, with a larger logit of the same total behind them."""
    x = torch.full((2, 1, 20000), -200.0, device="cuda")
    x[:, 0, 5] = 0.0
    x[0, 0, 1000::9] = -199.0
    x[0, 0, 15000] = -198.0
    x[1, 0, :3] = -250.0
    x[1, 0, 19999] = -199.0
    x = x.to(ref.DTYPES[dtype])
    for score in (-1.0, -1e9):
        for n_out in (1, 2, 3, 12):
            check_f32(lc, x, np.full((2, 1), score, np.float32), n_out)


def test_select_infinite_and_huge_scores(lc, gpu):
    """Scores that leave every candidate of a beam the same total."""
    x, _, _ = inputs(3, 3, 5001, "f32", 8)
    scores = np.array([[1e30, -1e30, -3e38], [np.inf, 0, np.inf], [-1e9, 0, -1e9]], np.float32)
    for n_out in (1, 4, 40):
        check_f32(lc, x[:2].contiguous(), scores[:2], n_out)
    few = x[2:, :, :5].contiguous()
    few[0, 1] = torch.tensor([0.0, -200, -201, -202, -203])
    check_f32(lc, few, scores[2:], 12)
