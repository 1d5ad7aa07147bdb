"""Plain 64-bit forms of the uncompressed paged cache's operators and of beam
selection, one row after the other, and the inputs their tests share."""
import numpy as np
import torch

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}

# One value's error, for unit-normal K, V and scores below about 30. f32 sums: a
# score of 256 products is off by at most 256 * 2^-24 * sum |q k| scale, some
# 1e-5 for these inputs, which weighs the values (|v| < 6) as much. Weights
# held as two 16-bit halves are off by 2^-17 (bf16; 2^-22 f16), 4e-5 with
# |v| < 6. Then half an ulp of the output's type.
ATOL = 1e-4
RTOL = {"f32": 1e-5, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}


def pool(layers, pages, heads, page, dim, dtype, seed, layout="phtd", offset=0, fill=float("nan")):
    """Two pools [layers, pages, heads, page, dim] full of `fill`, as views of the page layout and
    `offset` elements into their storage."""
    order = {"phtd": (0, 1, 2, 3, 4), "pthd": (0, 1, 3, 2, 4), "plhtd": (1, 0, 2, 3, 4)}[layout]
    shape = (layers, pages, heads, page, dim)
    stored = [shape[i] for i in order]
    back = [order.index(i) for i in range(5)]
    out = []
    for _ in range(2):
        flat = torch.full((int(np.prod(stored)) + offset,), fill, dtype=DTYPES[dtype], device="cuda")
        out.append(flat[offset:].view(stored).permute(back))
    return out


def tables_for(lens, page, pages, width, seed):
    """Distinct random pages for every sequence; unused entries -1."""
    g = np.random.default_rng(seed)
    ids = g.permutation(pages)
    t = np.full((len(lens), width), -1, np.int32)
    at = 0
    for s, n in enumerate(lens):
        need = -(-n // page)
        t[s, :need] = ids[at:at + need]
        at += need
    return torch.from_numpy(t).cuda()


def fill_slots(k, v, layer, tables, lens, seed):
    """Unit-normal rows in the used slots; returns them as [seq] of [heads, n, dim] (in the pool's type)."""
    g = torch.Generator().manual_seed(seed)
    page, rows = k.shape[3], []
    for s, n in enumerate(lens):
        kk = torch.randn((k.shape[2], n, k.shape[4]), generator=g).to(k.dtype).cuda()
        vv = torch.randn((k.shape[2], n, k.shape[4]), generator=g).to(k.dtype).cuda()
        for p in range(-(-n // page)):
            m = min(page, n - p * page)
            k[layer, int(tables[s, p]), :, :m] = kk[:, p * page:p * page + m]
            v[layer, int(tables[s, p]), :, :m] = vv[:, p * page:p * page + m]
        rows.append((kk, vv))
    return rows


def attn(rows, q, scale, window=0):
    """Outputs [seqs, heads, dim] and weights [seq] of [q heads, n], in f64."""
    out = torch.zeros(q.shape, dtype=torch.float64)
    weights = []
    for s, (k, v) in enumerate(rows):
        n = k.shape[1]
        lo = max(0, n - window) if window else 0
        w = torch.zeros((q.shape[1], n), dtype=torch.float64)
        share = q.shape[1] // k.shape[0]
        for i in range(q.shape[1] if n else 0):
            x = (k[i // share, lo:].double().cpu() @ q[s, i].double().cpu()) * scale
            w[i, lo:] = torch.softmax(x, 0)
            out[s, i] = w[i, lo:] @ v[i // share, lo:].double().cpu()
        weights.append(w)
    return out, weights


def evict_row(acc, pos, budget, n_sink, n_recent):
    """(kept acc, kept pos, [(from, to)]) of one row (lists), as the definition has it."""
    n = len(acc)
    if n <= budget:
        return list(acc), list(pos), []
    newest = max(pos)

    def weight(t):
        if pos[t] < n_sink or pos[t] > newest - n_recent:
            return float("inf")
        return -float("inf") if acc[t] != acc[t] else acc[t]

    # NaN ranks below -inf, held slots above +inf
    def rank(t):
        held = pos[t] < n_sink or pos[t] > newest - n_recent
        return (0 if held else 1 if acc[t] == acc[t] else 2, -weight(t) if not held and acc[t] == acc[t] else 0.0, t)

    stay = set(sorted(range(n), key=rank)[:budget])
    holes = [t for t in range(budget) if t not in stay]
    movers = [t for t in range(budget, n) if t in stay]
    a, p = list(acc), list(pos)
    for to, at in zip(holes, movers):
        a[to], p[to] = acc[at], pos[at]
    return a[:budget] + [0.0] * (n - budget), p[:budget] + [-1] * (n - budget), list(zip(movers, holes))


def reorder(tables, lens, parents, page):
    """New tables and the tail copies [(from page, to page, slots)] of each group."""
    groups, beams = parents.shape
    out, copies = tables.copy(), []
    for g in range(groups):
        full, fill = divmod(int(lens[g]), page)
        t = tables[g * beams:(g + 1) * beams]
        spare = [j for j in range(beams) if j not in parents[g].tolist()]
        seen = set()
        for j in range(beams):
            p = int(parents[g, j])
            out[g * beams + j, :full] = t[p, :full]
            if not fill:
                continue
            own = p
            if p in seen:
                own = spare.pop(0)
                copies.append((int(t[p, full]), int(t[own, full]), fill))
            seen.add(p)
            out[g * beams + j, full] = t[own, full]
    return out, copies


def select(logits, scores, finished, n_out, eos, pad):
    """The definition in f64, on one group's rows [beams, vocab]: (totals, parents, tokens, finished)."""
    beams, vocab = logits.shape
    x = logits.astype(np.float64)
    with np.errstate(all="ignore"):
        x = x - x.max(1, keepdims=True)
        z = scores.astype(np.float64)[:, None] + (x - np.log(np.exp(x).sum(1, keepdims=True)))
    for b in range(beams):
        if finished is not None and finished[b]:
            z[b] = -np.inf
            z[b, pad] = scores[b]
    z = np.where(np.isnan(z), -np.inf, z).reshape(-1)
    order = np.argsort(-z, kind="stable")[:n_out]
    res = []
    for r in range(n_out):
        if r < len(order) and z[order[r]] > -np.inf:
            b, t = divmod(int(order[r]), vocab)
            done = bool(finished is not None and finished[b]) or t == eos
            res.append((z[order[r]], b, t, int(done)))
        else:
            res.append((-np.inf, r % beams, pad, 1))
    return res
