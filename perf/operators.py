"""Cases of the uncompressed paged cache's operators and of beam search: decode attention over pages, the same with the
accumulated attention weights, eviction by those weights, the selection over beams and vocabulary, and the reordering
of the beams' pages. Each case runs as elementary torch operations in 32 bits, or (``own``) through this package."""
import importlib
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
ESIZE = {"f32": 4, "bf16": 2, "f16": 2}


def listed():
    """12 cases, two or more for each operator."""
    return [
        # the first steps of one short chat on a 32-bit cache with a head dimension that is no power of two: latency only
        dict(name="attn_short", op="attn", seqs=1, low=19, tokens=19, q_heads=8, kv_heads=2, dim=80, page=16, window=0, dtype="f32"),
        # batched decode, 32 sequences of 8192 tokens in 256-token blocks: the ordinary serving step
        dict(name="attn_batch", op="attn", seqs=32, low=8192, tokens=8192, q_heads=32, kv_heads=8, dim=128, page=256, window=0, dtype="bf16"),
        # a sliding layer (window 1024) of 16 sequences, head dimension 256, ragged lengths, one of them empty
        dict(name="attn_window", op="attn", seqs=16, low=0, tokens=4096, q_heads=16, kv_heads=8, dim=256, page=64, window=1024, dtype="f16"),
        # one long context alone on the card: the work has to be split over the length
        dict(name="attn_long", op="attn", seqs=1, low=131072, tokens=131072, q_heads=32, kv_heads=8, dim=128, page=64, window=0, dtype="bf16"),
        # decode steps that keep the attention weights for the eviction: a few short requests with odd lengths
        dict(name="weights_few", op="weights", seqs=3, low=1, tokens=777, q_heads=12, kv_heads=4, dim=64, page=16, window=0, dtype="f16"),
        # the same for a full batch of ragged lengths
        dict(name="weights_batch", op="weights", seqs=24, low=1000, tokens=6000, q_heads=32, kv_heads=8, dim=128, page=32, window=0, dtype="bf16"),
        # every step of a loop that holds its caches at a budget: one token came in, one goes
        dict(name="evict_step", op="evict", seqs=16, low=1025, tokens=1025, budget=1024, sink=4, recent=128, kv_heads=8, dim=128, page=32, dtype="bf16"),
        # long prompts cut down to their budget once
        dict(name="evict_prompt", op="evict", seqs=8, low=6001, tokens=8192, budget=2048, sink=4, recent=256, kv_heads=8, dim=128, page=64, dtype="bf16"),
        # one request with 4 beams, 32-bit logits over an odd vocabulary
        dict(name="select_one", op="select", groups=1, beams=4, n_out=4, vocab=50021, dtype="f32"),
        # 32 requests with 8 beams, twice as many candidates as beams, 16-bit logits
        dict(name="select_batch", op="select", groups=32, beams=8, n_out=16, vocab=131072, dtype="bf16"),
        # one request's beams change places between two tokens
        dict(name="reorder_one", op="reorder", groups=1, beams=4, tokens=531, kv_heads=4, dim=64, page=16, layers=4, dtype="f16"),
        # a batch of beam searches over many layers, with large pages
        dict(name="reorder_batch", op="reorder", groups=8, beams=8, tokens=2272, kv_heads=8, dim=128, page=64, layers=16, dtype="bf16"),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    """One more case of the listed ones' ranges."""
    op = rng.choice(["attn", "attn", "weights", "evict", "select", "reorder"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if op in ("attn", "weights"):
        kv = rng.choice([1, 2, 4, 8])
        dim = rng.choice([64, 80, 96, 128, 128, 192, 256])
        # at most half of the largest listed case's bytes
        tokens = min(_log(rng, 1, 131072), (1 << 29) // (kv * dim * 2 * ESIZE[dtype]))
        seqs = max(1, min(_log(rng, 1, 64), (1 << 29) // (tokens * kv * dim * 2 * ESIZE[dtype])))
        ragged = rng.random() < 0.7
        return dict(op=op, seqs=seqs, low=rng.randint(0, tokens) if ragged else tokens, tokens=tokens, q_heads=kv * rng.choice([1, 2, 3, 4, 6, 8]),
                    kv_heads=kv, dim=dim, page=rng.choice([8, 16, 32, 48, 64, 128, 256]), window=rng.choice([0, 0, 0, rng.randint(1, tokens)]), dtype=dtype)
    if op == "evict":
        kv = rng.choice([1, 2, 4, 8])
        dim = rng.choice([64, 80, 128, 256])
        tokens = min(_log(rng, 64, 32768), (1 << 27) // (kv * dim * 2 * ESIZE[dtype]))
        seqs = max(1, min(_log(rng, 1, 32), (1 << 27) // (tokens * kv * dim * 2 * ESIZE[dtype])))
        budget = rng.choice([tokens - 1, rng.randint(16, tokens - 1)])
        return dict(op=op, seqs=seqs, low=rng.randint(1, tokens), tokens=tokens, budget=budget, sink=rng.choice([0, 4]), recent=rng.randint(0, budget // 4),
                    kv_heads=kv, dim=dim, page=rng.choice([8, 16, 48, 64, 256]), dtype=dtype)
    if op == "select":
        beams = rng.randint(1, 16)
        vocab = _log(rng, 500, 131072)
        groups = max(1, min(_log(rng, 1, 32), (1 << 24) // (beams * vocab)))
        return dict(op=op, groups=groups, beams=beams, n_out=beams * rng.choice([1, 1, 2]), vocab=vocab, dtype=dtype)
    return dict(op=op, groups=rng.randint(1, 8), beams=rng.randint(2, 8), tokens=_log(rng, 2, 2272), kv_heads=rng.choice([1, 2, 4, 8]), dim=rng.choice([64, 80, 128]),
                page=rng.choice([8, 16, 64, 100]), layers=rng.randint(1, 16), dtype=rng.choice(["bf16", "f16"]))


def _lens(case):
    """The sequences' lengths, evenly between low and tokens, both among them."""
    n = case["seqs"]
    return [case["tokens"] - (case["tokens"] - case["low"]) * i // max(1, n - 1) for i in range(n)]


def _extra(case):
    """Beams that share a parent with an earlier one, on average over parents drawn at random."""
    w = case["beams"]
    return case["groups"] * w * (1.0 - 1.0 / w) ** w


def work(case):
    """Each input read once, each output written once."""
    op, e = case["op"], ESIZE[case["dtype"]]
    if op in ("attn", "weights"):
        kv, dim, heads = case["kv_heads"], case["dim"], case["q_heads"]
        seen = [min(n, case["window"]) if case["window"] else n for n in _lens(case)]
        moved = 2 * dim * e * kv * sum(seen) + 2 * case["seqs"] * heads * dim * e + 4 * sum(-(-n // case["page"]) for n in seen)
        moved += 8 * kv * sum(_lens(case)) if op == "weights" else 0
        return {"bytes": moved, "flops": 4 * dim * heads * sum(seen)}
    if op == "evict":
        kv, budget = case["kv_heads"], case["budget"]
        over = [n for n in _lens(case) if n > budget]
        # of the slots below the budget all stay that are sinks, and of the others the share that the rest of the budget leaves
        free = budget - case["sink"] - case["recent"]
        moves = sum((budget - case["sink"]) * (1.0 - max(0.0, min(1.0, free / max(1, n - case["sink"] - case["recent"])))) for n in over)
        return {"bytes": 16 * kv * sum(_lens(case)) + 4 * case["dim"] * e * kv * moves, "flops": 0}
    if op == "select":
        rows = case["groups"] * case["beams"]
        return {"bytes": rows * (case["vocab"] * e + 5) + case["groups"] * case["n_out"] * 13, "flops": 4 * rows * case["vocab"]}
    fill = case["tokens"] % case["page"]
    tail = 4 * case["dim"] * e * case["kv_heads"] * fill * case["layers"]
    return {"bytes": _extra(case) * tail + case["groups"] * case["beams"] * 8 * (-(-case["tokens"] // case["page"])), "flops": 0}


def _pool(case, layers, pages, gen):
    shape = (layers, pages, case["kv_heads"], case["page"], case["dim"])
    kind = DTYPES[case["dtype"]]
    return tuple(torch.empty(shape, device="cuda", dtype=kind).normal_(generator=gen) for _ in range(2))


def prepare(case, seed):
    """A program's pages, tables, lengths and handle, with what the step brings."""
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    op, kind = case["op"], DTYPES[case["dtype"]]
    state = {"case": dict(case)}
    if op == "select":
        groups, beams, vocab = case["groups"], case["beams"], case["vocab"]
        x = torch.randn((groups, beams, vocab), device="cuda", generator=gen) * 2.5
        # each beam has some tokens that it likes, and a share of the vocabulary that is banned
        liked = torch.randint(0, vocab, (groups, beams, 12), device="cuda", generator=gen)
        x.scatter_add_(2, liked, 9.0 + 4.0 * torch.rand((groups, beams, 12), device="cuda", generator=gen))
        banned = torch.randint(0, vocab, (groups, beams, 40), device="cuda", generator=gen)
        x.scatter_(2, banned, float("-inf"))
        state["logits"] = x.to(kind)
        state["scores"] = -3.0 - 4.0 * torch.rand((groups, beams), device="cuda", generator=gen)
        state["finished"] = (torch.rand((groups, beams), device="cuda", generator=gen) < 0.1).to(torch.uint8)
        state["eos"], state["pad"] = 2, 0
        if own:
            lc = importlib.import_module("lumen-rs_b200")
            state["beam"] = lc.BeamSearch(groups, beams, vocab, n_out=case["n_out"])
        return state
    if op == "reorder":
        groups, beams = case["groups"], case["beams"]
        width = -(-case["tokens"] // case["page"]) + 1
        shared = case["tokens"] // case["page"] // 2  # the prompt's pages: the same for all of a group's beams
        apart = width - shared
        pages = groups * (shared + beams * apart)
        at = torch.randperm(pages, device="cuda", generator=gen).to(torch.int32)
        head = at[: groups * shared].view(groups, 1, shared).expand(groups, beams, shared)
        tail = at[groups * shared:].view(groups, beams, apart)
        state["tables"] = torch.cat([head, tail], 2).reshape(groups * beams, width).contiguous()
        state["tables_out"] = torch.empty_like(state["tables"])
        state["lens"] = torch.full((groups,), case["tokens"], device="cuda", dtype=torch.int32)
        state["parents"] = torch.randint(0, beams, (groups, beams), device="cuda", generator=gen, dtype=torch.int32)
        state["k"], state["v"] = _pool(case, case["layers"], pages, gen)
        rows, heads = groups * beams, case["kv_heads"]
    else:
        rows = case["seqs"]
        width = -(-case["tokens"] // case["page"])
        pages = rows * width
        lens = torch.tensor(_lens(case), dtype=torch.int32, device="cuda")
        state["lens"] = lens[torch.randperm(rows, device="cuda", generator=gen)]
        state["tables"] = torch.randperm(pages, device="cuda", generator=gen).to(torch.int32).view(rows, width)
        state["k"], state["v"] = _pool(case, 1, pages, gen)
        heads, span = case.get("q_heads", case["kv_heads"]), width * case["page"]
        if op in ("attn", "weights"):
            state["q"] = (torch.randn((rows, heads, case["dim"]), device="cuda", generator=gen) * 1.5).to(kind)
            state["out"] = torch.empty_like(state["q"])
            state["scale"] = case["dim"] ** -0.5
        if op in ("weights", "evict"):
            # what earlier steps left: a few tokens hold most of the weight
            state["acc"] = torch.exp(2.0 * torch.randn((rows, case["kv_heads"], span), device="cuda", generator=gen))
            state["acc_out"] = torch.zeros_like(state["acc"])
        if op == "evict":
            # earlier evictions left the tokens out of order
            order = torch.rand((rows, case["kv_heads"], span), device="cuda", generator=gen)
            order = torch.where(torch.arange(span, device="cuda") < state["lens"].view(-1, 1, 1), order, 2.0)
            state["pos"] = order.argsort(-1).argsort(-1).to(torch.int32)
            state["pos_out"] = torch.zeros_like(state["pos"])
    if own:
        lc = importlib.import_module("lumen-rs_b200")
        state["cache"] = lc.PagedKvCache(state["k"], state["v"], max_seqs=rows, max_pages_per_seq=width, max_q_heads=heads)
    return state


def run(state):
    """One call, and what it wrote."""
    case = state["case"]
    op = case["op"]
    if op == "attn":
        if own:
            return state["cache"].attn(0, state["tables"], state["lens"], state["q"], state["scale"], window=case["window"], out=state["out"])
        return _attn(state)[0]
    if op == "weights":
        if own:
            out = state["cache"].attn_weights(0, state["tables"], state["lens"], state["q"], state["scale"], state["acc"], state["acc_out"],
                                              window=case["window"], out=state["out"])
            return {"out": out, "acc": state["acc_out"]}
        return _weights(state)
    if op == "evict":
        if own:
            state["cache"].evict(0, state["tables"], state["lens"], case["budget"], state["acc"], state["pos"], state["acc_out"], state["pos_out"],
                                 n_sink=case["sink"], n_recent=case["recent"])
            return {"k": state["k"], "v": state["v"], "acc": state["acc_out"], "pos": state["pos_out"]}
        return _evict(state)
    if op == "select":
        if own:
            scores, parents, tokens, finished = state["beam"].select(state["logits"], state["scores"], state["finished"], eos_id=state["eos"], pad_id=state["pad"])
            return {"scores": scores, "parents": parents, "tokens": tokens, "finished": finished}
        return _select(state)
    if own:
        state["cache"].reorder(state["tables"], state["lens"], state["parents"], state["tables_out"])
        return {"k": state["k"], "v": state["v"], "tables": state["tables_out"]}
    return _reorder(state)


def _rows(pool, tables):
    """[rows, kv heads, tokens, dim] in 32 bits."""
    x = pool[0][tables.long()].float()
    return x.transpose(1, 2).reshape(tables.shape[0], pool.shape[2], -1, pool.shape[4])


def _attn(state):
    """The attention's output, and the weights [rows, kv heads, queries a head, tokens]."""
    case, q = state["case"], state["q"]
    rows, kv = q.shape[0], case["kv_heads"]
    keys, values = _rows(state["k"], state["tables"]), _rows(state["v"], state["tables"])
    t = torch.arange(keys.shape[2], device=q.device)
    n = state["lens"].view(-1, 1, 1, 1)
    seen = (t < n) & (t >= n - (case["window"] or case["tokens"]))
    x = torch.matmul(q.float().view(rows, kv, -1, case["dim"]), keys.transpose(2, 3)) * state["scale"]
    x = torch.where(seen, x, float("-inf"))
    top = x.amax(-1, keepdim=True)
    p = torch.where(seen, torch.exp(x - top), 0.0)
    p = p / p.sum(-1, keepdim=True).clamp_min(1e-30)
    out = torch.matmul(p, values).reshape(q.shape).to(q.dtype)
    return out, p


def _weights(state):
    out, p = _attn(state)
    live = torch.arange(p.shape[3], device=p.device) < state["lens"].view(-1, 1, 1)
    return {"out": out, "acc": torch.where(live, state["acc"] + p.sum(2), 0.0)}


def _slots(case, tables, slot):
    """The pages and rows in them of slots [rows, kv heads, m]."""
    page = torch.gather(tables.long().unsqueeze(1).expand(-1, slot.shape[1], -1), 2, slot // case["page"])
    return page, slot % case["page"]


def _evict(state):
    case, acc, pos = state["case"], state["acc"], state["pos"]
    budget = case["budget"]
    t = torch.arange(acc.shape[2], device=acc.device)
    n = state["lens"].view(-1, 1, 1)
    live = t < n
    newest = torch.where(live, pos, -1).amax(-1, keepdim=True)
    held = (pos < case["sink"]) | (pos > newest - case["recent"])
    key = torch.where(live, torch.where(held, float("inf"), acc), float("-inf"))
    order = torch.sort(key, dim=-1, descending=True, stable=True).indices[..., :budget]
    stay = torch.zeros_like(live.expand_as(key)).scatter(2, order, True) & live
    hole, mover = ~stay & live & (t < budget), stay & (t >= budget)
    most = min(budget, acc.shape[2] - budget)
    dst = torch.sort(hole.to(torch.int8), dim=-1, descending=True, stable=True).indices[..., :most]
    src = torch.sort(mover.to(torch.int8), dim=-1, descending=True, stable=True).indices[..., :most]
    real = torch.arange(most, device=acc.device) < hole.sum(-1, keepdim=True)
    last = (n - 1).clamp_min(0).expand_as(dst)  # a pair that is none copies the last slot to itself: that is no hole where there are any
    src, dst = torch.where(real, src, last), torch.where(real, dst, last)
    new_acc = acc.scatter(2, dst, torch.gather(acc, 2, src))
    new_pos = pos.scatter(2, dst, torch.gather(pos, 2, src))
    gone = live & (t >= budget)
    heads = torch.arange(case["kv_heads"], device=acc.device).view(1, -1, 1)
    (sp, sr), (dp, dr) = _slots(case, state["tables"], src), _slots(case, state["tables"], dst)
    state["k"][0][dp, heads, dr] = state["k"][0][sp, heads, sr]
    state["v"][0][dp, heads, dr] = state["v"][0][sp, heads, sr]
    return {"k": state["k"], "v": state["v"], "acc": torch.where(gone | ~live, 0.0, new_acc), "pos": torch.where(live, torch.where(gone, -1, new_pos), 0)}


def _select(state):
    case, x = state["case"], state["logits"].float()
    beams, vocab, m = case["beams"], case["vocab"], case["n_out"]
    x = x - x.amax(-1, keepdim=True)
    z = state["scores"].unsqueeze(2) + (x - torch.log(torch.exp(x).sum(-1, keepdim=True)))
    done = state["finished"].bool().unsqueeze(2)
    only = torch.where(torch.arange(vocab, device=x.device) == state["pad"], state["scores"].unsqueeze(2), float("-inf"))
    z = torch.where(done, only, z)
    z = torch.where(torch.isnan(z), float("-inf"), z).flatten(1)
    z, at = torch.sort(z, dim=1, descending=True, stable=True)
    z, at = z[:, :m], at[:, :m]
    none = z == float("-inf")
    parents = torch.where(none, torch.arange(m, device=x.device) % beams, at // vocab)
    tokens = torch.where(none, state["pad"], at % vocab)
    finished = none | torch.gather(state["finished"].bool(), 1, parents) | (tokens == state["eos"])
    return {"scores": z.contiguous(), "parents": parents.int(), "tokens": tokens.int(), "finished": finished.to(torch.uint8)}


def _reorder(state):
    case, tables, parents = state["case"], state["tables"], state["parents"].long()
    groups, beams = parents.shape
    width = tables.shape[1]
    tables = tables.view(groups, beams, width).long()
    full, fill = (state["lens"] // case["page"]).long(), (state["lens"] % case["page"]).view(-1, 1)
    j = torch.arange(beams, device=parents.device)
    same = parents.unsqueeze(2) == parents.unsqueeze(1)
    later = (same & (j.view(-1, 1) > j)).any(2)  # an earlier beam has this parent too
    childless = ~(parents.unsqueeze(2) == j).any(1)
    spare = torch.sort(childless.to(torch.int8), dim=1, descending=True, stable=True).indices
    owner = torch.where(later, torch.gather(spare, 1, (later.cumsum(1) - 1).clamp_min(0)), parents)
    tails = torch.gather(tables, 2, full.clamp_max(width - 1).view(-1, 1, 1).expand(-1, beams, 1)).squeeze(2)
    src, dst = torch.gather(tails, 1, parents), torch.gather(tails, 1, owner)
    i = torch.arange(width, device=parents.device).view(1, 1, -1)
    at = full.view(-1, 1, 1)
    came = torch.gather(tables, 1, parents.unsqueeze(2).expand(-1, -1, width))
    out = torch.where(i < at, came, torch.where((i == at) & (fill.unsqueeze(2) > 0), dst.unsqueeze(2), tables))
    kept = torch.arange(case["page"], device=parents.device) < fill.expand(-1, beams).reshape(-1, 1)
    kept = kept.view(1, -1, 1, case["page"], 1)
    src, dst = src.reshape(-1), dst.reshape(-1)
    state["k"][:, dst] = torch.where(kept, state["k"][:, src], state["k"][:, dst])
    state["v"][:, dst] = torch.where(kept, state["v"][:, src], state["v"][:, dst])
    return {"k": state["k"], "v": state["v"], "tables": out.view(-1, width).int()}


def exact(case, seed):
    """From the definitions, one sequence (or row) after the other, in 64 bits."""
    state = prepare(case, seed)
    op = case["op"]
    if op in ("attn", "weights"):
        out = torch.zeros(state["q"].shape, dtype=torch.float64, device="cuda")
        acc = torch.zeros(state["acc"].shape, dtype=torch.float64, device="cuda") if op == "weights" else None
        share = case["q_heads"] // case["kv_heads"]
        for s, n in enumerate(state["lens"].tolist()):
            low = max(0, n - case["window"]) if case["window"] else 0
            if op == "weights":
                acc[s, :, :n] = state["acc"][s, :, :n].double()
            if not n:
                continue
            pages = state["tables"][s, : -(-n // case["page"])].long()
            for h in range(case["kv_heads"]):
                k = state["k"][0, pages, h].reshape(-1, case["dim"])[low:n].double()
                v = state["v"][0, pages, h].reshape(-1, case["dim"])[low:n].double()
                w = torch.softmax((k @ state["q"][s, h * share:(h + 1) * share].double().T).T * state["scale"], dim=1)
                out[s, h * share:(h + 1) * share] = w @ v
                if op == "weights":
                    acc[s, h, low:n] += w.sum(0)
        return {"out": out, "acc": acc} if op == "weights" else out
    if op == "select":
        scores = torch.full((case["groups"], case["n_out"]), float("-inf"), dtype=torch.float64)
        for g in range(case["groups"]):
            found = []
            for b in range(case["beams"]):
                if state["finished"][g, b]:
                    found.append(state["scores"][g, b].double().view(1))
                    continue
                z = torch.log_softmax(state["logits"][g, b].double(), 0) + state["scores"][g, b].double()
                found.append(torch.topk(z, min(case["n_out"], case["vocab"])).values)
            best = torch.sort(torch.cat(found), descending=True).values[: case["n_out"]].cpu()
            scores[g, : best.numel()] = best
        return {"scores": scores, "parents": None, "tokens": None, "finished": None}
    if op == "evict":
        k, v, budget = state["k"].double(), state["v"].double(), case["budget"]
        acc = torch.zeros(state["acc"].shape, dtype=torch.float64)
        for s, n in enumerate(state["lens"].tolist()):
            pages = state["tables"][s].long()
            for h in range(case["kv_heads"]):
                a, p = state["acc"][s, h, :n].double().tolist(), state["pos"][s, h, :n].tolist()
                if n > budget:
                    held = [x < case["sink"] or x > max(p) - case["recent"] for x in p]
                    stay = set(sorted(range(n), key=lambda t: (-math.inf if held[t] else -a[t], t))[:budget])
                    to, of = [t for t in range(budget) if t not in stay], sorted(t for t in stay if t >= budget)
                    for d, t in zip(to, of):
                        a[d] = a[t]
                    a[budget:] = [0.0] * (n - budget)
                    to, of = torch.tensor(to, dtype=torch.long, device="cuda"), torch.tensor(of, dtype=torch.long, device="cuda")
                    for x in (k, v):
                        x[0, pages[to // case["page"]], h, to % case["page"]] = x[0, pages[of // case["page"]], h, of % case["page"]]
                acc[s, h, :n] = torch.tensor(a, dtype=torch.float64)
        return {"k": k, "v": v, "acc": acc, "pos": None}
    return None  # the reordering moves values and computes none
