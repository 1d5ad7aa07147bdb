"""The uncompressed paged cache against its plain 64-bit forms: attention,
accumulated weights, append, eviction and reordering."""
import numpy as np
import pytest
import torch

import paged_ref as ref

pytestmark = pytest.mark.gpu


def make(lc, lens, heads, kv, dim, page, dtype, *, layers=2, layer=1, layout="phtd", offset=0, seed=0, spare=3, slack=1):
    width = max(1, max(-(-n // page) for n in lens)) + slack
    pages = sum(-(-n // page) for n in lens) + spare
    k, v = ref.pool(layers, pages, kv, page, dim, dtype, seed, layout, offset)
    tables = ref.tables_for(lens, page, pages, width, seed)
    rows = ref.fill_slots(k, v, layer, tables, lens, seed)
    cache = lc.PagedKvCache(k, v, max_seqs=len(lens), max_pages_per_seq=width, max_q_heads=heads)
    return cache, tables, torch.tensor(lens, dtype=torch.int32, device="cuda"), rows


def queries(n, heads, dim, dtype, seed, gain=1.0):
    g = torch.Generator().manual_seed(seed + 77)
    return (torch.randn((n, heads, dim), generator=g) * gain).to(ref.DTYPES[dtype]).cuda()


def check(out, want, dtype):
    got = out.double().cpu()
    assert not torch.isnan(got).any()
    err = (got - want).abs() - ref.RTOL[dtype] * want.abs()
    assert err.max().item() <= ref.ATOL, err.max().item()


LENS = [[1], [0, 1, 2], [15, 16, 17, 33], [300, 0, 7, 129, 64, 1000]]


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("heads,kv,dim,page", [(4, 2, 64, 16), (8, 1, 128, 32), (6, 2, 80, 20), (3, 3, 256, 64),
                                               (12, 1, 96, 8), (20, 1, 128, 16), (5, 5, 20, 7), (2, 1, 33, 16),
                                               (16, 2, 192, 256), (4, 4, 8, 1), (24, 3, 128, 48)])
@pytest.mark.parametrize("lens", LENS)
def test_attn_matches_plain(lc, gpu, dtype, heads, kv, dim, page, lens):
    cache, tables, ln, rows = make(lc, lens, heads, kv, dim, page, dtype)
    q = queries(len(lens), heads, dim, dtype, 1)
    out = cache.attn(1, tables, ln, q, dim ** -0.5)
    check(out, ref.attn(rows, q, dim ** -0.5)[0], dtype)
    assert cache.status() == lc.LC_OK


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("window", [1, 15, 64, 100, 5000])
def test_attn_window(lc, gpu, dtype, window):
    lens = [0, 1, 64, 65, 999, 2000]
    cache, tables, ln, rows = make(lc, lens, 8, 2, 128, 32, dtype)
    q = queries(len(lens), 8, 128, dtype, 2)
    check(cache.attn(1, tables, ln, q, 0.1, window=window), ref.attn(rows, q, 0.1, window)[0], dtype)


@pytest.mark.parametrize("layout,offset", [("pthd", 0), ("plhtd", 0), ("phtd", 1), ("phtd", 8)])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_attn_strides_and_alignment(lc, gpu, dtype, layout, offset):
    lens = [70, 3, 257]
    cache, tables, ln, rows = make(lc, lens, 8, 4, 64, 16, dtype, layout=layout, offset=offset)
    q = queries(3, 8, 64, dtype, 3)
    check(cache.attn(1, tables, ln, q, 0.125), ref.attn(rows, q, 0.125)[0], dtype)


@pytest.mark.parametrize("pool,qt,out", [("bf16", "f32", "f32"), ("f16", "f16", "f32"), ("bf16", "bf16", "f32"),
                                         ("f32", "bf16", "f16"), ("f16", "bf16", "bf16"), ("f32", "f32", "bf16")])
def test_attn_mixed_types(lc, gpu, pool, qt, out):
    lens = [500, 31]
    cache, tables, ln, rows = make(lc, lens, 8, 2, 128, 64, pool)
    q = queries(2, 8, 128, qt, 4)
    o = torch.full((2, 8, 128), float("nan"), dtype=ref.DTYPES[out], device="cuda")
    check(cache.attn(1, tables, ln, q, 0.08, out=o), ref.attn(rows, q, 0.08)[0], out)


def test_attn_q_at_odd_address(lc, gpu):
    lens = [500, 31]
    cache, tables, ln, rows = make(lc, lens, 8, 2, 128, 64, "bf16")
    q = queries(2, 8, 128, "bf16", 4)
    flat = torch.empty(q.numel() + 1, dtype=q.dtype, device="cuda")
    flat[1:] = q.view(-1)
    check(cache.attn(1, tables, ln, flat[1:].view(q.shape), 0.08), ref.attn(rows, q, 0.08)[0], "bf16")


@pytest.mark.parametrize("dtype,dim,heads,kv", [("bf16", 128, 8, 1), ("f16", 256, 4, 2), ("f32", 64, 3, 1)])
def test_attn_long_split(lc, gpu, dtype, dim, heads, kv):
    """One long sequence beside short ones: many partials of one item; peaked scores (gain 3)."""
    lens = [20011, 5, 0, 1203]
    cache, tables, ln, rows = make(lc, lens, heads, kv, dim, 64, dtype)
    q = queries(4, heads, dim, dtype, 5, gain=3.0)
    out = cache.attn(1, tables, ln, q, dim ** -0.5)
    check(out, ref.attn(rows, q, dim ** -0.5)[0], dtype)
    for _ in range(3):  # the order in which blocks finish changes nothing
        assert torch.equal(cache.attn(1, tables, ln, q, dim ** -0.5), out)


def test_attn_many_sequences(lc, gpu):
    """More sequences than threads of a block, mostly short and empty."""
    g = np.random.default_rng(8)
    lens = [int(x) for x in g.integers(0, 40, 700)]
    cache, tables, ln, rows = make(lc, lens, 2, 1, 64, 16, "bf16", layers=1, layer=0)
    q = queries(700, 2, 64, "bf16", 6)
    check(cache.attn(0, tables, ln, q, 0.125), ref.attn(rows, q, 0.125)[0], "bf16")


def test_attn_infinite_scores(lc, gpu):
    """A key row of -inf drops out; where no score is finite the row is zeros."""
    cache, tables, ln, rows = make(lc, [40, 16], 2, 1, 64, 16, "f32", layers=1, layer=0)
    q = queries(2, 2, 64, "f32", 7).abs()
    rows[0][0][0, 5] = -float("inf")
    cache.k_pages[0, int(tables[0, 0]), 0, 5] = -float("inf")
    cache.k_pages[0, int(tables[1, 0])] = -float("inf")
    out = cache.attn(0, tables, ln, q, 0.125)
    want = ref.attn(rows[:1], q[:1], 0.125)[0]
    check(out[:1], want, "f32")
    assert (out[1] == 0).all()


@pytest.mark.parametrize("dtype,dim", [("f32", 64), ("bf16", 128), ("f16", 80)])
@pytest.mark.parametrize("heads,kv", [(4, 4), (6, 2), (16, 2), (20, 1)])
@pytest.mark.parametrize("window,decay", [(0, 1.0), (50, 0.5)])
def test_weights_match_plain(lc, gpu, dtype, dim, heads, kv, window, decay):
    lens = [0, 1, 33, 64, 1500]
    cache, tables, ln, rows = make(lc, lens, heads, kv, dim, 16, dtype)
    q = queries(len(lens), heads, dim, dtype, 9)
    span = tables.shape[1] * 16 + 5
    acc = torch.rand((len(lens), kv, span), device="cuda")
    acc_out = torch.full_like(acc, 7.0)
    out = cache.attn_weights(1, tables, ln, q, dim ** -0.5, acc, acc_out, decay=decay, window=window)
    want, w = ref.attn(rows, q, dim ** -0.5, window)
    check(out, want, dtype)
    for s, n in enumerate(lens):
        add = w[s].view(kv, heads // kv, n).sum(1)
        got = acc_out[s, :, :n].double().cpu() - decay * acc[s, :, :n].double().cpu()
        # a weight's relative error is twice its score's absolute error (about 1e-5); acc rounds at 2^-24 of values below 22
        assert ((got - add).abs() <= 1e-4 * add + 2e-6).all()
        assert (acc_out[s, :, n:] == 7.0).all()
    same = acc.clone()
    cache.attn_weights(1, tables, ln, q, dim ** -0.5, same, decay=decay, window=window)
    for s, n in enumerate(lens):
        assert torch.equal(same[s, :, :n], acc_out[s, :, :n]) and torch.equal(same[s, :, n:], acc[s, :, n:])


@pytest.mark.parametrize("pool,src", [("bf16", "f32"), ("f16", "f16"), ("f32", "bf16"), ("bf16", "bf16")])
@pytest.mark.parametrize("n_tokens,dim,page", [(1, 128, 16), (37, 33, 8), (5, 256, 64)])
def test_append(lc, gpu, pool, src, n_tokens, dim, page):
    kv, lens = 3, [0, 1, page - 1, page, 2 * page + 3]
    width = -(-(max(lens) + n_tokens) // page)
    pages = len(lens) * width
    k, v = ref.pool(2, pages, kv, page, dim, pool, 0)
    tables = torch.randperm(pages, device="cuda").to(torch.int32).view(len(lens), width)
    cache = lc.PagedKvCache(k, v, max_seqs=len(lens), max_pages_per_seq=width, max_q_heads=kv)
    ln = torch.tensor(lens, dtype=torch.int32, device="cuda")
    keys = torch.randn((len(lens), kv, n_tokens, dim), device="cuda").to(ref.DTYPES[src])
    values = torch.randn((len(lens), kv, n_tokens, dim), device="cuda").to(ref.DTYPES[src])
    pos = torch.full((len(lens), kv, width * page), -9, dtype=torch.int32, device="cuda")
    pos0 = ln + 100
    cache.append(1, tables, ln, keys, values, pos, pos0)
    assert torch.isnan(k[0].float()).all()
    for pool_t, new in ((k, keys), (v, values)):
        flat = pool_t[1][tables.long()].transpose(1, 2).reshape(len(lens), kv, width * page, dim)
        for s, n in enumerate(lens):
            assert torch.equal(flat[s, :, n:n + n_tokens], new[s].to(k.dtype))
            assert torch.isnan(flat[s, :, :n].float()).all() and torch.isnan(flat[s, :, n + n_tokens:].float()).all()
    for s, n in enumerate(lens):
        assert (pos[s, :, n:n + n_tokens].cpu() == torch.arange(n_tokens) + n + 100).all()
        assert (pos[s, :, :n] == -9).all() and (pos[s, :, n + n_tokens:] == -9).all()


def run_evict(lc, lens, budget, sink, recent, *, kv=2, dim=64, page=16, dtype="bf16", layout="phtd", offset=0, acc=None,
              seed=3, inplace=False):
    cache, tables, ln, rows = make(lc, lens, kv, kv, dim, page, dtype, layout=layout, offset=offset, seed=seed)
    span = tables.shape[1] * page + 3
    g = torch.Generator().manual_seed(seed)
    if acc is None:
        acc = torch.exp(2 * torch.randn((len(lens), kv, span), generator=g))
    acc = acc.cuda()
    pos = torch.stack([torch.stack([torch.randperm(span, generator=g) for _ in range(kv)]) for _ in lens]).to(torch.int32)
    for s, n in enumerate(lens):  # positions 0 .. n - 1 in some order
        pos[s, :, :n] = torch.argsort(torch.argsort(pos[s, :, :n], dim=1), dim=1).to(torch.int32)
    pos = pos.cuda()
    a0, p0 = acc.cpu(), pos.cpu()
    k0, v0 = cache.k_pages.clone(), cache.v_pages.clone()
    acc_out = acc if inplace else torch.full_like(acc, 5.0)
    pos_out = pos if inplace else torch.full_like(pos, 5)
    cache.evict(1, tables, ln, budget, acc, pos, acc_out, pos_out, n_sink=sink, n_recent=recent)
    moved = 0
    for s, n in enumerate(lens):
        for h in range(kv):
            a, p, pairs = ref.evict_row(a0[s, h, :n].tolist(), p0[s, h, :n].tolist(), budget, sink, recent)
            got = acc_out[s, h, :n].cpu()
            np.testing.assert_array_equal(got.numpy(), np.array(a, np.float32))
            assert pos_out[s, h, :n].tolist() == p
            for at, to in pairs:
                sp, dp = int(tables[s, at // page]), int(tables[s, to // page])
                k0[1, dp, h, to % page] = k0[1, sp, h, at % page]
                v0[1, dp, h, to % page] = v0[1, sp, h, at % page]
            moved += len(pairs)
    if not inplace:
        for s, n in enumerate(lens):
            assert (acc_out[s, :, n:] == 5.0).all() and (pos_out[s, :, n:] == 5).all()
    else:
        for s, n in enumerate(lens):
            np.testing.assert_array_equal(acc_out[s, :, n:].cpu().numpy(), a0[s, :, n:].numpy())
    assert torch.equal(cache.k_pages.contiguous().view(torch.uint8), k0.contiguous().view(torch.uint8))
    assert torch.equal(cache.v_pages.contiguous().view(torch.uint8), v0.contiguous().view(torch.uint8))
    assert cache.status() == lc.LC_OK
    return moved


@pytest.mark.parametrize("lens,budget,sink,recent", [([0, 1, 5], 3, 0, 0), ([2], 1, 0, 1), ([17, 64, 65], 64, 4, 16),
                                                     ([300, 100], 37, 4, 33), ([1025, 900], 1024, 4, 128),
                                                     ([5000, 40, 2047], 900, 0, 0), ([9001], 8000, 10, 5)])
@pytest.mark.parametrize("inplace", [False, True])
def test_evict_matches_plain(lc, gpu, lens, budget, sink, recent, inplace):
    run_evict(lc, lens, budget, sink, recent, inplace=inplace)


@pytest.mark.parametrize("dtype,dim,layout,offset", [("f32", 128, "pthd", 0), ("f16", 33, "phtd", 0), ("bf16", 256, "plhtd", 0),
                                                     ("f32", 20, "phtd", 1), ("bf16", 64, "phtd", 3)])
def test_evict_layouts(lc, gpu, dtype, dim, layout, offset):
    assert run_evict(lc, [200, 77], 50, 2, 10, dtype=dtype, dim=dim, layout=layout, offset=offset) > 0


def test_evict_ties_and_odd_weights(lc, gpu):
    """Equal weights keep the lower slots; NaN goes first, then -inf; -0 equals 0; +inf stays."""
    n, kv = 3000, 2
    acc = torch.zeros((1, kv, 3100))
    acc[0, 1, ::3] = -0.0
    acc[0, 0, 5:2000:7] = float("nan")
    acc[0, 0, 6:2000:7] = -float("inf")
    acc[0, 0, 2500:2510] = float("inf")
    acc[0, 1, 100:2900:11] = 1e-42
    assert run_evict(lc, [n], 1200, 0, 0, acc=acc[:, :, :span_for(n)], kv=kv) > 100


def span_for(n, page=16, slack=1):
    return (-(-n // page) + slack) * page + 3


def test_evict_long_row(lc, gpu):
    """A row over several blocks of a cluster, with runs of equal weights across their borders."""
    n = 40000
    g = torch.Generator().manual_seed(4)
    acc = torch.randint(0, 5, (1, 1, span_for(n, 64)), generator=g).float()
    assert run_evict(lc, [n], 15000, 4, 100, kv=1, page=64, acc=acc) > 1000


def test_evict_keys_beyond_shared_memory(lc, gpu):
    """So long that a row's keys do not fit the cluster's shared memory."""
    n = 340000
    assert run_evict(lc, [n], 2000, 4, 100, kv=1, dim=8, page=256) > 1000


@pytest.mark.parametrize("dtype,dim,page,layout", [("bf16", 128, 16, "phtd"), ("f16", 33, 7, "phtd"), ("f32", 64, 32, "pthd"),
                                                   ("bf16", 80, 100, "plhtd")])
@pytest.mark.parametrize("groups,beams", [(1, 1), (1, 4), (3, 8), (2, 33)])
def test_reorder_matches_plain(lc, gpu, dtype, dim, page, layout, groups, beams):
    g = np.random.default_rng(groups * 100 + beams)
    for lens in ([page * 2 + 1] * groups, [page] * groups, [0] * groups, [int(x) for x in g.integers(0, 3 * page, groups)]):
        width, kv = 4, 2
        pages = groups * beams * width
        k, v = ref.pool(3, pages, kv, page, dim, dtype, 0, layout)
        for t in (k, v):
            t.copy_(torch.randn(t.shape, device="cuda"))
        cache = lc.PagedKvCache(k, v, max_seqs=groups * beams, max_pages_per_seq=width, max_q_heads=kv)
        tables = g.permutation(pages).astype(np.int32).reshape(groups * beams, width)
        parents = g.integers(0, beams, (groups, beams)).astype(np.int32)
        want, copies = ref.reorder(tables, lens, parents, page)
        k0, v0 = k.clone(), v.clone()
        for src, dst, fill in copies:
            k0[:, dst, :, :fill] = k0[:, src, :, :fill]
            v0[:, dst, :, :fill] = v0[:, src, :, :fill]
        out = cache.reorder(torch.from_numpy(tables).cuda(), torch.tensor(lens, dtype=torch.int32, device="cuda"),
                            torch.from_numpy(parents).cuda())
        np.testing.assert_array_equal(out.cpu().numpy(), want)
        assert torch.equal(k, k0) and torch.equal(v, v0)
        assert cache.status() == lc.LC_OK


def test_other_streams_and_graph(lc, gpu):
    """Calls on a side stream after the current one, and a captured call replayed with other lengths."""
    lens = [700, 90]
    cache, tables, ln, rows = make(lc, lens, 8, 2, 128, 32, "bf16")
    q = queries(2, 8, 128, "bf16", 11)
    want = ref.attn(rows, q, 0.1)[0]
    first = cache.attn(1, tables, ln, q, 0.1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = cache.attn(1, tables, ln, q, 0.1)
    third = cache.attn(1, tables, ln, q, 0.1)
    torch.cuda.synchronize()
    check(first, want, "bf16")
    assert torch.equal(first, second) and torch.equal(first, third)
    graph = torch.cuda.CUDAGraph()
    out = torch.empty_like(q)
    with torch.cuda.graph(graph):
        cache.attn(1, tables, ln, q, 0.1, out=out)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, first)
    ln.copy_(torch.tensor([650, 3], dtype=torch.int32))
    graph.replay()
    torch.cuda.synchronize()
    check(out, ref.attn([(k[:, :n], v[:, :n]) for (k, v), n in zip(rows, (650, 3))], q, 0.1)[0], "bf16")


def test_refusals(lc, gpu):
    k = torch.zeros((1, 4, 2, 16, 64), dtype=torch.bfloat16, device="cuda")
    cache = lc.PagedKvCache(k, k.clone(), max_seqs=2, max_pages_per_seq=2, max_q_heads=8)
    tables = torch.zeros((2, 2), dtype=torch.int32, device="cuda")
    ln = torch.ones(2, dtype=torch.int32, device="cuda")
    q = torch.zeros((2, 8, 64), dtype=torch.bfloat16, device="cuda")
    acc, pos = torch.zeros((2, 2, 32), device="cuda"), torch.zeros((2, 2, 32), dtype=torch.int32, device="cuda")

    def refused(f, *args, **kw):
        with pytest.raises(lc.LumenError) as e:
            f(*args, **kw)
        assert e.value.code == lc.LC_ERR_INVALID
        return str(e.value)

    refused(cache.attn, 1, tables, ln, q, 1.0)  # layer
    refused(cache.attn, 0, tables, ln, q[:, :7].contiguous(), 1.0)  # heads
    refused(cache.attn, 0, tables, ln, torch.zeros((2, 16, 64), dtype=q.dtype, device="cuda"), 1.0)
    refused(cache.attn, 0, tables, ln, q, float("nan"))
    refused(cache.attn, 0, tables, ln, q, 1.0, window=-1)
    wide = torch.zeros((2, 3), dtype=torch.int32, device="cuda")
    refused(cache.attn, 0, wide, ln, q, 1.0)
    refused(cache.attn_weights, 0, tables, ln, q, 1.0, acc[:, :, :31].contiguous())
    refused(cache.attn_weights, 0, tables, ln, q, 1.0, acc, decay=1.5)
    refused(cache.evict, 0, tables, ln, 0, acc, pos)
    refused(cache.evict, 0, tables, ln, 8, acc, pos, n_sink=4, n_recent=5)
    parents = torch.zeros((1, 2), dtype=torch.int32, device="cuda")
    refused(cache.reorder, tables, ln[:1].contiguous(), parents, tables)
    for bad in (q.cpu(), q.float().double(), q[:, :, :32], q.transpose(0, 1)):
        with pytest.raises((ValueError, TypeError)):
            cache.attn(0, tables, ln, bad, 1.0)
    with pytest.raises((ValueError, TypeError)):
        cache.attn(0, tables.long(), ln, q, 1.0)
    with pytest.raises((ValueError, TypeError)):
        cache.attn(0, tables.cpu(), ln, q, 1.0)
    # host pointers at the C entry
    L = lc.lib()
    host = np.zeros((2, 8, 64), np.float32)
    assert L.lc_paged_attn(cache._h, 0, 2, tables.data_ptr(), 2, ln.data_ptr(), host.ctypes.data, 0, 8, 1.0, 0, q.data_ptr(), 1,
                           None) == lc.LC_ERR_INVALID
    assert L.lc_paged_attn(None, 0, 2, tables.data_ptr(), 2, ln.data_ptr(), q.data_ptr(), 1, 8, 1.0, 0, q.data_ptr(), 1,
                           None) == lc.LC_ERR_INVALID
    with pytest.raises(lc.LumenError):  # overlapping rows
        lc.PagedKvCache(k[:, :1].expand(1, 4, 2, 16, 64), k[:, :1].expand(1, 4, 2, 16, 64), max_seqs=1, max_pages_per_seq=1,
                        max_q_heads=2)
    big = torch.zeros((1, 1, 1, 1, 264), device="cuda")
    with pytest.raises(lc.LumenError):
        lc.PagedKvCache(big, big.clone(), max_seqs=1, max_pages_per_seq=1, max_q_heads=1)


@pytest.mark.parametrize("what", ["len", "negative", "page", "page_low", "parent"])
def test_status_tells_of_bad_tables(lc, gpu, what):
    """Lengths, pages and parents out of range are not followed, and told."""
    k = torch.zeros((1, 4, 2, 16, 64), dtype=torch.bfloat16, device="cuda")
    cache = lc.PagedKvCache(k, k.clone(), max_seqs=2, max_pages_per_seq=2, max_q_heads=2)
    tables = torch.tensor([[0, 1], [2, 3]], dtype=torch.int32, device="cuda")
    ln = torch.tensor([20, 20], dtype=torch.int32, device="cuda")
    parents = torch.tensor([[0, 0]], dtype=torch.int32, device="cuda")
    assert cache.status() == lc.LC_OK
    if what == "len":
        ln[1] = 33
    elif what == "negative":
        ln[0] = -1
    elif what == "page":
        tables[1, 1] = 4
    elif what == "page_low":
        tables[0, 1] = -1
    else:
        parents[0, 1] = 2
    if what == "parent":
        cache.reorder(tables, ln[:1].contiguous(), parents)
    else:
        cache.attn(0, tables, ln, torch.zeros((2, 2, 64), dtype=torch.bfloat16, device="cuda"), 1.0)
    torch.cuda.synchronize()
    assert cache.status() == lc.LC_ERR_INVALID


def test_overlaps_are_refused(lc, gpu):
    """Outputs may be their inputs where the header says so, and never a part of them."""
    k = torch.zeros((1, 4, 2, 16, 64), dtype=torch.bfloat16, device="cuda")
    cache = lc.PagedKvCache(k, k.clone(), max_seqs=2, max_pages_per_seq=2, max_q_heads=2)
    tables = torch.zeros((2, 2), dtype=torch.int32, device="cuda")
    ln = torch.ones(2, dtype=torch.int32, device="cuda")
    q = torch.zeros((3, 2, 64), dtype=torch.bfloat16, device="cuda")
    acc, pos = torch.zeros((3, 2, 32), device="cuda"), torch.zeros((3, 2, 32), dtype=torch.int32, device="cuda")
    for f, args in ((cache.attn, (0, tables, ln, q[:2], 1.0)), ):
        for out in (q[:2], q[1:]):
            with pytest.raises(lc.LumenError):
                f(*args, out=out)
    with pytest.raises(lc.LumenError):
        cache.attn_weights(0, tables, ln, q[:2], 1.0, acc[:2], acc[1:])
    with pytest.raises(lc.LumenError):
        cache.evict(0, tables, ln, 8, acc[:2], pos[:2], acc[1:])
    with pytest.raises(lc.LumenError):
        cache.evict(0, tables, ln, 8, acc[:2], pos[:2], None, pos[1:])
    with pytest.raises(lc.LumenError):
        cache.evict(0, tables, ln, 8, acc[:2], pos[:2], pos_out=acc.view(torch.int32)[:2])


@pytest.mark.parametrize("dtype,dim", [("bf16", 128), ("f32", 64), ("f16", 40)])
def test_offsets_past_32_bits(lc, gpu, dtype, dim):
    """Pages whose elements lie beyond 2^32 of the pool: attention, append, eviction, reordering."""
    page, kv = 64, 2
    need = (1 << 32) // (kv * page * dim) + 40
    k, v = (torch.empty((1, need, kv, page, dim), dtype=ref.DTYPES[dtype], device="cuda") for _ in range(2))
    lens = [1000, 130]
    tables = torch.full((2, 17), -1, dtype=torch.int32)
    tables[0, :16] = torch.arange(need - 1, need - 17, -1, dtype=torch.int32)
    tables[1, :4] = torch.tensor([need - 20, 3, need - 30, need - 33], dtype=torch.int32)
    tables = tables.cuda()
    rows = ref.fill_slots(k, v, 0, tables, lens, 1)
    ln = torch.tensor(lens, dtype=torch.int32, device="cuda")
    cache = lc.PagedKvCache(k, v, max_seqs=2, max_pages_per_seq=17, max_q_heads=4)
    q = queries(2, 4, dim, dtype, 2)
    check(cache.attn(0, tables, ln, q, dim ** -0.5), ref.attn(rows, q, dim ** -0.5)[0], dtype)
    new = torch.randn((2, kv, 1, dim), device="cuda").to(k.dtype)
    cache.append(0, tables, ln, new, new)
    for s, n in enumerate(lens):
        assert torch.equal(k[0, int(tables[s, n // page]), :, n % page], new[s, :, 0])
    span = 17 * page
    acc = torch.rand((2, kv, span), device="cuda")
    pos = torch.arange(span, dtype=torch.int32, device="cuda").expand(2, kv, span).contiguous()
    a0 = acc.cpu()
    before = [k[0, tables[s, :-(-n // page)].long()].clone() for s, n in enumerate(lens)]
    cache.evict(0, tables, ln, 100, acc, pos)
    for s, n in enumerate(lens):
        for h in range(kv):
            _, _, pairs = ref.evict_row(a0[s, h, :n].tolist(), list(range(n)), 100, 0, 0)
            for at, to in pairs:
                assert torch.equal(k[0, int(tables[s, to // page]), h, to % page], before[s][at // page, h, at % page])
    tails = k[0, tables[:, 1].long()].clone()
    out = cache.reorder(tables, torch.tensor([100], dtype=torch.int32, device="cuda"),
                        torch.zeros((1, 2), dtype=torch.int32, device="cuda"))
    assert out[1, 0] == tables[0, 0] and torch.equal(k[0, int(tables[1, 1]), :, :36], tails[0, :, :36])
    assert cache.status() == lc.LC_OK


@pytest.mark.parametrize("pool,qt,dim,heads,kv,page,window", [
    ("bf16", "f32", 64, 10, 2, 16, 0), ("f16", "f32", 136, 4, 1, 24, 100), ("bf16", "f16", 256, 3, 1, 8, 0),
    ("f16", "bf16", 40, 4, 4, 7, 33), ("bf16", "f32", 100, 8, 2, 16, 0)])
def test_attn_queries_of_another_type(lc, gpu, pool, qt, dim, heads, kv, page, window):
    """16-bit pools whose slots outside the sequences hold NaN."""
    lens = [0, 1, 17, 333, 1200]
    cache, tables, ln, rows = make(lc, lens, heads, kv, dim, page, pool)
    q = queries(len(lens), heads, dim, qt, 4)
    out = torch.empty((len(lens), heads, dim), device="cuda")
    check(cache.attn(1, tables, ln, q, dim ** -0.5, window=window, out=out), ref.attn(rows, q, dim ** -0.5, window)[0],
          "f32")
    assert cache.status() == lc.LC_OK


@pytest.mark.parametrize("pool", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("src", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("dim,shift", [(128, 0), (128, 1), (128, 4), (200, 0), (36, 0)])
def test_append_types_and_alignment(lc, gpu, pool, src, dim, shift):
    """Sources at odd addresses, rows of odd 16-byte units, a length beyond the table."""
    k, v = ref.pool(1, 12, 2, 16, dim, pool, 0)
    cache = lc.PagedKvCache(k, v, max_seqs=3, max_pages_per_seq=4, max_q_heads=2)
    tables = torch.randperm(12, device="cuda").to(torch.int32).view(3, 4)
    lens = [13, 0, 40]
    ln = torch.tensor(lens, dtype=torch.int32, device="cuda")
    new = []
    for _ in range(2):
        flat = torch.randn(3 * 2 * 25 * dim + shift, device="cuda").to(ref.DTYPES[src])
        new.append(flat[shift:].view(3, 2, 25, dim))
    cache.append(0, tables, ln, *new)
    for pool_t, x in zip((k, v), new):
        flat = pool_t[0][tables.long()].transpose(1, 2).reshape(3, 2, 64, dim)
        for s, n in enumerate(lens):
            fit = min(25, 64 - n)
            assert torch.equal(flat[s, :, n:n + fit], x[s, :, :fit].to(k.dtype))
            assert torch.isnan(flat[s, :, :n].float()).all() and torch.isnan(flat[s, :, n + fit:].float()).all()
    assert cache.status() == lc.LC_ERR_INVALID  # sequence 2's last token is past its table


def test_weights_of_empty_sequences(lc, gpu):
    """No slot anywhere: the output's zeros are there when the call's work on the stream is done."""
    cache, tables, ln, rows = make(lc, [0, 0], 4, 2, 64, 16, "bf16")
    tables = torch.zeros((2, 1), dtype=torch.int32, device="cuda")
    acc = torch.ones((2, 2, 16), device="cuda")
    q = queries(2, 4, 64, "bf16", 1)
    for _ in range(20):
        out = torch.full_like(q, 3.0)
        cache.attn_weights(0, tables, ln, q, 1.0, acc, out=out)
        assert (out.clone() == 0).all() and (acc == 1).all()


@pytest.mark.parametrize("lens,budget", [([13000], 12999), ([13000, 9, 12500, 0], 3000), ([30000, 25001], 9000),
                                         ([60000], 20000)])
@pytest.mark.parametrize("inplace", [False, True])
def test_evict_rows_of_a_cluster(lc, gpu, lens, budget, inplace):
    """Rows of 2, 4 and 8 blocks, ragged, some of no more than the budget, with equal weights."""
    g = torch.Generator().manual_seed(len(lens))
    acc = torch.randint(0, 900, (len(lens), 2, span_for(max(lens), 64)), generator=g).float()
    run_evict(lc, lens, budget, 4, 100, kv=2, page=64, dim=8, acc=acc, inplace=inplace)


def two_slots(lc, dtype, dim, page, low, high):
    """Sequences of two slots: one of V 0 and one of V 1, whose score is `low` to `high` smaller in log2
    (head i's query picks dimension i, so scores are single products). The f32 outputs, and p / (1 + p) in f64."""
    seqs, heads = 48, 8
    cache, tables, ln, _ = make(lc, [2] * seqs, heads, 1, dim, page, dtype, layers=1, layer=0)
    g = torch.Generator().manual_seed(dim + page)
    less = ((low + (high - low) * torch.rand((seqs, heads), generator=g)) / 1.4426950408889634).to(ref.DTYPES[dtype])
    for pool_t, first, second in ((cache.k_pages, 0.0, -less), (cache.v_pages, 0.0, torch.ones_like(less))):
        for s in range(seqs):
            pool_t[0, int(tables[s, 0]), 0, :2] = first
            pool_t[0, int(tables[s, 0]), 0, 1, :heads] = second[s].cuda()
    q = torch.zeros((seqs, heads, dim), dtype=ref.DTYPES[dtype], device="cuda")
    q[:, range(heads), range(heads)] = 1.0
    out = cache.attn(0, tables, ln, q, 1.0, out=torch.empty((seqs, heads, dim), device="cuda"))
    p = torch.exp(-less.double())
    return out[:, range(heads), range(heads)].double().cpu(), p / (1 + p)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("dim,page", [(64, 16), (128, 7), (128, 8), (192, 16), (256, 16), (256, 3)])
def test_attn_weights_keep_24_bits(lc, gpu, dtype, dim, page):
    """A score below 8 (log2) is off by its factor's and its product's rounding, 8 * 2^-24 each, a weight
    by ln 2 of that, 2^-22 of exp2 and 2^-24 three times (sum, reciprocal, product): 1.2e-6 in all, below 2^-19."""
    got, want = two_slots(lc, dtype, dim, page, 0.0, 8.0)
    assert ((got - want).abs() <= 2.0 ** -19 * want).all()


@pytest.mark.parametrize("dim,page", [(64, 16), (128, 7), (256, 16)])
@pytest.mark.parametrize("low,high", [(8.0, 18.0), (18.0, 28.0)])
def test_attn_small_weights_under_a_large_one(lc, gpu, dim, page, low, high):
    """f16: a slot far below one whose V is 0. Scores below 28: 28 * 2^-24 twice, times ln 2, and 2^-22 and 3 * 2^-24
    as above, 2.8e-6, below 2^-18; two parts: 2^-22; and 2^-40 of the largest weight, two of them for two parts."""
    got, want = two_slots(lc, "f16", dim, page, low, high)
    assert ((got - want).abs() <= (2.0 ** -18 + 2.0 ** -22) * want + 2.0 ** -39).all()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_captured_calls_after_larger_ones(lc, gpu, dtype):
    """Graphs of attn_weights and evict of two sequences, replayed after calls of the same handle that need
    more workspace and after those of another handle, whose answers they leave alone."""
    heads, kv, dim, page, lens = 8, 2, 64, 16, [2000, 1500, 90, 70]
    cache, tables, ln, _ = make(lc, lens, heads, kv, dim, page, dtype, seed=5)
    span = tables.shape[1] * page
    q = queries(4, heads, dim, dtype, 3)
    g = torch.Generator().manual_seed(6)
    acc = torch.rand((4, kv, span), generator=g).cuda()
    pos = torch.arange(span, dtype=torch.int32, device="cuda").expand(4, kv, span).contiguous()
    k0, v0 = cache.k_pages.clone(), cache.v_pages.clone()

    class Call:
        """attn_weights or evict of the rows from `first` on of a handle, and all that it wrote."""

        def __init__(self, handle, name, first, budget=0):
            self.handle, self.name, self.budget = handle, name, budget
            self.t, self.n, self.q, self.acc, self.pos = (x[first:].clone() for x in (tables, ln, q, acc, pos))
            self.out, self.acc_out, self.pos_out = (torch.empty_like(x) for x in (self.q, self.acc, self.pos))

        def reset(self):
            self.handle.k_pages.copy_(k0)
            self.handle.v_pages.copy_(v0)
            for x in (self.out, self.acc_out, self.pos_out):
                x.fill_(3)

        def run(self):
            if self.name == "weights":
                self.handle.attn_weights(1, self.t, self.n, self.q, 0.125, self.acc, self.acc_out, out=self.out)
            else:
                self.handle.evict(1, self.t, self.n, self.budget, self.acc, self.pos, self.acc_out, self.pos_out)

        def wrote(self):
            torch.cuda.synchronize()
            k, v = self.handle.k_pages, self.handle.v_pages
            return [x.clone() for x in (self.out, self.acc_out, self.pos_out, k.contiguous().view(torch.uint8),
                                        v.contiguous().view(torch.uint8))]

        def eager(self):
            self.reset()
            self.run()
            return self.wrote()

    small = [Call(cache, "weights", 2), Call(cache, "evict", 2, 40), Call(cache, "evict", 2, 60)]
    want = [c.eager() for c in small]
    graphs = []
    for c in small:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            c.run()
    for c in (Call(cache, "weights", 0), Call(cache, "evict", 0, 700)):
        c.eager()
    other = lc.PagedKvCache(k0.clone(), v0.clone(), max_seqs=4, max_pages_per_seq=tables.shape[1], max_q_heads=heads)
    theirs = [Call(other, "weights", 1), Call(other, "evict", 1, 300), Call(other, "weights", 0), Call(other, "evict", 0, 700)]
    wanted = [c.eager() for c in theirs]
    for _ in range(2):
        for c, graph, w in zip(small, graphs, want):
            c.reset()
            graph.replay()
            assert all(torch.equal(a, b) for a, b in zip(c.wrote(), w))
        for c, w in zip(theirs, wanted):
            assert all(torch.equal(a, b) for a, b in zip(c.eager(), w))


def test_captured_append_and_reorder(lc, gpu):
    """Graphs of the two calls without a workspace do what the calls do."""
    k, v = ref.pool(2, 16, 2, 16, 64, "bf16", 0)
    for x in (k, v):
        x.copy_(torch.randn(x.shape, device="cuda"))
    cache = lc.PagedKvCache(k, v, max_seqs=4, max_pages_per_seq=4, max_q_heads=2)
    tables = torch.randperm(16, device="cuda").to(torch.int32).view(4, 4)
    ln = torch.tensor([37, 37, 37, 37], dtype=torch.int32, device="cuda")
    parents = torch.tensor([[2, 0, 2, 2]], dtype=torch.int32, device="cuda")
    new = torch.randn((4, 2, 1, 64), device="cuda").to(k.dtype)
    k0, v0, out = k.clone(), v.clone(), torch.empty_like(tables)

    def calls():
        cache.reorder(tables, ln[:1], parents, out)
        cache.append(0, out, ln, new, new)

    calls()
    want = [x.clone() for x in (out, k, v)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        calls()
    for _ in range(2):
        for x, x0 in ((k, k0), (v, v0)):
            x.copy_(x0)
        out.fill_(-1)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip((out, k, v), want))


def test_order_with_the_last_stream_in_capture(lc, gpu):
    """The last call's stream is being captured: a call on another stream runs at once, outside of that capture."""
    lens = [700, 90]
    cache, tables, ln, _ = make(lc, lens, 8, 2, 128, 32, "bf16")
    q = queries(2, 8, 128, "bf16", 11)
    want = cache.attn(1, tables, ln, q, 0.1)
    torch.cuda.synchronize()
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    first, inside, outside = (torch.zeros_like(q) for _ in range(3))
    torch.cuda.synchronize()
    cache.attn(1, tables, ln, q, 0.1, out=first, stream=a)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=a):
        cache.attn(1, tables, ln, q, 0.1, out=inside, stream=a)
        cache.attn(1, tables, ln, q, 0.1, out=outside, stream=b)
    torch.cuda.synchronize()
    assert torch.equal(first, want) and torch.equal(outside, want) and (inside == 0).all()
    outside.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(inside, want) and (outside == 0).all()


@pytest.mark.parametrize("handle", ["paged", "beam"])
def test_order_after_a_destroyed_stream(lc, gpu, handle):
    """Streams that are destroyed between the calls, whose values later ones may be given again."""
    import ctypes

    cudart = torch.cuda.cudart()
    lens = [700, 90]
    cache, tables, ln, _ = make(lc, lens, 8, 2, 128, 32, "bf16")
    q = queries(2, 8, 128, "bf16", 11)
    beam = lc.BeamSearch(2, 4, 30011)
    x, scores = torch.randn((2, 4, 30011), device="cuda"), torch.zeros((2, 4), device="cuda")

    def call(stream=None):
        if handle == "paged":
            return [cache.attn(1, tables, ln, q, 0.1, stream=stream)]
        return beam.select(x, scores, stream=stream)

    want = call()
    torch.cuda.synchronize()
    for _ in range(4):
        raw = ctypes.c_ulonglong()
        assert int(cudart.cudaStreamCreate(ctypes.addressof(raw))) == 0
        got = [call(raw.value)]
        torch.cuda.ExternalStream(raw.value).synchronize()
        assert int(cudart.cudaStreamDestroy(raw.value)) == 0
        got.append(call())
        torch.cuda.synchronize()
        for g in got:
            assert all(torch.equal(u, w) for u, w in zip(g, want))


def test_calls_on_streams_in_turn(lc, gpu):
    """Append, attention and eviction of one handle, each on another stream than the call before, no other wait between."""
    lens = [5000, 3000]
    cache, tables, ln, _ = make(lc, lens, 8, 2, 128, 32, "bf16")
    span = tables.shape[1] * 32
    new = torch.randn((2, 2, 1, 128), device="cuda").to(torch.bfloat16)
    q = queries(2, 8, 128, "bf16", 12)
    acc = torch.rand((2, 2, span), device="cuda")
    pos = torch.arange(span, dtype=torch.int32, device="cuda").expand(2, 2, span).contiguous()
    streams = [torch.cuda.Stream() for _ in range(3)]
    k0, v0 = cache.k_pages.clone(), cache.v_pages.clone()
    n1, n2 = ln + 1, torch.clamp(ln + 1, max=1000)
    outs = []
    for order in ([None] * 4, [streams[0], None, streams[1], streams[2]], [streams[2], streams[0], streams[1], None]):
        cache.k_pages.copy_(k0)
        cache.v_pages.copy_(v0)
        a, p, out = acc.clone(), pos.clone(), torch.empty_like(q)
        torch.cuda.synchronize()
        cache.append(1, tables, ln, new, new, stream=order[0])
        cache.attn_weights(1, tables, n1, q, 0.1, a, stream=order[1], out=torch.empty_like(q))
        cache.evict(1, tables, n1, 1000, a, p, n_recent=10, stream=order[2])
        cache.attn(1, tables, n2, q, 0.1, out=out, stream=order[3])
        torch.cuda.synchronize()
        outs.append((out, a, p))
    for got in outs[1:]:
        assert all(torch.equal(x, y) for x, y in zip(got, outs[0]))


def test_expanded_pools_are_refused(lc, gpu):
    """Strides of zero everywhere stand for a contiguous pool at the C entry, of which these have one row."""
    row = torch.zeros((1, 1, 1, 1, 64), dtype=torch.bfloat16, device="cuda")
    for shape in ((2, 4, 2, 16, 64), (1, 1, 1, 16, 64), (1, 8, 1, 1, 64)):
        with pytest.raises((ValueError, lc.LumenError)):
            lc.PagedKvCache(row.expand(shape), row.clone().expand(shape), max_seqs=1, max_pages_per_seq=1, max_q_heads=2)
    lone = torch.zeros(64, dtype=torch.bfloat16, device="cuda").as_strided((1, 1, 1, 1, 64), (0, 0, 0, 0, 1))
    lc.PagedKvCache(lone, lone.clone().as_strided((1, 1, 1, 1, 64), (0, 0, 0, 0, 1)), max_seqs=1, max_pages_per_seq=1, max_q_heads=1)


def test_too_many_slots_for_a_call(lc, gpu):
    """2^21 items of 991 tiles and, where their window begins inside one, 992, of 16 slots: with what an item costs
    beside, one more than 31 bits count, and refused; a little shorter windows fit, here of lengths 0."""
    seqs, kv, page, dim = 2048, 1024, 4096, 8
    k, v = (torch.zeros((1, 1, kv, page, dim), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    cache = lc.PagedKvCache(k, v, max_seqs=seqs, max_pages_per_seq=5, max_q_heads=kv)
    tables = torch.zeros((seqs, 5), dtype=torch.int32, device="cuda")
    ln = torch.zeros(seqs, dtype=torch.int32, device="cuda")
    q = torch.ones((seqs, kv, dim), dtype=torch.bfloat16, device="cuda")
    with pytest.raises(lc.LumenError) as e:
        cache.attn(0, tables, ln, q, 1.0, window=991 * 16)
    assert e.value.code == lc.LC_ERR_INVALID
    assert (cache.attn(0, tables, ln, q, 1.0, window=989 * 16) == 0).all()


@pytest.mark.parametrize("name", ["attn", "weights", "reorder", "select"])
def test_outputs_made_for_another_stream(lc, gpu, name):
    """The current stream has yet to write blocks that are free by now; outputs of calls on other streams are not those."""
    lens = [700, 90]
    cache, tables, ln, _ = make(lc, lens, 8, 2, 128, 32, "bf16")
    q = queries(2, 8, 128, "bf16", 11)
    acc = torch.rand((2, 2, tables.shape[1] * 32), device="cuda")
    beam = lc.BeamSearch(2, 4, 3011)
    x, scores = torch.randn((2, 4, 3011), device="cuda"), torch.zeros((2, 4), device="cuda")
    parents = torch.zeros((1, 2), dtype=torch.int32, device="cuda")

    def call(stream):
        if name == "attn":
            return [cache.attn(1, tables, ln, q, 0.1, stream=stream)]
        if name == "weights":
            return [cache.attn_weights(1, tables, ln, q, 0.1, acc, acc.clone() if stream is None else more, stream=stream)]
        if name == "reorder":
            return [cache.reorder(tables, full, parents, stream=stream)]
        return beam.select(x, scores, stream=stream)

    full, more = torch.tensor([64], dtype=torch.int32, device="cuda"), acc.clone()
    want = [t.clone() for t in call(None)]
    side = torch.cuda.Stream()
    for stream in (side, side.cuda_stream):
        torch.cuda.synchronize()
        torch.cuda._sleep(100_000_000)
        late = [torch.empty_like(t) for t in want for _ in range(64)]
        for t in late:
            t.fill_(1)
        del late, t
        got = call(stream)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    for stream in (0, 1, torch.cuda.current_stream()):
        assert all(torch.equal(a, b) for a, b in zip(call(stream), want))


def test_overlaps_with_other_inputs_are_refused(lc, gpu):
    """An output in the place of an input that is not its own, or of another output."""
    k = torch.zeros((1, 4, 2, 16, 64), dtype=torch.bfloat16, device="cuda")
    cache = lc.PagedKvCache(k, k.clone(), max_seqs=2, max_pages_per_seq=2, max_q_heads=2)
    tables = torch.zeros((2, 2), dtype=torch.int32, device="cuda")
    ln = torch.ones(2, dtype=torch.int32, device="cuda")
    acc, pos = torch.zeros((2, 2, 32), device="cuda"), torch.zeros((2, 2, 32), dtype=torch.int32, device="cuda")
    both = torch.zeros((2, 2, 64), device="cuda")  # q or out, and in its storage rows of weights
    rows, ints = both.view(-1)[:128].view(2, 2, 32), torch.zeros(16, dtype=torch.int32, device="cuda")

    def refused(f, *args, **kw):
        with pytest.raises(lc.LumenError) as e:
            f(*args, **kw)
        assert e.value.code == lc.LC_ERR_INVALID

    refused(cache.evict, 0, tables, ln, 8, acc, pos, pos.view(torch.float32), torch.empty_like(pos))
    refused(cache.evict, 0, tables, ln, 8, acc, pos, torch.empty_like(acc), acc.view(torch.int32))
    refused(cache.attn_weights, 0, tables, ln, both, 1.0, acc, rows)
    refused(cache.attn_weights, 0, tables, ln, torch.ones_like(both), 1.0, acc, rows, out=both)
    refused(cache.attn_weights, 0, tables, ln, torch.ones_like(both), 1.0, rows, acc, out=both)
    refused(cache.reorder, tables, ln[:1], ints[:2].view(1, 2), ints[1:5].view(2, 2))
    refused(cache.reorder, tables, ints[:1], ints[8:10].view(1, 2), ints[:4].view(2, 2))
    # the selection's, at the C entry
    logits, scores = torch.zeros((1, 2, 100), device="cuda"), torch.zeros((1, 2), device="cuda")
    beam, outs = lc.BeamSearch(1, 2, 100), torch.zeros(64, device="cuda")
    at = [outs.data_ptr(), outs.data_ptr() + 32, outs.data_ptr() + 64, outs.data_ptr() + 96]

    def select(a):
        return lc.lib().lc_beam_select(beam._h, 1, logits.data_ptr(), lc.LC_F32, 100, scores.data_ptr(), None, -1, 0, *a, None)

    torch.cuda.synchronize()
    assert select(at) == lc.LC_OK
    for o in range(4):
        for other in (logits.data_ptr() + 796, scores.data_ptr() + 4, at[(o + 1) % 4]):
            assert select(at[:o] + [other] + at[o + 1:]) == lc.LC_ERR_INVALID
    torch.cuda.synchronize()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("slots", [3000, 20000, 140000])
def test_tables_much_wider_than_the_sequences(lc, gpu, dtype, slots):
    """Tables for up to `slots`, none of their unused pages in the pool: the same answers as under tight ones."""
    lens, page, kv, dim = [1025, 0, 700, 64], 32, 2, 64
    cache, tables, ln, rows = make(lc, lens, 8, kv, dim, page, dtype, seed=9)
    width = slots // page
    wide = torch.full((4, width), -1, dtype=torch.int32, device="cuda")
    wide[:, :tables.shape[1]] = tables
    k0, v0 = cache.k_pages.clone(), cache.v_pages.clone()
    q = queries(4, 8, dim, dtype, 3)
    g = torch.Generator().manual_seed(2)
    acc = torch.rand((4, kv, tables.shape[1] * page), generator=g).cuda()
    pos = torch.arange(acc.shape[2], dtype=torch.int32, device="cuda").expand_as(acc).contiguous()
    got = []
    for t in (tables, wide):
        handle = lc.PagedKvCache(k0.clone(), v0.clone(), max_seqs=4, max_pages_per_seq=width, max_q_heads=8)
        a, p = (torch.zeros((4, kv, t.shape[1] * page), dtype=x.dtype, device="cuda") for x in (acc, pos))
        a[:, :, :acc.shape[2]], p[:, :, :acc.shape[2]] = acc, pos
        for window in (0, 100):
            check(handle.attn(1, t, ln, q, 0.125, window=window), ref.attn(rows, q, 0.125, window)[0], dtype)
        add = torch.zeros_like(a)
        check(handle.attn_weights(1, t, ln, q, 0.125, add), ref.attn(rows, q, 0.125)[0], dtype)
        handle.evict(1, t, ln, 600, a, p, n_sink=4, n_recent=30)
        handle.evict(1, t, torch.clamp(ln, max=600), 599, a, p, n_sink=4, n_recent=30)
        assert handle.status() == lc.LC_OK
        n = acc.shape[2]
        got.append([a[:, :, :n], p[:, :, :n]] + [x.contiguous().view(torch.uint8) for x in (handle.k_pages, handle.v_pages)])
        w = ref.attn(rows, q, 0.125)[1]
        for s, m in enumerate(lens):
            want = w[s].view(kv, 4, m).sum(1)
            # as in test_weights_match_plain
            assert ((add[s, :, :m].double().cpu() - want).abs() <= 1e-4 * want + 2e-6).all()
    assert all(torch.equal(x, y) for x, y in zip(*got))


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("dim,page,slots", [(64, 16, 16384), (128, 7, 8192), (256, 16, 4096)])
def test_attn_sums_are_rounded_and_not_cut(lc, gpu, dtype, dim, page, slots):
    """Values of 1: outputs are 1, and of 512 the errors' mean is small, if tiles are added up by rounding. A tile's
    products end by cutting, up to three times 2^-23 of its sum, and the roundings' mean is below 2^-24: below 2^-21
    in all. (Sums that the products themselves ran on, over 10 to 55 tiles of a warp, were off by 2^-20 to 2^-21 on average.)"""
    seqs, kv, group = 8, 8, 8
    width = -(-slots // page)
    g = torch.Generator(device="cuda").manual_seed(dim)
    k = torch.empty((1, seqs * width, kv, page, dim), dtype=ref.DTYPES[dtype], device="cuda").normal_(generator=g)
    cache = lc.PagedKvCache(k, torch.ones_like(k), max_seqs=seqs, max_pages_per_seq=width, max_q_heads=kv * group)
    tables = torch.randperm(seqs * width, device="cuda").to(torch.int32).view(seqs, width)
    ln = torch.full((seqs,), slots, dtype=torch.int32, device="cuda")
    q = queries(seqs, kv * group, dim, dtype, 1)
    out = cache.attn(0, tables, ln, q, dim ** -0.5, out=torch.empty((seqs, kv * group, dim), device="cuda")).double()
    assert (out - 1).abs().max() <= 2.0 ** -18
    assert (out - 1).mean().abs() <= 2.0 ** -21
