"""Attention of several new tokens per sequence over the paged cache (PagedCache.attend_prompts, attend_tree)
against a plain 64-bit restatement."""
import importlib
import math

import pytest
import torch

from prompts_reference import attend_many, close, make, signed, split_of, trees
from serving_reference import TYPES, values

engine = importlib.import_module("qwen-30brust_amd")
serving = importlib.import_module("qwen-30brust_amd.serving")

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    d = engine.Device(0)
    yield d
    d.close()


def ints(x):
    return torch.tensor(x, dtype=torch.int32).cuda()


def run(dev, context, new, heads, kvheads, dim, page, q, kv, *, tree=False, scale=None, seed=1, head_major=False,
        front=0, behind=0, change=None, most=None):
    """Prepares, calls and compares; change(cache, table, lengths, first, query) may alter the inputs."""
    cache, table, lengths, first, query = make(seed, context, new, heads, kvheads, dim, page, q, kv, head_major, front,
                                               behind)
    if change:
        change(cache, table, lengths, first, query)
    bits = None
    if tree:
        bits = [0] * front + trees(torch.Generator().manual_seed(seed), new)[1] + [0] * behind
        # some see nothing of the tree, some what is no ancestor
        bits = [0 if i % 7 == 3 else b | (1 if i % 5 == 2 else 0) for i, b in enumerate(bits)]
    scale = 0.9 / math.sqrt(dim) if scale is None else scale
    k, v = values(cache[0], cache[2]), values(cache[1], cache[3])
    sign = -1 if scale < 0 else 1  # the same of queries of the other sign; the bound is made for scales above 0
    want, bound = attend_many(sign * query, k, v, table, lengths, first, abs(scale), bits, split_of(q, kv))
    c = serving.PagedCache(dev, *cache)
    out = torch.full(query.shape, 7.0, dtype=query.dtype, device="cuda")
    args = (query.cuda(), table.cuda(), ints(lengths), ints(first))
    if tree:
        got = c.attend_tree(*args, signed(bits).cuda(), most, scale=scale, out=out)
    else:
        got = c.attend_prompts(*args, most, scale=scale, out=out)
    assert got is out
    assert (got[:front] == 7).all() and (got[first[-1]:] == 7).all()
    live = slice(front, first[-1])
    close(got[live], want[live], bound[live])
    return got


KINDS = [("f32", "f32"), ("f16", "f16"), ("bf16", "bf16"), ("bf16", "q8_0"), ("f16", "q8_0"), ("f32", "q8_0"), ("f32", "f16"),
         ("f16", "bf16"), ("bf16", "f32")]
SHAPES = [(32, 4, 128), (8, 8, 64), (6, 2, 128), (10, 1, 64), (36, 2, 64)]
EDGES = ([0, 0, 0, 0, 5, 64, 1, 100, 257, 40, 3, 64, 0, 31], [1, 2, 63, 64, 31, 1, 127, 33, 16, 0, 130, 64, 17, 1])


@pytest.mark.parametrize("q,kv", KINDS)
@pytest.mark.parametrize("heads,kvheads,dim", SHAPES)
def test_prompts_edges(dev, q, kv, heads, kvheads, dim):
    run(dev, *EDGES, heads, kvheads, dim, 16, q, kv, front=3, behind=2)


@pytest.mark.parametrize("q,kv", KINDS)
@pytest.mark.parametrize("heads,kvheads,dim", SHAPES)
def test_tree_edges(dev, q, kv, heads, kvheads, dim):
    run(dev, [0, 0, 5, 64, 1, 100, 257, 40, 700], [1, 2, 31, 64, 64, 33, 16, 0, 5], heads, kvheads, dim, 16, q, kv, tree=True,
        front=2, behind=1)


@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("q,kv", [("f32", "f32"), ("bf16", "bf16"), ("bf16", "q8_0")])
@pytest.mark.parametrize("page", [1, 7, 24, 64, 200])
def test_pages(dev, tree, q, kv, page):
    run(dev, [129, 0, 333, 64], [40, 33, 1, 64], 8, 2, 128, page, q, kv, tree=tree, head_major=page % 3 == 0, seed=page)


@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("q,kv,dim,heads,kvheads", [
    ("bf16", "bf16", 256, 4, 2), ("f16", "f16", 256, 16, 1), ("f32", "f32", 256, 4, 2), ("bf16", "q8_0", 256, 4, 2),
    ("bf16", "bf16", 96, 8, 2), ("f32", "f32", 96, 4, 4), ("f16", "q8_0", 160, 5, 5), ("f16", "f16", 80, 4, 2),
    ("bf16", "bf16", 5, 4, 2), ("f32", "f16", 1, 3, 1), ("f16", "f16", 250, 3, 1), ("f32", "q8_0", 32, 4, 2)])
def test_widths(dev, tree, q, kv, dim, heads, kvheads):
    run(dev, [70, 0, 200], [33, 60, 1], heads, kvheads, dim, 16, q, kv, tree=tree)


@pytest.mark.parametrize("q,kv", [("f32", "f32"), ("bf16", "bf16"), ("f16", "f16")])
@pytest.mark.parametrize("context,new", [([0], [1500]), ([1300], [300]), ([0, 900, 17], [700, 1, 650])])
def test_longer(dev, q, kv, context, new):
    """Sequences whose work is dealt to many workgroups."""
    run(dev, context, new, 8, 2, 128, 16, q, kv)


@pytest.mark.parametrize("q,kv", [("f32", "f32"), ("bf16", "bf16"), ("f16", "f16")])
@pytest.mark.parametrize("context,new", [([70001], [3]), ([20000, 3, 500], [64, 64, 1])])
def test_tree_long(dev, q, kv, context, new):
    run(dev, context, new, 8, 1, 64, 64, q, kv, tree=True)


@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("q,kv", [("f32", "f32"), ("bf16", "bf16"), ("f16", "f16")])
@pytest.mark.parametrize("heads", [1, 3, 130, 300])
def test_groups(dev, tree, q, kv, heads):
    """Query heads of one KV head: fewer and more than a tile has rows."""
    run(dev, [50, 0], [20, 9], heads, 1, 64, 16, q, kv, tree=tree)


@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("q,kv", [("f32", "f32"), ("bf16", "bf16"), ("f16", "f16"), ("f32", "q8_0")])
@pytest.mark.parametrize("scale", [0.0, -0.3, 3.0, 1e-30])
def test_scales(dev, tree, q, kv, scale):
    run(dev, [70, 0], [33, 20], 4, 2, 64, 16, q, kv, tree=tree, scale=scale)


# ------------------------------------------------------- values that are not finite
def at(table, b, t, page=16):
    return int(table[b, t // page]), t % page


@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("q,kv", [("f32", "f32"), ("bf16", "bf16"), ("f16", "f16"), ("f32", "bf16")])
@pytest.mark.parametrize("dim", [128, 64, 96, 256])
def test_masked_values(dev, tree, q, kv, dim):
    """NaN and infinities in keys and values that a row does not see change nothing; those that it sees come
    out as the formula has them."""
    context, new = [100, 0, 33], [40, 60, 30]

    def change(cache, table, lengths, first, query):
        k, v = cache[0], cache[1]
        for b, (c, n) in enumerate(zip(context, new)):
            for t, (x, value) in zip((c + n - 1, c + n // 2, c + n // 3, c + 5),
                                     ((v, math.nan), (v, math.inf), (v, -math.inf), (k, math.nan))):
                x[at(table, b, t)][b % 2, 3 + t % 7] = value
            # slots behind the keys, and a page of nobody's
            for t in range(c + n, -(-(c + n) // 16) * 16):
                k[at(table, b, t)] = math.nan
                v[at(table, b, t)] = math.inf

    run(dev, context, new, 8, 2, dim, 16, q, kv, tree=tree, change=change)


@pytest.mark.parametrize("q,kv", [("f32", "f32"), ("bf16", "bf16"), ("f16", "f16")])
def test_infinite_scores(dev, q, kv):
    """A score of -inf is no weight, rows of nothing but -inf are zeros, +inf gives NaN."""
    def change(cache, table, lengths, first, query):
        k = cache[0]
        query[:, :, 0] = query[:, :, 0].abs().clamp(min=0.5)
        for b in range(3):
            for t in range(lengths[b]):
                if b == 0 or (b == 1 and t % 3):
                    k[at(table, b, t)][:, 0] = -math.inf
        k[at(table, 2, 30)][0, 0] = math.inf

    got = run(dev, [0, 20, 10], [20, 40, 35], 4, 2, 64, 16, q, kv, change=change)
    assert (got[:20] == 0).all()


def test_large_values(dev):
    """Values near the end of the range, whose weighted means are in it."""
    for q, kv, most in (("bf16", "bf16", 2.0 ** 118), ("f16", "f16", 60000.0), ("f32", "f32", 2.0 ** 118)):
        def change(cache, table, lengths, first, query):
            cache[1].copy_((cache[1].float().sign() * most).to(cache[1].dtype))

        run(dev, [100, 0], [30, 50], 4, 2, 128, 16, q, kv, change=change)


def test_small_weights(dev):
    """Many weights far below the largest: f16 products keep them."""
    n, dim = 4000, 64

    def change(cache, table, lengths, first, query):
        query.zero_()
        query[:, :, 0] = 1.0
        k, v = cache[0], cache[1]
        k.zero_()
        v.zero_()
        k[..., 0] = -16.5  # weights of 2^-23.8, a thousand of them a tenth of a thousandth
        v[..., 0] = 8.0
        k[at(table, 0, 0)][:, 0] = 0.0
        v[at(table, 0, 0)][:, 0] = 0.0

    got = run(dev, [n], [3], 2, 1, dim, 16, "f16", "f16", scale=1.0, change=change)
    assert (got[:, :, 0].float() > 0.0015).all()


# ------------------------------------------------------- out of range
def test_out_of_range(dev):
    """Sequences out of range give NaN or are left as they were, and do not touch the others."""
    for q, kv in (("f32", "f32"), ("bf16", "bf16"), ("bf16", "q8_0")):
        context, new = [30, 40, 50, 20, 33, 10], [20] * 6
        cache, table, lengths, first, query = make(3, context, new, 4, 2, 64, 16, q, kv)
        c = serving.PagedCache(dev, *cache)
        k, v = values(cache[0], cache[2]), values(cache[1], cache[3])
        bits = trees(torch.Generator().manual_seed(1), new)[1]
        for tree in (False, True):
            want, bound = attend_many(query, k, v, table, lengths, first, 0.125, bits if tree else None, split_of(q, kv))

            def call(table, lengths, first, most=None):
                out = torch.full(query.shape, 7.0, dtype=query.dtype, device="cuda")
                args = (query.cuda(), table.cuda(), ints(lengths), ints(first))
                if tree:
                    return c.attend_tree(*args, signed(bits).cuda(), most, scale=0.125, out=out)
                return c.attend_prompts(*args, most, scale=0.125, out=out)

            # lengths: negative, past `most`, below the new tokens
            got = call(table, [-1, lengths[1], 71, 19, lengths[4], lengths[5]], first, 70)
            for b in range(6):
                rows = slice(first[b], first[b + 1])
                if b in (0, 2, 3):
                    assert got[rows].isnan().all()
                else:
                    close(got[rows], want[rows], bound[rows])
            # pages: of sequence 1's key 48, of 2's first, behind 4's keys (never read)
            t2 = table.clone()
            t2[1, 3], t2[2, 0], t2[4, -1 if table.shape[1] > 4 else 3] = 1 << 20, -5, 99999
            got = call(t2, lengths, first)
            for b in range(6):
                for i in range(20):
                    r = first[b] + i
                    bad = b == 2 or (b == 1 and (tree or context[1] + i >= 48)) or \
                        (b == 4 and table.shape[1] <= 4 and (tree or context[4] + i >= 48))
                    if bad:
                        assert got[r].isnan().all(), (b, i)
                    else:
                        close(got[r:r + 1], want[r:r + 1], bound[r:r + 1])
            # bounds of new tokens: past the rows, negative, descending (the next sequence then has others' rows)
            for f, left, others in (([0, 20, 40, 60, 80, 100, 121], 5, (0, 1, 2, 3, 4)),
                                    ([-20, 20, 40, 60, 80, 100, 120], 0, (1, 2, 3, 4, 5)),
                                    ([0, 20, 40, 30, 80, 100, 120], None, (0, 4, 5))):
                got = call(table, lengths, f)
                for b in others:
                    close(got[first[b]:first[b + 1]], want[first[b]:first[b + 1]], bound[first[b]:first[b + 1]])
                if left is not None:
                    assert (got[first[left]:first[left + 1]] == 7).all()


def test_too_many_nodes(dev):
    cache, table, lengths, first, query = make(1, [5, 5], [65, 64], 2, 1, 64, 16, "bf16", "bf16")
    c = serving.PagedCache(dev, *cache)
    got = c.attend_tree(query.cuda(), table.cuda(), ints(lengths), ints(first), torch.full((129,), -1, device="cuda"))
    assert got[:65].isnan().all() and not got[65:].isnan().any()


def test_nothing_to_do(dev):
    cache, table, lengths, first, query = make(1, [5], [3], 2, 1, 64, 16, "f32", "f32")
    c = serving.PagedCache(dev, *cache)
    assert c.attend_prompts(query[:0].cuda(), table.cuda(), ints(lengths), ints([0, 0])).shape == (0, 2, 64)
    none = torch.empty(0, 4, dtype=torch.int32, device="cuda")
    out = torch.full((3, 2, 64), 5.0, device="cuda")
    assert (c.attend_prompts(query.cuda(), none, ints([]), ints([0]), 16, out=out) == 5).all()
    # padding: a sequence without keys and tokens beside one of length 0 that has tokens
    got = c.attend_prompts(query.cuda(), table[[0, 0, 0]].cuda(), ints([0, 8, 0]), ints([0, 0, 3, 3]))
    assert torch.equal(got, c.attend_prompts(query.cuda(), table.cuda(), ints([8]), ints([0, 3])))
    assert c.attend_prompts(query.cuda(), table.cuda(), ints([0]), ints([0, 3])).isnan().all()


# ------------------------------------------------------- layouts
@pytest.mark.parametrize("q,kv", [("f32", "f32"), ("bf16", "bf16"), ("f16", "f16"), ("bf16", "q8_0"), ("f32", "f16")])
@pytest.mark.parametrize("dim", [64, 128])
def test_layouts(dev, q, kv, dim):
    """Queries and outputs in wider rows, off every alignment, in place; caches with strides of their own."""
    context, new, heads, G = [100, 3], [30, 70], 8, 2
    cache, table, lengths, first, query = make(5, context, new, heads, G, dim, 16, q, kv)
    c = serving.PagedCache(dev, *cache)
    args = (table.cuda(), ints(lengths), ints(first))
    want = c.attend_prompts(query.cuda(), *args)
    n = query.shape[0]

    def wide(t, extra, shift):
        rows = torch.zeros(n, heads * dim + extra, dtype=t.dtype, device="cuda")
        view = rows[:, shift:shift + heads * dim].unflatten(1, (heads, dim))
        view.copy_(t)
        return view

    for extra, shift in ((16, 8), (5, 1), (1, 0)):
        mine = wide(query.cuda(), extra, shift)
        assert torch.equal(c.attend_prompts(mine, *args), want)
        out = wide(torch.zeros_like(query).cuda(), extra, shift)
        assert c.attend_prompts(mine, *args, out=out) is out and torch.equal(out, want)
        assert c.attend_prompts(mine, *args, out=mine) is mine and torch.equal(mine, want)
    if kv == "q8_0":
        return
    # a cache off every alignment, and one of wide slots: the staged and the direct way agree to their sums' order
    k, v = values(cache[0], None), values(cache[1], None)
    exact, bound = attend_many(query, k, v, table, lengths, first, dim ** -0.5, None, split_of(q, kv))
    for extra, shift in ((1, 1), (32, 8)):
        held = []
        for x in cache[:2]:
            pool = torch.full((x.shape[0], 16, G, dim + extra), math.nan, dtype=x.dtype, device="cuda")
            pool[..., shift:shift + dim] = x
            held.append(pool[..., shift:shift + dim])
        got = serving.PagedCache(dev, *held).attend_prompts(query.cuda(), *args)
        close(got, exact, bound)


@pytest.mark.parametrize("kv", ["bf16", "f32"])
def test_far_pages(dev, kv):
    """Pages whose offsets pass 32 bits."""
    G, dim, page = 2, 128, 64
    x = TYPES[kv]
    pages = (1 << 32) // (page * G * dim) + 50  # past 2^32 elements
    k, v = (torch.empty(pages, page, G, dim, dtype=x, device="cuda") for _ in range(2))
    ids = [pages - 1, 0, pages - 2, pages // 2 + 1]
    g = torch.Generator().manual_seed(2)
    small = []
    for t in (k, v):
        part = torch.randn(4, page, G, dim, generator=g).to(x)
        small.append(part)
        for i, p in enumerate(ids):
            t[p] = part[i].cuda()
    query = torch.randn(50, 4, dim, generator=g).to(x)
    table = torch.arange(4, dtype=torch.int32)[None]
    want, bound = attend_many(query, small[0].double(), small[1].double(), table, [240], [0, 50], 0.1, None,
                              split_of(kv, kv))
    c = serving.PagedCache(dev, k, v)
    got = c.attend_prompts(query.cuda(), ints([ids]), ints([240]), ints([0, 50]), scale=0.1)
    close(got, want, bound)
    bits = [(1 << i + 1) - 1 for i in range(50)]
    got = c.attend_tree(query.cuda(), ints([ids]), ints([240]), ints([0, 50]), signed(bits).cuda(), scale=0.1)
    close(got, want, bound)


# ------------------------------------------------------- agreement, streams, graphs
@pytest.mark.parametrize("q,kv", [("f32", "f32"), ("bf16", "bf16"), ("f16", "f16"), ("bf16", "q8_0")])
def test_single_tokens(dev, q, kv):
    """One new token a sequence: what attend gives, to the order of the sums."""
    context = [0, 5, 300, 1000]
    cache, table, lengths, first, query = make(4, context, [1] * 4, 16, 2, 128, 16, q, kv)
    c = serving.PagedCache(dev, *cache)
    k, v = values(cache[0], cache[2]), values(cache[1], cache[3])
    want, bound = attend_many(query, k, v, table, lengths, first, 128 ** -0.5, None, split_of(q, kv))
    for got in (c.attend_prompts(query.cuda(), table.cuda(), ints(lengths), ints(first)),
                c.attend_tree(query.cuda(), table.cuda(), ints(lengths), ints(first), torch.ones(4, dtype=torch.int64, device="cuda"))):
        close(got, want, bound)


def test_streams_and_graphs(dev):
    """Calls under way on two streams, and graphs replayed beside each other and eager calls, give what a call
    alone gives, bit by bit; a replay reads lengths as they are then."""
    cache, table, lengths, first, query = make(6, [900, 0, 70], [64, 64, 5], 16, 2, 128, 16, "bf16", "bf16")
    c = serving.PagedCache(dev, *cache)
    bits = signed(trees(torch.Generator().manual_seed(1), [64, 64, 5])[1]).cuda()
    t, f, n = table.cuda(), ints(first), ints(lengths)
    qs = [query.cuda(), (query * 0.5).cuda()]

    def work(i):
        return c.attend_prompts(qs[i], t, n, f), c.attend_tree(qs[i], t, n, f, bits)

    want = [[x.clone() for x in work(i)] for i in range(2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(6):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(work(i))
    torch.cuda.synchronize()
    for i in range(2):
        for r in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(r, want[i]))
    graphs, held = [], []
    for i in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held.append(work(i))
        graphs.append(graph)
    for _ in range(4):
        for s, graph in zip(streams, graphs):
            with torch.cuda.stream(s):
                graph.replay()
        eager = work(0)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(eager, want[0]))
        for i in range(2):
            for a, b in zip(held[i], want[i]):
                assert torch.equal(a, b)
                a.zero_()
        torch.cuda.synchronize()
    n.sub_(ints([500, 0, 3]))
    shorter = [x.clone() for x in work(1)]
    graphs[1].replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(held[1], shorter)) and not torch.equal(shorter[0], want[1][0])


def test_many_sequences(dev):
    """More sequences than a workgroup has threads, ragged, in one call."""
    B = 1500
    g = torch.Generator().manual_seed(9)
    context = torch.randint(0, 40, (B,), generator=g).tolist()
    new = torch.randint(0, 4, (B,), generator=g).tolist()
    for q, kv in (("bf16", "bf16"), ("f32", "f32")):
        run(dev, context, new, 4, 2, 64, 8, q, kv)


def test_refusals(dev):
    cache, table, lengths, first, query = make(1, [5, 0], [3, 2], 4, 2, 64, 16, "bf16", "bf16")
    c = serving.PagedCache(dev, *cache)
    q, t, n, f, s = query.cuda(), table.cuda(), ints(lengths), ints(first), torch.ones(5, dtype=torch.int64, device="cuda")

    def refused(text, call):
        with pytest.raises(engine.EngineError, match=text):
            call()

    refused("3 dimensions", lambda: c.attend_prompts(q[0], t, n, f))
    refused("shape", lambda: c.attend_prompts(q[:, :, :32], t, n, f))
    refused("multiple of the KV heads", lambda: c.attend_prompts(q[:, :3], t, n, f))
    refused("one more than sequences", lambda: c.attend_prompts(q, t, n, f[:2]))
    refused("type torch.int64", lambda: c.attend_prompts(q, t, n, f.long()))
    refused("type torch.float64", lambda: c.attend_prompts(q.double(), t, n, f))
    refused("other sequences", lambda: c.attend_prompts(q, t, n[:1], f))
    refused("hold fewer keys", lambda: c.attend_prompts(q, t, n, f, 17))
    refused("one for each token", lambda: c.attend_tree(q, t, n, f, s[:4]))
    refused("type torch.int32", lambda: c.attend_tree(q, t, n, f, s.int()))
    refused("share memory", lambda: c.attend_prompts(q, t, n, f, out=q[:1].expand(5, 4, 64)))
    refused("not a tensor on", lambda: c.attend_prompts(query, t, n, f))
    refused("no gradient", lambda: c.attend_prompts(q.float().requires_grad_(), t, n, f))
