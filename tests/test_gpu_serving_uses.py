"""Uses of the serving operators that their documentation allows: in place, on two streams at once, as
graphs replayed beside each other, at the most sequences, with scales of any sign, after every kind of
step of the engine."""
import importlib
import math

import numpy as np
import pytest
import torch

from serving_reference import TYPES, attend, make_cache, make_table, values
from test_gpu_logprobs import check, exact

engine = importlib.import_module("qwen-30brust_amd")
serving = importlib.import_module("qwen-30brust_amd.serving")
synth = importlib.import_module("qwen-30brust_amd.synth")

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    d = engine.Device(0)
    yield d
    d.close()


def ints(x):
    return torch.tensor(x, dtype=torch.int32).cuda()


@pytest.mark.parametrize("q,kv", [("f32", "f32"), ("bf16", "bf16"), ("f16", "q8_0"), ("bf16", "f16")])
@pytest.mark.parametrize("heads,kvheads,dim", [(32, 4, 128), (24, 2, 64), (8, 2, 96), (20, 1, 256)])
@pytest.mark.parametrize("lengths", [[3000], [700, 5, 0, 1200], [40] * 70])
def test_queries_in_place(dev, q, kv, heads, kvheads, dim, lengths):
    """q_out may be q, out may be q: the same bits as apart."""
    g = torch.Generator().manual_seed(dim)
    page = 16
    table, pool, _ = make_table(g, lengths, page)
    cache = make_cache(g, pool, page, kvheads, dim, kv)
    c, n, table = serving.PagedCache(dev, *cache), ints(lengths), table.cuda()
    B = len(lengths)
    rows = torch.randn(B, (heads + 2 * kvheads) * dim, generator=g).to(TYPES[q]).cuda()
    query = rows[:, :heads * dim].unflatten(1, (heads, dim))
    k, v = (m.unflatten(1, (kvheads, dim)) for m in rows[:, heads * dim:].chunk(2, 1))
    w, rope = torch.ones(dim, device="cuda") * 1.1, torch.randn(4000, dim // 2, 2, generator=g).cuda()
    apart = torch.zeros(B, heads, dim, dtype=TYPES[q], device="cuda")
    c.append(k, v, table, n, q=query, q_out=apart, q_norm=w, rope=rope)
    live = n > 0
    got = c.append(k, v, table, n, q=query, q_out=query, q_norm=w, rope=rope)
    assert got is query and torch.equal(query[live], apart[live])
    want = c.attend(query, table, n)
    mine = query.clone()
    assert c.attend(mine, table, n, out=mine) is mine and torch.equal(mine, want)
    assert c.attend(query, table, n, out=query) is query and torch.equal(query, want)  # a slice of rows


@pytest.mark.parametrize("scale", [0.0, -0.3, 3.0, 1e-30])
@pytest.mark.parametrize("q,kv,dim", [("f32", "f32", 128), ("bf16", "bf16", 64), ("f16", "q8_0", 128), ("f32", "f16", 80)])
def test_scales(dev, scale, q, kv, dim):
    g = torch.Generator().manual_seed(dim)
    lengths = [100, 1, 33]
    table, pool, _ = make_table(g, lengths, 16)
    cache = make_cache(g, pool, 16, 2, dim, kv)
    query = torch.randn(3, 4, dim, generator=g).to(TYPES[q]).cuda()
    # the same of queries of the other sign; the bound is made for scales above 0
    want, _, bound = attend(-query if scale < 0 else query, values(cache[0], cache[2]), values(cache[1], cache[3]), table,
                            lengths, abs(scale))
    got = serving.PagedCache(dev, *cache).attend(query, table.cuda(), ints(lengths), scale=scale).cpu().double()
    half = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}[q]
    assert ((got - want).abs() <= bound + half * (want.abs() + bound) + 2.0 ** -17 * 5 * (q != "f32")).all()


def test_most_sequences(dev):
    """65,535 sequences of none to four keys: appended to, attended, evicted."""
    B, G, dim, page = 65535, 1, 64, 4
    g = torch.Generator(device="cuda").manual_seed(1)
    lengths = torch.randint(0, 5, (B,), generator=g, device="cuda", dtype=torch.int32)
    order = torch.randperm(2 * B, generator=g, device="cuda").int()
    table, to = order[:B, None].contiguous(), order[B:, None].contiguous()
    k, v = (torch.randn(2 * B, page, G, dim, generator=g, device="cuda") for _ in range(2))
    c = serving.PagedCache(dev, k, v)
    new = torch.randn(2, B, G, dim, generator=g, device="cuda")
    c.append(new[0], new[1], table, lengths)
    has = lengths > 0
    last = (table[has, 0].long(), lengths[has].long() - 1)
    assert torch.equal(k[last], new[0][has]) and torch.equal(v[last], new[1][has])
    q = torch.randn(B, 2, dim, generator=g, device="cuda")
    weights = torch.zeros(B, G, page, device="cuda")
    out, _ = c.attend(q, table, lengths, weights=weights)
    kk, vv = k[table[:, 0].long()].transpose(1, 2).double(), v[table[:, 0].long()].transpose(1, 2).double()
    s = (q.double()[:, :, None] * kk).sum(-1) / 8
    there = torch.arange(page, device="cuda") < lengths[:, None]
    s = s.masked_fill(~there[:, None], -math.inf)
    p = torch.where(has[:, None, None], s.softmax(-1), torch.zeros_like(s))
    # scores of up to 67 terms, each off by a half step of at most 60 in all; four keys
    tol = (4 * 67 * 60 + 100) * 2.0 ** -24
    assert ((out.double() - (p[..., None] * vv).sum(2)).abs() <= tol * 5).all()
    assert ((weights.double() - p.sum(1, keepdim=True)).abs() <= 2 * tol).all()
    kept, kw, n = c.evict(weights, table, lengths, 2, to, recent=1)
    assert torch.equal(n, lengths.clamp(max=2))
    rows = has.nonzero()[:, 0]
    assert torch.equal(k[to[rows, 0].long(), 0, 0], k[table[rows, 0].long(), kept[rows, 0, 0].long(), 0])


def test_two_streams_at_once(dev):
    """Calls under way on two streams, each with workspaces of its own, give what they give alone."""
    g = torch.Generator().manual_seed(5)
    lengths, G, H, dim = [4000, 900, 3000], 4, 32, 128
    table, pool, _ = make_table(g, lengths, 16)
    cache = make_cache(g, pool, 16, G, dim, "bf16")
    c, n, table = serving.PagedCache(dev, *cache), ints(lengths), table.cuda()
    q = [torch.randn(3, H, dim, generator=g).bfloat16().cuda() for _ in range(2)]
    x = [torch.randn(20, 151936, generator=g).cuda() for _ in range(2)]
    weights = torch.rand(3, G, 4000, generator=g).cuda()

    def work(i):
        out, w = c.attend(q[i], table, n, 4000, weights=weights, weights_out=torch.zeros_like(weights))
        return (out, w[0], w[1, :, :900], w[2, :, :3000], *(t for t in serving.logprobs(dev, x[i], top=9) if t is not None))

    want = [[t.clone() for t in work(i)] for i in range(2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(8):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(work(i))
    torch.cuda.synchronize()
    for i in range(2):
        for r in got[i]:
            for a, b in zip(r, want[i]):
                assert torch.equal(a, b)
    # two graphs, replayed on two streams together
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
        torch.cuda.synchronize()
        for i in range(2):
            for a, b in zip(held[i], want[i]):
                assert torch.equal(a, b)
                a.zero_()
        torch.cuda.synchronize()


def test_logprobs_after_every_kind_of_step(dev):
    """Model.logprobs reads the logits that prefill, generate and forward leave."""
    spec = synth.tiny_k()
    m = engine.Model(synth.build_image(spec, threads=4), spec.context, device=dev)

    def same(x):
        x = torch.from_numpy(np.ascontiguousarray(x))[None]
        lp, h, ids, alt = m.logprobs(4, 9)
        check((torch.tensor([lp]), torch.tensor([h]), torch.from_numpy(ids.astype(np.int32))[None], torch.from_numpy(alt)[None]),
              exact(x, torch.tensor([4]), 9, None), x, x.shape[1])

    same(m.prefill([7, 3, 5])[1])
    same(m.forward(2))
    _, logits = m.generate([1, 2], 3, want_logits=True)
    same(logits)
    m.reset()
    with pytest.raises(engine.EngineError, match="run a token step first"):
        m.logprobs()
