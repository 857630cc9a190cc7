"""Pages and slots of new tokens (PagePool.plan), the acceptance of drafted tokens (accept), and both with appends
and attention as a server uses them."""
import importlib

import pytest
import torch

from prompts_reference import signed, trees
from serving_reference import TYPES, make_cache, make_table

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


# ------------------------------------------------------- plan
class Plain:
    """The same on lists."""

    def __init__(self, pages, page, free):
        self.pages, self.page, self.free = pages, page, list(free)

    def plan(self, table, held, lengths, grow, n, parents=None):
        page, per = self.page, len(table[0]) if table else 0
        first, lengths = [0], list(lengths)
        fine = [0 <= L and 0 <= L + g and max(L, L + g) <= per * page and 0 <= h <= per
                for L, g, h in zip(lengths, grow, held)]
        need = [-(-(L + g) // page) for L, g in zip(lengths, grow)]
        for b in reversed(range(len(lengths))):
            if fine[b] and grow[b] <= 0 and held[b] > need[b]:
                self.free += reversed(table[b][need[b]:held[b]])
                held[b] = need[b]
        for b in range(len(lengths)):
            if fine[b] and grow[b] <= 0:
                lengths[b] += grow[b]
        rows, open_ = [], True
        for b in range(len(lengths)):
            if fine[b] and grow[b] > 0:
                claims = max(0, need[b] - held[b])
                open_ = open_ and claims <= len(self.free) and first[-1] + grow[b] <= n
                if open_:
                    for _ in range(claims):
                        table[b][held[b]] = self.free.pop()
                        held[b] += 1
                    for i in range(grow[b]):
                        t = lengths[b] + i
                        rows.append((table[b][t // page] * page + t % page, t, b))
                    lengths[b] += grow[b]
                    first.append(first[-1] + grow[b])
                    continue
            first.append(first[-1])
        slots, positions, sequences = ([r[k] for r in rows] + [-1] * (n - len(rows)) for k in range(3))
        seen = [0] * n
        if parents is not None:
            for b in range(len(lengths)):
                f, m = first[b], first[b + 1] - first[b]
                for j in range(min(m, 64)):
                    p = parents[f + j]
                    seen[f + j] = 1 << j | (seen[f + p] if 0 <= p < j else 0)
                    positions[f + j] = lengths[b] - m + bin(seen[f + j]).count("1") - 1
        return lengths, first, slots, positions, sequences, seen


def setup(dev, seed, batch, page, per, spare, most):
    g = torch.Generator().manual_seed(seed)
    lengths = torch.randint(0, most + 1, (batch,), generator=g).tolist()
    held = [-(-t // page) for t in lengths]
    order = torch.randperm(sum(held) + spare, generator=g).tolist()
    table, at = [[-9] * per for _ in range(batch)], 0
    for b, h in enumerate(held):
        table[b][:h] = order[at:at + h]
        at += h
    free = order[at:]
    plain = Plain(len(order), page, free)
    pool = serving.PagePool(dev, len(order), page, free=ints(free + [0] * at), count=ints([len(free)]))
    return g, lengths, held, table, plain, pool


def same(got, want, n, tree):
    lengths, first, slots, positions, sequences, seen = want
    assert got.lengths.tolist() == lengths and got.first.tolist() == first
    assert got.slots.tolist() == slots and got.positions.tolist() == positions and got.sequences.tolist() == sequences
    assert (got.ancestors is None) == (not tree) and (not tree or torch.equal(got.ancestors.cpu(), signed(seen)))


@pytest.mark.parametrize("batch,page,per,most,spare", [(1, 16, 40, 100, 50), (5, 1, 700, 30, 900), (64, 16, 300, 4000, 800),
                                                       (3, 64, 40, 900, 200), (1100, 4, 30, 40, 9000), (2500, 7, 12, 20, 9000)])
@pytest.mark.parametrize("tree", [False, True])
def test_plan(dev, batch, page, per, most, spare, tree):
    """Rounds of growth and shrinking, some more than fits, against lists; lengths in place on every other."""
    g, lengths, held, table, plain, pool = setup(dev, batch, batch, page, per, spare, most)
    t, h, n = ints(table), ints(held), ints(lengths)
    for step in range(5):
        grow = torch.randint(1, 20 if tree or batch > 100 else 300, (batch,), generator=g)
        if step % 2:
            grow = torch.where(torch.rand(batch, generator=g) < 0.6, -grow, grow)
        grow = [max(x, -L) if step != 3 else x for x, L in zip(grow.tolist(), lengths)]
        room = sum(max(0, x) for x in grow) + 3
        room = room // 2 if step == 4 else room
        parents = None
        if tree:
            parents = [int(torch.randint(-1, 20, (1,), generator=g)) for _ in range(room)]
            parents = [p if i % 3 else min(i % 9, p) for i, p in enumerate(parents)]
        got = pool.plan(t, h, n, ints(grow), room, parents=None if parents is None else ints(parents),
                        out=n if step % 2 else None)
        want = plain.plan(table, held, lengths, grow, room, parents)
        same(got, want, room, tree)
        lengths, n = want[0], got.lengths
        assert t.tolist() == table and h.tolist() == held
        assert pool.count.tolist() == [len(plain.free)] and pool.free[:len(plain.free)].tolist() == plain.free


def test_plan_large(dev):
    """As many tokens as a prefill of prompts has: filled by a second launch."""
    g, lengths, held, table, plain, pool = setup(dev, 3, 40, 16, 400, 9000, 900)
    t, h, n = ints(table), ints(held), ints(lengths)
    grow = torch.randint(1, 2100, (40,), generator=g).tolist()
    room = sum(grow) + 1000
    got = pool.plan(t, h, n, ints(grow), room)
    same(got, plain.plan(table, held, lengths, grow, room), room, False)
    assert t.tolist() == table
    # and back: the stack is what it was
    before = list(plain.free)
    back = pool.plan(t, h, got.lengths, -ints(grow), 0)
    assert back.lengths.tolist() == lengths and back.first.tolist() == [0] * 41 and back.slots.shape == (0,)
    plain.plan(table, held, got.lengths.tolist(), [-x for x in grow], 0)
    assert pool.free[:len(plain.free)].tolist() == plain.free and len(plain.free) > len(before)


def test_plan_out_of_range(dev):
    """Lengths, held pages and growth out of range leave a sequence as it was; a count out of range is read as the
    nearest in range; pages given back twice do not pass the stack's end."""
    table = ints([[0, 1, 2, 9]] * 7)
    held, lengths = ints([2, 2, 5, -1, 2, 2, 1]), ints([-1, 65, 20, 20, 20, 20, 9])
    grow = ints([5, 1, 1, 1, 50, -21, 3])
    pool = serving.PagePool(dev, 10, 16, free=ints([5, 6, 7, 8] + [0] * 6), count=ints([4]))
    keep = table.clone(), held.clone()
    got = pool.plan(table, held, lengths, grow, 100)
    assert got.lengths.tolist() == [-1, 65, 20, 20, 20, 20, 12] and got.first.tolist() == [0] * 7 + [3]
    assert got.slots.tolist() == [9, 10, 11] + [-1] * 97 and got.positions[:4].tolist() == [9, 10, 11, -1]
    assert torch.equal(table, keep[0]) and torch.equal(held, keep[1]) and pool.count.item() == 4
    for wrong, free in ((99, 10), (-5, 0)):
        pool = serving.PagePool(dev, 10, 16, free=torch.arange(10, dtype=torch.int32, device="cuda"), count=ints([wrong]))
        t = torch.full((1, 40), -1, dtype=torch.int32, device="cuda")
        got = pool.plan(t, ints([0]), ints([0]), ints([160]), 200)
        assert got.first.tolist() == [0, 160 if free == 10 else 0] and pool.count.item() == 0
    behind = torch.full((30,), 77, dtype=torch.int32, device="cuda")
    pool = serving.PagePool(dev, 10, 16, free=behind[:10], count=ints([8]))
    pool.plan(ints([[0, 1, 2, 3, 4]]), ints([5]), ints([80]), ints([-80]), 0)
    assert pool.count.item() == 10 and behind[8:10].tolist() == [4, 3] and (behind[10:] == 77).all()


def test_plan_empty(dev):
    pool = serving.PagePool(dev, 10, 16)
    none = torch.empty(0, dtype=torch.int32, device="cuda")
    got = pool.plan(none.reshape(0, 4), none, none, none, 5)
    assert got.first.tolist() == [0] and got.slots.tolist() == [-1] * 5 and pool.count.item() == 10
    t = torch.zeros(2, 4, dtype=torch.int32, device="cuda")
    got = pool.plan(t, ints([0, 0]), ints([0, 0]), ints([17, 1]), 18)
    assert t.tolist() == [[0, 1, 0, 0], [2, 0, 0, 0]] and got.slots.tolist() == list(range(17)) + [32]


def test_plan_graph(dev):
    """A captured step (lengths in place) replayed: each replay grows the sequences once more."""
    g, lengths, held, table, plain, pool = setup(dev, 5, 6, 4, 60, 200, 40)
    t, h, n, grow = ints(table), ints(held), ints(lengths), ints([1, 3, 0, 5, 1, 2])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = pool.plan(t, h, n, grow, 12, out=n)
    for _ in range(4):
        graph.replay()
        torch.cuda.synchronize()
        want = plain.plan(table, held, lengths, grow.tolist(), 12)
        same(got, want, 12, False)
        lengths = want[0]
        assert t.tolist() == table and h.tolist() == held and pool.free[:len(plain.free)].tolist() == plain.free
        grow[3] = grow[3] - 4 if grow[3] > 0 else grow[3]


def test_plan_refusals(dev):
    pool = serving.PagePool(dev, 10, 16)
    t, x = torch.zeros(2, 4, dtype=torch.int32, device="cuda"), ints([0, 0])

    def refused(text, call):
        with pytest.raises(engine.EngineError, match=text):
            call()

    refused("one for each row", lambda: pool.plan(t, x[:1], x, x, 5))
    refused("one for each row", lambda: pool.plan(t, x, x, ints([1]), 5))
    refused("type torch.int64", lambda: pool.plan(t, x, x.long(), x, 5))
    refused("share memory", lambda: pool.plan(t[:1].expand(2, 4), x.clone(), x, x.clone(), 5))
    refused("one for each new token", lambda: pool.plan(t, x.clone(), x, x.clone(), 5, parents=ints([1])))
    refused("new tokens out of range", lambda: pool.plan(t, x.clone(), x, x.clone(), -1))
    refused("overlap", lambda: pool.plan(t, x, x, x.clone(), 5))
    refused("overlap", lambda: pool.plan(t, x.clone(), x, x.clone(), 5, out=t[0, :2]))
    refused("too many keys", lambda: serving.PagePool(dev, 10, 1 << 30).plan(t, x.clone(), x, x.clone(), 5))
    refused("pages out of range", lambda: serving.PagePool(dev, 0, 16))
    refused("go together", lambda: serving.PagePool(dev, 2, 16, free=ints([0, 1])))
    refused("10 are needed", lambda: serving.PagePool(dev, 10, 16, free=ints([0]), count=ints([1])))


# ------------------------------------------------------- accept
def walk(parents, tokens, chosen):
    path = [0]
    while True:
        at = [j for j in range(path[-1] + 1, len(parents)) if parents[j] == path[-1] and tokens[j] == chosen[path[-1]]]
        if not at:
            return path
        path.append(at[0])


def drafted(seed, new, values=3):
    """(parents, tokens, chosen), packed: few different tokens, so that walks go on and siblings agree."""
    g = torch.Generator().manual_seed(seed)
    parents = trees(g, new)[0]
    n = len(parents)
    return parents, torch.randint(0, values, (n,), generator=g).tolist(), torch.randint(0, values, (n,), generator=g).tolist()


@pytest.mark.parametrize("kv,dim,page,head_major", [("f32", 128, 16, False), ("f16", 64, 7, True), ("bf16", 128, 1, False),
                                                    ("q8_0", 128, 16, True), ("q8_0", 32, 24, False), ("bf16", 5, 16, False),
                                                    ("f32", 256, 64, False)])
@pytest.mark.parametrize("values", [1, 2])
def test_accept(dev, kv, dim, page, head_major, values):
    context, new = [0, 100, 33, 5, 64, 200, 8], [1, 64, 20, 0, 33, 64, 2]
    lengths = [c + n for c, n in zip(context, new)]
    g = torch.Generator().manual_seed(dim)
    table, pool, _ = make_table(g, lengths, page)
    layers = [make_cache(g, pool, page, 3, dim, kv, head_major) for _ in range(2)]
    parents, tokens, chosen = drafted(dim + values, new, values)
    if values == 1:  # chains as long as the tree
        parents = [j - 1 for n in new for j in range(n)]
    before = [[None if x is None else x.clone() for x in layer] for layer in layers]
    first = [2]
    for n in new:
        first.append(first[-1] + n)
    pad = [7, 7], [1]  # rows of no sequence
    lists = [pad[0] + x + pad[1] for x in (parents, tokens, chosen)]
    caches = [serving.PagedCache(dev, *layer) for layer in layers]
    got = serving.accept(caches, *(ints(x) for x in lists), table.cuda(), ints(lengths), ints(first))
    path = [-1] * len(lists[0])
    for b, n in enumerate(new):
        at = slice(first[b], first[b + 1])
        steps = walk(lists[0][at], lists[1][at], lists[2][at]) if n else []
        path[first[b]:first[b] + len(steps)] = steps
        assert got[0][b].item() == context[b] + len(steps) and got[1][b].item() == len(steps)
        assert got[3][b].item() == (lists[2][first[b] + steps[-1]] if n else -1)
        for old in before:
            for x in old:
                if x is None:
                    continue
                rows = [x[table[b, (context[b] + s) // page], (context[b] + s) % page].clone() for s in steps]
                for i, row in enumerate(rows):
                    t = context[b] + i
                    x[table[b, t // page], t % page] = row
    assert got[2].tolist() == path
    for layer, old in zip(layers, before):
        for x, y in zip(layer, old):
            assert (x is None and y is None) or torch.equal(x, y)


def test_accept_many_layers(dev):
    """More caches than a launch takes."""
    g = torch.Generator().manual_seed(1)
    table, pool, _ = make_table(g, [20], 16)
    layers = [make_cache(g, pool, 16, 1, 32, "bf16") for _ in range(70)]
    want = [layer[0][table[0, 0], 9].clone() for layer in layers]
    got = serving.accept([serving.PagedCache(dev, *layer) for layer in layers], ints([-1, 0, 0]), ints([0, 4, 5]),
                         ints([5, 1, 2]), table[:, :1].cuda(), ints([10]), ints([0, 3]))
    assert [x.tolist() for x in got] == [[9], [2], [0, 2, -1], [2]]
    for layer, row in zip(layers, want):
        assert torch.equal(layer[0][table[0, 0], 8], row)


def test_accept_out_of_range(dev):
    """Sequences out of range keep what they have."""
    g = torch.Generator().manual_seed(1)
    lengths = [30] * 6
    table, pool, _ = make_table(g, lengths, 16)
    cache = make_cache(g, pool, 16, 2, 64, "f32")
    keep = cache[0].clone()
    table[3, 1] = 1 << 20
    first = [0, 3, 6, 9, 12, 12, 90]
    n = 100
    got = serving.accept([serving.PagedCache(dev, *cache)], ints([j % 3 - 1 for j in range(n)]), ints([0] * n), ints([0] * n),
                         table.cuda(), ints([-4, 2, 33, 30, 30, 30]), ints(first))
    assert got[0].tolist() == [-4, 2, 33, 30, 30, 30] and got[1].tolist() == [0] * 6 and got[3].tolist() == [-1] * 6
    assert (got[2] == -1).all() and torch.equal(cache[0], keep)
    # bounds of rows: descending, past the rows
    got = serving.accept([serving.PagedCache(dev, *cache)], ints([-1, 0, 1]), ints([0] * 3), ints([0] * 3), table.cuda(),
                         ints(lengths), ints([0, 3, 2, 3, 4, -1, 3]))
    assert got[1].tolist() == [3, 0, 1, 0, 0, 0] and got[0][3:].tolist() == [30] * 3


def test_accept_refusals(dev):
    g = torch.Generator().manual_seed(1)
    a, b = make_cache(g, 4, 16, 2, 64, "f32"), make_cache(g, 5, 16, 2, 64, "f32")
    ca, cb = serving.PagedCache(dev, *a), serving.PagedCache(dev, *b)
    x, t, n, f = ints([-1, 0, 0]), ints([[0, 1]]), ints([20]), ints([0, 3])

    def refused(text, call):
        with pytest.raises(engine.EngineError, match=text):
            call()

    refused("a list of caches", lambda: serving.accept([], x, x, x, t, n, f))
    refused("differ in shape", lambda: serving.accept([ca, cb], x, x, x, t, n, f))
    refused("for each node", lambda: serving.accept([ca], x, x[:2], x, t, n, f))
    refused("one more than sequences", lambda: serving.accept([ca], x, x, x, t, n, f[:1]))
    refused("type torch.int64", lambda: serving.accept([ca], x.long(), x, x, t, n, f))
    shared = serving.PagedCache(dev, a[0][:1].expand(4, 16, 2, 64), a[1][:1].expand(4, 16, 2, 64))
    refused("read only", lambda: serving.accept([shared], x, x, x, t, n, f))


# ------------------------------------------------------- together
@pytest.mark.parametrize("kv", ["f32", "bf16", "q8_0"])
def test_rounds(dev, kv):
    """Prompts, then rounds of drafted trees: plan, append, attend_tree, accept, plan. What the accepted tokens
    are answered with, and the cache, are those of a decode that takes them one by one."""
    G, H, dim, page, B, layers = 2, 8, 64, 16, 3, 2
    x = TYPES["bf16" if kv == "q8_0" else kv]
    g = torch.Generator().manual_seed(3)

    def randn(*shape):
        return torch.randn(*shape, generator=g).to(x).cuda()

    def caches():
        kinds = [make_cache(torch.Generator().manual_seed(i), 60, page, G, dim, kv) for i in range(layers)]
        return [serving.PagedCache(dev, *k) for k in kinds]

    # keys, values and queries by token and layer: the same in both decodes
    vocab = 6
    embed = [[randn(vocab, h, dim) for h in (G, G, H)] for _ in range(layers)]
    rope = torch.randn(400, dim // 2, 2, generator=g).cuda()

    def step(cs, tokens, table, lengths, first, positions, attend):
        outs = []
        for c, (ek, ev, eq) in zip(cs, embed):
            i = tokens.long()
            q = c.append(ek[i], ev[i], table, lengths, first=first, q=eq[i], rope=rope, positions=positions)
            outs.append(attend(c, q))
        return outs

    def empty():
        return (torch.zeros(B, 12, dtype=torch.int32, device="cuda"), ints([0] * B), ints([0] * B))

    prompts = [40, 3, 17]
    tokens = torch.randint(0, vocab, (sum(prompts),), generator=g, dtype=torch.int32).cuda()
    # the model's choice: some hash of what the layers answer, the same for the same token and place
    trail = [[] for _ in range(B)]
    # drafted: by trees
    cs, pool = caches(), serving.PagePool(dev, 60, page)
    table, held, lengths = empty()
    plan = pool.plan(table, held, lengths, ints(prompts), sum(prompts))
    outs = step(cs, tokens, table, plan.lengths, plan.first, plan.positions,
                lambda c, q: c.attend_prompts(q, table, plan.lengths, plan.first))
    answers = [[[o[plan.first[b]:plan.first[b + 1]] for o in outs] for b in range(B)]]
    lengths, root = plan.lengths, [1, 2, 3]
    choose = torch.randint(0, vocab, (400, vocab), generator=g)  # the model's choice after a token at a place
    accepted_tokens = [[] for _ in range(B)]
    for _ in range(4):
        new = [int(torch.randint(2, 30, (1,), generator=g)) for _ in range(B)]
        parents, drafts, _ = drafted(sum(new), new, vocab)
        n, begin = sum(new), [0, new[0], new[0] + new[1], sum(new)]
        for b in range(B):
            drafts[begin[b]] = root[b]
        plan = pool.plan(table, held, lengths, ints(new), n, parents=ints(parents))
        assert plan.first.tolist() == begin
        outs = step(cs, ints(drafts), table, plan.lengths, plan.first, plan.positions,
                    lambda c, q: c.attend_tree(q, table, plan.lengths, plan.first, plan.ancestors))
        chosen = [int(choose[p, t]) for p, t in zip(plan.positions.tolist(), drafts)]
        lengths, count, path, following = serving.accept(cs, ints(parents), ints(drafts), ints(chosen), table, plan.lengths,
                                                         plan.first)
        for b in range(B):
            steps = path[begin[b]:begin[b] + int(count[b])].tolist()
            accepted_tokens[b] += [drafts[begin[b] + s] for s in steps]
            for s in steps:
                trail[b].append([o[begin[b] + s] for o in outs])
        root = following.tolist()
        # pages that rejected tokens held go back
        lengths = pool.plan(table, held, lengths, ints([0] * B), 0).lengths
        assert held.tolist() == [-(-t // page) for t in lengths.tolist()]
    assert max(len(a) for a in accepted_tokens) > 4  # at least one draft was followed
    assert pool.count.item() == 60 - sum(held.tolist())
    # one by one, in a cache of its own
    ones, pool1 = caches(), serving.PagePool(dev, 60, page)
    table1, held1, lengths1 = empty()
    plan = pool1.plan(table1, held1, lengths1, ints(prompts), sum(prompts))
    outs = step(ones, tokens, table1, plan.lengths, plan.first, plan.positions,
                lambda c, q: c.attend_prompts(q, table1, plan.lengths, plan.first))
    for b in range(B):
        for a, o in zip(answers[0][b], outs):
            assert torch.equal(a, o[plan.first[b]:plan.first[b + 1]])
    lengths1 = plan.lengths
    half = 2.0 ** -7 if x == torch.bfloat16 else 2.0 ** -17  # two roundings of the outputs, of weights, of 32-bit sums
    for i in range(max(len(a) for a in accepted_tokens)):
        grow = [int(i < len(a)) for a in accepted_tokens]
        live = [b for b in range(B) if grow[b]]
        plan = pool1.plan(table1, held1, lengths1, ints(grow), sum(grow))
        lengths1 = plan.lengths
        outs = step(ones, ints([accepted_tokens[b][i] for b in live]), table1, lengths1, plan.first, plan.positions,
                    lambda c, q: c.attend_prompts(q, table1, lengths1, plan.first))
        for k, b in enumerate(live):
            for a, o in zip(trail[b][i], outs):
                assert (a.double() - o[k].double()).abs().max() <= 4 * half * 5  # values of at most 5
    assert lengths1.tolist() == lengths.tolist()
    for c, d in zip(cs, ones):
        for b in range(B):
            for t in range(int(lengths[b])):
                a, o = (int(table[b, t // page]), t % page), (int(table1[b, t // page]), t % page)
                assert torch.equal(c.k[a], d.k[o]) and torch.equal(c.v[a], d.v[o])
                assert c.k_scale is None or torch.equal(c.k_scale[a], d.k_scale[o])


@pytest.mark.parametrize("kv", ["f16", "q8_0"])
def test_round_in_a_graph(dev, kv):
    """A round captured whole (plan, append, attend_tree, accept, plan) and replayed from states put back, with eager
    rounds between: each replay leaves what the eager round left, bit for bit."""
    G, H, dim, page, B, n = 2, 8, 64, 16, 4, 75
    x = TYPES["bf16" if kv == "q8_0" else kv]
    g = torch.Generator().manual_seed(5)
    cache = serving.PagedCache(dev, *make_cache(g, 40, page, G, dim, kv))
    pool = serving.PagePool(dev, 40, page)
    table, held = torch.zeros(B, 12, dtype=torch.int32, device="cuda"), ints([0] * B)
    lengths = pool.plan(table, held, ints([0] * B), ints([37, 0, 16, 100]), 153).lengths
    nodes = [5, 1, 64, 3]  # two rows of 75 are no sequence's
    parents, drafts, _ = drafted(sum(nodes), nodes, 3)
    parents, drafts = ints(parents + [-1, -1]), ints(drafts + [0, 0])
    chosen = torch.randint(0, 3, (n,), generator=g, dtype=torch.int32).cuda()
    grow, none = ints(nodes), ints([0] * B)
    k, v, q = (torch.randn(n, h, dim, generator=g).to(x).cuda() for h in (G, G, H))
    rope = torch.randn(400, dim // 2, 2, generator=g).cuda()
    out = torch.empty_like(q)

    def one():
        out.fill_(7)
        plan = pool.plan(table, held, lengths, grow, n, parents=parents)
        turned = cache.append(k, v, table, plan.lengths, plan.first, q=q, rope=rope, positions=plan.positions)
        cache.attend_tree(turned, table, plan.lengths, plan.first, plan.ancestors, out=out)
        new, accepted, path, following = serving.accept([cache], parents, drafts, chosen, table, plan.lengths, plan.first)
        return [*plan, out, new, accepted, path, following, pool.plan(table, held, new, none, 0).lengths]

    state = [t for t in (table, held, pool.free, pool.count, cache.k, cache.v, cache.k_scale, cache.v_scale) if t is not None]
    before = [t.clone() for t in state]

    def back():
        for t, b in zip(state, before):
            t.copy_(b)

    want = [t.clone() for t in one()]
    after = [t.clone() for t in state]
    assert want[6][-2:].eq(7).all() and not want[6][:-2].eq(7).all() and want[8].tolist()[1] == 1
    back()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = one()
    for _ in range(4):
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)) and all(torch.equal(a, b) for a, b in zip(state, after))
        back()
        one()
        back()
