"""The key-value cache in pages (serving.PagedCache over qh_paged_*) against plain 64-bit
restatements: appending with norm and RoPE, attention of one token per sequence, eviction, and the
three together as a serving loop uses them."""
import importlib
import math

import pytest
import torch

from serving_reference import HALF, TINY, TYPES, attend, gathered, make_cache, make_table, quantise, values

engine = importlib.import_module("qwen-30brust_amd")
serving = importlib.import_module("qwen-30brust_amd.serving")

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    d = engine.Device(0)
    yield d
    d.close()


def close(got, want, bound):
    """Every value within `bound` of `want` and one rounding to its type."""
    g = got.cpu().double()
    assert torch.equal(torch.isfinite(g), torch.isfinite(want))
    fine = torch.isfinite(want)
    assert torch.equal(g[~fine & ~want.isnan()], want[~fine & ~want.isnan()])
    tol = bound + HALF[got.dtype] * (want.abs() + bound) + TINY[got.dtype]
    off = (g - want).abs()
    assert (off <= tol)[fine].all(), (off / tol)[fine].max()


# ------------------------------------------------------------------ attention
def case(seed, lengths, heads, kvheads, dim, page, q, kv, head_major=False):
    g = torch.Generator().manual_seed(seed)
    table, pool, _ = make_table(g, lengths, page)
    cache = make_cache(g, pool, page, kvheads, dim, kv, head_major)
    query = (2 * torch.randn(len(lengths), heads, dim, generator=g)).to(TYPES[q]).cuda()
    return cache, table, query


def split_error(q, kv):
    """Relative error of a softmax weight that goes to the matrix cores in two parts of the cache's
    16-bit type, each cut off: 2^-15 of bf16's two (8 bits each), 2^-21 of f16's; its sum is taken
    before."""
    if q == "f32" or kv == "f32":
        return 0.0
    return 2.0 ** -21 if kv == "f16" else 2.0 ** -15


def run_attend(dev, lengths, heads, kvheads, dim, page, q, kv, head_major=False, weights=True, most=None, seed=1):
    cache, table, query = case(seed, lengths, heads, kvheads, dim, page, q, kv, head_major)
    c = serving.PagedCache(dev, *cache)
    n = torch.tensor(lengths, dtype=torch.int32).cuda()
    k, v = values(cache[0], cache[2]), values(cache[1], cache[3])
    scale = 0.9 / math.sqrt(dim)
    want, p, bound = attend(query, k, v, table, lengths, scale)
    # sum p |v| is at most the largest |v|
    bound = bound + split_error(q, kv) * v.abs().max()
    got = c.attend(query, table.cuda(), n, most, scale=scale)
    close(got, want, bound)
    if not weights:
        return
    size = max(max(lengths), 1)
    before = torch.rand(len(lengths), kvheads, size + 3)
    after = torch.full((len(lengths), kvheads, size + 5), -5.0)
    wb, wa = before.cuda(), after.cuda()
    got2, w = c.attend(query, table.cuda(), n, size, scale=scale, weights=wb, weights_out=wa)
    assert w is wa
    close(got2, want, bound)
    for b, t in enumerate(lengths):
        exact = before[b, :, :t].double() + p[b]
        # as the output's: a sum of G weights of at most 1, each off by the bound for |v| = 1
        G, d = heads // kvheads, dim
        qq = query[b].cpu().double().reshape(kvheads, G, d)
        kk = gathered(k, table, b, t)
        size_s = scale * (qq.abs()[:, :, None] * kk.abs()[:, None]).sum(-1).amax() if t else 0.0
        rel = (4 * (d + 3) * size_s + 8 * 2 * size_s + 2 * (t + 8) + 64 + G) * 2.0 ** -24
        assert ((w[b, :, :t].cpu().double() - exact).abs() <= rel * p[b] + 2.0 ** -23 * exact).all()
    # left as they were
    for b, t in enumerate(lengths):
        assert (w[b, :, t:] == -5.0).all()
    # in place: the same values
    x = wb.clone()
    got3, y = c.attend(query, table.cuda(), n, size, scale=scale, weights=x)
    assert y is x and torch.equal(got3, got2)
    for b, t in enumerate(lengths):
        assert torch.equal(x[b, :, :t], wa[b, :, :t]) and torch.equal(x[b, :, t:], wb[b, :, t:])


KINDS = [("f32", "f32"), ("f16", "f16"), ("bf16", "bf16"), ("bf16", "q8_0"), ("f32", "q8_0"), ("f16", "bf16"),
         ("f32", "f16"), ("bf16", "f32"), ("f16", "q8_0")]
EDGES = [0, 1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 256, 257, 300]


@pytest.mark.parametrize("q,kv", KINDS)
@pytest.mark.parametrize("heads,kvheads,dim", [(32, 4, 128), (8, 8, 64), (6, 2, 128), (10, 1, 64), (16, 1, 128), (36, 2, 64)])
def test_attend_edges(dev, q, kv, heads, kvheads, dim):
    run_attend(dev, EDGES, heads, kvheads, dim, 16, q, kv)


@pytest.mark.parametrize("q,kv", KINDS)
@pytest.mark.parametrize("page", [1, 7, 16, 24, 32, 48, 64, 200])
def test_attend_pages(dev, q, kv, page):
    run_attend(dev, [129, 64, 201, 1, 0, 333], 8, 2, 128, page, q, kv, head_major=page % 3 == 0, seed=page)


@pytest.mark.parametrize("q,kv", [("f32", "f32"), ("bf16", "bf16"), ("f16", "f16"), ("bf16", "q8_0")])
@pytest.mark.parametrize("heads,kvheads,dim", [(4, 2, 96), (3, 1, 256), (4, 4, 32), (5, 5, 160), (20, 2, 256),
                                               (8, 4, 192)])
def test_attend_other_widths(dev, q, kv, heads, kvheads, dim):
    run_attend(dev, [200, 1, 77], heads, kvheads, dim, 16, q, kv)


@pytest.mark.parametrize("q,kv", [("f32", "f32"), ("bf16", "bf16"), ("f16", "f16")])
@pytest.mark.parametrize("dim", [1, 2, 5, 80, 97, 250])
def test_attend_odd_widths(dev, q, kv, dim):
    run_attend(dev, [90, 1, 33], 4, 2, dim, 16, q, kv)


@pytest.mark.parametrize("q,kv", [("f32", "f32"), ("bf16", "bf16"), ("f16", "f16"), ("bf16", "q8_0")])
@pytest.mark.parametrize("lengths", [[5003], [4096, 3, 0, 1025], [40000, 17]])
def test_attend_long(dev, q, kv, lengths):
    run_attend(dev, lengths, 16, 2, 128, 64 if lengths[0] > 5003 else 16, q, kv)


@pytest.mark.parametrize("batch", [1, 70, 300])
def test_attend_batches(dev, batch):
    lengths = [(37 * i * i) % 150 for i in range(batch)]
    run_attend(dev, lengths, 4, 2, 64, 16, "bf16", "bf16")


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
def test_attend_views(dev, kind):
    """Queries that are a slice of a projection's rows, at a data pointer and with strides that are
    not aligned to 16 bytes; an output with strides; keys and values in one tensor."""
    g = torch.Generator().manual_seed(3)
    lengths, page, G, d, H = [77, 130, 1], 16, 2, 128, 8
    table, pool, _ = make_table(g, lengths, page)
    both = torch.randn(pool, page, G, 2 * d + 1, generator=g).to(TYPES[kind]).cuda()
    k, v = both[..., :d], both[..., d:2 * d]
    rows = torch.randn(3, (H + 2 * G) * d + 3, generator=g).to(TYPES[kind]).cuda()
    q = rows[:, 1:1 + H * d].unflatten(1, (H, d))
    out = torch.full((3, H, d + 5), 7.0, dtype=TYPES[kind]).cuda()
    c = serving.PagedCache(dev, k, v)
    n = torch.tensor(lengths, dtype=torch.int32).cuda()
    want, _, bound = attend(q, values(k, None), values(v, None), table, lengths, 1 / math.sqrt(d))
    got = c.attend(q, table.cuda(), n, out=out[..., 2:2 + d])
    close(got, want, bound + split_error(kind, kind) * v.abs().max().cpu().double())
    assert (out[..., :2] == 7).all() and (out[..., 2 + d:] == 7).all()


@pytest.mark.parametrize("q,kv", [("f32", "f32"), ("bf16", "bf16"), ("f16", "f16"), ("bf16", "q8_0"), ("f32", "bf16")])
@pytest.mark.parametrize("dim", [128, 96])
def test_attend_values_that_are_not_finite(dev, q, kv, dim):
    """What lies behind the last key is never used; an infinite value of a key that has weight comes
    out infinite, a NaN as NaN, in its own column and sequence only; keys of -inf have no weight."""
    lengths, page = [33, 70, 20, 18, 5], 16
    cache, table, query = case(5, lengths, 8, 2, dim, page, q, kv)
    k, v, ks, vs = cache
    big = ks if kv == "q8_0" else k
    # slots behind the last key
    for b, n in enumerate(lengths):
        for t in range(n, -(-n // page) * page):
            p, s = table[b, t // page], t % page
            big[p, s] = math.nan
            (vs if kv == "q8_0" else v)[p, s] = math.inf
    query[:, :, 0] = query[:, :, 0].abs() + 0.5
    if kv != "q8_0":
        v[table[1, 2], 3, 1, 5] = math.inf           # sequence 1, key 35
        v[table[1, 1], 0, 0, 7] = math.nan           # key 16
        k[table[2, 0], 4, :, 0] = -math.inf          # sequence 2, key 4: no weight
        for t in range(18):                          # sequence 3: every score -inf
            k[table[3, t // page], t % page, :, 0] = -math.inf
    n = torch.tensor(lengths, dtype=torch.int32).cuda()
    scale = 1 / math.sqrt(dim)
    kk, vv = values(k, ks), values(v, vs)
    for b, t in enumerate(lengths):  # the restatement does not look behind the keys either
        for i in range(t, -(-t // page) * page):
            kk[table[b, i // page], i % page] = vv[table[b, i // page], i % page] = 0
    want, _, bound = attend(query, kk, vv, table, lengths, scale)
    got = serving.PagedCache(dev, *cache).attend(query, table.cuda(), n).cpu().double()
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.isinf(), want.isinf())
    if kv != "q8_0":
        assert want[1, 4:, 5].isinf().all() and want[1, :4, 7].isnan().all() and (want[3] == 0).all()
        assert (got[3] == 0).all()
    fine = torch.isfinite(want)
    top = vv[torch.isfinite(vv)].abs().max()
    assert ((got - want).abs()[fine] <= (2 ** -8 if q == "bf16" else 2 ** -10) * top).all()


def test_attend_out_of_range(dev):
    """Page ids and lengths out of range: NaN for that sequence, the others as without them."""
    lengths = [40, 50, 60, 70, 9]
    for q, kv in [("f32", "f32"), ("bf16", "bf16")]:
        for dim in (128, 80):
            cache, table, query = case(6, lengths, 4, 2, dim, 16, q, kv)
            c = serving.PagedCache(dev, *cache)
            n = torch.tensor(lengths, dtype=torch.int32)
            good = c.attend(query, table.cuda(), n.cuda(), 80).cpu()
            bad, m = table.clone(), n.clone()
            bad[0, 1], bad[1, 0] = cache[0].shape[0], -1
            m[2], m[3] = -3, 81
            w = torch.full((5, 2, 80), 2.0).cuda()
            got, _ = c.attend(query, bad.cuda(), m.cuda(), 80, weights=w)
            got = got.cpu()
            assert got[:4].isnan().all() and torch.equal(got[4], good[4])
            assert (w[2:4] == 2).all() and w[0, :, :40].isnan().all()
            got = c.attend(query, bad.cuda(), m.cuda(), 80).cpu()
            assert got[:4].isnan().all() and torch.equal(got[4], good[4])


def test_attend_far_offsets(dev):
    """Pages whose elements lie behind the 2^32nd."""
    g = torch.Generator().manual_seed(8)
    page, d, pages = 16, 64, (1 << 21) + 40
    big = torch.empty(pages, page, 1, 2 * d, dtype=torch.float16, device="cuda")
    ids = [pages - 1, 3, pages - 7, 1 << 20, (1 << 21) + 1]
    for p in ids:
        big[p] = torch.randn(page, 1, 2 * d, generator=g).half().cuda()
    table = torch.tensor([ids], dtype=torch.int32)
    small = torch.stack([big[p].cpu() for p in ids])
    n = [73]
    q = torch.randn(1, 4, d, generator=g).half().cuda()
    own = torch.arange(5, dtype=torch.int32)[None]
    want, _, bound = attend(q, small[..., :d].double(), small[..., d:].double(), own, n, 1 / 8)
    c = serving.PagedCache(dev, big[..., :d], big[..., d:])
    got = c.attend(q, table.cuda(), torch.tensor(n, dtype=torch.int32).cuda())
    close(got, want, bound + 2.0 ** -21 * 5)
    # an append there, and an eviction from there
    row = torch.randn(2, 1, 1, d, generator=g).half().cuda()
    n2 = torch.tensor([74], dtype=torch.int32).cuda()
    c.append(row[0], row[1], table.cuda(), n2)
    assert torch.equal(big[ids[4], 9, 0, :d], row[0, 0, 0]) and torch.equal(big[ids[4], 9, 0, d:], row[1, 0, 0])
    to = torch.tensor([[pages - 3, 5]], dtype=torch.int32)
    w = torch.rand(1, 1, 74, generator=g).cuda()
    kept, _, _ = c.evict(w, table.cuda(), n2, 20, to.cuda(), first=1, recent=2)
    kept = kept[0, 0].long()
    src = torch.stack([big[p] for p in ids]).flatten(0, 1)
    dst = torch.stack([big[p] for p in to[0].tolist()]).flatten(0, 1)
    assert torch.equal(dst[:20], src[kept])


# --------------------------------------------------------------------- append
def turned(x, w, eps, rope, pos):
    x = x.double()
    if w is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * w.double()
    if rope is not None:
        cs = rope[pos.long()].double()[:, None]
        a, b = x.chunk(2, -1)
        x = torch.cat([a * cs[..., 0] - b * cs[..., 1], a * cs[..., 1] + b * cs[..., 0]], -1)
    return x


def angles(n, d):
    a = torch.arange(n, dtype=torch.float64)[:, None] * 1e6 ** (-2 * torch.arange(d // 2, dtype=torch.float64) / d)
    return torch.stack([a.cos(), a.sin()], -1).float()


@pytest.mark.parametrize("x,kv", [("f32", "f32"), ("f32", "f16"), ("bf16", "bf16"), ("f16", "f16"), ("bf16", "f32")])
@pytest.mark.parametrize("heads,kvheads,dim", [(32, 4, 128), (4, 4, 64), (3, 1, 256), (2, 2, 34), (0, 2, 128), (1, 1, 2),
                                               (6, 2, 96)])
@pytest.mark.parametrize("norm", [True, False])
@pytest.mark.parametrize("skip", [1, 8])
def test_append(dev, x, kv, heads, kvheads, dim, norm, skip):
    """Ragged prompts with norm and RoPE (every second pattern: neither), rows in front of and behind
    the sequences left out; rows aligned to one element and to eight."""
    g = torch.Generator().manual_seed(dim + heads)
    page, counts, lengths = 16, [5, 1, 0, 19, 3], [37, 1, 8, 19, 3 + 2 * 16]
    table, pool, _ = make_table(g, lengths, page)
    k, v, _, _ = make_cache(g, pool, page, kvheads, dim, kv)
    lead, n = 2, 2 + sum(counts) + 3
    first = torch.tensor([lead] + [lead + sum(counts[:i + 1]) for i in range(len(counts))], dtype=torch.int32)
    rows = torch.randn(n, (heads + 2 * kvheads) * dim + skip, generator=g).to(TYPES[x]).cuda()[:, skip:]
    q_new = rows[:, :heads * dim].unflatten(1, (heads, dim)) if heads else None
    k_new, v_new = (m.unflatten(1, (kvheads, dim)) for m in rows[:, heads * dim:].chunk(2, 1))
    qw, kw = (1 + 0.3 * torch.randn(dim, generator=g) for _ in range(2))
    rope, pos = angles(600, dim), torch.randint(0, 600, (n,), generator=g).int()
    k0, v0 = k.cpu().clone(), v.cpu().clone()
    more, out = {}, None
    if heads:
        out = torch.full((n, heads, dim), 9.0, dtype=TYPES[x], device="cuda")
        more = dict(q=q_new, q_out=out)
    if norm:
        more.update(k_norm=kw.cuda(), eps=1e-5, rope=rope.cuda(), positions=pos.cuda())
        if heads:
            more["q_norm"] = qw.cuda()
    c = serving.PagedCache(dev, k, v)
    got = c.append(k_new, v_new, table.cuda(), torch.tensor(lengths, dtype=torch.int32).cuda(), first.cuda(), **more)
    assert got is out
    kx = turned(k_new.cpu(), kw if norm else None, 1e-5, rope if norm else None, pos)
    # a norm is off by at most dim + 8 half steps of 32 bits (sum, root, division, two products), a
    # rotation of two such values by four more
    tol = (dim + 12) * 2.0 ** -24 if norm else 0.0
    kd, vd = k0.double(), v0.double()
    kb = torch.zeros_like(kd)
    live = torch.zeros(n, dtype=torch.bool)
    for b, (m, t) in enumerate(zip(counts, lengths)):
        for i in range(m):
            r, s = lead + sum(counts[:b]) + i, t - m + i
            p = table[b, s // page]
            kd[p, s % page], vd[p, s % page] = kx[r], v_new[r].cpu().double()
            kb[p, s % page] = tol * (kx[r].abs() + kx[r].roll(dim // 2, -1).abs())
            live[r] = True
    step = HALF[k.dtype] if HALF[k.dtype] > 2.0 ** -24 or norm else 0.0
    off = (k.cpu().double() - kd).abs()
    moved = kd != k0.double()
    assert (off <= kb + step * (kd.abs() + kb) + TINY[k.dtype])[moved].all() and (off[~moved] <= TINY[k.dtype]).all()
    assert torch.equal(v.cpu(), vd.to(v.dtype))
    if heads:
        qx = turned(q_new.cpu(), qw if norm else None, 1e-5, rope if norm else None, pos)
        assert (out[~live] == 9).all()
        b = tol * (qx.abs() + qx.roll(dim // 2, -1).abs())
        close(out[live], qx[live], b[live])


@pytest.mark.parametrize("x", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("kvheads,dim", [(4, 128), (1, 32), (2, 96), (3, 256)])
def test_append_8bit(dev, x, kvheads, dim):
    """Codes and scales equal to the formula's, through a head-major cache too; a block of zeros, of
    values that are not finite, of tiny ones."""
    g = torch.Generator().manual_seed(kvheads)
    lengths = [40, 3]
    table, pool, _ = make_table(g, lengths, 16)
    for head_major in (False, True):
        c = make_cache(g, pool, 16, kvheads, dim, "q8_0", head_major)
        before = [t.clone() for t in c]
        k_new, v_new = (torch.randn(13, kvheads, dim, generator=g).to(TYPES[x]) for _ in range(2))
        k_new[3, 0, :32] = 0
        k_new[4] *= 1e-7
        k_new[5] *= 3e4
        v_new[6, 0, 1], v_new[7, 0, 31] = math.inf, math.nan
        serving.PagedCache(dev, *c).append(k_new.cuda(), v_new.cuda(), table.cuda(),
                                           torch.tensor(lengths, dtype=torch.int32).cuda(),
                                           torch.tensor([0, 11, 13], dtype=torch.int32).cuda())
        want = [t.cpu().clone() for t in before]
        for b, (r0, m, t) in enumerate([(0, 11, 40), (11, 2, 3)]):
            for i in range(m):
                s = t - m + i
                p = table[b, s // 16]
                for j, new in ((0, k_new), (1, v_new)):
                    codes, d = quantise(new[r0 + i])
                    fine = torch.isfinite(new[r0 + i].float()).unflatten(-1, (-1, 32)).all(-1)
                    want[2 + j][p, s % 16] = torch.where(fine, d, torch.full_like(d, math.nan))
                    want[j][p, s % 16] = torch.where(fine.repeat_interleave(32, -1), codes, torch.zeros_like(codes))
        for got, w in zip(c, want):
            assert torch.equal(got.cpu().nan_to_num(77.0) if got.dtype == torch.float16 else got.cpu(),
                               w.nan_to_num(77.0) if w.dtype == torch.float16 else w)


def test_append_8bit_next_to_ties(dev):
    """Values on, and one and two steps of f32 beside, the middle between two codes: the code of the
    exact quotient."""
    top = 0.987  # a scale of 1.99 * 2^-8: a step of a value is down to half a step of its quotient
    f = (torch.tensor(top) / 127).half().float()
    mid = (torch.arange(126) + 0.5).repeat_interleave(5).reshape(126, 5) * f  # exact: 7 + 11 bits
    near = [mid[:, 0]]
    for way in (-math.inf, math.inf):
        x = mid[:, 0]
        for _ in range(2):
            x = torch.nextafter(x, torch.tensor(way))
            near.append(x)
    x = torch.stack(near, 1).reshape(-1)
    x = torch.cat([x, -x])
    x = torch.cat([x, torch.zeros(-len(x) % 31)]).reshape(-1, 31)
    x = torch.cat([x, torch.full((len(x), 1), top)], 1)  # every block has the same scale
    want = (x.double() / f.double()).round().clamp(-127, 127).to(torch.int8)
    n, g = -(-len(x) // 8), torch.Generator().manual_seed(1)
    rows = torch.zeros(n * 8, 32)
    rows[:len(x)] = x
    for kvheads, dim in ((2, 128), (1, 256), (8, 32)):
        c = make_cache(g, 4, 64, kvheads, dim, "q8_0")
        k_new = rows.reshape(n, kvheads, dim)
        serving.PagedCache(dev, *c).append(k_new.cuda(), k_new.cuda(), torch.tensor([[2, 0, 3]], dtype=torch.int32).cuda(),
                                           torch.tensor([n], dtype=torch.int32).cuda(),
                                           torch.tensor([0, n], dtype=torch.int32).cuda())
        for held in c[:2]:
            got = held[[2, 0, 3]].reshape(-1, kvheads * dim)[:n].reshape(-1, 32)[:len(x)]
            assert torch.equal(got.cpu(), want)


def test_append_one_token_each(dev):
    """Without `first`: a token for each sequence at its end; padded rows, lengths and pages out of
    range and a position outside the table."""
    g = torch.Generator().manual_seed(2)
    lengths = [17, 0, 16, 1, 200, 33, 40]
    table, pool, _ = make_table(g, [17, 0, 16, 1, 0, 33, 40], 16)
    bad = torch.cat([table, torch.full((7, 2), -9, dtype=torch.int32)], 1)  # 80 keys a row
    bad[5, 2] = pool
    k, v, _, _ = make_cache(g, pool, 16, 2, 64, "f32")
    k0, v0 = k.cpu().clone(), v.cpu().clone()
    new = torch.randn(3, 7, 2, 64, generator=g)
    out = torch.full((7, 2, 64), 3.0, device="cuda")
    pos = torch.tensor([5, 0, 700, -1, 0, 1, 2], dtype=torch.int32)
    c = serving.PagedCache(dev, k, v)
    c.append(new[0].cuda(), new[1].cuda(), bad.cuda(), torch.tensor(lengths, dtype=torch.int32).cuda(), q=new[2].cuda(),
             q_out=out, rope=angles(100, 64).cuda(), positions=pos.cuda())
    turn = turned(new[0], None, 0, angles(100, 64), pos.clamp(0, 99))
    for b, s in [(0, 16), (2, 15), (3, 0), (6, 39)]:
        p = table[b, s // 16]
        k0[p, s % 16] = math.nan if b in (2, 3) else turn[b].float()
        v0[p, s % 16] = new[1, b]
    assert torch.equal(v.cpu(), v0)
    assert torch.equal(k.cpu().isnan(), k0.isnan())
    assert (k.cpu() - k0).nan_to_num().abs().max() <= 2.0 ** -22 * 5
    assert (out[[1, 4]] == 3).all() and out[[2, 3]].isnan().all() and not out[[0, 5, 6]].isnan().any()


# ------------------------------------------------------------------- eviction
def order(w):
    b = w.contiguous().view(torch.int32).long()
    return torch.where(b < 0, -b - 1 - (1 << 31), b)


def keep_of(w, n, keep, first, recent):
    """The kept indexes of one KV head, ascending."""
    if n <= keep:
        return list(range(n))
    o = order(w[:n]).tolist()
    mid = sorted(range(first, n - recent), key=lambda t: (-o[t], t))[:keep - first - recent]
    return sorted(list(range(first)) + mid + list(range(n - recent, n)))


def run_evict(dev, lengths, keep, first, recent, page, kv, kvheads=2, dim=64, weights=None, head_major=False, seed=1):
    g = torch.Generator().manual_seed(seed)
    new = -(-keep // page)
    table, pool, spare = make_table(g, lengths, page, spare=new * len(lengths) + 1)
    cache = make_cache(g, pool, page, kvheads, dim, kv, head_major)
    most = max(max(lengths), 1)
    w = torch.randn(len(lengths), kvheads, most + 2, generator=g).exp() if weights is None else weights(g, len(lengths), kvheads, most + 2)
    to = spare[:new * len(lengths)].reshape(len(lengths), new)
    before = [None if t is None else t.cpu().clone() for t in cache]
    c = serving.PagedCache(dev, *cache)
    n = torch.tensor(lengths, dtype=torch.int32).cuda()
    kept, kw, length = c.evict(w.cuda(), table.cuda(), n, keep, to.cuda(), first=first, recent=recent, most=most)
    assert length.tolist() == [min(t, keep) for t in lengths]
    kept, kw = kept.cpu(), kw.cpu()
    for b, t in enumerate(lengths):
        for h in range(kvheads):
            ids = keep_of(w[b, h], t, keep, first, recent)
            m = len(ids)
            assert kept[b, h, :m].tolist() == ids
            assert (kept[b, h, m:] == -1).all() and (kw[b, h, m:] == 0).all()
            assert torch.equal(kw[b, h, :m].view(torch.int32), w[b, h][ids].contiguous().view(torch.int32))
            if not m:
                continue
            src, dst = torch.tensor(ids), torch.arange(m)
            for x in before:
                if x is not None:
                    x[to[b].long()[dst // page], dst % page, h] = x[table[b].long()[src // page], src % page, h]
    for x, y in zip(before, cache):
        if x is not None:
            assert torch.equal(x, y.cpu())  # the kept rows moved, and nothing else


@pytest.mark.parametrize("kv", ["f32", "f16", "bf16", "q8_0"])
@pytest.mark.parametrize("keep,first,recent", [(64, 4, 16), (64, 0, 0), (1, 0, 0), (1, 1, 0), (40, 8, 32), (129, 1, 127)])
def test_evict(dev, kv, keep, first, recent):
    run_evict(dev, [0, 1, keep - 1, keep, keep + 1, 333, 1025, 2047], keep, first, recent, 16, kv)


@pytest.mark.parametrize("page", [1, 7, 64, 200])
@pytest.mark.parametrize("kvheads,dim", [(1, 128), (3, 96), (8, 256)])
def test_evict_shapes(dev, page, kvheads, dim):
    run_evict(dev, [500, 77], 100, 3, 20, page, "bf16", kvheads, dim, head_major=page == 64, seed=page)
    run_evict(dev, [500, 77], 100, 3, 20, page, "q8_0", kvheads, dim, head_major=page == 64, seed=page)


@pytest.mark.parametrize("dim", [1, 5, 33, 250])
def test_evict_odd_widths(dev, dim):
    for kv in ("f32", "f16"):
        run_evict(dev, [90, 20], 33, 1, 3, 16, kv, 2, dim)


def test_evict_ties_and_strange_weights(dev):
    """Equal weights (the lower index stays), zeros, infinities, NaN of both signs, -0 below 0."""
    def same(g, b, h, n):
        return torch.full((b, h, n), 0.25)

    def few(g, b, h, n):
        return torch.randint(0, 3, (b, h, n), generator=g).float()

    def strange(g, b, h, n):
        w = torch.tensor([0.0, -0.0, math.inf, -math.inf, math.nan, -math.nan, 1.0, -1.0, 1e-42, 3e38])
        return w[torch.randint(0, len(w), (b, h, n), generator=g)]

    for f in (same, few, strange):
        run_evict(dev, [1500, 300, 100], 100, 4, 16, 16, "f32", weights=f)


def test_evict_long(dev):
    run_evict(dev, [20011, 70000], 5000, 4, 700, 64, "f16", 2, 64)


def test_evict_out_of_range(dev):
    """A sequence with a length or a page out of range keeps nothing, the others as without it."""
    g = torch.Generator().manual_seed(4)
    lengths = [50, 60, 70, 80, 90]
    table, pool, spare = make_table(g, lengths, 16, spare=12)
    cache = make_cache(g, pool, 16, 2, 64, "bf16")
    to = spare[:10].reshape(5, 2).clone()
    table[0, 3], to[1, 1] = pool, -1
    n = torch.tensor(lengths, dtype=torch.int32)
    n[2], n[3] = -1, 97
    before = [t.cpu().clone() for t in cache[:2]]
    w = torch.rand(5, 2, 96, generator=g)
    kept, kw, length = serving.PagedCache(dev, *cache).evict(w.cuda(), table.cuda(), n.cuda(), 30, to.cuda(), recent=5)
    assert length.tolist() == [0, 0, 0, 0, 30]
    assert (kept[:4] == -1).all() and (kw[:4] == 0).all()
    assert kept[4, 0].tolist() == keep_of(w[4, 0], 90, 30, 0, 5)
    changed = {int(p) for x, y in zip(before, cache) for p in (x != y.cpu()).flatten(1).any(1).nonzero()}
    assert changed == set(to[4].tolist())


# ------------------------------------------------------------------- together
@pytest.mark.parametrize("x,kv", [("f32", "f32"), ("bf16", "bf16"), ("bf16", "q8_0")])
def test_serving_loop(dev, x, kv):
    """Prompts appended, decode steps that append, attend and add up weights, an eviction, more
    steps over the new pages: every output against attention over the keys that a plain program
    would hold."""
    g = torch.Generator().manual_seed(11)
    H, G, d, page, B = 8, 2, 64, 16, 3
    prompts, rope = [40, 9, 75], angles(400, d)
    per = 8
    order_ = torch.randperm(2 * B * per, generator=g).int()
    table, to = order_[:B * per].reshape(B, per), order_[B * per:].reshape(B, per)
    cache = make_cache(g, 2 * B * per, page, G, d, kv)
    c = serving.PagedCache(dev, *cache)
    qw, kw = (1 + 0.2 * torch.randn(d, generator=g) for _ in range(2))
    more = dict(q_norm=qw.cuda(), k_norm=kw.cuda(), rope=rope.cuda())

    def rows(n):
        r = torch.randn(n, (H + 2 * G) * d, generator=g).to(TYPES[x]).cuda()
        return r[:, :H * d].unflatten(1, (H, d)), *(m.unflatten(1, (G, d)) for m in r[:, H * d:].chunk(2, 1))

    n = torch.tensor(prompts, dtype=torch.int32).cuda()
    first = torch.tensor([0, 40, 49, 124], dtype=torch.int32).cuda()
    q, k, v = rows(124)
    c.append(k, v, table.cuda(), n, first, q=q, **more)
    weights = torch.zeros(B, G, per * page, device="cuda")
    position = n.clone()

    def step(table, n, weights, position):
        q, k, v = rows(B)
        n += 1
        q = c.append(k, v, table.cuda(), n, q=q, positions=position, **more)
        position += 1
        out, _ = c.attend(q, table.cuda(), n, per * page, weights=weights)
        want, p, bound = attend(q, values(cache[0], cache[2]), values(cache[1], cache[3]), table, n.tolist(),
                                1 / math.sqrt(d))
        close(out, want, bound + split_error(x, kv) * 6)
        return p

    total = [torch.zeros(G, 0, dtype=torch.float64) for _ in range(B)]
    for _ in range(5):
        p = step(table, n, weights, position)
        for b in range(B):
            total[b] = torch.nn.functional.pad(total[b], (0, p[b].shape[1] - total[b].shape[1])) + p[b]
    for b in range(B):
        t = total[b].shape[1]
        assert (weights[b, :, :t].cpu().double() - total[b]).abs().max() <= 1e-4
    kept, w, n = c.evict(weights, table.cuda(), n, 32, to.cuda(), first=2, recent=8)
    assert n.tolist() == [32, 14, 32]
    for b in range(B):
        for h in range(G):
            ids = keep_of(weights[b, h].cpu(), prompts[b] + 5, 32, 2, 8)
            assert kept[b, h, :len(ids)].tolist() == ids
    weights = torch.zeros(B, G, per * page, device="cuda")
    weights[:, :, :32] = w
    for _ in range(3):
        step(to, n, weights, position)


def test_streams_and_graphs(dev):
    """Calls on a side stream; a captured decode step (append, attend with weights, evict) replayed
    three times with new inputs, eager calls between, against eager results."""
    g = torch.Generator().manual_seed(12)
    lengths, page, H, G, d, keep = [300, 1, 90, 0], 16, 8, 2, 128, 64
    table, pool, spare = make_table(g, lengths, page, spare=16)
    to = spare[:16].reshape(4, 4).contiguous().cuda()
    cache = make_cache(g, pool, page, G, d, "bf16")
    c = serving.PagedCache(dev, *cache)
    table, n = table.cuda(), torch.tensor(lengths, dtype=torch.int32).cuda()
    q, k, v = (torch.randn(4, h, d, generator=g).bfloat16().cuda() for h in (H, G, G))
    w = torch.zeros(4, G, 304, device="cuda")

    def work():
        c.append(k, v, table, n)
        out, after = c.attend(q, table, n, 304, weights=w, weights_out=torch.zeros_like(w))
        return (out, *c.evict(after, table, n, keep, to, first=4, recent=8))

    eager = [t.clone() for t in work()]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = work()
    side.synchronize()
    for a, b in zip(got, eager):
        assert torch.equal(a, b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = work()
    for i in range(3):
        for t in (q, k, v):
            t.copy_(torch.randn(t.shape, generator=g).bfloat16())
        n.copy_(torch.tensor([300 - 40 * i, 1 - i % 2, 90, 0], dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        replayed = [t.clone() for t in held]
        torch.cuda.synchronize()
        for a, b in zip(replayed, work()):
            assert torch.equal(a, b)


def test_calls_agree(dev):
    """The same call twice gives the same bits."""
    cache, table, query = case(9, [900, 2000, 5], 32, 4, 128, 16, "bf16", "bf16")
    c = serving.PagedCache(dev, *cache)
    n = torch.tensor([900, 2000, 5], dtype=torch.int32).cuda()
    w = torch.zeros(3, 4, 2000, device="cuda")
    a = c.attend(query, table.cuda(), n, weights_out=w)
    a = [t.clone() for t in a]
    for _ in range(3):
        b = c.attend(query, table.cuda(), n, weights_out=torch.zeros_like(w))
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_no_sequences(dev):
    cache, table, _ = case(1, [5], 4, 2, 64, 16, "f32", "f32")
    c = serving.PagedCache(dev, *cache)
    n = torch.zeros(0, dtype=torch.int32, device="cuda")
    t = torch.zeros(0, 4, dtype=torch.int32, device="cuda")
    q = torch.zeros(0, 4, 64, device="cuda")
    assert c.attend(q, t, n).shape == (0, 4, 64)
    assert c.append(q[:, :2], q[:, :2], t, n) is None
    kept, w, m = c.evict(torch.zeros(0, 2, 9, device="cuda"), t, n, 4, t)
    assert kept.shape == w.shape == (0, 2, 4) and m.shape == (0,)
    # rows of padding alone
    n, t = torch.zeros(3, dtype=torch.int32, device="cuda"), torch.full((3, 0), 0, dtype=torch.int32, device="cuda")
    q = torch.ones(3, 4, 64, device="cuda")
    assert (c.attend(q, t, n) == 0).all()
    _, _, m = c.evict(torch.zeros(3, 2, 0, device="cuda"), t, n, 4, t)
    assert m.tolist() == [0, 0, 0]
