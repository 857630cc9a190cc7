"""What attention over the paged cache keeps of its scores, weights and values: weights in two parts
of 16 bits, queries over 8-bit codes, the ends of the types' ranges, outputs of another type than the
queries'."""
import importlib
import math

import pytest
import torch

from serving_reference import HALF, TINY, TYPES, attend, make_cache, make_table, values

engine = importlib.import_module("qwen-30brust_amd")
serving = importlib.import_module("qwen-30brust_amd.serving")

pytestmark = pytest.mark.gpu
U = 2.0 ** -24  # half a step of 32 bits


@pytest.fixture(scope="module")
def dev():
    d = engine.Device(0)
    yield d
    d.close()


def close(got, want, bound):
    g = got.cpu().double()
    assert torch.isfinite(g).all()
    tol = bound + HALF[got.dtype] * (want.abs() + bound) + TINY[got.dtype]
    off = (g - want).abs()
    assert (off <= tol).all(), (off / tol).max()


# Relative error of a weight that enters a product of 16 bits in two parts: the second part is off by
# half its step, and it is at most half a step of the first.
SPLIT = {"bf16": 2.0 ** -17, "f16": 2.0 ** -23, "q8_0": 2.0 ** -23}


def pairs(kv, dim, n, heads, g):
    """A cache of one sequence of n keys in pages of 16 and queries whose scores are exact: q = (a, 2^-13,
    0 ..), k = (s, 0 or 1, 0 ..) with s of few bits.  Key i's value is +1 or -1 (every second key) in
    column i / 2 alone, so that an output column is the difference of two weights, or (where heads'
    second element is 0 and values are not negated) a weight."""
    s = torch.randint(-60, 61, (n // 2,), generator=g).repeat_interleave(2)
    k, v = torch.zeros(n, dim), torch.zeros(n, dim)
    k[:, 0], k[1::2, 1] = s / 64, 1.0
    i = torch.arange(n)
    v[i, i // 2] = 1.0 - 2.0 * (i % 2)
    q = torch.zeros(1, heads, dim)
    q[0, :, 0] = 1 - torch.arange(heads) / 32
    q[0, :, 1] = 2.0 ** -13
    page = 16
    shape = (n // page, page, 1, dim)
    if kv == "q8_0":
        d = torch.full((n, dim // 32), 1.0)
        d[:, 0] = 1 / 64
        codes = k.clone()
        codes[:, :32] *= 64
        cache = (codes, v, d, torch.ones(n, dim // 32))
        cache = (cache[0].to(torch.int8).reshape(shape).cuda(), cache[1].to(torch.int8).reshape(shape).cuda(),
                 cache[2].half().reshape(*shape[:3], -1).cuda(), cache[3].half().reshape(*shape[:3], -1).cuda())
    else:
        cache = (k.to(TYPES[kv]).reshape(shape).cuda(), v.to(TYPES[kv]).reshape(shape).cuda(), None, None)
    return cache, q


# A weight in 32 bits of such a case (|s| <= 1): s off by 3 half steps, s - m by |s - m| <= 12 of them
# (m at most 8 from the top), the exponential by 2, all times ln 2 but the last; the sum by as much and
# its n / 4 + 8 additions; the division by 2
def weight_error(n):
    return (2 * (3 + 12 + 2) + n / 4 + 8 + 2) * U


@pytest.mark.parametrize("q,kv,dim", [("bf16", "bf16", 128), ("bf16", "bf16", 64), ("f16", "f16", 128), ("f16", "f16", 64),
                                      ("bf16", "q8_0", 128), ("f16", "q8_0", 64)])
@pytest.mark.parametrize("n", [16, 64, 128])
def test_differences_of_weights(dev, q, kv, dim, n):
    """Outputs that are a difference of two nearly equal weights show the weights' own error, not the
    output's rounding."""
    cache, query = pairs(kv, dim, n, 8, torch.Generator().manual_seed(n))
    query = query.to(TYPES[q]).cuda()
    table = torch.arange(n // 16, dtype=torch.int32)[None]
    k, v = values(cache[0], cache[2]), values(cache[1], cache[3])
    want, p, _ = attend(query, k, v, table, [n], 1.0)
    size = attend(query, k, v.abs(), table, [n], 1.0)[0]  # both weights
    c = serving.PagedCache(dev, *cache)
    lengths = torch.tensor([n], dtype=torch.int32).cuda()
    got = c.attend(query, table.cuda(), lengths, scale=1.0)
    close(got, want, (SPLIT[kv] + weight_error(n)) * size)
    # a 32-bit output keeps 32 bits
    out = torch.empty(1, 8, dim, device="cuda")
    c.attend(query, table.cuda(), lengths, scale=1.0, out=out)
    close(out, want, weight_error(n) * size)


@pytest.mark.parametrize("q,kv", [("bf16", "bf16"), ("f16", "f16"), ("bf16", "q8_0"), ("f32", "bf16"), ("f16", "f32")])
@pytest.mark.parametrize("out", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dim,heads,kvheads", [(128, 32, 4), (64, 6, 2), (256, 4, 2), (96, 4, 2)])
def test_output_types(dev, q, kv, out, dim, heads, kvheads):
    """Outputs of every type, ragged lengths, the same with and without key weights."""
    g = torch.Generator().manual_seed(dim)
    lengths = [129, 1, 0, 700]
    table, pool, _ = make_table(g, lengths, 16)
    cache = make_cache(g, pool, 16, kvheads, dim, kv)
    query = (2 * torch.randn(4, heads, dim, generator=g)).to(TYPES[q]).cuda()
    k, v = values(cache[0], cache[2]), values(cache[1], cache[3])
    want, _, bound = attend(query, k, v, table, lengths, 0.9 / math.sqrt(dim))
    narrow = out != "f32" and dim in (64, 128) and q != "f32" and (kv == "q8_0" or q == kv)
    bound = bound + (SPLIT[kv] if narrow else 0.0) * v.abs().max()
    c = serving.PagedCache(dev, *cache)
    n = torch.tensor(lengths, dtype=torch.int32).cuda()
    held = torch.full((4, heads, dim), 7.0, dtype=TYPES[out], device="cuda")
    assert c.attend(query, table.cuda(), n, scale=0.9 / math.sqrt(dim), out=held) is held
    close(held, want, bound)
    again = torch.full_like(held, 5.0)
    w = torch.zeros(4, kvheads, 704, device="cuda")
    c.attend(query, table.cuda(), n, 704, scale=0.9 / math.sqrt(dim), out=again, weights=w)
    assert torch.equal(held, again)


@pytest.mark.parametrize("q", ["bf16", "f16"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("small", [-12, -20, -24])
def test_small_query_elements_over_codes(dev, q, dim, small):
    """A query whose largest element meets keys of 0 there: the others, 2^small of it, keep their bits."""
    g = torch.Generator().manual_seed(dim - small)
    lengths, page = [5, 40, 333], 16
    table, pool, _ = make_table(g, lengths, page)
    cache = make_cache(g, pool, page, 2, dim, "q8_0")
    cache[0][..., 0] = 0
    # f16's own smallest values bound what it can hold
    top = 1.0 if q == "bf16" else 1024.0
    query = torch.randn(3, 8, dim, generator=g) * 2.0 ** small * top
    query[..., 0] = top
    query = query.to(TYPES[q]).cuda()
    scale = 2.0 ** -small / top / math.sqrt(dim)
    want, p, bound = attend(query, values(cache[0], cache[2]), values(cache[1], cache[3]), table, lengths, scale)
    w = torch.zeros(3, 2, 336, device="cuda")
    n = torch.tensor(lengths, dtype=torch.int32).cuda()
    got, _ = serving.PagedCache(dev, *cache).attend(query, table.cuda(), n, 336, scale=scale, weights=w)
    close(got, want, bound + SPLIT["q8_0"] * 5)
    for b, t in enumerate(lengths):
        # as the outputs' bound: a score's error is at most (d + 3) half steps of its terms' sum
        qq = query[b].cpu().double().reshape(2, 4, dim)
        kk = values(cache[0], cache[2])[table[b].long()[torch.arange(t) // page], torch.arange(t) % page].transpose(0, 1)
        size = scale * (qq.abs()[:, :, None] * kk.abs()[:, None]).sum(-1).amax()
        rel = (4 * (dim + 3) * size + 16 * size + 2 * (t + 8) + 64 + 4) * U
        assert ((w[b, :, :t].cpu().double() - p[b]).abs() <= rel * p[b] + 2.0 ** -23 * p[b]).all()


@pytest.mark.parametrize("kv,power", [("q8_0", p) for p in (-125, -112, -60, 0, 60, 112, 125)] +
                         [("bf16", p) for p in (-100, -60, 60, 112, 125)])
def test_queries_of_any_size(dev, kv, power):
    """bf16 queries near both ends of their range, with the scale that brings the scores back."""
    g = torch.Generator().manual_seed(200 + power)
    lengths, dim = [70, 3], 128
    table, pool, _ = make_table(g, lengths, 16)
    cache = make_cache(g, pool, 16, 1, dim, kv)
    # the largest lies at 3.9 x 2^power
    query = torch.randn(2, 4, dim, generator=g).clamp(-3.9, 3.9)
    query[0, 0, 0], query[1, 1, 5] = 3.9, -3.9
    query = (query * 2.0 ** power).bfloat16().cuda()
    scale = 2.0 ** -power / math.sqrt(dim)
    if power > 100:  # a scale, and scores, in 32 bits' normal range
        cache[0 if kv == "bf16" else 2].mul_(2.0 ** -10)
        scale *= 2.0 ** 10
    want, _, bound = attend(query, values(cache[0], cache[2]), values(cache[1], cache[3]), table, lengths, scale)
    got = serving.PagedCache(dev, *cache).attend(query, table.cuda(), torch.tensor(lengths, dtype=torch.int32).cuda(), scale=scale)
    close(got, want, bound + SPLIT[kv] * 5)


@pytest.mark.parametrize("q,kv", [("f16", "f16"), ("f16", "q8_0"), ("bf16", "q8_0"), ("bf16", "bf16"), ("f32", "f16")])
@pytest.mark.parametrize("gap", [12, 23, 25])
def test_one_key_far_above_the_others(dev, q, kv, gap):
    """A first key `gap` above all others whose value is 0: the output is the many others' alone, each
    weight e^-gap.  1,024 sequences and KV heads of 8,192 keys, so that no split over the keys gives the
    others a wave without the first one."""
    dim, n, page, G, B = 64, 8192, 16, 16, 64
    k, v = torch.zeros(2, page, G, dim), torch.zeros(2, page, G, dim)
    k[0, 0, :, 0] = gap
    v[:] = 96.0 + torch.arange(G)[:, None]
    v[0, 0] = 0.0
    if kv == "q8_0":
        ones = torch.ones(2, page, G, dim // 32, dtype=torch.float16)
        cache = (k.to(torch.int8).cuda(), v.to(torch.int8).cuda(), ones.cuda(), ones.clone().cuda())
    else:
        cache = (k.to(TYPES[kv]).cuda(), v.to(TYPES[kv]).cuda(), None, None)
    query = torch.zeros(B, G, dim)
    query[..., 0] = 1.0
    table = torch.ones(B, n // page, dtype=torch.int32)
    table[:, 0] = 0
    got = serving.PagedCache(dev, *cache).attend(query.to(TYPES[q]).cuda(), table.cuda(),
                                                 torch.full((B,), n, dtype=torch.int32).cuda(), scale=1.0)
    others = (n - 1) * math.exp(-gap)
    want = (others / (1 + others) * (96.0 + torch.arange(G, dtype=torch.float64)))[None, :, None].expand(B, G, dim)
    # scores are whole numbers: off by 3 |s| half steps, s - m by |s - m| < 64, the exponential by 2; sums
    # of n weights in runs, at most n additions; below 2^-43 of the largest weight nothing counts
    bound = (2 * (3 * gap + 64 + 2) + n + 64) * U * want + 2.0 ** -17 * want * (kv == "bf16") + n * 2.0 ** -43 * 112
    close(got, want, bound)


@pytest.mark.parametrize("q,kv", [("bf16", "bf16"), ("f32", "bf16"), ("f32", "f32"), ("bf16", "f32")])
@pytest.mark.parametrize("dim", [64, 128, 256, 96])
def test_large_values(dev, q, kv, dim):
    """Values whose sum over the keys is still in 32 bits' range."""
    g = torch.Generator().manual_seed(dim)
    lengths = [8, 1, 5, 0]
    table, pool, _ = make_table(g, lengths, 16)
    k, v, _, _ = make_cache(g, pool, 16, 2, dim, kv)
    v.clamp_(-2, 2).mul_(2e37)
    query = (2 * torch.randn(4, 8, dim, generator=g)).to(TYPES[q]).cuda()
    want, _, bound = attend(query, values(k, None), values(v, None), table, lengths, 1 / math.sqrt(dim))
    got = serving.PagedCache(dev, k, v).attend(query, table.cuda(), torch.tensor(lengths, dtype=torch.int32).cuda())
    close(got, want, bound + (SPLIT["bf16"] * 4e37 if q == kv == "bf16" else 0.0))


@pytest.mark.parametrize("x,to", [("f32", "bf16"), ("bf16", "f32"), ("f16", "bf16"), ("bf16", "f16")])
@pytest.mark.parametrize("dim", [128, 34])
def test_append_queries_of_another_type(dev, x, to, dim):
    """Queries rounded to the type of q_out, beside keys in a cache of another type."""
    g = torch.Generator().manual_seed(dim)
    H, G, n, page = 6, 2, 21, 16
    table = torch.tensor([[2, 0]], dtype=torch.int32)
    k, v, _, _ = make_cache(g, 3, page, G, dim, to)
    q_new = torch.randn(n, H, dim, generator=g).to(TYPES[x])
    kv_new = torch.randn(2, n, G, dim, generator=g).to(TYPES[x])
    w = 1 + 0.3 * torch.randn(dim, generator=g)
    out = torch.full((n, H, dim), 9.0, dtype=TYPES[to], device="cuda")
    c = serving.PagedCache(dev, k, v)
    got = c.append(kv_new[0].cuda(), kv_new[1].cuda(), table.cuda(), torch.tensor([n], dtype=torch.int32).cuda(),
                   torch.tensor([0, n], dtype=torch.int32).cuda(), q=q_new.cuda(), q_out=out, q_norm=w.cuda(), eps=1e-5)
    assert got is out
    y = q_new.double()
    want = y / torch.sqrt((y * y).mean(-1, keepdim=True) + 1e-5) * w.double()
    close(out, want, (dim + 12) * U * want.abs())
    at = torch.arange(n)
    assert torch.equal(k.cpu()[table[0].long()[at // page], at % page], kv_new[0].to(TYPES[to]))
    assert torch.equal(v.cpu()[table[0].long()[at // page], at % page], kv_new[1].to(TYPES[to]))


@pytest.mark.parametrize("q,kv,size", [("f16", "f16", -14), ("bf16", "q8_0", -14), ("f32", "q8_0", -14), ("f32", "f16", -14),
                                       ("bf16", "bf16", -90), ("f32", "f32", -90), ("f32", "bf16", -90)])
@pytest.mark.parametrize("dim", [128, 64])
def test_small_values(dev, q, kv, size, dim):
    """Values of 2^size, in f16 below its normal range (a step of 2^-24 there)."""
    g = torch.Generator().manual_seed(dim)
    lengths = [70, 1, 333]
    table, pool, _ = make_table(g, lengths, 16)
    cache = make_cache(g, pool, 16, 2, dim, kv)
    cache[3 if kv == "q8_0" else 1].mul_(2.0 ** size)
    query = (2 * torch.randn(3, 8, dim, generator=g)).to(TYPES[q]).cuda()
    out = torch.empty(3, 8, dim, dtype=torch.bfloat16 if q == "f16" else TYPES[q], device="cuda")
    v = values(cache[1], cache[3])
    want, _, bound = attend(query, values(cache[0], cache[2]), v, table, lengths, 1 / math.sqrt(dim))
    serving.PagedCache(dev, *cache).attend(query, table.cuda(), torch.tensor(lengths, dtype=torch.int32).cuda(), out=out)
    close(out, want, bound + (SPLIT[kv] if q != "f32" else 0.0) * v.abs().max())


def test_blocks_past_the_scale(dev):
    """An 8-bit block whose scale is past f16's range reads as NaN, its neighbours as they are."""
    g = torch.Generator().manual_seed(1)
    cache = make_cache(g, 2, 16, 1, 64, "q8_0")
    c = serving.PagedCache(dev, *cache)
    table, n = torch.tensor([[1]], dtype=torch.int32).cuda(), torch.tensor([3], dtype=torch.int32).cuda()
    new = torch.randn(2, 3, 1, 64, generator=g)
    new[1, 1, 0, 40] = 9e6
    new[1, 2, 0, 41] = -8.3e6  # 65,354 x 127
    c.append(new[0].cuda(), new[1].cuda(), table, n, torch.tensor([0, 3], dtype=torch.int32).cuda())
    for q in (torch.zeros(1, 2, 64, device="cuda"), torch.zeros(1, 2, 64, dtype=torch.bfloat16, device="cuda")):
        out = c.attend(q, table, n).cpu()
        assert torch.isfinite(out[..., :32]).all() and out[..., 32:].isnan().all()
