"""Attention of several new tokens where the range of its types ends: small and large queries, scales and values, codes
whose values pass f16, values that are not finite; and 8-bit caches under bf16 queries at the lengths and masks of the
other kinds."""
import importlib
import math

import pytest
import torch

from prompts_reference import attend_many, close, make, signed, split_of, trees
from serving_reference import values
from test_gpu_prompts import at, ints, run

engine = importlib.import_module("qwen-30brust_amd")
serving = importlib.import_module("qwen-30brust_amd.serving")

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    d = engine.Device(0)
    yield d
    d.close()


# ------------------------------------------------------- queries and scales of any size over codes
@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("scale,size", [(1e-30, 1e-12), (2.0 ** -12, 2.0 ** -126), (1e-30, 1.0), (0.0, 1.0), (-0.3, 1.0), (3.0, 1.0)])
def test_queries_of_any_size_over_codes(dev, tree, dim, scale, size):
    """The factor that takes a row's queries into f16's range, and its inverse in the scale, change no score, also where
    the product with the scale leaves 32 bits' range."""
    def change(cache, table, lengths, first, query):
        query.copy_((query.float().clamp(-3.9, 3.9) / 4 * size).to(query.dtype))
        query[:, 0] = (query[:, 0].float() / 64).to(query.dtype)  # rows of different sizes

    run(dev, [70, 0, 400], [33, 20, 40], 4, 2, dim, 16, "bf16", "q8_0", tree=tree, scale=scale, change=change)


@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("dim", [64, 128])
def test_subnormal_queries_over_codes(dev, tree, dim):
    """Rows of nothing but subnormal numbers, under a scale that brings the scores back."""
    def change(cache, table, lengths, first, query):
        query.copy_((query.float().clamp(-3.9, 3.9) / 4 * 2.0 ** -126).to(query.dtype))
        query[:, 0] = (query[:, 0].float() / 16).to(query.dtype)

    run(dev, [70, 0, 400], [33, 20, 40], 4, 2, dim, 16, "bf16", "q8_0", tree=tree, scale=2.0 ** 125, change=change)


@pytest.mark.parametrize("dim", [64, 128])
def test_large_scale_over_codes(dev, dim):
    """Scores of 0 under a scale whose product with the queries' factor passes 32 bits: the mean of the values."""
    def change(cache, table, lengths, first, query):
        query.copy_((query.float().clamp(-3.9, 3.9) * 2.0 ** 125).to(query.dtype))
        cache[0].zero_()

    run(dev, [70, 0], [33, 60], 4, 2, dim, 16, "bf16", "q8_0", scale=2.0 ** 20, change=change)


@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("dim", [64, 128])
def test_wide_query_rows_over_codes(dev, tree, dim):
    """Rows whose largest element meets codes of 0: the others, 2^-45 to 2^-20 of it, decide, and what is below 2^-39 is lost."""
    def change(cache, table, lengths, first, query):
        g = torch.Generator().manual_seed(7)
        power = torch.randint(-45, -19, query.shape, generator=g)
        power[..., 0] = 0
        query.copy_((query.double().clamp(-2, 2) * 2.0 ** power.double()).to(query.dtype))
        query[..., 0] = 2.0
        cache[0][..., 0] = 0

    run(dev, [70, 0, 300], [33, 20, 40], 4, 2, dim, 16, "bf16", "q8_0", tree=tree, scale=2.0 ** 18, change=change)


def test_infinite_queries_over_codes(dev):
    """An infinity beside large elements: the scores are its alone, -inf for codes above 0 under -inf."""
    cache, table, lengths, first, query = make(3, [20], [40], 4, 2, 64, 16, "bf16", "q8_0")
    query.copy_((query.float().sign() * 2.0 ** 100).to(query.dtype))
    cache[0][..., 5] = 3
    query[:, 0, 5], query[:, 1, 5] = -math.inf, math.inf
    c = serving.PagedCache(dev, *cache)
    got = c.attend_prompts(query.cuda(), table.cuda(), ints(lengths), ints(first), scale=2.0 ** -100)
    assert (got[:, 0] == 0).all() and got[:, 1].isnan().all()
    want, bound = attend_many(query[:, 2:], values(cache[0], cache[2])[:, :, 1:], values(cache[1], cache[3])[:, :, 1:], table,
                              lengths, first, 2.0 ** -100, None, split_of("bf16", "q8_0"))
    close(got[:, 2:], want, bound)


@pytest.mark.parametrize("q,kv,dim", [("bf16", "bf16", 64), ("f16", "f16", 128), ("bf16", "q8_0", 64), ("f32", "f32", 64), ("f32", "bf16", 64),
                                      ("bf16", "bf16", 96)])
@pytest.mark.parametrize("what", [math.nan, math.inf, -math.inf])
def test_scale_of_zero(dev, q, kv, dim, what):
    """0 times what is not finite is NaN; the other rows are means."""
    cache, table, lengths, first, query = make(3, [20, 0], [40, 9], 4, 2, dim, 16, q, kv)
    query[7, 1, 3] = query[45, 2, dim - 1] = what
    c = serving.PagedCache(dev, *cache)
    got = c.attend_prompts(query.cuda(), table.cuda(), ints(lengths), ints(first), scale=0.0)
    assert got[7, 1].isnan().all() and got[45, 2].isnan().all()
    query[7, 1, 3] = query[45, 2, dim - 1] = 0
    got[7, 1] = got[45, 2] = 0
    want, bound = attend_many(query, values(cache[0], cache[2]), values(cache[1], cache[3]), table, lengths, first, 0.0, None,
                              split_of(q, kv))
    want[7, 1] = want[45, 2] = 0
    close(got, want, bound)


# ------------------------------------------------------- values near the end of their range
@pytest.mark.parametrize("dim", [64, 128, 256, 96])
@pytest.mark.parametrize("q,kv", [("bf16", "bf16"), ("f32", "bf16"), ("f32", "f32"), ("f16", "f16")])
def test_sums_that_fit(dev, q, kv, dim):
    """Values of 2^128 / keys, under scores that run 7.5 powers of two ahead of those in front: no weight passes 1, so
    the sum stays in range."""
    n, new = 440, 40
    most = 60000.0 if kv == "f16" else 2.0 ** 119

    def change(cache, table, lengths, first, query):
        query.zero_()
        query[:, :, 0] = 1.0
        cache[0].zero_()
        cache[1].copy_((cache[1].float().sign() * most).to(cache[1].dtype))
        cache[1][..., 0] = most
        for t in range(64, n + new):
            cache[0][at(table, 0, t)][:, 0] = 5.1875  # 7.48 ln 2

    got = run(dev, [n], [new], 4, 2, dim, 16, q, kv, scale=1.0, change=change)
    assert torch.isfinite(got).all()


@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("dim", [64, 128])
def test_codes_past_f16(dev, tree, dim):
    """Code times scale past 65504 is not finite in every row that sees it, wherever it lies, and in no other."""
    context, new = [300, 40, 0], [40, 60, 64]
    cache, table, lengths, first, query = make(4, context, new, 4, 2, dim, 16, "bf16", "q8_0")
    for b, (c, n) in enumerate(zip(context, new)):
        for t in {c // 3, c + n // 2, c + n - 1}:
            cache[1][at(table, b, t)][b % 2, 1 + t % 9] = 127 if t % 2 else -127
            cache[3][at(table, b, t)][b % 2, 0] = 700.0
    k, v = values(cache[0], cache[2]), values(cache[1], cache[3])
    assert (v.abs() > 65520).sum() > 0 and (v.abs() > 65504).sum() == (v.abs() > 65520).sum()
    bits = trees(torch.Generator().manual_seed(1), new)[1] if tree else None
    rounded = v.float().half().double()
    want, bound = attend_many(query, k, rounded, table, lengths, first, 0.01, bits, split_of("bf16", "q8_0"))
    c = serving.PagedCache(dev, *cache)
    args = (query.cuda(), table.cuda(), ints(lengths), ints(first))
    got = c.attend_tree(*args, signed(bits).cuda(), scale=0.01) if tree else c.attend_prompts(*args, scale=0.01)
    assert not torch.isfinite(want).all()
    # values of up to 65504 beside the infinite ones, rounded as `rounded` is
    close(got, want, bound)


@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("dim", [64, 128])
def test_masked_scales(dev, tree, dim):
    """NaN and infinite scales of keys and values that a row does not see change nothing; those of values that it sees
    come out as the formula has them, and a NaN key scale as NaN."""
    context, new = [100, 0, 33], [40, 60, 30]
    cache, table, lengths, first, query = make(4, context, new, 8, 2, dim, 16, "bf16", "q8_0")
    ks, vs = cache[2], cache[3]
    for b, (c, n) in enumerate(zip(context, new)):
        for t, (x, value) in zip((c + n - 1, c + n // 2, c + n // 3, c + 5),
                                 ((vs, math.nan), (vs, math.inf), (vs, -math.inf), (ks, math.nan))):
            x[at(table, b, t)][b % 2, t % (dim // 32)] = value
        for t in range(c + n, -(-(c + n) // 16) * 16):
            ks[at(table, b, t)] = math.nan
            vs[at(table, b, t)] = math.inf
    k, v = values(cache[0], cache[2]), values(cache[1], cache[3])
    bits = trees(torch.Generator().manual_seed(1), new)[1] if tree else None
    more = table, lengths, first, 0.1, bits, split_of("bf16", "q8_0")
    want = attend_many(query, k, v, *more)[0]
    # rows that see a NaN key are NaN; the others' error has no part of it
    bound = attend_many(query, k.nan_to_num(0), v, *more)[1]
    c = serving.PagedCache(dev, *cache)
    args = (query.cuda(), table.cuda(), ints(lengths), ints(first))
    got = c.attend_tree(*args, signed(bits).cuda(), scale=0.1) if tree else c.attend_prompts(*args, scale=0.1)
    close(got, want, bound)


# ------------------------------------------------------- lengths over codes
@pytest.mark.parametrize("heads,kvheads,dim", [(8, 2, 128), (8, 1, 64), (16, 2, 64)])
@pytest.mark.parametrize("context,new", [([0], [1500]), ([3100], [400]), ([0, 2900, 17], [700, 130, 450])])
def test_longer_over_codes(dev, heads, kvheads, dim, context, new):
    run(dev, context, new, heads, kvheads, dim, 16, "bf16", "q8_0")


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("context,new", [([30001], [3]), ([9000, 3, 500], [64, 64, 1])])
def test_tree_long_over_codes(dev, dim, context, new):
    run(dev, context, new, 8, 1, dim, 64, "bf16", "q8_0", tree=True)


@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("heads", [1, 3, 130])
def test_groups_over_codes(dev, tree, heads):
    run(dev, [50, 0], [20, 9], heads, 1, 64, 16, "bf16", "q8_0", tree=tree)
