"""What attention of several new tokens keeps of its softmax weights: two parts of 16 bits, as the attention of single
tokens does."""
import importlib
import math

import pytest
import torch

from prompts_reference import attend_many, close, make, signed, trees
from serving_reference import TYPES, attend, values
from test_gpu_paged_precision import SPLIT, U, pairs
from test_gpu_prompts import ints

engine = importlib.import_module("qwen-30brust_amd")
serving = importlib.import_module("qwen-30brust_amd.serving")

pytestmark = pytest.mark.gpu

KINDS = [("bf16", "bf16"), ("f16", "f16")]


@pytest.fixture(scope="module")
def dev():
    d = engine.Device(0)
    yield d
    d.close()


def calls(c, query, table, lengths, first, bits, **more):
    args = (query.cuda(), table.cuda(), ints(lengths), ints(first))
    yield c.attend_prompts(*args, **more), False
    yield c.attend_tree(*args, signed(bits).cuda(), **more), True


def weight_error(n):
    """Relative error of a weight of scores up to 1.5 in 32 bits: their power of two lies up to 16 from the reference, so
    the difference is off by 16 half steps, the scale by 3 with the score's own products, the exponential by 2; the same
    in the sum, with its n / 4 + 8 additions; the division by 2."""
    return (2 * (16 + 3 + 2) + n / 4 + 8 + 2) * U


@pytest.mark.parametrize("q,kv", KINDS)
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("n", [16, 64, 128])
def test_differences_of_weights(dev, q, kv, dim, n):
    """Outputs that are a difference of two nearly equal weights show the weights' own error, not the output's."""
    cache, query = pairs(kv, dim, n, 8, torch.Generator().manual_seed(n))
    query = query.to(TYPES[q])
    table = torch.arange(n // 16, dtype=torch.int32)[None]
    k, v = values(cache[0], cache[2]), values(cache[1], cache[3])
    want = attend(query, k, v, table, [n], 1.0)[0]
    size = attend(query, k, v.abs(), table, [n], 1.0)[0]  # both weights
    # f16: and half a step of 2^-24 beside a largest weight of at least 2^11
    low = n * 2.0 ** -36 if kv != "bf16" else 0.0
    for got, _ in calls(serving.PagedCache(dev, *cache), query, table, [n], [0, 1], [1], scale=1.0):
        close(got, want, (SPLIT[kv] + weight_error(n)) * size + low * size.amax())


@pytest.mark.parametrize("q,kv", KINDS)
@pytest.mark.parametrize("heads,kvheads,dim", [(16, 2, 128), (8, 8, 64), (4, 2, 256), (6, 2, 96)])
def test_outputs_within_their_rounding(dev, q, kv, heads, kvheads, dim):
    """Prompts, pieces and trees: an output is off by its own rounding and what 17 or 23 bits of the weights leave."""
    context, new = [0, 700, 33, 2100], [64, 1, 40, 30]
    cache, table, lengths, first, query = make(9, context, new, heads, kvheads, dim, 16, q, kv)
    k, v = values(cache[0], cache[2]), values(cache[1], cache[3])
    bits, scale = trees(torch.Generator().manual_seed(2), new)[1], 0.9 / math.sqrt(dim)
    for got, tree in calls(serving.PagedCache(dev, *cache), query, table, lengths, first, bits, scale=scale):
        want, bound = attend_many(query, k, v, table, lengths, first, scale, bits if tree else None, SPLIT[kv])
        low = 2 * max(lengths) * 2.0 ** -36 * v.abs().max() if kv != "bf16" else 0.0
        close(got, want, bound + low)
