"""Sequences without new tokens between those that have some, and batches without sequences."""
import importlib

import pytest
import torch

from prompts_reference import attend_many, close, make, split_of
from serving_reference import make_cache, values
from test_gpu_prompts import ints

engine = importlib.import_module("qwen-30brust_amd")
serving = importlib.import_module("qwen-30brust_amd.serving")

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    d = engine.Device(0)
    yield d
    d.close()


def gaps(dev, places, batch, q, kv):
    """A call of `batch` sequences, of which those at `places` have tokens and the others some keys and no tokens."""
    context, new = [40, 0, 7, 100, 3], [30, 5, 1, 9, 2]
    cache, table, lengths, first, query = make(8, context, new, 4, 2, 64, 16, q, kv)
    k, v = values(cache[0], cache[2]), values(cache[1], cache[3])
    want, bound = attend_many(query, k, v, table, lengths, first, 0.1, None, split_of(q, kv))
    wide = torch.zeros(batch, table.shape[1], dtype=torch.int32)
    long, count = torch.full((batch,), 16, dtype=torch.int32), torch.zeros(batch, dtype=torch.int32)
    wide[places], long[places], count[places] = table, torch.tensor(lengths, dtype=torch.int32), torch.tensor(new, dtype=torch.int32)
    begin = torch.cat([torch.zeros(1, dtype=torch.int32), count.cumsum(0).int()])
    c = serving.PagedCache(dev, *cache)
    args = (query.cuda(), wide.cuda(), long.cuda(), begin.cuda(), table.shape[1] * 16)
    return lambda: c.attend_prompts(*args, scale=0.1), want, bound


@pytest.mark.parametrize("q,kv", [("f32", "f32"), ("bf16", "bf16"), ("bf16", "q8_0")])
@pytest.mark.parametrize("places,batch", [([0, 1, 2, 3, 4], 5), ([0, 255, 256, 257, 1030], 1040), ([3, 258, 259, 9000, 65534], 65535),
                                          ([65530, 65531, 65532, 65533, 65534], 65535)])
def test_sequences_without_tokens(dev, q, kv, places, batch):
    call, want, bound = gaps(dev, places, batch, q, kv)
    close(call(), want, bound)


def test_sequences_without_tokens_take_no_turns(dev):
    """Sequences far apart are found by all threads together: the same call, with the others behind, takes about as long."""
    def took(call):
        best = 1e9
        for _ in range(5):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            call()
            b.record()
            b.synchronize()
            best = min(best, a.elapsed_time(b))
        return best

    batch = 65535
    apart = gaps(dev, [0, 20000, 40000, 60000, 65534], batch, "bf16", "bf16")[0]
    beside = gaps(dev, [65530, 65531, 65532, 65533, 65534], batch, "bf16", "bf16")[0]
    assert took(apart) < 5 * took(beside)


def test_acceptance_without_sequences(dev):
    """No sequences, and rows of none: no node is accepted."""
    g = torch.Generator().manual_seed(1)
    cache = serving.PagedCache(dev, *make_cache(g, 4, 16, 2, 64, "f32"))
    x = ints([-1, 0, 0, 1, 2])
    held = torch.full((20,), 77, dtype=torch.int32, device="cuda")  # memory that the outputs may get
    del held
    new, accepted, path, following = serving.accept([cache], x, x, x, torch.zeros(0, 2, dtype=torch.int32, device="cuda"),
                                                    ints([]), ints([0]))
    assert new.shape == accepted.shape == following.shape == (0,) and path.tolist() == [-1] * 5
