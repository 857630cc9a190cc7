"""An append of more tokens and heads than one launch holds (2^32 threads)."""
import importlib

import pytest
import torch

engine = importlib.import_module("qwen-30brust_amd")
serving = importlib.import_module("qwen-30brust_amd.serving")

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    d = engine.Device(0)
    yield d
    d.close()


@pytest.mark.parametrize("kvheads,dim", [(8, 256), (3, 2)])
def test_many_tokens(dev, kvheads, dim):
    """2^24 tokens whose rows overlap in memory (every token's is four elements behind the one before
    it), into a sequence most of whose pages are out of range: the few pages that are in the cache, at
    both ends and all along, hold their own tokens."""
    n, page = 1 << 24, 16
    g = torch.Generator().manual_seed(dim)
    base = torch.randn(4 * n + kvheads * dim, generator=g).half().cuda()
    k_new, v_new = (x.as_strided((n, kvheads, dim), (4, dim, 1), at) for x, at in ((base, 0), (base, 4)))
    held = sorted(t // page for t in (0, n // 7, n // 4, n // 2 - 1, n // 2, n // 3 * 2, n - 40, n - 1))
    k = torch.zeros(len(held) + 1, page, kvheads, dim, dtype=torch.float16, device="cuda")
    v = torch.zeros_like(k)
    table = torch.full((1, n // page), -1, dtype=torch.int32)
    table[0, held] = torch.arange(len(held), dtype=torch.int32)
    serving.PagedCache(dev, k, v).append(k_new, v_new, table.cuda(), torch.tensor([n], dtype=torch.int32).cuda(),
                                         torch.tensor([0, n], dtype=torch.int32).cuda())
    for i, p in enumerate(held):
        at = p * page
        assert torch.equal(k[i], k_new[at:at + page]) and torch.equal(v[i], v_new[at:at + page])
    assert (k[len(held):] == 0).all() and (v[len(held):] == 0).all()
