"""Outputs whose elements share memory (expanded tensors) are refused; inputs that do are read."""
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


def test_expanded(dev):
    k, v = (torch.randn(6, 16, 2, 64, device="cuda") for _ in range(2))
    cache = serving.PagedCache(dev, k, v)
    table = torch.arange(4, dtype=torch.int32, device="cuda").reshape(2, 2)
    to, n = torch.tensor([[4], [5]], dtype=torch.int32, device="cuda"), torch.tensor([20, 9], dtype=torch.int32, device="cuda")
    q, new = torch.randn(2, 4, 64, device="cuda"), torch.randn(2, 2, 64, device="cuda")
    shared = torch.empty(1, 4, 64, device="cuda").expand(2, 4, 64)
    heavy = torch.rand(1, 2, 32, device="cuda").expand(2, 2, 32)
    with pytest.raises(engine.EngineError, match="attention outputs: elements of an output share memory"):
        cache.attend(q, table, n, out=shared)
    with pytest.raises(engine.EngineError, match="query outputs: elements of an output share memory"):
        cache.append(new, new, table, n, q=q, q_out=shared)
    with pytest.raises(engine.EngineError, match="weight outputs: elements of an output share memory"):
        cache.attend(q, table, n, 32, weights=heavy)
    one = serving.PagedCache(dev, k[:1].expand(6, 16, 2, 64), v[:1].expand(6, 16, 2, 64))
    with pytest.raises(engine.EngineError, match="read only"):
        one.append(new, new, table, n)
    with pytest.raises(engine.EngineError, match="read only"):
        one.evict(heavy, table, n, 8, to)
    # as inputs they are ordinary tensors
    assert torch.equal(cache.attend(q[:1].expand(2, 4, 64), table, n), cache.attend(q[:1].repeat(2, 1, 1), table, n))
    same = serving.PagedCache(dev, k[:1].repeat(6, 1, 1, 1), v[:1].repeat(6, 1, 1, 1))
    assert torch.equal(one.attend(q, table, n), same.attend(q, table, n))
    after = [torch.zeros(2, 2, 32, device="cuda") for _ in range(2)]
    cache.attend(q, table, n, 32, weights=heavy, weights_out=after[0])
    cache.attend(q, table, n, 32, weights=heavy.clone(), weights_out=after[1])
    assert torch.equal(after[0], after[1])
