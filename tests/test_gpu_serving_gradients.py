"""Every tensor argument of the serving operators that requires a gradient is refused while gradients are
recorded, and taken under no_grad with the same results."""
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


def test_arguments(dev):
    g = torch.Generator(device="cuda").manual_seed(1)

    def randn(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    cache = serving.PagedCache(dev, randn(6, 16, 2, 64), randn(6, 16, 2, 64))
    table = torch.arange(4, dtype=torch.int32, device="cuda").reshape(2, 2)
    to, n = torch.tensor([[4], [5]], dtype=torch.int32, device="cuda"), torch.tensor([20, 9], dtype=torch.int32, device="cuda")

    def append(k, v, q, q_norm, k_norm, rope):
        return cache.append(k, v, table, n, q=q, q_norm=q_norm, k_norm=k_norm, rope=rope)

    def attend(q, weights):
        out, w = cache.attend(q, table, n, 32, weights=weights, weights_out=torch.empty(2, 2, 32, device="cuda"))
        return out, w[0, :, :20], w[1, :, :9]

    def evict(weights):
        return cache.evict(weights, table, n, 8, to, first=1, recent=2)[:2]

    def logprobs(x):
        return serving.logprobs(dev, x, torch.tensor([3, 4], dtype=torch.int32, device="cuda"), top=2)

    for call, args in ((append, (randn(2, 2, 64), randn(2, 2, 64), randn(2, 4, 64), randn(64), randn(64), randn(40, 32, 2))),
                       (attend, (randn(2, 4, 64), randn(2, 2, 32))), (evict, (randn(2, 2, 32).abs(),)), (logprobs, (randn(2, 70),))):
        want = call(*args)
        want = [t.clone() for t in (want if isinstance(want, tuple) else (want,))]
        for i in range(len(args)):
            mine = [a.clone().requires_grad_(i == j) for j, a in enumerate(args)]
            with pytest.raises(engine.EngineError, match="no gradient is recorded here"):
                call(*mine)
            with torch.no_grad():
                got = call(*mine)
            for a, b in zip(got if isinstance(got, tuple) else (got,), want):
                assert torch.equal(a, b) and not a.requires_grad
