"""The serving operators' refusals at the ends of their ranges, and of tensors that want a gradient (on
the CPU: nothing is launched)."""
import importlib

import pytest
import torch

from test_serving import evict, message, seqs

engine = importlib.import_module("qwen-30brust_amd")
serving = importlib.import_module("qwen-30brust_amd.serving")


def test_keys_to_move():
    """No more than a launch moves."""
    long = seqs(most=(1 << 30) + 5, table_pages=1 << 27)
    assert "keys to keep out of range" in message(evict(s=long, keep=(1 << 30) - 1, to_pages=1 << 26))
    assert "keys to keep out of range" in message(evict(s=long, keep=(1 << 30) - 63, to_pages=1 << 26))
    assert message(evict(s=long, keep=(1 << 30) - 64, to_pages=1 << 26)) == "null context"
    assert message(evict(keep=(1 << 30) - 1, to_pages=1 << 26)) == "null context"  # no sequence is that long


class Closed:
    index, h = 0, None


def test_tensors_that_want_a_gradient():
    """Refused by name while gradients are recorded; under no_grad the next check is reached."""
    k, plain = torch.zeros(4, 16, 2, 64, requires_grad=True), torch.zeros(4, 16, 2, 64)
    x = torch.zeros(2, 5, requires_grad=True)
    for call, what in ((lambda: serving.PagedCache(Closed, k, plain), "cache keys"),
                       (lambda: serving.logprobs(Closed, x), "logits"), (lambda: serving.logprobs(Closed, 2 * x), "logits")):
        with pytest.raises(engine.EngineError, match=f"{what}: no gradient is recorded here"):
            call()
        with torch.no_grad():
            with pytest.raises(engine.EngineError, match="not a tensor on the engine's device"):
                call()
    with torch.inference_mode():
        with pytest.raises(engine.EngineError, match="not a tensor on the engine's device"):
            serving.logprobs(Closed, x)
