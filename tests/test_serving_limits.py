"""The serving operators' refusals at the ends of their ranges, and of tensors that want a gradient (on
the CPU: nothing is launched)."""
import importlib

import pytest
import torch

from test_serving import A, cache, evict, message, seqs

engine = importlib.import_module("qwen-30brust_amd")
serving = importlib.import_module("qwen-30brust_amd.serving")


def test_keys_to_move():
    """No more than a launch moves."""
    long = seqs(most=(1 << 30) + 5, table_pages=1 << 27)
    assert "keys to keep out of range" in message(evict(s=long, keep=(1 << 30) - 1, to_pages=1 << 26))
    assert "keys to keep out of range" in message(evict(s=long, keep=(1 << 30) - 63, to_pages=1 << 26))
    assert message(evict(s=long, keep=(1 << 30) - 64, to_pages=1 << 26)) == "null context"
    assert message(evict(keep=(1 << 30) - 1, to_pages=1 << 26)) == "null context"  # no sequence is that long
