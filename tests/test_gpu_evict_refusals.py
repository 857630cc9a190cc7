"""qh_paged_evict refuses outputs that lie on its inputs or on each other, before anything runs."""
import importlib

import pytest
import torch

engine = importlib.import_module("qwen-30brust_amd")

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    d = engine.Device(0)
    yield d
    d.close()


def test_outputs_apart(dev):
    B, G, page, dim, pool, most, keep = 3, 2, 16, 64, 30, 64, 32
    k, v = (torch.zeros(pool, page, G, dim, dtype=torch.float16, device="cuda") for _ in range(2))
    arena = torch.zeros(7, 4096, dtype=torch.int32, device="cuda")  # far apart

    def place(i, t):
        x = arena[i, :t.numel()].view(t.dtype).view(t.shape)
        x.copy_(t)
        return x

    table = place(0, torch.arange(B * 4, dtype=torch.int32).reshape(B, 4))
    to = place(1, (12 + torch.arange(B * 2, dtype=torch.int32)).reshape(B, 2))
    own = dict(lengths=place(2, torch.tensor([60, 5, 64], dtype=torch.int32)), weights=place(3, torch.rand(B, G, most)),
               kept=place(4, torch.zeros(B, G, keep, dtype=torch.int32)), kept_weights=place(5, torch.zeros(B, G, keep)),
               new=place(6, torch.zeros(B, dtype=torch.int32)))
    cache = engine._Pages(k.data_ptr(), v.data_ptr(), None, None, 1, page, G, dim, pool, page * G * dim, G * dim, dim)

    def call(**at):
        p = {name: t.data_ptr() for name, t in own.items()}
        p.update(at)
        seqs = engine._Sequences(table.data_ptr(), p["lengths"], 4, 4, B, most)
        dev._check(engine.lib().qh_paged_evict(dev.h, cache, seqs, p["weights"], G * most, most, keep, 2, 8, to.data_ptr(), 2, 2,
                                               p["kept"], p["kept_weights"], p["new"], None))

    def at(name, skip=0):
        return own[name].data_ptr() + skip

    torch.cuda.synchronize()  # the context's own stream runs the calls
    for kw, text in [(dict(new=at("lengths")), "new lengths overlap the lengths"),
                     (dict(new=at("lengths", 4)), "new lengths overlap the lengths"),
                     (dict(kept_weights=at("weights")), "kept weights overlap the weights"),
                     (dict(kept_weights=at("weights", B * G * (most - keep) * 4)), "kept weights overlap the weights"),
                     (dict(kept=table.data_ptr()), "kept indexes overlap the page table"),
                     (dict(new=to.data_ptr() + 8), "new lengths overlap the new pages"),
                     (dict(kept=at("kept_weights")), "kept indexes overlap the kept weights"),
                     (dict(new=at("kept", 12)), "kept indexes overlap the new lengths")]:
        with pytest.raises(engine.EngineError, match=text):
            call(**kw)
    # side by side they may lie
    both = torch.empty(2 * B * G * keep + 2 * B, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    n = B * G * keep * 4
    call(kept=both.data_ptr(), kept_weights=both.data_ptr() + n, new=both.data_ptr() + 2 * n)
    want = both.clone()
    call()
    assert torch.equal(want[:n // 4], own["kept"].flatten()) and want[2 * n // 4:][:B].tolist() == [32, 5, 32]
    assert torch.equal(want[n // 4:n // 2].view(torch.float32), own["kept_weights"].flatten())
