"""Inputs in device memory that another stream writes while calls read them: results may be wrong, but
nothing outside the outputs and the workspace is written, and later calls are right."""
import ctypes as C
import importlib

import pytest
import torch

from serving_reference import attend, make_cache, make_table, values

engine = importlib.import_module("qwen-30brust_amd")
serving = importlib.import_module("qwen-30brust_amd.serving")

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    d = engine.Device(0)
    yield d
    d.close()


class Guarded:
    """A tensor in the middle of a larger one whose other values must stay."""

    def __init__(self, shape, dtype):
        n = 1
        for s in shape:
            n *= s
        self.all = torch.full((n + 2048,), 77, dtype=dtype, device="cuda")
        self.t = self.all[1024:1024 + n].view(shape)

    def whole(self):
        return bool((self.all[:1024] == 77).all() and (self.all[-1024:] == 77).all())


@pytest.mark.parametrize("kv,dim", [("bf16", 128), ("f32", 64), ("f16", 96)])
def test_lengths_pages_and_weights_that_change(dev, kv, dim):
    g = torch.Generator().manual_seed(dim)
    longest, page, G, H, keep = [5000, 4100, 300, 2500], 16, 2, 8, 400
    most, B = 5008, 4
    table, pool, spare = make_table(g, longest, page, spare=B * keep // page + 5)
    to = spare[:B * keep // page].reshape(B, -1)
    cache = make_cache(g, pool, page, G, dim, kv)
    c = serving.PagedCache(dev, *cache)
    k0 = cache[0].clone()
    q = torch.randn(B, H, dim, generator=g).to(cache[0].dtype).cuda()
    states = [(torch.tensor(n, dtype=torch.int32).cuda(), t.cuda()) for n, t in
              ((longest, table), ([17, 4100, 0, 900], table.clone().fill_(-1)), ([4999, 1, 300, -4], table),
               ([0, 0, 0, 0], table), ([most + 1, 40, 1, 2500], table.roll(1, 1)))]
    lengths, held, to = states[0][0].clone(), states[0][1].clone(), to.cuda()
    heavy = torch.rand(B, G, most, generator=g).cuda()
    other = torch.rand(B, G, most, generator=g).cuda()
    kept, kw, new = (Guarded(s, t) for s, t in (((B, G, keep), torch.int32), ((B, G, keep), torch.float32), ((B,), torch.int32)))
    out, after = Guarded((B, H, dim), q.dtype), Guarded((B, G, most), torch.float32)
    seqs = engine._Sequences(held.data_ptr(), lengths.data_ptr(), held.stride(0), held.shape[1], B, most)
    lib, need = engine.lib(), C.c_size_t()
    dev._check(lib.qh_paged_attention_bytes(dev.h, c._pages, seqs, H, 1, need))
    work = Guarded((need.value,), torch.uint8)
    assert work.t.data_ptr() % 16 == 0
    kinds = serving.KIND[q.dtype]
    heads = [engine._Heads(t.data_ptr(), kinds, H * dim, dim) for t in (q, out.t)]
    weights = engine._KeyWeights(heavy.data_ptr(), after.t.data_ptr(), G * most, most, G * most, most)
    side, main = torch.cuda.Stream(), torch.cuda.current_stream()
    torch.cuda.synchronize()

    def calls():
        s = serving._stream(dev)
        dev._check(lib.qh_paged_attention(dev.h, c._pages, seqs, heads[0], H, dim ** -0.5, heads[1], weights,
                                          work.t.data_ptr(), need.value, s))
        dev._check(lib.qh_paged_evict(dev.h, c._pages, seqs, heavy.data_ptr(), G * most, most, keep, 4, 50, to.data_ptr(),
                                      to.stride(0), to.shape[1], kept.t.data_ptr(), kw.t.data_ptr(), new.t.data_ptr(), s))

    for i in range(40):
        with torch.cuda.stream(side):
            for j in range(12):
                lengths.copy_(states[(i + j) % len(states)][0])
                held.copy_(states[(i + j) % len(states)][1])
                heavy.copy_(other if j % 2 else 1 - other)
        calls()
    torch.cuda.synchronize()
    assert all(x.whole() for x in (kept, kw, new, out, after, work))
    assert ((kept.t >= -1) & (kept.t < most)).all() and ((new.t >= 0) & (new.t <= keep)).all()
    moved = torch.zeros(pool, dtype=torch.bool)
    moved[to.cpu().flatten().long()] = True
    assert torch.equal(cache[0][(~moved).cuda()], k0[(~moved).cuda()])
    # and a call beside nothing
    lengths.copy_(states[0][0])
    held.copy_(states[0][1])
    calls()
    torch.cuda.synchronize()
    want, _, bound = attend(q, values(cache[0], None), values(cache[1], None), table, longest, dim ** -0.5)
    # the other calls' tests hold the exact bound; here a rounding of the output and the weights' two parts
    assert ((out.t.cpu().double() - want).abs() <= 2 * bound + 2.0 ** -8 * want.abs() + 2.0 ** -12).all()
    assert new.t.tolist() == [400, 400, 300, 400]
