"""Log probabilities of rows whose maximum lies at or just above -2^24, where the sums' unit changes:
logits of both sides have weight, whichever lanes, batches and waves hold them."""
import importlib
import math

import pytest
import torch

from test_gpu_logprobs import exact

engine = importlib.import_module("qwen-30brust_amd")
serving = importlib.import_module("qwen-30brust_amd.serving")

pytestmark = pytest.mark.gpu
EDGE = -2.0 ** 24


@pytest.fixture(scope="module")
def dev():
    d = engine.Device(0)
    yield d
    d.close()


def rows_of(vocab, g):
    t = torch.arange(vocab)

    def steps(n):  # whole numbers, two apart below the edge
        return torch.randint(0, n, (vocab,), generator=g).double()

    low, high = EDGE - 2 - 2 * steps(8), EDGE + steps(4)
    return torch.stack([
        torch.where(t == 0, EDGE + 1, torch.full((vocab,), EDGE - 2, dtype=torch.float64)),
        torch.where(t == vocab - 1, EDGE + 1, low),
        torch.where(t % 97 == 5, high, low),
        torch.where(t < vocab // 2, low, high),
        torch.where(t < vocab // 2, high, low),
        torch.where(t % 64 < 3, high, EDGE - 2 - 3 * 2 * steps(4)),
        torch.where(t == vocab // 3, EDGE, torch.full((vocab,), EDGE - 4, dtype=torch.float64)),
        torch.where(t == vocab // 3, EDGE - 2, torch.full((vocab,), EDGE - 4, dtype=torch.float64)),
        torch.where(t == vocab // 3, EDGE + 30, low),
        torch.where(t == vocab // 3, EDGE + 300, low),
        EDGE + 200 + steps(9),
        torch.where(t % 5 == 0, -math.inf, torch.where(t % 31 == 1, high, low)),
    ]).float()


@pytest.mark.parametrize("vocab", [40, 1024, 2049, 5000, 151936])
def test_around_the_edge(dev, vocab):
    """Every difference of two logits is exact in 32 bits.  A term: a difference times log2(e) (|t| half
    steps, up to 60 where it has weight) and two for the exponential; a sum's parts vocab / 64 in order
    and 64 folded; the logarithm and its product two of a result of up to 400."""
    g = torch.Generator().manual_seed(vocab)
    x = rows_of(vocab, g)
    targets = torch.randint(0, vocab, (len(x),), generator=g).int()
    targets[0], targets[1] = 0, vocab - 1
    masks = [None, (torch.rand(vocab, generator=g) < 0.8).to(torch.uint8)]
    masks[1][targets.long()] = 1
    rel = (2 * 60 + 2 + vocab / 64 + 64) * 2.0 ** -24
    for valid in masks:
        for top in (0, 5, 40):
            want = exact(x, targets, top, valid)
            got = serving.logprobs(dev, x.cuda(), targets.cuda(), top=top, valid=None if valid is None else valid.cuda())
            for a, b in zip(got, want):
                if b is None:
                    assert a is None
                elif b.dtype == torch.int32:
                    assert torch.equal(a.cpu(), b)
                else:
                    a = a.cpu().double()
                    fine = b.abs() < 1e30  # a masked id's f32::MIN is its own log probability
                    assert (a < -1e30)[~fine].all()
                    off, tol = (a - b).abs(), rel * (21 + b.abs()) + 4 * 2.0 ** -24 * b.abs()
                    assert (off <= tol)[fine].all(), (off / tol)[fine].max()


def test_several_rows_a_wave_and_waves_a_row(dev):
    """The same rows among ordinary ones, where a wave holds several rows."""
    g = torch.Generator().manual_seed(3)
    x = torch.randn(9000, 70, generator=g)
    x[::7] = rows_of(70, g)[2]
    want = exact(x, None, 3, None)
    got = serving.logprobs(dev, x.cuda(), top=3)
    assert torch.equal(got[2].cpu(), want[2])
    tol = (2 * 60 + 2 + 70 + 64) * 2.0 ** -24
    assert ((got[1].cpu().double() - want[1]).abs() <= 30 * tol).all()
    assert ((got[3].cpu().double() - want[3]).abs() <= 30 * tol).all()
