"""Log probabilities, entropy and top alternatives of rows of logits (serving.logprobs over
qh_logprobs, Model.logprobs over qh_last_logprobs) against plain 64-bit restatements."""
import importlib
import math

import numpy as np
import pytest
import torch

from serving_reference import TYPES

engine = importlib.import_module("qwen-30brust_amd")
serving = importlib.import_module("qwen-30brust_amd.serving")
synth = importlib.import_module("qwen-30brust_amd.synth")

pytestmark = pytest.mark.gpu
MIN = torch.finfo(torch.float32).min


@pytest.fixture(scope="module")
def dev():
    d = engine.Device(0)
    yield d
    d.close()


def order(x):
    b = x.contiguous().view(torch.int32).long()
    return torch.where(b < 0, -b - 1 - (1 << 31), b)


def exact(x, targets, top, valid):
    """x: f32 on the CPU."""
    if valid is not None:
        x = torch.where(valid.bool(), x, torch.full_like(x, MIN))
    y = x.double()
    m = y.amax(-1, keepdim=True)
    e = torch.where(y == -math.inf, torch.zeros_like(y), (y - m).exp())
    s = e.sum(-1, keepdim=True)
    bad = (y.isnan() | (y == math.inf)).any(-1)
    none = (y == -math.inf).all(-1)
    h = s.log()[:, 0] - torch.where(e > 0, (y - m) * e, torch.zeros_like(y)).sum(-1) / s[:, 0]
    h[none], h[bad] = 0, math.nan

    def logp(v):
        r = torch.where(v == -math.inf, v, (v - m) - s.log())  # m may be f32::MIN
        r[bad] = math.nan
        return r

    lp = None
    if targets is not None:
        inside = (targets >= 0) & (targets < x.shape[1])
        lp = logp(y.gather(1, targets.long().clamp(0, x.shape[1] - 1)[:, None]))[:, 0]
        lp[~inside] = math.nan
    if not top:
        return lp, h, None, None
    rank = (order(x) << 25) - torch.arange(x.shape[1])
    ids = rank.sort(-1, descending=True).indices[:, :top]
    return lp, h, ids.int(), logp(y.gather(1, ids))


def check(got, want, x, vocab):
    """32-bit arithmetic: exponentials off by 2 + |x - m| half steps each, sums of 32-bit partial sums
    by at most vocab / 1024 + 64 of them; a log probability then by that and two half steps of its
    terms, the entropy by that times its size and the largest |x - m| that has weight (90)."""
    rel = (2 + 90 + vocab / 1024 + 64) * 2.0 ** -24
    size = x.float().nan_to_num(0, 0, 0).clamp(-1e4, 1e4).abs().amax(-1).double() + 20

    def near(a, b, tol):
        a = a.cpu().double()
        assert torch.equal(a.isnan(), b.isnan())
        fine = torch.isfinite(b)
        assert torch.equal(a[~fine & ~b.isnan()], b[~fine & ~b.isnan()])
        off, lim = (a - b).abs(), (tol + 2.0 ** -22 * b.abs())
        assert (off <= lim)[fine].all(), (off / lim)[fine].max()

    tol = rel + 4 * 2.0 ** -24 * size
    if want[0] is not None:
        near(got[0], want[0], tol)
    near(got[1], want[1], rel * (1 + want[1].nan_to_num(0).abs() + 20) + 4 * 2.0 ** -24 * size)
    if want[2] is not None:
        assert torch.equal(got[2].cpu(), want[2])
        near(got[3], want[3], tol[:, None])
    else:
        assert got[2] is None and got[3] is None


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,vocab,top", [(1, 1, 1), (3, 2, 2), (1, 63, 5), (2, 64, 64), (5, 65, 20), (4, 1000, 0),
                                            (2, 4096, 128), (7, 4097, 1), (3, 50257, 20), (1, 151936, 20),
                                            (2, 151936, 128), (9, 151936, 5), (300, 1031, 7), (1, 262147, 33)])
@pytest.mark.parametrize("mask", [False, True])
def test_logprobs(dev, kind, rows, vocab, top, mask):
    g = torch.Generator().manual_seed(vocab + rows)
    x = (3 * torch.randn(rows, vocab, generator=g)).to(TYPES[kind])
    targets = torch.randint(0, vocab, (rows,), generator=g).int()
    valid = (torch.rand(vocab, generator=g) < 0.9).to(torch.uint8) if mask else None
    if mask:
        valid[targets.long()] = 1
    want = exact(x.float(), targets, top, valid)
    got = serving.logprobs(dev, x.cuda(), targets.cuda(), top=top, valid=None if valid is None else valid.cuda())
    check(got, want, x, vocab)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("vocab", [500, 30011, 151936])
def test_patterns(dev, kind, vocab):
    """Rows that rise, fall, are all alike, hold few values, one spike, only -inf, only masked ids,
    and rows with infinities and NaN among them; targets outside the vocabulary."""
    g = torch.Generator().manual_seed(vocab)
    t = torch.arange(vocab).float()
    rows = [t / vocab, -t / vocab, torch.zeros(vocab), torch.randint(0, 3, (vocab,), generator=g).float(),
            torch.where(t == 77, 60.0, 0.0), torch.full((vocab,), -math.inf),
            torch.where(t % 3 == 0, -math.inf, torch.randn(vocab, generator=g)),
            torch.where(t == 5, math.inf, 0.0), torch.where(t == 9, math.nan, torch.randn(vocab, generator=g)),
            torch.where(t == 9, -math.nan, 1.0), torch.full((vocab,), 6e4), torch.full((vocab,), -6e4),
            torch.where(t < 3, -math.inf, torch.where(t == 300, 0.0, -math.inf)), torch.where(t % 2 == 0, 0.0, -0.0),
            50 * torch.randn(vocab, generator=g)]
    x = torch.stack(rows).to(TYPES[kind])
    n = len(rows)
    targets = torch.randint(0, vocab, (n,), generator=g).int()
    targets[1], targets[2], targets[12] = vocab, -1, 300
    valid = torch.ones(vocab, dtype=torch.uint8)
    valid[torch.randint(0, vocab, (vocab // 5,), generator=g)] = 0
    for v in (None, valid, torch.zeros(vocab, dtype=torch.uint8)):
        for top in (0, 1, 20, 128):
            if v is not None:  # a masked target's f32::MIN is its log probability
                inside = (targets >= 0) & (targets < vocab)
                assert inside.sum() == n - 2
            want = exact(x.float(), targets, top, v)
            got = serving.logprobs(dev, x.cuda(), targets.cuda(), top=top, valid=None if v is None else v.cuda())
            check(got, want, x, vocab)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("vocab", [7, 1000, 151936])
def test_ends_of_the_range(dev, kind, vocab):
    """Rows whose maximum lies near either end of the type, with ties there, one batch of such logits
    among ordinary ones, ordinary ones with the lowest value among them; a log probability past the
    type's range is -inf."""
    g = torch.Generator().manual_seed(vocab)
    t, big = torch.arange(vocab), torch.finfo(TYPES[kind]).max
    noise = torch.randn(vocab, generator=g)
    rows = [torch.where(t % 5 == 0, big, 0.9 * big), torch.where(t == vocab - 1, big, -big), torch.where(t % 3 == 0, -0.7 * big, -big),
            torch.full((vocab,), -big), torch.where(t == vocab // 2, 0.99 * big, noise), torch.where(t < 3, -big, noise),
            torch.where(t < 1100, -big, noise), torch.where(t >= 5, -math.inf, -0.8 * big),
            torch.where(t == 4, 1.9e38, torch.where(t == 6, -1.9e38, 0.0)), torch.where(t == vocab - 1, 2.1e38, -2.1e38),
            # between: past 2^24 half a step of the maximum is more than 1
            torch.where(t % 7 == 0, 1.01e9, noise), 1e4 * noise + 3e7, 1e4 * noise - 3e7, 1e3 * noise + 2 ** 24, 1e3 * noise - 2 ** 24,
            1e6 * noise, 1e12 * noise, torch.where(t % 64 < 9, -1e10, noise), torch.where(t < 2000, -1e10, noise),
            torch.where(t == 3, math.nan, 1e12 * noise), torch.where(t == 2, math.nan, -1e12)]
    x = torch.stack([r.float() for r in rows]).to(TYPES[kind])
    targets = torch.randint(0, vocab, (len(rows),), generator=g).int()
    for v in (None, (torch.rand(vocab, generator=g) < 0.9).to(torch.uint8)):
        for top in (0, min(vocab, 5), min(vocab, 100)):
            want = exact(x.float(), targets, top, v)
            want = [None if w is None else w if w.dtype == torch.int32 else w.float().double() for w in want]
            got = serving.logprobs(dev, x.cuda(), targets.cuda(), top=top, valid=None if v is None else v.cuda())
            check(got, want, x, vocab)


def test_views(dev):
    """Rows with a stride, at an odd element; without targets."""
    g = torch.Generator().manual_seed(1)
    for kind in TYPES:
        x = torch.randn(6, 2003, generator=g).to(TYPES[kind]).cuda()
        for lo, n in ((0, 2003), (1, 2000), (3, 1024)):
            y = x[::2, lo:lo + n]
            got = serving.logprobs(dev, y, top=9)
            assert got[0] is None
            check(got, exact(y.cpu().float(), None, 9, None), y.cpu(), n)


def test_stream_and_graph(dev):
    """On a side stream, and captured and replayed with new logits beside eager calls."""
    g = torch.Generator().manual_seed(1)
    x = torch.randn(3, 151936, generator=g).cuda()
    t = torch.tensor([5, 6, 7], dtype=torch.int32).cuda()
    eager = serving.logprobs(dev, x, t, top=20)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = serving.logprobs(dev, x, t, top=20)
    side.synchronize()
    for a, b in zip(got, eager):
        assert torch.equal(a, b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = serving.logprobs(dev, x, t, top=20)
    for _ in range(3):
        x.copy_(torch.randn(3, 151936, generator=g))
        graph.replay()
        torch.cuda.synchronize()
        replayed = [a.clone() for a in held]
        for a, b in zip(replayed, serving.logprobs(dev, x, t, top=20)):
            assert torch.equal(a, b)


def test_no_rows(dev):
    x = torch.zeros(0, 100, device="cuda")
    got = serving.logprobs(dev, x, torch.zeros(0, dtype=torch.int32, device="cuda"), top=3)
    assert [tuple(t.shape) for t in got] == [(0,), (0,), (0, 3), (0, 3)]


def test_last_step(dev):
    """Model.logprobs reads the last step's logits where they are, with the valid-token mask."""
    spec = synth.tiny_k()
    m = engine.Model(synth.build_image(spec, threads=4), spec.context, device=dev)
    with pytest.raises(engine.EngineError, match="run a token step first"):
        m.logprobs(1)
    for token in (7, 3):
        x = torch.from_numpy(m.forward(token))[None]
        vocab = x.shape[1]
        valid = np.ones(vocab, np.uint8)
        valid[5:vocab:3] = 0
        for v in (None, valid):
            m.set_valid_tokens(v)
            want = exact(x, torch.tensor([4]), 9, None if v is None else torch.from_numpy(v))
            lp, h, ids, alt = m.logprobs(4, 9)
            check((torch.tensor([lp]), torch.tensor([h]), torch.from_numpy(ids.astype(np.int32))[None],
                   torch.from_numpy(alt)[None]), want, x, vocab)
        assert ids[0] == int(np.argmax(np.where(valid, x[0].numpy(), MIN)))
        lp, h2, ids, alt = m.logprobs()
        assert lp is None and h2 == h and ids.size == 0 and alt.size == 0
        m.set_valid_tokens(None)
    with pytest.raises(engine.EngineError, match="token outside vocabulary"):
        m.logprobs(vocab)
    with pytest.raises(engine.EngineError, match="alternatives"):
        m.logprobs(1, 129)
