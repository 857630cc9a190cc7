"""Plain 64-bit restatements of the serving operators (CPU, torch), and the
inputs that their tests share."""
import math

import torch

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
HALF = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}  # half a step, relative
TINY = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -133}


def quantise(x):
    """(codes, scales) of Q8_0: blocks of 32, scale = f16(max |x| / 127)."""
    b = x.float().unflatten(-1, (-1, 32))
    d = (b.abs().amax(-1, keepdim=True) / 127).half()
    f = d.float()
    codes = torch.where(f > 0, (b / f).round().clamp(-127, 127), torch.zeros_like(b)).to(torch.int8)
    return codes.flatten(-2), d[..., 0]


def values(k, scale):
    """A cache tensor's values in 64 bits (CPU)."""
    k = k.cpu()
    if scale is None:
        return k.double()
    return (k.unflatten(-1, (-1, 32)).double() * scale.cpu().double()[..., None]).flatten(-2)


def make_cache(g, pages, page, kvheads, dim, kind, head_major=False):
    """(k, v, k_scale, v_scale) on the GPU: a pool of pages of normal values; head_major: tensors
    whose memory is [pages][kvheads][page][dim]."""
    out, scales = [], []
    for _ in range(2):
        x = torch.randn(pages, page, kvheads, dim, generator=g)
        x, s = quantise(x) if kind == "q8_0" else (x.to(TYPES[kind]), None)

        def laid(t):
            return t.cuda() if not head_major else t.transpose(1, 2).contiguous().cuda().transpose(1, 2)

        out.append(laid(x))
        scales.append(None if s is None else laid(s))
    return (*out, *scales)


def make_table(g, lengths, page, spare=2):
    """(table, number of pages): every sequence's pages, scattered over a pool; entries that no key
    needs are out of range."""
    need = [-(-t // page) for t in lengths]
    pool = sum(need) + spare
    order = torch.randperm(pool, generator=g).int()
    table = torch.full((len(lengths), max(max(need), 1)), -7, dtype=torch.int32)
    at = 0
    for b, m in enumerate(need):
        table[b, :m] = order[at:at + m]
        at += m
    return table, pool, order[at:]


def gathered(x, table, b, n):
    """[kvheads][n][dim] of sequence b."""
    t = torch.arange(n)
    page = x.shape[1]
    return x[table[b].long()[t // page], t % page].transpose(0, 1)


def attend(q, k, v, table, lengths, scale):
    """(out, weights per sequence, bound of the error per unit of half steps) in 64 bits; k and v
    from values()."""
    heads, d = q.shape[1:]
    outs, weights, bounds = [], [], []
    for b, n in enumerate(lengths):
        G = heads // k.shape[2]
        if n == 0:
            outs.append(torch.zeros(heads, d, dtype=torch.float64))
            bounds.append(torch.zeros(heads, d, dtype=torch.float64))
            weights.append(torch.zeros(k.shape[2], 0, dtype=torch.float64))
            continue
        kk, vv = gathered(k, table, b, n), gathered(v, table, b, n)
        qq = q[b].cpu().double().reshape(-1, G, d)
        s = scale * (qq[:, :, None, :] * kk[:, None]).sum(-1)
        m = s.amax(-1, keepdim=True)
        e = torch.where(m == -math.inf, torch.zeros_like(s), (s - m).exp())
        total = e.sum(-1, keepdim=True)
        p = torch.where(total == 0, torch.zeros_like(e), e / total)
        terms = p[..., None] * vv[:, None]
        if torch.isfinite(vv).all() and torch.isfinite(s).all():
            outs.append(terms.sum(2).reshape(heads, d))
            # 32-bit arithmetic: a score is off by at most (d + 3) half steps of sum |q k| scale, its
            # exponential by that and two steps of |s - m| more, twice (numerator and sum); the sums
            # of n terms by n + 8 half steps; rescalings and the join by 64 more
            size = scale * (qq.abs()[:, :, None, :] * kk.abs()[:, None]).sum(-1).amax(-1)
            ds = (d + 3) * size + 4 * (s - m).abs().amax(-1)
            rel = 2 * ds + 2 * (n + 8) + 64
            bounds.append((rel[..., None] * terms.abs().sum(2)).reshape(heads, d) * 2.0 ** -24)
        else:
            outs.append((p @ vv).reshape(heads, d))
            bounds.append(torch.zeros(heads, d, dtype=torch.float64))
        weights.append(p.sum(1))
    return torch.stack(outs), weights, torch.stack(bounds)
