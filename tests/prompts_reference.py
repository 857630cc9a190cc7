"""Plain 64-bit restatements of the operators for several new tokens per sequence (CPU, torch), and the inputs
that their tests share."""
import math

import torch

from serving_reference import HALF, TINY, TYPES, gathered, make_cache, make_table


def make(seed, context, new, heads, kvheads, dim, page, q, kv, head_major=False, front=0, behind=0):
    """(cache tensors, table, lengths, first, query [front + all new + behind][heads][dim]), on the CPU but the
    cache; the first `front` and last `behind` rows are no sequence's."""
    g = torch.Generator().manual_seed(seed)
    lengths = [c + n for c, n in zip(context, new)]
    table, pool, _ = make_table(g, lengths, page)
    cache = make_cache(g, pool, page, kvheads, dim, kv, head_major)
    first = [front]
    for n in new:
        first.append(first[-1] + n)
    query = (2 * torch.randn(first[-1] + behind, heads, dim, generator=g)).to(TYPES[q])
    return cache, table, lengths, first, query


def trees(g, new, wide=4):
    """(parents, ancestors) of random trees, packed: numbers within a sequence, and 64 bits."""
    parents, bits = [], []
    for n in new:
        own = []
        for j in range(n):
            p = -1 if j == 0 else max(0, j - 1 - int(torch.randint(0, wide, (1,), generator=g)))
            parents.append(p)
            own.append(1 << j | (own[p] if p >= 0 else 0))
        bits += own
    return parents, bits


def signed(bits):
    return torch.tensor([b - (1 << 64) if b >> 63 else b for b in bits], dtype=torch.int64)


def split_of(q, kv):
    """A softmax weight that enters a product of 16 bits is rounded once, to the type of queries and cache; bf16 queries
    over Q8_0 take f16 products, where the values (code times scale), too, are rounded to f16."""
    if (q, kv) == ("bf16", "q8_0"):
        return HALF[torch.float16]
    return HALF[TYPES[q]] if q == kv and q != "f32" else 0.0


def attend_many(q, k, v, table, lengths, first, scale, bits=None, split=0.0):
    """(out like q in 64 bits, its rows of no sequence 0; a bound of the error before the last rounding). k and v:
    values of the cache's slots. bits: each row's visible nodes, None: causal. A key that a row does not see takes no
    part, whatever it holds."""
    heads, d = q.shape[1:]
    out, bound = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64)
    G = heads // k.shape[2]
    q8 = split == HALF[torch.float16] and q.dtype == torch.bfloat16
    for b, n in enumerate(lengths):
        m = first[b + 1] - first[b]
        if not m:
            continue
        kk, vv = gathered(k, table, b, n), gathered(v, table, b, n)
        t = torch.arange(n)
        if bits is None:
            sees = t <= n - m + torch.arange(m)[:, None]
        else:
            own = torch.tensor([[bits[first[b] + i] >> j & 1 for j in range(m)] for i in range(m)], dtype=torch.bool)
            sees = torch.cat([torch.ones(m, n - m, dtype=torch.bool), own], 1)
        qq = q[first[b]:first[b + 1]].double().reshape(m, -1, G, d).permute(1, 2, 0, 3)  # [kvheads][G][m][d]
        s = scale * (qq @ kk[:, None].transpose(2, 3))
        s = s.masked_fill(~sees, -math.inf)
        top = s.amax(-1, keepdim=True)
        e = torch.where(top == -math.inf, torch.zeros_like(s), (s - top).exp())
        total = e.sum(-1, keepdim=True)
        p = torch.where(total == 0, torch.zeros_like(e), e / total)
        # products of keys that a row does not see are left out, not 0 times what they hold
        fine = torch.isfinite(vv)
        o = p @ torch.where(fine, vv, 0.0)[:, None]
        if not fine.all():
            for h, j in (~fine).any(-1).nonzero().tolist():
                add = p[h, :, :, j, None] * vv[h, j]
                o[h] = torch.where(sees[:, j, None], o[h] - p[h, :, :, j, None] * torch.where(fine[h, j], vv[h, j], 0.0) + add, o[h])
        rows = slice(first[b], first[b + 1])
        out[rows] = o.permute(2, 0, 1, 3).reshape(m, heads, d)
        # 32-bit arithmetic: a score is off by at most (d + 3) half steps of sum |q k| scale, its exponential by that
        # and four of |s - top| (the product with log2 e, the difference), twice (numerator and sum); the sums of n
        # terms by n + 8 half steps; rescalings and the join by 64 more. A weight rounded to 16 bits: `split`, in the
        # numerator and in the sum; in f16 weights below 2^-14 times 2^-7 of the running maximum are rounded to
        # steps of 2^-24 times 2^-7, half of that each
        finite = torch.where(fine, vv, 0.0)
        size = scale * (qq.abs() @ kk.abs()[:, None].transpose(2, 3)).masked_fill(~sees, 0).nan_to_num(0, 0, 0).amax(-1, keepdim=True)
        low = torch.where(s == -math.inf, torch.zeros_like(s), (s - top).abs()).nan_to_num(0, 0, 0).amax(-1, keepdim=True)
        rel = (2 * ((d + 3) * size + 4 * low) + 2 * (n + 8) + 64) * 2.0 ** -24 + 2 * split
        near = rel * (p @ finite.abs()[:, None])
        if q8:
            # values as f16, half a step of 2^-11 or 2^-25; a query's elements below 2^-39 of its largest, in every score
            lost = scale * 2.0 ** -39 * qq.abs().amax(-1, keepdim=True) * kk.abs().sum(-1).amax()
            near = near + split * (p @ finite.abs()[:, None]) + 2.0 ** -25 + 2 * lost * finite.abs().amax()
        if split == HALF[torch.float16]:
            near = near + 2 * n * 2.0 ** -32 * finite.abs().amax()
        bound[rows] = near.permute(2, 0, 1, 3).reshape(m, heads, d)
    return out, bound


def close(got, want, bound):
    """Every value within `bound` of `want` and one rounding to its type."""
    g = got.cpu().double()
    fine = torch.isfinite(want)
    assert torch.equal(torch.isnan(g), torch.isnan(want))
    assert torch.equal(g[~fine & ~want.isnan()], want[~fine & ~want.isnan()])
    tol = bound + HALF[got.dtype] * (want.abs() + bound) + TINY[got.dtype]
    off = (g - want).abs()
    assert (off <= tol)[fine].all(), ((off / tol)[fine].max(), (off > tol).nonzero()[:5])
