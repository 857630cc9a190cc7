"""Measured calls of the serving operators on device tensors: a paged key-value cache (append with
Q/K norm and RoPE, attention of one new token per sequence, eviction by accumulated attention
weight) and the log probabilities of an answer's tokens.

Each case names its `op`:
  append    new tokens' q, k and v: per-head RMSNorm and NeoX RoPE of q and k, k and v into pages
  attend    attention of one new token per sequence over its pages, and (where `weights`) each
            key's softmax weight, summed over the query heads of its KV head, added up
  evict     keeps the first, the last and the heaviest keys of every KV head, in new pages
  logprobs  log probabilities of given tokens, entropy and the top alternatives of rows of logits

With `own` false, run() computes them in elementary torch operations.
"""
import importlib
import math

import torch

own = False

VOCAB = 151936
FLOATS = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4.0, "f16": 2.0, "bf16": 2.0, "q8_0": 34 / 32}
EPS = 1e-6
THETA = 1e6


def listed():
    return [
        # one conversation's decode step in the engine's own types: latency counts
        {"name": "attend-one", "op": "attend", "batch": 1, "lo": 517, "hi": 517, "heads": 32, "kvheads": 4, "dim": 128,
         "page": 16, "q": "f32", "kv": "f32", "weights": False},
        # a serving batch of ragged histories that keeps the weights an eviction goes by
        {"name": "attend-ragged", "op": "attend", "batch": 48, "lo": 1, "hi": 4096, "heads": 32, "kvheads": 4,
         "dim": 128, "page": 16, "q": "bf16", "kv": "bf16", "weights": True},
        # two long documents
        {"name": "attend-long", "op": "attend", "batch": 2, "lo": 65537, "hi": 65537, "heads": 32, "kvheads": 4,
         "dim": 128, "page": 64, "q": "f16", "kv": "f16", "weights": False},
        # a larger batch on a cache held in 8 bits
        {"name": "attend-8bit", "op": "attend", "batch": 96, "lo": 33, "hi": 4096, "heads": 32, "kvheads": 4,
         "dim": 128, "page": 32, "q": "bf16", "kv": "q8_0", "weights": False},
        # the decode step of a batch: one token each
        {"name": "append-decode", "op": "append", "batch": 64, "each": 1, "lo": 1, "hi": 4096, "heads": 32,
         "kvheads": 4, "dim": 128, "page": 16, "x": "bf16", "kv": "bf16", "norm": True},
        # three prompts of one prefill
        {"name": "append-prompts", "op": "append", "batch": 3, "each": 667, "lo": 667, "hi": 2100, "heads": 32,
         "kvheads": 4, "dim": 128, "page": 64, "x": "f32", "kv": "f16", "norm": True},
        # keys and values that are ready, into a cache held in 8 bits
        {"name": "append-8bit", "op": "append", "batch": 2, "each": 512, "lo": 512, "hi": 900, "heads": 0,
         "kvheads": 4, "dim": 128, "page": 32, "x": "f32", "kv": "q8_0", "norm": False},
        # a batch brought back to a budget
        {"name": "evict-batch", "op": "evict", "batch": 16, "lo": 700, "hi": 4096, "keep": 1024, "first": 4,
         "recent": 256, "kvheads": 4, "dim": 128, "page": 16, "kv": "bf16"},
        # one long document
        {"name": "evict-long", "op": "evict", "batch": 1, "lo": 65537, "hi": 65537, "keep": 8192, "first": 4,
         "recent": 1024, "kvheads": 4, "dim": 128, "page": 64, "kv": "f16"},
        # the token just chosen, with the API's usual alternatives
        {"name": "logprobs-one", "op": "logprobs", "rows": 1, "vocab": VOCAB, "x": "f32", "top": 20, "mask": True},
        # a decode step of a batch
        {"name": "logprobs-batch", "op": "logprobs", "rows": 48, "vocab": VOCAB, "x": "bf16", "top": 5, "mask": False},
        # scoring a long answer
        {"name": "logprobs-score", "op": "logprobs", "rows": 777, "vocab": VOCAB, "x": "f32", "top": 20, "mask": True},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    op = rng.choice(["attend", "attend", "attend", "append", "append", "evict", "evict", "logprobs", "logprobs"])
    if op == "logprobs":
        vocab = rng.choice([VOCAB, _log_int(rng, 300, VOCAB)])
        rows = _log_int(rng, 1, 777)
        return {"op": op, "rows": rows, "vocab": vocab, "x": rng.choice(["f32", "f32", "bf16", "f16"]),
                "top": rng.choice([0, 1, 5, 20, rng.randint(2, 64)]), "mask": rng.random() < 0.5}
    kvheads, dim = rng.choice([1, 2, 4, 4, 8]), rng.choice([64, 128, 128, 128])
    heads, page = kvheads * rng.choice([1, 2, 4, 5, 8]), rng.choice([16, 16, 32, 64, 24, 128])
    c = {"op": op, "kvheads": kvheads, "dim": dim, "page": page}
    if op == "attend":
        q, kv = rng.choice([("f32", "f32"), ("f16", "f16"), ("bf16", "bf16"), ("bf16", "bf16"), ("bf16", "q8_0"),
                            ("f32", "q8_0"), ("f32", "f16")])
        hi = _log_int(rng, 16, 65537)
        batch = max(1, min(_log_int(rng, 1, 96), int(130e6 / (hi * kvheads * dim * BYTES[kv]))))
        c.update(batch=batch, lo=rng.randint(1, hi) if batch > 1 else hi, hi=hi, heads=heads, q=q, kv=kv,
                 weights=rng.random() < 0.4)
    elif op == "append":
        x, kv = rng.choice([("f32", "f32"), ("f32", "f16"), ("bf16", "bf16"), ("f16", "f16")])
        batch = _log_int(rng, 1, 64)
        each = rng.choice([1, max(1, _log_int(rng, 1, 2000) // batch)])
        c.update(batch=batch, each=each, lo=each, hi=each + rng.randint(0, 1500), heads=heads, x=x, kv=kv, norm=True)
    else:
        hi = _log_int(rng, 40, 65537)
        keep = _log_int(rng, 8, min(hi, 8192))
        first, recent = rng.randint(0, min(4, keep // 4)), rng.randint(0, keep // 2)
        kv = rng.choice(["f32", "bf16", "bf16", "f16"])
        batch = max(1, min(_log_int(rng, 1, 16), int(16e6 / (min(hi, keep) * kvheads * dim * BYTES[kv]))))
        c.update(batch=batch, lo=rng.randint(1, hi) if batch > 1 else hi, hi=hi, keep=keep, first=first, recent=recent,
                 kv=kv)
    return c


# ---------------------------------------------------------------- inputs --
_device = None


def _engine():
    """The program's one engine context."""
    global _device
    if _device is None:
        _device = importlib.import_module("qwen-30brust_amd").Device(0)
    return _device


def _serving():
    return importlib.import_module("qwen-30brust_amd.serving")


def _lengths(case):
    """The sequences' lengths, evenly from lo to hi (both reached)."""
    n = case["batch"]
    return [case["hi"] - (case["hi"] - case["lo"]) * i // max(1, n - 1) for i in range(n)]


def _quantised(x):
    """(codes, scales) of blocks of 32 values: scale = largest magnitude / 127 in 16 bits."""
    b = x.float().unflatten(-1, (-1, 32))
    d = (b.abs().amax(-1, keepdim=True) / 127).half()
    f = d.float()
    codes = torch.where(f > 0, (b / f).round().clamp(-127, 127), torch.zeros_like(b)).to(torch.int8)
    return codes.flatten(-2), d[..., 0]


def _values(codes, scales):
    return (codes.unflatten(-1, (-1, 32)).float() * scales.float()[..., None]).flatten(-2)


def _pages(case, g, lengths, extra=0):
    """(k, v, k_scale, v_scale, table): a pool of random pages in random order."""
    page, kv = case["page"], case["kv"]
    per = -(-max(lengths) // page)
    need = [-(-t // page) for t in lengths]
    pool = sum(need) + extra + 3
    shape = (pool, page, case["kvheads"], case["dim"])
    order = torch.randperm(pool, generator=g, device="cuda").int()
    table = torch.zeros(len(lengths), per, dtype=torch.int32)
    at = torch.zeros_like(table)
    done = 0
    for i, m in enumerate(need):
        at[i, :m] = torch.arange(done, done + m)
        done += m
    table = order[at.cuda().long()]
    held = []
    for _ in range(2):
        x = torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)
        held.append(_quantised(x) if kv == "q8_0" else (x.to(FLOATS[kv]), None))
    return held[0][0], held[1][0], held[0][1], held[1][1], table, order[done:]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def randn(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    state = dict(case)
    if case["op"] == "logprobs":
        n, vocab = case["rows"], case["vocab"]
        x = randn(n, vocab) * 2.5
        likely = torch.randint(0, vocab, (n, 8), generator=g, device="cuda")
        x.scatter_(1, likely, 8 + 4 * randn(n, 8).abs())
        state["logits"] = x.to(FLOATS[case["x"]])
        # ids past the tokenizer's are padding
        real = vocab - vocab // 570
        state["targets"] = torch.where(torch.rand(n, generator=g, device="cuda") < 0.7, likely[:, 0].clamp(max=real - 1),
                                       torch.randint(0, real, (n,), generator=g, device="cuda")).int()
        state["valid"] = (torch.arange(vocab, device="cuda") < real).to(torch.uint8) if case["mask"] else None
        if own:
            state["device"] = _engine()
        return state

    lengths = _lengths(case)
    order = torch.randperm(len(lengths), generator=g, device="cuda").tolist()
    lengths = [lengths[i] for i in order]
    new = -(-case["keep"] // case["page"]) if case["op"] == "evict" else 0
    k, v, ks, vs, table, spare = _pages(case, g, lengths, extra=new * len(lengths))
    state.update(k=k, v=v, k_scale=ks, v_scale=vs, table=table, most=max(lengths),
                 lengths=torch.tensor(lengths, dtype=torch.int32, device="cuda"))
    B, H, G, d = case["batch"], case.get("heads", 0), case["kvheads"], case["dim"]
    if case["op"] == "attend":
        state["query"] = (2 * randn(B, H, d)).to(FLOATS[case["q"]])
        state["before"] = randn(B, G, max(lengths)).exp() if case["weights"] else None
        state["after"] = torch.zeros(B, G, max(lengths), device="cuda") if case["weights"] else None
    elif case["op"] == "append":
        n, x = B * case["each"], FLOATS[case["x"]]
        # one projection's rows hold q, k and v
        qkv = randn(n, (H + 2 * G) * d).to(x)
        state["q_new"] = qkv[:, :H * d].unflatten(1, (H, d)) if H else None
        state["k_new"], state["v_new"] = (m.unflatten(1, (G, d)) for m in qkv[:, H * d:].chunk(2, 1))
        state["begin"] = torch.arange(0, n + 1, case["each"], device="cuda", dtype=torch.int32)
        state["q_weight"], state["k_weight"] = (1 + 0.2 * randn(d) for _ in range(2))
        # positions run on past what was evicted
        ahead = torch.randint(0, 2000, (B, 1), generator=g, device="cuda")
        slot = state["lengths"][:, None] - case["each"] + torch.arange(case["each"], device="cuda")
        state["positions"] = (slot + ahead).int().reshape(-1)
        angle = torch.arange(8192, device="cuda", dtype=torch.float64)[:, None] * THETA ** (
            -2 * torch.arange(d // 2, device="cuda", dtype=torch.float64) / d)
        state["rope"] = torch.stack([angle.cos(), angle.sin()], -1).float()
    else:
        # accumulated softmax weights: a heavy tail, and keys that no query looked at
        w = (2 * randn(B, G, max(lengths))).exp()
        state["heavy"] = torch.where(torch.rand(w.shape, generator=g, device="cuda") < 0.1, torch.zeros_like(w), w)
        state["to"] = spare[:new * B].reshape(B, new).contiguous()
    if own:
        state["cache"] = _serving().PagedCache(_engine(), k, v, ks, vs)
    return state


# ------------------------------------------------------------------ runs --
def run(state):
    return {"append": _append, "attend": _attend, "evict": _evict, "logprobs": _logprobs}[state["op"]](state)


def _gathered(state, which):
    """The sequences' rows [batch][kvheads][max length][dim] in 32 bits."""
    x, t = state[which], state["table"].long()
    rows = _values(x[t], state[which + "_scale"][t]) if state["kv"] == "q8_0" else x[t].float()
    return rows.flatten(1, 2)[:, :state["most"]].transpose(1, 2).contiguous()


def _attend(state):
    if own:
        if state["before"] is None:
            return state["cache"].attend(state["query"], state["table"], state["lengths"], state["most"])
        return state["cache"].attend(state["query"], state["table"], state["lengths"], state["most"],
                                     weights=state["before"], weights_out=state["after"])
    q = state["query"]
    k, v = _gathered(state, "k"), _gathered(state, "v")
    s = q.float().unflatten(1, (state["kvheads"], -1)) @ k.transpose(2, 3) / math.sqrt(state["dim"])
    there = torch.arange(state["most"], device="cuda") < state["lengths"][:, None]
    s = s.masked_fill(~there[:, None, None], -math.inf)
    e = (s - s.amax(-1, keepdim=True)).exp()
    p = e / e.sum(-1, keepdim=True)
    out = (p @ v).flatten(1, 2).to(q.dtype)
    if state["before"] is None:
        return out
    return out, torch.where(there[:, None], state["before"] + p.sum(2), state["after"])


def _append(state):
    x, norm = state["k_new"], state["norm"]
    if own:
        more = {}
        if norm:
            more = dict(q=state["q_new"], q_norm=state["q_weight"], k_norm=state["k_weight"], eps=EPS,
                        rope=state["rope"], positions=state["positions"])
        q = state["cache"].append(x, state["v_new"], state["table"], state["lengths"], first=state["begin"], **more)
    else:
        each, B = state["each"], state["batch"]

        def turned(y, w):
            y = y.float()
            y = y / (y.square().mean(-1, keepdim=True) + EPS).sqrt() * w
            cos, sin = state["rope"][state["positions"].long()][:, None].unbind(-1)
            a, b = y.chunk(2, -1)
            return torch.cat([a * cos - b * sin, a * sin + b * cos], -1)

        slot = (state["lengths"][:, None] - each + torch.arange(each, device="cuda")).long()
        at = state["table"].gather(1, slot // state["page"]).long().reshape(-1), (slot % state["page"]).reshape(-1)
        q = turned(state["q_new"], state["q_weight"]).to(x.dtype) if norm else None
        k = turned(x, state["k_weight"]) if norm else x.float()
        for which, y in (("k", k), ("v", state["v_new"].float())):
            if state["kv"] == "q8_0":
                state[which][at], state[which + "_scale"][at] = _quantised(y)
            else:
                state[which][at] = y.to(state[which].dtype)
    if state["kv"] == "q8_0":
        return _values(state["k"], state["k_scale"]), _values(state["v"], state["v_scale"])
    return q, state["k"], state["v"]


def _order(w):
    """Whole numbers in the total order of 32-bit floats."""
    b = w.contiguous().view(torch.int32).long()
    return torch.where(b < 0, -b - 1 - (1 << 31), b)


def _evict(state):
    keep, first, recent, page = state["keep"], state["first"], state["recent"], state["page"]
    if own:
        kept, weights, lengths = state["cache"].evict(state["heavy"], state["table"], state["lengths"], keep,
                                                      state["to"], first=first, recent=recent)
        return kept, weights, lengths, state["k"], state["v"]
    w, n = state["heavy"], state["lengths"].long()[:, None, None]
    t = torch.arange(state["most"], device="cuda").expand_as(w)
    # all that has to stay before the heaviest, these before the rest, ties by index
    must = (t < first) | (t >= n - recent) | (n <= keep)
    rank = (_order(w) << 24) - t
    rank = torch.where(must, torch.full_like(rank, 1 << 62), rank)
    rank = torch.where(t < n, rank, torch.full_like(rank, -(1 << 62)))
    if keep > w.shape[-1]:
        rank = torch.nn.functional.pad(rank, (0, keep - w.shape[-1]), value=-(1 << 62))
    ids = rank.topk(keep, -1).indices
    short = n.clamp(max=keep)
    ids = torch.where(ids < n, ids, torch.full_like(ids, 1 << 40)).sort(-1).values
    real = torch.arange(keep, device="cuda") < short
    ids = torch.where(real, ids, torch.zeros_like(ids))
    kept = torch.where(real, ids, torch.full_like(ids, -1)).int()
    weights = torch.where(real, w.gather(2, ids), torch.zeros_like(w[..., :1]))
    heads = torch.arange(state["kvheads"], device="cuda")[None, :, None].expand_as(ids)
    old = state["table"].long()[:, None].expand(-1, ids.shape[1], -1).gather(2, ids // page)
    j = torch.arange(keep, device="cuda").expand_as(ids)
    new = state["to"].long()[:, None].expand(-1, ids.shape[1], -1).gather(2, j // page)
    for which in ("k", "v"):
        x = state[which]
        x[new[real.expand_as(ids)], (j % page)[real.expand_as(ids)], heads[real.expand_as(ids)]] = \
            x[old, ids % page, heads][real.expand_as(ids)]
    return kept, weights, short[:, 0, 0].int(), state["k"], state["v"]


def _logprobs(state):
    top = state["top"]
    if own:
        return _serving().logprobs(state["device"], state["logits"], state["targets"], top=top, valid=state["valid"])
    x = state["logits"].float()
    if state["valid"] is not None:
        x = torch.where(state["valid"].bool(), x, torch.full_like(x[:, :1], torch.finfo(torch.float32).min))
    m = x.amax(-1, keepdim=True)
    e = (x - m).exp()
    total = e.sum(-1, keepdim=True)
    every = m + total.log()
    entropy = total.log() - (e * (x - m)).sum(-1, keepdim=True) / total
    found = x.gather(1, state["targets"].long()[:, None]) - every
    if not top:
        return found[:, 0], entropy[:, 0], None, None
    t = torch.arange(state["vocab"], device="cuda")
    ids = ((_order(x) << 24) - t).topk(top, -1).indices
    return found[:, 0], entropy[:, 0], ids.int(), x.gather(1, ids) - every


# ------------------------------------------------------------------ work --
def work(case):
    if case["op"] == "logprobs":
        n, vocab = case["rows"], case["vocab"]
        # one exponential and a product a logit
        return {"bytes": n * vocab * BYTES[case["x"]] + vocab * case["mask"] + n * (12 + 8 * case["top"]),
                "flops": 4 * n * vocab}
    lengths, g, d, kv = _lengths(case), case["kvheads"], case["dim"], BYTES[case["kv"]]
    pages = sum(-(-t // case["page"]) for t in lengths)
    if case["op"] == "attend":
        total, h, B = sum(lengths), case["heads"], case["batch"]
        return {"bytes": 2 * total * g * d * kv + 2 * B * h * d * BYTES[case["q"]] + 4 * pages + 4 * B
                + 8 * g * total * case["weights"],
                "flops": 4 * total * h * d}
    if case["op"] == "append":
        n, h = case["batch"] * case["each"], case["heads"]
        return {"bytes": n * d * ((2 * h + 2 * g) * BYTES[case["x"]] + 2 * g * kv) + n * (4 * d + 8) * case["norm"],
                "flops": n * d * (h + 2 * g) * 8}
    kept = sum(min(t, case["keep"]) for t in lengths)
    return {"bytes": 4 * g * sum(lengths) + kept * g * (4 * d * kv + 8) + 4 * pages, "flops": 2 * g * sum(lengths)}


# --------------------------------------------------------------- 64 bits --
def exact(case, seed):
    if case["op"] == "evict":
        return None  # choices and moves
    state = prepare(case, seed)
    if case["op"] == "logprobs":
        x = state["logits"].double()
        if state["valid"] is not None:
            x[:, state["valid"] == 0] = torch.finfo(torch.float32).min
        every = torch.logsumexp(x, -1)
        found = x[torch.arange(len(x)), state["targets"].long()] - every
        p = torch.softmax(x, -1)
        entropy = torch.special.entr(p).sum(-1)
        del p
        if not case["top"]:
            return found, entropy, None, None
        return found, entropy, None, x.sort(-1, descending=True).values[:, :case["top"]] - every[:, None]
    page, d, G = case["page"], case["dim"], case["kvheads"]
    if case["op"] == "append":
        if case["kv"] == "q8_0":
            outs, n = [], case["each"]
            for m in "kv":
                held = _values(state[m], state[m + "_scale"]).double()
                blocks = state[m + "_new"].double().unflatten(-1, (-1, 32))
                d = (blocks.abs().amax(-1, keepdim=True) / 127).half().double()
                new = (torch.round(blocks / d).clamp(-127, 127) * d).flatten(-2)
                for b, t in enumerate(state["lengths"].tolist()):
                    s = torch.arange(t - n, t, device="cuda")
                    held[state["table"][b, s // page].long(), s % page] = new[b * n:b * n + n]
                outs.append(held)
            return tuple(outs)
        outs = []
        for x, w in ((state["q_new"], state["q_weight"]), (state["k_new"], state["k_weight"])):
            x = x.double() * w.double() * torch.rsqrt(x.double().pow(2).mean(-1, keepdim=True) + EPS)
            r = torch.view_as_complex(state["rope"].double())[state["positions"].long()][:, None]
            z = torch.complex(x[..., :d // 2].contiguous(), x[..., d // 2:].contiguous()) * r
            outs.append(torch.cat([z.real, z.imag], -1))
        k, v, n = state["k"].double(), state["v"].double(), case["each"]
        for b, t in enumerate(state["lengths"].tolist()):
            s = torch.arange(t - n, t, device="cuda")
            p = state["table"][b, s // page].long()
            k[p, s % page] = outs[1][b * n:b * n + n]
            v[p, s % page] = state["v_new"][b * n:b * n + n].double()
        return outs[0], k, v
    out, weights = [], None if state["after"] is None else state["after"].double()
    for b, t in enumerate(state["lengths"].tolist()):
        s = torch.arange(t, device="cuda")
        p = state["table"][b, s // page].long()
        k, v = ((_values(state[m][p, s % page], state[m + "_scale"][p, s % page]) if case["kv"] == "q8_0"
                 else state[m][p, s % page]).double().permute(1, 0, 2).contiguous() for m in "kv")
        q = state["query"][b].double().reshape(G, -1, d)
        a = torch.softmax(torch.bmm(q, k.transpose(1, 2).contiguous()) / math.sqrt(d), -1)
        out.append(torch.bmm(a, v).reshape(-1, d))
        if weights is not None:
            weights[b, :, :t] = state["before"][b, :, :t].double() + a.sum(1)
    out = torch.stack(out)
    return out if weights is None else (out, weights)
