"""Measured calls of the serving operators for prompts and drafted tokens over a paged key-value cache: pages
and slots for new tokens, causal attention of prompts, attention of trees of drafted tokens, and the
acceptance of a tree's tokens.

Each case names its `op`:
  plan     pages for the tokens that sequences grow by, with their tables, slots and positions, and the pages
           back when the sequences shrink by as many
  prompts  causal attention of the new tokens of several sequences over their pages
  tree     attention of drafted tokens: each sees its sequence's context and its own ancestors
  accept   the drafted tokens' keys and values go into the cache (of each layer), the tree is walked by what
           the model chose, and the accepted ones move up behind the context

With `own` false, run() computes them in elementary torch operations.
"""
import importlib
import math
import random

import torch

own = False

VOCAB = 151936
FLOATS = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4.0, "f16": 2.0, "bf16": 2.0, "q8_0": 34 / 32}
ROWS = 1 << 28  # scores that the plain form holds at a time


def listed():
    return [
        # the decode step of a batch: one token each, few of them into a new page
        {"name": "plan-decode", "op": "plan", "batch": 64, "lo": 1, "hi": 4096, "new_lo": 1, "new": 1, "page": 16,
         "tree": False},
        # the requests of a busy second come and go
        {"name": "plan-prompts", "op": "plan", "batch": 48, "lo": 0, "hi": 900, "new_lo": 1, "new": 2100, "page": 16,
         "tree": False},
        # drafted trees of a batch
        {"name": "plan-tree", "op": "plan", "batch": 32, "lo": 1, "hi": 4096, "new_lo": 9, "new": 26, "page": 16,
         "tree": True},
        # one question in the engine's own types: latency counts
        {"name": "prompt-one", "op": "prompts", "batch": 1, "lo": 0, "hi": 0, "new_lo": 517, "new": 517, "heads": 32,
         "kvheads": 4, "dim": 128, "page": 16, "q": "f32", "kv": "f32"},
        # the prompts of one prefill, from one token on
        {"name": "prompts-packed", "op": "prompts", "batch": 24, "lo": 0, "hi": 300, "new_lo": 1, "new": 2100,
         "heads": 32, "kvheads": 4, "dim": 128, "page": 16, "q": "bf16", "kv": "bf16"},
        # a long document at once
        {"name": "prompt-long", "op": "prompts", "batch": 1, "lo": 0, "hi": 0, "new_lo": 16381, "new": 16381,
         "heads": 32, "kvheads": 4, "dim": 128, "page": 64, "q": "f16", "kv": "f16"},
        # the next pieces of two long documents, cache held in 8 bits
        {"name": "prompts-8bit", "op": "prompts", "batch": 2, "lo": 12000, "hi": 15000, "new_lo": 512, "new": 512,
         "heads": 32, "kvheads": 4, "dim": 128, "page": 32, "q": "bf16", "kv": "q8_0"},
        # one conversation's drafted tree: latency counts
        {"name": "tree-one", "op": "tree", "batch": 1, "lo": 517, "hi": 517, "new_lo": 16, "new": 16, "heads": 32,
         "kvheads": 4, "dim": 128, "page": 16, "q": "bf16", "kv": "bf16"},
        # a serving batch of ragged histories
        {"name": "tree-batch", "op": "tree", "batch": 48, "lo": 1, "hi": 4096, "new_lo": 9, "new": 26, "heads": 32,
         "kvheads": 4, "dim": 128, "page": 16, "q": "bf16", "kv": "bf16"},
        # two long documents, the largest trees
        {"name": "tree-long", "op": "tree", "batch": 2, "lo": 65537, "hi": 65537, "new_lo": 64, "new": 64, "heads": 32,
         "kvheads": 4, "dim": 128, "page": 64, "q": "f16", "kv": "f16"},
        # one conversation, two layers in the engine's own types
        {"name": "accept-one", "op": "accept", "batch": 1, "lo": 517, "hi": 517, "new_lo": 16, "new": 16, "kvheads": 4,
         "dim": 128, "page": 16, "q": "f32", "kv": "f32", "layers": 2},
        # a batch, four layers
        {"name": "accept-batch", "op": "accept", "batch": 48, "lo": 1, "hi": 4096, "new_lo": 9, "new": 26,
         "kvheads": 4, "dim": 128, "page": 16, "q": "bf16", "kv": "bf16", "layers": 4},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    op = rng.choice(["plan", "plan", "prompts", "prompts", "prompts", "tree", "tree", "tree", "accept", "accept"])
    page = rng.choice([16, 16, 32, 64, 24, 128])
    c = {"op": op, "page": page}
    if op == "plan":
        tree = rng.random() < 0.4
        batch = _log_int(rng, 1, 48)
        new = rng.randint(1, 64) if tree else rng.choice([1, _log_int(rng, 1, 2100)])
        c.update(batch=batch, lo=rng.randint(0, 60), hi=60 + _log_int(rng, 1, 4000), new_lo=rng.randint(1, new), new=new,
                 tree=tree)
        return c
    kvheads, dim = rng.choice([1, 2, 4, 4, 8]), rng.choice([64, 128, 128, 128])
    c.update(kvheads=kvheads, dim=dim)
    q, kv = rng.choice([("f32", "f32"), ("f16", "f16"), ("bf16", "bf16"), ("bf16", "bf16"), ("bf16", "q8_0"),
                        ("f32", "f16")])
    c.update(q=q, kv=kv)
    if op == "accept":
        batch, new = _log_int(rng, 1, 48), rng.randint(1, 64)
        c.update(batch=batch, lo=rng.randint(0, 60), hi=60 + _log_int(rng, 1, 2000), new_lo=rng.randint(1, new), new=new,
                 layers=rng.randint(1, 4))
        return c
    c["heads"] = heads = kvheads * rng.choice([1, 2, 4, 5, 8])
    if op == "tree":
        new = rng.randint(1, 64)
        hi = _log_int(rng, 16, 65537)
        batch = max(1, min(_log_int(rng, 1, 48), int(130e6 / (hi * kvheads * dim * BYTES[kv]))))
        c.update(batch=batch, lo=rng.randint(0, hi) if batch > 1 else hi, hi=hi, new_lo=rng.randint(1, new), new=new)
        return c
    new = _log_int(rng, 1, 8000)
    hi = rng.choice([0, _log_int(rng, 1, 16000)])
    # at most some 2e10 pairs of a query head and a key in 16 bits, less where all is in 32
    most = 2e10 if q == kv != "f32" else 4e9
    batch = max(1, min(_log_int(rng, 1, 24), int(most / (heads * new * (hi + new / 2)))))
    c.update(batch=batch, lo=rng.randint(0, hi) if batch > 1 else hi, hi=hi,
             new_lo=rng.randint(1, new) if batch > 1 else new, new=new)
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


def _evenly(lo, hi, n):
    """n whole numbers evenly from lo to hi (both reached)."""
    return [hi - (hi - lo) * i // max(1, n - 1) for i in range(n)]


def _sequences(case):
    """(keys of each sequence's context, its new tokens): both evenly over their ranges, in orders of their own."""
    n, rng = case["batch"], random.Random(case["batch"])
    context, new = _evenly(case["lo"], case["hi"], n), _evenly(case["new_lo"], case["new"], n)
    rng.shuffle(context)
    rng.shuffle(new)
    return context, new


def _ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device="cuda")


def _sums(values):
    out = [0]
    for v in values:
        out.append(out[-1] + v)
    return out


def _quantised(x):
    """(codes, scales) of blocks of 32 values: scale = largest magnitude / 127 in 16 bits."""
    b = x.float().unflatten(-1, (-1, 32))
    d = (b.abs().amax(-1, keepdim=True) / 127).half()
    f = d.float()
    codes = torch.where(f > 0, (b / f).round().clamp(-127, 127), torch.zeros_like(b)).to(torch.int8)
    return codes.flatten(-2), d[..., 0]


def _values(codes, scales):
    return (codes.unflatten(-1, (-1, 32)).float() * scales.float()[..., None]).flatten(-2)


def _table(lengths, page, g, extra=0):
    """(table, pages in all): every sequence's pages, scattered over the pool, and `extra` more entries a row."""
    need = [-(-t // page) for t in lengths]
    pool = sum(need) + 3
    order = torch.randperm(pool, generator=g, device="cuda").int()
    at, done = torch.zeros(len(need), max(max(need), 1) + extra, dtype=torch.long), 0
    for i, m in enumerate(need):
        at[i, :m] = torch.arange(done, done + m)
        done += m
    return order[at.cuda()], pool


def _trees(counts, g):
    """(parents, ancestors): random trees, packed; node 0 is the root and a parent lies in front of its children."""
    most = max(counts)
    back = (torch.rand(len(counts), most, generator=g, device="cuda") * 8).long().clamp(max=7)
    node = torch.arange(most, device="cuda")
    parent = (node - 1 - back).clamp(min=0)
    parent[:, 0] = -1
    seen = torch.zeros(len(counts), most, dtype=torch.long, device="cuda")
    for j in range(most):
        mine = torch.full_like(seen[:, :1], 1 << j if j < 63 else -(1 << 63))
        seen[:, j:j + 1] = mine | (seen.gather(1, parent[:, j:j + 1]) if j else 0)
    there = node < _ints(counts, torch.long)[:, None]
    return parent[there].int(), seen[there]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def randn(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    state = dict(case)
    B, page = case["batch"], case["page"]
    context, new = _sequences(case)
    n, begin = sum(new), _sums(new)
    state.update(context=context, counts=new, n=n, begin=begin)
    if case["op"] == "plan":
        # tables with room for more, sequences that hold what they need, and the other pages free
        grown = [-(-(a + b) // page) for a, b in zip(context, new)]
        held = [-(-a // page) for a in context]
        pages = sum(grown) + 37
        ids = torch.randperm(pages, generator=g, device="cuda").int()
        table = torch.zeros(B, max(grown) + 5, dtype=torch.int32, device="cuda")
        at = _sums(held)
        for b, m in enumerate(held):
            table[b, :m] = ids[at[b]:at[b] + m]
        free = torch.zeros(pages, dtype=torch.int32, device="cuda")
        free[:pages - at[-1]] = ids[at[-1]:]
        state.update(pages=pages, table=table, held=_ints(held), lengths=_ints(context), grow=_ints(new),
                     shrink=-_ints(new), free=free, count=_ints([pages - at[-1]]),
                     parents=_trees(new, g)[0] if case["tree"] else None)
        if own:
            state["pool"] = _serving().PagePool(_engine(), pages, page, free=free, count=state["count"])
        return state

    G, d, kv = case["kvheads"], case["dim"], case["kv"]
    lengths = [a + b for a, b in zip(context, new)]
    table, pool = _table(lengths, page, g)
    layers = []
    for _ in range(case.get("layers", 1)):
        held = []
        for _ in range(2):
            x = randn(pool, page, G, d)
            held += _quantised(x) if kv == "q8_0" else (x.to(FLOATS[kv]), None)
        layers.append({"k": held[0], "k_scale": held[1], "v": held[2], "v_scale": held[3]})
    state.update(table=table, most=max(lengths), lengths=_ints(lengths), first=_ints(begin), layers=layers)
    if case["op"] in ("prompts", "tree"):
        state["query"] = (2 * randn(n, case["heads"], d)).to(FLOATS[case["q"]])
    if case["op"] in ("tree", "accept"):
        state["parents"], state["ancestors"] = _trees(new, g)
    if case["op"] == "accept":
        # one projection's rows hold k and v
        for layer in layers:
            rows = randn(n, 2 * G * d).to(FLOATS[case["q"]])
            layer["k_new"], layer["v_new"] = (m.unflatten(1, (G, d)) for m in rows.chunk(2, 1))
        tokens = torch.randint(0, VOCAB, (n,), generator=g, device="cuda")
        # four nodes of five are followed by one of their children
        chosen = torch.randint(0, VOCAB, (n,), generator=g, device="cuda")
        base = torch.repeat_interleave(_ints(begin[:-1], torch.long), _ints(new, torch.long))
        child = state["parents"] >= 0
        where = (base + state["parents"])[child]
        likely = torch.rand(n, generator=g, device="cuda") < 0.8
        follow = torch.full_like(chosen, -1)
        follow.scatter_reduce_(0, where, tokens[child], "amax")
        state["tokens"] = tokens.int()
        state["chosen"] = torch.where((follow >= 0) & likely, follow, chosen).int()
    if own:
        s, dev = _serving(), _engine()
        state["caches"] = [s.PagedCache(dev, x["k"], x["v"], x["k_scale"], x["v_scale"]) for x in layers]
    return state


# ------------------------------------------------------------------ runs --
def run(state):
    return {"plan": _plan, "prompts": _prompts, "tree": _tree, "accept": _accept}[state["op"]](state)


def _plan(state):
    table, held, lengths = state["table"], state["held"], state["lengths"]
    if own:
        more = state["pool"].plan(table, held, lengths, state["grow"], state["n"], parents=state["parents"])
        less = state["pool"].plan(table, held, more.lengths, state["shrink"], 0)
        grown, seen = more.lengths, more.ancestors
        first, sequence, position, slot = more.first, more.sequences, more.positions, more.slots
        shrunk = less.lengths
    else:
        page, n, B = state["page"], state["n"], state["batch"]
        free, count = state["free"], state["count"]
        # all of these cases' sequences fit
        grown = lengths + state["grow"]
        need = (grown + page - 1) // page
        claims = (need - held).clamp(min=0)
        upto = claims.cumsum(0)
        at = torch.arange(table.shape[1], device="cuda")
        claimed = (at >= held[:, None]) & (at < need[:, None])
        which = count.long() - 1 - ((upto - claims)[:, None] + at - held[:, None])
        table.copy_(torch.where(claimed, free[which.clamp(0, len(free) - 1)], table))
        held.copy_(torch.maximum(need, held))
        count.sub_(upto[-1])
        first = torch.cat([torch.zeros_like(held[:1]), state["grow"].cumsum(0).int()])
        token = torch.arange(n, device="cuda", dtype=torch.int32)
        sequence = (torch.searchsorted(first, token, right=True) - 1).int()
        row = sequence.long()
        place = (lengths[row] + token - first[row]).int()
        slot = table[row, (place // page).long()].long() * page + place % page
        position, seen = place, None
        if state["parents"] is not None:
            # a node's ancestors: itself and its parent's, one level of the trees after the other
            parent, base = state["parents"].long(), first[row].long()
            node = token - base
            one = torch.where(node < 63, 1 << node.clamp(max=62), torch.full_like(node, -(1 << 63)))
            seen, up = one, torch.where(parent >= 0, base + parent, token.long())
            for _ in range(6):  # a path of up to 64 nodes
                seen, up = seen | seen[up], up[up]
            bits = (seen[:, None] >> torch.arange(64, device="cuda")) & 1
            position = (lengths[row] + bits.sum(1) - 1).int()
        # and back
        shrunk = grown + state["shrink"]
        keep = (shrunk + page - 1) // page
        back = (held - keep).clamp(min=0)
        behind = back.sum() - back.cumsum(0)
        gone = (at >= keep[:, None]) & (at < held[:, None])
        to = count.long() + behind[:, None] + (held[:, None] - 1 - at)
        free.scatter_(0, torch.where(gone, to, len(free) - 1)[gone], table[gone])
        held.copy_(torch.minimum(keep, held))
        count.add_(back.sum())
    return grown, first, sequence, position, slot, seen, shrunk, table, held, state["free"], state["count"]


def _rows(state, which, b, dtype=torch.float32):
    """Sequence b's keys or values [kvheads][length][dim]."""
    layer, t = state["layers"][0], state["context"][b] + state["counts"][b]
    page, at = state["page"], state["table"][b, :-(-t // state["page"])].long()
    x = layer[which][at]
    x = _values(x, layer[which + "_scale"][at]).to(dtype) if state["kv"] == "q8_0" else x.to(dtype)
    return x.flatten(0, 1)[:t].transpose(0, 1).contiguous()


def _visible(state, b, lo, hi):
    """[hi - lo][length]: which keys new tokens lo .. hi of sequence b see."""
    context, n, begin = state["context"][b], state["counts"][b], state["begin"][b]
    t = torch.arange(context + n, device="cuda")
    if state["op"] == "prompts":
        return t <= context + torch.arange(lo, hi, device="cuda")[:, None]
    bits = (state["ancestors"][begin + lo:begin + hi, None] >> (t - context).clamp(min=0)) & 1
    return (t < context) | (bits == 1)


def _attend(state):
    G, scale = state["kvheads"], state["dim"] ** -0.5
    out = torch.empty_like(state["query"])
    for b in range(state["batch"]):
        k, v = _rows(state, "k", b).transpose(1, 2).contiguous(), _rows(state, "v", b)
        per = max(1, ROWS // (state["heads"] * k.shape[2]))
        for lo in range(0, state["counts"][b], per):
            hi = min(state["counts"][b], lo + per)
            rows = slice(state["begin"][b] + lo, state["begin"][b] + hi)
            # [kvheads][tokens x query heads of one][dim]
            q = state["query"][rows].float().unflatten(1, (G, -1)).transpose(0, 1).contiguous()
            s = (q.flatten(1, 2) @ k * scale).unflatten(1, (hi - lo, -1))
            s = s.masked_fill_(~_visible(state, b, lo, hi)[:, None], -math.inf)
            e = s.sub_(s.amax(-1, keepdim=True)).exp_()
            p = e.div_(e.sum(-1, keepdim=True))
            o = (p.flatten(1, 2) @ v).unflatten(1, (hi - lo, -1))
            out[rows] = o.transpose(0, 1).flatten(1, 2).to(out.dtype)
    return out


def _prompts(state):
    if own:
        return state["caches"][0].attend_prompts(state["query"], state["table"], state["lengths"], state["first"],
                                                 state["most"])
    return _attend(state)


def _tree(state):
    if own:
        return state["caches"][0].attend_tree(state["query"], state["table"], state["lengths"], state["first"],
                                              state["ancestors"], state["most"])
    return _attend(state)


def _accept(state):
    layers = state["layers"]
    if own:
        for cache, x in zip(state["caches"], layers):
            cache.append(x["k_new"], x["v_new"], state["table"], state["lengths"], first=state["first"])
        lengths, accepted, path, following = _serving().accept(
            state["caches"], state["parents"], state["tokens"], state["chosen"], state["table"], state["lengths"],
            state["first"])
    else:
        n, page, first = state["n"], state["page"], state["first"]
        token = torch.arange(n, device="cuda")
        row = torch.searchsorted(first, token.int(), right=True) - 1
        base = first[row].long()
        parent = base + state["parents"].long()
        root = state["parents"] < 0
        place = (state["lengths"][row] - first[row + 1]).long() + token
        page_of, slot = state["table"][row, place // page].long(), place % page
        for x in layers:
            for which in "kv":
                y = x[which + "_new"]
                if state["kv"] == "q8_0":
                    x[which][page_of, slot], x[which + "_scale"][page_of, slot] = _quantised(y)
                else:
                    x[which][page_of, slot] = y.to(x[which].dtype)
        up = torch.where(root, token, parent)
        fits = root | (state["tokens"] == state["chosen"][up])
        # of siblings that fit, the first
        rank = torch.full_like(token, n).scatter_reduce(0, up, torch.where(fits & ~root, token, n), "amin")
        good = root | (rank[up] == token)
        for _ in range(6):  # every ancestor fits
            good, up = good & good[up], up[up]
        nodes = good.int()
        upto = nodes.cumsum(0)
        before = torch.cat([torch.zeros_like(upto[:1]), upto])[first.long()]
        accepted = (before[1:] - before[:-1]).int()
        lengths = state["lengths"] - (first[1:] - first[:-1]) + accepted
        step = (upto - 1 - before[:-1][row])[good]
        path = torch.full_like(state["parents"], -1)
        path[base[good] + step] = (token - base)[good].int()
        last = path.long()[first[:-1].long() + accepted.long() - 1]
        following = state["chosen"][first[:-1].long() + last]
        to = (state["lengths"][row] - first[row + 1] + first[row]).long()[good] + step
        to_page, to_slot = state["table"][row[good], to // page].long(), to % page
        for x in layers:
            for which in ("k", "v", "k_scale", "v_scale"):
                if x[which] is not None:
                    x[which][to_page, to_slot] = x[which][page_of[good], slot[good]]
    held = [(_values(x["k"], x["k_scale"]), _values(x["v"], x["v_scale"])) if state["kv"] == "q8_0" else (x["k"], x["v"])
            for x in layers]
    return lengths, accepted, path, following, held


# ------------------------------------------------------------------ work --
def _pairs(case):
    """(new tokens, keys that they see in all, keys) of the sequences. Of a tree a node sees some half."""
    context, new = _sequences(case)
    return sum(new), sum(c * n + n * (n + 1) / 2 for c, n in zip(context, new)), sum(context) + sum(new)


def work(case):
    B, page = case["batch"], case["page"]
    n, seen, keys = _pairs(case)
    if case["op"] == "plan":
        # lengths, growth and counts read and written twice, claimed pages, and what each token gets
        return {"bytes": 2 * 24 * B + 4 * (B + 1) + 4 * 4 * n / page + n * (28 if case["tree"] else 16), "flops": n}
    g, d, kv = case["kvheads"], case["dim"], BYTES[case["kv"]]
    if case["op"] == "accept":
        moved = n / 4
        return {"bytes": case["layers"] * 2 * g * d * (n * (BYTES[case["q"]] + kv) + 2 * moved * kv) + 16 * n + 16 * B,
                "flops": n}
    h = case["heads"]
    return {"bytes": 2 * keys * g * d * kv + 2 * n * h * d * BYTES[case["q"]] + 4 * keys / page + 8 * B
            + 8 * n * (case["op"] == "tree"), "flops": 4 * seen * h * d}


# --------------------------------------------------------------- 64 bits --
def exact(case, seed):
    if case["op"] in ("plan", "accept"):
        return None  # whole numbers, and moves
    state = prepare(case, seed)
    G, d, scale = case["kvheads"], case["dim"], 1 / math.sqrt(case["dim"])
    out = torch.empty(state["query"].shape, dtype=torch.float64, device="cuda")
    per = case["heads"] // G
    for b, (context, n) in enumerate(zip(state["context"], state["counts"])):
        k, v = _rows(state, "k", b, torch.float64), _rows(state, "v", b, torch.float64)
        if case["kv"] == "q8_0":
            at = state["table"][b, :-(-(context + n) // case["page"])].long()
            k, v = ((state["layers"][0][m][at].unflatten(-1, (-1, 32)).double()
                     * state["layers"][0][m + "_scale"][at].double()[..., None]).flatten(-2).flatten(0, 1)[:context + n]
                    .transpose(0, 1) for m in "kv")
        step = max(1, (1 << 27) // (context + n))
        for h in range(case["heads"]):
            kt, vt = k[h // per].T.contiguous(), v[h // per].contiguous()
            for lo in range(0, n, step):
                hi = min(n, lo + step)
                rows = slice(state["begin"][b] + lo, state["begin"][b] + hi)
                s = torch.mm(state["query"][rows, h].double(), kt) * scale
                s[~_visible(state, b, lo, hi)] = -math.inf
                out[rows, h] = torch.mm(torch.softmax(s, -1), vt)
    return out
