"""Operators on torch tensors of the GPU, for a program that serves several
sequences: a key-value cache held in pages (`PagedCache`: append, attend,
attend_prompts, attend_tree, evict), pages given out and taken back (`PagePool`),
drafted tokens accepted (`accept`) and the log probabilities of tokens
(`logprobs`), over the C ABI's entry points for device tensors
(include/qwen_hip.h: qh_paged_*, qh_logprobs).

Every call runs on torch's current stream of the tensors' device, which is the
given engine Device's, returns at once, and may be captured into a graph.  What
it allocates (outputs that are not given, workspaces) comes from torch's
allocator.  Arguments on the host are checked (EngineError); lengths, page ids
and targets lie on the device and are checked there: the header says what a call
does with those out of range.  Nothing here has a gradient: a tensor that requires
one is refused where torch records gradients (call under torch.no_grad()).

    serving = importlib.import_module("qwen-30brust_amd.serving")
"""
import collections
import ctypes as C
import importlib

import torch

engine = importlib.import_module(__package__)
EngineError = engine.EngineError

KIND = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 30}
_BYTES = C.c_size_t


def _need(ok, message):
    if not ok:
        raise EngineError(message)


def _on(dev, t, what, dtypes, ndim):
    """Checks a tensor's place, type and rank, and that its last dimension is contiguous; its shape and strides."""
    if not isinstance(t, torch.Tensor):
        raise EngineError(f"{what}: not a tensor on the engine's device")
    if t.requires_grad and torch.is_grad_enabled():
        raise EngineError(f"{what}: no gradient is recorded here; call under torch.no_grad()")
    if t.get_device() != dev.index:  # -1 on the host
        raise EngineError(f"{what}: not a tensor on the engine's device")
    if t.dtype not in dtypes:
        raise EngineError(f"{what}: type {t.dtype} is not supported")
    shape, strides = t.shape, t.stride()
    if len(strides) != ndim:
        raise EngineError(f"{what}: {ndim} dimensions are needed, {t.dim()} given")
    if strides[-1] != 1 and shape[-1] > 1:
        raise EngineError(f"{what}: the last dimension is not contiguous")
    return shape, strides


_I32, _F32 = (torch.int32,), (torch.float32,)


def _stream(dev):
    # the handle alone: a Stream object would take a microsecond more
    return torch._C._cuda_getCurrentRawStream(dev.index) or engine.NULL_STREAM


def _live(dev):
    if dev.h is None:
        raise EngineError("the device was closed")
    return dev.h


def _shared(t):
    """Whether elements share memory (an expanded dimension)."""
    return any(n > 1 and s == 0 for n, s in zip(t.shape, t.stride()))


def _apart(t, what):
    if _shared(t):
        raise EngineError(f"{what}: elements of an output share memory")


def _heads(dev, t, what, rows, heads, dim):
    shape, strides = _on(dev, t, what, KIND, 3)
    if shape != (rows, heads, dim):
        raise EngineError(f"{what}: shape {tuple(shape)}, not {(rows, heads, dim)}")
    return engine._Heads(t.data_ptr(), KIND[t.dtype], strides[0], strides[1])


class PagedCache:
    """A key-value cache in pages: k and v [pages][page][kvheads][dim] in f32,
    f16 or bf16, or int8 codes (Q8_0) with k_scale and v_scale
    [pages][page][kvheads][dim / 32] in f16.  The tensors stay the caller's; k
    and v have the same strides.  Heads are at most 256 wide."""

    def __init__(self, device, k, v, k_scale=None, v_scale=None):
        q8 = isinstance(k, torch.Tensor) and k.dtype == torch.int8
        for t, what in ((k, "cache keys"), (v, "cache values")):
            _on(device, t, what, (torch.int8,) if q8 else KIND, 4)
        _need(k.shape == v.shape and k.dtype == v.dtype and k.stride() == v.stride(),
              "cache keys and values differ in shape, type or strides")
        if q8:
            for t, what in ((k_scale, "cache key scales"), (v_scale, "cache value scales")):
                _on(device, t, what, (torch.float16,), 4)
                _need(k.shape[3] % 32 == 0 and t.shape == (*k.shape[:3], k.shape[3] // 32)
                      and all(n == 1 or 32 * a == b for n, a, b in zip(k.shape[:3], t.stride(), k.stride())),
                      f"{what}: one for each 32 codes, at their offset / 32")
        else:
            _need(k_scale is None and v_scale is None, "scales go with a cache of 8-bit codes")
        self.device, self.k, self.v, self.k_scale, self.v_scale = device, k, v, k_scale, v_scale
        self._writable = not (_shared(k) or _shared(v))
        pages, self.page, self.kvheads, self.dim = k.shape
        # a dimension of one has no stride of its own
        st = [s if n > 1 else 32 * -(-s // 32) for n, s in zip(k.shape[:3], k.stride())]
        self._pages = engine._Pages(k.data_ptr(), v.data_ptr(), k_scale.data_ptr() if q8 else None,
                                    v_scale.data_ptr() if q8 else None, 8 if q8 else KIND[k.dtype], self.page,
                                    self.kvheads, self.dim, pages, *st)

    def _sequences(self, table, lengths, most):
        dev = self.device
        (rows, pages), strides = _on(dev, table, "page table", _I32, 2)
        (batch,), _ = _on(dev, lengths, "lengths", _I32, 1)
        if rows != batch:
            raise EngineError("the page table has other sequences than the lengths")
        if most is None:
            most = min(pages * self.page, 0x7fffffff - (1 << 20))
        if not 0 <= most <= 0x7fffffff:
            raise EngineError("longest length out of range")
        return engine._Sequences(table.data_ptr(), lengths.data_ptr(), strides[0], pages, batch, most)

    def append(self, k, v, table, lengths, first=None, *, q=None, q_out=None, q_norm=None, k_norm=None, eps=1e-6,
               rope=None, positions=None):
        """Appends tokens' keys and values ([n][kvheads][dim]) to sequences
        whose `lengths` count them already; sequence b's tokens are first[b] ..
        first[b + 1] - 1 (None: one token each).  On the way k, and q
        ([n][heads][dim]) with it, are normed by head (q_norm, k_norm [dim]) and
        rotated by rope ([positions][dim / 2][2] of cos and sin) at `positions`
        [n] (None: their places).  Returns q_out (allocated if not given), or
        None without q."""
        dev, (n, d) = self.device, (k.shape[0], self.dim)
        _need(self._writable, "a cache whose elements share memory is read only")
        seqs = self._sequences(table, lengths, None)
        kh = _heads(dev, k, "keys", n, self.kvheads, d)
        vh = _heads(dev, v, "values", n, self.kvheads, d)
        if first is not None:
            _on(dev, first, "first tokens", _I32, 1)
            _need(first.shape[0] == lengths.shape[0] + 1, "first tokens: one more than sequences is needed")
        more = engine._Append(eps=eps)
        if q is not None:
            more.heads = heads = q.shape[1] if isinstance(q, torch.Tensor) and q.dim() == 3 else 0
            more.q = _heads(dev, q, "queries", n, heads, d)
            given = q_out is not None
            if not given:
                q_out = q.new_empty((n, heads, d))
            more.q_out = _heads(dev, q_out, "query outputs", n, heads, d)
            if given:
                _apart(q_out, "query outputs")
        else:
            _need(q_out is None and q_norm is None, "query outputs and weights go with queries")
        for name, w in (("q_norm", q_norm), ("k_norm", k_norm)):
            if w is not None:
                if _on(dev, w, name, _F32, 1)[0][0] != d:
                    raise EngineError(f"{name}: {d} weights are needed")
                setattr(more, name, w.data_ptr())
        if rope is not None:
            _on(dev, rope, "table of angles", _F32, 3)
            _need(tuple(rope.shape[1:]) == (d // 2, 2) and rope.is_contiguous(),
                  "table of angles: contiguous [positions][dim / 2][2] is needed")
            more.rope, more.rope_rows = rope.data_ptr(), rope.shape[0]
        if positions is not None:
            _need(rope is not None, "positions go with a table of angles")
            _on(dev, positions, "positions", _I32, 1)
            _need(positions.shape[0] == n, "positions: one for each token")
            more.position = positions.data_ptr()
        dev._check(engine.lib().qh_paged_append(_live(dev), self._pages, seqs,
                                                None if first is None else first.data_ptr(), n, kh, vh, more,
                                                _stream(dev)))
        return q_out

    def attend(self, q, table, lengths, most=None, *, scale=None, out=None, weights=None, weights_out=None):
        """Attention of one token per sequence, q [batch][heads][dim], over its
        cached keys: out like q (allocated if not given).  most: no length is
        above it (None: what the table's rows hold).  scale: 1 / sqrt(dim) if not
        given.  With weights and / or weights_out ([batch][kvheads][most or
        more] in f32) every key's softmax weight, summed over its KV head's query
        heads, is added to weights (zeros if not given) and written to
        weights_out (weights itself if not given); returns (out, weights_out).
        The call's workspace then holds every score: batch x heads x most x 4
        bytes."""
        dev, (batch, d) = self.device, (lengths.shape[0], self.dim)
        seqs = self._sequences(table, lengths, most)
        heads = q.shape[1] if isinstance(q, torch.Tensor) and q.dim() == 3 else 0
        qh = _heads(dev, q, "queries", batch, heads, d)
        given = out is not None
        if not given:
            out = q.new_empty((batch, heads, d))
        oh = _heads(dev, out, "attention outputs", batch, heads, d)
        if given:
            _apart(out, "attention outputs")
        w = None
        if weights_out is None:
            weights_out = weights
        if weights_out is not None:
            for t, what in ((weights, "weights"), (weights_out, "weight outputs")):
                if t is not None:
                    _on(dev, t, what, _F32, 3)
                    _need(t.shape[0] == batch and t.shape[1] == self.kvheads and t.shape[2] >= seqs.most,
                          f"{what}: [sequences][KV heads][longest length] is needed")
            _apart(weights_out, "weight outputs")
            i = (None, 0, 0) if weights is None else (weights.data_ptr(), weights.stride(0), weights.stride(1))
            w = engine._KeyWeights(i[0], weights_out.data_ptr(), i[1], i[2], weights_out.stride(0),
                                   weights_out.stride(1))
        lib, h = engine.lib(), _live(dev)
        need = _BYTES()
        dev._check(lib.qh_paged_attention_bytes(h, self._pages, seqs, heads, w is not None, need))
        work = torch.empty(need.value, dtype=torch.uint8, device=q.device) if need.value else None
        dev._check(lib.qh_paged_attention(h, self._pages, seqs, qh, heads, d ** -0.5 if scale is None else scale, oh,
                                          w, None if work is None else work.data_ptr(), need.value, _stream(dev)))
        return out if w is None else (out, weights_out)

    def attend_prompts(self, q, table, lengths, first, most=None, *, scale=None, out=None):
        """Causal attention of several new tokens per sequence, q
        [n][heads][dim]: sequence b's are rows first[b] .. first[b + 1] - 1, the
        last of its `lengths[b]` keys (appended before) their own, and each sees
        the keys up to its own.  A whole prompt, the next piece of one, or a single
        token.  out like q (allocated if not given); rows of no sequence are left as
        they were.  most and scale as in attend.  With 16-bit q and out over a
        cache of their type softmax weights keep attend's 17 bits (bf16) or 23 (f16);
        with bf16 ones over Q8_0 weights and values keep 11, where attend has 23; an
        f32 out keeps 32."""
        return self._many(q, table, lengths, first, None, most, scale, out)

    def attend_tree(self, q, table, lengths, first, ancestors, most=None, *, scale=None, out=None):
        """attend_prompts for drafted tokens: a sequence's new tokens are the nodes
        of a tree (at most 64), and node i sees every key in front of them and
        the key of node j where bit j of ancestors[i] ([n], int64) is set."""
        _on(self.device, ancestors, "ancestors", (torch.int64,), 1)
        return self._many(q, table, lengths, first, ancestors, most, scale, out)

    def _many(self, q, table, lengths, first, ancestors, most, scale, out):
        dev, d = self.device, self.dim
        seqs = self._sequences(table, lengths, most)
        n, heads = q.shape[:2] if isinstance(q, torch.Tensor) and q.dim() == 3 else (0, 0)
        qh = _heads(dev, q, "queries", n, heads, d)
        _on(dev, first, "first tokens", _I32, 1)
        _need(first.shape[0] == lengths.shape[0] + 1, "first tokens: one more than sequences is needed")
        _need(ancestors is None or ancestors.shape[0] == n, "ancestors: one for each token")
        given = out is not None
        if not given:
            out = q.new_empty((n, heads, d))
        oh = _heads(dev, out, "attention outputs", n, heads, d)
        if given:
            _apart(out, "attention outputs")
        lib, h = engine.lib(), _live(dev)
        need = _BYTES()
        dev._check(lib.qh_paged_prompts_bytes(h, self._pages, seqs, n, heads, need))
        work = torch.empty(need.value, dtype=torch.uint8, device=q.device) if need.value else None
        more = (qh, heads, d ** -0.5 if scale is None else scale, oh, None if work is None else work.data_ptr(),
                need.value, _stream(dev))
        if ancestors is None:
            dev._check(lib.qh_paged_prompts(h, self._pages, seqs, first.data_ptr(), n, *more))
        else:
            dev._check(lib.qh_paged_tree(h, self._pages, seqs, first.data_ptr(), n, ancestors.data_ptr(), *more))
        return out

    def evict(self, weights, table, lengths, keep, to, *, first=0, recent=0, most=None):
        """Brings sequences to at most `keep` keys: each KV head keeps its first
        `first` keys, its last `recent` and the heaviest between by `weights`
        ([batch][kvheads][most or more]), moved in order to the pages `to`
        [batch][pages], all different, which no sequence of the call reads.  Returns (kept
        indexes [batch][kvheads][keep] with -1 behind them, their weights, new
        lengths)."""
        dev = self.device
        _need(self._writable, "a cache whose elements share memory is read only")
        _on(dev, weights, "weights", _F32, 3)
        if most is None:
            most = min(weights.shape[2], table.shape[-1] * self.page)
        seqs = self._sequences(table, lengths, most)
        batch = lengths.shape[0]
        _need(weights.shape[0] == batch and weights.shape[1] == self.kvheads and weights.shape[2] >= most,
              "weights: [sequences][KV heads][longest length] is needed")
        _on(dev, to, "new pages", _I32, 2)
        _need(to.shape[0] == batch, "new pages: a row for each sequence is needed")
        _need(0 < keep < 1 << 30 and first >= 0 and recent >= 0, "keys to keep out of range")
        kept = torch.empty((batch, self.kvheads, keep), dtype=torch.int32, device=weights.device)
        kept_weights = torch.empty((batch, self.kvheads, keep), dtype=torch.float32, device=weights.device)
        new = torch.empty(batch, dtype=torch.int32, device=weights.device)
        dev._check(engine.lib().qh_paged_evict(_live(dev), self._pages, seqs, weights.data_ptr(), weights.stride(0),
                                               weights.stride(1), keep, first, recent, to.data_ptr(), to.stride(0),
                                               to.shape[1], kept.data_ptr(), kept_weights.data_ptr(), new.data_ptr(),
                                               _stream(dev)))
        return kept, kept_weights, new


Plan = collections.namedtuple("Plan", "lengths first slots positions sequences ancestors")


class PagePool:
    """The free pages of caches whose sequences share tables: a stack of page ids
    on the GPU, free [pages] of which the first count[0] are free (both int32;
    None: all pages, the lowest goes first).  They stay the caller's."""

    def __init__(self, device, pages, page, *, free=None, count=None):
        where = torch.device("cuda", device.index)
        _need(0 < pages < 1 << 31 and 0 < page <= 1 << 30, "pages out of range")
        _need((free is None) == (count is None), "free pages and their count go together")
        if free is None:
            free = torch.arange(pages - 1, -1, -1, dtype=torch.int32, device=where)
            count = torch.full((1,), pages, dtype=torch.int32, device=where)
        for t, what, n in ((free, "free pages", pages), (count, "count of free pages", 1)):
            _on(device, t, what, _I32, 1)
            _need(t.shape[0] == n, f"{what}: {n} are needed")
            _apart(t, what)
        self.device, self.pages, self.page, self.free, self.count = device, pages, page, free, count
        self._pool = engine._Pool(free.data_ptr(), count.data_ptr(), pages, page)

    def plan(self, table, held, lengths, grow, n, *, parents=None, out=None):
        """Grows sequences by `grow` tokens (shrinks them where it is negative):
        table [batch][pages] and held [batch], the entries of its rows in use, get pages
        or give them back in place.  One that grows keeps pages held beyond its
        length; with 0 or less all that its new length does not need go back.  n: room
        for new tokens; growth ends with the first sequence that does not fit into n
        or the free pages.  Returns a Plan:
        lengths [batch] (out, which may be lengths; allocated if not given), first
        [batch + 1], and for each of n rows, packed by first, slots (int64: page id * page
        + slot), positions, sequences (-1 behind the last token) and, with parents
        ([n], a tree per sequence: numbers within it, -1 for a root), ancestors
        (int64) for attend_tree, positions then counting a node's depth."""
        dev = self.device
        (batch, pages), strides = _on(dev, table, "page table", _I32, 2)
        for t, what in ((held, "held pages"), (lengths, "lengths"), (grow, "growth")):
            _on(dev, t, what, _I32, 1)
            _need(t.shape[0] == batch, f"{what}: one for each row of the page table")
        for t, what in ((table, "page table"), (held, "held pages")):
            _apart(t, what)
        _need(0 <= n <= 1 << 24, "new tokens out of range")
        if parents is not None:
            _on(dev, parents, "parents", _I32, 1)
            _need(parents.shape[0] == n, "parents: one for each new token")
        if out is None:
            out = torch.empty_like(lengths, memory_format=torch.contiguous_format)
        else:
            _on(dev, out, "new lengths", _I32, 1)
            _need(out.shape[0] == batch, "new lengths: one for each row of the page table")
            _apart(out, "new lengths")
        longs = torch.empty((2 if parents is not None else 1, n), dtype=torch.int64, device=table.device).unbind()
        slots, seen = longs if parents is not None else (longs[0], None)
        first, positions, sequences = torch.empty(batch + 1 + 2 * n, dtype=torch.int32,
                                                  device=table.device).split_with_sizes((batch + 1, n, n))
        plan = Plan(out, first, slots, positions, sequences, seen)
        places = engine._Plan(*(None if t is None else t.data_ptr() for t in plan))
        dev._check(engine.lib().qh_paged_plan(_live(dev), self._pool, table.data_ptr(), strides[0], pages, held.data_ptr(),
                                              lengths.data_ptr(), grow.data_ptr(), batch, n,
                                              None if parents is None else parents.data_ptr(), places, _stream(dev)))
        return plan


def accept(caches, parents, tokens, chosen, table, lengths, first):
    """Accepts drafted tokens after attend_tree: walks each sequence's tree from its
    root (its first new token) to the child whose token ([n]) is the one that the model
    chose ([n]) after the node reached, and moves the accepted nodes' keys and values,
    in all `caches` (PagedCaches of one shape: a model's layers), to the slots behind
    the context.  Returns (new lengths, accepted counts, path [n]: accepted nodes'
    numbers from each sequence's first row on and -1, next tokens)."""
    caches = list(caches)
    _need(caches and all(isinstance(c, PagedCache) for c in caches), "a list of caches is needed")
    dev, cache = caches[0].device, caches[0]
    _need(all(c.device is dev for c in caches), "caches of several devices")
    _need(all(c._writable for c in caches), "a cache whose elements share memory is read only")
    seqs = cache._sequences(table, lengths, None)
    batch = lengths.shape[0]
    for t, what in ((parents, "parents"), (tokens, "drafted tokens"), (chosen, "chosen tokens"), (first, "first tokens")):
        _on(dev, t, what, _I32, 1)
    n = parents.shape[0]
    _need(tokens.shape[0] == n and chosen.shape[0] == n, "a drafted and a chosen token for each node")
    _need(first.shape[0] == batch + 1, "first tokens: one more than sequences is needed")
    held = torch.empty(3 * batch + n, dtype=torch.int32, device=table.device)
    if not batch:
        held.fill_(-1)  # nothing is launched: rows of no sequence
    new, accepted, following, path = held.split_with_sizes((batch, batch, batch, n))
    pages = (engine._Pages * len(caches))(*(c._pages for c in caches))
    dev._check(engine.lib().qh_paged_accept(_live(dev), pages, len(caches), seqs, first.data_ptr(), n, parents.data_ptr(),
                                            tokens.data_ptr(), chosen.data_ptr(), new.data_ptr(), accepted.data_ptr(),
                                            path.data_ptr(), following.data_ptr(), _stream(dev)))
    return new, accepted, path, following


def logprobs(device, logits, targets=None, *, top=0, valid=None):
    """Of rows of logits ([rows][vocab] in f32, f16 or bf16): (log probability of
    targets [rows] or None, entropy [rows], ids [rows][top] of the top
    alternatives and their log probabilities, or None, None).  valid: uint8
    [vocab], ids with 0 read as f32::MIN."""
    _on(device, logits, "logits", KIND, 2)
    rows, vocab = logits.shape
    logp = ids = alt = None
    if targets is not None:
        _on(device, targets, "targets", _I32, 1)
        _need(targets.shape[0] == rows, "targets: one for each row")
        logp = torch.empty(rows, dtype=torch.float32, device=logits.device)
    if valid is not None:
        _on(device, valid, "valid-token mask", (torch.uint8,), 1)
        _need(valid.shape[0] == vocab, "valid-token mask length differs from the vocabulary")
    entropy = torch.empty(rows, dtype=torch.float32, device=logits.device)
    _need(0 <= top <= vocab, "more alternatives than logits")
    if top:
        ids = torch.empty((rows, top), dtype=torch.int32, device=logits.device)
        alt = torch.empty((rows, top), dtype=torch.float32, device=logits.device)
    lib, h = engine.lib(), _live(device)
    need = _BYTES()
    device._check(lib.qh_logprobs_bytes(h, rows, vocab, top, need))
    work = torch.empty(need.value, dtype=torch.uint8, device=logits.device) if need.value else None

    def at(t):
        return None if t is None else t.data_ptr()

    device._check(lib.qh_logprobs(h, logits.data_ptr(), KIND[logits.dtype], rows, vocab, logits.stride(0),
                                  at(targets), at(valid), top, at(logp), entropy.data_ptr(), at(ids), at(alt),
                                  at(work), need.value, _stream(device)))
    return logp, entropy, ids, alt
