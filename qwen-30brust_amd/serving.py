"""Operators on torch tensors of the GPU, for a program that serves several
sequences: a key-value cache held in pages (`PagedCache`: append, attend, evict)
and the log probabilities of tokens (`logprobs`), over the C ABI's entry points
for device tensors (include/qwen_hip.h: qh_paged_*, qh_logprobs).

Every call runs on torch's current stream of the tensors' device, which is the
given engine Device's, returns at once, and may be captured into a graph.  What
it allocates (outputs that are not given, workspaces) comes from torch's
allocator.  Arguments on the host are checked (EngineError); lengths, page ids
and targets lie on the device and are checked there: the header says what a call
does with those out of range.  Nothing here has a gradient: a tensor that requires
one is refused where torch records gradients (call under torch.no_grad()).

    serving = importlib.import_module("qwen-30brust_amd.serving")
"""
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
