"""Refusals of the operators on device tensors: the C ABI's checks of its host-side arguments (none
of which needs a GPU: a call that passes them all ends with "null context" here) and the package's
checks of tensors."""
import ctypes as C
import importlib

import pytest
import torch

engine = importlib.import_module("qwen-30brust_amd")
serving = importlib.import_module("qwen-30brust_amd.serving")

A = 1 << 20  # an aligned address that is never read


def message(rc):
    assert rc == 1
    return engine.lib().qh_last_error(None).decode()


def cache(**kw):
    d = dict(k=A, v=A, k_scale=None, v_scale=None, kind=1, page=16, kvheads=2, dim=64, pages=10, page_stride=2048,
             token_stride=128, head_stride=64)
    d.update(kw)
    return engine._Pages(**d)


def seqs(**kw):
    d = dict(table=A, length=A, table_stride=4, table_pages=4, batch=3, most=64)
    d.update(kw)
    return engine._Sequences(**d)


def heads(**kw):
    d = dict(data=A, kind=1, row_stride=256, head_stride=64)
    d.update(kw)
    return engine._Heads(**d)


CACHES = [(dict(k=None), "null cache keys"), (dict(v=A + 1), "cache values is not aligned"), (dict(kind=2), "element kind 2"),
          (dict(kind=12), "element kind 12"), (dict(page=0), "empty cache"), (dict(kvheads=0), "empty cache"),
          (dict(dim=0), "empty cache"), (dict(pages=0), "empty cache"), (dict(dim=257), "at most 256 wide"),
          (dict(pages=1 << 31), "too many pages"), (dict(kind=8), "null cache key scales"),
          (dict(kind=8, k_scale=A, v_scale=A + 1), "cache value scales is not aligned"),
          (dict(kind=8, k_scale=A, v_scale=A, dim=48), "multiples of 32"),
          (dict(kind=8, k_scale=A, v_scale=A, token_stride=129), "multiples of 32"),
          (dict(page_stride=1 << 60), "beyond the address space"), (dict(kvheads=1 << 17), "out of range")]
SEQS = [(dict(length=None), "null lengths"), (dict(table=None), "null page table"), (dict(table=A + 2), "page table is not aligned"),
        (dict(most=65), "hold fewer keys"), (dict(batch=65536), "at most 65535"), (dict(most=(1 << 31) - 1), "too long"),
        (dict(table_stride=1 << 60), "beyond the address space")]


def attention(c=None, s=None, q=None, n=4, out=None, w=None, work=(A, 1 << 30)):
    return engine.lib().qh_paged_attention(None, c or cache(), s or seqs(), q or heads(), n, 1.0, out or heads(), w,
                                           work[0], work[1], None)


def append(c=None, s=None, first=A, n=5, k=None, v=None, more=None):
    return engine.lib().qh_paged_append(None, c or cache(), s or seqs(), first, n, k or heads(), v or heads(), more, None)


def evict(c=None, s=None, w=A, keep=32, first=4, recent=8, to=A, to_pages=2, kept=A, kw=A, new=A):
    return engine.lib().qh_paged_evict(None, c or cache(), s or seqs(), w, 128, 64, keep, first, recent, to, to_pages,
                                       to_pages, kept, kw, new, None)


def logprobs(x=A, kind=0, rows=3, vocab=100, stride=100, target=A, valid=None, top=5, lp=A, h=A, ids=A, alt=A,
             work=(A, 1 << 40)):
    return engine.lib().qh_logprobs(None, x, kind, rows, vocab, stride, target, valid, top, lp, h, ids, alt, work[0],
                                    work[1], None)


def test_calls_that_pass_the_checks():
    for rc in (attention(), append(), evict(), logprobs(), append(first=None, n=3), attention(s=seqs(most=0, table=None)),
               logprobs(target=None, lp=None, h=None, top=0, ids=None, alt=None),
               attention(c=cache(kind=8, k_scale=A, v_scale=A)), attention(q=heads(kind=30))):
        assert message(rc) == "null context"
    # nothing to do
    assert attention(s=seqs(batch=0)) == 0 and append(n=0) == 0 and evict(s=seqs(batch=0)) == 0 and logprobs(rows=0) == 0


@pytest.mark.parametrize("call", [attention, append, evict])
@pytest.mark.parametrize("kw,text", CACHES)
def test_caches(call, kw, text):
    assert text in message(call(c=cache(**kw)))


@pytest.mark.parametrize("call", [attention, append, evict])
@pytest.mark.parametrize("kw,text", SEQS)
def test_sequences(call, kw, text):
    assert text in message(call(s=seqs(**kw)))


@pytest.mark.parametrize("kw,text", [
    (dict(n=3), "multiple of the KV heads"), (dict(n=0), "multiple of the KV heads"), (dict(q=heads(data=None)), "null queries"),
    (dict(q=heads(kind=8)), "element kind 8"), (dict(out=heads(data=A + 1)), "attention outputs is not aligned"),
    (dict(q=heads(row_stride=1 << 60)), "beyond the address space"), (dict(w=engine._KeyWeights(after=None)), "null weight outputs"),
    (dict(w=engine._KeyWeights(before=A + 1, after=A)), "weights is not aligned"), (dict(s=seqs(batch=60000), n=60000), "too many"),
    (dict(w=engine._KeyWeights(after=A), work=(A, 64)), "workspace of 64 bytes"),
    (dict(w=engine._KeyWeights(after=A), work=(None, 1 << 30)), "null workspace"),
    (dict(w=engine._KeyWeights(after=A), work=(A + 4, 1 << 30)), "workspace is not aligned")])
def test_attention(kw, text):
    assert text in message(attention(**kw))


@pytest.mark.parametrize("kw,text", [
    (dict(first=None), "as many tokens as sequences"), (dict(first=A + 1), "first tokens is not aligned"),
    (dict(n=(1 << 24) + 1), "at most 16777216 tokens"), (dict(k=heads(data=None)), "null keys"), (dict(v=heads(kind=8)), "element kind 8"),
    (dict(more=engine._Append(q=heads(), q_out=heads(), heads=3)), "multiple of the KV heads"),
    (dict(more=engine._Append(q=heads(), q_out=heads(data=None), heads=4)), "null query outputs"),
    (dict(more=engine._Append(k_norm=A + 2)), "key norm weights is not aligned"),
    (dict(more=engine._Append(rope=A)), "table of angles out of range"),
    (dict(more=engine._Append(rope=A + 4, rope_rows=5)), "table of angles is not aligned"),
    (dict(more=engine._Append(rope=A, rope_rows=5, position=A + 1)), "positions is not aligned"),
    (dict(c=cache(dim=63), more=engine._Append(rope=A, rope_rows=5)), "even head width"),
    (dict(n=1 << 24, more=engine._Append(q=heads(row_stride=1), q_out=heads(row_stride=1), heads=256)), "too many tokens")])
def test_append(kw, text):
    assert text in message(append(**kw))


@pytest.mark.parametrize("kw,text", [
    (dict(keep=0), "out of range"), (dict(keep=1 << 31), "out of range"), (dict(first=33), "more than those kept"),
    (dict(first=10, recent=23), "more than those kept"), (dict(keep=33), "hold fewer keys than those kept"),
    (dict(w=None), "null weights"), (dict(to=None), "null new pages"), (dict(kept=None), "null kept indexes"),
    (dict(kw=A + 1), "kept weights is not aligned"), (dict(new=None), "null new lengths")])
def test_evict(kw, text):
    assert text in message(evict(**kw))


@pytest.mark.parametrize("kw,text", [
    (dict(x=None), "null logits"), (dict(x=A + 1), "logits is not aligned"), (dict(kind=8), "element kind 8"),
    (dict(vocab=0, top=0), "1 to 16777216"), (dict(vocab=(1 << 24) + 1), "1 to 16777216"), (dict(top=129, vocab=1000), "at most 128"),
    (dict(top=6, vocab=5), "no more than logits"), (dict(target=None), "go together"), (dict(lp=None), "go together"),
    (dict(ids=None), "null alternatives"), (dict(alt=A + 2), "alternatives is not aligned"), (dict(h=A + 1), "entropies is not aligned"),
    (dict(stride=1 << 60), "beyond the address space"), (dict(rows=1 << 32), "too many rows")])
def test_logprobs(kw, text):
    assert text in message(logprobs(**kw))


def test_null_structures():
    lib, size = engine.lib(), C.c_size_t()
    assert "null cache" in message(lib.qh_paged_attention(None, None, seqs(), heads(), 4, 1.0, heads(), None, None, 0, None))
    assert "null sequences" in message(lib.qh_paged_append(None, cache(), None, A, 1, heads(), heads(), None, None))
    assert "null keys" in message(lib.qh_paged_append(None, cache(), seqs(), A, 1, None, heads(), None, None))
    assert "null output" in message(lib.qh_paged_attention_bytes(None, cache(), seqs(), 4, 0, None))
    assert "null output" in message(lib.qh_logprobs_bytes(None, 1, 5, 1, None))
    assert lib.qh_paged_attention_bytes(None, cache(), seqs(), 4, 1, size) == 0 and size.value >= 3 * 4 * 64 * 4
    assert lib.qh_logprobs_bytes(None, 1, 151936, 20, size) == 0


def test_tensors_off_the_device():
    """The package refuses tensors of another device before anything is launched."""
    class Closed:
        index, h = 0, None

    k = torch.zeros(4, 16, 2, 64)
    with pytest.raises(engine.EngineError, match="not a tensor on the engine's device"):
        serving.PagedCache(Closed, k, k)
    with pytest.raises(engine.EngineError, match="not a tensor on the engine's device"):
        serving.logprobs(Closed, torch.zeros(2, 5))
    with pytest.raises(engine.EngineError, match="not a tensor"):
        serving.PagedCache(Closed, [1], k)
