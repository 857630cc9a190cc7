"""Refusals of the operators for several new tokens per sequence: the C ABI's checks of its host-side arguments (none
of which needs a GPU: a call that passes them all ends with "null context" here)."""
import ctypes as C
import importlib

import pytest

from test_serving import A, CACHES, SEQS, cache, heads, message, seqs

engine = importlib.import_module("qwen-30brust_amd")


def prompts(c=None, s=None, first=A, n=5, q=None, h=4, out=None, work=(A, 1 << 40)):
    return engine.lib().qh_paged_prompts(None, c or cache(), s or seqs(), first, n, q or heads(), h, 1.0, out or heads(), work[0],
                                         work[1], None)


def tree(c=None, s=None, first=A, n=5, ancestors=A, q=None, h=4, out=None, work=(A, 1 << 40)):
    return engine.lib().qh_paged_tree(None, c or cache(), s or seqs(), first, n, ancestors, q or heads(), h, 1.0, out or heads(),
                                      work[0], work[1], None)


def accept(c=None, layers=1, s=None, first=1 * A, n=5, parents=2 * A, tokens=3 * A, chosen=4 * A, new=5 * A, accepted=6 * A,
           path=7 * A, following=8 * A):
    return engine.lib().qh_paged_accept(None, c or cache(), layers, s or seqs(), first, n, parents, tokens, chosen, new, accepted,
                                        path, following, None)


def pool(**kw):
    d = dict(free=11 * A, count=12 * A, pages=100, page=16)
    d.update(kw)
    return engine._Pool(**d)


def places(**kw):
    d = dict(length=13 * A, first=14 * A, slot=15 * A, position=16 * A, sequence=17 * A, ancestors=None)
    d.update(kw)
    return engine._Plan(**d)


def plan(p=None, table=1 * A, stride=8, pages=8, held=2 * A, length=3 * A, grow=4 * A, batch=3, n=20, parents=None, out=None):
    return engine.lib().qh_paged_plan(None, p or pool(), table, stride, pages, held, length, grow, batch, n, parents,
                                      out or places(), None)


def test_calls_that_pass_the_checks():
    two = (engine._Pages * 2)(cache(), cache(k=9 * A))
    for rc in (prompts(), tree(), accept(), plan(), accept(c=two, layers=2), plan(parents=5 * A, out=places(ancestors=6 * A)),
               plan(out=places(length=3 * A)), plan(out=places(slot=None, position=None, sequence=None)),
               plan(batch=0, table=None, held=None, length=None, grow=None), prompts(q=heads(kind=30)), tree(s=seqs(most=0, table=None)),
               accept(n=0, parents=None, tokens=None, chosen=None, path=None)):
        assert message(rc) == "null context"
    # nothing to do
    assert prompts(n=0) == 0 and prompts(s=seqs(batch=0)) == 0 and tree(n=0, ancestors=None) == 0 and accept(s=seqs(batch=0)) == 0


@pytest.mark.parametrize("call", [prompts, tree, accept])
@pytest.mark.parametrize("kw,text", CACHES)
def test_caches(call, kw, text):
    assert text in message(call(c=cache(**kw)))


@pytest.mark.parametrize("call", [prompts, tree, accept])
@pytest.mark.parametrize("kw,text", SEQS)
def test_sequences(call, kw, text):
    assert text in message(call(s=seqs(**kw)))


@pytest.mark.parametrize("call", [prompts, tree])
@pytest.mark.parametrize("kw,text", [
    (dict(h=3), "multiple of the KV heads"), (dict(h=0), "multiple of the KV heads"), (dict(q=heads(data=None)), "null queries"),
    (dict(q=heads(kind=8)), "element kind 8"), (dict(out=heads(data=A + 1)), "attention outputs is not aligned"),
    (dict(q=heads(row_stride=1 << 60)), "beyond the address space"), (dict(first=None), "null first tokens"),
    (dict(first=A + 2), "first tokens is not aligned"), (dict(n=(1 << 24) + 1), "at most 16777216 tokens"),
    (dict(n=1 << 24, h=256, q=heads(row_stride=1), out=heads(row_stride=1)), "too many tokens and heads")])
def test_attention(call, kw, text):
    assert text in message(call(**kw))


def test_tree():
    assert "null ancestors" in message(tree(ancestors=None))
    assert "ancestors is not aligned" in message(tree(ancestors=A + 4))
    size = C.c_size_t()
    assert "null output" in message(engine.lib().qh_paged_prompts_bytes(None, cache(), seqs(), 5, 4, None))
    assert "multiple of the KV heads" in message(engine.lib().qh_paged_prompts_bytes(None, cache(), seqs(), 5, 5, size))
    assert engine.lib().qh_paged_prompts_bytes(None, cache(), seqs(), 5, 4, size) == 0


@pytest.mark.parametrize("kw,text", [
    (dict(layers=0), "no caches"), (dict(c=(engine._Pages * 2)(cache(), cache(kind=30)), layers=2), "differ"),
    (dict(c=(engine._Pages * 2)(cache(), cache(page_stride=4096)), layers=2), "differ"),
    (dict(c=(engine._Pages * 2)(cache(), cache(k=None)), layers=2), "null cache keys"), (dict(first=None), "null first tokens"),
    (dict(parents=None), "null parents"), (dict(tokens=A + 1), "drafted tokens is not aligned"), (dict(chosen=None), "null chosen"),
    (dict(path=None), "null path"), (dict(new=None), "null new lengths"), (dict(accepted=None), "null accepted"),
    (dict(following=A + 2), "next tokens is not aligned"), (dict(n=(1 << 24) + 1), "at most 16777216 tokens"),
    (dict(new=A), "overlap"), (dict(path=2 * A + 16), "overlap"), (dict(accepted=5 * A + 8), "overlap")])
def test_accept(kw, text):
    assert text in message(accept(**kw))


@pytest.mark.parametrize("kw,text", [
    (dict(p=pool(free=None)), "null free pages"), (dict(p=pool(count=A + 1)), "not aligned"), (dict(p=pool(pages=0)), "empty pool"),
    (dict(p=pool(page=0)), "empty pool"), (dict(p=pool(pages=1 << 31)), "too many pages"), (dict(p=pool(page=1 << 31)), "out of range"),
    (dict(batch=65536), "at most 65535"), (dict(n=(1 << 24) + 1), "at most 16777216"), (dict(pages=0), "empty page table"),
    (dict(table=None), "null page table"), (dict(held=None), "null held"), (dict(length=None), "null lengths"),
    (dict(grow=A + 2), "growth is not aligned"), (dict(stride=7), "rows overlap"), (dict(stride=1 << 60), "beyond the address"),
    (dict(pages=1 << 30, stride=1 << 30), "page table out of range"), (dict(p=pool(page=1 << 30)), "too many keys"),
    (dict(out=places(length=None)), "null new lengths"), (dict(out=places(first=None)), "null first tokens"),
    (dict(out=places(slot=A + 4)), "slots is not aligned"), (dict(out=places(ancestors=A)), "go with parents"),
    (dict(parents=A + 1), "parents is not aligned"), (dict(out=places(length=3 * A + 4)), "overlap"),
    (dict(out=places(first=1 * A)), "overlap"), (dict(held=11 * A), "overlap"), (dict(out=places(slot=16 * A)), "overlap")])
def test_plan(kw, text):
    assert text in message(plan(**kw))


@pytest.mark.parametrize("call", [prompts, tree])
def test_workspace(call):
    size = C.c_size_t()
    assert engine.lib().qh_paged_prompts_bytes(None, cache(), seqs(), 5, 4, size) == 0 and size.value > 0
    assert "null workspace" in message(call(work=(None, size.value)))
    assert "workspace is not aligned" in message(call(work=(A + 8, size.value)))
    assert "bytes, " in message(call(work=(A, 0)))
    assert message(call(work=(A, size.value))) == "null context"


@pytest.mark.parametrize("call", [prompts, tree])
def test_more_work_than_is_counted(call):
    pages = 1 << 26
    big = dict(s=seqs(batch=1, table_pages=pages, table_stride=pages, most=(1 << 30) - 1))
    assert message(call(c=cache(kvheads=1), n=1 << 23, h=250, **big)) == "too many tokens, heads and keys"
    assert message(call(c=cache(kvheads=1), n=1 << 23, h=32, **big)) == "null context"


def test_one_cache_twice():
    three = (engine._Pages * 3)(cache(), cache(k=9 * A, v=10 * A), cache())
    assert message(accept(c=three, layers=3)) == "a cache is given twice"
    assert message(accept(c=three, layers=2)) == "null context"


def test_null_structures():
    lib = engine.lib()
    assert "null cache" in message(lib.qh_paged_prompts(None, None, seqs(), A, 5, heads(), 4, 1.0, heads(), None, 0, None))
    assert "null sequences" in message(lib.qh_paged_tree(None, cache(), None, A, 5, A, heads(), 4, 1.0, heads(), None, 0, None))
    assert "null pool" in message(lib.qh_paged_plan(None, None, A, 8, 8, A, A, A, 3, 5, None, places(), None))
    assert "null plan" in message(lib.qh_paged_plan(None, pool(), A, 8, 8, A, A, A, 3, 5, None, None, None))
    assert "null cache" in message(lib.qh_paged_accept(None, None, 1, seqs(), A, 5, A, A, A, A, A, A, A, None))
