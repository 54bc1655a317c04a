"""Reordered sequences whose ends lie in pages that others hold too, without a
GPU: every continuation can grow, as after a fork."""
import random

import pytest

import nanoinfer_amd as na
from nanoinfer_amd import _abi
from test_page_sharing import PAGE, _check_books, _grow, _kv


def _step(kv, *seqs):
    kv.step_begin([(s, 1, 1) for s in seqs])
    kv.step_end()


@pytest.mark.parametrize("listed", [False, True])
def test_an_end_inside_a_shared_page_is_copied(listed):
    """p was truncated into a page that another sequence holds: its continuation gets a page of its own."""
    kv = _kv()
    whole = kv.add_seq()
    _grow(kv, whole, 3 * PAGE)
    p, c = kv.fork([whole, whole])
    kv.truncate(p, PAGE + 5)
    shared = kv.block_table(p)[1]
    seqs, parents = ([c, p], [p, c]) if not listed else ([c, p, whole], [p, c, whole])
    kv.reorder(seqs, parents)
    assert kv.seq_len(c) == PAGE + 5 and kv.block_table(c)[0] == kv.block_table(whole)[0]
    assert kv.block_table(c)[1] != shared and kv.page_refs(kv.block_table(c)[1]) == 1
    _check_books(kv)
    _step(kv, c, p)
    assert kv.block_table(p)[:3] == kv.block_table(whole)
    _check_books(kv)


def test_two_ends_in_one_page():
    """Two sequences end in the same page, both are replaced: one continuation keeps it, the other gets a copy."""
    kv = _kv()
    a = kv.add_seq()
    _grow(kv, a, 2 * PAGE)
    (b,) = kv.fork([a])
    c, d = kv.add_seq(), kv.add_seq()
    kv.truncate(a, PAGE + 3)
    kv.truncate(b, PAGE + 9)
    page = kv.block_table(a)[1]
    kv.reorder([a, b, c, d], [c, d, a, b])
    assert [kv.seq_len(x) for x in (a, b, c, d)] == [0, 0, PAGE + 3, PAGE + 9]
    assert kv.block_table(c)[1] == page != kv.block_table(d)[1] and kv.page_refs(page) == 1
    _check_books(kv)
    _step(kv, c, d)
    _check_books(kv)


def test_a_whole_page_of_one_is_the_end_of_another():
    """Both go on elsewhere: the page stays with the one that holds it whole."""
    kv = _kv()
    a = kv.add_seq()
    _grow(kv, a, 2 * PAGE)
    (b,) = kv.fork([a])
    kv.truncate(b, PAGE + 9)
    page = kv.block_table(a)[1]
    kv.reorder([a, b], [b, a])
    assert kv.block_table(b)[1] == page != kv.block_table(a)[1] and kv.page_refs(page) == 1
    _check_books(kv)
    _step(kv, a, b)
    _check_books(kv)


def test_no_page_for_the_copy():
    kv = _kv(pages=2)
    whole = kv.add_seq()
    _grow(kv, whole, 2 * PAGE)
    p, c = kv.fork([whole, whole])
    kv.truncate(p, PAGE + 5)
    before = [kv.block_table(s) for s in (whole, p, c)]
    with pytest.raises(na.KvError) as e:
        kv.reorder([c, p], [p, c])
    assert e.value.code == _abi.NI_ERR_POOL_EXHAUSTED
    assert [kv.block_table(s) for s in (whole, p, c)] == before
    _check_books(kv)


@pytest.mark.parametrize("seed", range(4))
def test_continuations_grow_after_any_calls(seed):
    """Replaced sequences can always take a step, unless the pool is empty; pages are counted."""
    rng = random.Random(seed)
    kv = _kv(pages=40, seqs=8, ctx=150)
    for _ in range(300):
        live = [s for s in range(8) if kv.is_live(s)]
        op = rng.choice(["add", "grow", "fork", "fork", "reorder", "reorder", "reorder", "free", "truncate", "truncate"])
        try:
            if op == "add" or not live:
                kv.add_seq()
            elif op == "grow":
                s = rng.choice(live)
                kv.own(s)
                _grow(kv, s, rng.randint(0, 30))
            elif op == "fork":
                kv.fork(rng.choices(live, k=rng.randint(1, 3)))
            elif op == "reorder":
                seqs = rng.sample(live, rng.randint(1, len(live)))
                parents = rng.choices(live, k=len(seqs))
                lengths = [kv.seq_len(p) for p in parents]
                kv.reorder(seqs, parents)
                assert [kv.seq_len(s) for s in seqs] == lengths
                _check_books(kv)
                changed = [s for s, p in zip(seqs, parents) if s != p]
                if changed:
                    _step(kv, *changed)
            elif op == "free":
                kv.free_seq(rng.choice(live))
            else:
                s = rng.choice(live)
                kv.truncate(s, rng.randint(0, kv.seq_len(s)))
        except na.KvError as e:
            assert e.code in (_abi.NI_ERR_NO_SLOT, _abi.NI_ERR_POOL_EXHAUSTED, _abi.NI_ERR_CONTEXT_FULL)
        _check_books(kv)
