"""Books of shared pages (fork, reorder, own, compact), without a GPU: handles
that keep the books alone, against a model that holds each sequence's pages and
counts."""
import random

import numpy as np
import pytest

import nanoinfer_amd as na
from nanoinfer_amd import _abi

PAGE = na.KV_BLOCK


def _kv(pages=40, seqs=8, ctx=200, **kw):
    return na.PagedKv(na.BatchOpts(n_layer=2, n_head=3, head_dim=64, kv_blocks=pages, max_seqs=seqs, n_ctx=ctx,
                                   max_rows=64, host_only=True, **kw))


def _grow(kv, s, n):
    kv.reserve(s, kv.seq_len(s) + n)
    kv.commit(s, n)


def _check_books(kv):
    held = {}
    for s in range(kv.opts.max_seqs):
        table = kv.block_table(s)
        assert table == [] or kv.is_live(s)
        assert len(set(table)) == len(table)
        for p in table:
            held[p] = held.get(p, 0) + 1
    for p in range(kv.opts.kv_blocks):
        assert kv.page_refs(p) == held.get(p, 0)
    assert kv.blocks_used() == len(held)
    assert kv.free_block_count() == kv.opts.kv_blocks - len(held)


def test_fork_shares_whole_pages_and_takes_one_for_the_end():
    kv = _kv()
    s = kv.add_seq()
    _grow(kv, s, 2 * PAGE + 5)
    kv.reserve(s, 4 * PAGE)  # a page past the end is the parent's alone
    a, b = kv.fork([s, s])
    t = kv.block_table(s)
    assert (a, b) == (1, 2) and len(t) == 4
    for x, page in ((a, 4), (b, 5)):  # handed out in order
        assert kv.seq_len(x) == 2 * PAGE + 5
        assert kv.block_table(x) == t[:2] + [page]
    assert [kv.page_refs(p) for p in t] == [3, 3, 1, 1]
    _check_books(kv)
    kv.free_seq(s)
    assert [kv.page_refs(p) for p in t] == [2, 2, 0, 0]
    _check_books(kv)


@pytest.mark.parametrize("length", [0, PAGE, 3 * PAGE])
def test_fork_of_whole_pages_takes_none(length):
    kv = _kv(pages=4)
    s = kv.add_seq()
    _grow(kv, s, length)
    used = kv.blocks_used()
    forks = kv.fork([s] * 7)
    assert all(kv.block_table(f) == kv.block_table(s) and kv.seq_len(f) == length for f in forks)
    assert kv.blocks_used() == used
    _check_books(kv)


def test_fork_refusals_change_nothing():
    kv = _kv(pages=3, seqs=4)
    s = kv.add_seq()
    _grow(kv, s, PAGE + 1)
    for parents, code in (([s] * 4, _abi.NI_ERR_NO_SLOT), ([s, s], _abi.NI_ERR_POOL_EXHAUSTED), ([s, 2], _abi.NI_ERR_NOT_LIVE),
                          ([s, 9], _abi.NI_ERR_BAD_ARG)):
        with pytest.raises(na.KvError) as e:
            kv.fork(parents)
        assert e.value.code == code
        assert [kv.is_live(x) for x in range(4)] == [True, False, False, False]
        _check_books(kv)
    assert kv.fork([]) == []
    assert len(kv.fork([s])) == 1
    for bad in ([-1], [1 << 32], [0.5]):
        with pytest.raises(ValueError):
            kv.fork(bad)


def test_writes_into_shared_pages_are_refused():
    kv = _kv()
    s = kv.add_seq()
    _grow(kv, s, 2 * PAGE)
    (f,) = kv.fork([s])
    kv.truncate(f, PAGE + 3)  # the end lies inside a page that s holds too
    for call in (lambda: kv.step_begin([(f, 1, 1)]), lambda: kv.step_begin([(s, 1, 1), (f, 2, 1)])):
        with pytest.raises(na.KvError) as e:
            call()
        assert e.value.code == _abi.NI_ERR_SHARED and f"sequence {f}: position {PAGE + 3}" in str(e.value)
    kv.own(f)
    assert kv.block_table(f)[0] != kv.block_table(s)[0] and kv.block_table(f)[1] != kv.block_table(s)[1]
    _check_books(kv)
    kv.step_begin([(f, 1, 1)])
    for call in (lambda: kv.fork([s]), lambda: kv.reorder([s], [f]), lambda: kv.own(s), lambda: kv.compact()):
        with pytest.raises(na.KvError) as e:
            call()
        assert "still open" in str(e.value)
    kv.step_end()
    assert kv.seq_len(f) == PAGE + 4
    # whole shared pages before the end are no obstacle
    kv2 = _kv()
    s = kv2.add_seq()
    _grow(kv2, s, 2 * PAGE + 1)
    (f,) = kv2.fork([s])
    kv2.step_begin([(f, 3, 1), (s, 40, 1)])
    kv2.step_end()
    _check_books(kv2)


def test_own_takes_only_what_is_asked_for():
    kv = _kv(pages=8)
    s = kv.add_seq()
    _grow(kv, s, 4 * PAGE)
    (f,) = kv.fork([s])
    t = kv.block_table(s)
    kv.own(f, PAGE, PAGE)
    assert kv.block_table(f) == t
    kv.own(f, PAGE + 3, 2 * PAGE + 1)
    assert [a == b for a, b in zip(kv.block_table(f), t)] == [True, False, False, True]
    kv.own(f, PAGE, 3 * PAGE)  # its own already
    assert kv.blocks_used() == 6
    _check_books(kv)
    for begin, end in ((2, 1), (0, 4 * PAGE + 1)):
        with pytest.raises(na.KvError) as e:
            kv.own(f, begin, end)
        assert "not all reserved" in str(e.value)
    kv.own(s)
    assert kv.blocks_used() == 8
    (g,) = kv.fork([s])
    with pytest.raises(na.KvError) as e:
        kv.own(g)
    assert e.value.code == _abi.NI_ERR_POOL_EXHAUSTED
    assert kv.block_table(g) == kv.block_table(s)
    _check_books(kv)


def _search(kv, beams, shared, own):
    s = kv.add_seq()
    _grow(kv, s, shared)
    out = [s] + kv.fork([s] * (beams - 1))
    for b in out:
        _grow(kv, b, own)
    return out


def test_reorder_keeps_pages_in_place():
    kv = _kv()
    b = _search(kv, 4, 2 * PAGE + 3, PAGE + 4)  # the end inside page 3
    t = [kv.block_table(x) for x in b]
    kv.reorder(b, [b[0], b[0], b[2], b[2]])
    u = [kv.block_table(x) for x in b]
    assert u[0] == t[0] and u[2] == t[2]
    assert u[1] == t[0][:3] + [t[1][3]] and u[3] == t[2][:3] + [t[3][3]]  # copies into their own last pages
    _check_books(kv)
    kv.reorder(b, [b[0], b[0], b[2], b[2]])
    assert [kv.block_table(x) for x in b] == u
    # every beam replaced: the first continuation takes over the end
    kv.reorder(b, [b[1], b[0], b[1], b[0]])
    v = [kv.block_table(x) for x in b]
    assert v[0] == u[1] and v[1] == u[0] and v[2][:3] == u[1][:3] and v[3][:3] == u[0][:3]
    assert len({x[3] for x in v}) == 4
    _check_books(kv)


def test_reorder_of_other_lengths_and_of_unlisted_parents():
    kv = _kv()
    a, b, c = kv.add_seq(), kv.add_seq(), kv.add_seq()
    _grow(kv, a, 5 * PAGE + 2)
    _grow(kv, b, PAGE)
    kv.reserve(b, 3 * PAGE)
    kv.reorder([b, c], [a, a])
    assert kv.seq_len(b) == kv.seq_len(c) == 5 * PAGE + 2
    assert kv.block_table(b)[:5] == kv.block_table(c)[:5] == kv.block_table(a)[:5]
    assert kv.blocks_used() == 5 + 3
    _check_books(kv)
    d = kv.add_seq()
    kv.reorder([a, b], [d, d])  # an empty sequence
    assert kv.block_table(a) == [] and kv.seq_len(b) == 0
    _check_books(kv)


def test_reorder_refusals_change_nothing():
    kv = _kv(pages=4, seqs=4)
    a, b, c = kv.add_seq(), kv.add_seq(), kv.add_seq()
    _grow(kv, a, 3 * PAGE + 1)
    for seqs, parents, text in (([b, b], [a, a], "twice"), ([b, 3], [a, a], "not live"), ([b], [3], "not live"),
                                ([7], [a], "out of range"), ([b, c], [a, a], "exhausted")):
        with pytest.raises(na.KvError) as e:
            kv.reorder(seqs, parents)
        assert text in str(e.value)
        assert kv.block_table(b) == [] and kv.seq_len(b) == 0
        _check_books(kv)
    with pytest.raises(ValueError):
        kv.reorder([a], [a, b])
    kv.reorder([], [])


@pytest.mark.parametrize("order", [None, "shuffled"])
def test_compact_moves_pages_to_the_front(order):
    n = 20
    first = list(range(n))
    if order:
        random.Random(3).shuffle(first)
    kv = _kv(pages=n, page_order=first if order else None)
    s = [kv.add_seq() for _ in range(4)]
    for x in s:
        _grow(kv, x, 3 * PAGE + 2)
    (f,) = kv.fork([s[3]])
    kv.free_seq(s[0])
    kv.free_seq(s[2])
    before = {x: kv.block_table(x) for x in (s[1], s[3], f)}
    moved = kv.compact()
    used = kv.blocks_used()
    assert used == 4 + 4 + 1 and moved == sum(p != q for t, u in ((t, kv.block_table(x)) for x, t in before.items())
                                              for p, q in zip(t, u)) - 3  # three pages are held twice
    where = {}
    for x, t in before.items():
        for p, q in zip(t, kv.block_table(x)):
            assert where.setdefault(p, q) == q  # shared pages move once
    assert sorted(first.index(q) for q in where.values()) == list(range(used))
    for p, q in where.items():
        if first.index(p) < used:
            assert p == q
    _check_books(kv)
    assert kv.compact() == 0
    x = kv.add_seq()
    _grow(kv, x, 2 * PAGE)  # handed out in order again
    assert kv.block_table(x) == first[used:used + 2]
    _check_books(kv)


@pytest.mark.parametrize("seed", range(6))
def test_books_hold_over_many_calls(seed):
    rng = random.Random(seed)
    kv = _kv(pages=30, seqs=9, ctx=150)
    for _ in range(400):
        live = [s for s in range(9) if kv.is_live(s)]
        op = rng.choice(["add", "grow", "grow", "fork", "reorder", "reorder", "free", "truncate", "own", "compact"])
        try:
            if op == "add" or not live:
                kv.add_seq()
            elif op == "grow":
                _grow(kv, rng.choice(live), rng.randint(0, 40))
            elif op == "fork":
                kv.fork(rng.choices(live, k=rng.randint(1, 3)))
            elif op == "reorder":
                seqs = rng.sample(live, rng.randint(1, len(live)))
                parents = rng.choices(live, k=len(seqs))
                want = [(kv.seq_len(p), kv.block_table(p)) for p in parents]
                kv.reorder(seqs, parents)
                for s, (n, t) in zip(seqs, want):
                    assert kv.seq_len(s) == n and kv.block_table(s)[:n // PAGE] == t[:n // PAGE]
            elif op == "free":
                kv.free_seq(rng.choice(live))
            elif op == "truncate":
                s = rng.choice(live)
                kv.truncate(s, rng.randint(0, kv.seq_len(s)))
            elif op == "own":
                kv.own(rng.choice(live))
            else:
                kv.compact()
        except na.KvError as e:
            assert e.code in (_abi.NI_ERR_NO_SLOT, _abi.NI_ERR_POOL_EXHAUSTED, _abi.NI_ERR_CONTEXT_FULL)
        _check_books(kv)


def test_null_arguments():
    kv = _kv()
    L, h = kv._L, kv.handle
    assert L.ni_kv_fork(h, None, 1, None, None) == _abi.NI_ERR_BAD_ARG
    assert L.ni_kv_reorder(h, None, None, 1, None) == _abi.NI_ERR_BAD_ARG
    assert L.ni_kv_fork(h, None, 0, None, None) == _abi.NI_OK
    assert L.ni_kv_compact(h, None, None) == _abi.NI_OK
    assert L.ni_kv_own(h, 0, 0, 0, None) == _abi.NI_ERR_NOT_LIVE
    with pytest.raises(ValueError):
        kv.page_refs(40)
    assert np.array(kv.fork(np.zeros((0,), np.int64))).size == 0
