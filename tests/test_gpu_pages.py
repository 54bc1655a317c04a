"""Forked, reordered, owned and compacted sequences on the GPU: what every
sequence holds afterwards, bit for bit, against a model that copies rows."""
import random

import numpy as np
import pytest
import torch

import nanoinfer_amd as na
from nanoinfer_amd import _abi

pytestmark = pytest.mark.gpu
PAGE = na.KV_BLOCK


def _kv(fmt, pages=60, seqs=10, ctx=200, n_layer=2, n_head=3, head_dim=64, **kw):
    return na.PagedKv(na.BatchOpts(n_layer=n_layer, n_head=n_head, head_dim=head_dim, kv_blocks=pages, max_seqs=seqs,
                                   n_ctx=ctx, max_rows=1024, q8=fmt == "q8",
                                   block8=fmt == "block8", **kw))


def _grow(kv, s, n, g, stream=None):
    """n rows appended to s."""
    at = kv.seq_len(s)
    kv.reserve(s, at + n)
    shape = (kv.opts.n_layer, n, kv.opts.n_embd)
    k, v = (torch.randn(shape, generator=g, device="cuda") for _ in range(2))
    kv.append([(s, p) for p in range(at, at + n)], k, v, stream=stream)
    kv.commit(s, n)


def _held(kv, s, fmt, n=None):
    """The bits of K and V of every committed position of s, on the host."""
    n = kv.seq_len(s) if n is None else n
    if n == 0:
        return []
    rows = [(s, p) for p in range(n)]
    if fmt == "q8":
        (k, v), (ks, vs) = kv.gather_q8(rows)
        return [x.cpu() for x in (k, v, ks, vs)]
    return [x.cpu() for x in (kv.gather(rows) if fmt == "f16" else kv.gather_values(rows))]


def _equal(a, b):
    return len(a) == len(b) and all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("fmt", ["f16", "q8", "block8"])
@pytest.mark.parametrize("n_head,head_dim,n_layer", [(3, 64, 2), (1, 128, 1), (12, 64, 5)])
@pytest.mark.parametrize("length", [1, 15, 16, 17, 35, 64, 77])
def test_fork_holds_what_its_parent_held(gpu, fmt, n_head, head_dim, n_layer, length):
    g = torch.Generator("cuda").manual_seed(length)
    kv = _kv(fmt, n_head=n_head, head_dim=head_dim, n_layer=n_layer)
    s, other = kv.add_seq(), kv.add_seq()
    _grow(kv, other, 21, g)
    _grow(kv, s, length, g)
    want, aside = _held(kv, s, fmt), _held(kv, other, fmt)
    forks = kv.fork([s, s, other, s])
    for f, w in zip(forks, (want, want, aside, want)):
        assert _equal(_held(kv, f, fmt), w)
    for f in (*forks, s):  # each goes its own way
        _grow(kv, f, 1 + f, g)
    whole = (lambda n: n // PAGE * PAGE) if fmt == "block8" else (lambda n: n)  # (a scale that grows rounds rows again)
    for f, w, n in zip((*forks, s), (want, want, aside, want, want), (length, length, 21, length, length)):
        assert all(torch.equal(x, y[:, :whole(n)]) for x, y in zip(_held(kv, f, fmt, whole(n)), w))
    assert _equal(_held(kv, other, fmt), aside)


@pytest.mark.parametrize("fmt", ["f16", "q8", "block8"])
@pytest.mark.parametrize("seed", range(3))
def test_contents_over_many_calls(gpu, fmt, seed):
    """400 calls; after each the sequences that it touched, at the end all of them."""
    rng, g = random.Random(seed), torch.Generator("cuda").manual_seed(seed)
    kv = _kv(fmt, pages=40, n_head=2)
    want = {}
    for step in range(150):
        op = rng.choice(["grow", "grow", "grow", "fork", "reorder", "reorder", "free", "truncate", "compact"])
        live = list(want)
        try:
            if not live or (op == "grow" and len(live) < 3):
                s = kv.add_seq()
                want[s] = []
                live, op = [s], "grow"
            if op == "grow":
                s, n = rng.choice(live), rng.randint(1, 20)
                try:
                    _grow(kv, s, n, g)
                except na.KvError as e:
                    if e.code != _abi.NI_ERR_SHARED:
                        raise
                    kv.own(s)
                    _grow(kv, s, n, g)
                now = _held(kv, s, fmt)
                old = want[s][0].shape[1] if want[s] else 0
                # (a block's scale that grows rounds the rows before the end's page again)
                same = old if fmt != "block8" else old // PAGE * PAGE
                assert all(torch.equal(x[:, :same], y[:, :same]) for x, y in zip(now, want[s]) if same)
                want[s] = now
            elif op == "fork":
                parents = rng.choices(live, k=rng.randint(1, 3))
                for f, p in zip(kv.fork(parents), parents):
                    want[f] = want[p]
            elif op == "reorder":
                seqs = rng.sample(live, rng.randint(1, len(live)))
                parents = rng.choices(live, k=len(seqs))
                kv.reorder(seqs, parents)
                want.update({s: w for s, w in zip(seqs, [want[p] for p in parents])})
            elif op == "free" and len(live) > 2:
                s = rng.choice(live)
                kv.free_seq(s)
                del want[s]
            elif op == "truncate":
                s = rng.choice(live)
                n = rng.randint(0, kv.seq_len(s))
                kv.truncate(s, n)
                want[s] = [x[:, :n] for x in want[s]] if n else []
            elif op == "compact":
                kv.compact()
        except na.KvError as e:
            assert e.code in (_abi.NI_ERR_NO_SLOT, _abi.NI_ERR_POOL_EXHAUSTED, _abi.NI_ERR_CONTEXT_FULL)
            for s in rng.sample(live, len(live) // 2):
                kv.free_seq(s)
                want.pop(s)
        if step % 10 == 9 or op in ("fork", "reorder", "compact"):
            for s, w in want.items():
                assert _equal(_held(kv, s, fmt), w), (step, op, s)


@pytest.mark.parametrize("fmt", ["f16", "q8"])
def test_rows_past_the_end_and_other_pages_are_left(gpu, fmt):
    """Of a page that a sequence ends in only the rows before the end are written."""
    kv = _kv(fmt, pages=8)
    _, _, n = kv.pools()

    class Pool:
        __cuda_array_interface__ = dict(shape=(n,), typestr="|u1", data=(kv.pools()[0], False), version=2)

    pool = torch.as_tensor(Pool(), device="cuda")
    pool.copy_(torch.randint(0, 256, pool.shape, device="cuda", dtype=torch.uint8))
    s = kv.add_seq()
    kv.reserve(s, 2 * PAGE)
    kv.commit(s, PAGE + 6)
    before = pool.clone().view(2, 8, 3, 2, -1)
    (f,) = kv.fork([s])
    after = pool.view(2, 8, 3, 2, -1)
    src, dst = kv.block_table(s)[1], kv.block_table(f)[1]
    at = np.arange(6 * 128) if fmt == "f16" else np.concatenate([np.arange(6 * 64), 16 * 64 + np.arange(6 * 4)])
    want = before.clone()
    want[:, dst, :, :, at] = before[:, src, :, :, at]
    assert torch.equal(after, want)


def test_many_copies_in_one_call(gpu):
    """More copies than travel with the launch arguments, and pages of several tiles."""
    g = torch.Generator("cuda").manual_seed(1)
    kv = _kv("f16", pages=6600, seqs=3300, ctx=64, n_layer=1, n_head=12)
    s = kv.add_seq()
    _grow(kv, s, 18, g)
    want = _held(kv, s, "f16")
    forks = kv.fork([s] * 3200)
    for f in (forks[0], forks[1600], forks[-1]):
        assert _equal(_held(kv, f, "f16"), want)
    rows = [(f, 17) for f in forks[::8]]
    k, v = kv.gather(rows)
    assert all((k[0, i].cpu() == want[0][0, 17]).all() for i in (0, 5, len(rows) - 1))
    assert bool((k == k[:, :1]).all()) and bool((v == v[:, :1]).all())
    for f in forks[:1600]:
        kv.free_seq(f)
    assert kv.compact() > 1000
    assert _equal(_held(kv, forks[-1], "f16"), want)
    assert kv.block_table(forks[-1])[0] == kv.block_table(s)[0]


def test_calls_on_other_streams_run_in_order(gpu):
    """A fork on one stream, appends and gathers on others, without waiting in between."""
    g = torch.Generator("cuda").manual_seed(2)
    kv = _kv("f16", n_layer=4, n_head=12, ctx=1000, pages=400)
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    s = kv.add_seq()
    _grow(kv, s, 899, g)
    want = _held(kv, s, "f16")
    shape = (4, 1, 768)
    k, v = torch.randn(shape, device="cuda"), torch.randn(shape, device="cuda")
    torch.cuda.synchronize()
    for turn in range(20):
        (f,) = kv.fork([s], stream=a)
        kv.reserve(f, 900)
        kv.append([(f, 899)], k, v, stream=b)
        kv.commit(f, 1)
        kv.reorder([f], [s], stream=a)
        kv.compact(stream=b)
        with torch.cuda.stream(a):
            got = kv.gather([(f, p) for p in range(390, 899)])
        kv.free_seq(f)
        a.synchronize()
        assert all(torch.equal(x.cpu(), y[:, 390:]) for x, y in zip(got, want)), turn


def test_refused_while_capturing(gpu):
    kv = _kv("f16")
    g = torch.Generator("cuda").manual_seed(3)
    s = kv.add_seq()
    _grow(kv, s, 20, g)
    want, table = _held(kv, s, "f16"), kv.block_table(s)
    x = torch.zeros(4, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for call in (lambda: kv.fork([s]), lambda: kv.reorder([s], [s]), lambda: kv.own(s), lambda: kv.compact()):
            with pytest.raises(na.KvError) as e:
                call()
            assert "capturing" in str(e.value)
        x += 1
    for i in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert x.tolist() == [i + 1.0] * 4
    assert kv.block_table(s) == table and not kv.is_live(1)
    assert _equal(_held(kv, s, "f16"), want)


def test_steps_of_forked_sequences(gpu):
    """A prompt forked and continued through steps: attention of every beam over
    its own rows, against the same rows in sequences that share nothing."""
    g = torch.Generator("cuda").manual_seed(4)
    kv, ref = _kv("f16", ctx=100), _kv("f16", ctx=100)
    s, r = kv.add_seq(), [ref.add_seq() for _ in range(3)]
    n, c = 41, 192
    x = [torch.randn((2, n, c), generator=g, device="cuda") for _ in range(3)]
    kv.step([(s, n, 1)], *x)
    for i in r:
        ref.step([(i, n, 1)], *x)
    beams = [s] + kv.fork([s, s])
    for turn in range(20):
        y = [torch.randn((2, 3, c), generator=g, device="cuda") for _ in range(3)]
        out = kv.step([(b, 1, 1) for b in beams], *y)
        want = ref.step([(b, 1, 1) for b in r], *y)
        assert torch.equal(out, want), turn
        if turn % 3 == 2:  # the second continues the first from here on
            kv.reorder(beams, [beams[0], beams[0], beams[2]])
            t = ref.seq_len(r[0])
            k, v = ref.gather([(r[0], p) for p in range(t)])
            ref.append([(r[1], p) for p in range(t)], k.view(torch.float16).float(), v.view(torch.float16).float())
    with pytest.raises(na.KvError) as e:
        kv.truncate(beams[1], 20)
        z = [t[:, :1].contiguous() for t in y]
        kv.append([(beams[1], 20)], z[1], z[2])
    assert e.value.code == _abi.NI_ERR_SHARED
    for call in (lambda: kv.step([(beams[1], 1, 1)], *z), lambda: kv.step_noalloc([(beams[1], 1, 1)], *z)
                 if hasattr(kv, "step_noalloc") else kv.step([(beams[1], 1, 1)], *z),
                 lambda: kv.decode_steps([beams[1]], *[t[None] for t in z]),
                 lambda: kv.append_rotary([(beams[1], 20)], z[1], z[2], na.Rotary(64)),
                 lambda: kv.qkv_append([(beams[1], 20)], torch.zeros((1, 64), device="cuda"),
                                       torch.zeros((576, 64), device="cuda"))):
        with pytest.raises(na.KvError) as e:
            call()
        assert e.value.code == _abi.NI_ERR_SHARED
    kv.own(beams[1])
    kv.step([(beams[1], 1, 1)], *z)
