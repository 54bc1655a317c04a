"""The block-scaled cache (8-bit floats, a power-of-two scale for each page and
head) on the GPU: appends bit for bit against the rule written out on the
host, attention against 64 bits on what the cache holds."""
import math
import random

import numpy as np
import pytest
import torch

import nanoinfer_amd as na
from nanoinfer_amd import _abi

pytestmark = pytest.mark.gpu
PAGE = na.KV_BLOCK


def _kv(n_layer=2, n_head=3, head_dim=64, pages=64, seqs=6, ctx=600, max_rows=1024, **kw):
    return na.PagedKv(na.BatchOpts(n_layer=n_layer, n_head=n_head, head_dim=head_dim, kv_blocks=pages, max_seqs=seqs,
                                   n_ctx=ctx, max_rows=max_rows, block8=True, **kw))


class Model:
    """What blocks hold: [n_layer, n_head, 16, head_dim] values and their scale's exponent, by (sequence, page of it)."""

    def __init__(self, n_layer, n_head, head_dim):
        self.shape, self.blocks = (n_layer, n_head, PAGE, head_dim), {}

    @staticmethod
    def need(top):
        e = torch.full(top.shape, -117, dtype=torch.int64)
        for i, t in enumerate(top.flatten().tolist()):
            while t > 448.0 * 2.0 ** int(e.view(-1)[i]):
                e.view(-1)[i] += 1
        return e

    @staticmethod
    def e4m3(x):
        return x.clamp(-448, 448).float().to(torch.float8_e4m3fn).double()

    def append(self, rows, x):
        """x [n_layer, n, n_head * head_dim]; rows of one block go in together."""
        n_layer, n_head, _, d = self.shape
        x = x.cpu().double()
        x = torch.nan_to_num(x, nan=0.0, posinf=math.inf, neginf=-math.inf).view(n_layer, -1, n_head, d)
        by = {}
        for i, (s, p) in enumerate(rows):
            by.setdefault((s, p // PAGE), []).append((p % PAGE, i))
        for key, new in by.items():
            values, e = self.blocks.get(key, (torch.zeros(self.shape, dtype=torch.float64),
                                              torch.full(self.shape[:2], -1000, dtype=torch.int64)))
            slots, at = [a for a, _ in new], [b for _, b in new]
            y = x[:, at].transpose(1, 2)
            top = torch.where(y.abs() < math.inf, y.abs(), 0.0).amax((-1, -2))
            now = self.need(top) if 0 in slots else torch.maximum(e, self.need(top))
            by2 = torch.exp2((e - now).double())[..., None, None]
            values = torch.where(by2 == 1, values, self.e4m3(values * by2)) if 0 not in slots else values.clone()
            values[:, :, slots] = self.e4m3(y * torch.exp2(-now.double())[..., None, None])
            self.blocks[key] = (values, now)

    def values(self, rows):
        out = [(self.blocks[s, p // PAGE][0] * torch.exp2(self.blocks[s, p // PAGE][1].double())[..., None, None])[:, :, p % PAGE]
               for s, p in rows]
        return torch.stack(out, 1).flatten(2)


def _check(kv, models, rows):
    """Rows the cache holds, exactly."""
    for layer in (na.ALL_LAYERS, kv.opts.n_layer - 1):
        for got, m in zip(kv.gather_values(rows, layer=layer), models):
            want = m.values(rows)
            want = want if layer == na.ALL_LAYERS else want[layer]
            assert torch.equal(got.cpu().double(), want)


@pytest.mark.parametrize("n_layer,n_head,head_dim", [(2, 3, 64), (1, 1, 128), (3, 2, 128)])
@pytest.mark.parametrize("scale", [1.0, 1e-34, 1e33])
@pytest.mark.parametrize("ragged", [False, True])
def test_appends(gpu, n_layer, n_head, head_dim, scale, ragged):
    """Rows of several sequences, one or many at a time, whose size changes from row to row."""
    rng, g = random.Random(int(ragged) + head_dim), torch.Generator("cuda").manual_seed(head_dim)
    kv = _kv(n_layer, n_head, head_dim)
    c = n_head * head_dim
    models = [Model(n_layer, n_head, head_dim) for _ in range(2)]
    seqs = [kv.add_seq() for _ in range(3)]
    length = {s: 0 for s in seqs}
    for s in seqs:
        kv.reserve(s, 120)
    for _ in range(14):
        rows = []
        for s in rng.sample(seqs, rng.randint(1, 3)):
            n = rng.choice([1, 1, 2, 5, 16, 23]) if ragged else 1
            n = min(n, 120 - length[s])
            rows += [(s, length[s] + i) for i in range(n)]
            length[s] += n
        if not rows:
            continue
        x = [torch.randn((n_layer, len(rows), c), generator=g, device="cuda") *
             torch.exp2(torch.randint(-6, 7, (1, len(rows), 1), generator=g, device="cuda")) * scale for _ in range(2)]
        x[1][:, :, :head_dim] *= 0  # (a head of zeros)
        kv.append(rows, *x)
        for m, y in zip(models, x):
            m.append(rows, y)
        _check(kv, models, [(s, p) for s in seqs for p in range(length[s])])


def test_append_order_rewrites_and_other_rows(gpu):
    """Rows in any order, positions written again, a page that begins anew."""
    g = torch.Generator("cuda").manual_seed(3)
    kv = _kv(n_head=2, pages=20)
    models = [Model(2, 2, 64) for _ in range(2)]
    a, b = kv.add_seq(), kv.add_seq()
    for s in (a, b):
        kv.reserve(s, 3 * PAGE)

    def put(rows, size):
        x = [torch.randn((2, len(rows), 128), generator=g, device="cuda") * size for _ in range(2)]
        kv.append(rows, *x)
        for m, y in zip(models, x):
            m.append(rows, y)

    every = [(s, p) for s in (a, b) for p in range(3 * PAGE)]
    put(every, 1.0)
    mixed = every[::]
    random.Random(1).shuffle(mixed)
    put(mixed, 3.0)
    _check(kv, models, every)
    put([(b, 20), (a, 5), (b, 17), (a, 4)], 100.0)  # grows; the other rows of the pages are rounded again
    _check(kv, models, every)
    put([(a, 7), (a, 6)], 0.001)  # never shrinks
    _check(kv, models, every)
    put([(a, p) for p in range(PAGE)], 0.01)  # anew
    _check(kv, models, every)
    layer = [torch.randn((1, 128), generator=g, device="cuda") * 500 for _ in range(2)]
    before = kv.gather_values(every, layer=0)
    kv.append([(b, 40)], *layer, layer=1)  # one layer only
    after = kv.gather_values(every, layer=0)
    assert all(torch.equal(x, y) for x, y in zip(before, after))
    with pytest.raises(na.KvError) as e:
        kv.append([(a, 3), (b, 3), (a, 3)], *[torch.zeros((2, 3, 128), device="cuda")] * 2)
    assert "twice" in str(e.value)


def test_append_of_no_numbers(gpu):
    g = torch.Generator("cuda").manual_seed(4)
    kv = _kv(n_layer=1, n_head=1)
    models = [Model(1, 1, 64) for _ in range(2)]
    s = kv.add_seq()
    kv.reserve(s, 32)
    x = [torch.randn((1, 20, 64), generator=g, device="cuda") for _ in range(2)]
    for y in x:
        y[0, 3, 5], y[0, 4, 6], y[0, 5, 7] = math.nan, math.inf, -math.inf
        y[0, 17] = math.nan
    rows = [(s, p) for p in range(20)]
    kv.append(rows, *x)
    for m, y in zip(models, x):
        m.append(rows, y)
    _check(kv, models, rows)
    k, _ = kv.gather_values(rows)
    assert k[0, 3, 5] == 0 and bool(torch.isfinite(k).all()) and k[0, 4, 6] == -k[0, 5, 7] > 3


def test_strided_inputs_and_graphs(gpu):
    """k, v and q as views of one buffer, one layer at a time; the calls captured and replayed."""
    g = torch.Generator("cuda").manual_seed(5)
    kv, eager = _kv(), _kv()
    c, n = 192, 7
    for x in (kv, eager):
        s = x.add_seq()
        x.reserve(s, 100)
    held = [torch.randn((2, 90, c), generator=g, device="cuda") for _ in range(2)]
    for x in (kv, eager):
        x.append([(0, p) for p in range(90)], *held)
    fused = torch.randn((2, n, 3 * c), generator=g, device="cuda")
    q, k, v = fused.split(c, -1)
    rows = [(0, 90 + i) for i in range(n)]
    out = torch.empty((2, n, c), device="cuda")

    def step(x, out):
        x.append(rows, k, v)
        x.attention(q, rows, out=out)

    step(kv, out)  # (partials of the size)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(kv, out)
    want = torch.empty_like(out)
    for turn in range(4):
        fused.copy_(torch.randn(fused.shape, generator=g, device="cuda"))
        out.zero_()
        graph.replay()
        step(eager, want)
        torch.cuda.synchronize()
        assert torch.equal(out, want), turn
        one = [eager.attention(q[i], rows, layer=i) for i in range(2)]
        assert torch.equal(torch.stack(one), want)


def _exact(kv, q, rows, group, prefixes=()):
    """(attention in 64 bits over what the cache holds, a bound of the kernel's error)."""
    d, h = kv.opts.head_dim, kv.opts.n_head
    stored = {}

    def keys(s, n):
        if (s, n) not in stored:
            stored[s, n] = [x.double().view(kv.opts.n_layer, n, h, d) for x in kv.gather_values([(s, p) for p in range(n)])]
        return stored[s, n]

    ends = {}
    for s, p in rows:
        ends[s] = max(ends.get(s, 0), p + 1)
    front = []
    for s, n, count in prefixes:
        front += [(s, n)] * count
    front = front or [(0, 0)] * len(rows)
    out, bound = torch.empty_like(q, dtype=torch.float64), torch.empty_like(q, dtype=torch.float64)
    for i, ((s, p), (ps, pn)) in enumerate(zip(rows, front)):
        k, v = (x[:, :p + 1] for x in keys(s, ends[s]))
        if pn:
            pk, pv = keys(ps, pn)
            k, v = torch.cat([pk, k], 1), torch.cat([pv, v], 1)
        x = q[:, i].double().view(-1, h, group, d)
        score = (x[:, None] * k[:, :, :, None]).sum(-1) / math.sqrt(d)  # [layer, key, head, group]
        size = (x[:, None] * k[:, :, :, None]).abs().sum(-1).amax(1) / math.sqrt(d)
        w = torch.softmax(score, 1)
        out[:, i] = (w[..., None] * v[:, :, :, None]).sum(1).flatten(1)
        # Scores: q in two f16 parts (2^-22, and 2^-25 of the scale of its parts below their normal range), d
        # products added in f32 one after another at worst, the scaled sum rounded and taken relative to the reference.
        ds = size * (2.0 ** -21 + (d + 8) * 2.0 ** -24) + 2.0 ** -22 * k.abs().amax((1, 3))[..., None] * math.sqrt(d)
        # Weights in two f16 parts and through exp2 (2^-21 in all, and 2^-37 of the largest each), sums of the keys
        # of a lane or a wave and their joining in f32; the scores' error moves every weight twice.
        n = k.shape[1]
        rel = 2 * ds + 2.0 ** -20 + (n / 32 + 80) * 2.0 ** -24 + n * 2.0 ** -36
        bound[:, i] = (rel * v.abs().amax((1, 3))[..., None])[..., None].expand(-1, -1, -1, d).flatten(1)
    return out, bound


def _filled(kv, lengths, g, loud=0.05):
    c = kv.opts.n_embd
    for n in lengths:
        s = kv.add_seq()
        kv.reserve(s, max(n, 1))
        for at in range(0, n, kv.opts.max_rows // PAGE * PAGE):
            m = min(n - at, kv.opts.max_rows // PAGE * PAGE)
            x = [torch.randn((kv.opts.n_layer, m, c), generator=g, device="cuda") *
                 (1 + 5 * (torch.rand((c,), generator=g, device="cuda") < loud)) for _ in range(2)]
            kv.append([(s, at + p) for p in range(m)], *x)
        kv.commit(s, n)


@pytest.mark.parametrize("n_layer,n_head,head_dim,group", [(2, 3, 64, 1), (1, 2, 128, 4), (1, 1, 64, 7), (3, 2, 128, 1),
                                                           (1, 2, 64, 16), (1, 1, 128, 40)])
@pytest.mark.parametrize("rows_each", [1, 2, 5, 17, 40])
@pytest.mark.parametrize("split", [0, 16, 64])
def test_attention(gpu, n_layer, n_head, head_dim, group, rows_each, split):
    g = torch.Generator("cuda").manual_seed(head_dim + rows_each)
    lengths = [rows_each, rows_each + 1, 40, 47, 48, 49, 130, 277]
    kv = _kv(n_layer, n_head, head_dim, seqs=len(lengths), ctx=600)
    _filled(kv, lengths, g)
    rows = [(s, n - rows_each + i) for s, n in enumerate(lengths) for i in range(rows_each)]
    q = torch.randn((n_layer, len(rows), n_head * group * head_dim), generator=g, device="cuda") * 1.5
    out = kv.prefix_attention(q, rows, [(0, 0, len(rows))], split_tokens=split)
    want, bound = _exact(kv, q, rows, group)
    assert bool(((out.double() - want).abs() <= bound).all())
    if group == 1:
        assert torch.equal(kv.attention(q, rows, split_tokens=split), out)
    if n_layer == 1:
        assert torch.equal(kv.prefix_attention(q[0], rows, [(0, 0, len(rows))], layer=0, split_tokens=split), out[0])


@pytest.mark.parametrize("head_dim,group", [(64, 1), (128, 4)])
def test_long_contexts(gpu, head_dim, group):
    g = torch.Generator("cuda").manual_seed(7)
    lengths = [1, 16, 5000, 9001]
    kv = _kv(1, 2, head_dim, pages=1000, seqs=4, ctx=9100, max_rows=9100)
    _filled(kv, lengths, g)
    rows = [(s, n - 1) for s, n in enumerate(lengths)] + [(3, p) for p in (0, 15, 16, 4000)]
    q = torch.randn((1, len(rows), 2 * group * head_dim), generator=g, device="cuda") * 2
    want, bound = _exact(kv, q, rows, group)
    for split in (0, 512):
        out = kv.prefix_attention(q, rows, [(0, 0, len(rows))], split_tokens=split)
        assert bool(((out.double() - want).abs() <= bound).all())


@pytest.mark.parametrize("head_dim,group,rows_each", [(64, 1, 1), (128, 4, 1), (64, 3, 6)])
def test_behind_prefixes(gpu, head_dim, group, rows_each):
    g = torch.Generator("cuda").manual_seed(8)
    lengths = [rows_each, 30, 50, 61, 300, 17]
    kv = _kv(1, 2, head_dim, seqs=6)
    _filled(kv, lengths, g)
    rows = [(s, n - rows_each + i) for s, n in enumerate(lengths[:4]) for i in range(rows_each)]
    prefixes = [(4, 299, 2 * rows_each), (0, 0, rows_each), (5, 17, rows_each)]
    q = torch.randn((1, len(rows), 2 * group * head_dim), generator=g, device="cuda")
    want, bound = _exact(kv, q, rows, group, prefixes)
    for split in (0, 32):
        out = kv.prefix_attention(q, rows, prefixes, split_tokens=split)
        assert bool(((out.double() - want).abs() <= bound).all())
    inplace = q.clone()
    assert kv.prefix_attention(inplace, rows, prefixes, out=inplace, split_tokens=32) is inplace
    assert torch.equal(inplace, out)


def test_scales_far_apart_and_rows_not_seen(gpu):
    """Pages whose scales differ by 2^80, in any order; later rows, and what pages
    held before, do not matter."""
    g = torch.Generator("cuda").manual_seed(9)
    kv = _kv(1, 1, 64, pages=40, seqs=4)
    old = kv.add_seq()  # leaves large values in its pages
    kv.reserve(old, 20 * PAGE)
    x = torch.full((1, 20 * PAGE, 64), 1e30, device="cuda")
    kv.append([(old, p) for p in range(20 * PAGE)], x, x)
    kv.free_seq(old)
    sizes = [1.0, 1e12, 1e-12, 3.0, 1e-3, 1e6]
    s = kv.add_seq()
    kv.reserve(s, 6 * PAGE)
    rows = [(s, p) for p in range(6 * PAGE - 5)]
    k = torch.randn((1, len(rows), 64), generator=g, device="cuda")
    v = k.clone()
    for i, z in enumerate(sizes):
        v[:, i * PAGE:(i + 1) * PAGE] *= z
    kv.append(rows, k, v)
    ask = [(s, p) for p in (0, 7, 15, 16, 40, 47, 48, 63, 70, 90)]
    q = torch.randn((1, len(ask), 64), generator=g, device="cuda") * 4
    out = kv.attention(q, ask)
    kk, vv = kv.gather_values(rows)
    for i, (_, p) in enumerate(ask):
        score = (q[0, i].double() * kk[0, :p + 1].double()).sum(-1) / 8
        w = torch.softmax(score, 0)
        want = (w[:, None] * vv[0, :p + 1].double()).sum(0)
        # relative to what the value's page adds at most (its weights' parts), 2^-20, and the scores' error:
        # 2 * (|q| |k| / 8 * 68 * 2^-24)
        ds = (q[0, i].double() * kk[0, :p + 1].double()).abs().sum(-1).max() / 8 * (2.0 ** -21 + 72 * 2.0 ** -24) + 2e-6
        bound = (w[:, None] * vv[0, :p + 1].double().abs()).sum(0) * (2 * ds + 2.0 ** -17) + 1e-30
        assert bool(((out[0, i].double() - want).abs() <= bound + want.abs() * 2.0 ** -20).all()), p
    again = kv.attention(q[:, :4], ask[:4])
    big = torch.full((1, 1, 64), 1e25, device="cuda")
    kv.append([(s, 2 * PAGE + 3)], big, big)  # a page that the first four do not see
    assert torch.equal(kv.attention(q[:, :4], ask[:4]), again)


@pytest.mark.parametrize("n_layer,n_head,head_dim", [(4, 16, 128), (4, 16, 64), (1, 8, 128)])
def test_prompts_over_scales_far_apart(gpu, n_layer, n_head, head_dim):
    """Pages whose value scales lie up to 2^80 apart, in tiles of many rows (two at a time, and one)."""
    g = torch.Generator("cuda").manual_seed(19)
    n, c = 1056, n_head * head_dim
    kv = _kv(n_layer, n_head, head_dim, pages=n // PAGE, seqs=1, ctx=n, max_rows=n)
    s = kv.add_seq()
    kv.reserve(s, n)
    rows = [(s, p) for p in range(n)]
    k = torch.randn((n_layer, n, c), generator=g, device="cuda")
    v = torch.randn((n_layer, n, c), generator=g, device="cuda")
    sizes = torch.tensor([1.0, 1e-9, 1e12, 1e-12, 3.0, 1e6, 1e-3], device="cuda")
    v *= sizes[torch.arange(n, device="cuda") // PAGE % 7][None, :, None]
    kv.append(rows, k, v)
    q = torch.randn((n_layer, n, c), generator=g, device="cuda") * 3
    out = kv.attention(q, rows)
    kk, vv = kv.gather_values(rows)
    past = torch.ones((n, n), dtype=torch.bool, device="cuda").tril()
    for layer, head in ((0, 0), (n_layer - 1, n_head - 1)):
        at = slice(head * head_dim, (head + 1) * head_dim)
        qh, kh, vh = (x[layer, :, at].double().cpu() for x in (q, kk, vv))
        parts = (qh.abs() @ kh.abs().T) / math.sqrt(head_dim)
        w = torch.softmax(((qh @ kh.T) / math.sqrt(head_dim)).masked_fill(~past.cpu(), -math.inf), -1)
        # the scores' error (q's parts 2^-21, head_dim + 8 sums of 2^-24), weights and sums as for single rows
        ds = (parts * past.cpu()).amax(-1, keepdim=True) * (2.0 ** -21 + (head_dim + 8) * 2.0 ** -24) + 2e-6
        # (a weight is 2^10 and more at the largest key, f16 in steps of 2^-24 at the least, 2^6 smaller in the units of
        # a near page: half a step is 2^-29 of the largest weight)
        small = w.amax(-1, keepdim=True) * 2.0 ** -28 * (past.cpu().double() @ vh.abs())
        bound = (w @ vh.abs()) * (2 * ds + 2.0 ** -17) + small + 1e-30
        want = w @ vh
        assert bool(((out[layer, :, at].double().cpu() - want).abs() <= bound + want.abs() * 2.0 ** -20).all()), (layer, head)


def test_steps(gpu):
    """ni_kv_step and decode steps: the append, then the queried rows' attention."""
    rng, g = random.Random(1), torch.Generator("cuda").manual_seed(10)
    kv, ref = _kv(pages=120), _kv(pages=120)
    for x in (kv, ref):
        for _ in range(5):
            x.add_seq()
    for turn in range(8):
        work = []
        for s in rng.sample(range(5), 4):
            n = rng.choice([1, 1, 3, 30])
            work.append((s, n, rng.choice([0, 1, n])))
        n = sum(w[1] for w in work)
        q, k, v = (torch.randn((2, n, 192), generator=g, device="cuda") for _ in range(3))
        out = kv.step(work, q, k, v, out=torch.full_like(q, 7.0))
        rows, ask, at = [], [], []
        for s, m, nq in work:
            length = ref.seq_len(s)
            ref.reserve(s, length + m)
            rows += [(s, length + i) for i in range(m)]
            ask += rows[len(rows) - nq:] if nq else []
            at += range(len(rows) - nq, len(rows))
            ref.commit(s, m)
        ref.append(rows, k, v)
        want = torch.full_like(q, 7.0)
        if ask:
            exact, bound = _exact(ref, q[:, at], ask, 1)
            assert bool(((out[:, at].double() - exact).abs() <= bound).all()), turn
            want[:, at] = out[:, at]
        assert torch.equal(out, want), turn  # rows not queried are left
        assert [kv.seq_len(s) for s in range(5)] == [ref.seq_len(s) for s in range(5)]
    every = [(s, p) for s in range(5) for p in range(kv.seq_len(s))]
    assert all(torch.equal(a, b) for a, b in zip(kv.gather_values(every), ref.gather_values(every)))
    q, k, v = (torch.randn((3, 2, 2, 192), generator=g, device="cuda") for _ in range(3))
    got = kv.decode_steps([1, 3], q, k, v)
    for t in range(3):
        assert torch.equal(got[t], ref.step([(1, 1, 1), (3, 1, 1)], q[t].contiguous(), k[t].contiguous(), v[t].contiguous()))


def test_streams_without_waiting(gpu):
    g = torch.Generator("cuda").manual_seed(11)
    kv = _kv(4, 12, 64, pages=200, ctx=2000, max_rows=2048)
    s = kv.add_seq()
    kv.reserve(s, 1900)
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    q = torch.randn((4, 1, 768), generator=g, device="cuda")
    x = [torch.randn((4, 1900, 768), generator=g, device="cuda") for _ in range(2)]
    rows = [(s, p) for p in range(1900)]
    kv.append(rows, *x)
    want = kv.attention(q, [(s, 1899)])
    torch.cuda.synchronize()
    for _ in range(10):
        out = torch.empty_like(want)
        zero = torch.zeros_like(x[0])
        torch.cuda.synchronize()
        kv.append(rows, zero, zero, stream=a)
        kv.append(rows, *x, stream=b)
        kv.attention(q, [(s, 1899)], out=out, stream=a)
        torch.cuda.synchronize()
        assert torch.equal(out, want)


@pytest.mark.parametrize("fmt", ["f16", "q8"])
def test_values_of_the_other_caches(gpu, fmt):
    g = torch.Generator("cuda").manual_seed(12)
    for d in (64, 128):
        kv = na.PagedKv(na.BatchOpts(n_layer=2, n_head=3, head_dim=d, kv_blocks=20, max_seqs=2, n_ctx=200, max_rows=64,
                                     q8=fmt == "q8"))
        s = kv.add_seq()
        kv.reserve(s, 50)
        rows = [(s, p) for p in range(50)]
        kv.append(rows, *[torch.randn((2, 50, 3 * d), generator=g, device="cuda") for _ in range(2)])
        for layer in (na.ALL_LAYERS, 1):
            got = kv.gather_values(rows[3:40], layer=layer)
            if fmt == "f16":
                want = [x.view(torch.float16).float() for x in kv.gather(rows[3:40], layer=layer)]
            else:
                values, scales = kv.gather_q8(rows[3:40], layer=layer)
                want = [(x.float().view(*sc.shape, d) * sc[..., None]).view(x.shape) for x, sc in zip(values, scales)]
                want = want if layer == na.ALL_LAYERS else [x[0] for x in want]
            assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_calls_that_do_not_take_it(gpu):
    kv = _kv()
    s = kv.add_seq()
    kv.reserve(s, 20)
    z = torch.zeros((2, 1, 192), device="cuda")
    for call in (lambda: kv.gather([(s, 0)]), lambda: kv.gather_q8([(s, 0)]), lambda: kv.step_begin([(s, 1, 1)]),
                 lambda: kv.append_rotary([(s, 0)], z, z, na.Rotary(64)),
                 lambda: kv.qkv_append([(s, 0)], torch.zeros((1, 64), device="cuda"), torch.zeros((576, 64), device="cuda")),
                 lambda: kv.attention(z, [(s, 0)], split_tokens=8), lambda: kv.append([(s, 40)], z, z)):
        with pytest.raises(na.KvError) as e:
            call()
        assert e.value.code in (_abi.NI_ERR_BAD_ARG, _abi.NI_ERR_NOT_RESERVED)
    L, p = kv._L, z.data_ptr()
    w = (_abi.ni_work * 1)(_abi.ni_work(s, 1, 1))
    assert L.ni_kv_step_noalloc(kv.handle, w, 1, p, p, p, 192, 192, p, 192, 192, 0, None) == _abi.NI_ERR_BAD_ARG
    assert "block-scaled" in L.ni_kv_last_error(kv.handle).decode()
    rows = (_abi.ni_row * 2)(_abi.ni_row(s, 0), _abi.ni_row(s, 1))
    assert L.ni_kv_gather_values(kv.handle, 0, rows, 2, p, p, 64, 0, None) == _abi.NI_ERR_BAD_ARG
    assert L.ni_kv_gather_values(kv.handle, 0, rows, 2, p + 4, p, 192, 0, None) == _abi.NI_ERR_BAD_ARG
    assert kv.gather_values([])[0].shape == (2, 0, 192)
