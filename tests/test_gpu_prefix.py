"""Attention behind shared prefixes against its formula in 64 bits over the
stored f16 (or int8) keys and values.

Tolerance: q enters the products in two f16 parts (2^-22 of itself), a score
sums its products in f32, softmax weights enter PV in two parts (2^-22) and
every sum over keys is f32.  With scores of a few units and sums that round
like a random walk over up to 2^12 keys the relative error (norm) is about
2^-22 to 2^-21; asked is 2^-18, and of single values 2^-16 of the largest."""
import math

import numpy as np
import pytest
import torch

import nanoinfer_amd as na

pytestmark = pytest.mark.gpu


class Cache:
    """A PagedKv filled with random rows and what it stores, in 64 bits."""

    def __init__(self, lens, n_layer=1, n_head=2, head_dim=64, q8=False, seed=0, std=1.0, spare=2, far=False):
        pages = sum(-(-n // 16) for n in lens) + spare
        order = np.random.default_rng(seed).permutation(pages)
        self.opts = na.BatchOpts(n_layer=n_layer, n_head=n_head, head_dim=head_dim, kv_blocks=pages, max_seqs=len(lens),
                                 n_ctx=max(lens), max_rows=4096, q8=q8,
                                 page_order=np.sort(order)[::-1].copy() if far else order)
        self.kv = na.PagedKv(self.opts)
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.k, self.v = [], []
        for n in lens:
            s = self.kv.add_seq()
            self.kv.reserve(s, n)
            k, v = (torch.randn((n_layer, n, n_head * head_dim), generator=g, device="cuda") * std for _ in range(2))
            self.put(s, k, v)
            self.k.append(self.stored(k))
            self.v.append(self.stored(v))

    def put(self, s, k, v, p0=0):
        for i in range(0, k.shape[1], 4096):
            n = min(4096, k.shape[1] - i)
            self.kv.append([(s, p0 + i + j) for j in range(n)], k[:, i:i + n], v[:, i:i + n])

    def stored(self, x):
        o = self.opts
        x = x.reshape(o.n_layer, -1, o.n_head, o.head_dim)
        if not o.q8:
            return x.half().double()
        scale = (x.abs().amax(-1, keepdim=True).double() / 127).float()
        inv = torch.where(scale > 0, 1 / scale.double(), torch.zeros_like(scale).double()).float()
        return torch.round(x * inv).clamp(-127, 127).double() * scale.double()

    def expect(self, q, rows, prefixes):
        """q [n_layer, n, heads * hd] -> the result in 64 bits."""
        o = self.opts
        L, n = q.shape[:2]
        q = q.double().view(L, n, o.n_head, -1, o.head_dim)
        out = torch.empty_like(q)
        at = [(s, m) for s, m, c in prefixes for _ in range(c)]
        for i, ((s, p), (ps, m)) in enumerate(zip(rows, at)):
            k, v = self.k[s][:, :p + 1], self.v[s][:, :p + 1]
            if m:
                k, v = torch.cat([self.k[ps][:, :m], k], 1), torch.cat([self.v[ps][:, :m], v], 1)
            k, v = k.permute(0, 2, 3, 1).contiguous(), v.transpose(1, 2).contiguous()  # [L, heads, hd, keys] and back
            w = torch.softmax(torch.matmul(q[:, i], k) / math.sqrt(o.head_dim), -1)
            out[:, i] = torch.matmul(w, v)
        return out.reshape(L, n, -1).cpu()

    def queries(self, n, group=1, seed=1):
        o = self.opts
        g = torch.Generator(device="cuda").manual_seed(seed)
        return torch.randn((o.n_layer, n, o.n_head * group * o.head_dim), generator=g, device="cuda")


def close(got, want, what=""):
    got = got.double().cpu()
    assert torch.isfinite(got).all(), what
    err = got - want
    rel, top = (err.norm() / want.norm()).item(), (err.abs().max() / want.abs().max()).item()
    assert rel <= 2.0 ** -18 and top <= 2.0 ** -16, f"{what}: {rel:.2e} of the norm, {top:.2e} of the largest"


def check(c, rows, prefixes, group=1, seed=1, **kw):
    q = c.queries(len(rows), group, seed)
    got = c.kv.prefix_attention(q, rows, prefixes, **kw)
    close(got, c.expect(q, rows, prefixes), f"{rows[:3]}.. {prefixes} {kw}")
    return q, got


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("group", [1, 3, 4, 20])
def test_heads_and_lengths(gpu, d, group, q8):
    c = Cache([1, 2, 15, 16, 17, 40, 129, 33, 300], n_head=2, head_dim=d, q8=q8, seed=d + group)
    last = [(s, n - 1) for s, n in enumerate([1, 2, 15, 16, 17, 40, 129])]
    for m in (1, 15, 16, 17, 33):
        check(c, last, [(7, m, 7)], group)
    check(c, last, [(8, 300, 3), (7, 5, 2), (0, 0, 2)], group)
    check(c, last, [(8, 257, 7)], group, split_tokens=16)
    check(c, last, [(8, 300, 7)], group, split_tokens=64)
    check(c, last, [(0, 0, 7)], group)


@pytest.mark.parametrize("d,q8", [(64, False), (128, False), (64, True)])
@pytest.mark.parametrize("split", [0, 16, 48])
def test_runs_of_rows(gpu, d, q8, split):
    """Verify rows and prompt chunks: consecutive rows share their sequence's
    keys and see them causally; rows of one sequence in other orders do not."""
    c = Cache([60, 31, 200, 150], n_layer=2, n_head=3, head_dim=d, q8=q8, seed=7)
    rows = [(0, p) for p in range(50, 55)] + [(1, p) for p in range(0, 31)]
    rows += [(2, 10), (2, 9), (2, 150), (2, 150), (0, 3)]
    check(c, rows, [(3, 150, 5), (3, 77, 31), (3, 16, 3), (0, 0, 2)], split_tokens=split)
    check(c, rows, [(3, 150, 4), (3, 150, 2), (3, 1, 35)], 2, split_tokens=split)  # a run across two prefixes


def test_every_prompt_row(gpu):
    c = Cache([130, 90], n_head=2, seed=9)
    rows = [(0, p) for p in range(130)]
    check(c, rows, [(1, 90, 130)])
    check(c, rows, [(1, 90, 130)], 5)
    check(c, rows, [(0, 0, 130)], 3, split_tokens=32)


@pytest.mark.parametrize("q8", [False, True])
def test_many_rows_and_a_long_prefix(gpu, q8):
    """Wide tiles and many partitions; a plan past the launch arguments."""
    lens = [1 + (i * 37) % 90 for i in range(70)] + [5000, 2100]
    c = Cache(lens, n_head=4, q8=q8, seed=11)
    rows = [(i, lens[i] - 1) for i in range(70)]
    check(c, rows, [(70, 5000, 40), (71, 2099, 30)], 2)
    check(c, rows, [(70, 4999, 70)], 1, split_tokens=4096)


def large(d, q8):
    """(layers, heads, positions) from which 17 rows behind a prefix take wide tiles."""
    return (4, 16, 2400) if q8 and d == 64 else (2, 8, 2050)


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("n", [16, 17, 33, 65, 97, 129, 200])
def test_wide_tiles(gpu, n, d, q8):
    """One to four waves of slots, one workgroup or two, full and not; prefixes
    that end inside a tile, inside a page and on a border; one of few rows."""
    layers, heads, m = large(d, q8)
    c = Cache([n + 4, m + 40, 71], n_layer=layers, n_head=heads, head_dim=d, q8=q8, seed=n)
    rows = [(0, p) for p in range(4, n + 4)]
    check(c, rows, [(1, m, n)])
    check(c, rows, [(1, m + 33, n - 1), (2, 71, 1)], split_tokens=512)
    check(c, rows[:n // 2 + 1], [(1, m + 14, n // 2 + 1)], 2, split_tokens=352)
    check(c, rows[:n // 4 + 1], [(1, m + 16, n // 4 + 1)], 4, split_tokens=m // 16 * 16)


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("d", [64, 128])
def test_wide_tiles_of_one_row(gpu, d, q8):
    """Many query heads of a single row, and runs with keys of their own in parts."""
    layers, heads, m = large(d, q8)
    c = Cache([700, m], n_layer=layers, n_head=heads, head_dim=d, q8=q8, seed=3)
    check(c, [(0, 699)], [(1, m, 1)], 20)
    check(c, [(0, 650), (0, 651), (0, 652)], [(1, m, 3)], 8)


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("n,wide", [(3, False), (40, False), (40, True)])
def test_values_of_many_sizes(gpu, n, wide, q8):
    """Values that grow along the keys, to thousands: int8 scales past 1."""
    layers, heads, m = large(64, q8) if wide else (1, 2, 400)
    c = Cache([n, m], n_layer=layers, n_head=heads, q8=q8, seed=35)
    size = torch.logspace(-3, 3.5, m, device=gpu)[None, :, None]
    g = torch.Generator(device="cuda").manual_seed(36)
    k, v = (torch.randn((layers, m, heads * 64), generator=g, device="cuda") for _ in range(2))
    for flip in (False, True):
        k, v = (k.flip(1), v) if flip else (k, v * size)
        v = v.flip(1) if flip else v
        c.put(1, k, v)
        c.k[1], c.v[1] = c.stored(k), c.stored(v)
        check(c, [(0, p) for p in range(n)], [(1, m, n)])
        check(c, [(0, 0)] * n, [(1, m - 1, n)], 3, split_tokens=0 if wide else 96)


@pytest.mark.parametrize("d", [64, 128])
def test_what_lies_behind_a_prefix_does_not_matter_to_wide_tiles(gpu, d):
    layers, heads, m = large(d, False)
    c = Cache([30, m + 20], n_layer=layers, n_head=heads, head_dim=d, seed=37)
    bad = torch.full((layers, 17, heads * d), float("nan"), device=gpu)
    c.put(1, bad, bad, m + 3)
    check(c, [(0, p) for p in range(30)], [(1, m + 3, 30)])
    check(c, [(0, p) for p in range(30)], [(1, m, 30)], split_tokens=1024)


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("d", [64, 128])
def test_many_short_rows(gpu, d, q8):
    """A decode batch of every layer: single rows of one key to a few pages, in
    launches of several rounds, behind a long prefix and behind none; what lies
    behind their ends, to the last page's, is as bad as can be."""
    lens = [1 + (i * 7) % 75 for i in range(67)]
    c = Cache([n + 16 for n in lens] + [700], n_layer=12, n_head=4, head_dim=d, q8=q8, seed=41, spare=3)
    bad = torch.full((12, 16, 4 * d), float("inf"), device=gpu)
    for i, n in enumerate(lens):
        c.put(i, bad, bad, n)
    rows = [(i, n - 1) for i, n in enumerate(lens)]
    for group in (1, 2):
        check(c, rows, [(67, 700, 67)], group)
        check(c, rows, [(67, 689, 60), (0, 0, 7)], group)
        check(c, rows, [(0, 0, 67)], group)


def test_layers_and_one_layer(gpu):
    c = Cache([20, 50, 64], n_layer=4, n_head=2, head_dim=128, seed=13)
    rows, pre = [(0, 19), (1, 44), (1, 45)], [(2, 63, 3)]
    q, got = check(c, rows, pre, 4)
    for layer in range(4):
        one = c.kv.prefix_attention(q[layer], rows, pre, layer=layer)
        close(one[None], c.expect(q, rows, pre)[layer:layer + 1])


@pytest.mark.parametrize("q8", [False, True])
def test_offsets_past_32_bits(gpu, q8):
    """Pages behind 2^32 halves of the pool: every kernel, and the rotating append."""
    n_head, pages = 32, 68000 if q8 else 33200
    lens = [1 + 3 * i for i in range(18)] + [2000]
    c = Cache(lens, n_head=n_head, head_dim=128, q8=q8, seed=43, spare=pages - 200, far=True)
    page_bytes = n_head * 2 * 16 * (128 + 4 if q8 else 256)
    assert min(min(c.kv.block_table(s)) for s in range(19)) * page_bytes > 2 ** 33
    rows = [(i, n - 1) for i, n in enumerate(lens[:18])]
    g = torch.Generator(device="cuda").manual_seed(44)
    k, v = (torch.randn((1, 18, n_head * 128), generator=g, device="cuda") for _ in range(2))
    c.kv.append_rotary(rows, k, v, na.Rotary(128), positions=np.zeros(18, np.uint32))  # (no turn)
    for i, (s, p) in enumerate(rows):
        c.k[s][:, p:p + 1], c.v[s][:, p:p + 1] = c.stored(k[:, i:i + 1]), c.stored(v[:, i:i + 1])
    check(c, rows, [(18, 2000, 18)])  # wide tiles, single rows
    check(c, rows, [(18, 2000, 18)], 4)
    check(c, rows[-3:], [(18, 2000, 3)])
    check(c, rows[-3:], [(18, 2000, 3)], split_tokens=512)


def test_strides_in_place_and_rows_behind(gpu):
    c = Cache([20, 50, 64], n_layer=2, n_head=2, seed=15)
    rows, pre = [(0, 19), (1, 44), (1, 45)], [(2, 63, 3)]
    q = c.queries(3, 2)
    want = c.expect(q, rows, pre)
    wide = torch.full((2, 5, 2 * 2 * 64 + 12), 9.0, device=gpu)
    wide[:, :3, 4:4 + 256] = q
    view = wide[:, :, 4:4 + 256]
    out = torch.full((2, 6, 256), 5.0, device=gpu)
    close(c.kv.prefix_attention(view, rows, pre, out=out)[:, :3], want)
    assert (out[:, 3:] == 5).all()
    got = c.kv.prefix_attention(view, rows, pre, out=view)
    assert got.data_ptr() == view.data_ptr()
    close(view[:, :3], want)
    assert (wide[:, 3:] == 9).all() and (wide[:, :, :4] == 9).all() and (wide[:, :, 260:] == 9).all()


def test_no_prefix_agrees_with_paged_attention(gpu):
    c = Cache([700, 33, 16], n_head=12, seed=17)
    rows = [(0, 699), (1, 32), (2, 0)]
    q = c.queries(3)
    a = c.kv.attention(q, rows)
    b = c.kv.prefix_attention(q, rows, [(0, 0, 3)])
    assert (a - b).norm() <= 2.0 ** -18 * a.norm()


def test_a_prefix_is_the_whole_sequence_cut_in_two(gpu):
    """Behind a prefix a row's result is that of one sequence holding both."""
    c = Cache([300, 300, 300], n_head=3, seed=19)
    k, v = (torch.randn((1, 300, 192), device=gpu) for _ in range(2))
    c.put(0, k, v)
    c.put(1, k[:, :200], v[:, :200])
    c.put(2, k[:, 200:], v[:, 200:])
    q = c.queries(2)
    whole = c.kv.attention(q, [(0, 299), (0, 250)])
    cut = c.kv.prefix_attention(q, [(2, 99), (2, 50)], [(1, 200, 2)])
    assert (whole - cut).norm() <= 2.0 ** -18 * whole.norm()


@pytest.mark.parametrize("d", [64, 128])
def test_what_masked_places_hold_does_not_matter(gpu, d):
    """Infinities and NaN behind the last key of a page, of a prefix and of the
    earlier rows of a run."""
    c = Cache([40, 40, 50], n_head=2, head_dim=d, seed=21)
    bad = torch.full((1, 1, 2 * d), float("nan"), device=gpu)
    inf = torch.full((1, 1, 2 * d), float("inf"), device=gpu)
    for s, p in ((0, 31), (0, 33), (1, 39), (2, 37), (2, 49)):
        c.put(s, bad, inf, p)
    for s, p in ((0, 32), (1, 20), (2, 38)):
        c.put(s, inf, bad, p)
    for group in (1, 2, 9):
        check(c, [(0, 28), (0, 29), (0, 30), (1, 19)], [(2, 37, 4)], group)
        # rows 28..30 see finite keys, 31 does not
        q = c.queries(5, group)
        rows, pre = [(0, p) for p in range(28, 33)], [(2, 37, 5)]
        got = c.kv.prefix_attention(q, rows, pre).view(1, 5, -1)
        close(got[:, :3], c.expect(q, rows, pre)[:, :3], "the rows before the bad key")
        assert not torch.isfinite(got[:, 3:]).any()


def test_low_scores_and_peaked_ones(gpu):
    """Scores far below zero, and one key far above the others."""
    c = Cache([30, 200], n_head=2, seed=23, std=4.0)
    q = c.queries(1) * 30.0
    rows, pre = [(0, 29)], [(1, 200, 1)]
    want = c.expect(q, rows, pre)
    got = c.kv.prefix_attention(q, rows, pre).double().cpu()
    # scores reach thousands: their f32 roundings, 2^-24 of them, are the weights'
    assert (got - want).abs().max() <= 2.0 ** -8 * want.abs().max()


def test_a_prefix_with_all_the_weight_or_none(gpu):
    c = Cache([3, 40], n_head=1, seed=25)
    q = torch.ones((1, 1, 64), device=gpu)
    k, v = torch.full((1, 40, 64), -30.0, device=gpu), torch.randn((1, 40, 64), device=gpu)
    c.put(1, k, v)
    c.put(0, torch.full((1, 3, 64), 30.0, device=gpu), torch.full((1, 3, 64), 2.0, device=gpu))
    got = c.kv.prefix_attention(q, [(0, 2)], [(1, 40, 1)])
    assert torch.equal(got, torch.full_like(got, 2.0))
    c.put(0, torch.full((1, 3, 64), -90.0, device=gpu), torch.full((1, 3, 64), 2.0, device=gpu))
    got = c.kv.prefix_attention(q, [(0, 2)], [(1, 40, 1)])
    want = v.half().double().mean(1).cpu()
    assert (got.double().cpu()[0] - want).abs().max() <= 2.0 ** -16 * want.abs().max()


def test_refusals(gpu):
    c = Cache([20, 33, 16], n_head=2, seed=27)
    q = c.queries(2)
    rows = [(0, 19), (1, 32)]

    def refused(what, rows=rows, pre=[(2, 16, 2)], q=q, **kw):
        with pytest.raises(na.KvError, match=what):
            c.kv.prefix_attention(q, rows, pre, **kw)

    refused("cover 1 rows", pre=[(2, 16, 1)])
    refused("cover 3 rows", pre=[(2, 16, 2), (2, 16, 1)])
    refused("no page", pre=[(2, 17, 2)])
    refused("out of range", pre=[(9, 1, 2)])
    refused("own prefix", pre=[(1, 16, 2)])
    refused("no page", rows=[(0, 19), (0, 32)])
    refused("multiple of 16", split_tokens=40)
    refused("n_q_head 3", q=torch.zeros((1, 2, 192), device=gpu))
    refused("overlap", out=q[:, :1].expand(1, 2, 128))
    refused("layer 1", q=q[0], layer=1)
    c.kv.free_seq(2)
    refused("not live")
    c.kv.prefix_attention(q, rows, [(2, 0, 2)])  # an empty prefix is not looked at
    assert c.kv.prefix_attention(q[:, :0], [], []).shape == (1, 0, 128)
    assert c.kv.prefix_attention(q[:, :0], [], [(2, 5, 0)]).shape == (1, 0, 128)
    wide = torch.zeros((1, 2, 256), device=gpu)
    with pytest.raises(na.KvError, match="q's strides"):  # the same memory, other strides
        c.kv.prefix_attention(wide[:, :, :128], rows, [(2, 3, 2)], out=wide.view(-1)[:256].view(1, 2, 128))


def test_captured_and_replayed(gpu):
    """A captured call replays over changed inputs, between eager calls that
    outgrow the handle's partials; a capture that would allocate is refused."""
    c = Cache([100, 60, 800, 900], n_head=4, seed=29)
    rows, pre = [(0, 99), (1, 59)], [(2, 800, 2)]
    q, out = c.queries(2), torch.empty((1, 2, 256), device=gpu)
    with pytest.raises(na.KvError, match="outside the capture"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            c.kv.prefix_attention(q, rows, pre, out=out)
    torch.cuda.synchronize()
    c.kv.prefix_attention(q, rows, pre, out=out)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c.kv.prefix_attention(q, rows, pre, out=out)
    for i in range(4):
        q.copy_(c.queries(2, seed=50 + i))
        want = c.expect(q, rows, pre)
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        close(out, want, f"replay {i}")
        # the handle's partials grow and the outgrown ones are asked back
        big = [(0, 99 - j) for j in range(60 * (i + 1) if i < 1 else 60)]
        check(c, big, [(3, 900, len(big))], 4 + i, split_tokens=16)
        c.kv.sync()


def test_streams_follow_each_other(gpu):
    """Appends on one stream, attention on another: the handle orders them."""
    c = Cache([64, 500], n_head=8, seed=31)
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    k, v = (torch.randn((1, 500, 512), device=gpu) for _ in range(2))
    q = c.queries(1)
    torch.cuda.synchronize()
    for i in range(3):
        k2, v2 = k * (i + 1), v * (i + 1)
        torch.cuda.synchronize()
        c.kv.append([(1, p) for p in range(500)], k2, v2, stream=a)
        got = c.kv.prefix_attention(q, [(0, 63)], [(1, 500, 1)], stream=b)
        b.synchronize()
        c.k[1], c.v[1] = c.stored(k2), c.stored(v2)
        # (scores of up to three times the usual size)
        err = got.double().cpu() - c.expect(q, [(0, 63)], [(1, 500, 1)])
        assert err.abs().max() <= 2.0 ** -16 * (i + 1) ** 2 * 4


def test_calls_repeat_bit_for_bit(gpu):
    c = Cache([100, 60, 3000], n_head=4, seed=33)
    rows, pre = [(0, 99), (1, 59)], [(2, 3000, 2)]
    q = c.queries(2, 4)
    first = c.kv.prefix_attention(q, rows, pre)
    for _ in range(3):
        assert torch.equal(first, c.kv.prefix_attention(q, rows, pre))


@pytest.mark.parametrize("bad", [float("inf"), 1e30])
@pytest.mark.parametrize("d", [64, 128])
def test_scales_that_only_later_rows_see(gpu, d, bad):
    """On the Q8 cache an infinite or huge value of a later row makes that
    row's scale so; the rows before it keep their results."""
    c = Cache([60, 50], n_head=2, head_dim=d, q8=True, seed=45)
    v = torch.full((1, 1, 2 * d), bad, device=gpu)
    for p in (31, 33, 40):
        k = c.queries(1, seed=p)
        c.put(0, k, v, p)
        c.k[0][:, p:p + 1], c.v[0][:, p:p + 1] = c.stored(k), c.stored(v)
    for group in (2, 5, 9):
        for n in (3, 4, 5):
            rows, pre = [(0, p) for p in range(28, 28 + n)], [(1, 50, n)]
            for split in (0, 16):
                q = c.queries(n, group)
                got, want = c.kv.prefix_attention(q, rows, pre, split_tokens=split), c.expect(q, rows, pre)
                close(got[:, :3], want[:, :3], f"{group} {n} {split}: the rows before the bad value")
                if n > 3 and math.isfinite(bad):
                    close(got[:, 3:], want[:, 3:], f"{group} {n} {split}: the rows that see it")
                elif n > 3:
                    assert not torch.isfinite(got[:, 3:]).any()


@pytest.mark.parametrize("std", [1e-2, 1e-3, 1e-5, 1e-20])
@pytest.mark.parametrize("d,wide", [(64, False), (128, False), (64, True), (128, True)])
def test_small_values_on_the_q8_cache(gpu, d, wide, std):
    """Int8 scales far below 1 cost the weights no bits, in any kernel: values
    of one small size, and of several, zeros among them, along the keys."""
    layers, heads, m = large(d, True) if wide else (1, 2, 700)
    n = 33 if wide else 17
    c = Cache([n, m], n_layer=layers, n_head=heads, head_dim=d, q8=True, seed=47)
    g = torch.Generator(device="cuda").manual_seed(48)
    k, v = (torch.randn((layers, m, heads * d), generator=g, device="cuda") for _ in range(2))
    own = [torch.randn((layers, n, heads * d), generator=g, device="cuda") for _ in range(2)]
    c.put(0, own[0], own[1] * std)
    c.k[0], c.v[0] = c.stored(own[0]), c.stored(own[1] * std)
    # every 32 keys another size (a group of waves reads every second or fourth such tile)
    steps = torch.tensor([0.0, 1.0, 0.25, 0.0, 2.0, 1.0, 0.0, 0.5], device=gpu).repeat_interleave(32)
    for size in (torch.ones(m, device=gpu), steps.repeat(-(-m // 256))[:m], torch.linspace(1, 0, m, device=gpu).square()):
        c.put(1, k, v * std * size[None, :, None])
        c.k[1], c.v[1] = c.stored(k), c.stored(v * std * size[None, :, None])
        check(c, [(0, p) for p in range(n)], [(1, m, n)])
        check(c, [(0, p) for p in range(n)], [(1, m - 5, n)], 2, split_tokens=0 if wide else 96)
        check(c, [(0, n - 1)] * 3, [(1, 64, 3)], 5)


@pytest.mark.parametrize("wide", [False, True])
def test_values_of_zero_on_the_q8_cache(gpu, wide):
    layers, heads, m = large(64, True) if wide else (1, 2, 300)
    c = Cache([20, m], n_layer=layers, n_head=heads, q8=True, seed=49, std=0.0)
    rows = [(0, p) for p in range(20)]
    got = c.kv.prefix_attention(c.queries(20), rows, [(1, m, 20)])
    assert torch.equal(got, torch.zeros_like(got))


def test_eager_calls_beside_replays(gpu):
    """A replay and a call of the same handle on another stream, neither
    waiting for the other: each has partials of its own."""
    c = Cache([200, 200, 4000, 3000], n_head=8, head_dim=128, seed=51)
    rows_a, pre_a = [(0, 184 + i) for i in range(16)], [(2, 4000, 16)]
    rows_b, pre_b = [(1, 184 + i) for i in range(16)], [(3, 3000, 16)]
    qa, qb = c.queries(16, seed=2), c.queries(16, seed=3)
    out_a, out_b = torch.empty_like(qa), torch.empty((20, *qb.shape), device=gpu)
    want_b = c.kv.prefix_attention(qb, rows_b, pre_b)
    want_a = c.kv.prefix_attention(qa, rows_a, pre_a)
    close(want_a, c.expect(qa, rows_a, pre_a))
    close(want_b, c.expect(qb, rows_b, pre_b))
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c.kv.prefix_attention(qa, rows_a, pre_a, out=out_a)
    c.kv.prefix_attention(qb, rows_b, pre_b, out=out_b[0])
    torch.cuda.synchronize()
    for i in range(20):
        with torch.cuda.stream(a):
            graph.replay()
            graph.replay()
        c.kv.prefix_attention(qb, rows_b, pre_b, out=out_b[i], stream=b)
    torch.cuda.synchronize()
    assert torch.equal(out_a, want_a)
    assert all(torch.equal(x, want_b) for x in out_b)
    # later captures share the first one's partials, or take the handle's where they need more
    more = torch.cuda.CUDAGraph()
    with torch.cuda.graph(more):
        c.kv.prefix_attention(qb, rows_b, pre_b, out=out_b[0])
    big = [(0, 199 - i) for i in range(150)]
    q = c.queries(150, 2)
    want = c.kv.prefix_attention(q, big, [(2, 4000, 150)], split_tokens=256)
    out, most = torch.empty_like(want), torch.cuda.CUDAGraph()
    with torch.cuda.graph(most):
        c.kv.prefix_attention(q, big, [(2, 4000, 150)], split_tokens=256, out=out)
    for _ in range(3):
        for x in (out_a, out_b, out):
            x.zero_()
        graph.replay()
        more.replay()
        most.replay()
        c.kv.prefix_attention(qb, rows_b, pre_b, out=out_b[1])
        torch.cuda.synchronize()
        assert torch.equal(out_a, want_a) and torch.equal(out, want)
        assert torch.equal(out_b[0], want_b) and torch.equal(out_b[1], want_b)


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("d,top", [(64, 3.6e5), (128, 5.1e5)])
@pytest.mark.parametrize("wide", [False, True])
def test_queries_at_the_end_of_their_range(gpu, d, top, q8, wide):
    """The largest q of the contract, against keys that leave ordinary scores."""
    layers, heads, m = large(d, q8) if wide else (1, 2, 300)
    n = 33 if wide else 17
    c = Cache([n, m], n_layer=layers, n_head=heads, head_dim=d, q8=q8, seed=53)
    g = torch.Generator(device="cuda").manual_seed(54)
    for s, x in ((0, n), (1, m)):
        k, v = (torch.randn((layers, x, heads * d), generator=g, device="cuda") for _ in range(2))
        k *= d ** 0.5 / top  # (f16: halves of 2^-24, as stored)
        c.put(s, k, v)
        c.k[s], c.v[s] = c.stored(k), c.stored(v)
    q = c.queries(n).clamp(-3, 3) * (top / 3)
    q[..., ::7] = top
    rows, pre = [(0, p) for p in range(n)], [(1, m, n)]
    got, want = c.kv.prefix_attention(q, rows, pre), c.expect(q, rows, pre)
    # A score's products come to 2^6 in magnitude: 2^6 * (2^-22 of the split + up to 2^7 f32 sums of 2^-24) is
    # 2^-11 of a weight, and as much of the weights' sum.
    assert torch.isfinite(got).all()
    assert (got.double().cpu() - want).norm() <= 2.0 ** -10 * want.norm()


def test_outputs_of_every_layout(gpu):
    """Row and layer strides of any kind: rows that share memory are refused,
    others hold what rows one after another do."""
    import random

    c = Cache([20, 50, 64], n_layer=3, n_head=2, seed=55)
    rows, pre = [(0, 19), (1, 44), (1, 45)], [(2, 63, 3)]
    q, rot = c.queries(3), na.Rotary(64)
    want = c.kv.prefix_attention(q, rows, pre)
    turned = c.kv.append_rotary(rows, q, q, rot, q=q)
    want_after = c.kv.prefix_attention(q, rows, pre)
    assert not torch.equal(want, want_after)  # (the keys appended are new; from here on always the same)
    rng, seen = random.Random(56), set()
    layouts = [(128, 128), (128, 384), (384, 128), (128, 256), (256, 384), (384, 256), (260, 128), (128, 388)]
    layouts += [(4 * rng.randint(28, 110), 4 * rng.randint(28, 110)) for _ in range(60)]
    for a, b in layouts:
        at = sorted(i * a + j * b for i in range(3) for j in range(3))
        shared = any(y - x < 128 for x, y in zip(at, at[1:]))
        seen.add(shared)
        buf = torch.zeros(2 * a + 2 * b + 128, device=gpu)
        out = buf.as_strided((3, 3, 128), (b, a, 1))
        if shared:
            with pytest.raises(na.KvError, match="overlap"):
                c.kv.prefix_attention(q, rows, pre, out=out)
            with pytest.raises(na.KvError, match="overlap"):
                c.kv.append_rotary(rows, q, q, rot, q=q, q_out=out)
        else:
            c.kv.prefix_attention(q, rows, pre, out=out)
            assert torch.equal(out, want_after), (a, b)
            buf.zero_()
            c.kv.append_rotary(rows, q, q, rot, q=q, q_out=out)
            assert torch.equal(out, turned), (a, b)
    assert seen == {False, True}
