"""Attention over the block-scaled cache where rows of one call see different
pages: a row's output is that of the pages it sees, whatever later ones hold.
Tiles of every form, ragged ones too."""
import math

import pytest
import torch

from test_gpu_block8 import PAGE, _exact, _kv

pytestmark = pytest.mark.gpu


def _held(n_layer, n_head, head_dim, n, sizes, g, keys=None):
    """A sequence of n rows whose values' size in page i is sizes[i % len(sizes)]."""
    c = n_head * head_dim
    kv = _kv(n_layer, n_head, head_dim, pages=-(-n // PAGE) + 1, seqs=2, ctx=n + PAGE, max_rows=n)
    s = kv.add_seq()
    kv.reserve(s, n)
    v = torch.randn((n_layer, n, c), generator=g, device="cuda")
    v *= torch.tensor(sizes, dtype=torch.float64, device="cuda")[torch.arange(n, device="cuda") // PAGE % len(sizes)].float()[None, :, None]
    k = torch.randn((n_layer, n, c), generator=g, device="cuda") if keys is None else keys
    kv.append([(s, p) for p in range(n)], k, v)
    return kv, s


def _check_seen(kv, s, out, q, rows, group, layers=None, heads=None):
    """Against 64 bits over the keys that each row sees, relative to the values that it sees."""
    d, h = kv.opts.head_dim, kv.opts.n_head
    n = max(rows) + 1
    k, v = kv.gather_values([(s, p) for p in range(n)])
    for layer in layers or range(kv.opts.n_layer):
        for head in heads or range(h):
            at = slice(head * d, (head + 1) * d)
            kk, vv = k[layer, :, at].double().cpu(), v[layer, :, at].double().cpu()
            for j in range(group):
                x = q[layer, :len(rows), (head * group + j) * d:(head * group + j + 1) * d].double().cpu()
                got = out[layer, :len(rows), (head * group + j) * d:(head * group + j + 1) * d].double().cpu()
                past = torch.arange(n)[None] <= torch.tensor(rows)[:, None]
                w = torch.softmax((x @ kk.T / math.sqrt(d)).masked_fill(~past, -math.inf), -1)
                want = w @ vv
                # Scores: q's parts 2^-21 (2^-25 of what is below their normal range), d + 8 sums of 2^-24; a weight moves by
                # twice that, by its parts (2^-20) and the sums of the keys of a wave and their joining.
                parts = (x.abs() @ kk.abs().T / math.sqrt(d) * past).amax(-1, keepdim=True)
                ds = parts * (2.0 ** -21 + (d + 8) * 2.0 ** -24) + 2e-6
                # (a weight is 2^10 and more at the largest key of a wave, in f16 steps of 2^-24 at the least, 2^6 smaller in the
                # units of a near page: half a step is 2^-29 of the largest weight)
                small = w.amax(-1, keepdim=True) * 2.0 ** -28 * (past.double() @ vv.abs())
                bound = (w @ vv.abs()) * (2 * ds + 2.0 ** -17) + small + want.abs() * 2.0 ** -20
                # (values of scales 2^83 below the largest seen add nothing: at most 2^9 of their scale each)
                top = (past[:, :, None] * vv.abs()[None]).amax((1, 2))[:, None] if len(rows) * n * d < 1 << 24 else 0.0
                bound = bound + torch.as_tensor(top) * 2.0 ** -66
                bad = (got - want).abs() > bound
                assert not bool(bad.any()), (layer, head, j, [rows[i] for i in torch.nonzero(bad.any(1))[:5, 0].tolist()])


# Shapes, and the form that plan_prefix gives them at 200 rows: one tile with eight waves, with four, in partitions; tiles
# of many rows one at a time; two at a time.
FORMS = [(1, 1, 64, 1, 0), (1, 2, 128, 4, 0), (1, 2, 64, 3, 64), (4, 12, 64, 1, 0), (1, 32, 128, 2, 0), (8, 32, 64, 2, 0),
         (4, 32, 128, 4, 0)]


@pytest.mark.parametrize("n_layer,n_head,head_dim,group,split", FORMS)
@pytest.mark.parametrize("up", [90, 130, 200])
def test_rows_before_a_page_of_far_larger_values(gpu, n_layer, n_head, head_dim, group, split, up):
    """Neighbouring rows in one call; a later page's values, and those of one more, lie 2^up above those of the pages before."""
    n, small = 12 * PAGE + 11, 2.0 ** -(up // 2)
    for first, large in ((0, 1), (9, 1), (5, 8), (9, 3), (2, 2)):
        g = torch.Generator("cuda").manual_seed(up + first)
        sizes = [small] * 13
        sizes[large], sizes[large + 2] = small * 2.0 ** up, small * 2.0 ** (up - 5)
        kv, s = _held(n_layer, n_head, head_dim, n, sizes, g)
        rows = list(range(first, n))
        q = torch.randn((n_layer, len(rows), n_head * group * head_dim), generator=g, device="cuda") * 2
        out = kv.prefix_attention(q, [(s, p) for p in rows], [(0, 0, len(rows))], split_tokens=split)
        _check_seen(kv, s, out, q, rows, group, layers=sorted({0, n_layer - 1}), heads=sorted({0, n_head - 1}))
        # rows by themselves, on both sides of the large page's first row
        for at in ((large * PAGE - 1 - first, large * PAGE - first)):
            one = kv.prefix_attention(q[:, at:at + 1].contiguous(), [(s, rows[at])], [(0, 0, 1)])
            assert float((one - out[:, at:at + 1]).abs().max()) <= 1e-4 * float(one.abs().max()), (first, large, rows[at])


@pytest.mark.parametrize("n_layer,n_head,head_dim,group,split", FORMS)
def test_rows_do_not_move_with_rows_behind_them(gpu, n_layer, n_head, head_dim, group, split):
    """The last rows' values replaced by others of all sizes: rows that do not see their pages keep every bit."""
    g = torch.Generator("cuda").manual_seed(31)
    n, c = 3 * PAGE + 13, n_head * head_dim
    kv, s = _held(n_layer, n_head, head_dim, n, [1.0, 1e-3, 1e3], g)
    rows = [(s, p) for p in range(5, n)]
    q = torch.randn((n_layer, len(rows), n_head * group * head_dim), generator=g, device="cuda") * 2
    ask = lambda: kv.prefix_attention(q, rows, [(0, 0, len(rows))], split_tokens=split)  # noqa: E731
    first = ask()
    for page in (3, 2, 1):
        for size in (1e-30, 1e-3, 3.0, 30.0, 1e4, 1e12, 1e28):
            x = [torch.randn((n_layer, n - page * PAGE, c), generator=g, device="cuda") * z for z in (1.0, size)]
            kv.append([(s, p) for p in range(page * PAGE, n)], *x)
            assert torch.equal(ask()[:, :page * PAGE - 5], first[:, :page * PAGE - 5]), (page, size)


@pytest.mark.parametrize("up", [100, 130, 230])
def test_values_far_below_others_add_nothing(gpu, up):
    """A row that sees small values, then far larger ones that it does not attend to: what it has of the small ones stays
    small beside the large."""
    n, d = 40 * PAGE, 64
    g = torch.Generator("cuda").manual_seed(up)
    keys = torch.zeros((1, n, d), device="cuda")
    keys[:, n // 2:] = -200.0
    keys[:, :n // 2] = 200.0
    kv, s = _held(1, 1, d, n, [2.0 ** -(up // 2)] * 20 + [2.0 ** (up - up // 2)] * 20, g, keys=keys)
    q = torch.ones((1, n, d), device="cuda")
    out = kv.attention(q, [(s, p) for p in range(n)])
    assert bool((out.abs() <= 2.0 ** -(up // 2) * 8).all())
    _check_seen(kv, s, out[:, :n // 2], q, list(range(n // 2)), 1)


@pytest.mark.parametrize("n_layer,n_head,head_dim,group", [(4, 16, 128, 1), (4, 16, 64, 3), (2, 16, 128, 4), (8, 12, 64, 1)])
@pytest.mark.parametrize("rows,before", [(1041, 7), (1049, 0), (1057, 13), (1031, 16)])
@pytest.mark.parametrize("split", [0, 512])
def test_ragged_tiles_of_many_rows(gpu, n_layer, n_head, head_dim, group, rows, before, split):
    """Two tiles at a time, the last of them short or empty, heads of a row in two tiles, behind earlier rows, in partitions."""
    g = torch.Generator("cuda").manual_seed(rows)
    n = before + rows
    kv, s = _held(n_layer, n_head, head_dim, n, [1.0], g)
    q = torch.randn((n_layer, rows, n_head * group * head_dim), generator=g, device="cuda") * 1.5
    at = [(s, before + i) for i in range(rows)]
    out = kv.prefix_attention(q, at, [(0, 0, rows)], split_tokens=split)
    pick = sorted({0, 1, 15, 16, 17, rows // 2, rows - 33, rows - 17, rows - 16, rows - 2, rows - 1})
    want, bound = _exact(kv, q[:, pick].contiguous(), [at[i] for i in pick], group)
    assert bool(((out[:, pick].double() - want).abs() <= bound).all())
    _check_seen(kv, s, out, q, [before + i for i in range(rows)], group, layers=[n_layer - 1], heads=[n_head - 1])


@pytest.mark.parametrize("n_layer,n_head,head_dim,group", [(8, 16, 64, 1), (4, 16, 128, 4)])
@pytest.mark.parametrize("split", [0, 64])
def test_many_rows_behind_prefixes(gpu, n_layer, n_head, head_dim, group, split):
    g = torch.Generator("cuda").manual_seed(41)
    kv = _kv(n_layer, n_head, head_dim, pages=120, seqs=4, ctx=700, max_rows=700)
    c = n_head * head_dim
    for n in (300, 270, 331, 17):
        s = kv.add_seq()
        kv.reserve(s, n)
        kv.append([(s, p) for p in range(n)], *[torch.randn((n_layer, n, c), generator=g, device="cuda") for _ in range(2)])
    rows = [(0, p) for p in range(300)] + [(1, p) for p in range(9, 270)]
    q = torch.randn((n_layer, len(rows), c * group), generator=g, device="cuda")
    for prefixes in ([(2, 331, len(rows))], [(2, 40, 300), (3, 17, 261)], [(3, 16, 300), (0, 0, 261)]):
        out = kv.prefix_attention(q, rows, prefixes, split_tokens=split)
        pick = [0, 15, 16, 31, 32, 100, 299, 300, 315, 316, 560]
        at, front = [rows[i] for i in pick], []
        for ps, pn, count in prefixes:
            front += [(ps, pn, 1)] * count
        want, bound = _exact(kv, q[:, pick].contiguous(), at, group, [front[i] for i in pick])
        assert bool(((out[:, pick].double() - want).abs() <= bound).all()), prefixes
