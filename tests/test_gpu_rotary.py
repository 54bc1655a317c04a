"""Rotary positions on the device, contiguous rows and the cache append,
against their formulas in 64 bits.

Tolerance of a rotated value in f32: the angle within an eighth of a turn is
off by at most 3 roundings of itself (conversion, constant, product), <= 3 *
2^-24 * pi/4; the sums for sine and cosine by less than 3 * 2^-24 and their
scaling by 2^-24; the two products and their difference by 2^-24 of |x1| + |x2|
each.  Together under 8 * 2^-24 (|x1| + |x2|) m.  A narrower type adds half its
step (eps / 2 of the value, or half its smallest subnormal)."""
import numpy as np
import pytest
import torch

import nanoinfer_amd as na

pytestmark = pytest.mark.gpu

TINY = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -24, torch.bfloat16: 2.0 ** -133}


def freqs(rot):
    """Frequencies from the table the calls read (which the CPU tests hold to its formula)."""
    return np.array([int(rot._r.turns[i]) for i in range(rot.rot_dim // 2)], dtype=object)


def turn64(rot, x, pos):
    """x [..., n, heads, head_dim] in 64 bits turned to pos [n], and |x1| + |x2| of each value."""
    r = rot.rot_dim
    turns = np.array([[(int(p) * int(w)) % (1 << 64) for w in freqs(rot)] for p in pos], dtype=object)
    ang = torch.tensor((turns / (1 << 64)).astype(np.float64).reshape(len(pos), 1, r // 2) * 2 * np.pi)
    c, s = torch.cos(ang) * rot.scale, torch.sin(ang) * rot.scale
    x = x.double().cpu()
    y, mag = x.clone(), torch.zeros_like(x)
    i1, i2 = (slice(0, r, 2), slice(1, r, 2)) if rot.interleaved else (slice(0, r // 2), slice(r // 2, r))
    a, b = x[..., i1], x[..., i2]
    y[..., i1], y[..., i2] = a * c - b * s, b * c + a * s
    mag[..., i1] = mag[..., i2] = (a.abs() + b.abs()) * rot.scale
    return y, mag


def close(got, want, mag, dtype, what=""):
    tol = 8 * 2.0 ** -24 * mag + torch.finfo(dtype).eps / 2 * want.abs() * (dtype != torch.float32) + TINY[dtype]
    err = (got.double().cpu() - want).abs()
    assert (err <= tol).all(), f"{what}: worst {(err / tol).max()} of the tolerance"


CASES = [
    # rows, heads, head_dim, kwargs, dtype
    (1, 1, 64, {}, torch.float32),
    (1, 1, 2, {}, torch.float32),
    (3, 5, 64, dict(interleaved=True), torch.float32),
    (64, 12, 64, dict(rot_dim=32), torch.float32),
    (17, 3, 128, dict(rot_dim=64, interleaved=True, scaling="linear", factor=4.0), torch.bfloat16),
    (33, 7, 80, dict(rot_dim=72), torch.float16),
    (5, 3, 80, dict(rot_dim=20), torch.float32),                       # value by value
    (5, 4, 80, dict(rot_dim=20, interleaved=True), torch.bfloat16),
    (7, 4, 36, {}, torch.float16),
    (7, 4, 4, dict(rot_dim=2), torch.float32),
    (9, 2, 256, dict(base=1e6), torch.float16),
    (700, 33, 128, dict(scaling="yarn", factor=8.0, orig_ctx=8192, base=500000.0), torch.float32),
    (2050, 40, 64, dict(scaling="ntk", factor=5.5, rot_dim=56), torch.bfloat16),
    # chunks of eight values, one head a thread, two and four
    (900, 9, 80, dict(rot_dim=72), torch.float16),
    (500, 11, 128, dict(rot_dim=64, interleaved=True), torch.bfloat16),
    (300, 7, 256, dict(base=1e6), torch.float32),
    (1030, 33, 128, dict(interleaved=True), torch.float32),
    (2100, 41, 128, dict(rot_dim=96), torch.bfloat16),
]


@pytest.mark.parametrize("n,h,d,kw,dtype", CASES)
def test_rows(gpu, n, h, d, kw, dtype):
    rot = na.Rotary(d, **kw)
    g = torch.Generator().manual_seed(n * 31 + d)
    x = torch.randn((n, h * d), generator=g).to(dtype)
    pos = torch.randint(0, 1 << 20, (n,), generator=g, dtype=torch.int32)
    pos[0] = 0
    if n > 2:
        pos[1], pos[2] = 2 ** 31 - 1, -5
    pad = h * d + 24 + (-h * d) % 8  # rows stay on 16-byte borders
    wide = torch.full((n + 2, pad), 7.0, dtype=dtype, device=gpu)  # rows of a wider buffer
    wide[:n, :h * d] = x.cuda()
    want, mag = turn64(rot, x.view(n, h, d), pos.tolist())
    got = na.rotary(wide[:n], rot, h, positions=pos.cuda())
    assert got.shape == (n, h * d) and got.dtype == dtype
    close(got.view(n, h, d), want, mag, dtype, "positions")
    assert (got.view(n, h, d)[..., rot.rot_dim:].cpu() == x.view(n, h, d)[..., rot.rot_dim:]).all()
    # consecutive positions, in place: nothing else of the buffer changes
    want, mag = turn64(rot, x.view(n, h, d), range(100001, 100001 + n))
    back = na.rotary(wide[:n], rot, h, pos0=100001, out=wide[:n])
    assert back.data_ptr() == wide.data_ptr()
    close(wide[:n, :h * d].reshape(n, h, d), want, mag, dtype, "pos0, in place")
    assert (wide[:n, h * d:] == 7).all() and (wide[n:] == 7).all()
    # off those borders, value by value
    odd = torch.zeros((n, h * d + 3), dtype=dtype, device=gpu)
    odd[:, 1:1 + h * d] = x.cuda()
    out = torch.full((n + 1, h * d + 5), 3.0, dtype=dtype, device=gpu)
    na.rotary(odd[:, 1:], rot, h, pos0=100001, out=out[:, 2:])
    close(out[:n, 2:2 + h * d].reshape(n, h, d), want, mag, dtype, "off 16-byte borders")
    assert (out[:n, :2] == 3).all() and (out[:n, 2 + h * d:] == 3).all() and (out[n] == 3).all()


def test_rows_far_positions_keep_their_angles(gpu):
    """pos0 near 2^32: the first pair alone turns a radian a position."""
    rot = na.Rotary(64)
    x = torch.randn((4, 64), generator=torch.Generator().manual_seed(1))
    pos0 = (1 << 32) - 4
    want, mag = turn64(rot, x.view(4, 1, 64), range(pos0, pos0 + 4))
    close(na.rotary(x.cuda(), rot, 1, pos0=pos0).view(4, 1, 64), want, mag, torch.float32)


def test_rows_nothing_to_do(gpu):
    rot = na.Rotary(64)
    assert na.rotary(torch.empty((0, 64), device=gpu), rot, 1).shape == (0, 64)
    assert na.rotary(torch.empty((3, 64), device=gpu), rot, 0).shape == (3, 0)


def test_rows_non_finite_values_stay_in_their_pairs(gpu):
    rot = na.Rotary(64)
    x = torch.ones((1, 128))
    x[0, 3], x[0, 70] = float("inf"), float("nan")
    y = na.rotary(x.cuda(), rot, 2, pos0=9).cpu()[0]
    bad = {3, 35, 64 + 6, 64 + 38}
    assert [i for i in range(128) if not torch.isfinite(y[i])] == sorted(bad)


def test_rows_and_attention_stay_relative(gpu):
    """Rotated q and k, then contiguous attention: shifting every position
    leaves the result (scores depend on differences of positions alone)."""
    h, d, n = 4, 64, 50
    g = torch.Generator().manual_seed(5)
    q, k, v = (torch.randn((n, h * d), generator=g).cuda() for _ in range(3))
    rot = na.Rotary(d)
    outs = []
    for p0 in (0, 12345):
        outs.append(na.attention(na.rotary(q, rot, h, pos0=p0), na.rotary(k, rot, h, pos0=p0), v, n, 0, h, d))
    assert (outs[0] - outs[1]).norm() <= 1e-5 * outs[0].norm()


# ------------------------------------------------------------------- append


def f16_tol(want, mag):
    return 8 * 2.0 ** -24 * mag + 2.0 ** -11 * want.abs() + 2.0 ** -25


def _filled(opts, lens):
    kv = na.PagedKv(opts)
    for n in lens:
        kv.reserve(kv.add_seq(), n)
    return kv


def _gather(kv, rows, layer=na.ALL_LAYERS):
    k, v = kv.gather(rows, layer=layer)
    return k.view(torch.float16).cpu(), v.view(torch.float16).cpu()


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("group", [1, 4])
@pytest.mark.parametrize("kw", [{}, dict(interleaved=True, rot_dim=32), dict(rot_dim=24, scaling="linear", factor=2.0),
                                dict(scaling="yarn", factor=4.0, orig_ctx=64)])
def test_append(gpu, d, group, kw):
    L, H = 3, 2
    opts = na.BatchOpts(n_layer=L, n_head=H, head_dim=d, kv_blocks=24, max_seqs=4, n_ctx=128, max_rows=64,
                        page_order=np.random.default_rng(3).permutation(24))
    kv = _filled(opts, (40, 17, 1))
    rows = [(0, p) for p in range(14, 35)] + [(2, 0), (1, 16), (1, 3), (0, 39)]
    n, hq = len(rows), H * group
    g = torch.Generator().manual_seed(d + group)
    fused = torch.randn((L, n + 1, (hq + 2 * H) * d), generator=g).cuda()
    q, k, v = fused[..., :hq * d], fused[..., hq * d:(hq + H) * d], fused[..., (hq + H) * d:]
    rot = na.Rotary(d, **kw)
    before = _gather(kv, [(0, p) for p in range(40)])
    pos = np.array([p + 1000 * s for s, p in rows])
    q_out = kv.append_rotary(rows, k, v, rot, q=q, positions=pos)
    want, mag = turn64(rot, q[:, :n].reshape(L, n, hq, d), pos)
    assert q_out.shape == (L, n, hq * d)
    close(q_out.view(L, n, hq, d), want, mag, torch.float32, "q")
    kg, vg = _gather(kv, rows)
    want, mag = turn64(rot, k[:, :n].reshape(L, n, H, d), pos)
    err = (kg.double().view(L, n, H, d) - want).abs()
    assert (err <= f16_tol(want, mag)).all()
    assert torch.equal(vg, v[:, :n].cpu().half())
    # dims past rot_dim are the plain append's, bit for bit
    assert torch.equal(kg.view(L, n, H, d)[..., rot.rot_dim:], k[:, :n].reshape(L, n, H, d)[..., rot.rot_dim:].cpu().half())
    # rows that were not appended keep what they held
    after = _gather(kv, [(0, p) for p in range(40)])
    untouched = [p for p in range(40) if not (14 <= p < 35 or p == 39)]
    for x, y in zip(before, after):
        assert torch.equal(x[:, untouched], y[:, untouched])
    # one layer, rows' own positions, in place: the other layers stay
    kv.append_rotary(rows, k[1], v[1], rot, q=q[1], q_out=q[1], layer=1)
    own = [p for _, p in rows]
    want, mag = turn64(rot, k[1, :n].reshape(n, H, d), own)
    k1, _ = _gather(kv, rows, layer=1)
    assert ((k1.double().view(n, H, d) - want).abs() <= f16_tol(want, mag)).all()
    k2, _ = _gather(kv, rows)
    assert torch.equal(k2[0], kg[0]) and torch.equal(k2[2], kg[2])


def test_append_without_queries_at_position_zero_is_the_plain_append(gpu):
    opts = na.BatchOpts(n_layer=2, n_head=3, head_dim=64, kv_blocks=8, max_seqs=2, n_ctx=64, max_rows=32)
    g = torch.Generator().manual_seed(2)
    k, v = torch.randn((2, 20, 192), generator=g).cuda(), torch.randn((2, 20, 192), generator=g).cuda()
    rows = [(0, p) for p in range(20)]
    a, b = _filled(opts, (20,)), _filled(opts, (20,))
    a.append(rows, k, v)
    assert b.append_rotary(rows, k, v, na.Rotary(64), positions=np.zeros(20, int)) is None
    for x, y in zip(_gather(a, rows), _gather(b, rows)):
        assert torch.equal(x, y)


def test_append_many_rows_staged_plan(gpu):
    """More rows than the launch arguments hold, four heads to a thread."""
    H, d, n = 12, 64, 2500
    opts = na.BatchOpts(n_layer=1, n_head=H, head_dim=d, kv_blocks=160, max_seqs=1, n_ctx=2512, max_rows=4096)
    kv = _filled(opts, (n,))
    g = torch.Generator().manual_seed(4)
    q, k, v = (torch.randn((n, H * d), generator=g).cuda() for _ in range(3))
    rot = na.Rotary(d)
    rows = [(0, p) for p in range(n)]
    q_out = kv.append_rotary(rows, k, v, rot, q=q, layer=0)
    want, mag = turn64(rot, q.view(n, H, d), range(n))
    close(q_out.view(n, H, d), want, mag, torch.float32)
    kg, vg = _gather(kv, rows, layer=0)
    want, mag = turn64(rot, k.view(n, H, d), range(n))
    assert ((kg.double().view(n, H, d) - want).abs() <= f16_tol(want, mag)).all()
    assert torch.equal(vg, v.cpu().half())


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("kw", [{}, dict(interleaved=True, rot_dim=32), dict(rot_dim=16)])
def test_append_q8(gpu, d, kw):
    """The stored bytes are ni_kv_append's of the rotated keys: the scale within
    the rotated values' error of amax / 127, the values within half a step and
    that error of it."""
    L, H = 2, 3
    opts = na.BatchOpts(n_layer=L, n_head=H, head_dim=d, kv_blocks=8, max_seqs=2, n_ctx=64, max_rows=32, q8=True)
    kv = _filled(opts, (30, 3))
    rows = [(0, p) for p in range(25)] + [(1, 2)]
    n = len(rows)
    g = torch.Generator().manual_seed(d)
    k, v = torch.randn((L, n, H * d), generator=g).cuda(), torch.randn((L, n, H * d), generator=g).cuda()
    k[0, 0] = 0
    rot = na.Rotary(d, **kw)
    kv.append_rotary(rows, k, v, rot, positions=np.arange(n) * 7)
    (kq, vq), (ks, vs) = kv.gather_q8(rows)
    want, mag = turn64(rot, k.view(L, n, H, d), np.arange(n) * 7)
    slack = 8 * 2.0 ** -24 * mag.amax(-1, keepdim=True)
    scale = want.abs().amax(-1, keepdim=True) / 127
    ks, kq = ks.double().cpu()[..., None], kq.double().cpu().view(L, n, H, d)
    assert ((ks - scale).abs() <= slack / 127 + 2.0 ** -23 * scale).all()
    assert ((kq * ks - want).abs() <= ks * 0.5 * (1 + 2.0 ** -20) + slack + 2.0 ** -22 * want.abs()).all()
    other = _filled(opts, (30, 3))
    other.append(rows, k, v)
    (_, vq2), (_, vs2) = other.gather_q8(rows)
    assert torch.equal(vq, vq2) and torch.equal(vs, vs2)


def test_append_refusals(gpu):
    opts = na.BatchOpts(n_layer=1, n_head=2, head_dim=64, kv_blocks=8, max_seqs=2, n_ctx=64, max_rows=8)
    kv = _filled(opts, (20, 5))
    x = torch.zeros((8, 128), device=gpu)
    rot = na.Rotary(64)

    def refused(what, *args, **kw):
        with pytest.raises(na.KvError, match=what):
            kv.append_rotary(*args, layer=0, **kw)

    refused("heads of 128", [(0, 0)], x, x, na.Rotary(128))
    refused("rot_dim 20", [(0, 0)], x, x, na.Rotary(64, rot_dim=20))
    refused("appears twice", [(0, 0), (0, 1), (0, 0)], x, x, rot)
    refused("no page", [(1, 16)], x, x, rot)
    refused("out of range", [(2, 0)], x, x, rot)
    refused("max_rows", [(0, p) for p in range(9)], torch.zeros((9, 128), device=gpu), torch.zeros((9, 128), device=gpu), rot)
    refused("16-byte aligned", [(0, 0)], torch.zeros(132, device=gpu)[1:129].view(1, 128),
            torch.zeros(132, device=gpu)[1:129].view(1, 128), rot)
    refused("overlap", [(0, 0), (0, 1)], x, x, rot, q=x, q_out=x[:1].expand(8, 128))
    with pytest.raises(na.KvError, match="layer 1 out of range"):
        kv.append_rotary([(0, 0)], x, x, rot, layer=1)
    kv.append_rotary([(0, 0), (0, 1)], x, x, rot, layer=0)  # a refused call leaves nothing behind
    kv.append_rotary([], x, x, rot, layer=0)


@pytest.mark.parametrize("rows,heads", [(5, 1), (1500, 6)])
def test_far_positions_against_the_definition(gpu, rows, heads):
    """Angles from frequencies of the definition, in 50 digits: near 2^32 the
    table adds 2^-31 turns, 2 pi 2^-31 of |x1| + |x2|, below a twentieth of
    2^-24 and so within what the tolerance's eight roundings leave."""
    import decimal

    D = decimal.Decimal
    pi = D("3.14159265358979323846264338327950288419716939937510582097494459")
    rot = na.Rotary(64)
    x = torch.randn((rows, heads, 64), generator=torch.Generator().manual_seed(2))
    pos = [(1 << 32) - rows + i for i in range(rows)]
    with decimal.localcontext() as c:
        c.prec = 50
        w = [D(10000) ** (-D(2 * i) / 64) / (2 * pi) for i in range(32)]
        ang = torch.tensor([[float(p * f % 1) for f in w] for p in pos], dtype=torch.float64) * 2 * np.pi
    c, s = torch.cos(ang)[:, None], torch.sin(ang)[:, None]
    a, b = x.double()[..., :32], x.double()[..., 32:]
    want, mag = torch.cat([a * c - b * s, b * c + a * s], 2), (a.abs() + b.abs()).repeat(1, 1, 2)
    got = na.rotary(x.view(rows, -1).cuda(), rot, heads, pos0=pos[0])
    close(got.view(rows, heads, 64), want, mag, torch.float32)


def _resident_mb():
    for line in open("/proc/self/status"):
        if line.startswith("VmRSS"):
            return int(line.split()[1]) / 1024


def test_a_place_written_twice_among_many_rows(gpu):
    """Found whichever rows they are, with host memory that follows the rows
    of a call and not the pages of the pool."""
    def cache(pages):
        kv = na.PagedKv(na.BatchOpts(n_layer=1, n_head=1, head_dim=64, kv_blocks=pages, max_seqs=64, n_ctx=64, max_rows=4096))
        for s in range(64):
            kv.reserve(kv.add_seq(), 64)
        return kv

    rot, x = na.Rotary(64), torch.zeros((4096, 64), device=gpu)
    rows = np.array([(s, p) for s in range(64) for p in range(64)], dtype=np.uint32)
    rng = np.random.default_rng(5)
    cache(300).append_rotary(rows, x, x, rot, layer=0)
    kv = cache(1 << 20)
    torch.cuda.synchronize()
    before = _resident_mb()
    kv.append_rotary(rows[:64], x, x, rot, layer=0)
    assert _resident_mb() - before < 16
    for n in (2, 3, 17, 500, 4096):
        some = rng.permutation(rows)[:n].copy()
        kv.append_rotary(some, x, x, rot, layer=0)
        i, j = rng.choice(n, 2, replace=False)
        some[i] = some[j]
        with pytest.raises(na.KvError, match="appears twice"):
            kv.append_rotary(some, x, x, rot, layer=0)
