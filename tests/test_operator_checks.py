"""Refusals and host arithmetic of the rotary, shared-prefix and verification
calls, without a GPU: every check comes before anything touches the device."""
import ctypes as C
import decimal
import math

import numpy as np
import pytest
import torch

import nanoinfer_amd as na
from nanoinfer_amd import _abi, drivers


def _err(L):
    return L.ni_kv_last_error(None).decode()


# ------------------------------------------------------------------- rotary


def _turns(r):
    return [int(r._r.turns[i]) for i in range(r.rot_dim // 2)]


def _frac_turns(freq):
    """freq / 2 pi modulo a turn, in 2^-64 turns."""
    return [int((f / (2 * math.pi)) % 1.0 * 2.0 ** 64) for f in freq]


@pytest.mark.parametrize("head_dim,rot_dim,kw", [
    (64, None, {}), (128, 64, dict(interleaved=True)), (80, 20, {}), (2, None, {}), (256, None, dict(base=1e6)),
    (64, None, dict(base=0.5)),
    (64, 32, dict(scaling="linear", factor=4.0)), (128, None, dict(scaling="ntk", factor=8.0, base=500000.0)),
    (128, None, dict(scaling="yarn", factor=8.0, orig_ctx=8192)), (64, 16, dict(scaling="yarn", factor=2.5, orig_ctx=2048)),
    (64, None, dict(scaling="yarn", factor=1.0, orig_ctx=2048)),
])
def test_rotary_frequencies(head_dim, rot_dim, kw):
    r = na.Rotary(head_dim, rot_dim=rot_dim, **kw)
    d, base, s = rot_dim or head_dim, kw.get("base", 10000.0), kw.get("factor", 1.0)
    i = np.arange(d // 2, dtype=np.float64)
    want_scale = 1.0
    if kw.get("scaling") == "ntk":
        base = base * s ** (d / (d - 2))
    f = base ** (-2 * i / d)
    if kw.get("scaling") == "linear":
        f = f / s
    if kw.get("scaling") == "yarn":
        turns_at = lambda n: d * math.log(kw["orig_ctx"] / (n * 2 * math.pi)) / (2 * math.log(base))
        lo, hi = max(math.floor(turns_at(32)), 0), min(math.ceil(turns_at(1)), d - 1)
        ramp = np.clip((i - lo) / max(hi - lo, 0.001), 0, 1)
        f = f / s * ramp + f * (1 - ramp)
        want_scale = 0.1 * math.log(s) + 1
    # Frequencies agree to a few 64-bit roundings (2^-53 of themselves, each).
    for got, want, x in zip(_turns(r), _frac_turns(f), f):
        diff = (got - want) % (1 << 64)
        assert min(diff, (1 << 64) - diff) <= 16 * 2.0 ** -53 * max(x, 1e-300) / (2 * math.pi) * 2.0 ** 64 + 2
    assert r.scale == pytest.approx(want_scale, rel=2.0 ** -23)
    assert r.rot_dim == d


PI = decimal.Decimal("3.14159265358979323846264338327950288419716939937510582097494459230781640628620899862803")


def _decimal_turns(d, base=10000.0, scaling=None, factor=1.0, orig_ctx=0):
    """f_i / 2 pi modulo a turn, to 50 digits."""
    with decimal.localcontext() as c:
        c.prec = 60
        D = decimal.Decimal
        b, s = D(base), D(factor)
        if scaling == "ntk":
            b *= s ** (D(d) / D(d - 2))
        f = [b ** (-2 * D(i) / d) for i in range(d // 2)]
        if scaling == "linear":
            f = [x / s for x in f]
        if scaling == "yarn":
            at = lambda n: d * (D(orig_ctx) / (n * 2 * PI)).ln() / (2 * b.ln())
            lo = max(at(32).to_integral_value(decimal.ROUND_FLOOR), D(0))
            hi = min(at(1).to_integral_value(decimal.ROUND_CEILING), D(d - 1))
            ramp = [min(max((i - lo) / max(hi - lo, D("0.001")), D(0)), D(1)) for i in range(d // 2)]
            f = [x / s * r + x * (1 - r) for x, r in zip(f, ramp)]
        return [x / (2 * PI) % 1 for x in f]


@pytest.mark.parametrize("head_dim,kw", [
    (64, {}), (128, {}), (256, dict(base=1e6)), (80, dict(base=500000.0)), (2, {}), (128, dict(base=1.0)),
    (64, dict(scaling="linear", factor=5.5)), (128, dict(scaling="ntk", factor=8.0, base=500000.0)),
    (4, dict(scaling="ntk", factor=4.0)),
    (128, dict(scaling="yarn", factor=8.0, orig_ctx=8192)), (64, dict(scaling="yarn", factor=2.5, orig_ctx=2048)),
])
def test_rotary_frequencies_to_the_tables_last_bits(head_dim, kw):
    """Within two units of 2^-64 turns: the roundings of 2^-64 of f / 2 pi, at
    most 0.16 turns (2 of the power, 1 of the exponent, which shrinks with f, 2
    of the quotient by 2 pi, up to 4 of a scaling), and half a unit."""
    got, want = _turns(na.Rotary(head_dim, **kw)), _decimal_turns(head_dim, **kw)
    for i, (g, w) in enumerate(zip(got, want)):
        off = (decimal.Decimal(g) - w * 2 ** 64) % 2 ** 64
        off = min(off, 2 ** 64 - off)
        assert off <= 2, f"pair {i}: {off:.1f} units"


def test_rotary_attn_scale_replaces_the_scalings_own():
    assert na.Rotary(64, scaling="yarn", factor=4.0, orig_ctx=2048, attn_scale=1.5).scale == 1.5


@pytest.mark.parametrize("kw,what", [
    (dict(head_dim=63), "head_dim 63"), (dict(head_dim=0), "head_dim 0"), (dict(head_dim=258), "head_dim 258"),
    (dict(head_dim=64, rot_dim=66), "rot_dim 66"), (dict(head_dim=64, rot_dim=7), "rot_dim 7"),
    (dict(head_dim=64, base=0.0), "base"), (dict(head_dim=64, base=float("nan")), "base"),
    (dict(head_dim=64, base=float("inf")), "base"),
    (dict(head_dim=64, scaling="linear", factor=0.5), "factor"),
    (dict(head_dim=64, scaling="linear", factor=float("inf")), "factor"),
    (dict(head_dim=64, rot_dim=2, scaling="ntk", factor=2.0), "rot_dim above 2"),
    (dict(head_dim=64, scaling="yarn", factor=2.0), "orig_ctx"),
    (dict(head_dim=64, base=1.0, scaling="yarn", factor=2.0, orig_ctx=64), "base above 1"),
    (dict(head_dim=64, scaling="yarn", factor=2.0, orig_ctx=64, beta_fast=1.0, beta_slow=2.0), "beta_fast"),
    (dict(head_dim=64, attn_scale=float("inf")), "attn_scale"),
])
def test_rotary_refusals(kw, what):
    with pytest.raises(na.KvError) as e:
        na.Rotary(**kw)
    assert e.value.code == _abi.NI_ERR_BAD_ARG and what in str(e.value)


@pytest.mark.parametrize("kw", [dict(head_dim=64, scaling="other"), dict(head_dim=64, rot_dim=0),
                                dict(head_dim=-2), dict(head_dim=64, attn_scale=0.0), dict(head_dim=64, beta_fast=0.0)])
def test_rotary_python_refusals(kw):
    with pytest.raises(ValueError):
        na.Rotary(**kw)


def test_rotary_apply_refuses_before_any_launch():
    L = _abi.lib()
    r = na.Rotary(64)
    buf = (C.c_float * 256)()
    p = C.addressof(buf)
    p += -p % 16
    call = lambda rot, dt, x, xs, o, os, n, h, pos=None: L.ni_rotary_apply(rot, dt, x, xs, o, os, n, h, pos, 0, None)
    assert call(None, 0, p, 64, p, 64, 1, 1) == _abi.NI_ERR_BAD_ARG and "rotary is NULL" in _err(L)
    empty = _abi.ni_rotary()
    assert call(C.byref(empty), 0, p, 64, p, 64, 1, 1) == _abi.NI_ERR_BAD_ARG and "ni_rotary_init" in _err(L)
    assert call(r.ref, 3, p, 64, p, 64, 1, 1) == _abi.NI_ERR_BAD_ARG and "type" in _err(L)
    assert call(r.ref, 0, None, 64, p, 64, 1, 1) == _abi.NI_ERR_BAD_ARG and "x is NULL" in _err(L)
    assert call(r.ref, 0, p, 64, None, 64, 1, 1) == _abi.NI_ERR_BAD_ARG and "out is NULL" in _err(L)
    assert call(r.ref, 0, p + 2, 64, p, 64, 1, 1) == _abi.NI_ERR_BAD_ARG and "aligned" in _err(L)
    assert call(r.ref, 1, p, 64, p + 1, 64, 1, 1) == _abi.NI_ERR_BAD_ARG and "aligned" in _err(L)
    assert call(r.ref, 0, p, -64, p, 64, 2, 1) == _abi.NI_ERR_BAD_ARG and "non-negative" in _err(L)
    assert call(r.ref, 0, p, 64, p, 64, 2, 2) == _abi.NI_ERR_BAD_ARG and "overlap" in _err(L)
    assert call(r.ref, 0, p, 64, p, 64, 1, 1, p + 2) == _abi.NI_ERR_BAD_ARG and "positions" in _err(L)
    assert call(r.ref, 0, p, 1 << 33, p, 1 << 33, 1 << 31, 1 << 10) == _abi.NI_ERR_BAD_ARG and "too large" in _err(L)
    assert call(r.ref, 0, p, 128, p, 64, 2, 1) == _abi.NI_ERR_BAD_ARG and "with x's stride" in _err(L)
    # a launch holds less than 2^32 threads
    assert call(r.ref, 0, p, 1 << 12, p, 1 << 12, 1 << 20, 1 << 6) == _abi.NI_ERR_BAD_ARG and "too large" in _err(L)
    assert call(r.ref, 0, None, 64, None, 64, 0, 1) == _abi.NI_OK
    assert call(r.ref, 0, None, 64, None, 64, 1, 0) == _abi.NI_OK


def test_rotary_wrapper_refuses_what_it_cannot_rotate():
    r = na.Rotary(64)
    x = torch.zeros((3, 128))
    with pytest.raises(TypeError):
        na.rotary(x.double(), r, 2)
    with pytest.raises(TypeError):
        na.rotary(x[0], r, 2)
    with pytest.raises(ValueError):
        na.rotary(x, r, 3)
    with pytest.raises(ValueError):
        na.rotary(x.t().contiguous().t(), r, 2)
    with pytest.raises(TypeError):
        na.rotary(x, r, 2, positions=torch.arange(3))
    with pytest.raises(ValueError):
        na.rotary(x, r, 2, positions=torch.arange(2, dtype=torch.int32))
    with pytest.raises(ValueError):
        na.rotary(x, r, 2, pos0=-1)
    with pytest.raises(ValueError):
        na.rotary(x, r, 2, out=torch.zeros((2, 128)))
    with pytest.raises(ValueError):
        na.rotary(x, r, 2, out=torch.zeros((3, 128), dtype=torch.float16))
    with pytest.raises(TypeError, match="CUDA"):
        na.rotary(x, r, 2)


# ------------------------------------------------- append, prefix attention


def _host_kv(**kw):
    return na.PagedKv(na.BatchOpts(n_layer=2, n_head=2, head_dim=64, kv_blocks=16, max_seqs=4, n_ctx=64, max_rows=8,
                                   host_only=True, **kw))


def test_host_only_handle_refuses_the_new_calls():
    kv = _host_kv()
    s = kv.add_seq()
    kv.reserve(s, 1)
    rows = (_abi.ni_row * 1)(_abi.ni_row(s, 0))
    r = na.Rotary(64)
    rc = kv._L.ni_kv_append_rotary(kv.handle, -1, rows, 1, r.ref, None, None, None, 0, 0, None, 0, 0, 0, None, 0, 0, None)
    assert rc == _abi.NI_ERR_NO_DEVICE
    pre = (_abi.ni_prefix * 1)(_abi.ni_prefix(0, 0, 1))
    rc = kv._L.ni_kv_prefix_attention(kv.handle, -1, None, 0, 0, 2, rows, 1, pre, 1, None, 0, 0, 0, None)
    assert rc == _abi.NI_ERR_NO_DEVICE
    assert kv._L.ni_kv_append_rotary(None, -1, rows, 1, r.ref, None, None, None, 0, 0, None, 0, 0, 0, None, 0, 0,
                                     None) == _abi.NI_ERR_BAD_ARG
    assert kv._L.ni_kv_prefix_attention(None, -1, None, 0, 0, 2, rows, 1, pre, 1, None, 0, 0, 0,
                                        None) == _abi.NI_ERR_BAD_ARG


def test_wrappers_refuse_bad_layouts_on_the_host():
    kv = _host_kv()
    rows, k = [(0, 0), (0, 1)], torch.zeros((2, 2, 128))
    r = na.Rotary(64)
    with pytest.raises(ValueError, match="share strides"):
        kv.append_rotary(rows, k, torch.zeros((2, 2, 256))[..., :128], r)
    with pytest.raises(ValueError, match="k is"):
        kv.append_rotary(rows, k[:, :1], k, r)
    for bad in ([0], [0, -1], [0.5, 1], [0, 1 << 32]):
        with pytest.raises(ValueError, match="positions"):
            kv.append_rotary(rows, k, k, r, positions=bad)
    with pytest.raises(ValueError, match="whole heads"):
        kv.append_rotary(rows, k, k, r, q=torch.zeros((2, 2, 100)))
    with pytest.raises(ValueError, match="q_out is"):
        kv.append_rotary(rows, k, k, r, q=torch.zeros((2, 2, 256)), q_out=torch.zeros((2, 2, 128)))
    with pytest.raises(ValueError, match="without q"):
        kv.append_rotary(rows, k, k, r, q_out=torch.zeros((2, 2, 128)))
    with pytest.raises(TypeError):
        kv.append_rotary(rows, k, k, r)  # host tensors
    with pytest.raises(ValueError, match="prefixes"):
        kv.prefix_attention(k, rows, [(0, -1, 2)])
    with pytest.raises(ValueError, match="whole heads"):
        kv.prefix_attention(torch.zeros((2, 2, 100)), rows, [(0, 0, 2)])
    with pytest.raises(ValueError, match="out is"):
        kv.prefix_attention(k, rows, [(0, 0, 2)], out=torch.zeros((2, 1, 128)))
    with pytest.raises(TypeError):
        kv.prefix_attention(k, rows, [(0, 0, 2)])


# ------------------------------------------------------------- verification


def _verify_call(**kw):
    L = _abi.lib()
    buf = (C.c_float * 4096)()
    p = C.addressof(buf)
    p += -p % 16
    a = dict(dtype=0, target=p, tss=300, trs=100, draft=p, dss=200, drs=100, drafted=p, ds=2, n_drafts=None, au=p, aus=2,
             su=p, n_seq=2, n_draft=2, vocab=100, accepted=p, tokens=p, ts=3, work=p, wb=1 << 20)
    a.update(kw)
    rc = L.ni_verify_drafts(a["dtype"], a["target"], a["tss"], a["trs"], a["draft"], a["dss"], a["drs"], a["drafted"],
                            a["ds"], a["n_drafts"], a["au"], a["aus"], a["su"], a["n_seq"], a["n_draft"], a["vocab"],
                            a["accepted"], a["tokens"], a["ts"], a["work"], a["wb"], None)
    return rc, _err(L), p


@pytest.mark.parametrize("kw,what", [
    (dict(dtype=3), "type"), (dict(vocab=0), "vocab"), (dict(vocab=(1 << 30) + 1), "vocab"), (dict(n_seq=65536), "65535"),
    (dict(n_draft=(1 << 20) + 1), "n_draft"), (dict(target=None), "target is NULL"), (dict(drafted=None), "drafted is NULL"),
    (dict(au=None), "accept_u is NULL"), (dict(su=None), "sample_u is NULL"), (dict(accepted=None), "accepted is NULL"),
    (dict(tokens=None), "tokens is NULL"), (dict(trs=-1), "target must have"), (dict(dss=-4), "draft must have"),
    (dict(ts=2), "overlap"), (dict(work=None), "workspace"), (dict(wb=31), "workspace must be 32 bytes"),
])
def test_verify_refusals(kw, what):
    rc, msg, _ = _verify_call(**kw)
    assert rc == _abi.NI_ERR_BAD_ARG and what in msg


def test_verify_refuses_misaligned_pointers():
    _, _, p = _verify_call(vocab=0)
    for name in ("target", "draft", "drafted", "n_drafts", "au", "su", "accepted", "tokens", "work"):
        buf = (C.c_float * 16)()
        q = C.addressof(buf) + 2 if name != "work" else C.addressof(buf) // 16 * 16 + 8
        rc, msg, _ = _verify_call(**{name: q})
        assert rc == _abi.NI_ERR_BAD_ARG and "align" in msg, name


def test_verify_refuses_answers_over_its_inputs():
    other = (C.c_int32 * 64)()
    q = C.addressof(other)
    for kw in (dict(n_drafts=q, accepted=q), dict(tokens=q, drafted=q)):
        rc, msg, _ = _verify_call(**kw)
        assert rc == _abi.NI_ERR_BAD_ARG and "share" in msg


def test_verify_workspace_and_nothing_to_do():
    L = _abi.lib()
    assert L.ni_verify_workspace(3, 1) == 3 * 16
    assert L.ni_verify_workspace(1, 2048) == 16 and L.ni_verify_workspace(1, 2049) == 32
    assert L.ni_verify_workspace(0, 5) == 0
    rc, _, _ = _verify_call(n_seq=0)
    assert rc == _abi.NI_OK


def test_verify_wrapper_refusals():
    b, k, v = 2, 3, 50
    t, d = torch.zeros((b, k + 1, v)), torch.zeros((b, k), dtype=torch.int32)
    u, s = torch.zeros((b, k)), torch.zeros(b)
    with pytest.raises(TypeError):
        na.verify_drafts(t.double(), d, u, s)
    with pytest.raises(TypeError):
        na.verify_drafts(t, d.long(), u, s)
    with pytest.raises(TypeError):
        na.verify_drafts(t, d, u, s, draft=torch.zeros((b, k, v), dtype=torch.float16))
    with pytest.raises(ValueError):
        na.verify_drafts(t, d, u, s, draft=torch.zeros((b, k + 1, v)))
    with pytest.raises(ValueError):
        na.verify_drafts(t.transpose(1, 2).contiguous().transpose(1, 2), d, u, s)
    with pytest.raises(ValueError):
        na.verify_drafts(t[:, :0], d, u, s)
    with pytest.raises(ValueError):
        na.verify_drafts(t, d[:, :2], u, s)
    with pytest.raises(ValueError):
        na.verify_drafts(t, d, u, s[:1])
    with pytest.raises(ValueError):
        na.verify_drafts(t, d, u, s, tokens=torch.zeros((b, k), dtype=torch.int32))
    with pytest.raises(TypeError, match="CUDA"):
        na.verify_drafts(t, d, u, s)


# ------------------------------------------------------------ verify driver


def test_spec_commit_takes_the_callers_numbers():
    kv = na.PagedKv(na.BatchOpts(kv_blocks=32, max_seqs=3, n_ctx=256, max_rows=64, host_only=True))
    seqs = [kv.add_seq() for _ in range(3)]
    for s, n in zip(seqs, (5, 16, 30)):
        kv.reserve(s, n)
        kv.commit(s, n)
    sp = drivers.Spec(kv, seqs, 4, 1)

    def round_(accepted):
        work, _ = sp.plan()
        for s, n, _ in np.asarray(work).tolist():
            kv.reserve(s, kv.seq_len(s) + n)
            kv.commit(s, n)
        return sp.commit(accepted)

    assert round_([0, 4, 2]) == [0, 4, 2]
    assert [kv.seq_len(s) for s in seqs] == [6, 21, 33]
    assert round_(torch.tensor([1, 0, 4], dtype=torch.int32)) == [1, 0, 4]
    assert [kv.seq_len(s) for s in seqs] == [8, 22, 38]
    work, _ = sp.plan()
    for s, n, _ in np.asarray(work).tolist():
        kv.reserve(s, kv.seq_len(s) + n)
        kv.commit(s, n)
    with pytest.raises(Exception, match="5 drafts accepted of 4"):
        sp.commit([0, 0, 5])
    assert [kv.seq_len(s) for s in seqs] == [13, 27, 43]  # nothing truncated
    for bad in ([0, 0], [0, -1, 0], [0, 1 << 32, 0]):
        with pytest.raises(ValueError):
            sp.commit(bad)
    assert sp.commit([0, 0, 0]) == [0, 0, 0]
    with pytest.raises(Exception, match="without a planned round"):
        sp.commit([0, 0, 0])


def test_spec_commit_refuses_what_is_no_integer():
    """1.9 accepted drafts are not 1, nor is 2^64 - 1 a small number."""
    kv = na.PagedKv(na.BatchOpts(kv_blocks=32, max_seqs=2, n_ctx=256, max_rows=64, host_only=True))
    seqs = [kv.add_seq() for _ in range(2)]
    for s in seqs:
        kv.reserve(s, 5)
        kv.commit(s, 5)
    sp = drivers.Spec(kv, seqs, 4, 1)
    work, _ = sp.plan()
    for s, n, _ in np.asarray(work).tolist():
        kv.reserve(s, kv.seq_len(s) + n)
        kv.commit(s, n)
    for bad in ([0.0, 1.9], [0, float("nan")], torch.tensor([1.0, 2.5]), [False, True], ["0", "1"],
                np.array([0, 2 ** 64 - 1], dtype=np.uint64)):
        with pytest.raises(ValueError):
            sp.commit(bad)
    assert [kv.seq_len(s) for s in seqs] == [10, 10]
    assert sp.commit(np.array([0, 4], dtype=np.uint64)) == [0, 4]
    assert [kv.seq_len(s) for s in seqs] == [6, 10]


def test_prefixes_are_integers():
    kv = _host_kv()
    q = torch.zeros((2, 2, 128))
    for bad in ((0, 1.5, 2), (0, "1", 2), (0, None, 2)):
        with pytest.raises(TypeError, match="integer"):
            kv.prefix_attention(q, [(0, 0), (0, 1)], [bad])
    with pytest.raises(TypeError, match="CUDA"):  # as far as integers of any kind get on the host
        kv.prefix_attention(q, [(0, 0), (0, 1)], [(np.uint32(0), torch.tensor(0), 2)])


def test_a_stream_of_another_device_is_refused():
    """Its context would make that device the current one, and the launch its."""
    from nanoinfer_amd import batch

    other = type("S", (), dict(cuda_stream=64, stream_id=3, device_index=1))()
    with pytest.raises(ValueError, match="the stream is of cuda:1"):
        batch._on(0, other)


def test_verify_refuses_answers_that_share_any_value_with_its_inputs():
    """Views of one buffer, at every shift that overlaps (none of these calls
    gets as far as a launch)."""
    names = dict(drafted=("drafted", "ds"), accept_u=("au", "aus"), sample_u=("su", None), n_drafts=("n_drafts", None))
    n, k = 3, 4

    def buffer():
        b = (C.c_int32 * 512)()
        return b, C.addressof(b) + -C.addressof(b) % 16

    keep, at = zip(*[buffer() for _ in range(9)])
    base = dict(target=at[0], draft=None, drafted=at[1], ds=k, au=at[2], aus=k, su=at[3], n_drafts=at[4],
                accepted=at[5], tokens=at[6], ts=k + 1, work=at[7], n_seq=n, n_draft=k, vocab=9, tss=45, trs=9)
    cells = lambda p, stride, width: {p + 4 * (i * stride + j) for i in range(n) for j in range(width)}
    seen = 0
    for what, (name, stride_name) in names.items():
        for shift in range(-24, 25):
            for ts in (5, 6, 9, 11):
                for stride in ((0, 4, 6, 11) if stride_name else (1,)):
                    p = at[8] + 4 * (100 + shift)
                    kw = dict(base, tokens=at[8] + 400, ts=ts, **{name: p}, **({stride_name: stride} if stride_name else {}))
                    if not cells(p, stride, k if stride_name else 1) & cells(at[8] + 400, ts, k + 1):
                        continue
                    rc, msg, _ = _verify_call(**kw)
                    assert rc == _abi.NI_ERR_BAD_ARG and f"tokens may not share memory with {what}" in msg, (kw, msg)
                    seen += 1
        for shift in (-1, 0, 1):
            kw = dict(base, accepted=at[8] + 400, **{name: at[8] + 4 * (100 + shift)})
            if stride_name is None or shift <= 0:
                rc, msg, _ = _verify_call(**kw)
                assert rc == _abi.NI_ERR_BAD_ARG and f"accepted may not share memory with {what}" in msg
    rc, msg, _ = _verify_call(**dict(base, accepted=at[6] + 4))
    assert rc == _abi.NI_ERR_BAD_ARG and "tokens may not share memory with accepted" in msg
    assert seen > 500
