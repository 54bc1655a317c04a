"""Verification of drafted tokens against its definition in 64 bits, sequence
by sequence.  The outputs are whole numbers and must be equal: the comparisons
are exact in 64 bits, and the sums are ~2^-45 of the whole off, which a uniform
number of 24 bits falls into about once in 2^20 draws; the seeds are fixed."""
import numpy as np
import pytest
import torch

import nanoinfer_amd as na

pytestmark = pytest.mark.gpu


def expect(target, drafted, accept_u, sample_u, draft=None, n_drafts=None):
    t, d = target.double().cpu().numpy(), None if draft is None else draft.double().cpu().numpy()
    drafted, au, su = drafted.cpu().numpy(), accept_u.cpu().double().numpy(), sample_u.cpu().double().numpy()
    b, k1, v = t.shape
    acc, tok = np.zeros(b, np.int32), np.full((b, k1), -1, np.int32)
    for s in range(b):
        n = k1 - 1 if n_drafts is None else min(max(int(n_drafts[s]), 0), k1 - 1)
        a = 0
        while a < n:
            x = drafted[s, a]
            if not 0 <= x < v or not au[s, a] * (1.0 if d is None else d[s, a, x]) < t[s, a, x]:
                break
            tok[s, a] = x
            a += 1
        clean = lambda w: np.where(w > 0, w, 0.0)
        w = clean(t[s, a])
        if a < n:
            if d is None:
                r = w.copy()
                if 0 <= drafted[s, a] < v:
                    r[drafted[s, a]] = 0
            else:
                r = clean(t[s, a] - d[s, a])
            if r.sum() > 0:
                w = r
        c = np.cumsum(w)
        acc[s] = a
        if c[-1] > 0:
            past = np.flatnonzero((c > su[s] * c[-1]) & (w > 0))
            tok[s, a] = past[0] if len(past) else np.flatnonzero(w > 0)[-1]
    return acc, tok


def inputs(b, k, v, dtype=torch.float32, seed=0, spread=2.5, near=0.5):
    g = torch.Generator(device="cuda").manual_seed(seed)
    lt = torch.randn((b, k + 1, v), generator=g, device="cuda") * spread
    ld = lt[:, :k] + near * torch.randn((b, k, v), generator=g, device="cuda")
    noise = -torch.log(-torch.log(torch.rand((b, k, v), generator=g, device="cuda").clamp(1e-9, 1 - 1e-6)))
    drafted = (ld + noise).argmax(-1).to(torch.int32)
    return (torch.softmax(lt, -1).to(dtype), drafted, torch.rand((b, k), generator=g, device="cuda"),
            torch.rand((b,), generator=g, device="cuda"), torch.softmax(ld, -1).to(dtype))


def check(args, **kw):
    acc, tok = na.verify_drafts(*args, **kw)
    want = expect(*args, **kw)
    assert np.array_equal(acc.cpu().numpy(), want[0])
    assert np.array_equal(tok.cpu().numpy(), want[1])
    return want


@pytest.mark.parametrize("b,k,v", [(1, 1, 1), (1, 1, 2), (3, 2, 7), (2, 4, 2047), (2, 4, 2048), (2, 3, 2049), (5, 5, 4097),
                                   (64, 4, 1003), (1, 7, 50257), (4, 3, 131071), (2, 70, 300), (300, 2, 33)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_verify(gpu, b, k, v, dtype):
    t, d, au, su, q = inputs(b, k, v, dtype, seed=b * 1000 + v)
    acc, _ = check((t, d, au, su), draft=q)
    n = torch.from_numpy(np.random.default_rng(v).integers(-1, k + 2, b).astype(np.int32)).cuda()  # held to 0..k
    check((t, d, au, su), draft=q, n_drafts=n)
    check((t, d, au, su))  # a drafter that was certain


def test_all_accepted_and_none(gpu):
    t, d, au, su, q = inputs(6, 5, 999, seed=3)
    acc, _ = check((t, d, torch.zeros_like(au), su), draft=q)
    assert (acc == 5).all()
    t2 = t.clone()
    for s in range(6):
        t2[s, 0, d[s, 0]] = 0
    acc, _ = check((t2, d, torch.zeros_like(au), su), draft=q)
    assert (acc == 0).all()


def test_no_drafts_draws_from_the_target(gpu):
    t, _, _, su, _ = inputs(7, 1, 5003, seed=4)
    d, au = torch.zeros((7, 0), dtype=torch.int32, device=gpu), torch.zeros((7, 0), device=gpu)
    acc, tok = check((t[:, :1], d, au, su))
    assert (acc == 0).all() and tok.shape == (7, 1)
    assert na.verify_drafts(t[:0, :1], d[:0], au[:0], su[:0])[1].shape == (0, 1)


def test_ends_of_the_unit_interval_and_zero_weights(gpu):
    """u = 0 draws the first entry with weight, the largest u below 1 the last."""
    v = 6000
    t = torch.zeros((2, 1, v), device=gpu)
    t[:, 0, [17, 2100, 4097, 5000]] = torch.tensor([0.25, 0.5, 0.125, 0.125], device=gpu)
    d, au = torch.zeros((2, 0), dtype=torch.int32, device=gpu), torch.zeros((2, 0), device=gpu)
    su = torch.tensor([0.0, 1 - 2.0 ** -24], device=gpu)
    _, tok = check((t, d, au, su))
    assert tok[:, 0].tolist() == [17, 5000]
    # a border of the sums belongs to the entry after it
    _, tok = check((t, d, au, torch.tensor([0.25, 0.75], device=gpu)))
    assert tok[:, 0].tolist() == [2100, 4097]


def test_target_under_the_drafter_draws_from_the_target(gpu):
    """Equal rows and a rejected token: nothing is left of the difference."""
    t, d, au, su, _ = inputs(4, 2, 700, seed=6)
    q = t[:, :2].clone()
    au = torch.ones_like(au)  # (u = 1 rejects where p = q)
    acc, tok = check((t, d, au, su), draft=q)
    assert (acc == 0).all() and (tok[:, 0] >= 0).all()


def test_bad_values_stay_in_bounds(gpu):
    """Tokens outside the vocabulary are rejected; NaN and negative
    probabilities weigh nothing; a row without any weight draws -1."""
    t, d, au, su, q = inputs(6, 3, 3001, seed=8)
    d = d.clone()
    d[0, 0], d[1, 1], d[2, 2] = -1, 3001, 2 ** 31 - 1
    check((t, d, torch.zeros_like(au), su), draft=q)
    check((t, d, torch.zeros_like(au), su))
    t2 = t.clone()
    t2[3, :, 100:2500] = float("nan")
    t2[4, :, ::2] = -1.0
    t2[5] = 0.0
    acc, tok = check((t2, d, au, su), draft=q)
    assert tok[5, 0] == -1
    t2[5] = float("nan")
    _, tok = check((t2, d, au, su), draft=q)
    assert tok[5, 0] == -1
    # infinities: some entry of the row (what is drawn is not defined)
    t3 = t.clone()
    t3[:, :, 7] = float("inf")
    _, tok = na.verify_drafts(t3, d, au, su, draft=q)
    tok = tok.cpu().numpy()
    assert ((tok >= -1) & (tok < 3001)).all()


def test_strided_inputs_and_given_outputs(gpu):
    b, k, v = 3, 4, 1500
    t, d, au, su, q = inputs(b, k, v, torch.float16, seed=9)
    big = torch.zeros((b, 9, v + 5), dtype=torch.float16, device=gpu)
    big[:, 2:2 + k + 1, 3:3 + v] = t
    qb = torch.zeros((b, k, v + 1), dtype=torch.float16, device=gpu)
    qb[..., 1:] = q
    db = torch.full((b, k + 3), -7, dtype=torch.int32, device=gpu)
    db[:, 1:1 + k] = d
    acc = torch.full((b,), 99, dtype=torch.int32, device=gpu)
    tokb = torch.full((b + 1, k + 4), 77, dtype=torch.int32, device=gpu)
    tok = tokb[:b, 1:k + 2]
    got = na.verify_drafts(big[:, 2:2 + k + 1, 3:3 + v], db[:, 1:1 + k], au, su, draft=qb[..., 1:], accepted=acc, tokens=tok)
    assert got[0] is acc and got[1] is tok
    want = expect(t, d, au, su, draft=q)
    assert np.array_equal(acc.cpu().numpy(), want[0]) and np.array_equal(tok.cpu().numpy(), want[1])
    assert (tokb[:, 0] == 77).all() and (tokb[:, k + 2:] == 77).all() and (tokb[b] == 77).all()


def test_one_sequence_of_a_column(gpu):
    """A dimension of one entry has no stride to hold to."""
    t, d, _, _, q = inputs(1, 4, 500, seed=10)
    u = torch.rand((1, 5), device=gpu)
    check((t, d, u[:, :4], u[:, 4]), draft=q)
    u = torch.rand((3, 2), device=gpu)
    t, d, _, _, q = inputs(3, 1, 500, seed=11)
    check((t, d, u[:, :1], u[:, 1].contiguous()), draft=q)


def test_the_tokens_follow_the_target(gpu):
    """Over many sequences alike the first token's frequencies are the target's
    (within 5 standard deviations of each count), whatever the drafter."""
    v, b = 8, 40000
    g = torch.Generator(device="cuda").manual_seed(1)
    p = torch.softmax(torch.randn(v, generator=g, device="cuda"), 0)
    q = torch.softmax(torch.randn(v, generator=g, device="cuda"), 0)
    d = torch.multinomial(q.expand(b, v), 1, generator=g).to(torch.int32)
    au, su = torch.rand((b, 1), generator=g, device="cuda"), torch.rand((b,), generator=g, device="cuda")
    _, tok = na.verify_drafts(p.expand(b, 2, v).contiguous(), d, au, su, draft=q.expand(b, 1, v).contiguous())
    count = torch.bincount(tok[:, 0].long(), minlength=v).double()
    want = p.double() * b
    assert ((count - want).abs() <= 5 * torch.sqrt(want * (1 - p.double()))).all()


def test_captured_and_replayed(gpu):
    t, d, au, su, q = inputs(8, 4, 9001, seed=12)
    acc, tok = torch.empty((8,), dtype=torch.int32, device=gpu), torch.empty((8, 5), dtype=torch.int32, device=gpu)
    na.verify_drafts(t, d, au, su, draft=q)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        na.verify_drafts(t, d, au, su, draft=q, accepted=acc, tokens=tok)
    for i in range(4):
        t2, d2, au2, su2, q2 = inputs(8, 4, 9001, seed=20 + i)
        for x, y in ((t, t2), (d, d2), (au, au2), (su, su2), (q, q2)):
            x.copy_(y)
        graph.replay()
        torch.cuda.synchronize()
        want = expect(t2, d2, au2, su2, draft=q2)
        assert np.array_equal(acc.cpu().numpy(), want[0]) and np.array_equal(tok.cpu().numpy(), want[1])
        check((t2, d2, au2, su2), draft=q2)  # eager work between the replays


def test_another_stream(gpu):
    t, d, au, su, q = inputs(16, 3, 20001, seed=13)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    acc, tok = na.verify_drafts(t, d, au, su, draft=q, stream=s)
    s.synchronize()
    want = expect(t, d, au, su, draft=q)
    assert np.array_equal(acc.cpu().numpy(), want[0]) and np.array_equal(tok.cpu().numpy(), want[1])


def test_any_object_with_a_streams_handle(gpu):
    """What the call allocates belongs to the stream it runs on, whatever names it."""
    from nanoinfer_amd import batch

    t, d, au, su, q = inputs(16, 3, 20001, seed=14)
    want = expect(t, d, au, su, draft=q)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    for stream in (s, torch.cuda.default_stream()):
        handle = type("S", (), dict(cuda_stream=stream.cuda_stream))()
        with batch._on(t.get_device(), handle) as at:
            assert at == stream.cuda_stream == torch.cuda.current_stream().cuda_stream
        assert torch.cuda.current_stream() == torch.cuda.default_stream()
        acc, tok = na.verify_drafts(t, d, au, su, draft=q, stream=handle)
        stream.synchronize()
        assert np.array_equal(acc.cpu().numpy(), want[0]) and np.array_equal(tok.cpu().numpy(), want[1])


def test_answers_beside_their_inputs_in_one_buffer(gpu):
    """Columns of one buffer share no value: [drafted | tokens | other], any order."""
    t, d, au, su, q = inputs(9, 4, 700, seed=15)
    want = expect(t, d, au, su, draft=q)
    for first, second in ((0, 4), (5, 0)):
        buf = torch.full((9, 12), -7, dtype=torch.int32, device=gpu)
        drafted, tokens = buf[:, first:first + 4], buf[:, second:second + 5]
        drafted.copy_(d)
        acc, tok = na.verify_drafts(t, drafted, au, su, draft=q, tokens=tokens)
        assert np.array_equal(acc.cpu().numpy(), want[0]) and np.array_equal(tok.cpu().numpy(), want[1])
        assert (buf[:, 9:] == -7).all() and torch.equal(drafted, d)
    for shift in (-4, -1, 0, 1, 3):  # the drafts inside the answer's columns
        buf = torch.zeros((9, 14), dtype=torch.int32, device=gpu)
        with pytest.raises(na.KvError, match="tokens may not share memory with drafted"):
            na.verify_drafts(t, buf[:, 5 + shift:9 + shift], au, su, draft=q, tokens=buf[:, 5:10] if shift != -4 else buf[:, 4:9])
