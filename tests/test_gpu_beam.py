"""Beam search's selection on the GPU, against totals sorted in 64 bits."""
import math

import numpy as np
import pytest
import torch

import nanoinfer_amd as na
from nanoinfer_amd import _abi

pytestmark = pytest.mark.gpu
# The normaliser is 2e-6 off at most (beam_kernels.hip); the score is rounded once.
LSE = 2e-6
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def _totals(logits, scores, finished=None, pad=0):
    x = logits.double().cpu()
    x = torch.where(torch.isnan(x), -math.inf, x)
    t = scores.double().cpu()[..., None] + (x - torch.logsumexp(x, -1, keepdim=True))
    t = torch.where((scores.cpu() > -math.inf)[..., None], t, -math.inf)
    if finished is not None:
        for b, w in torch.nonzero(finished.cpu()).tolist():
            t[b, w] = -math.inf
            t[b, w, pad] = scores[b, w].double()
    return torch.nan_to_num(t, nan=-math.inf, posinf=math.inf, neginf=-math.inf)


def _check(got, logits, scores, k, finished=None, pad=0, history=None, exact=False):
    """exact: near ties are exact ones, so that beams and tokens have to be the oracle's."""
    t = _totals(logits, scores, finished, pad)
    b, w, v = t.shape
    flat = t.view(b, w * v)
    best, at = torch.sort(flat, dim=-1, descending=True, stable=True)
    best, at = best[:, :k], at[:, :k]
    if best.shape[1] < k:
        best = torch.nn.functional.pad(best, (0, k - best.shape[1]), value=-math.inf)
        at = torch.nn.functional.pad(at, (0, k - at.shape[1]))
    s, p, n = (x.cpu() for x in got[:3])
    none = best == -math.inf
    assert bool((torch.isneginf(s) == none).all()) and bool(((p == -1) == none).all()) and bool(((n == -1) == none).all())
    close = LSE + best.abs() * 2.0 ** -24
    assert bool((none | ((s.double() - best).abs() <= close)).all())
    mine = p.long() * v + n.long()
    chosen = flat.gather(1, mine.clamp_min(0))
    assert bool((none | ((chosen - best).abs() <= (0 if exact else 2 * LSE))).all())
    assert all(len(set(r[~e].tolist())) == int((~e).sum()) for r, e in zip(mine, none))
    if exact:
        assert torch.equal(torch.where(none, -1, at // v).int(), p) and torch.equal(torch.where(none, -1, at % v).int(), n)
    if history is not None:
        h = history.cpu().gather(1, p.long().clamp_min(0)[..., None].expand(-1, -1, history.shape[2]))
        h = torch.where((p < 0)[..., None], torch.full_like(h, -1), h)
        assert torch.equal(got[3].cpu(), torch.cat([h, n[..., None]], -1))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("b,w,v,k", [(1, 1, 1, 1), (1, 1, 7, 5), (2, 3, 127, 6), (3, 2, 128, 4), (1, 4, 129, 8), (2, 5, 2047, 10),
                                     (1, 8, 2049, 64), (1, 4, 50257, 8), (7, 3, 4096, 3), (2, 64, 1000, 64), (1, 1, 131071, 64),
                                     (5, 6, 32003, 12), (1, 2, 262144, 4)])
def test_selection(gpu, dtype, b, w, v, k):
    g = torch.Generator("cuda").manual_seed(v)
    logits = (torch.randn((b, w, v), generator=g, device="cuda") * 3).to(dtype)
    scores = -torch.rand((b, w), generator=g, device="cuda") * 8
    history = torch.randint(0, v, (b, w, 9), generator=g, device="cuda", dtype=torch.int32)
    _check(na.beam_select(logits, scores, k, history=history), logits, scores, k, history=history)


@pytest.mark.parametrize("dtype", TYPES)
def test_equal_totals_go_to_the_lowest(gpu, dtype):
    g = torch.Generator("cuda").manual_seed(1)
    for v in (130, 5000, 40000):
        few = torch.randint(-2, 3, (2, 4, v), generator=g, device="cuda").to(dtype)
        few[:, 1:] = few[:, :1]  # the same row four times
        scores = torch.tensor([[-1.0, -1.0, -0.5, -1.0], [0.0] * 4], device="cuda")
        for k in (1, 7, 64):
            _check(na.beam_select(few, scores, k), few, scores, k, exact=True)
        flat = torch.zeros((1, 3, v), device="cuda", dtype=dtype)
        s, p, t = na.beam_select(flat, torch.zeros((1, 3), device="cuda"), 20)
        assert p.tolist() == [[0] * 20] and t.tolist() == [list(range(20))]
        up = torch.arange(v, device="cuda").float().div(v).to(dtype).expand(1, 2, v)  # each better than the one before
        _check(na.beam_select(up, torch.zeros((1, 2), device="cuda"), 64), up, torch.zeros((1, 2)), 64, exact=True)


@pytest.mark.parametrize("dtype", TYPES)
def test_candidates_in_one_place(gpu, dtype):
    """All the best within one group of the vocabulary, on its borders, in the last entries."""
    for v, at in ((9000, range(256, 320)), (9000, [0, 127, 128, 255, 256, 8959, 8960, 8999]), (2049, [2047, 2048])):
        logits = torch.full((2, 2, v), -4.0, device="cuda", dtype=dtype)
        for i, x in enumerate(at):
            logits[0, i % 2, x] = 3 + i / 64
            logits[1, 0, x] = 5
        scores = torch.zeros((2, 2), device="cuda")
        _check(na.beam_select(logits, scores, 64), logits, scores, 64, exact=True)


@pytest.mark.parametrize("dtype", TYPES)
def test_masks_and_what_is_no_number(gpu, dtype):
    g = torch.Generator("cuda").manual_seed(2)
    v = 3001
    logits = torch.randn((6, 4, v), generator=g, device="cuda").to(dtype)
    logits[0, :, 5:] = -math.inf             # few candidates
    logits[1] = -math.inf                    # none
    logits[2, 0] = -math.inf
    logits[2, 1, 100] = math.inf             # no candidates in that beam
    logits[2, 2, ::3] = math.nan
    logits[3, 1] = math.nan
    logits[3, 2, 1:] = torch.finfo(dtype).min  # one that takes it all
    logits[4] *= 200                         # exp of differences far below the smallest float
    logits[5, :, 17:] = torch.finfo(dtype).min
    scores = -torch.rand((6, 4), generator=g, device="cuda")
    scores[3, 3] = -math.inf
    scores[5, 0], scores[5, 1] = math.nan, -math.inf
    for k in (1, 8, 30):
        _check(na.beam_select(logits, scores, k), logits, scores, k)
    first = torch.full((6, 4), -math.inf, device="cuda")
    first[:, 0] = 0
    _check(na.beam_select(logits, first, 8), logits, first, 8)


@pytest.mark.parametrize("dtype", TYPES)
def test_finished_beams(gpu, dtype):
    g = torch.Generator("cuda").manual_seed(3)
    b, w, v = 5, 6, 1500
    logits = torch.randn((b, w, v), generator=g, device="cuda").to(dtype)
    scores = -torch.rand((b, w), generator=g, device="cuda") * 9
    finished = torch.zeros((b, w), dtype=torch.int32, device="cuda")
    finished[0, 2], finished[1] = 1, 5
    finished[2, :5], finished[3, ::2] = 1, -1
    logits[finished != 0] = math.nan  # not looked at
    scores[3, 0] = -math.inf
    for pad in (0, 700, v - 1):
        _check(na.beam_select(logits, scores, 12, finished=finished, pad_token=pad), logits, scores, 12, finished, pad)
    with pytest.raises(na.KvError) as e:
        na.beam_select(logits, scores, 12, finished=finished, pad_token=v)
    assert e.value.code == _abi.NI_ERR_BAD_ARG


def test_strides_and_given_outputs(gpu):
    g = torch.Generator("cuda").manual_seed(4)
    whole = torch.randn((4, 5, 1, 1003), generator=g, device="cuda")
    scores = -torch.rand((3, 4), generator=g, device="cuda")
    view = whole[1:, :4, 0, 2:1000]
    out = dict(out_scores=torch.full((3, 6), 7.0, device="cuda"), parents=torch.full((3, 6), 7, dtype=torch.int32, device="cuda"),
               tokens=torch.full((3, 6), 7, dtype=torch.int32, device="cuda"))
    got = na.beam_select(view, scores, 6, **out)
    assert got[0] is out["out_scores"] and got[1] is out["parents"] and got[2] is out["tokens"]
    _check(got, view, scores, 6)
    same = whole[:1, :1, 0].expand(3, 4, -1)  # one row for all beams, half apart
    got = na.beam_select(same, scores, 6)
    _check(got, same, scores, 6)
    half = torch.randn((2, 3, 2, 777), generator=g, device="cuda").half()[:, :, 1]
    _check(na.beam_select(half, scores[:2, :3].contiguous(), 4), half, scores[:2, :3], 4)
    assert [x.shape for x in na.beam_select(view, scores)] == [(3, 4)] * 3
    assert na.beam_select(view[:0], scores[:0], 3)[0].shape == (0, 3)
    assert na.beam_select(view, scores, 0)[0].shape == (3, 0)
    empty = torch.zeros((3, 4, 0), dtype=torch.int32, device="cuda")
    got = na.beam_select(view, scores, 5, history=empty)
    assert torch.equal(got[3][..., 0], got[2])


def test_captured_and_on_other_streams(gpu):
    g = torch.Generator("cuda").manual_seed(5)
    logits = torch.randn((3, 4, 60000), generator=g, device="cuda")
    scores = -torch.rand((3, 4), generator=g, device="cuda")
    history = torch.randint(0, 9, (3, 4, 50), generator=g, device="cuda", dtype=torch.int32)
    na.beam_select(logits, scores, 8, history=history)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = na.beam_select(logits, scores, 8, history=history)
    for turn in range(4):
        logits.copy_(torch.randn(logits.shape, generator=g, device="cuda"))
        history += 1
        graph.replay()
        torch.cuda.synchronize()
        want = na.beam_select(logits, scores, 8, history=history)
        assert all(torch.equal(a, b) for a, b in zip(got, want)), turn
        _check(got, logits, scores, 8, history=history)
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    many = [na.beam_select(logits, scores, 8, history=history, stream=s) for _ in range(10) for s in (a, b)]
    torch.cuda.synchronize()
    for m in many:
        assert all(torch.equal(x, y) for x, y in zip(m, want))


def test_refusals(gpu):
    logits, scores = torch.zeros((2, 3, 40), device="cuda"), torch.zeros((2, 3), device="cuda")
    for args, kw, kind in (((logits.double(), scores), {}, TypeError), ((logits[0], scores), {}, TypeError),
                           ((logits, scores.double()), {}, TypeError), ((logits, scores[:, :2]), {}, ValueError),
                           ((logits.transpose(1, 2), scores), {}, ValueError), ((logits[..., :0], scores), {}, ValueError),
                           ((logits, scores, -1), {}, ValueError), ((logits, scores, 65), {}, na.KvError),
                           ((logits, scores), dict(finished=scores), TypeError),
                           ((logits, scores), dict(out_history=scores), ValueError),
                           ((logits.cpu(), scores.cpu()), {}, TypeError), ((logits, scores.cpu()), {}, ValueError),
                           ((logits, scores, 3), dict(out_scores=scores), na.KvError),
                           ((logits, scores, 3), dict(out_scores=logits.view(-1)[:6].view(2, 3)), na.KvError),
                           ((logits.expand(2, 3, 40)[:, :1].expand(2, 70, 40), torch.zeros((2, 70), device="cuda")), {}, na.KvError)):
        with pytest.raises(kind):
            na.beam_select(*args, **kw)
    i = torch.zeros((2, 3), dtype=torch.int32, device="cuda")
    with pytest.raises(na.KvError):
        na.beam_select(logits, scores, 3, parents=i, tokens=i)
    h = torch.zeros((2, 3, 5), dtype=torch.int32, device="cuda")
    with pytest.raises(na.KvError):
        na.beam_select(logits, scores, 3, history=h[:, :, :4].contiguous(), tokens=h.view(-1)[:6].view(2, 3),
                       out_history=h)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("w,v,k", [(8, 131071, 16), (64, 40000, 64), (3, 2000, 33)])
def test_more_equal_totals_than_are_ranked_at_once(gpu, dtype, w, v, k):
    g = torch.Generator("cuda").manual_seed(6)
    logits = torch.randint(0, 2, (2, w, v), generator=g, device="cuda").to(dtype)
    logits[1] = logits[1, :1]
    logits[1, -1, v // 2:] = 2
    scores = torch.zeros((2, w), device="cuda")
    logits[0] = logits[0, 0].sort().values  # the best at the end of every row
    _check(na.beam_select(logits, scores, k), logits, scores, k, exact=True)
