"""The operators as a serving step uses them together: drafted rows rotated and
appended behind a shared prefix, attended, the drafts verified, the rejected
ones rolled back, and the next round over what is left -- against the same
rounds in 64 bits."""
import math

import numpy as np
import pytest
import torch

import nanoinfer_amd as na
from nanoinfer_amd import drivers
from test_gpu_rotary import turn64
from test_gpu_verify import expect

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n_head,group,d", [(3, 1, 64), (2, 4, 128)])
def test_rounds(gpu, n_head, group, d):
    L, K, V, P = 2, 3, 777, 83
    own = [1, 16, 30]
    S = len(own)
    kv = na.PagedKv(na.BatchOpts(n_layer=L, n_head=n_head, head_dim=d, kv_blocks=32, max_seqs=S + 1, n_ctx=128,
                                 max_rows=128))
    rot = na.Rotary(d, base=500000.0, rot_dim=d // 2)
    g = torch.Generator(device="cuda").manual_seed(d)
    rand = lambda *shape: torch.randn(shape, generator=g, device="cuda")
    c = n_head * d
    keys, vals = {}, {}  # what the cache holds, in 64 bits [L, n, heads, d]

    def append(rows, pos, q=None):
        k, v = rand(L, len(rows), c), rand(L, len(rows), c)
        q = kv.append_rotary(rows, k, v, rot, q=q, positions=pos)
        k64, _ = turn64(rot, k.view(L, -1, n_head, d), pos)
        for i, (s, p) in enumerate(rows):
            old = keys.get(s, torch.zeros((L, 0, n_head, d), dtype=torch.float64))[:, :p]
            keys[s] = torch.cat([old, k64[:, i:i + 1].half().double()], 1)
            old = vals.get(s, torch.zeros((L, 0, n_head, d), dtype=torch.float64))[:, :p]
            vals[s] = torch.cat([old, v.view(L, -1, n_head, d)[:, i:i + 1].half().double().cpu()], 1)
        return q

    prefix = kv.add_seq()
    kv.reserve(prefix, P)
    append([(prefix, p) for p in range(P)], np.arange(P))
    kv.commit(prefix, P)
    seqs = []
    for n in own:
        s = kv.add_seq()
        kv.reserve(s, n)
        append([(s, p) for p in range(n)], P + np.arange(n))
        kv.commit(s, n)
        seqs.append(s)
    head = rand(n_head * group * d, V) * 0.4
    spec = drivers.Spec(kv, seqs, K, 1)
    for _ in range(4):
        work, _ = spec.plan()
        rows = []
        for s, n, _ in np.asarray(work).tolist():
            p0 = kv.seq_len(s)
            kv.reserve(s, p0 + n)
            rows += [(s, p0 + i) for i in range(n)]
        pos = np.array([P + p for _, p in rows])
        q_in = rand(L, len(rows), c * group)
        q = append(rows, pos, q_in)
        out = kv.prefix_attention(q, rows, [(prefix, P, len(rows))])
        for s, n, _ in np.asarray(work).tolist():
            kv.commit(s, n)
        # against 64 bits, from the unrotated queries
        q64, _ = turn64(rot, q_in.view(L, len(rows), -1, d), pos)
        q64 = q64.view(L, len(rows), n_head, group, d)
        for i, (s, p) in enumerate(rows):
            k = torch.cat([keys[prefix], keys[s][:, :p + 1]], 1)
            v = torch.cat([vals[prefix], vals[s][:, :p + 1]], 1)
            w = torch.softmax(torch.einsum("lhgd,lkhd->lhgk", q64[:, i], k) / math.sqrt(d), -1)
            want = torch.einsum("lhgk,lkhd->lhgd", w, v).reshape(L, -1)
            # keys are f16: a rotated value at a border rounds to its neighbour, 2^-10 of it,
            # in a few of the thousands of values a score sums
            err = (out[:, i].double().cpu() - want).abs().max()
            assert err <= 2.0 ** -12 * want.abs().max()
        # a target and a drafter over the attention's output
        logits = (out[-1] @ head).view(S, K + 1, V)
        target = torch.softmax(logits * 4, -1)
        draft = torch.softmax(logits[:, :K] * 3, -1)
        drafted = torch.multinomial(draft.reshape(-1, V), 1, generator=g).view(S, K).to(torch.int32)
        au, su = torch.rand((S, K), generator=g, device="cuda"), torch.rand((S,), generator=g, device="cuda")
        accepted, tokens = na.verify_drafts(target, drafted, au, su, draft=draft)
        want = expect(target, drafted, au, su, draft=draft)
        assert np.array_equal(accepted.cpu().numpy(), want[0]) and np.array_equal(tokens.cpu().numpy(), want[1])
        lens = [kv.seq_len(s) - K - 1 for s in seqs]
        assert spec.commit(accepted) == want[0].tolist()
        assert [kv.seq_len(s) for s in seqs] == [n + 1 + a for n, a in zip(lens, want[0].tolist())]


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("d,n_head,P", [(64, 12, 1700), (128, 8, 3000)])
def test_a_captured_round(gpu, d, n_head, P, q8):
    """Append, attention over wide tiles and verification in one graph: every
    replay, over other inputs and between eager calls, gives the eager call's bits."""
    S, K, V, L = 10, 1, 1234, 1 if d == 128 else 2
    kv = na.PagedKv(na.BatchOpts(n_layer=L, n_head=n_head, head_dim=d, kv_blocks=P // 16 + 1 + 4 * S, max_seqs=S + 1,
                                 n_ctx=P, max_rows=P, q8=q8))
    rot = na.Rotary(d, interleaved=True)
    g = torch.Generator(device="cuda").manual_seed(d)
    rand = lambda *shape: torch.randn(shape, generator=g, device="cuda")
    c = n_head * d
    lens = [P] + [3 + 5 * i for i in range(S)]
    seqs = []
    for n in lens:
        s = kv.add_seq()
        kv.reserve(s, n)
        kv.append([(s, p) for p in range(n)], rand(L, n, c), rand(L, n, c))
        kv.commit(s, n)
        seqs.append(s)
    rows = []
    for s, n in zip(seqs[1:], lens[1:]):
        kv.reserve(s, n + K + 1)
        rows += [(s, n + i) for i in range(K + 1)]
    n = len(rows)
    pos = np.array([P + p for _, p in rows], dtype=np.uint32)
    head = rand(c, V) * 0.2
    k, v, q = rand(L, n, c), rand(L, n, c), rand(L, n, c)
    au, su = torch.rand((S, K), generator=g, device="cuda"), torch.rand((S,), generator=g, device="cuda")
    drafted = torch.randint(0, V, (S, K), generator=g, device="cuda", dtype=torch.int32)

    def round_(to):
        qr, out, acc, tok = to
        kv.append_rotary(rows, k, v, rot, q=q, q_out=qr, positions=pos)
        kv.prefix_attention(qr, rows, [(seqs[0], P, n)], out=out)
        target = torch.softmax((out[-1] @ head).view(S, K + 1, V), -1)
        na.verify_drafts(target, drafted, au, su, accepted=acc, tokens=tok)

    def outputs():
        return (torch.empty((L, n, c), device="cuda"), torch.empty((L, n, c), device="cuda"),
                torch.empty((S,), dtype=torch.int32, device="cuda"),
                torch.empty((S, K + 1), dtype=torch.int32, device="cuda"))

    eager, replayed = outputs(), outputs()
    round_(eager)  # (the handle's partials, the library's workspaces)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        round_(replayed)
    for i in range(4):
        for x in (k, v, q):
            x.copy_(rand(*x.shape))
        au.copy_(torch.rand((S, K), generator=g, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        got = [x.clone() for x in replayed]
        round_(eager)
        for a, b in zip(eager, got):
            assert torch.equal(a, b), i
