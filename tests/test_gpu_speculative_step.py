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
