"""Beam search over a cache, the calls together as a server makes them: a
prompt in one step, forks, then steps of attention, selection and reordering,
on each kind of cache.  Every beam's cache holds, bit for bit, what a cache of
its own would after its own rows alone; what beams share is held once."""
import math

import pytest
import torch

import nanoinfer_amd as na

pytestmark = pytest.mark.gpu
L, H, D, V, PROMPT = 2, 2, 64, 700, 37


def _cache(fmt, seqs):
    return na.PagedKv(na.BatchOpts(n_layer=L, n_head=H, head_dim=D, kv_blocks=200, max_seqs=seqs, n_ctx=160, max_rows=256,
                                   q8=fmt == "q8", block8=fmt == "block8"))


def _held(kv, s):
    return [x.clone() for x in kv.gather_values([(s, p) for p in range(kv.seq_len(s))])]


@pytest.mark.parametrize("fmt", ["f16", "q8", "block8"])
@pytest.mark.parametrize("searches,beams", [(2, 3), (3, 5)])
def test_search(gpu, fmt, searches, beams):
    g = torch.Generator("cuda").manual_seed(beams)
    c, pad = H * D, 0
    table = torch.randn((V, 3, L, c), generator=g, device="cuda")  # a token's q, k and v of every layer
    heads = torch.randn((c, V), generator=g, device="cuda") / 6
    kv = _cache(fmt, searches * beams + 1)
    prompts = torch.randint(1, V, (searches, PROMPT), generator=g, device="cuda")

    def rows(tokens):  # [n] -> q, k, v [L, n, c]
        return (x.contiguous() for x in table[tokens].permute(1, 2, 0, 3))

    first = [kv.add_seq() for _ in range(searches)]
    out = kv.step([(s, PROMPT, 1) for s in first], *rows(prompts.flatten()))
    out = out[-1, PROMPT - 1::PROMPT]  # the prompts' last rows
    live = torch.tensor([[s] + kv.fork([s] * (beams - 1)) for s in first])
    assert kv.blocks_used() == searches * (PROMPT // 16 + beams)
    logits = (out @ heads).view(searches, 1, V).expand(-1, beams, -1)
    scores = torch.full((searches, beams), -math.inf, device="cuda")
    scores[:, 0] = 0
    finished = torch.zeros((searches, beams), dtype=torch.int32, device="cuda")
    history = prompts[:, None].expand(-1, beams, -1).to(torch.int32).contiguous()
    for step in range(24):
        scores, parents, tokens, history = na.beam_select(logits, scores, finished=finished, pad_token=pad, history=history)
        finished = (finished.gather(1, parents.long()) != 0).int() | (tokens == pad).int()
        # The cache of a finished beam goes on with its pad tokens, as the others' do with theirs.
        kv.reorder(live.flatten().tolist(), live.gather(1, parents.cpu().long()).flatten().tolist())
        order = live.flatten().tolist()
        q, k, v = rows(tokens.flatten().long())
        out = kv.step([(s, 1, 1) for s in order], q, k, v)
        if step % 8 == 7:
            kv.compact()
        logits = (out[-1] @ heads).view(searches, beams, V)
        for i in (0, len(order) - 1):  # against 64 bits over what the cache holds
            kk, vv = (x.double().view(L, -1, H, D) for x in _held(kv, order[i]))
            score = (q[:, i].double().view(L, 1, H, D) * kk).sum(-1) / math.sqrt(D)
            want = (torch.softmax(score, 1)[..., None] * vv).sum(1).flatten(1)
            assert float((out[:, i].double() - want).abs().max()) <= 1e-4 * float(vv.abs().max())
    assert history.shape == (searches, beams, PROMPT + 24) and bool((scores[:, :-1] >= scores[:, 1:]).all())
    # Whole prompt pages are held once, by all beams of their search.
    for b in range(searches):
        tables = [kv.block_table(s) for s in live[b].tolist()]
        assert all(t[:PROMPT // 16] == tables[0][:PROMPT // 16] for t in tables)
        assert all(kv.page_refs(p) == beams for p in tables[0][:PROMPT // 16])
    # Each beam's rows, in the same steps, into a cache of its own.
    alone = _cache(fmt, 1)
    for b in range(searches):
        for w in range(beams):
            s = alone.add_seq()
            tokens = history[b, w].long()
            alone.step([(s, PROMPT, 1)], *rows(tokens[:PROMPT]))
            for t in range(PROMPT, len(tokens)):
                alone.step([(s, 1, 1)], *rows(tokens[t:t + 1]))
            assert all(torch.equal(x, y) for x, y in zip(_held(alone, s), _held(kv, int(live[b, w]))))
            alone.free_seq(s)
    for s in live.flatten().tolist():
        kv.free_seq(s)
    assert kv.blocks_used() == 0
