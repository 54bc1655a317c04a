"""Beam search on a paged cache as measurable cases: copies of pages (forked,
reordered and compacted sequences), the selection over beams and vocabulary,
and the cache held in 8 bits with a scale for each block of tokens and head.

* ``fork``: sequences continued several times, whole pages shared, the page
  with the end copied;
* ``reorder``: beams that continue other beams, in place;
* ``compact``: the pages of a new batch moved to where the last one's lay;
* ``beam``: the best continuations of every search, with their histories;
* ``append``: keys and values into the 8-bit cache, read back as what they stand for;
* ``attend``: rows appended to the 8-bit cache, and their attention.

Where ``own`` is false a pass is elementary torch operations; where it is true
it is the package's calls on the same inputs.  Lengths and page orders follow
from a case's ``ctx_seed`` (so its work is fixed), every value from
``prepare``'s seed.
"""
import math
import random

import numpy as np
import torch

own = False

GPT2 = dict(n_q_head=12, n_head=12, head_dim=64)  # the benchmark's model shape
GROUPED = dict(n_q_head=32, n_head=8, head_dim=128)  # the long-context shape, four query heads a cache head
LONG = dict(n_q_head=32, n_head=32, head_dim=128)  # the long-context shape
PAGE = 16
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def _pages(op, shape, n_layer, seqs, ctx_lo, ctx_hi, fmt="f16", beams=1, grown=0, ctx_seed=1):
    """seqs sequences (of `beams` beams each, `grown` positions past what they
    share) of ctx_lo..ctx_hi positions in a cache of f16 or int8 values."""
    return dict(kind="pages", op=op, **shape, n_layer=n_layer, seqs=seqs, ctx_lo=ctx_lo, ctx_hi=ctx_hi, fmt=fmt,
                beams=beams, grown=grown, ctx_seed=ctx_seed)


def _beam(searches, beams, vocab, k, dtype="f32", history=0, finished=0.0, banned=0.0, first=False):
    """finished, banned: shares of the beams and of the logits; first: only beam 0 has begun."""
    return dict(kind="beam", searches=searches, beams=beams, vocab=vocab, k=k, dtype=dtype, history=history,
                finished=finished, banned=banned, first=first)


def _block(op, shape, n_layer, seqs, ctx_lo, ctx_hi, new, ctx_seed=1):
    """seqs sequences of ctx_lo..ctx_hi positions, to which `new` are appended (and attended)."""
    return dict(kind="block", op=op, **shape, n_layer=n_layer, seqs=seqs, ctx_lo=ctx_lo, ctx_hi=ctx_hi, new=new,
                ctx_seed=ctx_seed)


def listed():
    return [
        # A prompt of one request, continued four times: the smallest call.
        dict(_pages("fork", GPT2, 12, 1, 1003, 1003, beams=4, ctx_seed=2), name="fork-4"),
        # A serving batch of beam searches after a step, every layer's pages.
        dict(_pages("reorder", GPT2, 12, 16, 200, 900, beams=4, grown=37, ctx_seed=3), name="reorder-16x4"),
        # A batch of long requests moved to the front of the pool when the one before it ends.
        dict(_pages("compact", LONG, 4, 6, 500, 2040, ctx_seed=4), name="compact-6"),
        # One user's search, its first step.
        dict(_beam(1, 4, 50257, 8, first=True), name="beam-1x4"),
        # Searches over a large vocabulary with f16-sized logits, some beams finished, tokens banned.
        dict(_beam(16, 6, 131071, 12, "bf16", history=100, finished=0.2, banned=0.05), name="beam-16x6-bf16"),
        # A serving batch of searches over the same vocabulary.
        dict(_beam(64, 8, 131071, 16, history=57), name="beam-64x8"),
        # One layer of a decode batch: every sequence appends a token.
        dict(_block("append", GPT2, 1, 64, 1, 40, 1, ctx_seed=5), name="append-64"),
        # One layer of a long prompt with grouped heads, behind an earlier part that ends inside a page.
        dict(_block("append", GROUPED, 1, 1, 13, 13, 2047, ctx_seed=6), name="append-prompt-2047"),
        # A decode batch, every layer in one call.
        dict(_block("attend", GPT2, 12, 64, 1, 767, 1, ctx_seed=7), name="attend-64-layers"),
        # Drafts attended for verification, one layer.
        dict(_block("attend", GPT2, 1, 32, 5, 1000, 5, ctx_seed=8), name="attend-32x5"),
        # A few users with a book each, grouped heads: the cache is the whole cost.
        dict(_block("attend", GROUPED, 1, 16, 30011, 32750, 1, ctx_seed=9), name="attend-16x32k"),
        # One layer of a prompt, every row queried.
        dict(_block("attend", GROUPED, 1, 1, 7, 7, 2041, ctx_seed=10), name="attend-prompt-2041"),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


def draw(rng: random.Random):
    kind = rng.choice(["fork", "reorder", "compact", "beam", "beam", "append", "append-prompt", "attend", "attend",
                       "attend-long", "attend-prompt"])
    cs = rng.randrange(1 << 30)
    if kind == "beam":
        beams = rng.randint(1, 8)
        return _beam(_log(rng, 1, 64), beams, _log(rng, 500, 131071), rng.randint(1, 2 * beams),
                     rng.choice(["f32", "f16", "bf16"]), history=rng.choice([0, rng.randint(1, 500)]),
                     finished=rng.choice([0.0, 0.3]), banned=rng.choice([0.0, 0.1]), first=rng.random() < 0.2)
    shape = rng.choice([GPT2, GROUPED])
    n_layer = rng.choice([1, 1, 12]) if shape is GPT2 else rng.choice([1, 4])
    if kind in ("fork", "reorder"):
        lo = rng.randint(1, 900)
        return _pages(kind, shape, n_layer, _log(rng, 1, 16), lo, rng.randint(lo, 1000), rng.choice(["f16", "int8"]),
                      beams=rng.randint(2, 6), grown=rng.randint(1, 50) if kind == "reorder" else 0, ctx_seed=cs)
    if kind == "compact":
        lo = rng.randint(1, 500)
        return _pages(kind, shape, n_layer, _log(rng, 1, 16), lo, rng.randint(lo, 700), rng.choice(["f16", "int8"]),
                      ctx_seed=cs)
    if kind == "append":
        lo = rng.randint(1, 40)
        return _block("append", shape, n_layer, _log(rng, 1, 64), lo, rng.randint(lo, 100), rng.choice([1, 1, 2, 5, 9]),
                      ctx_seed=cs)
    if kind == "append-prompt":
        ctx = rng.randint(1, 200)
        return _block("append", shape, 1, rng.randint(1, 2), ctx, ctx, _log(rng, 17, 1000), ctx_seed=cs)
    if kind == "attend":
        lo = rng.randint(1, 500)
        return _block("attend", shape, n_layer, _log(rng, 1, 64), lo, rng.randint(lo, 700), rng.choice([1, 1, 1, 3, 5, 8]),
                      ctx_seed=cs)
    if kind == "attend-long":
        n = _log(rng, 2000, 32000)
        return _block("attend", shape, 1, rng.randint(1, max(1, 300000 // n)), n - rng.randint(0, 500), n, rng.choice([1, 1, 4]),
                      ctx_seed=cs)
    ctx = rng.randint(1, 200)
    return _block("attend", shape, 1, rng.randint(1, 2), ctx, ctx, _log(rng, 17, 1000), ctx_seed=cs)


# ------------------------------------------------------------------- shapes


def _contexts(case):
    rng = random.Random(case["ctx_seed"])
    return [rng.randint(case["ctx_lo"], case["ctx_hi"]) for _ in range(case["seqs"])]


def _order(case, n_pages):
    order = list(range(n_pages))
    random.Random(case["ctx_seed"] + 1).shuffle(order)
    return order


def _parents(case):
    """reorder: the beam of its search that each beam continues; those continued by others continue themselves."""
    rng = random.Random(case["ctx_seed"] + 2)
    out = []
    for _ in range(case["seqs"]):
        keep = sorted(rng.sample(range(case["beams"]), max(1, case["beams"] // 2)))
        out.append([w if w in keep else rng.choice(keep) for w in range(case["beams"])])
    return out


def _block_bytes(case):
    """Bytes of a page's K (or V) of one head: f16 values, or int8 values and 16 f32 scales."""
    return PAGE * (2 * case["head_dim"] if case["fmt"] == "f16" else case["head_dim"] + 4)


def _row_bytes(case, rows):
    """Which bytes of such a block belong to its first `rows` rows."""
    d = case["head_dim"]
    if case["fmt"] == "f16":
        return np.arange(2 * d * rows)
    return np.concatenate([np.arange(d * rows), PAGE * d + np.arange(4 * rows)])


def _beams_tables(case):
    """fork, reorder: (pages in the pool, their order, the table and length of
    every sequence that lives before the measured call).  Pages are handed out
    in order; a fork shares whole pages and takes one page for the rest."""
    tables, lengths, at = [], [], 0
    need = sum(-(-n // PAGE) + case["beams"] * (1 + -(-case["grown"] // PAGE)) for n in _contexts(case)) + 3
    order = _order(case, need)

    def take(n):
        nonlocal at
        at += n
        return order[at - n:at]

    for n in _contexts(case):
        tables.append(take(-(-n // PAGE)))
        lengths.append(n)
    if case["op"] == "reorder":
        prompts, tables_, lengths_ = list(zip(tables, lengths)), [], []
        forks = [[(t if w == 0 else t[:n // PAGE] + take(1 if n % PAGE else 0)) for w in range(case["beams"])]
                 for t, n in prompts]
        for (_, n), beams in zip(prompts, forks):
            for t in beams:
                end = n + case["grown"]
                tables_.append(t + take(-(-end // PAGE) - len(t)))
                lengths_.append(end)
        tables, lengths = tables_, lengths_
    return need, order, tables, lengths, order[at:]


# ------------------------------------------------------------------- inputs


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(g, shape, std=1.0):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32) * std


def _pool_inputs(case, g, n_pages):
    """The bytes of a pool [n_layer, pages, heads, K|V, block]."""
    shape = (case["n_layer"], n_pages, case["n_head"], 2, _block_bytes(case))
    return torch.randint(0, 256, shape, generator=g, device="cuda", dtype=torch.uint8)


def _beam_inputs(case, seed):
    g = _gen(seed)
    b, w, v = case["searches"], case["beams"], case["vocab"]
    logits = _normal(g, (b, w, v), 2.5).to(DTYPES[case["dtype"]])
    if case["banned"]:
        logits.masked_fill_(torch.rand((b, w, v), generator=g, device="cuda") < case["banned"], -math.inf)
    scores = -torch.rand((b, w), generator=g, device="cuda") * 6 - 3
    if case["first"]:
        scores[:, 0] = 0
        scores[:, 1:] = -math.inf
    finished = None
    if case["finished"]:
        finished = (torch.rand((b, w), generator=g, device="cuda") < case["finished"]).to(torch.int32)
    history = None
    if case["history"]:
        history = torch.randint(0, v, (b, w, case["history"]), generator=g, device="cuda", dtype=torch.int32)
    return logits, scores, finished, history


def _block_inputs(case, seed):
    """Keys and values [n_layer, positions, heads * head_dim] f32 already in the cache, sequence after sequence, then
    those to append, and the queries of the appended rows."""
    g = _gen(seed)
    c, d = case["n_head"] * case["head_dim"], case["head_dim"]
    held, n = sum(_contexts(case)), case["seqs"] * case["new"]
    loud = 1 + 5 * (torch.rand((c,), generator=g, device="cuda") < 0.03)  # a few channels larger than the others
    old = [_normal(g, (case["n_layer"], held, c)) * loud for _ in range(2)]
    new = [_normal(g, (case["n_layer"], n, c), 1.3) * loud for _ in range(2)]
    return old, new, _normal(g, (case["n_layer"], n, case["n_q_head"] * d))


# ------------------------------------------------------------------ prepare


class _Pool:
    """A device pool's memory, for torch to view."""

    def __init__(self, kv):
        self.kv = kv  # keeps the pool alive
        at, _, n = kv.pools()
        self.__cuda_array_interface__ = dict(shape=(n,), typestr="|u1", data=(at, False), version=2)


def _cache(case, n_pages, order, max_seqs, n_ctx, **kw):
    import nanoinfer_amd as na

    return na.PagedKv(na.BatchOpts(n_layer=case["n_layer"], n_head=case["n_head"], head_dim=case["head_dim"],
                                   kv_blocks=n_pages, max_seqs=max_seqs, n_ctx=n_ctx, max_rows=8192, page_order=order, **kw))


def _prepare_pages(case, seed):
    g, ctx = _gen(seed), _contexts(case)
    if case["op"] == "compact":
        half = sum(-(-n // PAGE) for n in ctx)
        n_pages = 2 * half + 3
        order = _order(case, n_pages)
    else:
        n_pages, order, tables, lengths, free = _beams_tables(case)
    contents = _pool_inputs(case, g, n_pages)
    if own:
        kv = _cache(case, n_pages, order, 2 * case["seqs"] * case["beams"] + case["seqs"], max(ctx) + case["grown"],
                    q8=case["fmt"] == "int8")
        pool = torch.as_tensor(_Pool(kv), device="cuda").view(contents.shape)
        state = dict(case=case, kv=kv, pool=pool, ctx=ctx, live=[])
        for n in ctx:
            state["live"].append(kv.add_seq())
            kv.reserve(state["live"][-1], n)
            kv.commit(state["live"][-1], n)
        if case["op"] == "reorder":
            groups = [[s] + kv.fork([s] * (case["beams"] - 1)) for s in state["live"]]
            for beams in groups:
                for s in beams:
                    kv.reserve(s, kv.seq_len(s) + case["grown"])
                    kv.commit(s, case["grown"])
            state["beams"] = [s for beams in groups for s in beams]
            state["parents"] = [beams[w] for beams, p in zip(groups, _parents(case)) for w in p]
        pool.copy_(contents)  # (behind the copies that forks have made)
        return state
    state = dict(case=case, pool=contents)
    if case["op"] == "compact":
        state["dst"], state["src"] = (torch.tensor(x, device="cuda") for x in (order[:half], order[half:2 * half]))
        return state
    pairs = []  # (from, to, rows)
    if case["op"] == "fork":
        for t, n in zip(tables, lengths):
            for _ in range(case["beams"]):
                if n % PAGE:
                    pairs.append((t[-1], free[len(pairs)], n % PAGE))
    else:
        for i, p in enumerate(p + s * case["beams"] for s, ps in enumerate(_parents(case)) for p in ps):
            if p != i and lengths[p] % PAGE:
                pairs.append((tables[p][-1], tables[i][-1], lengths[p] % PAGE))
    rows = sorted({r for _, _, r in pairs})
    state["copies"] = [(torch.tensor([f for f, _, r in pairs if r == n], device="cuda")[:, None],
                        torch.tensor([t for _, t, r in pairs if r == n], device="cuda")[:, None],
                        torch.tensor(_row_bytes(case, n), device="cuda")) for n in rows]
    return state


def _prepare_block(case, seed):
    old, new, q = _block_inputs(case, seed)
    ctx, n_new, c = _contexts(case), case["new"], case["n_head"] * case["head_dim"]
    need = [-(-(n + n_new) // PAGE) for n in ctx]
    n_pages = sum(need) + 3
    order = _order(case, n_pages)
    rows = np.array([(s, n + t) for s, n in enumerate(ctx) for t in range(n_new)], dtype=np.uint32)
    # every position of the pages that the new rows go to
    touched = np.array([(s, p) for s, n in enumerate(ctx) for p in range(n // PAGE * PAGE, n + n_new)], dtype=np.uint32)
    one = case["n_layer"] == 1
    new, q = [x[0] if one else x for x in new], q[0] if one else q
    state = dict(case=case, rows=rows, touched=touched, k=new[0], v=new[1], q=q, out=torch.empty_like(q))
    if own:
        kv = _cache(case, n_pages, order, case["seqs"], max(ctx) + n_new, block8=True)
        held = np.array([(s, p) for s, n in enumerate(ctx) for p in range(n)], dtype=np.uint32)
        for n in ctx:
            s = kv.add_seq()
            kv.reserve(s, n + n_new)
        at = 0
        while at < len(held):  # whole pages of one sequence at a time, as prompts come
            s, p = held[at]
            m = min(8192, ctx[s] - int(p))
            kv.append(held[at:at + m], old[0][:, at:at + m], old[1][:, at:at + m])
            at += m
        for s, n in enumerate(ctx):
            kv.commit(s, n)
        state["kv"] = kv
        return state
    # Blocks of a sequence one after another, [n_layer, blocks, heads, 16, head_dim] each of K and V.
    first = np.concatenate([[0], np.cumsum(need)])
    state["first"], state["ctx"] = first, ctx
    at = np.concatenate([first[s] * PAGE + np.arange(n) for s, n in enumerate(ctx)])
    at = torch.tensor(at, device="cuda")
    state["held"] = []
    for x in old:
        dense = torch.zeros((case["n_layer"], int(first[-1]) * PAGE, c), device="cuda")
        dense[:, at] = x
        state["held"].append(list(_quantise(_blocks(case, dense))))
    return state


def prepare(case, seed):
    if case["kind"] == "pages":
        return _prepare_pages(case, seed)
    if case["kind"] == "block":
        return _prepare_block(case, seed)
    logits, scores, finished, history = _beam_inputs(case, seed)
    state = dict(case=case, logits=logits, scores=scores, finished=finished, history=history)
    shape = (case["searches"], case["k"])
    state["out"] = dict(out_scores=torch.empty(shape, device="cuda"),
                        parents=torch.empty(shape, dtype=torch.int32, device="cuda"),
                        tokens=torch.empty(shape, dtype=torch.int32, device="cuda"))
    if history is not None:
        state["out"]["out_history"] = torch.empty((*shape, case["history"] + 1), dtype=torch.int32, device="cuda")
    return state


# ---------------------------------------------------------------------- run


def run(s):
    return (_run_own if own else _run_plain)(s)


def _run_own(s):
    import nanoinfer_amd as na

    case = s["case"]
    if case["kind"] == "pages":
        kv = s["kv"]
        if case["op"] == "fork":
            seqs = kv.fork([x for x in s["live"] for _ in range(case["beams"])])
            for x in reversed(seqs):  # (the next pass finds the cache as this one did)
                kv.free_seq(x)
        elif case["op"] == "reorder":
            kv.reorder(s["beams"], s["parents"])
        else:
            fresh = []
            for n in s["ctx"]:
                fresh.append(kv.add_seq())
                kv.reserve(fresh[-1], n)
                kv.commit(fresh[-1], n)
            for x in s["live"]:
                kv.free_seq(x)
            kv.compact()
            s["live"] = fresh
        return {"pool": s["pool"]}
    if case["kind"] == "beam":
        na.beam_select(s["logits"], s["scores"], case["k"], finished=s["finished"], pad_token=case["vocab"] - 1,
                       history=s["history"], **s["out"])
        return s["out"]
    kv, layer = s["kv"], 0 if case["n_layer"] == 1 else na.ALL_LAYERS
    kv.append(s["rows"], s["k"], s["v"], layer=layer)
    if case["op"] == "append":
        k, v = kv.gather_values(s["touched"], layer=layer)
        return {"k": k, "v": v}
    if case["n_q_head"] == case["n_head"]:
        return kv.attention(s["q"], s["rows"], out=s["out"], layer=layer)
    return kv.prefix_attention(s["q"], s["rows"], [(0, 0, len(s["rows"]))], out=s["out"], layer=layer)


def _run_plain(s):
    kind = s["case"]["kind"]
    if kind == "pages":
        return _plain_pages(s)
    if kind == "beam":
        return _plain_beam(s)
    return _plain_block(s)


def _plain_pages(s):
    pool = s["pool"]
    if s["case"]["op"] == "compact":
        pool[:, s["dst"]] = pool[:, s["src"]]
    else:
        for src, dst, at in s["copies"]:
            moved = pool.permute(1, 4, 0, 2, 3)
            moved[dst, at] = moved[src, at]
    return {"pool": pool}


def _plain_beam(s):
    case, logits = s["case"], s["logits"]
    b, w, v, k = case["searches"], case["beams"], case["vocab"], case["k"]
    x = logits.double()
    top = x.amax(-1, keepdim=True)
    total = s["scores"].double()[..., None] + (x - (top + torch.log(torch.exp(x - top).sum(-1, keepdim=True))))
    if s["finished"] is not None:
        done = s["finished"] != 0
        total.masked_fill_(done[..., None], -math.inf)
        total[..., v - 1] = torch.where(done, s["scores"].double(), total[..., v - 1])
    total = total.masked_fill(torch.isnan(total), -math.inf).view(b, w * v)
    best, at = [], []
    for _ in range(k):
        i = total.argmax(-1, keepdim=True)
        best.append(total.gather(1, i))
        at.append(i)
        total.scatter_(1, i, -math.inf)
    best, at = torch.cat(best, 1), torch.cat(at, 1)
    none = best == -math.inf
    parents = torch.where(none, -1, at // v)
    tokens = torch.where(none, -1, at % v)
    out = dict(out_scores=best.float(), parents=parents.to(torch.int32), tokens=tokens.to(torch.int32))
    if s["history"] is not None:
        h = s["history"].gather(1, parents.clamp_min(0)[..., None].expand(-1, -1, case["history"]))
        h = torch.where(none[..., None], torch.full_like(h, -1), h)
        out["out_history"] = torch.cat([h, out["tokens"][..., None]], -1)
    return out


def _blocks(case, dense):
    """[n_layer, positions, heads * head_dim] as [n_layer, blocks, heads, 16, head_dim]."""
    n_layer, n, _ = dense.shape
    return dense.view(n_layer, n // PAGE, PAGE, case["n_head"], case["head_dim"]).transpose(2, 3).contiguous()


def _scale(top):
    """The power of two that a block with this largest value needs: top / scale <= 448, the largest e4m3 value."""
    m, e = torch.frexp(top)  # top = m 2^e, m in [0.5, 1); 448 = 0.875 * 2^9
    e = torch.where(top > 0, e - torch.where(m <= 0.875, 9, 8), -117).clamp(-117, 120)
    return ((e + 127) << 23).to(torch.int32).view(torch.float32)


def _quantise(x):
    """Blocks as (bytes of e4m3 values, scale of each block)."""
    scale = _scale(x.abs().amax((-1, -2)))
    return (x / scale[..., None, None]).to(torch.float8_e4m3fn).view(torch.uint8), scale


def _values(held, blocks):
    values, scale = held
    return values[:, blocks].view(torch.float8_e4m3fn).float() * scale[:, blocks][..., None, None]


def _plain_append(s, which):
    """The new rows into the blocks they go to; gives those blocks' values."""
    case, first, n_new = s["case"], s["first"], s["case"]["new"]
    values, scale = s["held"][which]
    if "blocks" not in s:
        blocks = np.concatenate([first[i] + np.arange(n // PAGE, -(-(n + n_new) // PAGE)) for i, n in enumerate(s["ctx"])])
        start = np.cumsum([0] + [-(-(n + n_new) // PAGE) - n // PAGE for n in s["ctx"]])
        at = np.concatenate([start[i] * PAGE + n % PAGE + np.arange(n_new) for i, n in enumerate(s["ctx"])])
        s["blocks"], s["at"] = torch.tensor(blocks, device="cuda"), torch.tensor(at, device="cuda")
    blocks, at = s["blocks"], s["at"]
    x = s["k"] if which == 0 else s["v"]
    x = x if case["n_layer"] > 1 else x[None]
    dense = torch.zeros((case["n_layer"], len(blocks) * PAGE, x.shape[-1]), device="cuda")
    dense[:, at] = x
    isnew = torch.zeros((len(blocks) * PAGE,), dtype=torch.bool, device="cuda")
    isnew[at] = True
    isnew = isnew.view(-1, PAGE)
    dense = _blocks(case, dense)
    before = scale[:, blocks]
    after = _scale(dense.abs().amax((-1, -2)))
    # a block whose first row is new begins anew, the others keep or grow their scale
    after = torch.where(isnew[:, 0][None, :, None], after, torch.maximum(after, before))
    kept = values[:, blocks].view(torch.float8_e4m3fn).float() * (before / after)[..., None, None]
    merged = torch.where(isnew[None, :, None, :, None], dense / after[..., None, None], kept)
    merged = merged.clamp(-448, 448).to(torch.float8_e4m3fn)
    values[:, blocks] = merged.view(torch.uint8)
    scale[:, blocks] = after
    return merged.float() * after[..., None, None]


def _plain_block(s):
    case, n_new = s["case"], s["case"]["new"]
    touched = [_plain_append(s, i) for i in (0, 1)]
    if case["op"] == "append":
        keep = torch.tensor(np.concatenate([np.arange(-(-(n + n_new) // PAGE) * PAGE - n // PAGE * PAGE)
                                            < n + n_new - n // PAGE * PAGE for n in s["ctx"]]), device="cuda")
        out = {}
        for name, x in zip("kv", touched):
            x = x.transpose(2, 3).reshape(case["n_layer"], len(keep), -1)[:, keep]
            out[name] = x if case["n_layer"] > 1 else x[0]
        return out
    d, h, hq = case["head_dim"], case["n_head"], case["n_q_head"]
    q = s["q"] if case["n_layer"] > 1 else s["q"][None]
    out = torch.empty_like(q)
    for i, n in enumerate(s["ctx"]):
        blocks = torch.arange(int(s["first"][i]), int(s["first"][i + 1]), device="cuda")
        k, v = (_values(held, blocks).transpose(1, 2).flatten(2, 3)[:, :, :n + n_new] for held in s["held"])
        x = q[:, i * n_new:(i + 1) * n_new].view(-1, n_new, h, hq // h, d).permute(0, 2, 3, 1, 4).reshape(-1, h, hq // h * n_new, d)
        score = torch.matmul(x / math.sqrt(d), k.transpose(-1, -2).contiguous())
        if n_new > 1:
            late = torch.arange(n + n_new, device="cuda") > n + torch.arange(n_new, device="cuda")[:, None]
            score = score.masked_fill(late.repeat(hq // h, 1), -math.inf)
        e = torch.exp(score - score.amax(-1, keepdim=True))
        y = torch.matmul(e, v) / e.sum(-1, keepdim=True)
        out[:, i * n_new:(i + 1) * n_new] = y.view(-1, h, hq // h, n_new, d).permute(0, 3, 1, 2, 4).flatten(2)
    return out if case["n_layer"] > 1 else out[0]


# --------------------------------------------------------------------- work


def work(case):
    if case["kind"] == "pages":
        head = 2 * case["n_layer"] * case["n_head"]  # blocks of a page
        if case["op"] == "compact":
            n = sum(-(-n // PAGE) for n in _contexts(case)) * _block_bytes(case)
        elif case["op"] == "fork":
            n = case["beams"] * sum(len(_row_bytes(case, n % PAGE)) for n in _contexts(case))
        else:
            n = sum(len(_row_bytes(case, (n + case["grown"]) % PAGE)) * sum(w != p for w, p in enumerate(ps))
                    for n, ps in zip(_contexts(case), _parents(case)))
        return {"bytes": 2 * head * n, "flops": 0}
    if case["kind"] == "beam":
        rows = case["searches"] * case["beams"] * (1 - case["finished"])
        size = 4 if case["dtype"] == "f32" else 2
        out = case["searches"] * case["k"] * (12 + 8 * case["history"])
        return {"bytes": int(rows * size * case["vocab"]) + out, "flops": int(4 * rows * case["vocab"])}
    layers, d, h, hq = case["n_layer"], case["head_dim"], case["n_head"], case["n_q_head"]
    ctx, r = _contexts(case), case["new"]
    rows = len(ctx) * r
    append = rows * h * d * 2 * 5  # f32 in, 8 bits out
    if case["op"] == "append":
        touched = sum(n % PAGE + r for n in ctx)
        return {"bytes": layers * (append + touched * h * d * 2 * 5), "flops": layers * rows * h * d * 4}
    keys = sum(n + r for n in ctx)
    pairs = sum(r * (n + r) - r * (r - 1) // 2 for n in ctx)
    return {"bytes": layers * (append + keys * h * d * 2 + rows * hq * d * 8), "flops": layers * 4 * d * hq * pairs}


# -------------------------------------------------------------------- exact


def exact(case, seed):
    if case["kind"] == "pages":
        return None  # bytes that are moved: nothing is computed
    return _exact_beam(case, seed) if case["kind"] == "beam" else _exact_block(case, seed)


def _exact_beam(case, seed):
    """Every search's candidates sorted, in 64 bits."""
    logits, scores, finished, history = _beam_inputs(case, seed)
    v, k = case["vocab"], case["k"]
    out = dict(out_scores=[], parents=[], tokens=[], out_history=[])
    for i in range(case["searches"]):
        total = torch.log_softmax(logits[i].double(), -1) + scores[i].double()[:, None]
        if finished is not None:
            for w in torch.nonzero(finished[i])[:, 0].tolist():
                total[w] = -math.inf
                total[w, v - 1] = scores[i, w].double()
        total = torch.nan_to_num(total, nan=-math.inf, neginf=-math.inf)
        best, at = torch.sort(total.flatten(), descending=True, stable=True)
        best, at = best[:k], at[:k]
        if len(best) < k:
            best, at = (torch.nn.functional.pad(x, (0, k - len(best)), value=y) for x, y in ((best, -math.inf), (at, 0)))
        at = torch.where(best == -math.inf, -1, at)
        out["out_scores"].append(best)
        out["parents"].append(torch.div(at, v, rounding_mode="floor").to(torch.int32))
        out["tokens"].append(torch.where(at < 0, at, at % v).to(torch.int32))
        if history is not None:
            rows = [history[i, p].tolist() if p >= 0 else [-1] * case["history"] for p in out["parents"][-1].tolist()]
            rows = [r + [t] for r, t in zip(rows, out["tokens"][-1].tolist())]
            out["out_history"].append(torch.tensor(rows, dtype=torch.int32, device="cuda"))
    return {name: torch.stack(x) for name, x in out.items() if x}


def _exact_stored(old, new):
    """What a block of 16 rows [.., rows, head_dim] holds of earlier rows and rows appended behind them, in 64 bits."""
    def power(x):
        top = x.abs().amax((-1, -2)).clamp_min(1e-300)
        return torch.exp2(torch.ceil(torch.log2(top / 448)).clamp(-117, 120))[..., None, None]

    def nearest(x):
        step = torch.exp2(torch.floor(torch.log2(x.abs().clamp_min(1e-300))).clamp_min(-6) - 3)
        return torch.round(x / step) * step

    if old is None:
        s = power(new)
        return nearest(new / s) * s
    s0 = power(old)
    s = torch.maximum(s0, power(new))
    return torch.cat([nearest(nearest(old / s0) * s0 / s), nearest(new / s)], -2) * s


def _exact_block(case, seed):
    old, new, q = _block_inputs(case, seed)
    d, h, hq, r = case["head_dim"], case["n_head"], case["n_q_head"], case["new"]
    heads = [x.double().view(case["n_layer"], -1, h, d).transpose(1, 2) if case["op"] == "append" or x.numel() < 1 << 28
             else x.view(case["n_layer"], -1, h, d).transpose(1, 2) for x in (*old, *new)]
    touched, out, at = ([], []), torch.empty(q.shape, dtype=torch.float64, device="cuda"), 0
    for i, n in enumerate(_contexts(case)):
        stored = []
        for j in (0, 1):
            a, b = heads[j][:, :, at:at + n].double(), heads[2 + j][:, :, i * r:(i + 1) * r].double()
            whole, parts = n // PAGE * PAGE, []
            if whole and case["op"] != "append":
                x = a[:, :, :whole].unflatten(2, (-1, PAGE))
                parts.append(_exact_stored(None, x).flatten(2, 3))
            m = min(r, PAGE - n % PAGE)  # the new rows in the block that holds the end
            parts.append(_exact_stored(a[:, :, whole:] if n > whole else None, b[:, :, :m]))
            full = (r - m) // PAGE * PAGE
            if full:
                parts.append(_exact_stored(None, b[:, :, m:m + full].unflatten(2, (-1, PAGE))).flatten(2, 3))
            if r > m + full:
                parts.append(_exact_stored(None, b[:, :, m + full:]))
            x = torch.cat(parts, 2)
            stored.append(x)
            if case["op"] == "append":
                touched[j].append(x.transpose(1, 2).flatten(2))
        at += n
        if case["op"] == "append":
            continue
        k, v = stored
        for layer in range(case["n_layer"]):
            x = q[layer, i * r:(i + 1) * r].double().view(r, h, hq // h, d)
            for g in range(hq // h):
                score = torch.matmul(x[:, :, g].transpose(0, 1), k[layer].transpose(1, 2).contiguous()) / math.sqrt(d)
                late = torch.arange(n + r, device="cuda") > torch.arange(n, n + r, device="cuda")[:, None]
                y = torch.matmul(torch.softmax(score.masked_fill(late, -math.inf), -1), v[layer])
                out[layer, i * r:(i + 1) * r].view(r, h, hq // h, d)[:, :, g] = y.transpose(0, 1)
    if case["op"] == "append":
        k, v = (torch.cat(x, 1) for x in touched)
        return {"k": k, "v": v} if case["n_layer"] > 1 else {"k": k[0], "v": v[0]}
    return out if case["n_layer"] > 1 else out[0]
