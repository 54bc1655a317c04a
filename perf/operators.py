"""Rotary positions, the rotating append, shared-prefix attention and draft
verification as measurable cases: one step of sampled speculative decoding
with a model that has rotary positions and grouped heads.

* ``rotary``: rows of heads rotated to their positions (contiguous rows);
* ``append``: keys rotated on their way into the paged cache, values beside
  them, queries rotated on their way to the attention;
* ``prefix``: paged attention of sequences that share prefixes held once;
* ``verify``: drafted tokens accepted or rejected against the target's
  probabilities, and the token after them drawn.

Where ``own`` is false a pass is elementary torch operations; where it is true
it is the package's calls on the same inputs.  Contexts and page orders follow
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


def _rope(base=10000.0, rot_dim=0, interleaved=False, scaling="none", factor=1.0, orig_ctx=0):
    """rot_dim 0: the whole head."""
    return dict(base=base, rot_dim=rot_dim, interleaved=interleaved, scaling=scaling, factor=factor, orig_ctx=orig_ctx)


def _rotary(rows, n_head, head_dim, pos_lo, pos_hi, dtype="f32", rope=None):
    """Rows at positions pos_lo..pos_hi: consecutive from pos_lo where pos_hi is 0."""
    return dict(kind="rotary", rows=rows, n_head=n_head, head_dim=head_dim, pos_lo=pos_lo, pos_hi=pos_hi, dtype=dtype,
                **(rope or _rope()))


def _append(shape, n_layer, seqs, ctx_lo, ctx_hi, new, offset=0, rope=None, ctx_seed=1):
    """seqs sequences of ctx_lo..ctx_hi positions, each appending `new` rows;
    their positions count from `offset` (the length of a prefix before them)."""
    return dict(kind="append", **shape, n_layer=n_layer, seqs=seqs, ctx_lo=ctx_lo, ctx_hi=ctx_hi, new=new,
                offset=offset, **(rope or _rope()), ctx_seed=ctx_seed)


def _prefix(shape, n_layer, seqs, ctx_lo, ctx_hi, query, prefix, groups=1, bare=False, q8=False, ctx_seed=1):
    """seqs sequences of ctx_lo..ctx_hi positions of their own, the last
    `query` of them queried, behind `groups` prefixes of `prefix` positions at
    most; `bare`: the last sequence has no prefix."""
    return dict(kind="prefix", **shape, n_layer=n_layer, seqs=seqs, ctx_lo=ctx_lo, ctx_hi=ctx_hi, query=query,
                prefix=prefix, groups=groups, bare=bare, q8=q8, ctx_seed=ctx_seed)


def _verify(seqs, drafts, vocab, dtype="f32", draft_probs=True, ragged=False, temp=2.5):
    return dict(kind="verify", seqs=seqs, drafts=drafts, vocab=vocab, dtype=dtype, draft_probs=draft_probs,
                ragged=ragged, temp=temp)


def listed():
    return [
        # A decode batch's queries rotated to their positions: the smallest launch.
        dict(_rotary(64, 12, 64, 1, 1023), name="rotary-64"),
        # A document's queries and keys at far positions, scaled for a long context, half of each head rotated.
        dict(_rotary(4095, 40, 128, 28001, 0, "bf16", _rope(rot_dim=64, interleaved=True, scaling="linear",
                                                            factor=4.0)), name="rotary-prompt-bf16"),
        # One layer of a decode batch: every sequence appends a token.
        dict(_append(GPT2, 1, 64, 32, 767, 1, ctx_seed=2), name="append-64"),
        # Every layer of a verify step: four drafts and a token a sequence, behind a shared prefix.
        dict(_append(GPT2, 12, 32, 3, 60, 5, offset=2047, ctx_seed=3), name="append-32x5-layers"),
        # One layer of a long prompt with grouped heads at far positions of a stretched context.
        dict(_append(GROUPED, 1, 1, 1, 1, 2047, offset=30000, rope=_rope(base=500000.0, scaling="yarn", factor=8.0,
                                                                         orig_ctx=8192), ctx_seed=4),
             name="append-prompt-2047"),
        # Two users of one short instruction: the smallest attention call.
        dict(_prefix(GPT2, 1, 2, 17, 60, 1, 515, ctx_seed=5), name="prefix-2"),
        # A serving batch behind one system prompt, every layer in one call.
        dict(_prefix(GPT2, 12, 64, 1, 255, 1, 1023, ctx_seed=6), name="prefix-64-layers"),
        # Drafts verified on the int8 cache behind two prompts, one sequence without any.
        dict(_prefix(GPT2, 1, 32, 5, 300, 5, 2001, groups=2, bare=True, q8=True, ctx_seed=7), name="prefix-32x5-q8"),
        # Many questions about one document, grouped heads.
        dict(_prefix(GROUPED, 1, 48, 1, 511, 1, 8185, ctx_seed=8), name="prefix-48-grouped"),
        # A few questions about a book: the cache is the whole cost.
        dict(_prefix(LONG, 1, 16, 1, 511, 1, 32767, ctx_seed=9), name="prefix-16x32k"),
        # One user's drafts.
        dict(_verify(1, 4, 50257), name="verify-1x4"),
        # A serving batch's drafts over a large vocabulary, each sequence with as many drafts as it had time for.
        dict(_verify(64, 7, 131071, ragged=True), name="verify-64x7"),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


def _draw_rope(rng, head_dim):
    scaling = rng.choice(["none", "linear", "ntk", "yarn"])
    return _rope(base=rng.choice([10000.0, 500000.0, 1000000.0]),
                 rot_dim=rng.choice([0, 0, head_dim // 2, head_dim // 4, head_dim - 8]), interleaved=rng.random() < 0.5,
                 scaling=scaling, factor=1.0 if scaling == "none" else rng.choice([2.0, 4.0, 8.0, 5.5]),
                 orig_ctx=rng.choice([2048, 4096, 8192]) if scaling == "yarn" else 0)


def draw(rng: random.Random):
    kind = rng.choice(["rotary", "append", "append-prompt", "prefix", "prefix", "prefix-long", "verify"])
    cs = rng.randrange(1 << 30)
    if kind == "rotary":
        head_dim = rng.choice([64, 64, 128, 80, 256])
        rows = _log(rng, 1, 4000)
        lo, hi = rng.randint(0, 100000), 0
        if rng.random() < 0.5:
            hi = lo + rng.randint(1, 1000000)
        return _rotary(rows, rng.randint(1, 32 if head_dim <= 128 else 16), head_dim, lo, hi,
                       rng.choice(["f32", "f16", "bf16"]), _draw_rope(rng, head_dim))
    shape = rng.choice([GPT2, GROUPED, LONG])
    n_layer = rng.choice([1, 1, 1, 12]) if shape is GPT2 else 1
    if kind == "append":
        hi = rng.randint(2, 60 if n_layer > 1 else 600 if shape is GPT2 else 120)
        return _append(shape, n_layer, _log(rng, 1, 64 if n_layer == 1 else 32), rng.randint(1, hi), hi,
                       rng.choice([1, 1, 2, 5, 9]), rng.choice([0, rng.randint(1, 100000)]),
                       _draw_rope(rng, shape["head_dim"]), cs)
    if kind == "append-prompt":
        ctx = rng.choice([1, rng.randint(1, 200)])
        return _append(shape, 1, rng.randint(1, 2), ctx, ctx, _log(rng, 17, 1000),
                       rng.choice([0, rng.randint(1, 30000)]), _draw_rope(rng, shape["head_dim"]), cs)
    if kind == "prefix":
        query = rng.choice([1, 1, 1, 3, 5, 8])
        hi = rng.randint(query, 400)
        n = _log(rng, 1, 4000)
        most, pairs = (64, 500000) if n_layer == 1 else (32, 220000)
        seqs = _log(rng, 1, max(1, min(most, pairs // (query * (n + hi)))))
        return _prefix(shape, n_layer, seqs, rng.randint(query, hi), hi, query, n,
                       groups=rng.randint(1, min(4, seqs)), bare=rng.random() < 0.3, q8=rng.random() < 0.3, ctx_seed=cs)
    if kind == "prefix-long":
        hi, n = rng.randint(1, 500), _log(rng, 4000, 32000)
        return _prefix(rng.choice([GPT2, GROUPED]), 1, rng.randint(1, 390000 // n), rng.randint(1, hi), hi, 1, n,
                       q8=rng.random() < 0.3, ctx_seed=cs)
    return _verify(_log(rng, 1, 64), rng.randint(1, 7), _log(rng, 500, 131071), rng.choice(["f32", "f16", "bf16"]),
                   draft_probs=rng.random() < 0.75, ragged=rng.random() < 0.5, temp=rng.choice([1.0, 2.5, 4.0]))


# ------------------------------------------------------------------- shapes


def _contexts(case):
    rng = random.Random(case["ctx_seed"])
    return [rng.randint(case["ctx_lo"], case["ctx_hi"]) for _ in range(case["seqs"])]


def _prefixes(case):
    """(length, sequences behind it) of each prefix; a last one of length 0 where the case has a bare sequence."""
    rng = random.Random(case["ctx_seed"] + 2)
    behind = case["seqs"] - (1 if case["bare"] and case["seqs"] > 1 else 0)
    groups = min(case["groups"], behind)
    cuts = [behind * i // groups for i in range(groups + 1)]
    out = [(case["prefix"] if i == 0 else rng.randint(1, case["prefix"]), cuts[i + 1] - cuts[i]) for i in range(groups)]
    return out + ([(0, 1)] if behind < case["seqs"] else [])


def _tables(case, lengths):
    """(pages in the pool, their order, the pages of each sequence) where
    sequences of these lengths are reserved one after another."""
    need = [-(-n // PAGE) for n in lengths]
    total = sum(need) + 3
    order = list(range(total))
    random.Random(case["ctx_seed"] + 1).shuffle(order)
    tables, at = [], 0
    for n in need:
        tables.append(order[at:at + n])
        at += n
    return total, order, tables


# ------------------------------------------------------------------- inputs


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(g, shape, std=1.0):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32) * std


def _positions(case, seed):
    if case["pos_hi"] == 0:
        return np.arange(case["pos_lo"], case["pos_lo"] + case["rows"])
    return np.random.default_rng(seed).integers(case["pos_lo"], case["pos_hi"] + 1, case["rows"])


def _cache_inputs(case, g, n_pages):
    """The cache's contents: [n_layer, pages, heads, K|V, 16, head_dim] f16, or
    (int8 values of that shape, f32 scales without the last axis)."""
    shape = (case["n_layer"], n_pages, case["n_head"], 2, PAGE, case["head_dim"])
    if not case.get("q8"):
        return torch.randn(shape, generator=g, device="cuda", dtype=torch.float16)
    x = torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)
    scale = x.abs().amax(-1) / 127
    return torch.round(x / scale[..., None]).clamp(-127, 127).to(torch.int8), scale


def _verify_inputs(case, seed):
    g = _gen(seed)
    b, k, v = case["seqs"], case["drafts"], case["vocab"]
    logits = _normal(g, (b, k + 1, v), case["temp"])
    target = torch.softmax(logits, -1).to(DTYPES[case["dtype"]])
    draft, guess = None, logits[:, :k] + _normal(g, (b, k, v), 0.7)
    if case["draft_probs"]:
        draft = torch.softmax(guess, -1).to(DTYPES[case["dtype"]])
    # the drafter's own choice: drawn from its probabilities, or the most likely token
    if case["draft_probs"]:
        u = torch.rand(guess.shape, generator=g, device="cuda").clamp_min(1e-20)
        guess = guess - torch.log(-torch.log(u).clamp_min(1e-20))
    drafted = guess.argmax(-1).to(torch.int32)
    u = torch.rand((b, k + 1), generator=g, device="cuda")
    n_drafts = torch.full((b,), k, dtype=torch.int32, device="cuda")
    if case["ragged"]:
        n_drafts = torch.randint(0, k + 1, (b,), generator=g, device="cuda", dtype=torch.int32)
    return target, draft, drafted, u[:, :k].contiguous(), u[:, k].contiguous(), n_drafts


# ------------------------------------------------------------------ prepare


class _Pool:
    """A device pool's memory, for torch to view."""

    def __init__(self, kv, n_bytes):
        self.kv = kv  # keeps the pool alive
        self.__cuda_array_interface__ = dict(shape=(n_bytes,), typestr="|u1", data=(kv.pools()[0], False), version=2)


def _cache(case, contents, n_pages, order, lengths):
    """(the cache, its contents as tensors): the package's PagedKv with each
    sequence's pages reserved, its memory viewed in place, or the tensors alone."""
    if not own:
        return None, contents
    import nanoinfer_amd as na

    kv = na.PagedKv(na.BatchOpts(n_layer=case["n_layer"], n_head=case["n_head"], head_dim=case["head_dim"],
                                 kv_blocks=n_pages, max_seqs=len(lengths), n_ctx=max(lengths), max_rows=4096,
                                 page_order=order, q8=bool(case.get("q8"))))
    for n in lengths:
        kv.reserve(kv.add_seq(), n)
    raw = torch.as_tensor(_Pool(kv, kv.pools()[2]), device="cuda")
    if not case.get("q8"):
        view = raw.view(torch.float16).view(contents.shape)
        view.copy_(contents)
        return kv, view
    values, scale = contents
    blocks = raw.view(*scale.shape[:-1], PAGE * case["head_dim"] + 4 * PAGE)
    blocks[..., :PAGE * case["head_dim"]].copy_(values.reshape(*scale.shape[:-1], -1).view(torch.uint8))
    blocks[..., PAGE * case["head_dim"]:].copy_(scale.contiguous().view(torch.uint8))
    return kv, raw


def _rotation(case):
    """What a program keeps of the model's rotation: the package's Rotary, or the frequencies and the scale."""
    if own:
        import nanoinfer_amd as na

        scaling = None if case["scaling"] == "none" else case["scaling"]
        return na.Rotary(case["head_dim"], base=case["base"], rot_dim=case["rot_dim"] or None,
                         interleaved=case["interleaved"], scaling=scaling, factor=case["factor"],
                         orig_ctx=case["orig_ctx"])
    freq, scale = _frequencies(case)
    return torch.tensor(freq, dtype=torch.float64, device="cuda"), scale


def _frequencies(case):
    r, base, s = case["rot_dim"] or case["head_dim"], case["base"], case["factor"]
    i = np.arange(r // 2, dtype=np.float64)
    if case["scaling"] == "ntk":
        base = base * s ** (r / (r - 2))
    freq = base ** (-2 * i / r)
    if case["scaling"] == "linear":
        return freq / s, 1.0
    if case["scaling"] == "yarn":
        def pair(turns):  # the pair that makes this many turns over the original context
            return r * math.log(case["orig_ctx"] / (turns * 2 * math.pi)) / (2 * math.log(base))

        lo, hi = max(math.floor(pair(32.0)), 0), min(math.ceil(pair(1.0)), r - 1)
        ramp = np.clip((i - lo) / max(hi - lo, 0.001), 0, 1)
        return freq / s * ramp + freq * (1 - ramp), 0.1 * math.log(s) + 1 if s > 1 else 1.0
    return freq, 1.0


def _append_inputs(case, seed):
    """Rows (seq, pos), positions, the fused [n_layer, n, q|k|v] buffer, the cache and its tables."""
    g = _gen(seed)
    ctx, new = _contexts(case), case["new"]
    n_pages, order, tables = _tables(case, [c + new for c in ctx])
    rows = np.array([(s, c + t) for s, c in enumerate(ctx) for t in range(new)], dtype=np.uint32)
    width = (case["n_q_head"] + 2 * case["n_head"]) * case["head_dim"]
    fused = _normal(g, (case["n_layer"], len(rows), width))
    return rows, fused, _cache_inputs(case, g, n_pages), n_pages, order, tables, [c + new for c in ctx]


def _split_fused(case, fused):
    """q, k and v as views of the fused buffer; of one layer without the layer axis."""
    if case["n_layer"] == 1:
        fused = fused[0]
    c, cq = case["n_head"] * case["head_dim"], case["n_q_head"] * case["head_dim"]
    return fused[..., :cq], fused[..., cq:cq + c], fused[..., cq + c:]


def prepare(case, seed):
    g = _gen(seed)
    kind = case["kind"]
    if kind == "rotary":
        pos = _positions(case, seed)
        x = _normal(g, (case["rows"], case["n_head"] * case["head_dim"])).to(DTYPES[case["dtype"]])
        return dict(case=case, x=x, out=torch.empty_like(x), rotation=_rotation(case),
                    positions=torch.tensor(pos, dtype=torch.int32, device="cuda"))
    if kind == "append":
        rows, fused, contents, n_pages, order, tables, lengths = _append_inputs(case, seed)
        kv, pool = _cache(case, contents, n_pages, order, lengths)
        q, k, v = _split_fused(case, fused)
        pos = (rows[:, 1] + case["offset"]).astype(np.uint32)
        state = dict(case=case, kv=kv, pool=pool, rows=rows, q=q, k=k, v=v, positions=pos, rotation=_rotation(case),
                     q_out=torch.empty(q.shape, device="cuda"))
        if not own:
            state["angles_at"] = torch.tensor(pos.astype(np.int64), device="cuda")
            state["page"] = torch.tensor([tables[s][p // PAGE] for s, p in rows.tolist()], device="cuda")
            state["slot"] = torch.tensor(rows[:, 1].astype(np.int64) % PAGE, device="cuda")
        return state
    if kind == "prefix":
        ctx, prefixes = _contexts(case), _prefixes(case)
        shared = [(n, s) for n, s in prefixes if n > 0]
        lengths = ctx + [n for n, _ in shared]
        n_pages, order, tables = _tables(case, lengths)
        contents = _cache_inputs(case, g, n_pages)
        kv, pool = _cache(case, contents, n_pages, order, lengths)
        r = case["query"]
        rows = np.array([(s, c - r + t) for s, c in enumerate(ctx) for t in range(r)], dtype=np.uint32)
        q = _normal(g, (case["n_layer"], len(rows), case["n_q_head"] * case["head_dim"]))
        q = q[0] if case["n_layer"] == 1 else q
        state = dict(case=case, kv=kv, pool=pool, rows=rows, q=q, out=torch.empty_like(q),
                     prefixes=[(len(ctx) + min(i, len(shared) - 1), n, s * r) for i, (n, s) in enumerate(prefixes)])
        if not own:
            longest = max(len(tables[s]) for s in range(len(ctx)))
            padded = [tables[s] + [0] * (longest - len(tables[s])) for s in range(len(ctx))]
            state["own_pages"] = torch.tensor(padded, device="cuda")
            state["shared_pages"] = [torch.tensor(t, device="cuda") for t in tables[len(ctx):]]
            state["last"] = torch.tensor(rows[:, 1].astype(np.int64), device="cuda").view(len(ctx), r)
            state["groups"] = prefixes
        return state
    target, draft, drafted, accept_u, sample_u, n_drafts = _verify_inputs(case, seed)
    return dict(case=case, target=target, draft=draft, drafted=drafted, accept_u=accept_u, sample_u=sample_u,
                n_drafts=n_drafts if case["ragged"] else None,
                accepted=torch.empty((case["seqs"],), dtype=torch.int32, device="cuda"),
                tokens=torch.empty((case["seqs"], case["drafts"] + 1), dtype=torch.int32, device="cuda"))


# ---------------------------------------------------------------------- run


def run(s):
    return (_run_own if own else _run_plain)(s)


def _run_own(s):
    import nanoinfer_amd as na

    case, kind = s["case"], s["case"]["kind"]
    if kind == "rotary":
        return na.rotary(s["x"], s["rotation"], case["n_head"], positions=s["positions"], out=s["out"])
    if kind == "append":
        layer = 0 if case["n_layer"] == 1 else na.ALL_LAYERS
        q = s["kv"].append_rotary(s["rows"], s["k"], s["v"], s["rotation"], q=s["q"], q_out=s["q_out"],
                                  positions=s["positions"], layer=layer)
        return {"q": q, "pool": s["pool"]}
    if kind == "prefix":
        layer = 0 if case["n_layer"] == 1 else na.ALL_LAYERS
        return s["kv"].prefix_attention(s["q"], s["rows"], s["prefixes"], out=s["out"], layer=layer)
    accepted, tokens = na.verify_drafts(s["target"], s["drafted"], s["accept_u"], s["sample_u"], draft=s["draft"],
                                        n_drafts=s["n_drafts"], accepted=s["accepted"], tokens=s["tokens"])
    return {"accepted": accepted, "tokens": tokens}


def _turn(case, x, cos, sin):
    """x [..., rows, heads, head_dim] f32 turned by cos and sin [rows, 1, pairs]."""
    r = case["rot_dim"] or case["head_dim"]
    out = x.clone()
    if case["interleaved"]:
        a, b = x[..., 0:r:2], x[..., 1:r:2]
        out[..., 0:r:2], out[..., 1:r:2] = a * cos - b * sin, b * cos + a * sin
    else:
        a, b = x[..., :r // 2], x[..., r // 2:r]
        out[..., :r // 2], out[..., r // 2:r] = a * cos - b * sin, b * cos + a * sin
    return out


def _cos_sin(rotation, positions):
    freq, scale = rotation
    angle = positions.double()[:, None, None] * freq
    return (torch.cos(angle) * scale).float(), (torch.sin(angle) * scale).float()


def _heads(x, case):
    return x.reshape(*x.shape[:-1], -1, case["head_dim"])


def _run_plain(s):
    case, kind = s["case"], s["case"]["kind"]
    if kind == "rotary":
        cos, sin = _cos_sin(s["rotation"], s["positions"])
        return _turn(case, _heads(s["x"].float(), case), cos, sin).reshape(s["x"].shape).to(s["x"].dtype)
    if kind == "append":
        cos, sin = _cos_sin(s["rotation"], s["angles_at"])
        q = _turn(case, _heads(s["q"], case), cos, sin).reshape(s["q"].shape)
        k, v = _turn(case, _heads(s["k"], case), cos, sin), _heads(s["v"], case)
        for i, x in enumerate((k, v)):
            x = x if case["n_layer"] > 1 else x[None]
            s["pool"][:, s["page"], :, i, s["slot"], :] = x.transpose(0, 1).to(torch.float16)
        return {"q": q, "pool": s["pool"]}
    if kind == "prefix":
        return _plain_attention(s)
    return _plain_verify(s)


def _keys_values(s, layer, pages):
    """K and V f32 [..., heads, 16 * pages, head_dim] of page ids [..., pages]."""
    case = s["case"]
    if case["q8"]:
        values, scale = s["pool"]
        kv = values[layer][pages].float() * scale[layer][pages][..., None]
    else:
        kv = s["pool"][layer][pages].float()
    # [..., pages, heads, 2, 16, hd] -> [2, ..., heads, pages, 16, hd]
    n = kv.dim()
    kv = kv.permute(n - 3, *range(n - 5), n - 4, n - 5, n - 2, n - 1)
    return kv.reshape(*kv.shape[:-3], -1, case["head_dim"]).unbind(0)


def _plain_attention(s):
    case = s["case"]
    h, d, g, r = case["n_head"], case["head_dim"], case["n_q_head"] // case["n_head"], case["query"]
    n_seq = case["seqs"]
    out = torch.empty_like(s["q"])
    hidden = torch.arange(s["own_pages"].shape[1] * PAGE, device="cuda")[None, None, :] > s["last"][:, :, None]
    hidden = hidden.repeat_interleave(g, 1)[:, None]  # [seqs, 1, rows * g, keys]
    for layer in range(case["n_layer"]):
        q = (s["q"] if case["n_layer"] == 1 else s["q"][layer]).view(n_seq, r, h, g, d)
        q = q.permute(0, 2, 1, 3, 4).reshape(n_seq, h, r * g, d) / math.sqrt(d)
        k, v = _keys_values(s, layer, s["own_pages"])
        score = torch.matmul(q, k.transpose(-1, -2).contiguous()).masked_fill(hidden, -math.inf)
        parts, at = [], 0
        for i, (n, behind) in enumerate(s["groups"]):
            mine = score[at:at + behind]
            if n == 0:
                e = torch.exp(mine - mine.amax(-1, keepdim=True))
                parts.append(torch.matmul(e, v[at:at + behind]) / e.sum(-1, keepdim=True))
                continue
            pk, pv = (x[:, :n] for x in _keys_values(s, layer, s["shared_pages"][i]))
            pq = q[at:at + behind].transpose(0, 1).reshape(h, behind * r * g, d)
            shared = torch.matmul(pq, pk.transpose(-1, -2).contiguous()).view(h, behind, r * g, n).transpose(0, 1)
            m = torch.maximum(shared.amax(-1, keepdim=True), mine.amax(-1, keepdim=True))
            shared, mine = torch.exp(shared - m), torch.exp(mine - m)
            o = torch.matmul(shared.transpose(0, 1).reshape(h, behind * r * g, n), pv)
            o = o.view(h, behind, r * g, d).transpose(0, 1) + torch.matmul(mine, v[at:at + behind])
            parts.append(o / (shared.sum(-1, keepdim=True) + mine.sum(-1, keepdim=True)))
            at += behind
        o = torch.cat(parts).view(n_seq, h, r, g, d).permute(0, 2, 1, 3, 4).reshape(n_seq * r, h * g * d)
        (out if case["n_layer"] == 1 else out[layer]).copy_(o)
    return out


def _plain_verify(s):
    case = s["case"]
    target, draft, drafted = s["target"], s["draft"], s["drafted"].long()
    b, k = drafted.shape
    n = torch.full((b,), k, device="cuda") if s["n_drafts"] is None else s["n_drafts"].long()
    p = target[:, :k].gather(2, drafted[..., None])[..., 0].double()
    q = torch.ones_like(p) if draft is None else draft.gather(2, drafted[..., None])[..., 0].double()
    step = torch.arange(k, device="cuda")
    ok = (s["accept_u"].double() * q < p) & (step < n[:, None])
    accepted = ok.long().cumprod(1).sum(1)
    rejected = accepted < n
    each = torch.arange(b, device="cuda")
    row = target[each, accepted].double()
    at = accepted.clamp_max(k - 1)
    if draft is None:
        left = row.clone()
        left[each, drafted[each, at]] = 0
    else:
        left = (row - draft[each, at].double()).clamp_min(0)
    left = torch.where(rejected[:, None] & (left.sum(1, keepdim=True) > 0), left, row)
    run_sum = left.cumsum(1)
    drawn = (run_sum <= s["sample_u"].double()[:, None] * run_sum[:, -1:]).sum(1).clamp_max(case["vocab"] - 1)
    place = torch.arange(k + 1, device="cuda")
    tokens = torch.where(place < accepted[:, None], torch.cat([drafted, drafted[:, :1]], 1), torch.full_like(place, -1))
    tokens = torch.where(place == accepted[:, None], drawn[:, None], tokens)
    return {"accepted": accepted.to(torch.int32), "tokens": tokens.to(torch.int32)}


# --------------------------------------------------------------------- work


def work(case):
    kind = case["kind"]
    if kind == "rotary":
        n = case["rows"] * case["n_head"] * case["head_dim"]
        size = 4 if case["dtype"] == "f32" else 2
        return {"bytes": 2 * size * n + 4 * case["rows"], "flops": 3 * n}
    if kind == "append":
        rows = case["seqs"] * case["new"] * case["n_layer"]
        d, hq, h = case["head_dim"], case["n_q_head"], case["n_head"]
        return {"bytes": rows * d * (8 * hq + 12 * h), "flops": 3 * rows * d * (hq + h)}
    if kind == "prefix":
        d, hq, h, r = case["head_dim"], case["n_q_head"], case["n_head"], case["query"]
        ctx, prefixes = _contexts(case), _prefixes(case)
        keys = sum(ctx) + sum(n for n, _ in prefixes)
        pairs = sum(r * c - r * (r - 1) // 2 for c in ctx) + sum(n * s * r for n, s in prefixes)
        rows = len(ctx) * r
        key_bytes = 2 * (d + 4) if case["q8"] else 4 * d
        layers = case["n_layer"]
        return {"bytes": layers * (keys * h * key_bytes + rows * hq * d * 8), "flops": layers * 4 * d * hq * pairs}
    # the distribution after the last accepted token, and the drafter's where that is a rejection
    size = 4 if case["dtype"] == "f32" else 2
    rows = 2 if case["draft_probs"] else 1
    return {"bytes": case["seqs"] * (rows * size * case["vocab"] + case["drafts"] * (2 * size + 12)),
            "flops": 2 * case["seqs"] * case["vocab"]}


# -------------------------------------------------------------------- exact


def exact(case, seed):
    kind = case["kind"]
    if kind == "rotary":
        g = _gen(seed)
        x = _normal(g, (case["rows"], case["n_head"] * case["head_dim"])).to(DTYPES[case["dtype"]])
        return _exact_turn(case, x.double(), _positions(case, seed))
    if kind == "append":
        rows, fused, pool, _, _, tables, _ = _append_inputs(case, seed)
        q, k, v = _split_fused(case, fused.double())
        pos = rows[:, 1].astype(np.int64) + case["offset"]
        pool = pool.double()
        k = _exact_turn(case, k, pos)
        for i, (s, p) in enumerate(rows.tolist()):
            block = pool[:, tables[s][p // PAGE], :, :, p % PAGE]  # [n_layer, heads, 2, hd]
            for j, x in enumerate((k, v)):
                block[:, :, j] = x[..., i, :].reshape(-1, case["n_head"], case["head_dim"])
        return {"q": _exact_turn(case, q, pos), "pool": pool}
    if kind == "prefix":
        return _exact_attention(case, seed)
    return _exact_verify(case, seed)


def _exact_turn(case, x, positions):
    """Pairs as complex numbers times scale * e^(i angle), in 64 bits."""
    r = case["rot_dim"] or case["head_dim"]
    freq, scale = _frequencies(case)
    angle = torch.tensor(np.asarray(positions, dtype=np.float64)[:, None] * freq, device="cuda")
    turn = torch.polar(torch.full_like(angle, scale), angle)[:, None]
    y = x.reshape(*x.shape[:-1], -1, case["head_dim"]).clone()
    part = y[..., :r]
    pairs = part.unflatten(-1, (r // 2, 2)) if case["interleaved"] else part.unflatten(-1, (2, r // 2)).transpose(-1, -2)
    z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
    y[..., :r] = (z if case["interleaved"] else z.transpose(-1, -2)).flatten(-2)
    return y.reshape(x.shape)


def _exact_attention(case, seed):
    g = _gen(seed)
    ctx, prefixes = _contexts(case), _prefixes(case)
    shared = [n for n, _ in prefixes if n > 0]
    n_pages, _, tables = _tables(case, ctx + shared)
    contents = _cache_inputs(case, g, n_pages)
    h, d, hq, r = case["n_head"], case["head_dim"], case["n_q_head"], case["query"]
    q = _normal(g, (case["n_layer"], len(ctx) * r, hq * d)).double()
    out = torch.empty_like(q)

    def stored(layer, table, n):
        """K and V [heads, n, hd] of a sequence."""
        table = torch.tensor(table, device="cuda")
        if case["q8"]:
            x = contents[0][layer][table].double() * contents[1][layer][table].double()[..., None]
        else:
            x = contents[layer][table].double()
        return x.permute(2, 1, 0, 3, 4).reshape(2, h, -1, d)[:, :, :n]

    for layer in range(case["n_layer"]):
        seq = 0
        for i, (n, behind) in enumerate(prefixes):
            front = stored(layer, tables[len(ctx) + i], n) if n else None
            for s in range(seq, seq + behind):
                k, v = stored(layer, tables[s], ctx[s])
                row = slice(s * r, (s + 1) * r)
                x = q[layer, row].reshape(r, h, hq // h, d).permute(1, 2, 0, 3).reshape(h, -1, d)
                score = torch.matmul(x, k.transpose(1, 2).contiguous()) / math.sqrt(d)
                late = torch.arange(ctx[s], device="cuda") > torch.arange(ctx[s] - r, ctx[s], device="cuda")[:, None]
                score = score.masked_fill(late.repeat(hq // h, 1), -math.inf)
                if n:
                    before = torch.matmul(x, front[0].transpose(1, 2).contiguous()) / math.sqrt(d)
                    weight = torch.softmax(torch.cat([before, score], -1), -1)
                    y = torch.matmul(weight[..., :n], front[1]) + torch.matmul(weight[..., n:], v)
                else:
                    y = torch.matmul(torch.softmax(score, -1), v)
                out[layer, row] = y.reshape(h, hq // h, r, d).permute(2, 0, 1, 3).reshape(r, hq * d)
            seq += behind
    return out[0] if case["n_layer"] == 1 else out


def _exact_verify(case, seed):
    target, draft, drafted, accept_u, sample_u, n_drafts = _verify_inputs(case, seed)
    drafted, accept_u, sample_u = drafted.cpu().numpy(), accept_u.double().cpu().numpy(), sample_u.double().cpu().numpy()
    n_drafts = n_drafts.cpu().numpy()
    k = case["drafts"]
    accepted = np.zeros(case["seqs"], dtype=np.int32)
    tokens = np.full((case["seqs"], k + 1), -1, dtype=np.int32)
    for b in range(case["seqs"]):
        a = 0
        while a < n_drafts[b]:
            t = int(drafted[b, a])
            q = 1.0 if draft is None else float(draft[b, a, t])
            if not accept_u[b, a] * q < float(target[b, a, t]):
                break
            tokens[b, a] = t
            a += 1
        p = target[b, a].double().cpu().numpy()
        w = p
        if a < n_drafts[b]:
            q = np.zeros_like(p) if draft is None else draft[b, a].double().cpu().numpy()
            if draft is None:
                q[drafted[b, a]] = p[drafted[b, a]]
            w = np.maximum(p - q, 0)
            w = w if w.sum() > 0 else p
        total = np.cumsum(w)
        accepted[b], tokens[b, a] = a, min(np.searchsorted(total, sample_u[b] * total[-1], side="right"), len(p) - 1)
    return {"accepted": torch.tensor(accepted, device="cuda"), "tokens": torch.tensor(tokens, device="cuda")}
