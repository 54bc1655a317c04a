"""Block-scaled pages that change hands: what a sequence writes is scaled by its
own rows, in whatever order and calls they come, whoever held the page before."""
import random

import pytest
import torch

import nanoinfer_amd as na
from test_gpu_block8 import PAGE, Model, _kv

pytestmark = pytest.mark.gpu


class Blocks(Model):
    """Model, where a block begins anew with a call that writes every row there is in it."""

    def __init__(self, *shape):
        super().__init__(*shape)
        self.rows = {}  # (sequence, page of it) -> rows written

    def append(self, rows, x):
        x = x.cpu().double().view(self.shape[0], -1, self.shape[1], self.shape[3])
        by = {}
        for i, (s, p) in enumerate(rows):
            by.setdefault((s, p // PAGE), []).append((p % PAGE, i))
        for key, new in by.items():
            slots, at = [a for a, _ in new], [b for _, b in new]
            there = self.rows.setdefault(key, set())
            y = x[:, at].transpose(1, 2)
            now = self.need(y.abs().amax((-1, -2)))
            values = torch.zeros(self.shape, dtype=torch.float64)
            if not there <= set(slots):
                values, e = self.blocks[key]
                now = torch.maximum(e, now)
                by2 = torch.exp2((e - now).double())[..., None, None]
                values = torch.where(by2 == 1, values, self.e4m3(values * by2))
            values[:, :, slots] = self.e4m3(y * torch.exp2(-now.double())[..., None, None])
            there.update(slots)
            self.blocks[key] = (values, now)

    def cut(self, s, n):
        """Truncated to n rows."""
        for key in [k for k in self.rows if k[0] == s]:
            self.rows[key] = {x for x in self.rows[key] if key[1] * PAGE + x < n}

    def become(self, s, parent, n):
        """s holds the first n rows of parent."""
        kept = {k[1]: (self.blocks[k], set(self.rows[k])) for k in self.rows if k[0] == parent and self.rows[k]}
        for key in [k for k in self.rows if k[0] == s]:
            del self.rows[key], self.blocks[key]
        for page, ((values, e), rows) in kept.items():
            self.blocks[s, page], self.rows[s, page] = (values.clone(), e.clone()), rows
        self.cut(s, n)


class Caches:
    """A cache whose pages all hold values of 1e30 of a sequence that is gone, and its models."""

    def __init__(self, pages=12, seqs=4, n_layer=2, n_head=2, head_dim=64, seed=1):
        self.g = torch.Generator("cuda").manual_seed(seed)
        self.kv = _kv(n_layer, n_head, head_dim, pages=pages, seqs=seqs)
        self.models = [Blocks(n_layer, n_head, head_dim) for _ in range(2)]
        old = self.kv.add_seq()
        n = pages * PAGE
        self.kv.reserve(old, n)
        x = torch.full((n_layer, n, n_head * head_dim), 1e30, device="cuda")
        self.kv.append([(old, p) for p in range(n)], x, x)
        self.kv.free_seq(old)

    def put(self, rows, size=1.0, models=True):
        x = [torch.randn((self.kv.opts.n_layer, len(rows), self.kv.opts.n_embd), generator=self.g, device="cuda") * size
             for _ in range(2)]
        self.kv.append(rows, *x)
        if models:
            for m, y in zip(self.models, x):
                m.append(rows, y)
        return x

    def check(self):
        rows = sorted((s, page * PAGE + x) for (s, page), there in self.models[0].rows.items() for x in there)
        for got, m in zip(self.kv.gather_values(rows), self.models):
            assert torch.equal(got.cpu().double(), m.values(rows))


@pytest.mark.parametrize("head_dim", [64, 128])
@pytest.mark.parametrize("parts", [[range(5, 10), range(5)], [[5], [0]], [[15], [3, 4], range(3), range(5, 15)],
                                   [[i] for i in (7, 6, 0, 1, 15)], [range(1, 16), [0]]])
def test_a_page_that_was_anothers_begins_past_its_first_row(gpu, head_dim, parts):
    """Rows of 1 after another's 1e30, the first of them not in the page's first row, each part a call."""
    c = Caches(head_dim=head_dim)
    s = c.kv.add_seq()
    c.kv.reserve(s, 3 * PAGE)
    for part in parts:
        c.put([(s, PAGE + p) for p in part])
        c.check()


@pytest.mark.parametrize("size", [0.01, 1.0, 100.0])
def test_the_first_row_written_again_under_others(gpu, size):
    c = Caches()
    s = c.kv.add_seq()
    c.kv.reserve(s, 2 * PAGE)
    c.put([(s, p) for p in range(2 * PAGE)])
    c.check()
    c.put([(s, 0), (s, PAGE + 1)], size)
    c.check()
    c.put([(s, PAGE), (s, 3)], 1 / size)
    c.check()
    c.put([(s, p) for p in range(PAGE)], 1e-3)  # all of them: anew
    c.check()


def test_a_row_alone_in_its_page_is_written_again(gpu):
    """Draft rows written, and written again, before anything else is in their page."""
    c = Caches()
    s = c.kv.add_seq()
    c.kv.reserve(s, PAGE)
    for size in (1e20, 1.0, 1e-20):
        c.put([(s, 0)], size)
        c.check()
        c.put([(s, p) for p in range(4)], size / 7)
        c.check()


def test_rows_rolled_back_count_no_more(gpu):
    c = Caches()
    s = c.kv.add_seq()
    c.kv.reserve(s, 2 * PAGE)
    c.put([(s, p) for p in range(PAGE + 9)], 1e10)
    c.kv.commit(s, PAGE + 9)
    c.kv.truncate(s, PAGE + 4)
    for m in c.models:
        m.cut(s, PAGE + 4)
    c.put([(s, PAGE + p) for p in range(4)])  # all that is left: anew
    c.check()
    c.put([(s, PAGE + 4)])
    c.check()
    c.kv.truncate(s, PAGE)  # its second page goes and comes back
    c.kv.reserve(s, 2 * PAGE)
    for m in c.models:
        m.cut(s, PAGE)
    c.put([(s, PAGE + 6)], 1e-10)
    c.check()


def test_copies_know_what_their_pages_hold(gpu):
    """Forked, reordered, owned and compacted pages go on with the rows they took over."""
    c = Caches(pages=16)
    kv, models = c.kv, c.models
    a = kv.add_seq()
    kv.reserve(a, PAGE + 5)
    c.put([(a, p) for p in range(PAGE + 5)])
    kv.commit(a, PAGE + 5)
    b, d = kv.fork([a, a])
    for x in (b, d):
        for m in models:
            m.become(x, a, PAGE + 5)
    for x, size in ((a, 1.0), (b, 1e-6), (d, 1e6)):  # a row of its own behind the end that was copied
        c.put([(x, PAGE + 5)], size)
        kv.commit(x, 1)
        c.check()
    kv.reorder([b], [d])
    for m in models:
        m.become(b, d, PAGE + 6)
    c.put([(b, PAGE + 6)], 1e-6)
    kv.commit(b, 1)
    c.check()
    kv.reorder([a, d], [d, a])  # ends change hands
    held = [[(k, m.blocks[k], m.rows[k]) for k in list(m.rows) if k[0] in (a, d)] for m in models]
    for m, h in zip(models, held):
        for k, values, rows in h:
            other = (d if k[0] == a else a, k[1])
            m.blocks[other], m.rows[other] = values, rows
    for x in (a, d):
        c.put([(x, PAGE + 6)], 1e-3)
        kv.commit(x, 1)
    c.check()
    kv.own(a, 0, PAGE)
    c.put([(a, 3)], 1e-3)  # one row among fifteen
    c.check()
    kv.free_seq(b)
    for m in models:
        for k in [k for k in m.rows if k[0] == b]:
            del m.rows[k]
    assert kv.compact() > 0
    c.check()
    c.put([(a, PAGE + 7), (d, PAGE + 7)], 1e-3)
    c.check()


@pytest.mark.parametrize("head_dim,seed", [(64, 1), (64, 2), (128, 3)])
def test_rows_in_any_order(gpu, head_dim, seed):
    """Rows of any position, several times, calls of all sizes; sequences freed and their pages taken by others."""
    rng = random.Random(seed)
    c = Caches(pages=6, seqs=3, head_dim=head_dim, seed=seed)
    live = []
    for _ in range(60):
        if len(live) < 2 or (rng.random() < 0.1 and len(live) < 3):
            s = c.kv.add_seq()
            c.kv.reserve(s, 2 * PAGE)
            live.append(s)
        if rng.random() < 0.1:
            s = live.pop(rng.randrange(len(live)))
            c.kv.free_seq(s)
            for m in c.models:
                m.cut(s, 0)
            continue
        rows = [(s, p) for s in live for p in range(2 * PAGE)]
        c.put(rng.sample(rows, rng.choice([1, 1, 2, 7, 30, len(rows)])), 2.0 ** rng.randint(-40, 40))
        c.check()


def test_captured_appends_keep_what_other_calls_wrote(gpu):
    """A captured append counts as made when it is captured: calls after it keep its rows, replays theirs."""
    c = Caches(pages=4, seqs=2)
    kv = c.kv
    s = kv.add_seq()
    kv.reserve(s, PAGE)
    kv.append([(s, 2)], *[torch.zeros((2, 1, 128), device="cuda")] * 2)  # (whatever a first call sets up)
    x = [torch.randn((2, 2, 128), generator=c.g, device="cuda") for _ in range(2)]
    rows = [(s, 4), (s, 5)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kv.append(rows, *x)
    graph.replay()
    for m in c.models:
        m.append([(s, 2)], torch.zeros((2, 1, 128)))
    for m, y in zip(c.models, x):
        m.append(rows, y)
    c.check()
    c.put([(s, 0)], 0.3)
    c.check()
    for size in (3.0, 0.1):
        for y in x:
            y.copy_(torch.randn(y.shape, generator=c.g, device="cuda") * size)
        graph.replay()
        for m, y in zip(c.models, x):
            m.append(rows, y)
        c.check()


@pytest.mark.parametrize("head_dim", [64, 128])
def test_layers_written_one_after_another(gpu, head_dim):
    """A prompt in parts, all of them in one layer and then in the next; then calls of all layers, which hold different rows."""
    c = Caches(n_layer=3, head_dim=head_dim)
    kv = c.kv
    s = kv.add_seq()
    kv.reserve(s, 2 * PAGE)

    def put(layer, rows, size=1.0):
        x = [torch.randn((len(rows), kv.opts.n_embd), generator=c.g, device="cuda") * size for _ in range(2)]
        kv.append([(s, p) for p in rows], *x, layer=layer)
        for m, y in zip(layers[layer], x):
            m.append([(s, p) for p in rows], y[None])

    def check():
        for layer, models in layers.items():
            rows = sorted((q, page * PAGE + x) for (q, page), there in models[0].rows.items() for x in there)
            for got, m in zip(kv.gather_values(rows, layer=layer) if rows else (), models):
                assert torch.equal(got.cpu().double(), m.values(rows)[0]), layer

    layers = {layer: [Blocks(1, 2, head_dim) for _ in range(2)] for layer in range(3)}
    for layer in (0, 2):
        for rows in (range(3, 9), range(3), range(9, 21)):
            put(layer, list(rows))
            check()
    put(0, [21], 1e-5)
    for rows in ([22], [5], list(range(PAGE)), list(range(4, 24)), list(range(2 * PAGE))):  # all layers
        x = [torch.randn((3, len(rows), kv.opts.n_embd), generator=c.g, device="cuda") * 0.1 for _ in range(2)]
        kv.append([(s, p) for p in rows], *x)
        for layer, models in layers.items():
            for m, y in zip(models, x):
                m.append([(s, p) for p in rows], y[layer:layer + 1])
        check()
    kv.commit(s, PAGE + 7)
    (f,) = kv.fork([s])
    for layer, models in layers.items():
        for m in models:
            m.become(f, s, PAGE + 7)
    check()
    x = [torch.randn((3, 1, kv.opts.n_embd), generator=c.g, device="cuda") * 0.1 for _ in range(2)]
    kv.append([(f, PAGE + 6)], *x)
    for layer, models in layers.items():
        for m, y in zip(models, x):
            m.append([(f, PAGE + 6)], y[layer:layer + 1])
    check()


@pytest.mark.parametrize("head_dim,n_head", [(64, 3), (128, 1), (128, 8)])
@pytest.mark.parametrize("rows", [1, 4, 6, 13, 15])
def test_copies_leave_what_lies_behind_the_end(gpu, head_dim, n_head, rows):
    """Of a page that a sequence ends in the rows before the end go over (of V with the rest of the word of four that
    holds the last), and its scales; nothing else of the pool changes."""
    kv = _kv(2, n_head, head_dim, pages=6)
    at, _, size = kv.pools()

    class Pool:
        __cuda_array_interface__ = dict(shape=(size,), typestr="|u1", data=(at, False), version=2)

    pool = torch.as_tensor(Pool(), device="cuda")
    pool.copy_(torch.randint(0, 256, pool.shape, device="cuda", dtype=torch.uint8))
    s = kv.add_seq()
    kv.reserve(s, 2 * PAGE)
    kv.commit(s, PAGE + rows)
    before = pool.clone().view(2, 6, -1)
    (f,) = kv.fork([s])
    after = pool.view(2, 6, -1)
    src, dst = kv.block_table(s)[1], kv.block_table(f)[1]
    block = PAGE * head_dim
    copied = torch.zeros((before.shape[2],), dtype=torch.bool)
    maybe = copied.clone()
    for head in range(n_head):
        for d in range(head_dim):
            for p in range(PAGE):
                k = head * 2 * block + d // 64 * 1024 + d % 64 // 16 * 256 + p * 16 + d % 16
                v = (head * 2 + 1) * block + d // 64 * 1024 + p // 4 * 256 + d % 16 * 16 + d % 64 // 16 * 4 + p % 4
                copied[k] = copied[v] = p < rows
                maybe[v] = p < (rows + 3) // 4 * 4
    scales = 2 * n_head * block
    copied[scales:scales + 8 * n_head] = True
    maybe[scales:scales + (8 * n_head + 15) // 16 * 16] = True  # (and what fills the unit of the last)
    copied, maybe = copied.cuda(), maybe.cuda()
    assert torch.equal(after[:, dst][:, copied], before[:, src][:, copied])
    left = ~(copied | maybe)
    assert torch.equal(after[:, dst][:, left], before[:, dst][:, left])
    others = [p for p in range(6) if p != dst]
    assert torch.equal(after[:, others], before[:, others])


@pytest.mark.parametrize("length", [5, 16, 21, 47])
def test_rows_brought_into_the_pool_by_other_means(gpu, length):
    """A pool's bytes from another cache of the same tables: appends go on behind the committed rows."""
    a, b = Caches(), Caches()
    sa, sb = a.kv.add_seq(), b.kv.add_seq()
    a.kv.reserve(sa, 4 * PAGE)
    a.put([(sa, p) for p in range(length)], 2.0)
    a.kv.commit(sa, length)
    b.kv.reserve(sb, 4 * PAGE)
    b.kv.commit(sb, length)
    assert a.kv.block_table(sa) == b.kv.block_table(sb)

    def pool(kv):
        at, _, n = kv.pools()

        class Pool:
            __cuda_array_interface__ = dict(shape=(n,), typestr="|u1", data=(at, False), version=2)

        return torch.as_tensor(Pool(), device="cuda")

    pool(b.kv).copy_(pool(a.kv))
    b.models = a.models
    for i, size in enumerate((1e-4, 1.0, 300.0)):
        b.put([(sb, length + i)], size)
        b.kv.commit(sb, 1)
        b.check()
    (f,) = b.kv.fork([sb])
    for m in b.models:
        m.become(f, sb, length + 3)
    b.put([(f, length + 3), (f, length + 4)], 1e-4)
    b.check()
