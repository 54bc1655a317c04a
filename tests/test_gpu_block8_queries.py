"""Queries of any size over the block-scaled cache, whose keys may be of any size
too: what counts is their product."""
import math

import pytest
import torch

from test_gpu_block8 import PAGE, _kv
from test_gpu_block8_rows import FORMS

pytestmark = pytest.mark.gpu


def _filled(n_layer, n_head, head_dim, n, g):
    kv = _kv(n_layer, n_head, head_dim, pages=2 * (-(-n // PAGE)), seqs=2, ctx=n, max_rows=n)
    k, v = (torch.randn((n_layer, n, n_head * head_dim), generator=g, device="cuda") for _ in range(2))
    s = kv.add_seq()
    kv.reserve(s, n)
    rows = [(s, p) for p in range(n)]
    kv.append(rows, k, v)
    return kv, rows, k, v


@pytest.mark.parametrize("n_layer,n_head,head_dim,group,split", FORMS)
@pytest.mark.parametrize("rows_each", [1, 12, 203])
def test_small_queries_of_large_keys_and_large_of_small(gpu, n_layer, n_head, head_dim, group, split, rows_each):
    """q and the keys by powers of two that cancel: the same scores, and every bit of the outputs."""
    g = torch.Generator("cuda").manual_seed(rows_each)
    n = 203
    kv, rows, k, v = _filled(n_layer, n_head, head_dim, n, g)
    q = torch.randn((n_layer, rows_each, n_head * group * head_dim), generator=g, device="cuda") * 1.5
    at = rows[n - rows_each:]
    want = kv.prefix_attention(q, at, [(0, 0, rows_each)], split_tokens=split)
    for by in (20, -17, 60, -60, 100):
        kv.append(rows, k * 2.0 ** by, v)
        got = kv.prefix_attention(q * 2.0 ** -by, at, [(0, 0, rows_each)], split_tokens=split)
        assert torch.equal(got, want), by


@pytest.mark.parametrize("head_dim,rows_each", [(64, 1), (128, 40)])
@pytest.mark.parametrize("by", [0, 16, 40, -40])
def test_each_head_and_row_by_itself(gpu, head_dim, rows_each, by):
    """Rows and heads of one tile whose queries differ by powers of ten, zeros among them, against 64 bits."""
    g = torch.Generator("cuda").manual_seed(by + 50)
    n, n_head, group = 203, 8, 4
    kv, rows, k, v = _filled(1, n_head, head_dim, n, g)
    kv.append(rows, k * 2.0 ** by, v)
    q = torch.randn((1, rows_each, n_head * group, head_dim), generator=g, device="cuda") * 2.0 ** -by
    q *= 10.0 ** torch.randint(-6, 2, (1, rows_each, n_head * group, 1), generator=g, device="cuda")
    q[:, :, 3] = 0
    q[:, 0, 5, 1:] = 0  # (one dim)
    out = kv.prefix_attention(q.flatten(2), rows[n - rows_each:], [(0, 0, rows_each)])
    kk, vv = (x[0].double().cpu().view(n, n_head, head_dim) for x in kv.gather_values(rows))
    past = torch.arange(n)[None] <= torch.arange(n - rows_each, n)[:, None]
    for head in range(n_head * group):
        x, kh, vh = q[0, :, head].double().cpu(), kk[:, head // group], vv[:, head // group]
        w = torch.softmax((x @ kh.T / math.sqrt(head_dim)).masked_fill(~past, -math.inf), -1)
        # q's two parts, 2^-21 of a value and 2^-36 of the row's largest; head_dim + 8 sums of 2^-24; weights as two parts and
        # their sums, 2^-17
        parts = ((x.abs() + x.abs().amax(-1, keepdim=True) * 2.0 ** -15) @ kh.abs().T / math.sqrt(head_dim) * past).amax(-1, keepdim=True)
        ds = parts * (2.0 ** -21 + (head_dim + 8) * 2.0 ** -24)
        bound = (w @ vh.abs()) * (2 * ds + 2.0 ** -17)
        got = out[0, :, head * head_dim:(head + 1) * head_dim].double().cpu()
        assert bool(((got - w @ vh).abs() <= bound).all()), head
