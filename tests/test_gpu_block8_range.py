"""The block-scaled cache at the ends of f32's range: what is stored is finite,
and means of finite values are finite."""
import math

import pytest
import torch

from test_gpu_block8 import PAGE, _kv

pytestmark = pytest.mark.gpu
TOP = torch.finfo(torch.float32).max


@pytest.mark.parametrize("head_dim", [64, 128])
@pytest.mark.parametrize("each", [1, 16])
def test_the_largest_values_are_stored_finite(gpu, head_dim, each):
    """Half a step is 2^-4 of a value, the largest of f32 among them; an infinity is stored as the largest value there is."""
    kv = _kv(1, 1, head_dim)
    s = kv.add_seq()
    kv.reserve(s, 2 * PAGE)
    x = torch.full((1, 2 * PAGE, head_dim), TOP, device="cuda")
    x *= torch.linspace(0.4, 1, 2 * PAGE * head_dim, device="cuda").view(x.shape)
    x[:, ::3] *= -1
    x[0, PAGE + 3, 7] = math.inf
    minus = -x
    for at in range(0, 2 * PAGE, each):
        kv.append([(s, p) for p in range(at, at + each)], x[:, at:at + each], minus[:, at:at + each])
    k, v = kv.gather_values([(s, p) for p in range(2 * PAGE)])
    assert torch.equal(k, -v) and bool(torch.isfinite(k).all())
    assert float(k[0, PAGE + 3, 7]) >= float(x[0, :PAGE + 3].abs().max()) * 0.9  # (the block's largest value by then)
    k[0, PAGE + 3, 7] = x[0, PAGE + 3, 7] = 0
    assert bool(((k.double() - x.double()).abs() <= x.double().abs() * 2.0 ** -4).all())


@pytest.mark.parametrize("n_layer,n_head,head_dim,rows_each,split", [(1, 1, 64, 1, 0), (1, 2, 128, 3, 0), (1, 2, 64, 16, 64),
                                                                    (12, 16, 64, 40, 0), (4, 32, 128, 40, 0)])
@pytest.mark.parametrize("size", [1e38, 1e35, 1e-30, 1e-36])
def test_means_of_large_and_small_values(gpu, n_layer, n_head, head_dim, rows_each, split, size):
    """Every key alike: the mean of the values, which neither passes f32's range on the way nor falls out of it."""
    g = torch.Generator("cuda").manual_seed(5)
    n, c = 500, n_head * head_dim
    kv = _kv(n_layer, n_head, head_dim, pages=40)
    s = kv.add_seq()
    kv.reserve(s, n)
    v = (0.5 + torch.rand((n_layer, n, c), generator=g, device="cuda")) * size
    kv.append([(s, p) for p in range(n)], torch.ones_like(v), v)
    q = torch.randn((n_layer, rows_each, c), generator=g, device="cuda")
    out = kv.attention(q, [(s, n - rows_each + i) for i in range(rows_each)], split_tokens=split)
    _, vv = kv.gather_values([(s, p) for p in range(n)])
    vv = vv.double()
    want = torch.stack([vv[:, :n - rows_each + i + 1].mean(1) for i in range(rows_each)], 1)
    # equal weights of two f16 parts (2^-21), sums of 500 in f32, a division; below 2^-126 f32 has steps of 2^-149
    assert bool(((out.double() - want).abs() <= want * (2.0 ** -20 + 500 * 2.0 ** -24) + 2.0 ** -148).all())


def test_large_values_beside_small(gpu):
    """Values of 1e37 and of 1e-20 in a row that attends to either."""
    g = torch.Generator("cuda").manual_seed(6)
    n, d = 20 * PAGE, 64
    for first in (True, False):
        kv = _kv(1, 1, d, pages=20)
        s = kv.add_seq()
        kv.reserve(s, n)
        size = torch.full((n, 1), 1e-20, device="cuda")
        size[(slice(0, n // 2) if first else slice(n // 2, n))] = 1e37
        v = (0.5 + torch.rand((1, n, d), generator=g, device="cuda")) * size
        kv.append([(s, p) for p in range(n)], torch.ones_like(v), v)
        out = kv.attention(torch.ones((1, 1, d), device="cuda"), [(s, n - 1)])
        _, vv = kv.gather_values([(s, p) for p in range(n)])
        want = vv[0].double().mean(0)
        assert bool(((out[0, 0].double() - want).abs() <= want * (2.0 ** -20 + 500 * 2.0 ** -24)).all())
