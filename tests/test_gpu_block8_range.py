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
