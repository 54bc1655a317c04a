"""Steps on the block-scaled cache that cannot be made: nothing of them is."""
import pytest
import torch

import nanoinfer_amd as na
from test_gpu_block8 import PAGE, _kv

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("why", ["plan", "partials"])
def test_a_step_that_cannot_be_captured_appends_nothing(gpu, why):
    """The attention's plan does not travel with the launch, or its partials are not there: the append is not captured either."""
    g = torch.Generator("cuda").manual_seed(1)
    n, seqs = (2500, 64) if why == "plan" else (4000, 1)
    kv = _kv(1, 1, 64, pages=seqs * (n // PAGE + 2), seqs=seqs, ctx=n + 32, max_rows=64)
    work = []
    for _ in range(seqs):
        s = kv.add_seq()
        kv.reserve(s, n + 1)
        kv.commit(s, n)
        work.append((s, 1, 1))
    rows = [(s, n) for s, _, _ in work]
    held = [torch.randn((1, seqs, 64), generator=g, device="cuda") for _ in range(2)]
    kv.append(rows, *held)  # (a draft, not committed)
    want = [x.clone() for x in kv.gather_values(rows)]
    q, k, v = (torch.randn((1, seqs, 64), generator=g, device="cuda") * 3 for _ in range(3))
    out, other = torch.zeros_like(q), torch.zeros(4, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        other += 1
        with pytest.raises(na.KvError) as e:
            kv.step(work, q, k, v, out=out, split_tokens=0 if why == "plan" else 16)
    assert why in str(e.value)
    for turn in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert other.tolist() == [turn + 1.0] * 4
        assert all(torch.equal(x, y) for x, y in zip(kv.gather_values(rows), want))
    assert [kv.seq_len(s) for s, _, _ in work] == [n] * seqs
    kv.step(work, q, k, v, out=out)  # outside it can be made
    assert kv.seq_len(0) == n + 1 and bool(torch.isfinite(out).all()) and bool((out != 0).any())


def test_a_step_too_large_appends_nothing(gpu):
    """More (partition, layer, head) items than a call takes."""
    g = torch.Generator("cuda").manual_seed(2)
    n, n_layer, n_head = 2048 * PAGE, 64, 64
    kv = _kv(n_layer, n_head, 64, pages=n // PAGE + 1, seqs=1, ctx=n + PAGE, max_rows=1)
    s = kv.add_seq()
    kv.reserve(s, n + 1)
    kv.commit(s, n)
    held = [torch.randn((n_layer, 1, n_head * 64), generator=g, device="cuda") for _ in range(2)]
    kv.append([(s, n)], *held)
    want = [x.clone() for x in kv.gather_values([(s, n)])]
    q, k, v = (torch.randn((n_layer, 1, n_head * 64), generator=g, device="cuda") * 3 for _ in range(3))
    with pytest.raises(na.KvError) as e:
        kv.step([(s, 1, 1)], q, k, v, split_tokens=16)
    assert "too large" in str(e.value) and kv.seq_len(s) == n
    assert all(torch.equal(x, y) for x, y in zip(kv.gather_values([(s, n)]), want))
    kv.step([(s, 1, 1)], q, k, v)
    assert kv.seq_len(s) == n + 1
    assert not torch.equal(kv.gather_values([(s, n)])[0], want[0])
