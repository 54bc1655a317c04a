"""Numbers that the calls of shared pages and beam selection take, without a GPU."""
import pytest
import torch

import nanoinfer_amd as na
from test_page_sharing import PAGE, _grow, _kv


@pytest.mark.parametrize("bad", [1 << 32, -1, (1 << 32) + 1, 1 << 40])
def test_numbers_past_32_bits_are_refused(bad):
    kv = _kv()
    s = kv.add_seq()
    _grow(kv, s, PAGE)
    (f,) = kv.fork([s])
    for call in (lambda: kv.page_refs(bad), lambda: kv.own(f, bad), lambda: kv.own(f, 0, bad), lambda: kv.own(bad, 0, 0)):
        with pytest.raises(ValueError):
            call()
    for call in (lambda: kv.page_refs(0.0), lambda: kv.own(f, 0.0), lambda: kv.own(f, 0, 1.0), lambda: kv.own("0")):
        with pytest.raises(TypeError):
            call()
    assert kv.block_table(f) == kv.block_table(s)


@pytest.mark.parametrize("k", [2.7, (1 << 32) + 1, 1 << 40, -1])
def test_numbers_of_answers(k):
    logits, scores = torch.zeros((1, 3, 40)), torch.zeros((1, 3))
    with pytest.raises(ValueError):
        na.beam_select(logits, scores, k)
    with pytest.raises(TypeError, match="CUDA"):  # a whole number goes on to the next check
        na.beam_select(logits, scores, 2.0)
