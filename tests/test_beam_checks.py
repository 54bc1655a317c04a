"""Refusals of beam selection, without a GPU: every check comes before anything
touches the device."""
import pytest

from nanoinfer_amd import _abi

P = 1 << 20  # an address that nothing reads


def _select(b=1, w=2, v=100, k=2, history=P, history_stride=8, n_history=5, out_history=P << 3, out_history_stride=8):
    L = _abi.lib()
    need = L.ni_beam_workspace(b, w, v)
    rc = L.ni_beam_select(_abi.NI_F32, P << 20, w * v, v, P << 11, None, 0, b, w, v, k, P << 12, P << 13, P << 14, history,
                          history_stride, n_history, out_history, out_history_stride, P << 15, need, None)
    return rc, L.ni_kv_last_error(None).decode()


@pytest.mark.parametrize("stride", [1 << 62, (1 << 62) + 1, 1 << 60, (1 << 63) - 1])
@pytest.mark.parametrize("name", ["history", "out_history"])
def test_histories_that_pass_the_address_space(name, stride):
    """Strides whose rows lie further apart than memory reaches: the extents that overlaps are sought in would wrap."""
    for b, w, k in ((1, 2, 2), (2, 4, 4), (1, 5, 3)):
        rc, text = _select(b=b, w=w, k=k, **{name + "_stride": stride})
        assert rc == _abi.NI_ERR_BAD_ARG and text == f"{name}'s strides are too large", text


def test_histories_that_share_memory():
    for kw, text in ((dict(out_history=P), "out_history may not share memory with history"),
                     (dict(history=P, history_stride=8, out_history=P + 4 * 12), "out_history may not share memory with history"),
                     (dict(history=P, history_stride=1 << 20, out_history=P + (1 << 22)), "out_history may not share memory")):
        rc, got = _select(**kw)
        assert rc == _abi.NI_ERR_BAD_ARG and text in got, got
