"""Beam search's selection over beams and vocabulary (``ni_beam_select``).  The
cache follows the selected beams by :meth:`~nanoinfer_amd.PagedKv.reorder`."""
from __future__ import annotations

import functools

from . import _abi
from .batch import KvError, _on, _stream_now, _torch
from .rotation import dtype_code
from .verify import _fits, _need


def beam_select(logits, scores, k=None, finished=None, pad_token=0, history=None, out_scores=None, parents=None,
                tokens=None, out_history=None, stream=None):
    """The ``k`` best continuations (default: as many as beams) of each search,
    best first.

    ``logits`` [B, W, V] of B searches with W beams, float32, float16 or
    bfloat16, rows of V dense; ``scores`` [B, W] float32, the beams' totals so far
    (-inf: a beam that has not begun); ``finished`` [B, W] int32: beams that
    are (nonzero) go on with ``pad_token`` alone, their score unchanged;
    ``history`` [B, W, T] int32: the beams' tokens so far.  All are CUDA tensors.
    A continuation's total is ``score + log_softmax(logits)`` of its token;
    equal ones go to the lowest (beam, token).

    Returns ``(scores [B, k] float32, parents [B, k], tokens [B, k])`` (int32) and,
    where ``history`` is given, the answers' histories [B, k, T + 1], allocated if
    not given (``out_scores``, ``parents``, ``tokens``, ``out_history``; they
    share no memory with the inputs).  Where there are fewer continuations:
    -inf, -1 and -1."""
    torch = _torch()
    if not isinstance(logits, torch.Tensor) or logits.dim() != 3 or dtype_code(logits.dtype) is None:
        raise TypeError("logits must be a float32, float16 or bfloat16 tensor [searches, beams, vocabulary]")
    b, w, v = logits.shape
    given, k = k, w if k is None else int(k)
    if given is not None and k != given:
        raise ValueError(f"k {given} is no whole number")
    if not 0 <= k <= 0xffffffff or v == 0 or w == 0:
        raise ValueError(f"logits are {list(logits.shape)}, k {k}: needs [searches, beams, vocabulary] and k in 0..2^32-1")
    if not 0 <= pad_token <= 0xffffffff:
        raise ValueError("pad_token must be in 0..2^32-1")
    device, f32, i32 = logits.get_device(), torch.float32, torch.int32
    t = 0
    if history is not None:
        if not isinstance(history, torch.Tensor) or history.dim() != 3:
            raise TypeError("history must be an int32 tensor [searches, beams, tokens]")
        t = history.shape[2]
    elif out_history is not None:
        raise ValueError("out_history without history")
    Tensor = torch.Tensor
    s = _stream_now(device, stream) if logits.is_cuda else None
    if (s is not None and logits.stride(2) == 1 and type(scores) is Tensor and _fits(scores, f32, (b, w), device)
            and type(out_scores) is Tensor and _fits(out_scores, f32, (b, k), device)
            and type(parents) is Tensor and _fits(parents, i32, (b, k), device)
            and type(tokens) is Tensor and _fits(tokens, i32, (b, k), device)
            and (finished is None or type(finished) is Tensor and _fits(finished, i32, (b, w), device))
            and (history is None or type(history) is Tensor and _fits(history, i32, (b, w, t), device)
                 and type(out_history) is Tensor and _fits(out_history, i32, (b, k, t + 1), device))):
        _call(torch, logits, scores, finished, pad_token, history, out_scores, parents, tokens, out_history, b, w, v, k, t, s)
    else:
        _need(logits, "logits", logits.dtype, (b, w, v), strided=True)
        for name, x, dtype, shape in (("scores", scores, f32, (b, w)), ("finished", finished, i32, (b, w)),
                                      ("history", history, i32, (b, w, t)), ("out_scores", out_scores, f32, (b, k)),
                                      ("parents", parents, i32, (b, k)), ("tokens", tokens, i32, (b, k)),
                                      ("out_history", out_history, i32, (b, k, t + 1))):
            if x is not None or name == "scores":
                _need(x, name, dtype, shape)
        if not logits.is_cuda:
            raise TypeError("logits must be a CUDA tensor")
        for name, x in (("scores", scores), ("finished", finished), ("history", history), ("out_scores", out_scores),
                        ("parents", parents), ("tokens", tokens), ("out_history", out_history)):
            if x is not None and x.device != logits.device:
                raise ValueError(f"{name} is on {x.device}, logits on {logits.device}")
        with _on(device, stream) as s:
            def made(x, dtype, *shape):
                return torch.empty(shape, dtype=dtype, device=logits.device) if x is None else x

            out_scores, parents, tokens = made(out_scores, f32, b, k), made(parents, i32, b, k), made(tokens, i32, b, k)
            if history is not None:
                out_history = made(out_history, i32, b, k, t + 1)
            _call(torch, logits, scores, finished, pad_token, history, out_scores, parents, tokens, out_history, b, w, v, k,
                  t, s)
    return (out_scores, parents, tokens) if history is None else (out_scores, parents, tokens, out_history)


@functools.lru_cache(maxsize=64)
def _workspace(b, w, v) -> int:
    return _abi.lib().ni_beam_workspace(b, w, v)


def _call(torch, logits, scores, finished, pad_token, history, out_scores, parents, tokens, out_history, b, w, v, k, t, s):
    L = _abi.lib()
    need = _workspace(b, w, v)
    # From torch's allocator: of this stream, and of the graph where one is captured.
    work = torch.empty((need,), dtype=torch.uint8, device=logits.device)
    rc = L.ni_beam_select(dtype_code(logits.dtype), logits.data_ptr(), logits.stride(0), logits.stride(1),
                          scores.data_ptr(), None if finished is None else finished.data_ptr(), pad_token, b, w, v, k,
                          out_scores.data_ptr(), parents.data_ptr(), tokens.data_ptr(),
                          None if history is None or t == 0 else history.data_ptr(), t, t,
                          None if history is None else out_history.data_ptr(), t + 1, work.data_ptr(), need, s)
    if rc != 0:
        raise KvError(rc, (L.ni_kv_last_error(None) or b"").decode())
