"""Verification of drafted tokens against a target model's probabilities
(``ni_verify_drafts``), beside the verify driver ``drivers.Spec``, whose
``commit`` takes the accepted numbers."""
from __future__ import annotations

import functools

from . import _abi
from .batch import KvError, _on, _stream_now, _torch
from .rotation import dtype_code


def _fits(t, dtype, shape, device) -> bool:
    """The quick form of the checks below for a contiguous tensor."""
    return t.dtype is dtype and t.shape == shape and t.is_contiguous() and t.get_device() == device


def _need(t, name, dtype, shape, strided=False):
    torch = _torch()
    if not isinstance(t, torch.Tensor) or t.dtype != dtype:
        raise TypeError(f"{name} must be a {dtype} tensor")
    dense = t.numel() == 0 or t.shape[-1] == 1 or t.stride(-1) == 1
    if tuple(t.shape) != shape or not dense or not (strided or t.is_contiguous()):
        raise ValueError(f"{name} must be a {'' if strided else 'contiguous '}{list(shape)} tensor with unit stride, "
                         f"not {list(t.shape)}")


def verify_drafts(target, drafted, accept_u, sample_u, draft=None, n_drafts=None, accepted=None, tokens=None,
                  stream=None):
    """Accept the drafted tokens that the target's probabilities allow and
    draw the one after them, so that the tokens that come out are distributed
    as the target's own (speculative sampling).

    ``target`` [B, K+1, V] holds the target's probabilities after each prefix
    of the drafts, ``draft`` [B, K, V] the drafter's (None: it was certain), in
    float32, float16 or bfloat16; ``drafted`` [B, K] int32 the tokens,
    ``accept_u`` [B, K] and ``sample_u`` [B] float32 uniform numbers in [0, 1),
    ``n_drafts`` [B] int32 how many drafts each sequence has (None: K).  All
    are CUDA tensors; rows of V are dense.  Draft i stays while ``accept_u *
    draft < target`` at its token; the next token is drawn from ``max(target -
    draft, 0)`` at the first that does not (from the target's row after the
    last), the first entry at which the sum passes ``sample_u`` times the whole.

    Returns ``(accepted [B], tokens [B, K+1])`` int32 (allocated if not
    given; they share no memory with the inputs or each other): the accepted drafts, the
    drawn token, then -1."""
    torch = _torch()
    if not isinstance(target, torch.Tensor) or target.dim() != 3 or dtype_code(target.dtype) is None:
        raise TypeError("target must be a float32, float16 or bfloat16 tensor [sequences, drafts + 1, vocabulary]")
    b, k, v = target.shape[0], target.shape[1] - 1, target.shape[2]
    dtype, device = target.dtype, target.get_device()
    s = _stream_now(device, stream) if target.is_cuda else None
    Tensor, i32 = torch.Tensor, torch.int32
    if (s is not None and k > 0 and v > 0 and target.is_contiguous() and type(drafted) is Tensor
            and type(accept_u) is Tensor and type(sample_u) is Tensor and type(accepted) is Tensor
            and type(tokens) is Tensor
            and (draft is None or type(draft) is Tensor and _fits(draft, dtype, (b, k, v), device))
            and (n_drafts is None or type(n_drafts) is Tensor and _fits(n_drafts, i32, (b,), device))
            and _fits(drafted, i32, (b, k), device) and _fits(accept_u, torch.float32, (b, k), device)
            and _fits(sample_u, torch.float32, (b,), device) and _fits(accepted, i32, (b,), device)
            and _fits(tokens, i32, (b, k + 1), device)):
        _call(torch, target, drafted, accept_u, sample_u, draft, n_drafts, accepted, tokens, b, k, v, s,
              ((k + 1) * v, v), (k * v, v), k, k, k + 1)
        return accepted, tokens
    if k < 0 or v == 0:
        raise ValueError(f"target is {list(target.shape)}: needs [sequences, drafts + 1, vocabulary]")
    _need(target, "target", target.dtype, (b, k + 1, v), strided=True)
    if draft is not None:
        _need(draft, "draft", target.dtype, (b, k, v), strided=True)
    _need(drafted, "drafted", torch.int32, (b, k), strided=True)
    _need(accept_u, "accept_u", torch.float32, (b, k), strided=True)
    _need(sample_u, "sample_u", torch.float32, (b,))
    if n_drafts is not None:
        _need(n_drafts, "n_drafts", torch.int32, (b,))
    if accepted is not None:
        _need(accepted, "accepted", torch.int32, (b,))
    if tokens is not None:
        _need(tokens, "tokens", torch.int32, (b, k + 1), strided=True)
    if not target.is_cuda:
        raise TypeError("target must be a CUDA tensor")
    for name, t in (("draft", draft), ("drafted", drafted), ("accept_u", accept_u), ("sample_u", sample_u),
                    ("n_drafts", n_drafts), ("accepted", accepted), ("tokens", tokens)):
        if t is not None and t.device != target.device:
            raise ValueError(f"{name} is on {t.device}, target on {target.device}")
    with _on(target.get_device(), stream) as s:
        if accepted is None:
            accepted = torch.empty((b,), dtype=torch.int32, device=target.device)
        if tokens is None:
            tokens = torch.empty((b, k + 1), dtype=torch.int32, device=target.device)
        _call(torch, target, drafted, accept_u, sample_u, draft, n_drafts, accepted, tokens, b, k, v, s,
              target.stride(), (0, 0) if draft is None else draft.stride(), drafted.stride(0), accept_u.stride(0),
              tokens.stride(0))
    return accepted, tokens


@functools.lru_cache(maxsize=64)
def _workspace(b, v) -> int:
    return _abi.lib().ni_verify_workspace(b, v)


def _call(torch, target, drafted, accept_u, sample_u, draft, n_drafts, accepted, tokens, b, k, v, s, target_strides,
          draft_strides, drafted_stride, accept_stride, tokens_stride):
    L = _abi.lib()
    need = _workspace(b, v)
    # From torch's allocator: of this stream, and of the graph where one is captured.
    work = torch.empty((need,), dtype=torch.uint8, device=target.device)
    rc = L.ni_verify_drafts(dtype_code(target.dtype), target.data_ptr(), target_strides[0], target_strides[1],
                            None if draft is None or k == 0 else draft.data_ptr(), draft_strides[0], draft_strides[1],
                            drafted.data_ptr() if k else None, drafted_stride,
                            None if n_drafts is None else n_drafts.data_ptr(), accept_u.data_ptr() if k else None,
                            accept_stride, sample_u.data_ptr(), b, k, v, accepted.data_ptr(), tokens.data_ptr(),
                            tokens_stride, work.data_ptr(), need, s)
    if rc != 0:
        raise KvError(rc, (L.ni_kv_last_error(None) or b"").decode())
