"""Scores of actions from a policy's logits, as sm_100a kernels: the log-probability of each token's chosen action, the
entropy of its distribution and its best alternatives, and their gradient.

    normalizer = log sum exp(logits),   log_prob = logits[action] - normalizer,   entropy = - sum p log p

logits (..., A) are float32 or bfloat16, actions (...) integers, `allowed` (..., A) bool says which actions there are in
a token (None: all; what stands in the others' places is not looked at). Results are float32. Everything is formed in
one reading of the logits; the gradient is one reading and one writing.

- A negative action marks a token without one (padding): its log_prob is 0 and has no gradient. One of A or above gives
  NaN, and a gradient that is NaN throughout.
- A token that allows nothing has normalizer and log_prob -infinity, entropy 0 and no gradient, whatever its action; an
  action that is not allowed, or whose logit is -infinity, has log_prob -infinity and no gradient of its own place.
- A NaN or +infinity among a token's allowed logits makes its results NaN, and its gradient throughout.
- What a token's logits have in common changes no result but the normalizer, a float32: `remainder` is what its rounding
  leaves.

The reference's policies act greedily and have no gradient (es.py:156-175); there is no counterpart there.
"""

from typing import NamedTuple

import torch
from torch.autograd.function import once_differentiable

import rlenv_lib as _rl

MOST_ALTERNATIVES = 32


class _Scores(NamedTuple):
    log_prob: torch.Tensor
    entropy: torch.Tensor
    normalizer: torch.Tensor
    top_log_probs: torch.Tensor | None = None
    top_actions: torch.Tensor | None = None


class Scores(_Scores):
    """Of logits (..., A): log_prob, entropy and normalizer (...) float32; of the alternatives asked for, best first
    (ties: the lower action), top_log_probs (..., n) float32 and top_actions (..., n) int64, None without. `remainder`
    (...) float32, no item of the tuple, is what the normalizer's rounding has left, None unless asked for."""
    remainder = None


def _check(logits, actions, allowed):
    """(rows, A, the type's code, the actions' code, the device's index)"""
    if not isinstance(logits, torch.Tensor) or not logits.is_cuda or logits.dtype not in _rl.FLOAT_DTYPES:
        _rl.as_floats("logits", logits)
    shape, index = logits.shape, logits.get_device()
    if not shape or shape[-1] == 0:
        raise ValueError(f"logits must be (..., A) with A of at least 1; got shape {tuple(shape)}")
    if not isinstance(actions, torch.Tensor) or actions.dtype not in _ACTIONS or actions.shape != shape[:-1]:
        raise ValueError(f"actions must be an int64, int32 or uint8 tensor of shape {tuple(shape[:-1])}")
    if allowed is not None and (not isinstance(allowed, torch.Tensor) or allowed.dtype not in (torch.bool, torch.uint8)
                                or allowed.shape != shape):
        raise ValueError(f"allowed must be a bool or uint8 tensor of shape {tuple(shape)}")
    if actions.get_device() != index or (allowed is not None and allowed.get_device() != index):
        _rl.one_device(index, actions=actions, allowed=allowed)
    return shape[:-1].numel(), shape[-1], _rl.FLOAT_DTYPES[logits.dtype], _ACTIONS[actions.dtype], index


_MANY, _MANY_LOGITS = 1 << 26, 1 << 40  # rows and logits that the library no longer takes in one launch


def _launches(m, v):
    """(first row, rows) of each launch that a call of m rows of v takes."""
    most = min(_MANY - 16, (_MANY_LOGITS - 1) // v & ~15)
    return ((0, m),) if m <= most else tuple((at, min(most, m - at)) for at in range(0, m, most))


def _in_launches(index, entry, code, m, v, args, rows):
    """entry(code, m, v, *args) in several launches; rows: of each argument the bytes from row to row, 0 where it is no
    address of rows."""
    for at, n in _launches(m, v):
        _rl.launch(index, entry, code, n, v, *(x + at * step if x else x for x, step in zip(args, rows)))


_ACTIONS = {torch.int64: _rl.I64, torch.int32: _rl.I32, torch.uint8: _rl.U8}


def forward(logits, actions, allowed=None, alternatives=0, remainder=False):
    """Scores of the actions, and of the `alternatives` (up to 32) best ones; with `remainder`, the normalizer's, for
    `backward`."""
    m, v, code, action_code, index = _check(logits, actions, allowed)
    if not 0 <= alternatives <= min(v, MOST_ALTERNATIVES):
        raise ValueError(f"alternatives must be from 0 to {min(v, MOST_ALTERNATIVES)}; got {alternatives}")
    logits, stride = _rl.as_rows(logits)
    allowed, allowed_stride = (None, 0) if allowed is None else _rl.as_rows(allowed)
    actions = actions.contiguous()
    log_prob = _rl.empty_lead(logits, torch.float32)
    entropy, normalizer = torch.empty_like(log_prob), torch.empty_like(log_prob)
    rest = torch.empty_like(log_prob) if remainder else None
    top = best = None
    if alternatives:
        top, best = _rl.empty_rows(logits, alternatives, torch.float32), _rl.empty_rows(logits, alternatives, torch.int64)
    entry = _rl.lib().log_probs_forward_remainder
    args = (logits.data_ptr(), stride, actions.data_ptr(), action_code, _rl.ptr(allowed), allowed_stride, log_prob.data_ptr(),
            entropy.data_ptr(), normalizer.data_ptr(), _rl.ptr(rest), alternatives, _rl.ptr(best), _rl.ptr(top))
    if m < _MANY and m * v < _MANY_LOGITS:
        _rl.launch(index, entry, code, m, v, *args)
    else:
        _in_launches(index, entry, code, m, v, args,
                     (stride * logits.element_size(), 0, actions.element_size(), 0, allowed_stride, 0, 4, 4, 4, 4, 0,
                      8 * alternatives, 4 * alternatives))
    scores = Scores(log_prob, entropy, normalizer, top, best)
    if remainder:
        scores.remainder = rest
    return scores


def backward(grad_log_prob, grad_entropy, logits, actions, normalizer, entropy, allowed=None, remainder=None):
    """The gradient (..., A) of the logits from those of log_prob and entropy (either may be None), with `forward`'s
    normalizer and entropy. With its remainder a token whose logits lie far from zero has as precise a gradient as
    another; without, its probabilities are off by a factor of up to e^(2^-24 |normalizer|)."""
    m, v, code, action_code, index = _check(logits, actions, allowed)
    lead = logits.shape[:-1]
    rows = []
    for name, x in (("grad_log_prob", grad_log_prob), ("grad_entropy", grad_entropy), ("normalizer", normalizer),
                    ("entropy", entropy), ("remainder", remainder)):
        if x is None and name not in ("normalizer", "entropy"):
            rows.append(None)
            continue
        if not isinstance(x, torch.Tensor) or x.get_device() != index or x.dtype is not torch.float32 or x.shape != lead:
            _rl.as_floats(name, x, lead, torch.float32)
            _rl.one_device(index, **{name: x})
        rows.append(x.contiguous())
    grad_log_prob, grad_entropy, normalizer, entropy, remainder = rows
    logits, stride = _rl.as_rows(logits)
    allowed, allowed_stride = (None, 0) if allowed is None else _rl.as_rows(allowed)
    actions, grad = actions.contiguous(), _rl.empty_rows(logits, v, logits.dtype)
    entry, size = _rl.lib().log_probs_backward_remainder, logits.element_size()
    args = (_rl.ptr(grad_log_prob), _rl.ptr(grad_entropy), logits.data_ptr(), stride, actions.data_ptr(), action_code,
            normalizer.data_ptr(), _rl.ptr(remainder), entropy.data_ptr(), _rl.ptr(allowed), allowed_stride, grad.data_ptr())
    if m < _MANY and m * v < _MANY_LOGITS:
        _rl.launch(index, entry, code, m, v, *args)
    else:
        _in_launches(index, entry, code, m, v, args,
                     (4, 4, stride * size, 0, actions.element_size(), 0, 4, 4, 4, allowed_stride, 0, v * size))
    return grad


class _Apply(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, actions, allowed):
        scores = forward(logits, actions, allowed, remainder=True)
        ctx.save_for_backward(logits, actions, allowed, scores.normalizer, scores.entropy, scores.remainder)
        ctx.set_materialize_grads(False)
        return scores.log_prob, scores.entropy

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_log_prob, grad_entropy):
        logits, actions, allowed, normalizer, entropy, remainder = ctx.saved_tensors
        grad = backward(grad_log_prob, grad_entropy, logits, actions, normalizer, entropy, allowed, remainder)
        return grad, None, None


def apply(logits, actions, allowed=None):
    """(log_prob, entropy) as differentiable operations of the logits."""
    return _Apply.apply(logits, actions, allowed)
