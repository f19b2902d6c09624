"""Decayed linear attention: the memory of a policy, as sm_100a kernels.

A head of an environment carries a D x D state S; a token with query q, key k, value v does

    S <- keep decay[h] S + k' v,    out = scale q S

with keep = 0 where `resets` marks the token as the first of an episode, so that nothing of the
episode before it is seen, not even an infinity. Trajectories are time-major, as the rewards and
dones of the step_many calls: q, k, v (T, N, H, D), resets (T, N). The `dones` of step t mark the
token t + 1: `episode_starts(dones)`.

- `forward` and `backward` take whole trajectories (chunks of tokens as matrix products);
- `step` takes one token for every environment and updates the state in place (acting);
- `attend` is forward with its gradient through torch.autograd.

Tensors are float32 or bfloat16, D in {16, 32, 64, 128}, the state always float32. The reference's
policies have no memory (es.py:156-164); there is no counterpart there. The decay is a constant:
it gets no gradient. Values outside [0, 1] are not looked at: the formula then grows, or is NaN
where a negative decay is raised to a power.
"""

import ctypes
from functools import lru_cache
from math import gcd

import torch
from torch.autograd.function import once_differentiable
from torch.autograd.graph import increment_version

import rlenv_lib as _rl

WIDTHS = (16, 32, 64, 128)


def _rows(x):
    """(x, its strides without the last) with rows dense and on 16-byte boundaries; anything else is
    copied. Axes of one element get stride 0 where torch's, which is any number, would not do."""
    strides, dense = x.stride(), x.is_contiguous() and x.data_ptr() % 16 == 0
    if dense and gcd(*strides[:-1]) % 16 == 0:
        return x, strides[:-1]
    strides = tuple(0 if n == 1 else s for s, n in zip(strides, x.shape))
    if dense:
        return x, strides[:-1]
    size = x.element_size()
    if strides[-1] != 1 or x.data_ptr() % 16 or any(s * size % 16 or s < 0 for s in strides[:-1]):
        x = x.clone(memory_format=torch.contiguous_format)
        strides = x.stride()
    return x, strides[:-1]


@lru_cache(maxsize=64)
def _stride_array(*strides):
    flat = [s for triple in strides for s in triple]
    return (ctypes.c_int64 * len(flat))(*flat)


def _check(lead, decay, state, resets, grad_state, names, tokens):
    """The tokens' common shape, dtype and device, and the resets as bytes. lead: leading axes. What fits passes
    on a few comparisons; what does not is looked at again for the message."""
    first = tokens[0]
    if not isinstance(first, torch.Tensor) or not first.is_cuda or first.dtype not in _rl.FLOAT_DTYPES:
        _rl.as_floats(names[0], first)
    shape, dtype, index = first.shape, first.dtype, first.get_device()
    for name, x in zip(names[1:], tokens[1:]):
        if not isinstance(x, torch.Tensor) or x.get_device() != index or x.dtype is not dtype or x.shape != shape:
            _rl.as_floats(name, x, shape, dtype)
            _rl.one_device(index, **{name: x})
    if len(shape) != lead + 2:
        raise ValueError(f"{', '.join(names)} must have {lead + 2} axes; got shape {tuple(shape)}")
    n, h, d = shape[-3:]
    if d not in WIDTHS:
        raise ValueError(f"the heads' width must be one of {WIDTHS}; got {d}")
    if not isinstance(decay, torch.Tensor) or decay.get_device() != index or decay.dtype is not torch.float32 \
            or decay.shape != (h,):
        _rl.as_floats("decay", decay, (h,), torch.float32)
        _rl.one_device(index, decay=decay)
    for s in (state, grad_state):
        if s is not None and (not isinstance(s, torch.Tensor) or s.get_device() != index
                              or s.dtype is not torch.float32 or s.shape != (n, h, d, d)):
            name = "state" if s is state else "grad_state"
            _rl.as_floats(name, s, (n, h, d, d), torch.float32)
            _rl.one_device(index, **{name: s})
    if resets is not None:
        if not isinstance(resets, torch.Tensor) or resets.dtype not in (torch.bool, torch.uint8) \
                or resets.shape != shape[:-2]:
            raise ValueError(f"resets must be a bool or uint8 tensor of shape {tuple(shape[:-2])}")
        _rl.one_device(index, resets=resets)
        resets = resets.contiguous()
    return shape, dtype, index, resets


def _like(x):
    """A dense tensor of x's shape and type (empty_like is the quicker call, but keeps x's strides)."""
    return torch.empty_like(x) if x.is_contiguous() else x.new_empty(x.shape)


def _state_like(state, q, n, h, d):
    return _like(state) if state is not None else q.new_empty((n, h, d, d), dtype=torch.float32)


def _scale(scale, d):
    return d ** -0.5 if scale is None else float(scale)


def forward(q, k, v, decay, state=None, resets=None, scale=None):
    """(out (T, N, H, D), state after the last token (N, H, D, D)). state None starts from zero; the
    given one is not changed. scale None is D ** -0.5."""
    shape, dtype, index, resets = _check(2, decay, state, resets, None, ("q", "k", "v"), (q, k, v))
    t, n, h, d = shape
    (q, qs), (k, ks), (v, vs) = _rows(q), _rows(k), _rows(v)
    decay, state = decay.contiguous(), None if state is None else state.contiguous()
    lib, code = _rl.lib(), _rl.FLOAT_DTYPES[dtype]
    out, new = _like(q), _state_like(state, q, n, h, d)
    nbytes = lib.linear_attention_scratch_bytes(code, d, t, n, h, 0)
    tmp = _rl.scratch(nbytes, q)
    _rl.launch(index, lib.linear_attention_forward, code, d, t, n, h, q.data_ptr(), k.data_ptr(), v.data_ptr(),
               _stride_array(qs, ks, vs), decay.data_ptr(), _rl.ptr(resets), _scale(scale, d), _rl.ptr(state),
               out.data_ptr(), new.data_ptr(), _rl.ptr(tmp), nbytes)
    return out, new


def backward(grad_out, q, k, v, decay, state=None, resets=None, scale=None, grad_state=None):
    """Gradients (dq, dk, dv (T, N, H, D), dstate (N, H, D, D)) of `forward` from grad_out and, where the
    final state is used further, grad_state."""
    shape, dtype, index, resets = _check(2, decay, state, resets, grad_state, ("grad_out", "q", "k", "v"),
                                         (grad_out, q, k, v))
    t, n, h, d = shape
    (g, gs), (q, qs), (k, ks), (v, vs) = _rows(grad_out), _rows(q), _rows(k), _rows(v)
    decay = decay.contiguous()
    state, grad_state = (None if s is None else s.contiguous() for s in (state, grad_state))
    lib, code = _rl.lib(), _rl.FLOAT_DTYPES[dtype]
    dq, dk, dv, dstate = _like(q), _like(q), _like(q), _state_like(state, q, n, h, d)
    nbytes = lib.linear_attention_scratch_bytes(code, d, t, n, h, 1)
    tmp = _rl.scratch(nbytes, q)
    _rl.launch(index, lib.linear_attention_backward, code, d, t, n, h, g.data_ptr(), q.data_ptr(), k.data_ptr(),
               v.data_ptr(), _stride_array(gs, qs, ks, vs), decay.data_ptr(), _rl.ptr(resets), _scale(scale, d),
               _rl.ptr(state), _rl.ptr(grad_state), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), dstate.data_ptr(),
               _rl.ptr(tmp), nbytes)
    return dq, dk, dv, dstate


def step(q, k, v, decay, state, resets=None, scale=None):
    """One token for every environment, q, k, v (N, H, D), resets (N,): updates `state` (N, H, D, D) in
    place and returns out (N, H, D). For acting: out carries no gradient, whatever its inputs do (`attend` is the
    differentiable form), and a graph that saved `state` before its update raises in its backward pass."""
    shape, dtype, index, resets = _check(1, decay, state, resets, None, ("q", "k", "v"), (q, k, v))
    if state is None or not state.is_contiguous() or state.data_ptr() % 16:
        raise ValueError("state must be contiguous and on a 16-byte boundary: it is updated in place")
    n, h, d = shape
    (q, qs), (k, ks), (v, vs) = _rows(q), _rows(k), _rows(v)
    decay, out = decay.contiguous(), _like(q)
    _rl.launch(index, _rl.lib().linear_attention_step, _rl.FLOAT_DTYPES[dtype], d, n, h, q.data_ptr(), k.data_ptr(),
               v.data_ptr(), _stride_array(qs, ks, vs), decay.data_ptr(), _rl.ptr(resets),
               _scale(scale, d), state.data_ptr(), out.data_ptr())
    increment_version(state)
    return out


def episode_starts(dones, first=False):
    """resets (T, N) for a trajectory's tokens from the dones (T, N) of its steps: token 0 is marked as
    `first` says (a bool, or (N,) flags), token t + 1 where step t ended an episode."""
    starts = torch.empty_like(dones, dtype=torch.bool)
    if starts.shape[0]:
        starts[0] = first
        starts[1:] = dones[:-1]
    return starts


class _Attend(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, decay, state, resets, scale):
        ctx.save_for_backward(q, k, v, decay, state, resets)
        ctx.scale = scale
        return forward(q, k, v, decay, state, resets, scale)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_out, grad_state):
        q, k, v, decay, state, resets = ctx.saved_tensors
        dq, dk, dv, dstate = backward(grad_out.contiguous(), q, k, v, decay, state, resets, ctx.scale, grad_state)
        return dq, dk, dv, None, dstate if state is not None else None, None, None


def attend(q, k, v, decay, state=None, resets=None, scale=None):
    """`forward` as a differentiable operation of q, k, v and state."""
    return _Attend.apply(q, k, v, decay, state, resets, scale)
