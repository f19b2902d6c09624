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

import torch

import rlenv_lib as _rl

WIDTHS = (16, 32, 64, 128)


def _rows(x):
    """(x, its strides without the last) with rows dense and on 16-byte boundaries; anything else is
    copied. Axes of one element have stride 0."""
    size = x.element_size()
    strides = [0 if n == 1 else s for s, n in zip(x.stride(), x.shape)]
    if strides[-1] != 1 or x.data_ptr() % 16 or any(s * size % 16 or s < 0 for s in strides[:-1]):
        x = x.contiguous() if not x.is_contiguous() else x.clone(memory_format=torch.contiguous_format)
        strides = [0 if n == 1 else s for s, n in zip(x.stride(), x.shape)]
    return x, strides[:-1]


def _check(lead, decay, state, resets, grad_state=None, **tokens):
    """The tokens' common shape, dtype and device, and the resets as bytes. lead: leading axes."""
    names = list(tokens)
    first = _rl.as_floats(names[0], tokens[names[0]], (None,) * (lead + 2))
    for name in names[1:]:
        _rl.as_floats(name, tokens[name], first.shape, first.dtype)
    *_, n, h, d = first.shape
    if d not in WIDTHS:
        raise ValueError(f"the heads' width must be one of {WIDTHS}; got {d}")
    _rl.as_floats("decay", decay, (h,), torch.float32)
    for name, s in (("state", state), ("grad_state", grad_state)):
        if s is not None:
            _rl.as_floats(name, s, (n, h, d, d), torch.float32)
    if resets is not None:
        if not isinstance(resets, torch.Tensor) or resets.dtype not in (torch.bool, torch.uint8) \
                or resets.shape != first.shape[:-2]:
            raise ValueError(f"resets must be a bool or uint8 tensor of shape {tuple(first.shape[:-2])}")
        resets = resets.contiguous()
    dev = _rl.same_device(decay=decay, state=state, resets=resets, grad_state=grad_state, **tokens)
    return first.shape, first.dtype, dev, resets


def _scale(scale, d):
    return d ** -0.5 if scale is None else float(scale)


def _strides(rows):
    flat = [s for _, strides in rows for s in strides]
    return (ctypes.c_int64 * len(flat))(*flat)


def forward(q, k, v, decay, state=None, resets=None, scale=None):
    """(out (T, N, H, D), state after the last token (N, H, D, D)). state None starts from zero; the
    given one is not changed. scale None is D ** -0.5."""
    (t, n, h, d), dtype, dev, resets = _check(1 + 1, decay, state, resets, q=q, k=k, v=v)
    rows = [_rows(x) for x in (q, k, v)]
    decay, state = decay.contiguous(), None if state is None else state.contiguous()
    lib, code = _rl.lib(), _rl.FLOAT_DTYPES[dtype]
    with torch.cuda.device(dev):
        out = torch.empty((t, n, h, d), dtype=dtype, device=dev)
        new = torch.empty((n, h, d, d), dtype=torch.float32, device=dev)
        nbytes = lib.linear_attention_scratch_bytes(code, d, t, n, h, 0)
        tmp = _rl.scratch(nbytes, dev)
        _rl.check(lib.linear_attention_forward(
            code, d, t, n, h, *(x.data_ptr() for x, _ in rows), _strides(rows), decay.data_ptr(), _rl.ptr(resets),
            _scale(scale, d), _rl.ptr(state), out.data_ptr(), new.data_ptr(), _rl.ptr(tmp), nbytes,
            _rl.stream_ptr(dev)))
    return out, new


def backward(grad_out, q, k, v, decay, state=None, resets=None, scale=None, grad_state=None):
    """Gradients (dq, dk, dv (T, N, H, D), dstate (N, H, D, D)) of `forward` from grad_out and, where the
    final state is used further, grad_state."""
    (t, n, h, d), dtype, dev, resets = _check(1 + 1, decay, state, resets, grad_state, grad_out=grad_out, q=q, k=k, v=v)
    rows = [_rows(x) for x in (grad_out, q, k, v)]
    decay = decay.contiguous()
    state, grad_state = (None if s is None else s.contiguous() for s in (state, grad_state))
    lib, code = _rl.lib(), _rl.FLOAT_DTYPES[dtype]
    with torch.cuda.device(dev):
        dq, dk, dv = (torch.empty((t, n, h, d), dtype=dtype, device=dev) for _ in range(3))
        dstate = torch.empty((n, h, d, d), dtype=torch.float32, device=dev)
        nbytes = lib.linear_attention_scratch_bytes(code, d, t, n, h, 1)
        tmp = _rl.scratch(nbytes, dev)
        _rl.check(lib.linear_attention_backward(
            code, d, t, n, h, *(x.data_ptr() for x, _ in rows), _strides(rows), decay.data_ptr(), _rl.ptr(resets),
            _scale(scale, d), _rl.ptr(state), _rl.ptr(grad_state), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(),
            dstate.data_ptr(), _rl.ptr(tmp), nbytes, _rl.stream_ptr(dev)))
    return dq, dk, dv, dstate


def step(q, k, v, decay, state, resets=None, scale=None):
    """One token for every environment, q, k, v (N, H, D), resets (N,): updates `state` (N, H, D, D) in
    place and returns out (N, H, D)."""
    (n, h, d), dtype, dev, resets = _check(1, decay, state, resets, q=q, k=k, v=v)
    if state is None or not state.is_contiguous() or state.data_ptr() % 16:
        raise ValueError("state must be contiguous and on a 16-byte boundary: it is updated in place")
    rows = [_rows(x) for x in (q, k, v)]
    decay = decay.contiguous()
    with torch.cuda.device(dev):
        out = torch.empty((n, h, d), dtype=dtype, device=dev)
        _rl.check(_rl.lib().linear_attention_step(
            _rl.FLOAT_DTYPES[dtype], d, n, h, *(x.data_ptr() for x, _ in rows), _strides(rows), decay.data_ptr(),
            _rl.ptr(resets), _scale(scale, d), state.data_ptr(), out.data_ptr(), _rl.stream_ptr(dev)))
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
    def backward(ctx, grad_out, grad_state):
        q, k, v, decay, state, resets = ctx.saved_tensors
        dq, dk, dv, dstate = backward(grad_out.contiguous(), q, k, v, decay, state, resets, ctx.scale, grad_state)
        return dq, dk, dv, None, dstate if state is not None else None, None, None


def attend(q, k, v, decay, state=None, resets=None, scale=None):
    """`forward` as a differentiable operation of q, k, v and state."""
    return _Attend.apply(q, k, v, decay, state, resets, scale)
