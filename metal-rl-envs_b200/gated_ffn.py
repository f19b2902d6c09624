"""Gated feed-forward block: out = act(x w_gate) * (x w_up), both products, the activation and the
product in one sm_100a kernel, and its gradient.

x is (..., K), the weights (K, F) as es.unflatten's (in, out) layout, out (..., F), all of one type,
float32 or bfloat16; sums are in 32 bits. activation is "silu" or "gelu" (the exact normal
distribution). `backward` forms both products again instead of keeping them. `apply` is the
differentiable form. The projection back to K is a plain matrix product and is left to the caller.
float32 operands go through the tensor cores as sums of three bfloat16 terms, but for few rows: results
have float32's precision, but an infinity, or a magnitude above bfloat16's 3.39e38, may come out as NaN, and of
operands below 2^-110 (8e-34) the lower terms are lost. bfloat16 gradients: the two products' own gradients,
grad_out act'(x w_gate) (x w_up) and grad_out act(x w_gate), are rounded to bfloat16 before the products that
follow.
The reference's policies are tanh MLPs (es.py:156-164); there is no counterpart there.
"""

import ctypes

import torch
from torch.autograd.function import once_differentiable

import rlenv_lib as _rl

ACTIVATIONS = {"silu": 0, "gelu": 1}


def _dense(x):
    """x itself where it is dense and on a 16-byte boundary, else a copy that is."""
    x = x.contiguous()
    return x if x.data_ptr() % 16 == 0 else x.clone()


def _check(x, w_gate, w_up, activation, *grad_out):
    """(M, K, F, the type's code, the device's index). What fits passes on a few comparisons; what does not is
    looked at again for the message."""
    _rl.as_floats("x", x)
    if not isinstance(w_gate, torch.Tensor):
        _rl.as_floats("w_gate", w_gate)
    index, dtype = x.get_device(), x.dtype
    if x.dim() < 1 or w_gate.dim() != 2 or w_gate.shape[0] != x.shape[-1]:
        raise ValueError(f"x must be (..., K) and w_gate (K, F); got {tuple(x.shape)} and {tuple(w_gate.shape)}")
    k, f = w_gate.shape
    for name, w in (("w_gate", w_gate), ("w_up", w_up)):
        if not isinstance(w, torch.Tensor) or w.get_device() != index or w.dtype is not dtype or w.shape != (k, f):
            _rl.as_floats(name, w, (k, f), dtype)
            _rl.one_device(index, **{name: w})
    for g in grad_out:
        _rl.as_floats("grad_out", g, (*x.shape[:-1], f), dtype)
        _rl.one_device(index, grad_out=g)
    if activation not in ACTIVATIONS:
        raise ValueError(f"activation must be one of {sorted(ACTIVATIONS)}; got {activation!r}")
    return x.numel() // k if k else x.shape[:-1].numel(), k, f, _rl.FLOAT_DTYPES[dtype], index


def forward(x, w_gate, w_up, activation="silu"):
    """act(x w_gate) * (x w_up), (..., F)."""
    m, k, f, code, index = _check(x, w_gate, w_up, activation)
    x, w_gate, w_up = _dense(x), _dense(w_gate), _dense(w_up)
    lib = _rl.lib()
    out = x.new_empty((*x.shape[:-1], f))
    nbytes = lib.gated_ffn_scratch_bytes(code, m, k, f, 0)
    tmp = _rl.scratch(nbytes, x)
    _rl.launch(index, lib.gated_ffn_forward, code, ACTIVATIONS[activation], m, k, f, x.data_ptr(), w_gate.data_ptr(),
               w_up.data_ptr(), out.data_ptr(), _rl.ptr(tmp), nbytes)
    return out


def backward(grad_out, x, w_gate, w_up, activation="silu"):
    """(dx, dw_gate, dw_up) of `forward` from grad_out (..., F)."""
    m, k, f, code, index = _check(x, w_gate, w_up, activation, grad_out)
    if 0 in (m, k, f):  # sums over nothing
        return torch.zeros_like(x), torch.zeros_like(w_gate), torch.zeros_like(w_up)
    grad_out, x, w_gate, w_up = _dense(grad_out), _dense(x), _dense(w_gate), _dense(w_up)
    lib = _rl.lib()
    dx, dwg, dwu = torch.empty_like(x), torch.empty_like(w_gate), torch.empty_like(w_up)
    nbytes = lib.gated_ffn_scratch_bytes(code, m, k, f, 1)
    tmp = _rl.scratch(nbytes, x)
    _rl.launch(index, lib.gated_ffn_backward, code, ACTIVATIONS[activation], m, k, f, grad_out.data_ptr(), x.data_ptr(),
               w_gate.data_ptr(), w_up.data_ptr(), dx.data_ptr(), dwg.data_ptr(), dwu.data_ptr(), _rl.ptr(tmp), nbytes)
    return dx, dwg, dwu


def gave_up(device=None, clear=True):
    """How many thread blocks on `device` (None: the current one) ended with a wait that ran out since the last
    clear: zero unless something is wrong with the machine. Results of such a call hold NaN. Waits for the
    device."""
    count = ctypes.c_uint(0)
    with torch.cuda.device(device):
        _rl.check(_rl.lib().gated_ffn_status(ctypes.byref(count), int(clear)))
    return count.value


class _Apply(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w_gate, w_up, activation):
        ctx.save_for_backward(x, w_gate, w_up)
        ctx.activation = activation
        return forward(x, w_gate, w_up, activation)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_out):
        x, w_gate, w_up = ctx.saved_tensors
        return (*backward(grad_out, x, w_gate, w_up, ctx.activation), None)


def apply(x, w_gate, w_up, activation="silu"):
    """`forward` as a differentiable operation of x and both weights."""
    return _Apply.apply(x, w_gate, w_up, activation)
