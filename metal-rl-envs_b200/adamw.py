"""One AdamW step over many tensors at once (Loshchilov & Hutter 2019), as an sm_100a kernel:

    m <- b1 m + (1 - b1) g,   v <- b2 v + (1 - b2) g^2,
    p <- p (1 - lr wd) - lr (m / (1 - b1^t)) / (sqrt(v / (1 - b2^t)) + eps)

Parameters are float32 (views of one flat vector, as es.unflatten's, are fine); gradients float32 or
bfloat16; `copies` are optional bfloat16 tensors that receive the stepped parameters in the same pass.
The moments live in a `State`: 32 bits an element, or 8 bits with an exponent byte for each block of
256 elements and stochastic rounding (csrc/adamw.cu says how). ES (es.py) needs no optimizer state;
the reference has no counterpart.

Gradients are expected to be finite; a value that is not makes its own element's parameter and moments
NaN or infinite and no other's.
"""

from array import array
from dataclasses import dataclass
from functools import lru_cache
from operator import attrgetter

import torch
from torch.autograd.graph import increment_version

import rlenv_lib as _rl

BLOCK = 256


@dataclass
class State:
    """The moments of a list of tensors. m and v are flat; tensor i starts at the sum of the earlier
    sizes, each rounded up to BLOCK. bits 32: float32; bits 8: uint8 codes, with m_exp and v_exp one byte
    a block. `step` counts the steps taken and `seed` picks the rounding's random stream: a saved State
    continues exactly."""
    bits: int
    sizes: tuple
    m: torch.Tensor
    v: torch.Tensor
    m_exp: torch.Tensor | None = None
    v_exp: torch.Tensor | None = None
    step: int = 0
    seed: int = 0


@lru_cache(maxsize=64)
def _blocks(sizes):
    return sum(-(-n // BLOCK) for n in sizes)


def init_state(params, bits=32, seed=0):
    """Zero moments for params."""
    if bits not in (8, 32):
        raise ValueError(f"moments are held in 8 or 32 bits; got {bits}")
    sizes = tuple(p.numel() for p in params)
    dev = params[0].device if params else _rl.device()
    blocks = _blocks(sizes)

    def zeros(n, dtype):
        return torch.zeros(n, dtype=dtype, device=dev)

    if bits == 32:
        return State(32, sizes, zeros(blocks * BLOCK, torch.float32), zeros(blocks * BLOCK, torch.float32), seed=seed)
    return State(8, sizes, zeros(blocks * BLOCK, torch.uint8), zeros(blocks * BLOCK, torch.uint8),
                 zeros(blocks, torch.uint8), zeros(blocks, torch.uint8), seed=seed)


def _check_state(state):
    """The state's device index; raises where its tensors do not fit its sizes."""
    blocks = _blocks(tuple(state.sizes))
    if state.bits not in (8, 32):
        raise ValueError(f"moments are held in 8 or 32 bits; got {state.bits}")
    kind = torch.float32 if state.bits == 32 else torch.uint8
    index = state.m.get_device()
    _expect("state.m", state.m, kind, blocks * BLOCK, index)
    _expect("state.v", state.v, kind, blocks * BLOCK, index)
    if state.bits == 8:
        _expect("state.m_exp", state.m_exp, torch.uint8, blocks, index)
        _expect("state.v_exp", state.v_exp, torch.uint8, blocks, index)
    return index


def _expect(name, x, dtype, n, index):
    if not isinstance(x, torch.Tensor) or x.dtype is not dtype or x.numel() != n or not x.is_contiguous() or x.get_device() != index \
            or index < 0:
        raise ValueError(f"{name} must be {n} contiguous {dtype} elements on the state's CUDA device")


_dtype, _numel, _index = attrgetter("dtype"), torch.Tensor.numel, torch.Tensor.get_device
_dense, _pointer = torch.Tensor.is_contiguous, torch.Tensor.data_ptr


def _check_list(name, tensors, dtype, sizes, index):
    """Every tensor dense, of dtype, on the device, of its size: the whole list in a few passes that run in
    the interpreter's C loops (a policy has dozens of small tensors and a step of some microseconds)."""
    try:
        fit = set(map(_dtype, tensors)) == {dtype} and set(map(_index, tensors)) == {index} \
            and all(map(_dense, tensors)) and tuple(map(_numel, tensors)) == sizes
    except (AttributeError, TypeError):  # None, say: a parameter without a gradient
        fit = False
    if not fit:
        raise ValueError(f"{name} must be contiguous {dtype} tensors on cuda:{index} of the state's sizes {sizes}")


def step(params, grads, state, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01, copies=None,
         grad_scale=None):
    """Updates params, state and copies in place. grads: one tensor a parameter, all of one dtype.
    grad_scale, a one-element float32 CUDA tensor, multiplies every gradient (clipping by a norm that
    stays on the device). Autograd sees the tensors as written in place: a graph that saved one of them raises in
    its backward pass."""
    count, sizes = len(state.sizes), tuple(state.sizes)
    if len(params) != count or len(grads) != count or (copies is not None and len(copies) != count):
        raise ValueError(f"{len(params)} params need as many grads, copies and state.sizes")
    if count == 0:
        state.step += 1
        return
    index, grad_dtype = _check_state(state), getattr(grads[0], "dtype", None)
    if grad_dtype not in _rl.FLOAT_DTYPES:
        raise ValueError(f"grads must be float32 or bfloat16; got {grad_dtype}")
    _check_list("params", params, torch.float32, sizes, index)
    try:
        _check_list("grads", grads, grad_dtype, sizes, index)
    except ValueError:  # a gradient with strides is copied; anything else raises here
        grads = [g.contiguous() if isinstance(g, torch.Tensor) else g for g in grads]
        _check_list("grads", grads, grad_dtype, sizes, index)
    if copies is not None:
        _check_list("copies", copies, torch.bfloat16, sizes, index)
    if grad_scale is not None:
        _expect("grad_scale", grad_scale, torch.float32, 1, index)
    b1, b2 = betas
    # the lists of pointers and sizes, alive until the call returns
    lists = [array("Q", map(_pointer, params)), array("Q", map(_pointer, grads)),
             array("Q", map(_pointer, copies)) if copies is not None else None, array("q", sizes)]
    params_at, grads_at, copies_at, sizes_at = (None if x is None else x.buffer_info()[0] for x in lists)
    _rl.launch(index, _rl.lib().adamw_step, state.bits, _rl.FLOAT_DTYPES[grad_dtype], count, params_at, grads_at,
               copies_at, sizes_at, state.m.data_ptr(), state.v.data_ptr(), _rl.ptr(state.m_exp), _rl.ptr(state.v_exp),
               lr, b1, b2, eps, weight_decay, _rl.ptr(grad_scale), state.step + 1, state.seed & 0xFFFFFFFF)
    increment_version([*params, *(copies or ()), state.m, state.v])
    state.step += 1


def moments(state):
    """(m, v), flat float32 tensors laid out as the state's: the state's own where it holds 32 bits, the
    values that its codes stand for where it holds 8."""
    if state.bits == 32:
        return state.m, state.v
    index = _check_state(state)
    m, v = (state.m.new_empty(state.m.numel(), dtype=torch.float32) for _ in range(2))
    _rl.launch(index, _rl.lib().adamw_moments, state.m_exp.numel(), state.m.data_ptr(), state.v.data_ptr(),
               state.m_exp.data_ptr(), state.v_exp.data_ptr(), m.data_ptr(), v.data_ptr())
    return m, v
