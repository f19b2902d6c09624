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

import ctypes
from dataclasses import dataclass

import torch

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


def _blocks(sizes):
    return sum(-(-n // BLOCK) for n in sizes)


def init_state(params, bits=32, seed=0):
    """Zero moments for params."""
    if bits not in (8, 32):
        raise ValueError(f"moments are held in 8 or 32 bits; got {bits}")
    sizes = tuple(p.numel() for p in params)
    dev = _rl.same_device(**{f"params[{i}]": p for i, p in enumerate(params)}) if params else _rl.device()
    blocks = _blocks(sizes)

    def zeros(n, dtype):
        return torch.zeros(n, dtype=dtype, device=dev)

    if bits == 32:
        return State(32, sizes, zeros(blocks * BLOCK, torch.float32), zeros(blocks * BLOCK, torch.float32), seed=seed)
    return State(8, sizes, zeros(blocks * BLOCK, torch.uint8), zeros(blocks * BLOCK, torch.uint8),
                 zeros(blocks, torch.uint8), zeros(blocks, torch.uint8), seed=seed)


def _check_state(state, dev):
    blocks = _blocks(state.sizes)
    if state.bits not in (8, 32):
        raise ValueError(f"moments are held in 8 or 32 bits; got {state.bits}")
    kinds = [("m", torch.float32 if state.bits == 32 else torch.uint8, blocks * BLOCK)]
    kinds.append(("v",) + kinds[0][1:])
    if state.bits == 8:
        kinds += [("m_exp", torch.uint8, blocks), ("v_exp", torch.uint8, blocks)]
    for name, dtype, n in kinds:
        x = getattr(state, name)
        if x is None or x.dtype != dtype or x.numel() != n or not x.is_contiguous() or x.device != dev:
            raise ValueError(f"state.{name} must be {n} contiguous {dtype} elements on {dev}")


def step(params, grads, state, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01, copies=None,
         grad_scale=None):
    """Updates params, state and copies in place. grads: one tensor a parameter, all of one dtype.
    grad_scale, a one-element float32 CUDA tensor, multiplies every gradient (clipping by a norm that
    stays on the device)."""
    count = len(params)
    if len(grads) != count or (copies is not None and len(copies) != count) or len(state.sizes) != count:
        raise ValueError(f"{count} params need as many grads, copies and state.sizes")
    if count == 0:
        state.step += 1
        return
    dev, grad_dtype = params[0].device, grads[0].dtype
    if grad_dtype not in _rl.FLOAT_DTYPES:
        raise ValueError(f"grads must be float32 or bfloat16; got {grad_dtype}")
    for i, (p, g, n) in enumerate(zip(params, grads, state.sizes)):
        if p.dtype != torch.float32 or not p.is_contiguous() or p.device != dev or not p.is_cuda or p.numel() != n:
            raise ValueError(f"params[{i}] must be {n} contiguous float32 elements on one CUDA device")
        if g.dtype != grad_dtype or g.device != dev or g.shape != p.shape:
            raise ValueError(f"grads[{i}] must be {grad_dtype} on {dev}, of its parameter's shape")
    if copies is not None:
        for i, (p, c) in enumerate(zip(params, copies)):
            if c.dtype != torch.bfloat16 or not c.is_contiguous() or c.device != dev or c.shape != p.shape:
                raise ValueError(f"copies[{i}] must be contiguous bfloat16 on {dev}, of its parameter's shape")
    if grad_scale is not None:
        _rl.as_floats("grad_scale", grad_scale, dtype=torch.float32)
        if grad_scale.numel() != 1 or grad_scale.device != dev:
            raise ValueError(f"grad_scale must be one float32 on {dev}")
    _check_state(state, dev)
    b1, b2 = betas
    grads = [g.contiguous() for g in grads]
    pointers = ctypes.c_void_p * count
    with torch.cuda.device(dev):
        _rl.check(_rl.lib().adamw_step(
            state.bits, _rl.FLOAT_DTYPES[grad_dtype], count, pointers(*[p.data_ptr() for p in params]),
            pointers(*[g.data_ptr() for g in grads]),
            pointers(*[c.data_ptr() for c in copies]) if copies is not None else None,
            (ctypes.c_int64 * count)(*state.sizes), state.m.data_ptr(), state.v.data_ptr(), _rl.ptr(state.m_exp),
            _rl.ptr(state.v_exp), lr, b1, b2, eps, weight_decay, _rl.ptr(grad_scale), state.step + 1,
            state.seed & 0xFFFFFFFF, _rl.stream_ptr(dev)))
    state.step += 1


def moments(state):
    """(m, v), flat float32 tensors laid out as the state's: the state's own where it holds 32 bits, the
    values that its codes stand for where it holds 8."""
    dev = state.m.device
    _check_state(state, dev)
    if state.bits == 32:
        return state.m, state.v
    with torch.cuda.device(dev):
        m = torch.empty(state.m.numel(), dtype=torch.float32, device=dev)
        v = torch.empty_like(m)
        _rl.check(_rl.lib().adamw_moments(state.m_exp.numel(), state.m.data_ptr(), state.v.data_ptr(),
                                          state.m_exp.data_ptr(), state.v_exp.data_ptr(), m.data_ptr(), v.data_ptr(),
                                          _rl.stream_ptr(dev)))
    return m, v
