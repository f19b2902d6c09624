"""Matrix products of 8-bit integers with scales, as sm_100a kernels: a policy that acts in 8 bits.

    out = (codes w_codes') * scale * w_scale

codes (..., K) int8 with a scale for each token (rms_norm.forward8 or `quantise` make them), a weight's codes (F, K)
int8 with a scale for each of its F channels (`quantise_weight`, once). Sums are exact in 32-bit integers, K up to
131,071, and multiplied in float32 by the token's scale, then by the channel's; the result, float32 or bfloat16, is
rounded from that. Tokens and channels are fewer than 2^31 - 256. There is no gradient: this is for acting. The
reference's policies are float32 MLPs (es.py:156-164); there is no counterpart there.
"""

import ctypes
from dataclasses import dataclass

import torch

import rlenv_lib as _rl
import rms_norm

MOST_TERMS = 131_071  # whose products of 8-bit integers sum below 2^31


@dataclass
class Weight:
    """A weight in 8 bits: codes (F, K) int8 with rows on 16-byte boundaries, scale (F,) float32. The value of row f is
    codes[f] * scale[f]: a channel's inputs lie side by side, unlike in the (K, F) matrix that it is made of."""
    codes: torch.Tensor
    scale: torch.Tensor


def quantise(x):
    """(codes (..., K) int8, scale (...) float32) of x (..., K), float32 or bfloat16: each row's largest magnitude
    over 127 is its scale. Rows of codes start on 16-byte boundaries; tokens that are zero or not finite are as
    rms_norm.forward8's."""
    m, k, code, index = rms_norm._check("x", x, None, 0.0)
    x, xs = _rl.as_rows(x)
    codes, scale = rms_norm.codes_like(x, k), _rl.empty_lead(x, torch.float32)
    _rl.launch(index, _rl.lib().rms_norm_codes, code, m, k, x.data_ptr(), xs, 0, 0, 0, 0.0, 0, codes.data_ptr(),
               (k + 15) // 16 * 16, scale.data_ptr(), 0)
    return codes, scale


def quantise_weight(w):
    """The Weight of w (K, F), the layout of the other operators' weights: a scale for each column of it."""
    _rl.as_floats("w", w)
    if w.dim() != 2:
        raise ValueError(f"w must be (K, F); got shape {tuple(w.shape)}")
    return Weight(*quantise(w.detach().t().contiguous()))


def _on_boundaries(codes, rows):
    """(codes, bytes between rows) with rows on 16-byte boundaries; anything else is copied."""
    k = codes.shape[-1]
    codes, pitch = _rl.as_rows(codes)
    if rows <= 1:
        pitch = (k + 15) // 16 * 16  # of one row, any
    if pitch % 16 or pitch < k or codes.data_ptr() % 16:
        room = rms_norm.codes_like(codes, k)
        room.copy_(codes)
        return room, (k + 15) // 16 * 16
    return codes, pitch


def forward(codes, scale, weight, dtype=torch.bfloat16):
    """(codes * scale) times the weight's transpose, (..., F) of dtype, from codes (..., K) and scale (...)."""
    if not isinstance(weight, Weight):
        raise ValueError(f"weight must be a Weight, as quantise_weight makes them; got {type(weight).__name__}")
    w, ws = weight.codes, weight.scale
    try:  # what fits passes on a few comparisons
        index = codes.get_device()
        fit = index >= 0 and scale.get_device() == index and w.get_device() == index and ws.get_device() == index \
            and codes.dtype is torch.int8 and w.dtype is torch.int8 and scale.dtype is ws.dtype is torch.float32
    except (AttributeError, TypeError):
        fit = False
    if not fit:
        for name, x, kind in (("codes", codes, torch.int8), ("scale", scale, torch.float32), ("weight.codes", w, torch.int8),
                              ("weight.scale", ws, torch.float32)):
            if not isinstance(x, torch.Tensor) or x.dtype is not kind or not x.is_cuda:
                raise ValueError(f"{name} must be a CUDA tensor of {kind}: there is no CPU path")
        _rl.one_device(index, scale=scale, **{"weight.codes": w, "weight.scale": ws})
    lead, of_w = scale.shape, w.shape
    if len(of_w) != 2 or codes.shape != (*lead, of_w[1]) or ws.shape != of_w[:1]:
        raise ValueError(f"codes (..., K), scale (...), weight.codes (F, K) and weight.scale (F,) do not fit: got "
                         f"{tuple(codes.shape)}, {tuple(lead)}, {tuple(of_w)} and {tuple(ws.shape)}")
    f, k = of_w
    if not 1 <= k <= MOST_TERMS:
        raise ValueError(f"K must be from 1 to {MOST_TERMS}, so that sums fit 32 bits; got {k}")
    if dtype not in _rl.FLOAT_DTYPES:
        raise ValueError(f"dtype must be float32 or bfloat16; got {dtype}")
    m = scale.numel()
    (codes, pitch), (w, w_pitch) = _on_boundaries(codes, m), _on_boundaries(w, f)
    scale, ws, lib = scale.contiguous(), ws.contiguous(), _rl.lib()
    out = _rl.empty_rows(codes, f, dtype)
    nbytes = lib.int8_linear_scratch_bytes(m, k, f)
    tmp = _rl.scratch(nbytes, codes)
    _rl.launch(index, lib.int8_linear_forward, _rl.FLOAT_DTYPES[dtype], m, k, f, codes.data_ptr(), pitch, scale.data_ptr(),
               w.data_ptr(), w_pitch, ws.data_ptr(), out.data_ptr(), _rl.ptr(tmp), nbytes)
    return out


def product(x, weight, dtype=None):
    """`forward` of x (..., K) in 8 bits, (..., F) of dtype (None: x's)."""
    return forward(*quantise(x), weight, dtype or x.dtype)


def gave_up(device=None, clear=True):
    """As gated_ffn.gave_up, for this module's kernels: how many thread blocks on `device` ended with a wait that ran
    out. Zero unless something is wrong with the machine. Waits for the device."""
    count = ctypes.c_uint(0)
    with torch.cuda.device(device):
        _rl.check(_rl.lib().int8_linear_status(ctypes.byref(count), int(clear)))
    return count.value
