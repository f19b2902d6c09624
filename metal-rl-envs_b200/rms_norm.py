"""Root-mean-square norm with the residual's addition, as sm_100a kernels:

    total = x + residual,   out = total / sqrt(mean(total^2) + eps) * weight

x and residual are (..., K), weight (K,), all of one type, float32 or bfloat16; sums are in 32 bits. `total` is the
residual stream that the next layer adds to; out is formed from it before it is rounded to the tensors' type.

- `forward` and `backward`, and `apply`, forward with its gradient through torch.autograd;
- `forward8` gives out in 8-bit integers with a scale for each token, for int8_linear's products.

Rows, fewer than 2^31 of them, may be any even step apart (slices of wider rows, expanded ones); other strides are
copied. Squares are summed in float32: magnitudes above 1.8e19 overflow to a norm of zeros, squares of those below 1e-19
lose precision and below 4e-23 are 0, which only an eps near 0 shows. With an eps of 0 a token of zeros is NaN, and one
whose squares are all 0 infinite. The reference's policies are tanh MLPs (es.py:156-164); there is no counterpart there.
"""

import torch
from torch.autograd.function import once_differentiable

import rlenv_lib as _rl


def _check(name, x, weight, eps, others=()):
    """(rows, K, the type's code, the device's index); others are (name, tensor) of x's kind or None. What fits passes on
    a few comparisons; what does not is looked at again for the message."""
    if not isinstance(x, torch.Tensor) or not x.is_cuda or x.dtype not in _rl.FLOAT_DTYPES:
        _rl.as_floats(name, x)
    shape, dtype, index = x.shape, x.dtype, x.get_device()
    if not shape or shape[-1] == 0:
        raise ValueError(f"{name} must be (..., K) with K of at least 1; got shape {tuple(shape)}")
    for other, y in others:
        if y is not None and (not isinstance(y, torch.Tensor) or y.get_device() != index or y.dtype is not dtype
                              or y.shape != shape):
            _rl.as_floats(other, y, shape, dtype)
            _rl.one_device(index, **{other: y})
    k = shape[-1]
    if weight is not None and (not isinstance(weight, torch.Tensor) or weight.get_device() != index
                               or weight.dtype is not dtype or weight.shape != (k,)):
        _rl.as_floats("weight", weight, (k,), dtype)
        _rl.one_device(index, weight=weight)
    if not eps >= 0.0:
        raise ValueError(f"eps must not be negative; got {eps}")
    return x.numel() // k, k, _rl.FLOAT_DTYPES[dtype], index


def _like(x):
    """A dense tensor of x's shape and type."""
    return torch.empty_like(x) if x.is_contiguous() else x.new_empty(x.shape)


def forward(x, weight=None, residual=None, eps=1e-6):
    """(out, total), both (..., K). residual None: total is x itself; weight None: ones."""
    m, k, code, index = _check("x", x, weight, eps, (("residual", residual),))
    if weight is not None:
        weight = weight.contiguous()
    x, xs = _rl.as_rows(x)
    out = _like(x)
    if residual is None:
        total, res_at, rs, total_at = x, 0, 0, 0
    else:
        residual, rs = _rl.as_rows(residual)
        total = torch.empty_like(out)
        res_at, total_at = residual.data_ptr(), total.data_ptr()
    _rl.launch(index, _rl.lib().rms_norm_forward, code, m, k, x.data_ptr(), xs, res_at, rs, _rl.ptr(weight), eps,
               out.data_ptr(), total_at)
    return out, total


def codes_like(x, k):
    """Room for 8-bit rows of k as int8_linear takes them: (..., K) int8, rows on 16-byte boundaries."""
    return _rl.empty_rows(x, k, torch.int8, (k + 15) // 16 * 16)


def forward8(x, weight=None, residual=None, eps=1e-6):
    """(codes (..., K) int8, scale (...) float32, total): out = codes * scale, each token's scale its largest magnitude
    over 127, rounded to the nearest. Rows of codes start on 16-byte boundaries. A token whose out is below 2^-100 is
    zeros with scale 0; one that holds a value that is not finite is zeros with scale NaN."""
    m, k, code, index = _check("x", x, weight, eps, (("residual", residual),))
    if weight is not None:
        weight = weight.contiguous()
    x, xs = _rl.as_rows(x)
    if residual is None:
        total, res_at, rs, total_at = x, 0, 0, 0
    else:
        residual, rs = _rl.as_rows(residual)
        total = _like(x)
        res_at, total_at = residual.data_ptr(), total.data_ptr()
    codes, scale = codes_like(x, k), _rl.empty_lead(x, torch.float32)
    _rl.launch(index, _rl.lib().rms_norm_codes, code, m, k, x.data_ptr(), xs, res_at, rs, _rl.ptr(weight), eps, 1,
               codes.data_ptr(), (k + 15) // 16 * 16, scale.data_ptr(), total_at)
    return codes, scale, total


def backward(grad_out, total, weight=None, eps=1e-6, grad_total=None):
    """(grad, grad_weight) from grad_out and, where the total is used further, grad_total: grad (..., K) is the
    gradient of x and of the residual alike, grad_weight (K,) or None without a weight."""
    return _backward(grad_out, total, weight, eps, grad_total, weight is not None)


def _backward(grad_out, total, weight, eps, grad_total, of_weight):
    """`backward`; of_weight: whether the weight's gradient, sums over all rows, is wanted."""
    m, k, code, index = _check("total", total, weight, eps, (("grad_out", grad_out), ("grad_total", grad_total)))
    lib = _rl.lib()
    if m == 0:
        return torch.empty_like(total), torch.zeros_like(weight) if of_weight else None
    (g, gs), (t, ts) = _rl.as_rows(grad_out), _rl.as_rows(total)
    s, ss = (None, 0) if grad_total is None else _rl.as_rows(grad_total)
    grad = _like(t)
    grad_weight, tmp, nbytes = None, None, 0
    if weight is not None:
        weight = weight.contiguous()
    if of_weight:
        grad_weight, nbytes = torch.empty_like(weight), lib.rms_norm_scratch_bytes(m, k)
        tmp = _rl.scratch(nbytes, t)
    _rl.launch(index, lib.rms_norm_backward, code, m, k, g.data_ptr(), gs, t.data_ptr(), ts, _rl.ptr(weight), eps,
               _rl.ptr(s), ss, grad.data_ptr(), _rl.ptr(grad_weight), _rl.ptr(tmp), nbytes)
    return grad, grad_weight


class _Apply(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, residual, eps):
        out, total = forward(x, weight, residual, eps)
        ctx.save_for_backward(total, weight)
        ctx.eps, ctx.with_residual = eps, residual is not None
        ctx.set_materialize_grads(False)
        return (out, total) if ctx.with_residual else out

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_out, grad_total=None):
        total, weight = ctx.saved_tensors
        if grad_out is None:  # the norm is not used
            return grad_total, None, grad_total if ctx.with_residual else None, None
        # a frozen weight's gradient would be a second kernel for what is dropped
        grad, grad_weight = _backward(grad_out, total, weight, ctx.eps, grad_total, ctx.needs_input_grad[1])
        return grad, grad_weight, grad if ctx.with_residual else None, None


def apply(x, weight=None, residual=None, eps=1e-6):
    """`forward` as a differentiable operation of x, weight and residual: (out, total). The gradient is taken at the
    total as it is stored."""
    if residual is not None:
        return _Apply.apply(x, weight, residual, eps)
    return _Apply.apply(x, weight, None, eps), x
