"""The norm, the 8-bit products and the scores of actions on the GPU against the oracle in 64 bits.

Tolerances are bounds on rounding, element by element. A float32 sum whose longest chain of additions is n is within
(n + the roundings of a term) 2^-24 of the same sum of magnitudes; a team of threads adds up to 128 terms a thread and
then in a tree, longer rows K / 512 a thread. rsqrtf errs by 2^-22, expf's fast form by (2 + 1.2 |x|) 2^-23, a product or
quotient by 2^-24. Results of type t are rounded by at most finfo(t).eps / 2 of their value."""

import numpy as np
import pytest
import torch

import rlenv_lib
from oracle import policy

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
HALF = 2.0 ** -24


def to64(x):
    return x.detach().double().cpu().numpy()


def half(dtype):
    return torch.finfo(TYPES[dtype]).eps / 2


def close(got, want, tol, what):
    got = to64(got)
    assert got.shape == want.shape, what
    bad = ~np.isfinite(want)
    assert np.array_equal(got[bad], want[bad], equal_nan=True), f"{what}: values that are not finite"
    off = np.abs(np.where(bad, 0.0, got) - np.where(bad, 0.0, want)) - np.where(bad, 0.0, tol)
    assert (off <= 0).all(), f"{what}: {(~(off <= 0)).sum()} of {off.size} outside, worst by {np.nanmax(off):.3g} at " \
                             f"{np.unravel_index(np.nanargmax(off), off.shape)}"


def chain(k):
    return min(k, 128) + k / 512 + 12


def normal(cuda, *shape, seed=0, scale=1.0, dtype="f32"):
    g = torch.Generator(device=cuda).manual_seed(seed)
    return (torch.randn(shape, generator=g, device=cuda) * scale).to(TYPES[dtype])


# ---- the norm ------------------------------------------------------------------------------------------

NORM_SIZES = [(1, 1), (3, 7), (1, 8), (9, 96), (18, 97), (5, 256), (2, 257), (33, 512), (7, 513), (300, 40), (4, 1000),
              (3, 1024), (2, 1032), (2, 2047), (3, 4096), (2, 4097), (1, 8200), (2, 16384), (1, 16383), (2, 20001),
              (1, 40000), (700, 128)]


def norm_tol(k, want, dtype):
    # t is exact to half a step, its square's sum to chain(k) halves, r to half of that and rsqrtf's, two products
    return ((chain(k) + 4) / 2 + 10) * HALF * abs(want) + half(dtype) * abs(want) + 1e-37


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("m,k", NORM_SIZES)
def test_norm_forward(cuda, m, k, dtype):
    import rms_norm

    x, y = normal(cuda, m, k, dtype=dtype), normal(cuda, m, k, seed=1, scale=3.0, dtype=dtype)
    w = (1 + 0.2 * normal(cuda, k, seed=2)).to(TYPES[dtype])
    for weight, residual in ((w, y), (None, None), (w, None), (None, y)):
        out, total = rms_norm.forward(x, weight, residual, 1e-5)
        t = to64(x) if residual is None else to64(x) + to64(residual)
        assert out.dtype == total.dtype == x.dtype and out.is_contiguous()
        close(total, t, (HALF + half(dtype)) * abs(t), "total")
        assert residual is not None or total is x
        want = policy.norm(t, None if weight is None else to64(weight), 1e-5)
        close(out, want, norm_tol(k, want, dtype), "out")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("m,k", NORM_SIZES)
def test_norm_in_8_bits(cuda, m, k, dtype):
    import int8_linear
    import rms_norm

    x, y = normal(cuda, m, k, dtype=dtype), normal(cuda, m, k, seed=1, scale=3.0, dtype=dtype)
    w = (1 + 0.2 * normal(cuda, k, seed=2)).to(TYPES[dtype])
    codes, scale, total = rms_norm.forward8(x, w, y, 1e-5)
    t = to64(x) + to64(y)
    want = policy.norm(t, to64(w), 1e-5)
    close(total, t, (HALF + half(dtype)) * abs(t), "total")
    off = norm_tol(k, want, "f32")  # of the values before their codes
    top = abs(want).max(-1, keepdims=True)
    rel = off.max(-1, keepdims=True) / np.where(top > 0, top, 1) + 3 * HALF
    close(scale, top[:, 0] / 127, rel[:, 0] * top[:, 0] / 127, "scale")
    # a code is the nearest whole number to the value over the scale, each a little off
    close(codes, want / np.where(top > 0, top / 127, 1.0), 0.5 + 127 * 2 * rel, "codes")
    assert codes.dtype == torch.int8 and scale.dtype == torch.float32
    assert codes.data_ptr() % 16 == 0 and (m == 1 or codes.stride(0) % 16 == 0)
    # without a norm: the values themselves, whose scale and codes are known but for ties' neighbours
    codes, scale = int8_linear.quantise(x)
    want = to64(x)
    top = abs(want).max(-1, keepdims=True)
    close(scale, top[:, 0] / 127, HALF * top[:, 0] / 127, "scale of rows")
    close(codes, want * 127 / np.where(top > 0, top, 1.0), 0.5 + 127 * 3 * HALF, "codes of rows")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("m,k", NORM_SIZES + [(5000, 72), (4999, 33), (3000, 333), (701, 2049), (1300, 1001), (700, 4096),
                                              (333, 8193)])
def test_norm_backward(cuda, m, k, dtype):
    import rms_norm

    t, g = normal(cuda, m, k, scale=3.0, dtype=dtype), normal(cuda, m, k, seed=1, dtype=dtype)
    s, w = normal(cuda, m, k, seed=2, dtype=dtype), (1 + 0.2 * normal(cuda, k, seed=3)).to(TYPES[dtype])
    for weight, stream in ((w, s), (None, None), (w, None), (None, s)):
        grad, grad_weight = rms_norm.backward(g, t, weight, 1e-5, stream)
        args = (to64(g), to64(t), None if weight is None else to64(weight), 1e-5, None if stream is None else to64(stream))
        want, want_w = policy.norm_grad(*args)
        mag, mag_w = policy.norm_grad(*args, absolute=True)
        n = 2.5 * chain(k) + 24  # the two sums, r to the third power, some products
        close(grad, want, n * HALF * mag + half(dtype) * abs(want), "grad")
        assert (grad_weight is None) == (weight is None)
        if weight is not None:
            rows = min(m, m / 296 + 60)  # a team's rows, a block's teams, the blocks' sums
            close(grad_weight, want_w, (rows + chain(k) / 2 + 16) * HALF * mag_w + half(dtype) * abs(want_w), "grad_weight")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("vectors", [16, 32, 64, 96, 128, 192, 256, 384, 512, 768, 1024, 1536, 2048, 4096])
def test_norm_at_the_borders_between_forms(cuda, vectors, dtype):
    """Rows of as many vectors of 16 bytes and of one more, whole and with values before and after them; gradients of
    blocks with a second row."""
    each = 4 if dtype == "f32" else 8
    for k in (vectors * each, vectors * each + 1, vectors * each + each, vectors * each + each + 3):
        test_norm_forward(cuda, 9, k, dtype)
        test_norm_in_8_bits(cuda, 9, k, dtype)
        test_norm_backward(cuda, 150 if k > 2000 else 1500, k, dtype)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_norm_takes_rows_of_any_layout(cuda, dtype):
    """Slices, expanded rows, strides that are copied and bases off every boundary."""
    import int8_linear
    import rms_norm

    wide = normal(cuda, 6, 5, 136, dtype=dtype)
    views = [wide[..., :128], wide[..., 8:], wide[..., 1:129], wide[:, 2, 3:100], wide[0, :1, :128].expand(7, 128),
             wide.transpose(0, 1)[..., :64], wide[..., ::2], wide[0, 0, 5:69], wide[:1, :1, :64]]
    for x in views:
        k, y = x.shape[-1], torch.flip(x, (0,))
        w = normal(cuda, k, seed=5, dtype=dtype)
        t = to64(x) + to64(y)
        want = policy.norm(t, to64(w), 1e-6)
        out, total = rms_norm.forward(x, w, y)
        close(out, want, norm_tol(k, want, dtype), "out")
        close(total, t, (HALF + half(dtype)) * abs(t), "total")
        codes, scale, total = rms_norm.forward8(x, w, y)
        close(total, t, (HALF + half(dtype)) * abs(t), "total of codes")
        close(codes * scale[..., None], want, 0.501 * abs(want).max(-1, keepdims=True) / 127, "codes")
        dense = x.clone(memory_format=torch.contiguous_format)
        assert all(torch.equal(a, b) for a, b in zip(int8_linear.quantise(x), int8_linear.quantise(dense)))
        grad, grad_weight = rms_norm.backward(x, x, w, 1e-6, x)
        args = (to64(x), to64(x), to64(w), 1e-6, to64(x))
        (want, want_w), (mag, mag_w) = policy.norm_grad(*args), policy.norm_grad(*args, absolute=True)
        n = 2.5 * chain(k) + 24
        close(grad, want, n * HALF * mag + half(dtype) * abs(want), "grad")
        close(grad_weight, want_w, (60 + n) * HALF * mag_w + half(dtype) * abs(want_w), "grad_weight")


def test_norm_of_rows_that_are_zero_or_not_finite(cuda):
    """A row that holds an infinity or a NaN changes no other row, and says so; a row of zeros is zeros."""
    import int8_linear
    import rms_norm

    for k in (40, 97, 2000, 40000):
        x = normal(cuda, 6, k)
        want, want8 = rms_norm.forward(x)[0], rms_norm.forward8(x)
        bad = x.clone()
        bad[1, k // 2], bad[2, 0], bad[3, k - 1], bad[4] = float("inf"), float("nan"), -float("inf"), 0.0
        out, _ = rms_norm.forward(bad)
        assert torch.equal(out[0], want[0]) and torch.equal(out[5], want[5]) and not out[4].any()
        assert torch.isnan(out[2]).all() and torch.isnan(out[1, k // 2]) and torch.isnan(out[3, k - 1])
        codes, scale, _ = rms_norm.forward8(bad)
        for i in (0, 5):
            assert torch.equal(codes[i], want8[0][i]) and scale[i] == want8[1][i]
        assert torch.isnan(scale[1:4]).all() and scale[4] == 0 and not codes[1:5].any()
        bad[5] *= 2.0 ** -110  # too small for codes of their own
        codes, scale = int8_linear.quantise(bad)
        assert torch.isnan(scale[1:4]).all() and not scale[4:].any() and not codes[1:].any() and scale[0] > 0


@pytest.mark.parametrize("k", [8, 64, 100, 1000, 1001])
def test_norm_without_epsilon(cuda, k):
    """eps 0 is the formula too: rows that share a warp with rows past the last one are not touched by those."""
    import rms_norm

    t, g, w = normal(cuda, 1501, k), normal(cuda, 1501, k, seed=1), 1 + 0.2 * normal(cuda, k, seed=2)
    want = policy.norm(to64(t), to64(w), 0.0)
    close(rms_norm.forward(t, w, None, 0.0)[0], want, norm_tol(k, want, "f32"), "out")
    grad, grad_weight = rms_norm.backward(g, t, w, 0.0)
    args = (to64(g), to64(t), to64(w), 0.0)
    (want, want_w), (mag, mag_w) = policy.norm_grad(*args), policy.norm_grad(*args, absolute=True)
    n = 2.5 * chain(k) + 24
    close(grad, want, n * HALF * mag, "grad")
    close(grad_weight, want_w, (80 + n) * HALF * mag_w, "grad_weight")


def test_norm_without_epsilon_of_rows_near_zero(cuda):
    """What the module says of squares that float32 does not hold: NaN, infinities, and any eps ends both."""
    import rms_norm

    for k in (8, 97, 4096, 20_001):
        x = torch.zeros((3, k), device=cuda)
        x[1], x[2] = 1e-25, -1e-18
        out, _ = rms_norm.forward(x, None, None, 0.0)
        assert out[0].isnan().all() and (out[1] == torch.inf).all()
        close(out[2], np.full(k, -1.0), norm_tol(k, np.ones(k), "f32"), "out")
        out, _ = rms_norm.forward(x, None, None, 1e-30)
        assert out.isfinite().all() and not out[0].any()


def test_codes_leave_the_bytes_past_a_row(cuda):
    x = normal(cuda, 5, 21)
    room, scale = torch.full((5, 32), 99, dtype=torch.int8, device=cuda), torch.empty(5, device=cuda)
    rlenv_lib.launch(0, rlenv_lib.lib().rms_norm_codes, rlenv_lib.F32, 5, 21, x.data_ptr(), 21, 0, 0, 0, 0.0, 0,
                     room.data_ptr(), 32, scale.data_ptr(), 0)
    assert (room[:, 21:] == 99).all() and (room[:, :21].abs().amax(1) == 127).all()


def test_norm_of_no_rows(cuda):
    import int8_linear
    import rms_norm

    x, w = torch.zeros((0, 3, 8), device=cuda), torch.ones(8, device=cuda)
    out, total = rms_norm.forward(x, w, x)
    codes, scale, _ = rms_norm.forward8(x, w)
    grad, grad_weight = rms_norm.backward(x, x, w)
    assert out.shape == total.shape == grad.shape == codes.shape == (0, 3, 8) and scale.shape == (0, 3)
    assert grad_weight.shape == (8,) and not grad_weight.any()
    weight = int8_linear.quantise_weight(torch.ones((8, 5), device=cuda))
    assert int8_linear.forward(codes, scale, weight).shape == (0, 3, 5)


@pytest.mark.parametrize("with_residual", [True, False])
def test_norm_through_autograd(cuda, with_residual):
    import rms_norm

    x, y, g, gt = (normal(cuda, 5, 3, 40, seed=i) for i in range(4))
    w = 1 + 0.2 * normal(cuda, 40, seed=9)
    leaves = [v.clone().requires_grad_() for v in ((x, w, y) if with_residual else (x, w))]
    out, total = rms_norm.apply(leaves[0], leaves[1], leaves[2] if with_residual else None, 1e-5)
    grads = torch.autograd.grad((out * g).sum() + (total * gt).sum(), leaves)
    t = to64(x) + to64(y) if with_residual else to64(x)
    args = [v.reshape(15, 40) if v.size > 40 else v for v in (to64(g), t, to64(w))] + [1e-5, to64(gt).reshape(15, 40)]
    want, want_w = policy.norm_grad(*args)
    mag, mag_w = policy.norm_grad(*args, absolute=True)
    n = 2.5 * chain(40) + 28
    close(grads[0].reshape(15, 40), want, n * HALF * mag, "x")
    close(grads[1], want_w, n * HALF * mag_w, "weight")
    if with_residual:
        assert torch.equal(grads[0], grads[2])
    outs = rms_norm.apply(leaves[0], leaves[1], leaves[2] if with_residual else None, 1e-5)
    alone = torch.autograd.grad((outs[0] * g).sum(), leaves, retain_graph=True)
    want, want_w = policy.norm_grad(*args[:4])
    close(alone[0].reshape(15, 40), want, n * HALF * mag, "x without the total")
    close(alone[1], want_w, n * HALF * mag_w, "weight without the total")
    if with_residual:  # the total alone: the weight has no part in it
        alone = torch.autograd.grad((outs[1] * gt).sum(), leaves, allow_unused=True)
        assert torch.equal(alone[0], gt) and alone[1] is None and torch.equal(alone[2], gt)
    with pytest.raises(RuntimeError):
        again = torch.autograd.grad(rms_norm.apply(*leaves)[0].square().sum(), leaves[0], create_graph=True)[0]
        torch.autograd.grad(again.sum(), leaves[0])


@pytest.mark.parametrize("m,k", [(1, 8), (40, 64), (3000, 333), (500, 1001), (200, 4096), (40, 16_384), (3, 20_001)])
def test_norm_with_a_frozen_weight(cuda, m, k, monkeypatch):
    """The gradient of x is what it is beside the weight's, and nothing is done for the weight's: no room for its sums."""
    import rms_norm

    x, w, g = normal(cuda, m, k).requires_grad_(), 1 + 0.2 * normal(cuda, k, seed=1), normal(cuda, m, k, seed=2)
    both = [x, w.clone().requires_grad_()]
    want = torch.autograd.grad(rms_norm.apply(*both)[0], both, g)
    assert want[1].shape == (k,)

    def refuse(*_):
        raise AssertionError("room for sums that nobody asked for")

    monkeypatch.setattr(rlenv_lib, "scratch", refuse)
    assert torch.equal(torch.autograd.grad(rms_norm.apply(x, w)[0], x, g)[0], want[0])
    empty = x[:0].detach().requires_grad_()
    assert torch.autograd.grad(rms_norm.apply(empty, w)[0].sum(), empty)[0].shape == (0, k)


# ---- products of 8-bit integers ----------------------------------------------------------------------------

def codes(cuda, rows, cols, seed):
    import rms_norm

    g = torch.Generator(device=cuda).manual_seed(seed)
    room = rms_norm.codes_like(torch.empty((rows, cols), device=cuda), cols)
    return room.copy_(torch.randint(-128, 128, (rows, cols), generator=g, device=cuda))


def product_want(a, sa, w, sw):
    # whole numbers below 2^53 / 128^2 terms: exact in 64 bits
    return (to64(a) @ to64(w).T) * to64(sa)[..., None] * to64(sw)


PRODUCT_SIZES = [(1, 1, 1), (1, 15, 3), (1, 16, 8), (2, 17, 9), (1, 1024, 4096), (3, 1000, 100), (7, 33, 257), (8, 64, 64),
                 (9, 4097, 31), (16, 256, 512), (17, 640, 96), (33, 100, 130), (64, 2048, 100), (100, 97, 2720),
                 (128, 128, 128), (129, 129, 129), (256, 512, 256), (257, 1000, 300), (300, 1000, 2720), (511, 96, 1040),
                 (1000, 64, 17), (2050, 200, 264)]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("m,k,f", PRODUCT_SIZES)
def test_int8_product(cuda, m, k, f, dtype):
    import int8_linear

    a, w = codes(cuda, m, k, 0), codes(cuda, f, k, 1)
    sa, sw = normal(cuda, m, seed=2).abs() + 0.1, normal(cuda, f, seed=3).abs() + 0.1
    out = int8_linear.forward(a, sa, int8_linear.Weight(w, sw), TYPES[dtype])
    want = product_want(a, sa, w, sw)
    # the sum exact, its conversion and two products
    close(out, want, 3.1 * HALF * abs(want) + half(dtype) * abs(want), "out")
    assert out.dtype == TYPES[dtype] and out.shape == (m, f)
    assert torch.equal(out, int8_linear.forward(a, sa, int8_linear.Weight(w, sw), TYPES[dtype]))


@pytest.mark.parametrize("m", [1, 8, 40, 300])
def test_int8_sums_reach_the_ends_of_32_bits(cuda, m):
    import int8_linear

    k, f = int8_linear.MOST_TERMS, 5
    pitch = k + 1
    low, high = (torch.full((r, pitch), v, dtype=torch.int8, device=cuda)[:, :k] for r, v in ((m, -128), (f, 127)))
    one = torch.ones(max(m, f), device=cuda)
    assert (int8_linear.forward(low, one[:m], int8_linear.Weight(high, one[:f]), torch.float32) == -128 * 127 * k).all()
    low_w = int8_linear.Weight(torch.full((f, pitch), -128, dtype=torch.int8, device=cuda)[:, :k], one[:f])
    assert (int8_linear.forward(low, one[:m], low_w, torch.float32) == float(128 * 128 * k)).all()


@pytest.mark.parametrize("m", [1, 5, 200])
def test_int8_product_of_other_layouts(cuda, m):
    """Rows off the boundaries, expanded and transposed ones, leading axes: the results of their copies."""
    import int8_linear

    g = torch.Generator(device=cuda).manual_seed(0)
    a = torch.randint(-128, 128, (m, 3, 50), generator=g, device=cuda).to(torch.int8)
    w = torch.randint(-128, 128, (40, 70), generator=g, device=cuda).to(torch.int8)
    sa, sw = normal(cuda, m, 6, seed=1)[:, ::2], normal(cuda, 40, seed=2)
    for x, y in ((a, w[:, :50]), (a, w[:, 7:57]), (a[:, :1].expand(m, 3, 50), w.t()[:50].t()), (a[..., 1:34], w[:, 16:49]),
                 (a.flip(0), w[:, :50].contiguous())):
        out = int8_linear.forward(x, sa, int8_linear.Weight(y, sw), torch.float32)
        want = product_want(x, sa, y, sw)
        close(out, want, 3.1 * HALF * abs(want), "out")


def test_a_layer_in_8_bits(cuda):
    """Norm, codes and product as a policy that acts in 8 bits runs them, against the same from the definitions: the
    codes' rounding is the largest error, half a step of each term."""
    import int8_linear
    import rms_norm

    for m, k, f in ((1, 64, 192), (33, 100, 70), (500, 1000, 2720)):
        x, y, w = normal(cuda, m, k), normal(cuda, m, k, seed=1), normal(cuda, k, f, seed=2, scale=k ** -0.5)
        weight = int8_linear.quantise_weight(w)
        assert weight.codes.shape == (f, k) and weight.scale.shape == (f,)
        w64 = to64(w)
        close(weight.codes * weight.scale[:, None], w64.T, (0.5 + 1e-4) * abs(w64).max(0)[:, None] / 127, "weight")
        got = int8_linear.forward(*rms_norm.forward8(x, None, y)[:2], weight, torch.float32)
        v = policy.norm(to64(x) + to64(y), None, 1e-6)
        step, wstep = abs(v).max(1, keepdims=True) / 127, abs(w64).max(0) / 127
        # |v w - v' w'| <= |v - v'| |w| + |v'| |w - w'|
        tol = 0.5 * step * abs(w64).sum(0) + 0.5 * (abs(v) + 0.5 * step).sum(1, keepdims=True) * wstep
        close(got, v @ w64, 1.001 * tol, "layer")
        assert torch.equal(int8_linear.product(x, weight), int8_linear.forward(*int8_linear.quantise(x), weight, x.dtype))


def test_int8_refusals(cuda):
    import int8_linear

    a, w, one = codes(cuda, 4, 20, 0), codes(cuda, 6, 20, 1), torch.ones(6, device=cuda)
    fine = int8_linear.Weight(w, one)
    for args in ((a.float(), one[:4], fine), (a, one[:3], fine), (a[:, :19], one[:4], fine), (a, one[:4].double(), fine),
                 (a, one[:4], int8_linear.Weight(w, one[:5])), (a, one[:4], int8_linear.Weight(w.float(), one)),
                 (a, one[:4], fine, torch.float16), (a, one[:4].cpu(), fine), (a, one[:4], None), (a, one[:4], (w, one)), (a[:, :0], one[:4], int8_linear.Weight(w[:, :0], one))):
        with pytest.raises(ValueError):
            int8_linear.forward(*args)
    with pytest.raises(ValueError):
        int8_linear.quantise_weight(torch.ones(3, device=cuda))
    with pytest.raises(ValueError, match="K must be"):
        big = torch.zeros((1, 131072), dtype=torch.int8, device=cuda)
        int8_linear.forward(big, one[:1], int8_linear.Weight(big, one[:1]))


# ---- scores -------------------------------------------------------------------------------------------------

def score_inputs(cuda, m, v, dtype, beside=0, masked=False, seed=0):
    l = normal(cuda, m, v + beside, seed=seed, scale=2.0, dtype=dtype)[:, :v]
    g = torch.Generator(device=cuda).manual_seed(seed + 1)
    allowed = torch.rand((m, v), generator=g, device=cuda) < 0.6 if masked else None
    actions = torch.randint(0, v, (m,), generator=g, device=cuda)
    if masked:
        allowed[torch.arange(m, device=cuda), actions] = True
        if m > 2:
            allowed[1] = False
    return l, actions, allowed


def score_bounds(l, allowed, v):
    """Of (log_prob's and the normalizer's, the entropy's) errors, but for log_prob's last subtraction."""
    e64 = np.where(allowed, l, -np.inf) if allowed is not None else l
    with np.errstate(all="ignore"):
        _, h, z, lp = policy.scores(l, np.zeros(l.shape[0], np.int64), allowed)
        top = e64.max(-1, keepdims=True)
        p, d = np.exp(lp), np.where(e64 > -np.inf, e64 - np.where(top > -np.inf, top, 0), 0)
        one, two = (p * -d).sum(-1), (p * d * d).sum(-1)  # means of |d| and d^2
        n = chain(v)
        sums = (n + 6) * 2 ** -23 + (2.4 * one) * 2 ** -23       # of log S
        z_off = sums + 2 ** -23 * (abs(z) + abs(np.log(v)))
        h_off = sums * (1 + one) + ((n + 8) * one + 2.4 * two) * 2 ** -23 + 2 ** -22 * (one + np.log(v) + 1)
    return np.where(np.isfinite(z), z_off, 0), np.where(np.isfinite(z), h_off, 0)


def check_scores(got, l, actions, allowed, top):
    l64, a = to64(l), actions.cpu().numpy().astype(np.int64)
    al = None if allowed is None else allowed.cpu().numpy() != 0
    lp, h, z, every = policy.scores(l64, a, al)
    z_off, h_off = score_bounds(l64, al, l64.shape[1])
    close(got.normalizer, z, z_off, "normalizer")
    close(got.entropy, h, h_off, "entropy")
    last = HALF * abs(np.where(np.isfinite(lp), lp, 0)) + 2 ** -23
    close(got.log_prob, lp, z_off + last, "log_prob")
    if top:
        best = policy.best(l64, top, al)
        assert got.top_actions.dtype == torch.int64
        assert np.array_equal(got.top_actions.cpu().numpy(), best), "top_actions"
        want = np.take_along_axis(every, best, -1)
        close(got.top_log_probs, want, z_off[:, None] + HALF * abs(np.where(np.isfinite(want), want, 0)) + 2 ** -23, "top_log_probs")
    else:
        assert got.top_actions is None and got.top_log_probs is None


SCORE_SIZES = [(1, 1), (5, 2), (300, 3), (7, 8), (5, 9), (4, 16), (9, 17), (6, 33), (5, 64), (3, 65), (4, 255), (3, 256),
               (9, 257), (5, 300), (3, 513), (4, 1000), (9, 1025), (3, 2047), (2, 2049), (3, 5000), (2, 8193), (1, 9001),
               (2, 32768), (1, 50021), (400, 4100), (1, 131071)]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("m,v", SCORE_SIZES)
def test_scores(cuda, m, v, dtype):
    import log_probs

    for beside, masked, top in ((0, False, min(v, 8)), (1, True, min(v, 32)), (0, True, 0), (3, False, 1)):
        l, actions, allowed = score_inputs(cuda, m, v, dtype, beside, masked, seed=beside)
        check_scores(log_probs.forward(l, actions, allowed, top), l, actions, allowed, top)


@pytest.mark.parametrize("m,v,dtype", [(1, 300_001, "bf16"), (2, 150_001, "f32"), (200, 40_000, "f32"), (700, 70_000, "bf16")])
def test_scores_of_long_rows(cuda, m, v, dtype):
    """Rows that registers do not hold, alone and with their clusters over all of the GPU."""
    import log_probs

    l, actions, allowed = score_inputs(cuda, m, v, dtype, masked=m < 10)
    check_scores(log_probs.forward(l, actions, allowed, 20), l, actions, allowed, 20)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("v", [5, 40, 200, 700, 1500, 6000, 20_000, 60_000, 140_000])
def test_alternatives_of_equal_logits(cuda, v, dtype):
    """Rows of one value, of two, of steps up and down, of both zeros, and the largest all in one thread's reach: ties go
    to the lower action however many there are."""
    import log_probs

    top = min(v, 32)
    l = torch.zeros((9, v), device=cuda)
    l[1] = torch.arange(v, device=cuda) % 2
    l[2] = torch.arange(v, device=cuda) // 100
    l[3] = -l[2]
    l[4, ::2] = -0.0
    l[5, v // 2:] = 3.0
    l[6, ::512 * 8] = 5.0
    l[7, -1] = 1.0
    l[8] = -torch.inf
    l[8, v // 3] = -4.0
    l = l.to(TYPES[dtype])
    actions = torch.zeros(9, dtype=torch.int32, device=cuda)
    check_scores(log_probs.forward(l, actions, None, top), l, actions, None, top)
    allowed = torch.ones((9, v), dtype=torch.uint8, device=cuda) * 3
    allowed[:, 1::3] = 0
    check_scores(log_probs.forward(l, actions, allowed, top), l, actions, allowed, top)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("m", [5, 8192, 8193])
def test_scores_at_the_borders_between_forms(cuda, m, dtype):
    """Rows of lanes' single values, by a few lanes or a warp, and the first of the longer ones, few rows and many: the
    last team of a block's is not full. Rows repeat; those that start alike on the boundaries of 16 bytes, eight
    repetitions further on, are the same bit for bit, and the first eight repetitions are checked."""
    import log_probs

    for v in (8, 9, 32, 33, 64, 65, 127, 128, 129, 255, 256, 257, 511, 512, 513, 1023, 1024, 1025):
        some = min(m, 37)
        l, actions, allowed = score_inputs(cuda, some, v, dtype, v % 2, v % 3 > 0, seed=v)
        every, again = torch.arange(m, device=cuda) % some, torch.arange(m, device=cuda) % (8 * some)
        many = torch.full((m, v + 3), 7.0, dtype=l.dtype, device=cuda)[:, :v].copy_(l[every])
        al = None if allowed is None else allowed[every]
        for top in sorted({0, 1, min(v, 9), min(v, 32)}):
            got = log_probs.forward(many, actions[every], al, top)
            for n in range(0, min(m, 8 * some), some):
                check_scores(log_probs.Scores(*(None if x is None else x[n:n + some] for x in got)), l, actions, allowed, top)
            for x in got:
                assert x is None or torch.equal(x.nan_to_num(), x[again].nan_to_num())
        g, h = normal(cuda, some, seed=2), normal(cuda, some, seed=3)
        for logits in (many, many.contiguous()):
            grad = log_probs.backward(g[every], h[every], logits, actions[every], got.normalizer, got.entropy, al)
            first = log_probs.backward(g, h, l, actions, got.normalizer[:some], got.entropy[:some], allowed)
            # forms differ by an instruction's rounding of a power's argument, one of each of the sums of two
            assert (grad[:some].double() - first.double()).abs().max() <= 2 * torch.finfo(l.dtype).eps * max(1.0, first.double().abs().max())
            assert torch.equal(grad.nan_to_num(), grad[again].nan_to_num())


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("v", [8, 16, 31, 60, 128, 250, 500, 1000, 1500, 5000, 40_000, 140_000])
def test_alternatives_where_logits_are_not_numbers(cuda, v, dtype):
    """NaN is above all logits, and ties go to the lower action, also where a row is nothing but NaN."""
    import log_probs

    top = min(v, 32)
    l = normal(cuda, 4, v).to(TYPES[dtype])
    l[0] = torch.nan
    l[1, :] = -torch.inf
    l[1, v // 2:] = torch.nan
    l[2, -1] = torch.nan
    for m in (4, 10_000):
        if m * v > 2 ** 25:
            continue
        rows = l[torch.arange(m, device=cuda) % 4]
        got = log_probs.forward(rows, torch.zeros(m, dtype=torch.int32, device=cuda), None, top)
        above = torch.where(l.isnan(), torch.inf, l.float())
        want = above.cpu().sort(dim=-1, descending=True, stable=True).indices[:, :top]
        assert torch.equal(got.top_actions[:4].cpu(), want) and torch.equal(got.top_actions, got.top_actions[:4].repeat(m // 4, 1))
        assert got.top_log_probs[:3].isnan().all() and got.top_log_probs[3].isfinite().all()


@pytest.mark.parametrize("v", [2, 30, 100, 400, 1200, 3000, 20_000, 70_000])
def test_scores_where_rows_are_odd(cuda, v):
    """Padding, actions outside, rows that allow nothing, logits that are not finite in and out of masked places: each
    row as documented and no other changed."""
    import log_probs

    l, actions, _ = score_inputs(cuda, 12, v, "f32")
    clean = log_probs.forward(l, actions, None, 2)
    allowed = torch.ones((12, v), dtype=torch.bool, device=cuda)
    bad, a = l.clone(), actions.clone()
    a[1], a[2] = -1, v
    allowed[3] = False
    bad[4, v // 2] = torch.nan
    bad[5, 0] = torch.inf
    bad[6, v - 1], allowed[6, v - 1], a[6] = torch.nan, False, 0
    bad[7, v - 1], allowed[7, v - 1], a[7] = torch.inf, False, v - 1
    bad[8, v - 1], a[8] = -torch.inf, v - 1
    bad[9] = torch.finfo(torch.float32).min
    got = log_probs.forward(bad, a, allowed, 2)
    for i in (0, 10, 11):
        assert all(x[i].equal(y[i]) for x, y in zip(got, clean))
    assert got.log_prob[1] == 0 and torch.isnan(got.log_prob[2])
    assert got.entropy[1] == clean.entropy[1] and got.entropy[2] == clean.entropy[2]
    assert got.normalizer[3] == -torch.inf and got.log_prob[3] == -torch.inf and got.entropy[3] == 0
    assert got.top_actions[3].tolist() == [0, 1] and (got.top_log_probs[3] == -torch.inf).all()
    for i in (4, 5):
        assert all(torch.isnan(x[i]) for x in (got.log_prob, got.entropy, got.normalizer))
    assert got.top_actions[4, 0] == v // 2 and got.top_actions[5, 0] == 0
    rest = l[6:8].clone()
    rest[:, v - 1] = -torch.inf
    check_scores(log_probs.Scores(*(x[6:9] for x in got)), torch.cat([rest, bad[8:9]]), a[6:9], None, 2)
    want = -np.log(v)
    assert abs(got.log_prob[9].item() - want) <= 2.0 ** 104 and abs(got.entropy[9].item() + want) < 1e-4
    g, h = normal(cuda, 12, seed=5), normal(cuda, 12, seed=6)
    grad = log_probs.backward(g, h, bad, a, got.normalizer, got.entropy, allowed)
    ref = log_probs.backward(g, h, l, actions, clean.normalizer, clean.entropy)
    for i in (0, 10, 11):
        assert torch.equal(grad[i], ref[i])
    assert torch.equal(grad[1], log_probs.backward(None, h, l, actions, clean.normalizer, clean.entropy)[1])
    assert torch.isnan(grad[2]).all() and not grad[3].any()
    assert torch.isnan(grad[4]).any() and torch.isnan(grad[5]).any()
    assert not grad[6:9, v - 1].any() and torch.isfinite(grad[6:9]).all()


def test_the_check_build_reports_actions_outside(cuda):
    import ctypes

    lib = ctypes.CDLL(str(rlenv_lib.CHECKS_LIB_PATH))
    for name in ("rlenv_log_probs_forward", "rlenv_log_probs_backward", "rlenv_checks_status"):
        getattr(lib, name).argtypes = rlenv_lib._SIGNATURES[name]
    word = ctypes.c_uint(0)
    for v in (5, 100, 3000):
        l, out = normal(cuda, 4, v), torch.empty((3, 4), device=cuda)
        for last, want in ((v - 1, 0), (v, 1)):
            actions = torch.tensor([0, -1, 1, last], device=cuda)
            assert lib.rlenv_checks_status(ctypes.byref(word), 1) == 0
            assert lib.rlenv_log_probs_forward(rlenv_lib.F32, 4, v, l.data_ptr(), v, actions.data_ptr(), rlenv_lib.I64, 0, 0,
                                               out[0].data_ptr(), out[1].data_ptr(), out[2].data_ptr(), 0, 0, 0, 0) == 0
            torch.cuda.synchronize()
            assert lib.rlenv_checks_status(ctypes.byref(word), 1) == 0 and word.value & 1 == want
            assert lib.rlenv_log_probs_backward(rlenv_lib.F32, 4, v, out[0].data_ptr(), 0, l.data_ptr(), v,
                                                actions.data_ptr(), rlenv_lib.I64, out[2].data_ptr(), out[1].data_ptr(), 0, 0,
                                                l.data_ptr(), 0) == 0
            torch.cuda.synchronize()
            assert lib.rlenv_checks_status(ctypes.byref(word), 1) == 0 and word.value & 1 == want


@pytest.mark.parametrize("m,v", [(4, 1500), (700, 3000), (3000, 9000), (600, 20_000), (4, 30_000), (1, 140_000)])
def test_alternatives_whose_list_is_shortened_often(cuda, m, v):
    """Rows that rise, fall, or rise in stretches of a lane's reach, by a warp, a block and a cluster: far more logits reach
    the list of alternatives than it holds, again and again. Called over and over, always the same."""
    import log_probs

    at = torch.arange(v, device=cuda, dtype=torch.float32)
    rows = torch.stack([at, -at, at % 1024, at // 8 % 64 * 8 + at % 8])
    want = torch.tensor(np.stack([policy.best(to64(rows), 32)]), device=cuda)[0]
    which = torch.arange(m, device=cuda) % 4
    l, actions = rows[which], torch.zeros(m, dtype=torch.int64, device=cuda)
    for top in (32, 5, 32, 5):
        got = log_probs.forward(l, actions, None, top)
        assert torch.equal(got.top_actions, want[which, :top])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("v", [7, 60, 250, 400, 1500, 5000, 40_000, 140_000])
def test_scores_of_rows_that_grow(cuda, v, dtype):
    """Rows whose largest logits come late, by steps and at once, after the type's lowest value too: the sums' base moves,
    and stands 20 below the largest logit at most, so that a sum's error counts up to 20 times in the entropy."""
    import log_probs

    low = torch.finfo(TYPES[dtype]).min
    l = normal(cuda, 8, v, seed=3)
    l[1] = torch.arange(v, device=cuda) * (300.0 / v)
    l[2] = -l[1]
    l[3] = torch.arange(v, device=cuda) // (v // 3) * 19.0
    l[4, -1] = 1e4
    l[5, : v // 2] = low
    l[6, :-1] = low
    l[7] = low
    l = l.to(TYPES[dtype])
    actions = torch.full((8,), v - 1, device=cuda)
    got = log_probs.forward(l, actions, None, 5)
    l64 = to64(l)
    lp, h, z, every = policy.scores(l64, actions.cpu().numpy())
    z_off, h_off = score_bounds(l64, None, v)
    extra = (chain(v) + 8) * 20 * 2 ** -23
    close(got.normalizer, z, z_off + extra, "normalizer")
    close(got.entropy, h, h_off + extra, "entropy")
    close(got.log_prob, lp, z_off + extra + HALF * abs(lp) + 2 ** -23, "log_prob")
    assert np.array_equal(got.top_actions.cpu().numpy(), policy.best(l64, 5))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("m,v", [(64, 60), (64, 1000), (64, 1500), (700, 3000), (3000, 9000), (64, 16_384), (400, 20_000), (2, 60_000), (1, 140_000)])
def test_the_entropy_of_rows_whose_largest_logit_is_the_last(cuda, m, v, dtype):
    """A policy that has learnt what to do: one logit 17 to 21 above ones of order one, so that the entropy is 1e-2 to 1e-5
    and the sum S is the one term. Against a base that lies close to it S is 1 and what a bit more, and so are the numbers that
    are rounded: once where the last logit is added, once for its lane, at most five times among lanes, four among warps and three
    among blocks. The others' part of S, and of the entropy, has its usual error in proportion to it."""
    import log_probs

    l = normal(cuda, m, v, seed=9).clamp(-4, 4)
    l[:, -1] = torch.linspace(17, 21, m, device=cuda)
    l = l.to(TYPES[dtype])
    got = log_probs.forward(l, torch.full((m,), v - 1, device=cuda))
    l64 = to64(l)
    lp, h, z, every = policy.scores(l64, np.full(m, v - 1))
    others = 1 - np.exp(lp)
    tol = 15 * HALF + others * (chain(v) + 20) * 26 * 2 ** -23  # 26: the others lie up to 25 below
    close(got.entropy, h, tol, "entropy")
    close(got.log_prob, lp, tol, "log_prob")


FAR = [("f32", 1024.0, 0.125), ("f32", 2.0 ** 17, 0.125), ("f32", 2.0 ** 24, 2.0), ("f32", -2.0 ** 24, 2.0),
       ("bf16", 1024.0, 8.0), ("bf16", -2.0 ** 17, 1024.0), ("bf16", 2.0 ** 24, 2.0 ** 17), ("f32", None, 0.0), ("bf16", None, 0.0)]


def far_logits(cuda, m, v, dtype, shift, unit, seed=0):
    """(logits that have `shift` in common, the same without it): whole units, exact in the type. None: its lowest value."""
    g = torch.Generator(device=cuda).manual_seed(seed)
    near = torch.randint(-20, 1, (m, v), generator=g, device=cuda).float() * unit
    near[:, v // 2] = 0.0
    far = (near + (torch.finfo(TYPES[dtype]).min if shift is None else shift)).to(TYPES[dtype])
    assert shift is None or torch.equal(far.double() - shift, near.double())
    return far, near


@pytest.mark.parametrize("dtype,shift,unit", FAR)
@pytest.mark.parametrize("m,v", [(9, 7), (9, 31), (5, 60), (8300, 60), (4, 250), (3, 700), (5, 1500), (700, 3000), (2, 30_000), (1, 140_000)])
def test_scores_of_rows_far_from_zero(cuda, m, v, dtype, shift, unit):
    """What a row's logits have in common changes neither its log-probabilities nor its entropy, nor how precise they are:
    the bounds are those of the rows without it."""
    import log_probs

    far, near = far_logits(cuda, m, v, dtype, shift, unit)
    actions = torch.arange(m, device=cuda) % v
    got = log_probs.forward(far, actions, None, min(v, 4))
    l64, some = to64(near[:50]), slice(0, 50)
    lp, h, z, every = policy.scores(l64, to64(actions[:50]).astype(np.int64))
    z_off, h_off = score_bounds(l64, None, v)
    close(got.log_prob[some], lp, z_off + HALF * abs(lp) + 2 ** -23, "log_prob")
    close(got.entropy[some], h, h_off, "entropy")
    want = np.take_along_axis(every, policy.best(l64, min(v, 4)), -1)
    close(got.top_log_probs[some], want, z_off[:, None] + HALF * abs(want) + 2 ** -23, "top_log_probs")
    z = z + (torch.finfo(TYPES[dtype]).min if shift is None else shift)
    close(got.normalizer[some], z, z_off + 2 * HALF * abs(z), "normalizer")


def grad_tol(g, h, l, actions, allowed, dtype):
    lp, entropy, z, every = policy.scores(l, actions, allowed)
    z_off, h_off = score_bounds(l, allowed, l.shape[1])
    with np.errstate(all="ignore"):
        some = every > -np.inf
        p, lp = np.where(some, np.exp(every), 0), np.where(some, every, 0)
        lp_off = z_off[:, None] + HALF * abs(lp) + 2 ** -23
        rel = lp_off + (2 + 1.2 * abs(lp)) * 2 ** -23  # of p
        far = abs(lp) > 80  # e^-87 is below float32's normal numbers
    want = policy.scores_grad(g, h, l, actions, allowed)
    inner = abs(lp + entropy[:, None])
    tol = abs(g)[:, None] * (p * rel + HALF * (p + (p > 0.1)) + 2 * HALF * abs(1 - p) * (p > 0.5)) \
        + abs(h)[:, None] * p * (inner * (rel + 4 * HALF) + lp_off + h_off[:, None]) + 4 * HALF * abs(want) \
        + (abs(g) + 90 * abs(h))[:, None] * (far * 2.0 ** -110 + 2.0 ** -125)
    chosen = np.arange(l.shape[1]) == actions[:, None]
    return want, tol + chosen * abs(g)[:, None] * 2 * HALF + half(dtype) * abs(want)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("m,v", SCORE_SIZES)
def test_scores_gradient(cuda, m, v, dtype):
    import log_probs

    for beside, masked in ((0, False), (1, True), (0, True), (3, False)):
        l, actions, allowed = score_inputs(cuda, m, v, dtype, beside, masked, seed=7 + beside)
        if m > 3:
            actions[3] = -1
        s = log_probs.forward(l, actions, allowed)
        g, h = normal(cuda, m, seed=5), normal(cuda, m, seed=6)
        a, al = actions.cpu().numpy(), None if allowed is None else allowed.cpu().numpy()
        for gg, hh in ((g, h), (None, h), (g, None), (None, None)):
            grad = log_probs.backward(gg, hh, l, actions, s.normalizer, s.entropy, allowed)
            zero = np.zeros(m)
            want, tol = grad_tol(zero if gg is None else to64(gg), zero if hh is None else to64(hh), to64(l), a, al, dtype)
            close(grad, want, tol, "grad")
            assert grad.dtype == l.dtype and grad.is_contiguous()


@pytest.mark.parametrize("dtype,shift,unit", FAR)
@pytest.mark.parametrize("m,v", [(9, 7), (5, 60), (8300, 60), (4, 250), (3, 700), (5, 1500), (2, 30_001), (1, 140_000)])
def test_scores_gradient_of_rows_far_from_zero(cuda, m, v, dtype, shift, unit):
    """The gradient of rows that have much in common is that of the rows without it, in its precision too, by the
    remainder of the normalizer's rounding: rows that lie as the gradient's do on the boundaries and others."""
    import log_probs

    far, near = far_logits(cuda, m, v + 1, dtype, shift, unit)
    actions = torch.arange(m, device=cuda) % v
    actions[m // 2] = -1
    g, h = normal(cuda, m, seed=5), normal(cuda, m, seed=6)
    n = min(m, 50)
    want, tol = grad_tol(to64(g[:n]), to64(h[:n]), to64(near[:n, :v]), to64(actions[:n]).astype(np.int64), None, dtype)
    for l in (far[:, :v], far[:, :v].contiguous()):
        s = log_probs.forward(l, actions, remainder=True)
        z = policy.scores(to64(near[:n, :v]), np.zeros(n, np.int64))[2]
        left = (to64(s.normalizer[:n]) - (torch.finfo(TYPES[dtype]).min if shift is None else shift)) + to64(s.remainder[:n])
        assert (abs(left - z) <= score_bounds(to64(near[:n, :v]), None, v)[0]).all()
        grad = log_probs.backward(g, h, l, actions, s.normalizer, s.entropy, None, s.remainder)
        close(grad[:n], want, tol, "grad")
        leaf = l.detach().clone().requires_grad_()
        both = torch.autograd.grad(log_probs.apply(leaf, actions), leaf, (g, h))[0]
        close(both[:n], want, tol, "apply's gradient")


def test_a_normalizers_remainder(cuda):
    """It is asked for, is no item of the tuple, and is 0 where the normalizer is not finite; what does not fit is refused."""
    import log_probs

    l, a = normal(cuda, 6, 5), torch.zeros(6, dtype=torch.int64, device=cuda)
    l[1], l[2, 0], l[3, 1] = -torch.inf, torch.nan, torch.inf
    s = log_probs.forward(l, a)
    assert s.remainder is None and len(s) == 5
    s = log_probs.forward(l, a, None, 2, remainder=True)
    log_prob, entropy, normalizer, top, best = s
    assert s.remainder.shape == (6,) and not s.remainder[1:4].any() and s.remainder[[0, 4, 5]].abs().max() <= HALF * 8
    assert not log_probs.backward(log_prob, entropy, l, a, normalizer, entropy, None, s.remainder)[1].any()
    for bad in (s.remainder[:5], s.remainder.double(), s.remainder.cpu(), 0.0):
        with pytest.raises(ValueError):
            log_probs.backward(log_prob, None, l, a, normalizer, entropy, None, bad)


@pytest.mark.parametrize("kind", [torch.int64, torch.int32, torch.uint8])
def test_scores_through_autograd(cuda, kind):
    """The loss of an actor: log_prob and entropy, their gradient against the oracle's; leading axes, a slice."""
    import log_probs

    l = normal(cuda, 6, 5, 10, scale=2.0).requires_grad_()
    actions = torch.randint(0, 9, (6, 5), device=cuda).to(kind)
    allowed = torch.rand((6, 1, 9), device=cuda) < 0.8
    allowed[..., 0] = True
    allowed = allowed.expand(6, 5, 9)
    g = normal(cuda, 6, 5, seed=3)
    lp, entropy = log_probs.apply(l[..., :9], actions, allowed)
    chosen = allowed.gather(-1, actions.long()[..., None])[..., 0]
    loss = (g * torch.where(chosen, lp, 0.0)).sum() + 0.3 * entropy.sum()
    grad, = torch.autograd.grad(loss, l)
    assert not grad[..., 9].any()
    g64 = np.where(chosen.cpu().numpy(), to64(g), 0.0).reshape(30)
    want, tol = grad_tol(g64, np.full(30, 0.3), to64(l)[..., :9].reshape(30, 9), actions.long().cpu().numpy().reshape(30),
                         allowed.cpu().numpy().reshape(30, 9), "f32")
    close(grad[..., :9].reshape(30, 9), want, tol, "grad")
    alone, = torch.autograd.grad(0.3 * log_probs.apply(l[..., :9], actions, allowed)[1].sum(), l)
    want, tol = grad_tol(np.zeros(30), np.full(30, 0.3), to64(l)[..., :9].reshape(30, 9),
                         actions.long().cpu().numpy().reshape(30), allowed.cpu().numpy().reshape(30, 9), "f32")
    close(alone[..., :9].reshape(30, 9), want, tol, "the entropy's gradient alone")


def test_scores_of_no_rows_and_refusals(cuda):
    import log_probs

    l, a = torch.zeros((0, 4, 7), device=cuda), torch.zeros((0, 4), dtype=torch.int64, device=cuda)
    s = log_probs.forward(l, a, None, 3)
    assert s.log_prob.shape == (0, 4) and s.top_actions.shape == (0, 4, 3)
    assert log_probs.backward(s.log_prob, None, l, a, s.normalizer, s.entropy).shape == l.shape
    l, a = torch.zeros((3, 7), device=cuda), torch.zeros(3, dtype=torch.int64, device=cuda)
    for args in ((l, a.float()), (l, a[:2]), (l.double(), a), (l, a, torch.ones((3, 6), dtype=torch.bool, device=cuda)),
                 (l, a, l), (l, a, None, 8), (l, a, None, -1), (l[:, :0], a), (l, a.cpu()), (l, None), (l.half(), a),
                 (torch.zeros((3, 99), device=cuda), a, None, 33)):
        with pytest.raises(ValueError):
            log_probs.forward(*args)
    s = log_probs.forward(l, a)
    for args in ((s.log_prob.double(), None, l, a, s.normalizer, s.entropy), (None, None, l, a, None, s.entropy),
                 (None, None, l, a, s.normalizer[:2], s.entropy), (s.log_prob.cpu(), None, l, a, s.normalizer, s.entropy)):
        with pytest.raises(ValueError):
            log_probs.backward(*args)


def test_scores_of_2_to_the_26_rows(cuda):
    """A million environments' 64 steps and some more, with masks and alternatives and their gradient: rows repeat, and each
    is what it is among a few."""
    import log_probs

    some, m = 1 << 12, (65 << 20) + 77
    every = torch.arange(m, device=cuda) % some
    allowed = torch.rand((some, 2), device=cuda) < 0.8
    for l, mask in ((normal(cuda, some, 2, scale=2.0), None), (normal(cuda, some, 2, seed=1).bfloat16(), allowed)):
        actions = torch.randint(-1, 2, (some,), device=cuda).to(torch.int32)
        g, h = normal(cuda, some, seed=2), normal(cuda, some, seed=3)
        few = log_probs.forward(l, actions, mask, 2, remainder=True)
        grad = log_probs.backward(g, h, l, actions, few.normalizer, few.entropy, mask, few.remainder)
        many, acts, masks = l[every], actions[every], None if mask is None else mask[every]
        got = log_probs.forward(many, acts, masks, 2, remainder=True)
        for x, y in zip((*got, got.remainder), (*few, few.remainder)):
            assert torch.equal(x, y[every])
        out = log_probs.backward(g[every], h[every], many, acts, got.normalizer, got.entropy, masks, got.remainder)
        assert torch.equal(out, grad[every])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("v", [5, 60, 250, 700, 1500, 30_001])
def test_gradients_of_rows_that_are_not_numbers(cuda, v, dtype):
    """A row with an action past the last one or a NaN among its allowed logits is NaN throughout, places that are not
    allowed too; one that allows nothing is zeros whatever its action; none changes another."""
    import log_probs

    l, actions, _ = score_inputs(cuda, 6, v, dtype)
    g, h = normal(cuda, 6, seed=5), normal(cuda, 6, seed=6)
    allowed = torch.ones((6, v), dtype=torch.bool, device=cuda)
    allowed[:, v // 2], actions[:] = False, 0
    clean = log_probs.forward(l, actions, allowed)
    want = log_probs.backward(g, h, l, actions, clean.normalizer, clean.entropy, allowed)
    a, bad = actions.clone(), l.clone()
    a[1], a[2], a[3], bad[4, 1] = v, v + 7, v, torch.nan
    allowed[2:4] = False
    s = log_probs.forward(bad, a, allowed, remainder=True)
    assert s.log_prob[1:5].isnan().all() and (s.normalizer[2:4] == -torch.inf).all()
    for rest in (None, s.remainder):
        grad = log_probs.backward(g, h, bad, a, s.normalizer, s.entropy, allowed, rest)
        assert grad[1].isnan().all() and grad[4].isnan().all() and not grad[2:4].any()
    grad = log_probs.backward(g, h, bad, a, s.normalizer, s.entropy, allowed)
    assert torch.equal(grad[0], want[0]) and torch.equal(grad[5], want[5])
    s = log_probs.forward(l, a, allowed)  # without an upstream gradient of log_prob too
    assert log_probs.backward(None, h, l, a, s.normalizer, s.entropy, allowed)[1].isnan().all()


# ---- streams and graphs ---------------------------------------------------------------------------------------

def test_operators_in_a_captured_graph_and_on_other_streams(cuda):
    """Everything once eagerly, then on a side stream, then captured and replayed on new inputs, two graphs' replays
    interleaved: the same bits."""
    import int8_linear
    import log_probs
    import rms_norm

    def inputs(seed):
        return [normal(cuda, 300, 96, seed=seed), normal(cuda, 300, 96, seed=seed + 1), normal(cuda, 300, 700, seed=seed + 2),
                normal(cuda, 3, 90_001, seed=seed + 3), normal(cuda, 200, 6000, seed=seed + 4)]

    w, weight = 1 + 0.1 * normal(cuda, 96, seed=50), int8_linear.quantise_weight(normal(cuda, 96, 300, seed=51))
    actions, long_weight = torch.arange(300, device=cuda), int8_linear.quantise_weight(normal(cuda, 6000, 40, seed=52))

    def everything(x, y, l, few, wide):
        out, total = rms_norm.forward(x, w, y)
        c, s, _ = rms_norm.forward8(x, w, y)
        got = log_probs.forward(l, actions, None, 4)
        return [out, total, c, s, *rms_norm.backward(x, total, w, 1e-6, y), int8_linear.forward(c, s, weight),
                int8_linear.forward(c[:3], s[:3], weight), *got, *log_probs.forward(few, actions[:3], None, 4),
                int8_linear.product(wide, long_weight), *rms_norm.backward(wide, wide, wide[0]),
                log_probs.backward(got.log_prob, got.entropy, l, actions, got.normalizer, got.entropy)]

    first, second = inputs(0), inputs(10)
    want = [everything(*first), everything(*second)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = everything(*first)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(other, want[0]))
    graphs, outs, rooms = [], [], []
    for _ in range(2):
        room = [x.clone() for x in first]
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(everything(*room))
        graphs.append(graph)
        rooms.append(room)
    for order in ((0, 1), (1, 0)):
        for which in (0, 1):
            for to, x in zip(rooms[which], (first, second)[order[which]]):
                to.copy_(x)
        graphs[0].replay()
        graphs[1].replay()
        torch.cuda.synchronize()
        for which in (0, 1):
            assert all(torch.equal(a, b) for a, b in zip(outs[which], want[order[which]]))


def test_gradients_in_a_captured_graph(cuda):
    """The norm and the scores through autograd, captured with their backward pass and replayed on other inputs: what the
    same steps give eagerly. No eager graph of the same leaves lives meanwhile, which torch asks for."""
    import log_probs
    import rms_norm

    def inputs(seed):
        return [normal(cuda, 300, 96, seed=seed), 1 + 0.1 * normal(cuda, 96, seed=seed + 1), normal(cuda, 300, 96, seed=seed + 2)]

    actions = torch.arange(300, device=cuda) % 96
    leaves = [v.requires_grad_() for v in inputs(0)]

    def grads():
        out, total = rms_norm.apply(*leaves)
        log_prob, entropy = log_probs.apply(out, actions)
        return torch.autograd.grad(log_prob.mean() + 0.1 * entropy.mean() + total.square().mean(), leaves)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        grads()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = grads()
    for seed in (10, 0):
        with torch.no_grad():
            for leaf, v in zip(leaves, inputs(seed)):
                leaf.copy_(v)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, grads()))


def test_offsets_past_32_bits(cuda):
    """Tensors of more than 2^31 and 2^32 elements: rows around those places and the last ones are what the same rows
    alone give."""
    import int8_linear
    import log_probs
    import rms_norm

    m, k = 4_300_000, 1000
    x, w = torch.empty((m, k), dtype=torch.bfloat16, device=cuda).normal_(), torch.ones(k, dtype=torch.bfloat16, device=cuda)
    weights = [int8_linear.quantise_weight(normal(cuda, k, f, seed=f)) for f in (1000, 1001)]
    out, _ = rms_norm.forward(x, w)
    codes, scale, _ = rms_norm.forward8(x, w)
    grad, _ = rms_norm.backward(x, x, w)
    products = [int8_linear.forward(codes, scale, weight) for weight in weights]
    places = [slice(at, at + 40) for at in (2 ** 31 // k - 20, 2 ** 32 // k - 20, m - 40)]
    for at in places:
        alone = x[at].clone()
        assert torch.equal(out[at], rms_norm.forward(alone, w)[0]) and torch.equal(grad[at], rms_norm.backward(alone, alone, w)[0])
        assert all(torch.equal(a[at], b) for a, b in zip((codes, scale), rms_norm.forward8(alone, w)))
        for product, weight in zip(products, weights):
            assert torch.equal(product[at], int8_linear.forward(codes[at], scale[at], weight))
    del out, codes, grad, products
    l, actions = x.view(-1)[: 40_000 * 100_000].view(40_000, 100_000), torch.arange(40_000, device=cuda) % 100_000
    got = log_probs.forward(l, actions, None, 3)
    grad = log_probs.backward(got.log_prob, got.entropy, l, actions, got.normalizer, got.entropy)
    for at in (slice(21_460, 21_490), slice(39_970, 40_000)):
        alone = l[at].clone()
        check_scores(log_probs.Scores(*(y[at] for y in got)), alone, actions[at], None, 3)
        assert torch.equal(grad[at], log_probs.backward(got.log_prob[at], got.entropy[at], alone, actions[at], got.normalizer[at],
                                                        got.entropy[at]))


def test_calls_at_the_same_time(cuda):
    """Two streams run the same operators on other inputs at once, over and over: nothing is shared between them."""
    import int8_linear
    import log_probs
    import rms_norm

    def inputs(seed):
        return (normal(cuda, 700, 2048, seed=seed), normal(cuda, 64, 50_000, seed=seed + 1),
                int8_linear.quantise_weight(normal(cuda, 2048, 300, seed=seed + 2)))

    def everything(x, l, weight):
        c, s, _ = rms_norm.forward8(x)
        grad, grad_weight = rms_norm.backward(x, x, x[0])
        got = log_probs.forward(l, torch.arange(64, device=cuda), None, 9)
        return [int8_linear.forward(c, s, weight), int8_linear.forward(c[:100], s[:100], weight), grad, grad_weight, *got]

    sets, streams = [inputs(0), inputs(10)], [torch.cuda.Stream(), torch.cuda.Stream()]
    want = [everything(*x) for x in sets]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i in (0, 1):
            with torch.cuda.stream(streams[i]):
                got[i].append(everything(*sets[i]))
    torch.cuda.synchronize()
    for i in (0, 1):
        for run in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(run, want[i]))
    assert int8_linear.gave_up() == 0


# ---- the policy that runs them together ------------------------------------------------------------------------

def rollout_of(cfg):
    import cartpole_metal
    import memory_policy as mp

    policy = mp.MemoryPolicy(cfg)
    g = torch.Generator(device=policy.decay.device).manual_seed(0)
    cartpole_metal.reseed(5)
    state, memory = cartpole_metal.reset(cfg.envs), policy.fresh_state(cfg.envs)
    resets = torch.ones(cfg.envs, dtype=torch.bool, device=policy.decay.device)
    return policy, mp.collect(policy, state, memory, resets, cfg.steps, g)[0]


def test_the_policys_gradients_with_and_without_the_fused_operators(cuda):
    """The same rollout's loss and gradients, norms and scores by torch and by the kernels: some twenty chained float32
    operations of up to 2,000 terms, each within 2^-16 of the sum of its terms' magnitudes."""
    import memory_policy as mp

    cfg = mp.Config(envs=33, steps=40)
    policy, rollout = rollout_of(cfg)
    found = []
    for fused in (0, 1):
        cfg.fused = fused
        loss = mp.loss_of(policy, rollout)
        found.append((loss, torch.autograd.grad(loss, policy.parameters)))
    (loss, grads), (loss1, grads1) = found
    assert abs(loss.item() - loss1.item()) <= 1e-3 * (1 + abs(loss.item()))
    for a, b in zip(grads, grads1):
        assert torch.isfinite(b).all() and (a - b).abs().max() <= 2e-3 * a.abs().max()


def test_the_policy_acts_in_8_bits(cuda):
    """Logits acted on in 8 bits against the trajectory form's in float32. A code is off by half of a 127th of its row's
    largest magnitude at most, which is below five times the root mean square of rows of 64 to 128 such values: 2% of that
    for a token's codes and for a channel's, as many independent errors as terms, so below 3% a product; five in a row
    below 7%, and a norm keeps a relative error."""
    import memory_policy as mp

    cfg = mp.Config(envs=65, steps=30, act_bits=8)
    policy, rollout = rollout_of(cfg)
    logits, _ = policy.trajectory(rollout.tokens, rollout.memory, rollout.resets)
    off, size = (logits - rollout.logits).norm(), logits.norm()
    assert 0 < off <= 0.1 * size
    with pytest.raises(ValueError, match="act_bits"):
        mp.MemoryPolicy(mp.Config(act_bits=4))


@pytest.mark.parametrize("act_bits,fused", [(8, 0), (32, 1), (8, 1)])
def test_the_policy_trains_with_them(cuda, act_bits, fused):
    import memory_policy as mp

    policy, lengths = mp.train(mp.Config(envs=64, steps=16, updates=3, act_bits=act_bits, fused=fused))
    assert len(lengths) == 3 and all(torch.isfinite(p).all() for p in policy.parameters)
