"""The norm, the 8-bit products and the scores of actions without a GPU: the oracle against differences and known
answers, the row plumbing, and every refusal that the library or its wrappers make before touching a GPU."""

import ctypes

import numpy as np
import pytest
import torch

from oracle import policy

FAKE = ctypes.c_void_p(0x1000)   # never dereferenced: each call is rejected first
ODD = ctypes.c_void_p(0x1001)
FOUR = ctypes.c_void_p(0x1004)


def difference(f, args, i, way, eps=1e-6):
    up, down = list(args), list(args)
    up[i], down[i] = args[i] + eps * way, args[i] - eps * way
    return (f(*up) - f(*down)) / (2 * eps)


@pytest.mark.parametrize("weighted", [True, False])
def test_norm_gradient_is_the_derivative(weighted):
    r = np.random.default_rng(0)
    t, g, gt = (r.normal(size=(4, 7)) for _ in range(3))
    w = 1 + 0.3 * r.normal(size=7) if weighted else None

    def loss(t, w):
        return (g * policy.norm(t, w, 1e-3)).sum() + (gt * t).sum()

    dt, dw = policy.norm_grad(g, t, w, 1e-3, gt)
    way = r.normal(size=t.shape)
    # rounding: some 60 terms of 1e-16 over 2e-6; the third derivative times eps^2 is far below
    assert abs(difference(loss, [t, w], 0, way) - (dt * way).sum()) < 1e-7
    if weighted:
        way = r.normal(size=w.shape)
        assert abs(difference(loss, [t, w], 1, way) - (dw * way).sum()) < 1e-7


def test_scores_gradient_is_the_derivative():
    r = np.random.default_rng(1)
    l, g, h = r.normal(size=(6, 5)) * 2, r.normal(size=6), r.normal(size=6)
    allowed = r.random((6, 5)) < 0.7
    allowed[:, 2] = True
    allowed[5] = False
    actions = np.array([2, 2, -1, 2, 2, 0])

    def loss(l):
        lp, entropy, _, _ = policy.scores(l, actions, allowed)
        return (g * lp)[:5].sum() + (h * entropy).sum()  # row 5 allows nothing: a constant -infinity

    grad, way = policy.scores_grad(g, h, l, actions, allowed), r.normal(size=l.shape)
    assert abs(difference(loss, [l], 0, way) - (grad * way).sum()) < 1e-7
    assert (grad[5] == 0).all() and (grad[~allowed] == 0).all()


def test_scores_gradient_of_an_action_that_is_all_but_impossible():
    """Its own gradient is g (1 - p), also where p is no number of 64 bits any more."""
    l = np.array([[0.0, -2000.0, -np.inf]])
    for action, want in ((0, [0, 0, 0]), (1, [-1.5, 1.5, 0]), (2, [-1.5, 0, 0])):
        assert policy.scores_grad(np.array([1.5]), np.array([0.3]), l, np.array([action])).tolist() == [want]


def test_scores_of_known_distributions():
    lp, entropy, normalizer, _ = policy.scores(np.zeros((2, 8)), np.array([3, -1]))
    np.testing.assert_allclose(entropy, np.log(8))
    np.testing.assert_allclose(lp, [-np.log(8), 0])
    lp, entropy, normalizer, _ = policy.scores(np.full((1, 3), -np.inf), np.array([1]))
    assert lp == -np.inf and entropy == 0 and normalizer == -np.inf
    assert policy.best(np.array([1.0, 3.0, 3.0, -np.inf]), 4).tolist() == [1, 2, 0, 3]


def test_quantised_rows():
    codes, scale = policy.quantise(np.array([[1.0, -2.54, 0.0], [0.0, 0.0, 0.0], [1e-40, 0.0, -1e-35]]))
    assert codes[0].tolist() == [50, -127, 0] and scale[0] == 2.54 / 127
    assert (codes[1:] == 0).all() and (scale[1:] == 0).all()


def test_rows_of_tensors():
    """as_rows keeps every layout that is one even step from row to row, and copies the others."""
    import rlenv_lib as rl

    x = torch.arange(5 * 6 * 8.0).reshape(5, 6, 8)
    kept = [(x, 8), (x[..., :7], 8), (x[:, :, 3:4], 8), (x[::2, 0], 96), (x[1:2, :, :5], 8), (x[0, 0], 8),
            (x[:, :1].expand(5, 1, 8), 48), (x[0, 0].expand(4, 3, 8), 0), (x[:, 0, :5], 48), (x[:1, 2, 1:], None)]
    for view, step in kept:
        y, got = rl.as_rows(view)
        assert y.data_ptr() == view.data_ptr() and (step is None or got == step), (view.shape, view.stride(), got)
        flat = torch.as_strided(y, (y[..., 0].numel(), y.shape[-1]), (got, 1), y.storage_offset())
        assert torch.equal(flat.reshape(view.shape), view)
    for view in (x.transpose(1, 2), x[..., ::2], x[:, :4, :7], x.transpose(0, 1)[..., :7], x[0, 0, ::2],
                 x[0].expand(5, 6, 8)):
        y, got = rl.as_rows(view)
        assert y.is_contiguous() and got == view.shape[-1] and torch.equal(y, view)


def test_norm_arguments_rejected_before_launch():
    import rlenv_lib

    lib = rlenv_lib.load()
    f32, bf16 = rlenv_lib.F32, rlenv_lib.BF16

    def fwd(dtype=f32, m=4, k=8, x=FAKE, xs=8, res=FAKE, rs=8, w=FAKE, eps=1e-6, out=FAKE, total=FAKE):
        return lib.rms_norm_forward(dtype, m, k, x, xs, res, rs, w, eps, out, total, None)

    assert fwd(dtype=0) == -1 and fwd(m=-1) == -1 and fwd(k=0) == -1 and fwd(m=1 << 31) == -1 and fwd(k=1 << 31) == -1
    assert fwd(x=None) == -1 and fwd(out=None) == -1 and fwd(xs=-1) == -1 and fwd(rs=-8) == -1
    assert fwd(eps=-1.0) == -1 and fwd(eps=float("nan")) == -1
    for name in ("x", "res", "w", "out", "total"):
        assert fwd(**{name: ODD}) == -1 and fwd(dtype=bf16, **{name: ODD}) == -1
    assert fwd(m=0, x=None, out=None) == 0

    def codes(m=4, k=8, x=FAKE, codes=FAKE, pitch=16, scale=FAKE):
        return lib.rms_norm_codes(f32, m, k, x, 8, None, 0, None, 1e-6, 1, codes, pitch, scale, None, None)

    assert codes(pitch=7) == -1 and codes(codes=None) == -1 and codes(scale=None) == -1 and codes(scale=ODD) == -1
    assert codes(x=None) == -1 and codes(m=0) == 0

    def bwd(m=4, g=FAKE, t=FAKE, grad=FAKE, gw=FAKE, tmp=FAKE, nbytes=None, gts=8):
        nbytes = lib.rms_norm_scratch_bytes(m, 8) if nbytes is None else nbytes
        return lib.rms_norm_backward(f32, m, 8, g, 8, t, 8, FAKE, 1e-6, FAKE, gts, grad, gw, tmp, nbytes, None)

    assert lib.rms_norm_scratch_bytes(4, 8) > 0 and lib.rms_norm_scratch_bytes(4, 0) == -1
    assert bwd(g=None) == -1 and bwd(t=None) == -1 and bwd(grad=None) == -1 and bwd(gts=-1) == -1
    assert bwd(tmp=None) == -1 and bwd(tmp=FOUR) == -1 and bwd(nbytes=4) == -1
    assert bwd(m=0) == -1 and bwd(m=0, gw=None) == 0


def test_int8_arguments_rejected_before_launch():
    import rlenv_lib

    lib = rlenv_lib.load()

    def fwd(dtype=rlenv_lib.F32, m=4, k=16, f=8, a=FAKE, ap=16, sa=FAKE, w=FAKE, wp=16, sw=FAKE, out=FAKE, tmp=FAKE,
            less=0):
        nbytes = max(0, lib.int8_linear_scratch_bytes(m, k, f)) - less
        return lib.int8_linear_forward(dtype, m, k, f, a, ap, sa, w, wp, sw, out, tmp, nbytes, None)

    assert fwd(dtype=0) == -1 and fwd(m=-1) == -1 and fwd(f=-1) == -1 and fwd(k=0) == -1
    assert fwd(k=131072, ap=131072, wp=131072) == -1  # 131,072 x 128 x 128 = 2^31
    assert fwd(ap=0) == -1 and fwd(wp=0) == -1 and fwd(ap=24, k=17) == -1 and fwd(wp=40) == -1
    for name in ("a", "w"):
        assert fwd(**{name: None}) == -1 and fwd(**{name: FOUR}) == -1
    for name in ("sa", "sw", "out"):
        assert fwd(**{name: None}) == -1 and fwd(**{name: ODD}) == -1
    assert fwd(m=0) == 0 and fwd(f=0) == 0
    assert lib.int8_linear_scratch_bytes(4, 0, 8) == -1


def test_scores_arguments_rejected_before_launch():
    import rlenv_lib

    lib = rlenv_lib.load()
    f32, i64 = rlenv_lib.F32, rlenv_lib.I64

    def fwd(dtype=f32, m=4, v=8, l=FAKE, stride=8, actions=FAKE, kind=i64, allowed=None, astride=0, lp=FAKE, h=FAKE, z=FAKE,
            top=0, best=None, blp=None):
        return lib.log_probs_forward(dtype, m, v, l, stride, actions, kind, allowed, astride, lp, h, z, top, best, blp, None)

    assert fwd(dtype=0) == -1 and fwd(m=-1) == -1 and fwd(v=0) == -1 and fwd(v=1 << 31) == -1 and fwd(stride=-1) == -1
    assert fwd(m=1 << 26) == -1 and fwd(kind=3) == -1 and fwd(kind=5) == -1 and fwd(astride=-1) == -1
    for name in ("l", "actions", "lp", "h", "z"):
        assert fwd(**{name: None}) == -1 and fwd(**{name: ODD}) == -1
    assert fwd(actions=FOUR) == -1
    assert fwd(top=-1) == -1 and fwd(top=9, best=FAKE, blp=FAKE) == -1 and fwd(v=99, top=33, best=FAKE, blp=FAKE) == -1
    assert fwd(top=2) == -1 and fwd(top=2, best=FAKE) == -1 and fwd(top=2, best=FOUR, blp=FAKE) == -1
    assert fwd(m=0, l=None) == 0

    def bwd(g=FAKE, h=FAKE, l=FAKE, z=FAKE, e=FAKE, grad=FAKE, m=4):
        return lib.log_probs_backward(f32, m, 8, g, h, l, 8, FAKE, i64, z, e, None, 0, grad, None)

    for name in ("l", "z", "e", "grad"):
        assert bwd(**{name: None}) == -1 and bwd(**{name: ODD}) == -1
    assert bwd(g=ODD) == -1 and bwd(h=ODD) == -1 and bwd(m=0) == 0


def test_scores_with_a_remainder_rejected_before_launch():
    import rlenv_lib

    lib = rlenv_lib.load()
    f32, i64 = rlenv_lib.F32, rlenv_lib.I64

    def fwd(rest=FAKE, l=FAKE, m=4, z=FAKE):
        return lib.log_probs_forward_remainder(f32, m, 8, l, 8, FAKE, i64, None, 0, FAKE, FAKE, z, rest, 0, None, None, None)

    def bwd(rest=FAKE, l=FAKE, m=4, z=FAKE):
        return lib.log_probs_backward_remainder(f32, m, 8, FAKE, FAKE, l, 8, FAKE, i64, z, rest, FAKE, None, 0, FAKE, None)

    for call in (fwd, bwd):
        assert call(rest=ODD) == -1 and call(l=None) == -1 and call(z=None) == -1 and call(m=-1) == -1
        assert call(m=0) == 0 and call(m=0, rest=None) == 0


def test_many_rows_of_scores_take_several_launches():
    """Every row once, in order, and no launch beyond what the library takes."""
    import log_probs

    for m, v in ((0, 3), (1, 1), ((1 << 26) - 16, 2), (1 << 26, 2), (1 << 28, 1), (5_000_000_000, 7), (2000, (1 << 31) - 64),
                 (3, 1 << 30), (1 << 20, 1 << 21)):
        launches, after = log_probs._launches(m, v), 0
        for at, n in launches:
            assert at == after and n < 1 << 26 and n * v < 1 << 40 and at % 16 == 0
            after += n
        assert after == m and (len(launches) == 1) == (m <= (1 << 26) - 16 and m * v <= (1 << 40) - 16 * v)


def test_wrappers_refuse_what_is_no_cuda_tensor():
    import int8_linear
    import log_probs
    import rms_norm

    x, a = torch.zeros(3, 4), torch.zeros(3, dtype=torch.int64)
    for call in (lambda: rms_norm.forward(x), lambda: rms_norm.forward(None), lambda: rms_norm.forward8(x),
                 lambda: rms_norm.backward(x, x), lambda: rms_norm.apply(x), lambda: int8_linear.quantise(x),
                 lambda: int8_linear.quantise_weight(x), lambda: int8_linear.product(x, None),
                 lambda: int8_linear.forward(x.to(torch.int8), x[:, 0], int8_linear.Weight(x.to(torch.int8), x[:, 0])),
                 lambda: log_probs.forward(x, a), lambda: log_probs.forward([1.0], a), lambda: log_probs.apply(x, a),
                 lambda: log_probs.backward(None, None, x, a, x[:, 0], x[:, 0])):
        with pytest.raises(ValueError, match="CUDA tensor"):
            call()
