"""The memory policy's operators without a GPU: the oracle against differences and known answers,
the 8-bit format, and every refusal that the library or its wrappers make before touching a GPU."""

import ctypes

import numpy as np
import pytest
import torch

from oracle import policy

FAKE = ctypes.c_void_p(0x1000)   # never dereferenced: each call is rejected first
ODD = ctypes.c_void_p(0x1004)


def test_attention_gradient_is_the_derivative():
    r = np.random.default_rng(0)
    t, n, h, d = 7, 2, 2, 4
    q, k, v, do = (r.normal(size=(t, n, h, d)) for _ in range(4))
    s, gs = r.normal(size=(2, n, h, d, d))
    resets = r.random((t, n)) < 0.3
    decay = np.array([0.9, 0.0])

    def loss(q, k, v, s):
        out, end = policy.scan(q, k, v, decay, s, resets, 0.7)
        return (do * out).sum() + (gs * end).sum()

    grads = policy.attention_grad(do, q, k, v, decay, s, resets, 0.7, gs)
    args, eps = [q, k, v, s], 1e-6
    for i, g in enumerate(grads):
        way = r.normal(size=g.shape)
        up, down = list(args), list(args)
        up[i], down[i] = args[i] + eps * way, args[i] - eps * way
        # loss is of second degree along any one argument: the difference is exact up to rounding,
        # some 1e3 terms of 1e-16 over 2e-6
        assert abs((loss(*up) - loss(*down)) / (2 * eps) - (g * way).sum()) < 1e-6


@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_ffn_gradient_is_the_derivative(act):
    r = np.random.default_rng(1)
    x, wg, wu, dh = r.normal(size=(5, 3)), r.normal(size=(3, 4)), r.normal(size=(3, 4)), r.normal(size=(5, 4))
    grads, args, eps = policy.ffn_grad(dh, x, wg, wu, act)[:3], [x, wg, wu], 1e-5
    for i, g in enumerate(grads):
        way = r.normal(size=g.shape)
        up, down = list(args), list(args)
        up[i], down[i] = args[i] + eps * way, args[i] - eps * way
        diff = ((dh * policy.ffn(*up, act)).sum() - (dh * policy.ffn(*down, act)).sum()) / (2 * eps)
        assert abs(diff - (g * way).sum()) < 1e-7  # third derivative times eps^2, and rounding over eps


@pytest.mark.parametrize("ebits", [4, 5])
def test_moment_codes_keep_their_values(ebits):
    """Every code of a block decodes to a value that encodes to the same code whatever the random bits'
    size (the value lies on the grid), and rounding errs by less than an eighth, on average by nothing."""
    top = (1 << (ebits + 3)) - 1
    codes = np.zeros(policy.BLOCK, np.uint8)
    codes[: top - 1] = np.arange(1, top)
    for e in (32, 100, 127, 254):
        x = policy.decode(codes, np.array([e], np.uint8), ebits)
        for rand in (0, 0xFFFF):
            again, e2 = policy.encode(x, np.full(x.shape, rand), ebits)
            assert e2[0] == e and (again == codes).all()
    r = np.random.default_rng(2)
    x = (r.normal(size=64 * policy.BLOCK).astype(np.float32)) ** 2 + np.float32(1e-3)
    words = r.integers(0, 1 << 16, (400, x.size))
    got = np.stack([policy.decode(*policy.encode(x, w, ebits), ebits) for w in words]).astype(np.float64)
    assert (abs(got - x) <= x / 8).all()
    # a rounding error is at most x / 8, so its standard deviation at most x / 16; 6 deviations of the mean
    assert (abs(got.mean(0) - x) <= 6 * x / 16 / np.sqrt(400) + x * 2.0 ** -16).all()


def test_moment_codes_of_zeros_infinities_and_tiny_values():
    x = np.zeros(policy.BLOCK, np.float32)
    x[:5] = [np.inf, np.nan, 1.0, 1e-30, -0.0]
    codes, e = policy.encode(x, np.zeros(x.shape, np.int64), 5)
    back = policy.decode(codes, e, 5)
    assert np.isnan(back[:2]).all() and back[2] == 1.0 and 0 < back[3] < 1e-9 and (back[4:] == 0).all()
    assert e[0] == 127  # the neighbours of an infinity keep their scale
    codes, e = policy.encode(np.zeros(policy.BLOCK, np.float32), np.full(policy.BLOCK, 0xFFFF), 4)
    assert (codes == 0).all() and e[0] == 32


def test_attention_arguments_rejected_before_launch():
    import rlenv_lib

    lib = rlenv_lib.load()
    st = (ctypes.c_int64 * 12)(*[64] * 12)
    f32, bf16 = rlenv_lib.F32, rlenv_lib.BF16

    def fwd(dtype=f32, d=64, t=4, n=2, h=2, q=FAKE, scale=1.0, decay=FAKE, out=FAKE, end=FAKE, strides=st, start=None):
        need = max(0, lib.linear_attention_scratch_bytes(dtype, d, t, n, h, 0))
        return lib.linear_attention_forward(dtype, d, t, n, h, q, FAKE, FAKE, strides, decay, None, scale, start, out,
                                            end, FAKE, need, None)

    assert fwd(dtype=0) == -1 and fwd(d=48) == -2 and fwd(t=-1) == -1 and fwd(h=-1) == -1
    assert fwd(q=None) == -1 and fwd(q=ODD) == -1 and fwd(decay=None) == -1 and fwd(end=None) == -1
    assert fwd(out=None) == -1 and fwd(strides=None) == -1
    assert fwd(scale=0.0) == -1 and fwd(scale=float("nan")) == -1 and fwd(scale=float("inf")) == -1
    assert fwd(start=FAKE) == -1                                  # the state in place
    assert fwd(n=1 << 40, h=1 << 40) == -1
    bad = (ctypes.c_int64 * 12)(*[64] * 11, 66)
    assert fwd(strides=(ctypes.c_int64 * 9)(*[64] * 8, 66)) == -1  # rows off the 16-byte boundary
    assert fwd(dtype=bf16, strides=(ctypes.c_int64 * 9)(*[64] * 8, 68)) == -1
    assert fwd(n=0) == 0 and fwd(h=0) == 0
    assert lib.linear_attention_scratch_bytes(f32, 48, 1, 1, 1, 0) == -1

    def bwd(strides=st, dstate=FAKE, gs=None, dq=FAKE, t=4):
        need = max(0, lib.linear_attention_scratch_bytes(f32, 64, t, 2, 2, 1))
        return lib.linear_attention_backward(f32, 64, t, 2, 2, FAKE, FAKE, FAKE, FAKE, strides, FAKE, None, 1.0, None,
                                             gs, dq, FAKE, FAKE, dstate, FAKE, need, None)

    assert bwd(strides=bad) == -1 and bwd(dq=None) == -1 and bwd(dstate=FAKE, gs=FAKE) == -1 and bwd(t=-1) == -1
    two = (ctypes.c_int64 * 6)(*[64] * 6)
    assert lib.linear_attention_step(f32, 64, 2, 2, FAKE, FAKE, FAKE, two, FAKE, None, 1.0, ODD, FAKE, None) == -1
    assert lib.linear_attention_step(f32, 64, 2, 2, FAKE, FAKE, FAKE, two, FAKE, None, 1.0, None, FAKE, None) == -1
    assert lib.linear_attention_step(f32, 24, 2, 2, FAKE, FAKE, FAKE, two, FAKE, None, 1.0, FAKE, FAKE, None) == -2
    assert lib.linear_attention_step(f32, 64, 0, 2, None, None, None, None, None, None, 1.0, None, None, None) == 0


def test_scratch_that_is_missing_or_small_is_rejected():
    import rlenv_lib

    lib = rlenv_lib.load()
    f32 = rlenv_lib.F32
    st = (ctypes.c_int64 * 12)(*[64] * 12)
    need = lib.linear_attention_scratch_bytes(f32, 64, 1 << 16, 1, 1, 0)
    if need > 0:  # one long sequence is split over the time axis
        for ptr, size in ((None, need), (FAKE, need - 1), (ODD, need)):
            assert lib.linear_attention_forward(f32, 64, 1 << 16, 1, 1, FAKE, FAKE, FAKE, st, FAKE, None, 1.0, None,
                                                FAKE, FAKE, ptr, size, None) == -1
    need = lib.gated_ffn_scratch_bytes(f32, 256, 128, 128, 1)
    assert need > 0
    for ptr, size in ((None, need), (FAKE, need - 1), (ODD, need)):
        assert lib.gated_ffn_backward(f32, 0, 256, 128, 128, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, ptr, size,
                                      None) == -1


def test_ffn_arguments_rejected_before_launch():
    import rlenv_lib

    lib = rlenv_lib.load()
    f32 = rlenv_lib.F32

    def fwd(dtype=f32, act=0, m=4, k=4, f=4, x=FAKE, out=FAKE):
        need = max(0, lib.gated_ffn_scratch_bytes(dtype, max(m, 0), max(k, 0), max(f, 0), 0))
        return lib.gated_ffn_forward(dtype, act, m, k, f, x, FAKE, FAKE, out, FAKE, need, None)

    assert fwd(dtype=2) == -1 and fwd(act=2) == -1 and fwd(m=-1) == -1 and fwd(k=-1) == -1 and fwd(x=None) == -1
    assert fwd(out=None) == -1 and fwd(f=1 << 31) == -1
    assert fwd(m=0) == 0 and fwd(f=0) == 0
    assert lib.gated_ffn_scratch_bytes(2, 4, 4, 4, 0) == -1 and lib.gated_ffn_scratch_bytes(f32, -4, 4, 4, 0) == -1
    assert lib.gated_ffn_backward(f32, 0, 0, 4, 4, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, 1 << 20, None) == -1


def test_adamw_arguments_rejected_before_launch():
    import rlenv_lib

    lib = rlenv_lib.load()
    f32 = rlenv_lib.F32
    one = (ctypes.c_void_p * 1)(0x1000)
    none = (ctypes.c_void_p * 1)(None)

    def step(bits=8, dtype=f32, p=one, size=10, m=FAKE, m_exp=FAKE, b1=0.9, b2=0.999, eps=1e-8, t=1, count=1):
        return lib.adamw_step(bits, dtype, count, p, one, None, (ctypes.c_int64 * 1)(size), m, FAKE, m_exp, FAKE, 1e-3,
                              b1, b2, eps, 0.0, None, t, 0, None)

    assert step(bits=16) == -1 and step(dtype=0) == -1 and step(p=None) == -1 and step(p=none) == -1
    assert step(size=-1) == -1 and step(size=(1 << 32) + 1) == -1 and step(m=None) == -1 and step(m_exp=None) == -1
    assert step(b1=1.0) == -1 and step(b2=-0.1) == -1 and step(eps=-1.0) == -1 and step(t=0) == -1
    assert step(bits=32, m=ODD) == -1 and step(b1=float("nan")) == -1 and step(count=-1) == -1
    assert step(count=0) == 0 and step(size=0) == 0
    assert lib.adamw_moments(-1, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, None) == -1
    assert lib.adamw_moments(1, FAKE, FAKE, FAKE, FAKE, ODD, FAKE, None) == -1
    assert lib.adamw_moments(0, None, None, None, None, None, None, None) == 0


def test_wrappers_refuse_host_tensors():
    """There is no CPU path: a host tensor raises."""
    import adamw
    import gated_ffn
    import linear_attention

    x = torch.zeros(2, 3, 1, 16)
    with pytest.raises(ValueError, match="CUDA"):
        linear_attention.forward(x, x, x, torch.ones(1))
    with pytest.raises(ValueError, match="CUDA"):
        linear_attention.step(x[0], x[0], x[0], torch.ones(1), torch.zeros(3, 1, 16, 16))
    with pytest.raises(ValueError, match="CUDA"):
        gated_ffn.forward(x, torch.zeros(16, 4), torch.zeros(16, 4))
    p = [torch.zeros(5)]
    with pytest.raises(ValueError, match="bits"):
        adamw.init_state(p, bits=4)
    with pytest.raises(ValueError):
        adamw.step(p, p, adamw.init_state(p))


def test_episode_starts():
    import linear_attention

    dones = torch.tensor([[0, 1], [1, 0], [0, 0]], dtype=torch.bool)
    want = [[False, False], [False, True], [True, False]]
    assert linear_attention.episode_starts(dones).tolist() == want
    assert linear_attention.episode_starts(dones, torch.tensor([True, False]))[0].tolist() == [True, False]
    assert linear_attention.episode_starts(dones[:0]).shape == (0, 2)


@pytest.mark.parametrize("bits", [8, 32])
def test_adamw_of_empty_tensors_needs_no_moments(bits):
    """A tensor without elements has no moments: their pointers may be NULL, as torch's empty tensors' are."""
    import rlenv_lib

    lib = rlenv_lib.load()

    def step(sizes, at=None, m=None):
        n = len(sizes)
        return lib.adamw_step(bits, rlenv_lib.F32, n, (ctypes.c_void_p * n)(*[at] * n), (ctypes.c_void_p * n)(*[at] * n),
                              None, (ctypes.c_int64 * n)(*sizes), m, m, m, m, 1e-3, 0.9, 0.999, 1e-8, 0.0, None, 1, 0, None)

    assert step([0]) == 0 and step([0, 0, 0]) == 0
    assert step([0, 5], 0x1000) == -1 and step([5], None, FAKE) == -1 and step([0, -1]) == -1


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows_have_strides_that_the_kernels_take(dtype):
    """Bases and strides on 16-byte boundaries, and the same values through them: axes of one element may have any
    stride in torch, a contiguous tensor's among them."""
    import linear_attention

    flat = torch.arange(4000, dtype=torch.float32).to(dtype)
    views = [flat.as_strided((1, 3, 2, 16), (97, 32, 16, 1)), flat.as_strided((3, 1, 2, 16), (32, 7, 16, 1)),
             flat.as_strided((5, 3, 1, 16), (48, 16, 3, 1)), flat.as_strided((1, 1, 1, 32), (1, 3, 5, 1)),
             flat.as_strided((4, 3, 2, 16), (97, 32, 16, 1)), flat.as_strided((4, 3, 2, 16), (0, 32, 16, 1)),
             flat.as_strided((4, 3, 2, 16), (32, 128, 16, 1)), flat[1:97].view(1, 3, 2, 16)]
    for x in views:
        y, strides = linear_attention._rows(x)
        assert len(strides) == 3 and y.data_ptr() % 16 == 0, x.stride()
        assert all(s * x.element_size() % 16 == 0 for s in strides), (x.stride(), strides)
        assert torch.equal(y.as_strided(x.shape, (*strides, 1)), x)
