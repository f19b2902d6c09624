"""The memory policy's operators on the GPU against the oracle in 64 bits.

Tolerances are bounds on rounding, element by element: `mag` is the same sum with every term's
magnitude. A float32 sum of n terms, accumulated in any order, truncating or rounding, is within
(n + the roundings of a term) 2^-23 of mag. bfloat16 outputs add half an ulp, 2^-8 of the value at
most, and intermediates held in two 16-bit terms 2^-15 of mag."""

import numpy as np
import pytest
import torch

from oracle import policy

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def to64(x):
    return x.detach().double().cpu().numpy()


def close(got, want, tol, what):
    got = to64(got)
    assert np.isfinite(got).all(), what
    off = np.abs(got - want) - tol
    assert (off <= 0).all(), f"{what}: {(off > 0).sum()} of {off.size} outside, worst by {off.max():.3g} at " \
                             f"{np.unravel_index(off.argmax(), off.shape)}"


# ---- decayed linear attention ------------------------------------------------------------------------

def inputs(cuda, t, n, h, d, dtype, seed=0, p_reset=0.05):
    g = torch.Generator(device=cuda).manual_seed(seed)
    x = [torch.randn((t, n, h, d), generator=g, device=cuda).to(TYPES[dtype]) for _ in range(4)]
    decay = torch.tensor([0.9, 1.0, 0.0, 0.999, 0.5, 0.99])[torch.arange(h) % 6].to(cuda)
    state, gstate = torch.randn((2, n, h, d, d), generator=g, device=cuda)
    resets = torch.rand((t, n), generator=g, device=cuda) < p_reset
    return x, decay, state, gstate, resets


def attention_tol(dtype, d, t, mag, want):
    terms = d + 64 + 2 * (t // 64 + 1) + 16
    tol = terms * 2.0 ** -23 * mag
    return tol + 2.0 ** -15 * mag + 2.0 ** -8 * np.abs(want) if dtype == "bf16" else tol


SHAPES = [(0, 2, 2, 16), (1, 1, 1, 16), (1, 3, 2, 128), (2, 2, 3, 32), (17, 1, 2, 64), (63, 2, 1, 32), (64, 1, 2, 64),
          (65, 3, 1, 128), (129, 1, 3, 16), (203, 5, 3, 32), (257, 2, 2, 64), (1000, 1, 1, 64), (2500, 1, 2, 16)]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("t,n,h,d", SHAPES)
def test_attention_forward(cuda, t, n, h, d, dtype):
    import linear_attention as la

    (q, k, v, _), decay, state, _, resets = inputs(cuda, t, n, h, d, dtype)
    for s, r in ((state, resets), (None, None), (state, None), (None, resets)):
        out, end = la.forward(q, k, v, decay, s, r, scale=0.3)
        args = (to64(q), to64(k), to64(v), to64(decay), None if s is None else to64(s),
                None if r is None else r.cpu().numpy(), 0.3)
        want, wend = policy.scan(*args)
        mag, mend = policy.scan(*args, absolute=True)
        close(out, want, attention_tol(dtype, d, t, mag, want), "out")
        close(end, wend, attention_tol("f32", d, t, mend, wend), "state")
        assert out.dtype == q.dtype and end.dtype == torch.float32


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("t,n,h,d", [s for s in SHAPES if s[0] < 1000] + [(700, 1, 1, 128)])
def test_attention_backward(cuda, t, n, h, d, dtype):
    import linear_attention as la

    (q, k, v, do), decay, state, gstate, resets = inputs(cuda, t, n, h, d, dtype, seed=1)
    for s, r, gs in ((state, resets, gstate), (None, None, None), (None, resets, gstate), (state, None, None)):
        got = la.backward(do, q, k, v, decay, s, r, scale=0.3, grad_state=gs)
        args = (to64(do), to64(q), to64(k), to64(v), to64(decay), None if s is None else to64(s),
                None if r is None else r.cpu().numpy(), 0.3, None if gs is None else to64(gs))
        want, mag = policy.attention_grad(*args), policy.attention_grad(*args, absolute=True)
        for name, x, w, m in zip(("dq", "dk", "dv", "dstate"), got, want, mag):
            close(x, w, attention_tol("f32" if name == "dstate" else dtype, d, t, m, w), name)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("n,h,d", [(1, 1, 16), (3, 5, 32), (7, 2, 64), (33, 3, 128)])
def test_attention_step_continues_a_trajectory(cuda, n, h, d, dtype):
    """Steps from a state, against the oracle; and the same tokens as one trajectory."""
    import linear_attention as la

    t = 9
    (q, k, v, _), decay, state, _, resets = inputs(cuda, t, n, h, d, dtype, seed=2, p_reset=0.2)
    args = (to64(q), to64(k), to64(v), to64(decay), to64(state), resets.cpu().numpy(), d ** -0.5)
    want, wend = policy.scan(*args)
    mag, mend = policy.scan(*args, absolute=True)
    s = state.clone()
    out = torch.stack([la.step(q[i], k[i], v[i], decay, s, resets[i]) for i in range(t)])
    close(out, want, attention_tol(dtype, d, t, mag, want), "out")
    close(s, wend, attention_tol("f32", d, t, mend, wend), "state")
    long, _ = la.forward(q, k, v, decay, state, resets)
    close(long, want, attention_tol(dtype, d, t, mag, want), "trajectory")


def test_attention_in_two_halves_is_the_whole(cuda):
    import linear_attention as la

    (q, k, v, _), decay, state, _, resets = inputs(cuda, 300, 2, 2, 32, "f32", seed=3)
    out, end = la.forward(q, k, v, decay, state, resets)
    a, mid = la.forward(q[:111], k[:111], v[:111], decay, state, resets[:111])
    b, end2 = la.forward(q[111:], k[111:], v[111:], decay, mid, resets[111:])
    args = (to64(q), to64(k), to64(v), to64(decay), to64(state), resets.cpu().numpy(), 32 ** -0.5)
    mag, mend = policy.scan(*args, absolute=True)
    close(torch.cat([a, b]), to64(out), 2 * attention_tol("f32", 32, 300, mag, mag), "out")
    close(end2, to64(end), 2 * attention_tol("f32", 32, 300, mend, mend), "state")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("t,d", [(150, 32), (150, 128), (5, 64), (4000, 16)])
def test_what_a_reset_cuts_off_is_not_seen(cuda, t, d, dtype):
    """Infinities and NaN in an earlier episode, in later tokens and in a dropped state leave the other
    tokens as if they were not there: equal to the same call with those values replaced."""
    import linear_attention as la

    (q, k, v, do), decay, state, gstate, _ = inputs(cuda, t, 2, 2, d, dtype, seed=4)
    cut, late = t // 2, t - 1
    resets = torch.zeros((t, 2), dtype=torch.bool, device=cuda)
    resets[cut] = True
    bad = [x.clone() for x in (q, k, v, state)]
    bad[0][0, :, :, 1], bad[1][cut - 1, :, :, 0], bad[2][1, :, :, 2], bad[3][...] = np.nan, np.inf, -np.inf, np.inf
    for x in bad[:3]:
        x[late] = np.nan
    clean = [x.clone() for x in (q, k, v, state)]
    out, _ = la.forward(*bad[:3], decay, bad[3], resets)
    want, _ = la.forward(*clean[:3], decay, clean[3], resets)
    args = (to64(q), to64(k), to64(v), to64(decay), None, resets.cpu().numpy(), d ** -0.5)
    mag, _ = policy.scan(*args, absolute=True)
    tol = 2 * attention_tol(dtype, d, t, mag, mag)
    close(out[cut:late], to64(want)[cut:late], tol[cut:late], "after the cut")
    assert torch.isnan(out[late]).all()
    # the gradient: tokens before the cut see nothing of what comes after it, and the other way round
    grads = [x.clone() for x in (do, q, k, v)]
    for x in grads:
        x[:cut - 1] = np.nan
    gq, gk, gv, _ = la.backward(*grads, decay, None, resets, grad_state=gstate)
    args = (to64(do), to64(q), to64(k), to64(v), to64(decay), None, resets.cpu().numpy(), d ** -0.5, to64(gstate))
    want, mags = policy.attention_grad(*args), policy.attention_grad(*args, absolute=True)
    for name, x, w, m in zip(("dq", "dk", "dv"), (gq, gk, gv), want, mags):
        close(x[cut:], w[cut:], attention_tol(dtype, d, t, m, w)[cut:], name)
    # a single token whose old state is dropped
    s = torch.full_like(state, np.inf)
    la.step(q[0], k[0], v[0], decay, s, torch.ones(2, dtype=torch.bool, device=cuda))
    close(s, to64(k[0])[..., :, None] * to64(v[0])[..., None, :], 2.0 ** -23 * 100, "step")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_attention_takes_any_strides(cuda, dtype):
    """Slices of one fused tensor, environment-major views, broadcast heads and rows off the 16-byte
    boundary give the bits of dense copies."""
    import linear_attention as la

    t, n, h, d = 70, 3, 2, 32
    g = torch.Generator(device=cuda).manual_seed(5)
    fused = torch.randn((n, t, 3, h, d), generator=g, device=cuda).to(TYPES[dtype]).transpose(0, 1)
    decay = torch.tensor([0.9, 0.99], device=cuda)
    odd = torch.randn(t * n * h * d + 1, generator=g, device=cuda).to(TYPES[dtype])[1:].view(t, n, h, d)
    wide = torch.randn((t, n, 1, d), generator=g, device=cuda).to(TYPES[dtype]).expand(t, n, h, d)
    for q, k, v in ((fused[:, :, 0], fused[:, :, 1], fused[:, :, 2]), (odd, fused[:, :, 1], wide)):
        resets = (torch.rand((n, t), generator=g, device=cuda) < 0.1).t()
        got = la.forward(q, k, v, decay, None, resets)
        want = la.forward(q.contiguous(), k.contiguous(), v.contiguous(), decay, None, resets.contiguous())
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        got = la.backward(v, q, k, v, decay, None, resets)
        want = la.backward(*(x.contiguous() for x in (v, q, k, v)), decay, None, resets.contiguous())
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        s1, s2 = torch.ones((2, n, h, d, d), device=cuda)
        assert torch.equal(la.step(q[3], k[3], v[3], decay, s1),
                           la.step(q[3].contiguous(), k[3].contiguous(), v[3].contiguous(), decay, s2))
        assert torch.equal(s1, s2)


def test_attention_gradients_through_autograd_and_differences(cuda):
    import linear_attention as la

    (q, k, v, do), decay, state, gstate, resets = inputs(cuda, 40, 2, 2, 16, "f32", seed=6)
    leaves = [x.clone().requires_grad_() for x in (q, k, v, state)]
    out, end = la.attend(*leaves[:3], decay, leaves[3], resets)
    ((out * do).sum() + (end * gstate).sum()).backward()
    args = [to64(x) for x in (q, k, v, state)]

    def loss(a):
        o, e = policy.scan(a[0], a[1], a[2], to64(decay), a[3], resets.cpu().numpy(), 16 ** -0.5)
        return (o * to64(do)).sum() + (e * to64(gstate)).sum()

    r = np.random.default_rng(0)
    for i, leaf in enumerate(leaves):
        way = r.normal(size=args[i].shape)
        up, down = list(args), list(args)
        up[i], down[i] = args[i] + 1e-3 * way, args[i] - 1e-3 * way
        diff = (loss(up) - loss(down)) / 2e-3
        # an exact difference (degree two); the gradient's float32 errors, 2^-18 of its size at most, against way
        assert abs(diff - (to64(leaf.grad) * way).sum()) < 2.0 ** -18 * np.abs(to64(leaf.grad) * way).sum() * 4 + 1e-6


def test_attention_offsets_past_32_bits(cuda):
    """A batch whose last environments lie beyond 2^31 elements, against those environments alone."""
    import linear_attention as la

    t, n, h, d = 33, 260_000, 2, 128
    g = torch.Generator(device=cuda).manual_seed(7)
    base = torch.randn((t, 1000, h, d), generator=g, device=cuda, dtype=torch.float32).to(torch.bfloat16)
    x = base.repeat(1, n // 1000, 1, 1)
    assert x.numel() > 2 ** 31
    x[:, -2:] *= 2
    decay = torch.tensor([0.9, 0.99], device=cuda)
    out, end = la.forward(x, x, x, decay)
    tail = x[:, -2:].contiguous()
    want, wend = la.forward(tail, tail, tail, decay)
    assert torch.equal(out[:, -2:], want) and torch.equal(end[-2:], wend)
    first, _ = la.forward(base, base, base, decay)
    assert torch.equal(out[:, :1000], first)
    del out, want, first
    o = la.step(x[0], x[1], x[2], decay, end)
    w = la.step(tail[0], tail[1], tail[2], decay, wend)
    assert end.numel() > 2 ** 31 and torch.equal(o[-2:], w) and torch.equal(end[-2:], wend)


def test_operators_follow_the_current_stream(cuda):
    """On a side stream, behind work that delays its inputs, with other work on the default stream."""
    import gated_ffn
    import linear_attention as la

    (q, k, v, _), decay, state, _, resets = inputs(cuda, 500, 8, 4, 64, "bf16", seed=8)
    w = torch.randn((64, 96), device=cuda, dtype=torch.bfloat16)
    want, wend = la.forward(q, k, v, decay, state, resets)
    whid = gated_ffn.forward(want, w, w)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    late = [torch.zeros_like(x) for x in (q, k, v)]
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        big = torch.randn((4096, 4096), device=cuda)
        for _ in range(20):
            big = big @ big * 1e-3
        for x, y in zip(late, (q, k, v)):
            x.copy_(y)
        out, end = la.forward(*late, decay, state, resets)
        hid = gated_ffn.forward(out, w, w)
    side.synchronize()
    assert torch.equal(out, want) and torch.equal(end, wend) and torch.equal(hid, whid)


def test_attention_refusals(cuda):
    import linear_attention as la

    x = torch.zeros((4, 2, 2, 32), device=cuda)
    decay, state = torch.ones(2, device=cuda), torch.zeros((2, 2, 32, 32), device=cuda)
    for args, kw in [((x, x, x[:3], decay), {}), ((x, x.bfloat16(), x, decay), {}), ((x.half(),) * 3 + (decay,), {}),
                     ((x, x, x, decay[:1]), {}), ((x, x, x, decay.double()), {}), ((x, x, x, decay), {"state": state[:1]}),
                     ((x, x, x, decay), {"state": state.bfloat16()}),
                     ((x, x, x, decay), {"resets": torch.zeros((2, 4), dtype=torch.bool, device=cuda)}),
                     ((x, x, x, decay), {"resets": torch.zeros((4, 2), device=cuda)}),
                     ((x, x, x, decay.cpu()), {}), ((x, x, x, decay), {"scale": 0.0}),
                     ((x, x, x, decay), {"scale": float("nan")}),
                     ((x[..., :24], x[..., :24], x[..., :24], decay), {})]:
        with pytest.raises(ValueError):
            la.forward(*args, **kw)
    with pytest.raises(ValueError):
        la.step(x[0], x[0], x[0], decay, state.transpose(2, 3))
    with pytest.raises(ValueError):
        la.step(x[0], x[0], x[0], decay, None)


# ---- gated feed-forward block --------------------------------------------------------------------------

FFN_SHAPES = [(1, 1, 1), (1, 64, 256), (3, 97, 250), (8, 1024, 512), (17, 16, 33), (128, 64, 128), (129, 65, 131),
              (200, 32, 1000), (300, 520, 72), (1000, 61, 173), (257, 1000, 264)]


def ffn_inputs(cuda, m, k, f, dtype, seed=0):
    g = torch.Generator(device=cuda).manual_seed(seed)

    def draw(*shape, scale=1.0):
        return (torch.randn(shape, generator=g, device=cuda) * scale).to(TYPES[dtype])

    return draw(m, k), draw(k, f, scale=k ** -0.5), draw(k, f, scale=k ** -0.5), draw(m, f)


def ffn_errors(x, wg, wu, act):
    """g, u and bounds on their errors as float32 sums of k terms."""
    unit = (x.shape[1] + 8) * 2.0 ** -23
    return x @ wg, x @ wu, unit * (abs(x) @ abs(wg)), unit * (abs(x) @ abs(wu))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("m,k,f", FFN_SHAPES)
def test_ffn_forward(cuda, m, k, f, act, dtype):
    import gated_ffn

    x, wg, wu, _ = ffn_inputs(cuda, m, k, f, dtype)
    out = gated_ffn.forward(x, wg, wu, act)
    x, wg, wu = to64(x), to64(wg), to64(wu)
    want = policy.ffn(x, wg, wu, act)
    g, u, eg, eu = ffn_errors(x, wg, wu, act)
    y, slope = policy.activation(g, act)
    # |act'| <= 1.13 for both; the activation itself is good to some 2^-20 of |g|
    tol = 1.13 * eg * (abs(u) + eu) + abs(y) * eu + 2.0 ** -20 * abs(g * u)
    close(out, want, tol + (2.0 ** -8 * abs(want) if dtype == "bf16" else 0.0), "h")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("m,k,f", FFN_SHAPES)
def test_ffn_backward(cuda, m, k, f, act, dtype):
    import gated_ffn

    x, wg, wu, dh = ffn_inputs(cuda, m, k, f, dtype, seed=1)
    got = gated_ffn.backward(dh, x, wg, wu, act)
    x, wg, wu, dh = to64(x), to64(wg), to64(wu), to64(dh)
    *want, dg, du = policy.ffn_grad(dh, x, wg, wu, act)
    g, u, eg, eu = ffn_errors(x, wg, wu, act)
    y, slope = policy.activation(g, act)
    # |act''| <= 0.8; dg and du pass through the inputs' type
    low = 2.0 ** -8 if dtype == "bf16" else 0.0
    edg = abs(dh) * (1.13 * eu + (abs(u) + eu) * 0.8 * eg + 2.0 ** -20 * abs(u) * (1 + abs(g))) + low * abs(dg)
    edu = abs(dh) * (1.13 * eg + 2.0 ** -20 * abs(g)) + low * abs(du)
    adg, adu = abs(dg) + edg, abs(du) + edu
    tols = (edg @ abs(wg.T) + edu @ abs(wu.T) + (2 * f + 8) * 2.0 ** -23 * (adg @ abs(wg.T) + adu @ abs(wu.T)),
            abs(x.T) @ edg + (m + 8) * 2.0 ** -23 * (abs(x.T) @ adg),
            abs(x.T) @ edu + (m + 8) * 2.0 ** -23 * (abs(x.T) @ adu))
    for name, a, w, tol in zip(("dx", "dw_gate", "dw_up"), got, want, tols):
        close(a, w, tol + low * abs(w), name)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("t,n,h,d", [(1, 200, 6, 16), (3, 200, 6, 16), (8, 100, 6, 32), (16, 75, 4, 64), (7, 50, 3, 128),
                                     (9, 50, 3, 128), (17, 200, 6, 16), (16, 200, 6, 16), (5, 20, 5, 64)])
def test_attention_of_few_tokens(cuda, t, n, h, d, dtype):
    test_attention_forward(cuda, t, n, h, d, dtype)
    test_attention_backward(cuda, t, n, h, d, dtype)


def test_attention_of_few_tokens_with_infinities(cuda):
    """What a reset cuts off is dropped, an infinity too, and other sequences see nothing of it."""
    import linear_attention as la

    (q, k, v, g), decay, state, gstate, resets = inputs(cuda, 6, 300, 2, 32, "f32", p_reset=0.0)
    resets[3, 1] = True
    bad = [x.clone() for x in (q, k, v, g)]
    for x in bad[1:3]:
        x[2, 1, 0] = float("inf")
    out, end = la.forward(bad[0], bad[1], bad[2], decay, state, resets)
    want, wend = la.forward(q, k, v, decay, state, resets)
    assert not torch.isfinite(out[2, 1, 0]).any()
    assert torch.equal(out[3:], want[3:]) and torch.equal(end, wend)
    assert torch.equal(out[:, [0, 2]], want[:, [0, 2]]) and torch.equal(out[:2], want[:2])
    bad = g.clone()
    bad[4, 1, 0] = float("inf")  # of the second episode: the first one's gradients do not see it
    got, want = la.backward(bad, q, k, v, decay, state, resets, None, gstate), la.backward(g, q, k, v, decay, state,
                                                                                       resets, None, gstate)
    for a, b in zip(got[:3], want[:3]):
        assert torch.equal(a[:3], b[:3]) and torch.equal(a[:, [0, 2]], b[:, [0, 2]])
    assert torch.equal(got[3], want[3]) and not torch.isfinite(got[0][4, 1, 0]).all()


def test_attention_states_off_the_vector_boundary(cuda):
    import linear_attention as la

    (q, k, v, g), decay, state, gstate, resets = inputs(cuda, 4, 600, 2, 16, "f32")
    flat = torch.empty(2 * state.numel() + 1, device=cuda)
    off, goff = (flat[1 + i * state.numel():][:state.numel()].view(state.shape) for i in (0, 1))
    off.copy_(state), goff.copy_(gstate)
    for a, b in zip(la.forward(q, k, v, decay, off, resets), la.forward(q, k, v, decay, state, resets)):
        assert torch.allclose(a, b, rtol=1e-5, atol=1e-5)
    for a, b in zip(la.backward(g, q, k, v, decay, off, resets, None, goff),
                    la.backward(g, q, k, v, decay, state, resets, None, gstate)):
        assert torch.allclose(a, b, rtol=1e-5, atol=1e-5)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("m,k,f", [(1, 97, 250), (2, 300, 77), (3, 64, 256), (5, 1, 5), (9, 129, 131), (32, 65, 1030),
                                   (33, 70, 68), (77, 31, 36), (128, 97, 250), (129, 97, 250)])
def test_ffn_backward_of_few_rows(cuda, m, k, f, dtype):
    test_ffn_backward(cuda, m, k, f, "gelu", dtype)


@pytest.mark.parametrize("m,k,f", [(300, 40, 200), (1500, 97, 250), (6000, 17, 129), (700, 128, 511), (2100, 250, 97)])
def test_ffn_backward_of_narrow_weights(cuda, m, k, f):
    """float32 weights' gradients formed as their transposes, whole and in parts, and a shape that is not."""
    test_ffn_backward(cuda, m, k, f, "silu", "f32")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("m,k,f", [(5000, 300, 520), (9000, 130, 70), (2600, 600, 260)])
def test_ffn_backward_dealt_unevenly(cuda, m, k, f, dtype):
    """Several tiles a pair of SMs, of both kinds and of unequal lengths."""
    test_ffn_backward(cuda, m, k, f, "gelu", dtype)


def test_ffn_gradient_of_few_rows_with_infinities(cuda):
    """Sums of products as the formula has them: what is not finite stays with its own token and column."""
    import gated_ffn

    x, wg, wu, dh = ffn_inputs(cuda, 3, 20, 23, "f32")
    want = gated_ffn.backward(dh, x, wg, wu)
    bad = dh.clone()
    bad[1, 22] = float("inf")
    dx, dwg, dwu = gated_ffn.backward(bad, x, wg, wu)
    assert not torch.isfinite(dx[1]).any() and torch.equal(dx[[0, 2]], want[0][[0, 2]])
    for got, w in ((dwg, want[1]), (dwu, want[2])):
        assert not torch.isfinite(got[:, 22]).any() and torch.equal(got[:, :22], w[:, :22])


def test_ffn_shapes_strides_and_empties(cuda):
    import gated_ffn

    x, wg, wu, dh = ffn_inputs(cuda, 60, 32, 48, "f32")
    want = gated_ffn.forward(x, wg, wu)
    assert torch.equal(gated_ffn.forward(x.view(3, 4, 5, 32), wg, wu), want.view(3, 4, 5, 48))
    assert torch.equal(gated_ffn.forward(x[7], wg, wu)[None], gated_ffn.forward(x[7:8], wg, wu))
    turned = wg.t().contiguous().t()
    assert torch.equal(gated_ffn.forward(x.t().contiguous().t(), turned, wu), want)
    off = torch.cat([torch.zeros(1, device=cuda), x.reshape(-1)])[1:].view(60, 32)  # off the 16-byte boundary
    assert torch.equal(gated_ffn.forward(off, wg, wu), want)
    for a, b in zip(gated_ffn.backward(dh, off, turned, wu), gated_ffn.backward(dh, x, wg, wu)):
        assert torch.equal(a, b)
    assert gated_ffn.forward(x[:0], wg, wu).shape == (0, 48)
    assert gated_ffn.forward(x[:, :0], wg[:0], wu[:0]).abs().sum() == 0
    assert [g.abs().sum().item() for g in gated_ffn.backward(dh[:0], x[:0], wg, wu)] == [0, 0, 0]
    leaves = [y.clone().requires_grad_() for y in (x, wg, wu)]
    (gated_ffn.apply(*leaves) * dh).sum().backward()
    for leaf, g in zip(leaves, gated_ffn.backward(dh, x, wg, wu)):
        assert torch.equal(leaf.grad, g)
    with pytest.raises(ValueError):
        gated_ffn.forward(x, wg[:3], wu)
    with pytest.raises(ValueError):
        gated_ffn.forward(x, wg, wu.bfloat16())
    with pytest.raises(ValueError):
        gated_ffn.forward(x, wg, wu, "relu6")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_ffn_rows_do_not_share_infinities(cuda, dtype):
    """A row with an infinity or NaN leaves the other rows' bits as they are, at sizes that end inside
    tiles; far-out values do not turn into NaN."""
    import gated_ffn

    for m, k, f in ((4, 32, 64), (300, 97, 250)):
        x, wg, wu, _ = ffn_inputs(cuda, m, k, f, dtype)
        want = gated_ffn.forward(x, wg, wu)
        bad = x.clone()
        bad[m - 1, k - 1], bad[m // 2, 0] = np.nan, np.inf
        out = gated_ffn.forward(bad, wg, wu)
        keep = [i for i in range(m) if i not in (m - 1, m // 2)]
        assert torch.equal(out[keep], want[keep]) and torch.isnan(out[m - 1]).all()
    big = torch.full((2, 32), 200.0, device=cuda).to(TYPES[dtype])
    w = torch.ones((32, 16), device=cuda).to(TYPES[dtype])
    for act in ("silu", "gelu"):
        assert torch.equal(gated_ffn.forward(big, -w, w, act), torch.zeros((2, 16), device=cuda).to(TYPES[dtype]) * -1)
        assert (gated_ffn.forward(big, w, w, act) == 6400.0 ** 2).all() if dtype == "f32" else True


# ---- AdamW ---------------------------------------------------------------------------------------------

def padded(tensors):
    return np.concatenate([np.pad(x.reshape(-1), (0, -x.size % policy.BLOCK)) for x in tensors])


def adam_inputs(cuda, sizes, dtype, seed, misaligned):
    g = torch.Generator(device=cuda).manual_seed(seed)

    def draw(n, scale, t):
        x = (torch.randn(n + 1, generator=g, device=cuda) * scale).to(t)
        return x[1:] if misaligned and n % 2 else x[:n].clone()

    return [draw(n, 0.1, torch.float32) for n in sizes], [draw(n, 1e-2, TYPES[dtype]) for n in sizes]


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("sizes", [(1,), (256, 255, 257), (3, 0, 1000, 77, 4096), tuple(range(1, 220))])
def test_adamw_steps(cuda, sizes, dtype, bits):
    """Three steps with different gradients. The moments' arithmetic is exactly rounded float32, so 8-bit
    codes must be equal; 32-bit moments too; the parameters are within the float32 error of an update."""
    import adamw

    f = np.float32
    params, _ = adam_inputs(cuda, sizes, dtype, 0, True)
    copies = [torch.zeros_like(p, dtype=torch.bfloat16) for p in params] if dtype == "bf16" else None
    state = adamw.init_state(params, bits, seed=77)
    lr, betas, eps, wd = 1e-2, (0.9, 0.999), 1e-8, 0.1
    scale = torch.tensor([0.5], device=cuda)
    p = padded([x.cpu().numpy() for x in params]).astype(np.float64)
    total = p.size
    m, v = np.zeros(total, f), np.zeros(total, f)
    for t in (1, 2, 3):
        _, grads = adam_inputs(cuda, sizes, dtype, t, True)
        adamw.step(params, grads, state, lr, betas, eps, wd, copies, scale)
        g = padded([x.float().cpu().numpy() for x in grads]) * f(0.5)
        m64, v64 = betas[0] * m.astype(float) + (1 - betas[0]) * g, betas[1] * v.astype(float) + (1 - betas[1]) * g.astype(float) ** 2
        m = m * f(betas[0]) + g * f(1 - betas[0])
        v = v * f(betas[1]) + (g * g) * f(1 - betas[1])
        rate, root = lr / (1 - betas[0] ** t), np.sqrt(v64 / (1 - betas[1] ** t)) + eps
        p = p * (1 - lr * wd) - rate * m64 / root
        if bits == 8:
            words = policy.rounding_words(total, 77, t)
            (cm, em), (cv, ev) = policy.encode(m, words & 0xFFFF, 4), policy.encode(v, words >> 16, 5)
            for name, want in (("m", cm), ("m_exp", em), ("v", cv), ("v_exp", ev)):
                assert (getattr(state, name).cpu().numpy() == want).all(), name
            m, v = policy.decode(cm, em, 4), policy.decode(cv, ev, 5)
        gm, gv = (x.cpu().numpy() for x in adamw.moments(state))
        assert (gm == m).all() and (gv == v).all()
        got = padded([to64(x) for x in params])
        # the update is at most some lr large: 16 roundings of it, and two of the parameter, a step
        tol = t * (2.0 ** -20 * (abs(rate * m64 / root) + lr) + 2.0 ** -22 * abs(p))
        assert (abs(got - p) <= tol).all(), abs(got - p).max()
    assert state.step == 3
    for c, x in zip(copies or [], params):
        assert torch.equal(c, x.to(torch.bfloat16))


@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_keeps_what_is_not_finite_to_itself(cuda, bits):
    import adamw

    p = [torch.ones(600, device=cuda)]
    g = [torch.full((600,), 0.1, device=cuda)]
    want, clean = [p[0].clone()], adamw.init_state(p, bits)
    adamw.step(want, g, clean)
    bad = [g[0].clone()]
    bad[0][5], bad[0][300] = np.nan, np.inf
    state = adamw.init_state(p, bits)
    adamw.step(p, bad, state)
    keep = torch.ones(600, dtype=torch.bool, device=cuda)
    keep[[5, 300]] = False
    assert torch.equal(p[0][keep], want[0][keep]) and not torch.isfinite(p[0][~keep]).any()
    for a, b in zip(adamw.moments(state), adamw.moments(clean)):
        assert torch.equal(a[:600][keep], b[:600][keep]) and not torch.isfinite(a[:600][~keep]).any()


def test_adamw_leaves_neighbours_alone(cuda):
    """Parameters that are views of one flat vector, gaps between them: the gaps keep their values, and a
    step over views is the step over copies."""
    import adamw

    flat = torch.randn(5000, device=cuda)
    before = flat.clone()
    cuts = [(3, 500), (501, 1001), (1500, 1501), (1777, 4999)]
    views = [flat[a:b] for a, b in cuts]
    own = [x.clone() for x in views]
    grads = [torch.randn_like(x) for x in own]
    for bits in (8, 32):
        s1, s2 = adamw.init_state(views, bits), adamw.init_state(own, bits)
        adamw.step(views, grads, s1)
        adamw.step(own, grads, s2)
        assert all(torch.equal(a, b) for a, b in zip(views, own)) and torch.equal(s1.m, s2.m)
    inside = torch.zeros(5000, dtype=torch.bool, device=cuda)
    for a, b in cuts:
        inside[a:b] = True
    assert torch.equal(flat[~inside], before[~inside])


def test_adamw_8bit_moments_follow_32bit_ones(cuda):
    """After 300 steps of noisy gradients the 8-bit second moment is right on average: each step's rounding
    errs by at most an eighth of v with zero mean, and v keeps 0.99 of it, so the errors' standard deviation
    is within v / 16 / sqrt(1 - 0.99^2) = 0.45 v; averaged over 2^16 elements, 6 deviations are 0.0105 of v's
    root mean square (chi-squared gradients: 1.02 of its mean)."""
    import adamw

    n = 1 << 16
    g = torch.Generator(device=cuda).manual_seed(3)
    p8, p32 = [torch.zeros(n, device=cuda)], [torch.zeros(n, device=cuda)]
    s8, s32 = adamw.init_state(p8, 8), adamw.init_state(p32, 32)
    for _ in range(300):
        grad = [torch.randn(n, generator=g, device=cuda)]
        adamw.step(p8, grad, s8, betas=(0.9, 0.99))
        adamw.step(p32, grad, s32, betas=(0.9, 0.99))
    v8, v32 = adamw.moments(s8)[1].double(), s32.v.double()
    assert abs((v8.mean() / v32.mean()).item() - 1) < 0.0115
    assert ((v8 / v32 - 1).abs() < 3).all() and ((v8 > 0) == (v32 > 0)).all()


def test_adamw_refusals(cuda):
    import adamw

    p, g = [torch.zeros(10, device=cuda)], [torch.zeros(10, device=cuda)]
    s = adamw.init_state(p)
    for args in [(p, [], s), (p, [g[0][:5]], s), (p, [g[0].double()], s), ([p[0].bfloat16()], g, s),
                 ([torch.zeros(20, device=cuda)[::2]], g, s), (p, g, adamw.init_state([p[0][:5]])),
                 (p, [g[0].cpu()], s), (p * 2, g * 2, s)]:
        with pytest.raises(ValueError):
            adamw.step(*args)
    with pytest.raises(ValueError):
        adamw.step(p, g, s, copies=[p[0]])
    with pytest.raises(ValueError):
        adamw.step(p, g, s, betas=(1.0, 0.9))
    with pytest.raises(ValueError):
        adamw.step(p, g, s, grad_scale=torch.ones(2, device=cuda))
    bad = adamw.init_state(p, 8)
    bad.m_exp = None
    with pytest.raises(ValueError):
        adamw.step(p, g, bad)
    assert s.step == 0 and p[0].abs().sum() == 0


def test_what_is_no_tensor_is_refused(cuda):
    import adamw
    import gated_ffn
    import linear_attention as la

    (q, k, v, g), decay, state, _, _ = inputs(cuda, 4, 1, 2, 16, "f32")
    for args in ((q, k, None, decay), (q, None, v, decay), (None, k, v, decay), (q, k, v, 0.9), (q, k, v, None),
                 (q, k, v, decay, 1.0), (q, k, v, decay, None, [True])):
        with pytest.raises(ValueError):
            la.forward(*args)
    with pytest.raises(ValueError):
        la.backward(None, q, k, v, decay)
    x, wg, wu, dh = ffn_inputs(cuda, 4, 8, 16, "f32")
    for args in ((None, wg, wu), (x, None, wu), (x, wg, None), (x, wg.cpu(), wu)):
        with pytest.raises(ValueError):
            gated_ffn.forward(*args)
    with pytest.raises(ValueError):
        gated_ffn.backward(None, x, wg, wu)
    params = [torch.zeros(4, device=cuda), torch.zeros(3, device=cuda)]
    grads, opt = [torch.ones_like(p) for p in params], adamw.init_state(params)
    for a, b, more in ((params, [grads[0], None], {}), (params, [None, None], {}), ([None, params[1]], grads, {}),
                       (params, grads, {"grad_scale": 0.5}), (params, grads, {"copies": [None, None]})):
        with pytest.raises(ValueError):
            adamw.step(a, b, opt, **more)
    assert opt.step == 0 and not params[0].any()


def test_second_derivatives_are_refused(cuda):
    import gated_ffn
    import linear_attention as la

    (q, k, v, _), decay, _, _, _ = inputs(cuda, 4, 1, 2, 16, "f32")
    x, wg, wu, _ = ffn_inputs(cuda, 4, 8, 16, "f32")
    for leaf, y in ((q.requires_grad_(), la.attend(q, k, v, decay)[0]), (x.requires_grad_(), gated_ffn.apply(x, wg, wu))):
        grad, = torch.autograd.grad(y.sum(), leaf, create_graph=True)
        with pytest.raises(RuntimeError):
            grad.sum().backward()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("blocks", [1, 2, 3, 5, 6, 7, 11, 12, 13])
def test_ffn_rings_filled_any_number_of_times(cuda, blocks, dtype):
    """A pair of SMs whose only tile fills its ring of five or six buffers less than once, exactly, once more, twice;
    the blocks of the pair end behind the last release of every buffer."""
    test_ffn_forward(cuda, 1200, 64 * blocks - 3, 520, "silu", dtype)
    test_ffn_backward(cuda, 257, 64 * blocks - 3, 264, "silu", dtype)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("d", [16, 32, 64, 128])
def test_attention_of_chunks_that_end_anywhere(cuda, d, dtype):
    """Rows and columns of a warp's tiles that are partly there, in the last of two chunks."""
    for t in (66, 71, 73, 80, 97, 111, 127):
        test_attention_forward(cuda, t, 1, 3, d, dtype)
    test_attention_backward(cuda, 75, 1, 3, d, dtype)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("m,k,f", [(450, 70, 530), (513, 64, 519), (700, 90, 390)])
def test_ffn_tiles_that_end_anywhere(cuda, m, k, f, dtype):
    """Tiles of which a warp's lanes have some rows and columns and not others."""
    test_ffn_forward(cuda, m, k, f, "gelu", dtype)
    test_ffn_backward(cuda, m, k, f, "gelu", dtype)


def test_a_state_stepped_before_the_backward_pass_is_noticed(cuda):
    """`attend` saves its state; `step` writes it in place, as autograd has to see."""
    import linear_attention as la

    (q, k, v, _), decay, state, _, _ = inputs(cuda, 5, 2, 2, 16, "f32")
    leaf = q.clone().requires_grad_()
    out, _ = la.attend(leaf, k, v, decay, state)
    version = state._version
    stepped = la.step(leaf[0], k[0], v[0], decay, state)
    assert state._version == version + 1 and not stepped.requires_grad
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.sum().backward()
    out, _ = la.attend(leaf, k, v, decay, state.clone())
    la.step(q[1], k[1], v[1], decay, state)
    out.sum().backward()
    assert leaf.grad is not None
    with torch.inference_mode():  # such tensors keep no versions
        la.step(q[0], k[0], v[0], decay, torch.zeros_like(state))


@pytest.mark.parametrize("bits", [32, 8])
def test_weights_stepped_before_the_backward_pass_are_noticed(cuda, bits):
    """`apply` saves the weights; `adamw.step` writes them and their copies in place, as autograd has to see."""
    import adamw
    import gated_ffn

    x, wg, wu, dh = ffn_inputs(cuda, 9, 16, 24, "f32")
    low = [w.to(torch.bfloat16).requires_grad_() for w in (wg, wu)]
    weights = [wg.requires_grad_(), wu.requires_grad_()]
    state = adamw.init_state(weights, bits)
    for used, inputs_ in ((weights, x), (low, x.to(torch.bfloat16))):
        out = gated_ffn.apply(inputs_, *used)
        versions = [w._version for w in weights + low + [state.m, state.v]]
        adamw.step(weights, [torch.ones_like(w) for w in weights], state, copies=[w.detach() for w in low])
        assert [w._version for w in weights + low + [state.m, state.v]] == [v + 1 for v in versions]
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            out.sum().backward()
    gated_ffn.apply(x, *weights).sum().backward()
    assert all(w.grad is not None for w in weights)
    with torch.no_grad():
        adamw.step([w.detach() for w in weights], [w.grad for w in weights], state)


@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_of_empty_tensors(cuda, bits):
    import adamw

    for sizes in ((0,), (0, 0), (0, 7)):
        params = [torch.ones(n, device=cuda) for n in sizes]
        state = adamw.init_state(params, bits)
        adamw.step(params, [torch.ones_like(p) for p in params], state)
        assert state.step == 1 and [x.numel() for x in adamw.moments(state)] == [256 * any(sizes)] * 2
        assert (params[-1] < 1).all()


def test_attention_takes_any_stride_of_an_axis_of_one(cuda):
    """One step, environment or head out of a tensor whose rows lie an odd number of elements apart."""
    import linear_attention as la

    decay = torch.tensor([0.9, 0.5, 0.7], device=cuda)
    for axis in range(3):
        shape = [1 if i == axis else n for i, n in enumerate((5, 4, 3))] + [16]
        strides = [0, 0, 0, 1]
        for i in range(2, -1, -1):
            strides[i] = strides[i + 1] * shape[i + 1]
        strides[axis] = 4097
        flat = torch.randn(8000, device=cuda)
        x = flat.as_strided(shape, strides)
        assert x.is_contiguous()
        y, g = torch.empty(shape, device=cuda).copy_(x), decay[:shape[2]]
        for a, b in zip(la.forward(x, x, x, g), la.forward(y, y, y, g)):
            assert torch.equal(a, b)
        for a, b in zip(la.backward(x, x, x, x, g), la.backward(y, y, y, y, g)):
            assert torch.equal(a, b)
        s, z = torch.ones((2, *shape[1:], 16), device=cuda)
        assert torch.equal(la.step(x[0], x[0], x[0], g, s), la.step(y[0], y[0], y[0], g, z)) and torch.equal(s, z)


def test_copies_that_a_call_makes_live_until_its_launch(cuda, monkeypatch):
    """A decay with strides is copied: memory taken from torch between the checks and the launch is not the copy's."""
    import linear_attention as la
    import rlenv_lib

    (q, k, v, g), _, state, _, _ = inputs(cuda, 3, 2, 4, 16, "f32")
    decay = torch.tensor([[0.9, 0.0], [0.5, 0.0], [0.7, 0.0], [0.1, 0.0]], device=cuda)[:, 0]
    states = [state.clone() for _ in range(2)]
    want = [la.step(q[0], k[0], v[0], decay.contiguous(), states[0]), *la.forward(q, k, v, decay.contiguous()),
            *la.backward(g, q, k, v, decay.contiguous())]
    launch, taken = rlenv_lib.launch, []

    def launch_late(index, entry, *args):
        taken.extend(torch.full((n,), 7.0, device=cuda) for n in (4, 4, 4, q.numel(), q[0].numel()))
        launch(index, entry, *args)

    monkeypatch.setattr(rlenv_lib, "launch", launch_late)
    got = [la.step(q[0], k[0], v[0], decay, states[1]), *la.forward(q, k, v, decay), *la.backward(g, q, k, v, decay)]
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and torch.equal(*states)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("eps", [0.0, 1e-16, 1e-13, 1e-8])
def test_adamw_of_tiny_gradients(cuda, bits, eps):
    """Gradients down to 1e-20, whose second moments lie below float32's smallest normal number: the update is the
    formula's for every epsilon, some lr without one. From parameters of zero, so that the update alone counts; its
    roundings, of root, product, sum and quotient, are some ulps of 2^-23 each."""
    import adamw

    f, n = np.float32, 1000
    g = np.geomspace(1e-20, 1e-16, n).astype(f) * np.where(np.arange(n) % 2, f(1), f(-1))
    params, lr, (b1, b2) = [torch.zeros(n, device=cuda)], 1e-3, (0.9, 0.999)
    adamw.step(params, [torch.from_numpy(g).to(cuda)], adamw.init_state(params, bits), lr, (b1, b2), eps, 0.0)
    m, v = (g * f(1 - b1)).astype(float), ((g * g) * f(1 - b2)).astype(float)
    assert (v > 0).all() and (v < 2.0 ** -126).any()
    want = -lr / (1 - b1) * m / (np.sqrt(v / (1 - b2)) + eps)
    assert (abs(to64(params[0]) - want) <= 2.0 ** -20 * abs(want)).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_infinities_of_long_sequences_are_the_definitions(cuda, dtype):
    """Without resets an infinity stays one, however long it decays, and is NaN where the decay is zero: in
    sequences that are split over the time axis too."""
    import linear_attention as la

    t, d = 4000, 16
    (q, k, v, do), _, state, gstate, _ = inputs(cuda, t, 1, 3, d, dtype, seed=9)
    q, k, v, do = (x.abs() for x in (q, k, v, do))
    decay = torch.tensor([0.9, 0.1, 0.0], device=cuda)  # 0.1^64 is below float32's smallest number
    for at in (3, 2000):
        bad = k.clone()
        bad[at, :, :, 1] = np.inf
        with np.errstate(invalid="ignore"):
            want, wend = policy.scan(to64(q), to64(bad), to64(v), to64(decay), None, None, d ** -0.5)
        out, end = la.forward(q, bad, v, decay)
        for got, w in ((out, want), (end, wend)):
            got = to64(got)
            assert (np.isposinf(got) == np.isposinf(w)).all() and (np.isnan(got) == np.isnan(w)).all()
        assert np.isposinf(wend[0, :2, 1]).all() and np.isnan(wend[0, 2, 1]).all()
    bad = do.clone()  # and from the last token to the first
    bad[t - 3, :, :, 2] = np.inf
    with np.errstate(invalid="ignore"):
        wants = policy.attention_grad(to64(bad), to64(q), to64(k), to64(v), to64(decay), None, None, d ** -0.5, None)
    for got, w in zip(la.backward(bad, q, k, v, decay), wants):
        got = to64(got)
        assert (np.isposinf(got) == np.isposinf(w)).all() and (np.isnan(got) == np.isnan(w)).all()


# ---- what the larger sizes reach ---------------------------------------------------------------------


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("sizes", [(700_001, 255, 1_300_007, 0, 3, 1_000_000, 77),
                                   (9, 300_000) * 20 + (1,)])
def test_adamw_of_more_blocks_than_warps(cuda, sizes, dtype, bits):
    """Warps that take several blocks of 256 elements, read ahead and cross from tensor to tensor: two steps against
    the definition in 64 bits, moments as in the small cases exactly."""
    import adamw

    f, lr, betas, eps, wd = np.float32, 1e-2, (0.9, 0.999), 1e-8, 0.1
    params, _ = adam_inputs(cuda, sizes, dtype, 0, True)
    copies = [torch.zeros_like(p, dtype=torch.bfloat16) for p in params]
    state = adamw.init_state(params, bits, seed=5)
    p = padded([x.cpu().numpy() for x in params]).astype(np.float64)
    assert p.size // 256 > 4736 and all(x.is_contiguous() for x in params)
    m, v = np.zeros(p.size, f), np.zeros(p.size, f)
    for t in (1, 2):
        _, grads = adam_inputs(cuda, sizes, dtype, t, True)
        adamw.step(params, grads, state, lr, betas, eps, wd, copies)
        g = padded([x.float().cpu().numpy() for x in grads])
        before = p
        p, m64, v64 = policy.adamw(p, g.astype(float), m.astype(float), v.astype(float), t, lr, betas, eps, wd)
        m = m * f(betas[0]) + g * f(1 - betas[0])
        v = v * f(betas[1]) + (g * g) * f(1 - betas[1])
        assert np.allclose(m, m64, rtol=1e-6, atol=1e-9) and np.allclose(v, v64, rtol=1e-6, atol=1e-12)
        if bits == 8:
            words = policy.rounding_words(p.size, 5, t)
            (cm, em), (cv, ev) = policy.encode(m, words & 0xFFFF, 4), policy.encode(v, words >> 16, 5)
            for name, want in (("m", cm), ("m_exp", em), ("v", cv), ("v_exp", ev)):
                assert (getattr(state, name).cpu().numpy() == want).all(), name
            m, v = policy.decode(cm, em, 4), policy.decode(cv, ev, 5)
        gm, gv = (x.cpu().numpy() for x in adamw.moments(state))
        assert (gm == m).all() and (gv == v).all()
        # the update is at most some lr large: 16 roundings of it, and two of the parameter, a step
        off = abs(padded([to64(x) for x in params]) - p)
        assert (off <= t * (2.0 ** -20 * (abs(p - before) + lr) + 2.0 ** -22 * abs(p))).all(), off.max()
    for c, x in zip(copies, params):
        assert torch.equal(c, x.to(torch.bfloat16))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("m,k,f", [(5000, 300, 520), (2100, 70, 2300), (20_000, 61, 173)])
def test_ffn_forward_of_several_tiles_a_pair(cuda, m, k, f, dtype):
    """More tiles than pairs of SMs: accumulators, rings and epilogues go on from tile to tile."""
    test_ffn_forward(cuda, m, k, f, "gelu", dtype)


@pytest.mark.parametrize("rows", [2, 700])
def test_ffn_of_large_bfloat16_values(cuda, rows):
    """By matrix-vector products and by tiles: 6400 x 6400 to half an ulp of bfloat16, 2^-8 of it at most."""
    import gated_ffn

    big = torch.full((rows, 32), 200.0, device=cuda, dtype=torch.bfloat16)
    w = torch.ones((32, 264), device=cuda, dtype=torch.bfloat16)
    for act in ("silu", "gelu"):
        out = gated_ffn.forward(big, w, w, act).double()
        assert ((out - 6400.0 ** 2).abs() <= 2.0 ** -8 * 6400.0 ** 2).all()
        assert not gated_ffn.forward(big, -w, w, act).any()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_attention_of_few_tokens_takes_any_strides(cuda, dtype):
    """Tokens one after the other, every operand with strides of its own: the bits of dense copies."""
    import linear_attention as la

    t, n, h, d = 5, 150, 4, 32
    g = torch.Generator(device=cuda).manual_seed(15)

    def draw(*shape):
        return torch.randn(shape, generator=g, device=cuda).to(TYPES[dtype])

    fused = draw(n, t, 3, h, d).transpose(0, 1)
    q, k = fused[:, :, 0], draw(h, t, n, d).permute(1, 2, 0, 3)
    v, do = draw(t, n, 1, d).expand(t, n, h, d), draw(t, h, n, d + 16)[..., 16:].transpose(1, 2)
    assert len({x.stride() for x in (q, k, v, do)}) == 4
    decay = torch.tensor([0.9, 0.99, 0.5, 0.0], device=cuda)
    state, gstate = torch.randn((2, n, h, d, d), generator=g, device=cuda)
    resets = (torch.rand((n, t), generator=g, device=cuda) < 0.1).t()
    for order in ((q, k, v, do), (k, v, do, q), (v, do, q, k), (do, q, k, v)):
        dense = [x.contiguous() for x in order]
        for a, b in zip(la.forward(*order[:3], decay, state, resets), la.forward(*dense[:3], decay, state, resets)):
            assert torch.equal(a, b)
        for a, b in zip(la.backward(*order, decay, state, resets, None, gstate),
                        la.backward(*dense, decay, state, resets, None, gstate)):
            assert torch.equal(a, b)
