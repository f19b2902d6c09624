"""The memory policy's operators in numpy, in 64 bits, from their definitions.

- `scan`: decayed linear attention token by token, and with `absolute` its terms' magnitudes
  summed instead (what rounding errors are measured against);
- `attention_grad`: its gradient, by the adjoint recurrence;
- `ffn`, `ffn_grad`: the gated feed-forward block;
- `norm`, `norm_grad`: the root-mean-square norm; `quantise`: rows in 8-bit integers;
- `scores`, `scores_grad`, `best`: log-probabilities of actions, entropy, alternatives;
- `adamw`: one step of AdamW; `encode`, `decode`: the 8-bit moments in float32, bit for bit.
"""

import math

import numpy as np

BLOCK = 256


def scan(q, k, v, decay, state, resets, scale, absolute=False):
    """(out (T, N, H, D), state): S <- keep g S + k'v, out = scale q S."""
    if absolute:
        q, k, v, state, scale = abs(q), abs(k), abs(v), None if state is None else abs(state), abs(scale)
    t, n, h, d = q.shape
    s = np.zeros((n, h, d, d)) if state is None else state.astype(np.float64)
    g = np.asarray(decay, np.float64)[:, None, None]
    out = np.zeros((t, n, h, d))
    for i in range(t):
        s = g * s
        if resets is not None:
            s = np.where(resets[i][:, None, None, None] != 0, 0.0, s)
        s = s + k[i][..., :, None] * v[i][..., None, :]
        out[i] = scale * np.einsum("nhd,nhde->nhe", q[i], s)
    return out, s


def attention_grad(do, q, k, v, decay, state, resets, scale, grad_state, absolute=False):
    """(dq, dk, dv, dstate) of sum(do * out) + sum(grad_state * final state)."""
    if absolute:
        do, q, k, v, scale = abs(do), abs(q), abs(k), abs(v), abs(scale)
        state, grad_state = (None if x is None else abs(x) for x in (state, grad_state))
    t, n, h, d = q.shape
    g = np.asarray(decay, np.float64)[:, None, None]

    def kept(i, x):
        x = g * x
        return x if resets is None else np.where(resets[i][:, None, None, None] != 0, 0.0, x)

    dq, dk, dv = (np.zeros((t, n, h, d)) for _ in range(3))
    s = np.zeros((n, h, d, d)) if state is None else state.astype(np.float64)
    for i in range(t):
        s = kept(i, s) + k[i][..., :, None] * v[i][..., None, :]
        dq[i] = scale * np.einsum("nhe,nhde->nhd", do[i], s)
    r = np.zeros((n, h, d, d)) if grad_state is None else grad_state.astype(np.float64)
    for i in range(t - 1, -1, -1):
        r = r + scale * q[i][..., :, None] * do[i][..., None, :]
        dk[i] = np.einsum("nhe,nhde->nhd", v[i], r)
        dv[i] = np.einsum("nhd,nhde->nhe", k[i], r)
        r = kept(i, r)
    return dq, dk, dv, r


_erf = np.vectorize(math.erf, otypes=[np.float64])


def activation(g, act):
    """act(g) and act'(g)."""
    if act == "silu":
        s = 0.5 * (1.0 + np.tanh(0.5 * g))
        return g * s, s + g * s * (1.0 - s)
    cdf = 0.5 * (1.0 + _erf(g / math.sqrt(2.0)))
    return g * cdf, cdf + g * np.exp(-0.5 * g * g) / math.sqrt(2.0 * math.pi)


def ffn(x, wg, wu, act):
    return activation(x @ wg, act)[0] * (x @ wu)


def ffn_grad(dh, x, wg, wu, act):
    """(dx, dwg, dwu, dg, du)"""
    y, slope = activation(x @ wg, act)
    dg, du = dh * (x @ wu) * slope, dh * y
    return dg @ wg.T + du @ wu.T, x.T @ dg, x.T @ du, dg, du


def norm(t, w, eps):
    """t / sqrt(mean(t^2) + eps) * w over the last axis; w None: ones."""
    out = t / np.sqrt((t * t).mean(-1, keepdims=True) + eps)
    return out if w is None else out * w


def norm_grad(g, t, w, eps, gt=None, absolute=False):
    """(dt, dw) of sum(g * norm(t, w)) + sum(gt * t); with `absolute` the sums of their terms' magnitudes."""
    if absolute:
        g, t, w, gt = (None if x is None else abs(x) for x in (g, t, w, gt))
    k = t.shape[-1]
    r = 1.0 / np.sqrt((t * t).mean(-1, keepdims=True) + eps)
    gw = g if w is None else g * w
    along = r ** 3 * (gw * t).sum(-1, keepdims=True) / k * t
    dt = r * gw + along if absolute else r * gw - along
    return dt if gt is None else dt + gt, (g * t * r).reshape(-1, k).sum(0)


def quantise(y):
    """(whole numbers, scale) of rows: the largest magnitude is 127 steps."""
    top = abs(y).max(-1, keepdims=True)
    some = top >= 2.0 ** -100
    return np.where(some, np.rint(y * 127 / np.where(some, top, 1.0)), 0.0), np.where(some, top / 127, 0.0)[..., 0]


def scores(l, actions, allowed=None):
    """(log_prob, entropy, normalizer, log-probabilities (..., A)) of logits l (..., A)."""
    l = l if allowed is None else np.where(allowed, l, -np.inf)
    with np.errstate(divide="ignore", invalid="ignore"):
        top = l.max(-1, keepdims=True)
        base = np.where(top == -np.inf, 0.0, top)
        e = np.exp(l - base)
        s = e.sum(-1, keepdims=True)
        normalizer = base + np.log(s)
        lp = np.where(l == -np.inf, -np.inf, l - normalizer)
        entropy = np.where(s > 0, np.log(s) - np.where(e > 0, e * (l - base), 0.0).sum(-1, keepdims=True) / s, 0.0)
    chosen = np.take_along_axis(lp, np.maximum(actions, 0)[..., None], -1)[..., 0]
    return np.where(actions < 0, 0.0, chosen), entropy[..., 0], normalizer[..., 0], lp


def scores_grad(g, h, l, actions, allowed=None):
    """The gradient of sum(g * log_prob) + sum(h * entropy)."""
    _, entropy, _, lp = scores(l, actions, allowed)
    some = lp > -np.inf  # not p > 0: the chosen action has a gradient where its p is below 64 bits' numbers too
    p, lp = np.exp(lp), np.where(some, lp, 0.0)
    chosen = np.arange(l.shape[-1]) == actions[..., None]
    grad = np.where(actions < 0, 0.0, g)[..., None] * (chosen - p) - h[..., None] * p * (lp + entropy[..., None])
    return np.where(some, grad, 0.0)


def best(l, n, allowed=None):
    """Places (..., n) of the largest logits, ties to the lower place."""
    l = l if allowed is None else np.where(allowed, l, -np.inf)
    return np.argsort(-l, -1, kind="stable")[..., :n]


def adamw(p, g, m, v, step, lr, betas, eps, weight_decay):
    """(p, m, v) after step number `step` (from 1)."""
    b1, b2 = betas
    m, v = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
    update = lr * (m / (1 - b1 ** step)) / (np.sqrt(v / (1 - b2 ** step)) + eps)
    return p - lr * weight_decay * p - update, m, v


# ---- 8-bit moments ---------------------------------------------------------------------------------

def pcg_hash(v):
    """The environments' reset hash on uint32 arrays."""
    v = np.asarray(v, np.uint32)
    with np.errstate(over="ignore"):
        s = v * np.uint32(747796405) + np.uint32(2891336453)
        w = ((s >> ((s >> np.uint32(28)) + np.uint32(4))) ^ s) * np.uint32(277803737)
    return (w >> np.uint32(22)) ^ w


def rounding_words(total, seed, step):
    key = pcg_hash(np.uint32((seed ^ (step * 0x9E3779B9)) & 0xFFFFFFFF))
    return pcg_hash(np.arange(total, dtype=np.uint32) ^ key)


def encode(x, rand16, ebits):
    """(codes, exponents) of float32 x, a multiple of BLOCK long."""
    bits = (x.view(np.uint32) & 0x7FFFFFFF).astype(np.int64)
    top = (1 << (ebits + 3)) - 1
    finite = np.where(bits < 0x7F800000, bits, 0).reshape(-1, BLOCK)
    e = np.maximum((finite.max(1) + 0x1FFFFF) >> 23, 32)
    c = ((bits + (rand16.astype(np.int64) << 4)) >> 20) - np.repeat(e - ((1 << ebits) - 1), BLOCK) * 8
    c = np.maximum(c, 0)
    if ebits == 5:
        c = np.where(bits > 0, np.maximum(c, 1), c)
    c = np.where(bits < 0x7F800000, c, top)
    if ebits == 4:
        c = c | np.where(x.view(np.int32) < 0, 128, 0)
    return c.astype(np.uint8), e.astype(np.uint8)


def decode(codes, e, ebits):
    top = (1 << (ebits + 3)) - 1
    mag = codes.astype(np.int64) & top
    bits = (mag + np.repeat(e.astype(np.int64) - ((1 << ebits) - 1), BLOCK) * 8) << 20
    x = np.where(mag == 0, 0, bits).astype(np.uint32).view(np.float32)
    x = np.where(mag == top, np.float32(np.nan), x)
    return np.where(codes > 127, -x, x).astype(np.float32) if ebits == 4 else x
