"""What stands around the memory of a policy, as it is measured: the root-mean-square norm with the
residual's addition (its gradient, and its output in 8 bits), products of 8-bit integers with scales for
each token and channel, and the log-probabilities of chosen actions with their entropy and the best
alternatives (and their gradient).

Each case can be computed in two ways on the same inputs: in plain torch operations, or by the
framework's kernels (`own`). `exact` gives the results from the definitions in 64 bits.

Rows are tokens: T steps of N environments in the framework's trajectories (500 x 256 of them in the
batches), one in the smallest acting calls. Weights of 8-bit products are held channel by channel, rows on
16-byte boundaries.
"""

import math
import sys
from pathlib import Path

import torch

own = False

_ROOT = Path(__file__).resolve().parent.parent
_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
_SIZE = {"f32": 4, "bf16": 2}
_EPS = 1e-6
_TINY = 2.0 ** -100  # rows whose largest magnitude is below are zero in 8 bits
_SPAN = 1024         # terms of a product of 8-bit integers whose float32 sum is exact: 1024 x 127 x 127 < 2^24


def _framework():
    """The framework's modules (a flat directory, imported by bare name)."""
    pkg = str(_ROOT / "metal-rl-envs_b200")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import int8_linear
    import log_probs
    import rms_norm
    return rms_norm, int8_linear, log_probs


# ---- cases -------------------------------------------------------------------------------------

def listed():
    return [
        # one environment acting: a single token's norm between two layers, all latency
        {"name": "norm_one", "op": "norm", "m": 1, "k": 1024, "dtype": "bf16", "residual": True},
        # the norm over collected rollouts (500 steps of 256 environments), 8 heads of 64: a stream of memory
        {"name": "norm_rollouts", "op": "norm", "m": 128_000, "k": 512, "dtype": "bf16", "residual": True},
        # its gradient, with the gradient that comes down the residual stream
        {"name": "norm_rollouts_grad", "op": "norm_grad", "m": 128_000, "k": 512, "dtype": "bf16", "stream": True},
        # the gradient over 500 x 37 tokens in float32, of a width that no vector load divides
        {"name": "norm_ragged_grad", "op": "norm_grad", "m": 18_500, "k": 97, "dtype": "f32", "stream": False},
        # one token through an 8-bit matrix: bounded by reading the weights, or by latency where L2 holds them
        {"name": "product_one", "op": "product8", "m": 1, "k": 1024, "f": 4096, "dtype": "bf16"},
        # a large batch of tokens: the tensor cores' rate
        {"name": "product_batch", "op": "product8", "m": 16_384, "k": 4096, "f": 4096, "dtype": "bf16"},
        # a few hundred environments acting through norm and product at odd sizes, float32 activations
        {"name": "layer_ragged", "op": "layer8", "m": 300, "k": 1000, "f": 2720, "dtype": "f32"},
        # a training batch of environments acting: norm, 8-bit activations, product
        {"name": "layer_batch", "op": "layer8", "m": 8192, "k": 1024, "f": 4096, "dtype": "bf16"},
        # one environment with a large discrete set of actions: chosen action, entropy and the best eight
        {"name": "scores_one", "op": "scores", "m": 1, "v": 50_021, "dtype": "bf16", "top": 8, "masked": False,
         "beside": 0, "padded": False},
        # CartPole's two actions over collected rollouts, the value's column beside them as the policy's head has it
        {"name": "scores_cartpole", "op": "scores", "m": 128_000, "v": 2, "dtype": "f32", "top": 0, "masked": False,
         "beside": 1, "padded": False},
        # a batch over a large set of actions with the best eight: one stream of logits
        {"name": "scores_large", "op": "scores", "m": 4096, "v": 32_768, "dtype": "bf16", "top": 8, "masked": False,
         "beside": 0, "padded": False},
        # the gradient over such a set, some actions not allowed, rows that start anywhere, padded tokens
        {"name": "scores_large_grad", "op": "scores_grad", "m": 4096, "v": 32_771, "dtype": "bf16", "top": 0,
         "masked": True, "beside": 0, "padded": True},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _draw_once(rng):
    op = rng.choice(["norm", "norm_grad", "product8", "layer8", "scores", "scores_grad"])
    dtype = rng.choice(["f32", "bf16"])
    if op in ("norm", "norm_grad"):
        # widths of eights as models have them, and odd ones
        k = _log_int(rng, 8, 16_384)
        k = k if rng.random() < 0.5 else -(-k // 8) * 8
        case = {"op": op, "m": _log_int(rng, 1, 131_072), "k": k, "dtype": dtype}
        case["residual" if op == "norm" else "stream"] = rng.random() < 0.6
        return case
    if op in ("product8", "layer8"):
        k, f = _log_int(rng, 16, 8192), _log_int(rng, 16, 8192)
        if rng.random() < 0.5:
            k, f = -(-k // 32) * 32, -(-f // 32) * 32
        return {"op": op, "m": _log_int(rng, 1, 16_384), "k": k, "f": f, "dtype": dtype}
    v = _log_int(rng, 2, 131_072)
    top = rng.choice([0, 1, 4, 8, 20]) if op == "scores" else 0
    return {"op": op, "m": _log_int(rng, 1, 262_144), "v": v, "dtype": dtype, "top": min(top, v),
            "masked": rng.random() < 0.4, "beside": rng.choice([0, 0, 1]), "padded": rng.random() < 0.3}


def draw(rng):
    """A case of the listed ones' ranges that costs no more than the largest of its operator's."""
    family = {"norm": ("norm", "norm_grad"), "norm_grad": ("norm", "norm_grad"), "product8": ("product8",),
              "layer8": ("layer8",), "scores": ("scores", "scores_grad"), "scores_grad": ("scores", "scores_grad")}
    while True:
        case = _draw_once(rng)
        most = [work(c) for c in listed() if c["op"] in family[case["op"]]]
        w = work(case)
        if w["bytes"] <= max(m["bytes"] for m in most) and w["flops"] <= max(m["flops"] for m in most):
            return case


def work(case):
    """Bytes that a pass has to read and write once, and its operations (a multiply-add is two)."""
    c, op, size = case, case["op"], _SIZE[case["dtype"]]
    if op == "norm":  # x, the result; with a residual that and the sum
        return {"bytes": c["m"] * c["k"] * float(size) * (4 if c["residual"] else 2) + c["k"] * size,
                "flops": c["m"] * c["k"] * 5.0}
    if op == "norm_grad":  # the sum, its norm's gradient, the result; the stream's gradient
        return {"bytes": c["m"] * c["k"] * float(size) * (4 if c["stream"] else 3) + 2 * c["k"] * size,
                "flops": c["m"] * c["k"] * 12.0}
    if op == "product8":
        return {"bytes": float(c["m"] * c["k"] + c["f"] * c["k"] + c["m"] * c["f"] * size + 4 * (c["m"] + c["f"])),
                "flops": 2.0 * c["m"] * c["k"] * c["f"]}
    if op == "layer8":  # x, the residual and the sum; the weights; the product in bfloat16
        return {"bytes": c["m"] * c["k"] * 3.0 * size + c["f"] * c["k"] + c["m"] * c["f"] * 2.0 + 4 * c["f"]
                + c["k"] * size, "flops": c["m"] * c["k"] * (2.0 * c["f"] + 7.0)}
    cells = c["m"] * c["v"]
    per = size + (1 if c["masked"] else 0)
    if op == "scores":  # logits; actions; log-probability, entropy, normalizer; the alternatives
        return {"bytes": float(cells * per + c["m"] * (8 + 12 + 12 * c["top"])), "flops": cells * 6.0}
    return {"bytes": float(cells * (per + size) + c["m"] * (8 + 16)), "flops": cells * 8.0}


# ---- inputs ------------------------------------------------------------------------------------

def _codes_buffer(rows, cols):
    """(rows, cols) 8-bit integers with rows on 16-byte boundaries."""
    return torch.zeros((rows, -(-cols // 16) * 16), dtype=torch.int8, device="cuda")[:, :cols]


def _quantised(y):
    """8-bit integers and scales of the rows of y (float32)."""
    largest = y.abs().amax(-1, keepdim=True)
    some = (largest >= _TINY) & (largest < math.inf)
    codes = torch.where(some, torch.round(y * torch.where(some, 127.0 / largest, 0.0)), 0.0)
    scale = torch.where(some, largest / 127.0, torch.where(largest < _TINY, 0.0, math.nan))
    return codes, scale[..., 0]


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    op, dtype = case["op"], _TYPES[case["dtype"]]

    def normal(*shape, scale=1.0, dtype=dtype):
        return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)

    s = {"case": dict(case)}
    m = case["m"]
    if op in ("norm", "norm_grad", "layer8"):
        k = case["k"]
        s["weight"] = (1.0 + 0.2 * torch.randn(k, generator=g, device="cuda")).to(dtype)
        # a residual stream that has grown over its layers, and what a layer adds
        if op == "norm_grad":
            s["total"], s["grad"] = normal(m, k, scale=3.0), normal(m, k)
            s["stream"] = normal(m, k) if case["stream"] else None
        else:
            s["x"] = normal(m, k)
            s["residual"] = normal(m, k, scale=3.0) if case.get("residual", True) else None
    if op in ("product8", "layer8"):
        k, f = case["k"], case["f"]
        codes, s["w_scale"] = _quantised(normal(f, k, scale=k ** -0.5, dtype=torch.float32))
        s["w_codes"] = _codes_buffer(f, k)
        s["w_codes"].copy_(codes)
    if op == "product8":
        codes, s["scale"] = _quantised(normal(m, k, dtype=torch.float32))
        s["codes"] = _codes_buffer(m, k)
        s["codes"].copy_(codes)
    if op in ("scores", "scores_grad"):
        v = case["v"]
        s["logits"] = normal(m, v + case["beside"], scale=2.0)[:, :v]
        s["allowed"] = None
        if case["masked"]:
            s["allowed"] = torch.rand((m, v), generator=g, device="cuda") < 0.7
            s["allowed"] &= torch.rand((m, 1), generator=g, device="cuda") >= 0.01  # rows that allow nothing
        # the chosen actions, drawn from the policy
        noise = torch.empty((m, v), device="cuda").exponential_(generator=g)
        drawn = s["logits"].float() - torch.log(noise)
        s["actions"] = (drawn if s["allowed"] is None else torch.where(s["allowed"], drawn, -math.inf)).argmax(-1)
        if case["padded"]:
            s["actions"][torch.rand(m, generator=g, device="cuda") < 0.1] = -1
        if op == "scores_grad":
            s["normalizer"], s["entropy"] = _plain_normalizer(_effective(s))[:2]
            s["grad"] = torch.randn(m, generator=g, device="cuda") / m
            s["grad_entropy"] = torch.full((m,), -0.01 / m, device="cuda")
    return s


# ---- the plain forms ---------------------------------------------------------------------------

def _plain_total(s):
    total = s["x"].float()
    return total if s["residual"] is None else total + s["residual"].float()


def _plain_norm_values(s, total):
    return total * torch.rsqrt(total.square().mean(-1, keepdim=True) + _EPS) * s["weight"].float()


def _plain_norm(s):
    total = _plain_total(s)
    out = _plain_norm_values(s, total).to(s["x"].dtype)
    return {"out": out} if s["residual"] is None else {"out": out, "total": total.to(s["x"].dtype)}


def _plain_norm_grad(s):
    total, g = s["total"].float(), s["grad"].float()
    r = torch.rsqrt(total.square().mean(-1, keepdim=True) + _EPS)
    unit, gw = total * r, g * s["weight"].float()
    grad = r * (gw - unit * (gw * unit).mean(-1, keepdim=True))
    if s["stream"] is not None:
        grad = grad + s["stream"].float()
    return {"grad": grad.to(s["total"].dtype), "grad_weight": (g * unit).sum(0).to(s["weight"].dtype)}


def _plain_product(codes, scale, w_codes, w_scale, dtype):
    """Sums of _SPAN terms in float32, which are whole numbers below 2^24, and their sum in 64 bits."""
    m, k = codes.shape
    spans = -(-k // _SPAN)

    def split(c):
        c = torch.nn.functional.pad(c.float(), (0, spans * _SPAN - k))
        return c.reshape(c.shape[0], spans, _SPAN).transpose(0, 1)

    if spans == 1:
        sums = codes.float() @ w_codes.float().t()
    else:
        sums = (split(codes) @ split(w_codes).transpose(1, 2)).sum(0, dtype=torch.float64).float()
    return (sums * scale[:, None] * w_scale).to(dtype)


def _plain_product8(s):
    return {"out": _plain_product(s["codes"], s["scale"], s["w_codes"], s["w_scale"], _TYPES[s["case"]["dtype"]])}


def _plain_layer8(s):
    total = _plain_total(s)
    codes, scale = _quantised(_plain_norm_values(s, total))
    return {"out": _plain_product(codes, scale, s["w_codes"], s["w_scale"], torch.bfloat16),
            "total": total.to(s["x"].dtype)}


def _effective(s):
    """Logits in 32 bits, -infinity where an action is not allowed."""
    l = s["logits"].float()
    return l if s["allowed"] is None else torch.where(s["allowed"], l, -math.inf)


def _plain_normalizer(l):
    """(normalizer, entropy, log-probabilities) of rows: -infinity, 0 and -infinities where nothing is allowed."""
    top = l.amax(-1, keepdim=True)
    top = torch.where(top > -math.inf, top, 0.0)
    away = l - top
    e = torch.exp(away)
    total = e.sum(-1)
    normalizer = top[:, 0] + torch.log(total)
    weighed = torch.where(e > 0, e * away, 0.0).sum(-1)
    entropy = torch.where(total > 0, torch.log(total) - weighed / total, 0.0)
    return normalizer, entropy, torch.where(l > -math.inf, l - normalizer[:, None], -math.inf)


def _plain_top(l, k):
    """Places of each row's k largest values, ties to the lowest place: one whole number a value, ordered by the
    value and then by the place."""
    bits = (l + 0.0).view(torch.int32)
    order = torch.where(bits >= 0, bits, bits ^ 0x7FFFFFFF).to(torch.int64)
    key = (order << 32) + (0xFFFFFFFF - torch.arange(l.shape[1], device=l.device))
    return 0xFFFFFFFF - (torch.topk(key, k, -1).values & 0xFFFFFFFF)


def _plain_scores(s):
    l, actions = _effective(s), s["actions"]
    normalizer, entropy, logp = _plain_normalizer(l)
    chosen = logp.gather(-1, actions.clamp(min=0)[:, None])[:, 0]
    out = {"log_prob": torch.where(actions < 0, 0.0, chosen), "entropy": entropy, "normalizer": normalizer}
    if s["case"]["top"]:
        out["top_actions"] = _plain_top(l, s["case"]["top"])
        out["top_log_probs"] = logp.gather(-1, out["top_actions"])
    return out


def _plain_scores_grad(s):
    l, actions = _effective(s), s["actions"]
    some = (l > -math.inf) & (s["normalizer"] > -math.inf)[:, None]
    logp = torch.where(some, l - s["normalizer"][:, None], 0.0)
    p = torch.where(some, torch.exp(logp), 0.0)
    g = torch.where(actions < 0, 0.0, s["grad"])[:, None]
    chosen = (torch.arange(l.shape[1], device=l.device) == actions[:, None]) & some
    grad = g * (chosen.float() - p) - s["grad_entropy"][:, None] * p * (logp + s["entropy"][:, None])
    return {"grad": grad.to(s["logits"].dtype)}


# ---- the framework's kernels ---------------------------------------------------------------------

def _own(s):
    rms_norm, int8_linear, log_probs = _framework()
    op = s["case"]["op"]
    if op == "norm":
        out, total = rms_norm.forward(s["x"], s["weight"], s["residual"], _EPS)
        return {"out": out} if s["residual"] is None else {"out": out, "total": total}
    if op == "norm_grad":
        grad, grad_weight = rms_norm.backward(s["grad"], s["total"], s["weight"], _EPS, s["stream"])
        return {"grad": grad, "grad_weight": grad_weight}
    if op == "product8":
        weight = int8_linear.Weight(s["w_codes"], s["w_scale"])
        return {"out": int8_linear.forward(s["codes"], s["scale"], weight, _TYPES[s["case"]["dtype"]])}
    if op == "layer8":
        codes, scale, total = rms_norm.forward8(s["x"], s["weight"], s["residual"], _EPS)
        weight = int8_linear.Weight(s["w_codes"], s["w_scale"])
        return {"out": int8_linear.forward(codes, scale, weight, torch.bfloat16), "total": total}
    if op == "scores":
        got = log_probs.forward(s["logits"], s["actions"], s["allowed"], s["case"]["top"])
        out = {"log_prob": got.log_prob, "entropy": got.entropy, "normalizer": got.normalizer}
        if s["case"]["top"]:
            out["top_actions"], out["top_log_probs"] = got.top_actions, got.top_log_probs
        return out
    return {"grad": log_probs.backward(s["grad"], s["grad_entropy"], s["logits"], s["actions"], s["normalizer"],
                                       s["entropy"], s["allowed"])}


def run(state):
    if own:
        return _own(state)
    op = state["case"]["op"]
    if op == "norm":
        return _plain_norm(state)
    if op == "norm_grad":
        return _plain_norm_grad(state)
    if op == "product8":
        return _plain_product8(state)
    if op == "layer8":
        return _plain_layer8(state)
    if op == "scores":
        return _plain_scores(state)
    return _plain_scores_grad(state)


# ---- the definitions in 64 bits ------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    d = {n: x.double() for n, x in s.items() if isinstance(x, torch.Tensor) and x.is_floating_point()}
    if op in ("norm", "layer8"):
        total = d["x"] + d["residual"] if "residual" in d else d["x"]
        out = total / (total.pow(2).sum(1, keepdim=True) / case["k"] + _EPS).sqrt() * d["weight"]
        if op == "norm":
            return {"out": out, "total": total} if "residual" in d else {"out": out}
        step = out.abs().max(1, keepdim=True).values / 127
        codes = torch.where(step > 0, (out / step).round(), 0.0)
        return {"out": (codes * step) @ (s["w_codes"].double() * d["w_scale"][:, None]).t(), "total": total}
    if op == "norm_grad":
        # with r(t) = (t't / K + eps)^-1/2: d(w r t)/dt = w r - r^3 (w t) t' / K
        t, k = d["total"], case["k"]
        r = (t.pow(2).sum(1, keepdim=True) / k + _EPS) ** -0.5
        seen = d["grad"] * d["weight"]
        grad = r * seen - r ** 3 * t * (seen * t).sum(1, keepdim=True) / k
        return {"grad": grad + d["stream"] if "stream" in d else grad,
                "grad_weight": torch.einsum("mk,mk->k", d["grad"], r * t)}
    if op == "product8":
        return {"out": (s["codes"].double() * d["scale"][:, None]) @ (s["w_codes"].double() * d["w_scale"][:, None]).t()}
    l = d["logits"]
    if s["allowed"] is not None:
        l = l.masked_fill(~s["allowed"], -math.inf)
    normalizer = torch.logsumexp(l, -1)
    logp = l - normalizer.clamp(min=-1e300)[:, None]
    p = logp.exp()
    entropy = -(p * logp.clamp(min=-1e300)).sum(-1)
    chosen = torch.zeros_like(p).scatter_(1, s["actions"].clamp(min=0)[:, None], 1.0)
    real = (s["actions"] >= 0).double()
    if op == "scores":
        rows = torch.arange(case["m"], device="cuda")
        picked = logp[rows, s["actions"].clamp(min=0)]
        out = {"log_prob": torch.where(real > 0, picked, 0.0), "entropy": entropy, "normalizer": normalizer}
        if case["top"]:
            places = torch.sort(l, dim=-1, descending=True, stable=True).indices[:, :case["top"]]
            out["top_actions"], out["top_log_probs"] = places, logp.gather(1, places)
        return out
    by_choice = (d["grad"] * real)[:, None] * (chosen - p)
    by_entropy = -d["grad_entropy"][:, None] * p * (logp.clamp(min=-1e300) + entropy[:, None])
    grad = by_choice + by_entropy
    live = (l > -math.inf) & (normalizer > -math.inf)[:, None]
    return {"grad": torch.where(live, grad, 0.0)}
