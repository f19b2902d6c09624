"""The operators of a memory policy, as they are measured: a decayed linear attention over
trajectories (with its gradient, and its one-token form for acting), a gated feed-forward block
(with its gradient), and the AdamW step that trains both.

Each case can be computed in two ways on the same inputs: in plain torch operations in 32 bits,
or by the framework's kernels (`own`). `exact` gives the results from the definitions in 64 bits.

Shapes are the framework's: trajectories are time-major, T steps of N environments (as the
`rewards` and `dones` of its step_many calls), with H heads of width D per token; weights are
(in, out), as es.unflatten's.
"""

import math
import sys
from pathlib import Path

import torch

own = False

_ROOT = Path(__file__).resolve().parent.parent
_CHUNK = 64    # tokens per chunk of the plain trajectory form
_BLOCK = 256   # elements per block of the 8-bit optimizer state

_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
_SIZE = {"f32": 4, "bf16": 2}


def _framework():
    """The framework's modules (a flat directory, imported by bare name)."""
    pkg = str(_ROOT / "metal-rl-envs_b200")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import adamw
    import gated_ffn
    import linear_attention
    return linear_attention, gated_ffn, adamw


# ---- cases -------------------------------------------------------------------------------------

def listed():
    return [
        # one environment acting: the lowest latency a policy sees, float32 as the environments are
        {"name": "attend_step_one", "op": "attend_step", "n": 1, "h": 4, "d": 32, "dtype": "f32", "p_reset": 0.0},
        # a training batch of environments acting, some of them just reset: a stream of states
        {"name": "attend_step_batch", "op": "attend_step", "n": 4096, "h": 8, "d": 64, "dtype": "bf16",
         "p_reset": 0.01},
        # collected CartPole-length rollouts (500 steps), episodes ending inside them
        {"name": "attend_rollouts", "op": "attend_forward", "t": 500, "n": 256, "h": 8, "d": 64, "dtype": "bf16",
         "p_reset": 0.01, "carry": True},
        # one long history, no resets: little to split but the time axis; float32
        {"name": "attend_history", "op": "attend_forward", "t": 16384, "n": 1, "h": 8, "d": 128, "dtype": "f32",
         "p_reset": 0.0, "carry": False},
        # the gradient over a training batch of rollouts
        {"name": "attend_rollouts_grad", "op": "attend_backward", "t": 500, "n": 128, "h": 8, "d": 64,
         "dtype": "bf16", "p_reset": 0.01, "carry": True},
        # the gradient at odd sizes in float32, short episodes (a reset every 20 steps or so)
        {"name": "attend_ragged_grad", "op": "attend_backward", "t": 203, "n": 77, "h": 3, "d": 32, "dtype": "f32",
         "p_reset": 0.05, "carry": True},
        # one token through the block: a matrix-vector product, bounded by reading the weights
        {"name": "ffn_one", "op": "ffn_forward", "m": 1, "k": 1024, "f": 4096, "dtype": "bf16", "act": "silu"},
        # a large batch of tokens forward
        {"name": "ffn_batch", "op": "ffn_forward", "m": 16384, "k": 1024, "f": 4096, "dtype": "bf16", "act": "silu"},
        # its gradient, a width that ends inside a tile
        {"name": "ffn_batch_grad", "op": "ffn_backward", "m": 8192, "k": 1024, "f": 2720, "dtype": "bf16",
         "act": "silu"},
        # the gradient of a small policy's block over 500 x 37 tokens in float32, widths that no vector load divides
        {"name": "ffn_ragged_grad", "op": "ffn_backward", "m": 18500, "k": 97, "f": 250, "dtype": "f32",
         "act": "gelu"},
        # a policy's sixty small tensors, state in 32 bits: latency
        {"name": "adamw_policy", "op": "adamw", "tensors": 60, "total": 100_000, "bits": 32, "dtype": "f32",
         "copies": False, "step": 10},
        # a large model: bf16 gradients, 8-bit state, bf16 working copies of the weights written in the same step
        {"name": "adamw_large_8bit", "op": "adamw", "tensors": 24, "total": 60_000_000, "bits": 8, "dtype": "bf16",
         "copies": True, "step": 1000},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _draw_once(rng):
    op = rng.choice(["attend_step", "attend_forward", "attend_backward", "ffn_forward", "ffn_backward", "adamw"])
    dtype = rng.choice(["f32", "bf16"])
    if op == "attend_step":
        return {"op": op, "n": _log_int(rng, 1, 16384), "h": rng.randint(1, 12), "d": rng.choice([16, 32, 64, 128]),
                "dtype": dtype, "p_reset": rng.choice([0.0, 0.01, 0.2])}
    if op in ("attend_forward", "attend_backward"):
        return {"op": op, "t": _log_int(rng, 1, 16384), "n": _log_int(rng, 1, 4096), "h": rng.randint(1, 12),
                "d": rng.choice([16, 32, 64, 128]), "dtype": dtype, "p_reset": rng.choice([0.0, 0.002, 0.05, 0.3]),
                "carry": rng.random() < 0.5}
    if op in ("ffn_forward", "ffn_backward"):
        return {"op": op, "m": _log_int(rng, 1, 32768), "k": _log_int(rng, 16, 2048), "f": _log_int(rng, 32, 8192),
                "dtype": dtype, "act": rng.choice(["silu", "gelu"])}
    total, copies = _log_int(rng, 1000, 60_000_000), rng.random() < 0.5
    return {"op": op, "tensors": rng.randint(1, 30 if copies else 60), "total": total, "bits": rng.choice([8, 32]),
            "dtype": dtype, "copies": copies, "step": _log_int(rng, 1, 100_000)}


def draw(rng):
    """A case of the listed ones' ranges that costs no more than the largest of its operator's."""
    family = {"attend_step": ("attend_step",), "attend_forward": ("attend_forward", "attend_backward"),
              "attend_backward": ("attend_forward", "attend_backward"), "ffn_forward": ("ffn_forward", "ffn_backward"),
              "ffn_backward": ("ffn_forward", "ffn_backward"), "adamw": ("adamw",)}
    while True:
        case = _draw_once(rng)
        most = [work(c) for c in listed() if c["op"] in family[case["op"]]]
        w = work(case)
        if w["bytes"] <= max(m["bytes"] for m in most) and w["flops"] <= max(m["flops"] for m in most):
            return case


def work(case):
    """Bytes that a pass has to read and write once, and its operations (a multiply-add is two)."""
    c, op = case, case["op"]
    if op == "attend_step":
        rows = c["n"] * c["h"]
        return {"bytes": rows * (8.0 * c["d"] ** 2 + 4 * c["d"] * _SIZE[c["dtype"]]), "flops": rows * 5.0 * c["d"] ** 2}
    if op in ("attend_forward", "attend_backward"):
        rows, tokens = c["n"] * c["h"], c["t"] * c["n"] * c["h"]
        back = op == "attend_backward"
        tensors, scans = (7, 3) if back else (4, 1)  # q k v do dq dk dv; q k v o
        # the recurrence itself: the state's update and the read-out, 2 D^2 multiply-adds a token and scan
        states = (1 if c["carry"] else 0) + 1 + (1 if back else 0)
        return {"bytes": tokens * c["d"] * float(_SIZE[c["dtype"]]) * tensors + rows * 4.0 * c["d"] ** 2 * states
                + c["t"] * c["n"], "flops": tokens * scans * 4.0 * c["d"] ** 2}
    if op == "ffn_forward":
        return {"bytes": float(_SIZE[c["dtype"]]) * (c["m"] * c["k"] + 2 * c["k"] * c["f"] + c["m"] * c["f"]),
                "flops": 4.0 * c["m"] * c["k"] * c["f"]}
    if op == "ffn_backward":  # both products again, then dx and both weights' gradients
        return {"bytes": float(_SIZE[c["dtype"]]) * (2 * c["m"] * c["k"] + 4 * c["k"] * c["f"] + c["m"] * c["f"]),
                "flops": 12.0 * c["m"] * c["k"] * c["f"]}
    # parameter read and written, gradient read, both moments read and written, and the moments' values
    # given out where they are held in 8 bits
    per = 8.0 + _SIZE[c["dtype"]] + (4 + 8 if c["bits"] == 8 else 16) + (2 if c["copies"] else 0)
    return {"bytes": c["total"] * per, "flops": c["total"] * 16.0}


# ---- inputs ------------------------------------------------------------------------------------

def _tensor_sizes(case):
    """Sizes of a model's tensors: matrices and vectors of very unequal sizes, summing to `total`."""
    n, total = case["tensors"], case["total"]
    weights = [((i * 7919) % 97 + 1) ** 2 for i in range(n)]
    sizes = [max(1, total * w // sum(weights)) for w in weights]
    sizes[-1] = max(1, sizes[-1] + total - sum(sizes))
    return sizes


def _offsets(sizes):
    """Where each tensor's state starts in the flat state (a block's boundary), and the flat length."""
    starts, at = [], 0
    for s in sizes:
        starts.append(at)
        at += -(-s // _BLOCK) * _BLOCK
    return starts, at


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    op = case["op"]

    def normal(*shape, scale=1.0, dtype=None):
        return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype or _TYPES[case["dtype"]])

    s = {"case": dict(case)}
    if op.startswith("attend"):
        n, h, d = case["n"], case["h"], case["d"]
        lead = (n, h) if op == "attend_step" else (case["t"], n, h)
        s.update(q=normal(*lead, d), k=normal(*lead, d, scale=d ** -0.5), v=normal(*lead, d))
        # memories from a few steps to thousands, one per head
        s["decay"] = 1.0 - 2.0 ** (-2.0 - torch.arange(h, device="cuda", dtype=torch.float32) % 9)
        s["resets"] = torch.rand(lead[:-1], generator=g, device="cuda") < case["p_reset"] if case["p_reset"] else None
        s["state"] = normal(n, h, d, d, dtype=torch.float32) if case.get("carry", True) else None
        if op == "attend_backward":
            s["grad"] = normal(*lead, d)
            s["grad_state"] = normal(n, h, d, d, dtype=torch.float32) if case["carry"] else None
    elif op.startswith("ffn"):
        m, k, f = case["m"], case["k"], case["f"]
        s.update(x=normal(m, k), w_gate=normal(k, f, scale=k ** -0.5), w_up=normal(k, f, scale=k ** -0.5))
        if op == "ffn_backward":
            s["grad"] = normal(m, f)
    else:
        sizes = _tensor_sizes(case)
        starts, total = _offsets(sizes)
        s.update(sizes=sizes, starts=starts, step=case["step"], total=total, seed=int(seed))
        s["params"] = [normal(n, scale=0.05, dtype=torch.float32) for n in sizes]
        s["grads"] = [normal(n, scale=1e-3 * (1 + i % 5)) for i, n in enumerate(sizes)]
        s["copies"] = [p.to(torch.bfloat16) for p in s["params"]] if case["copies"] else None
        m = torch.zeros(total, device="cuda")
        v = torch.zeros(total, device="cuda")
        for at, n in zip(starts, sizes):  # moments as some steps in: zero where no element stands
            m[at:at + n] = normal(n, scale=3e-4, dtype=torch.float32)
            v[at:at + n] = normal(n, scale=1e-3, dtype=torch.float32).square()
        if case["bits"] == 8:
            rand = torch.randint(0, 1 << 32, (total,), generator=g, device="cuda")
            s["m"], s["m_exp"] = _encode(m, rand & 0xFFFF, 4)
            s["v"], s["v_exp"] = _encode(v, rand >> 16, 5)
        else:
            s["m"], s["v"] = m, v
    return s


# ---- the plain forms ---------------------------------------------------------------------------

def _plain_scan(x, a, b, decay, carry, resets, reverse):
    """out_i = sum_{j <= i} w_ij (x_i . a_j) b_j + w_i x_i carry over (T, N, H, D) tensors, by chunks:
    products inside a chunk, and a decayed sum over the earlier chunks' states. `reverse` runs from the
    last token to the first, the decay applied after a token instead of before it. Returns out and the
    carry at the other end, in 32 bits."""
    t, n, h, d = x.shape
    if reverse:
        x, a, b = x.flip(0), a.flip(0), b.flip(0)
        resets = None if resets is None else resets.flip(0)
    f = 0 if reverse else 1
    chunks, dev = -(-t // _CHUNK), x.device

    def split(y):  # (T, N, H, D) -> (N, H, chunks, CHUNK, D), zeros past T
        y = torch.nn.functional.pad(y.float(), (0, 0, 0, 0, 0, 0, 0, chunks * _CHUNK - t))
        return y.reshape(chunks, _CHUNK, n, h, d).permute(2, 3, 0, 1, 4)

    x, a, b = split(x), split(a), split(b)
    r = torch.zeros((t, n), device=dev) if resets is None else resets.float()
    r = torch.nn.functional.pad(r, (0, 0, 0, chunks * _CHUNK - t))
    seen = r.cumsum(0)                                        # resets up to and with each token
    count = (seen - r if reverse else seen).t().reshape(n, 1, chunks, _CHUNK)
    ends = seen.reshape(chunks, _CHUNK, n)[:, -1].t()         # (N, chunks): resets before a chunk's end
    ends0 = torch.cat([torch.zeros((n, 1), device=dev), ends], 1)  # at 0, 1, ..: before a chunk's start
    i = torch.arange(_CHUNK, device=dev)
    g = decay.float().reshape(h, 1, 1, 1)

    apart = i[:, None] - i[None, :]
    w = torch.pow(g, apart.clamp(min=0)) * (apart >= 0) * (count[..., :, None] == count[..., None, :])
    out = ((x @ a.transpose(-1, -2)) * w) @ b

    start = torch.arange(chunks + 1, device=dev) * _CHUNK
    start[-1] = t
    end = start[1:]
    left = (end[:, None] - start[:-1, None] - i - f)          # decays from a token to its chunk's end
    wj = torch.pow(g.reshape(h, 1, 1), left.clamp(min=0)) * (left >= 0) * (count == ends[:, None, :, None])
    local = (a * wj[..., None]).transpose(-1, -2) @ b         # (N, H, chunks, D, D)
    gap = start[:, None] - end[None, :]
    wc = torch.pow(g.reshape(h, 1, 1), gap.clamp(min=0)) * (gap >= 0) * (ends0[:, None, :, None] == ends[:, None, None, :])
    state = (wc @ local.reshape(n, h, chunks, d * d)).reshape(n, h, chunks + 1, d, d)
    if carry is not None:
        w0 = torch.pow(g.reshape(h, 1), start) * (ends0[:, None, :] == 0)
        state = state + w0[..., None, None] * carry[:, :, None]
    wi = torch.pow(g.reshape(h, 1, 1), i + f) * (count == ends0[:, None, :-1, None])
    out = out + wi[..., None] * (x @ state[:, :, :-1])
    out = out.permute(2, 3, 0, 1, 4).reshape(chunks * _CHUNK, n, h, d)[:t]
    return (out.flip(0) if reverse else out), state[:, :, -1]


def _plain_attend_forward(s):
    q, scale = s["q"], s["q"].shape[-1] ** -0.5
    out, state = _plain_scan(q, s["k"], s["v"], s["decay"], s["state"], s["resets"], False)
    return {"out": (out * scale).to(q.dtype), "state": state}


def _plain_attend_backward(s):
    """With the state S_t and its adjoint R_t: dq_t = S_t do_t, dk_t = R_t v_t, dv_t = R_t' k_t, each a
    scan of the same kind over the other three tensors."""
    q, k, v, do, r = s["q"], s["k"], s["v"], s["grad"], s["resets"]
    scale = q.shape[-1] ** -0.5
    turned = None if s["state"] is None else s["state"].transpose(-1, -2)
    gs = None if s["grad_state"] is None else s["grad_state"] / scale
    dq, _ = _plain_scan(do, v, k, s["decay"], turned, r, False)
    dv, carry = _plain_scan(k, q, do, s["decay"], gs, r, True)
    dk, _ = _plain_scan(v, do, q, s["decay"], None if gs is None else gs.transpose(-1, -2), r, True)
    return {"dq": (dq * scale).to(q.dtype), "dk": (dk * scale).to(q.dtype), "dv": (dv * scale).to(q.dtype),
            "dstate": carry * scale}


def _plain_attend_step(s):
    q, k, v = s["q"].float(), s["k"].float(), s["v"].float()
    old = s["state"] if s["resets"] is None else torch.where(s["resets"][:, None, None, None], 0.0, s["state"])
    s["state"] = s["decay"][:, None, None] * old + k[..., :, None] * v[..., None, :]
    out = (q[..., None, :] @ s["state"])[..., 0, :] * q.shape[-1] ** -0.5
    return {"out": out.to(s["q"].dtype), "state": s["state"]}


def _activation(g, act):
    """act(g) and its derivative."""
    if act == "silu":
        sig = 1.0 / (1.0 + torch.exp(-g))
        return g * sig, sig * (1.0 + g * (1.0 - sig))
    cdf = 0.5 * (1.0 + torch.erf(g * math.sqrt(0.5)))
    return g * cdf, cdf + g * torch.exp(-0.5 * g * g) * (1.0 / math.sqrt(2.0 * math.pi))


def _plain_ffn_forward(s):
    x = s["x"].float()
    y, _ = _activation(x @ s["w_gate"].float(), s["case"]["act"])
    return (y * (x @ s["w_up"].float())).to(s["x"].dtype)


def _plain_ffn_backward(s):
    x, wg, wu, dy = s["x"].float(), s["w_gate"].float(), s["w_up"].float(), s["grad"].float()
    y, slope = _activation(x @ wg, s["case"]["act"])
    dg, du = dy * (x @ wu) * slope, dy * y
    t = s["x"].dtype
    return {"dx": (dg @ wg.t() + du @ wu.t()).to(t), "dw_gate": (x.t() @ dg).to(t), "dw_up": (x.t() @ du).to(t)}


# The 8-bit state. A block of 256 elements shares an exponent e; an element is held as a sign (first
# moment only), `ebits` bits of exponent below e and three bits of mantissa: the code c > 0 stands for the
# float whose bits are (c + 8 (e - 2^ebits + 1)) << 20, and 0 for zero. Rounding is stochastic: 16 random
# bits, a hash of (seed, step, place), are added below the last kept bit. The second moment never rounds
# to zero. The largest code is kept for NaN.

def _encode(x, rand, ebits):
    bits = x.abs().view(torch.int32).to(torch.int64)
    top = (1 << (ebits + 3)) - 1
    finite = torch.where(bits < 0x7F800000, bits, 0).reshape(-1, _BLOCK)
    e = ((finite.amax(1) + 0x1FFFFF) >> 23).clamp(min=32)
    c = ((bits + (rand << 4)) >> 20).reshape(-1, _BLOCK) - (e - ((1 << ebits) - 1))[:, None] * 8
    c = c.clamp(min=0).reshape(-1)
    if ebits == 5:
        c = torch.where((bits > 0) & (c < 1), 1, c)
    c = torch.where(bits < 0x7F800000, c, top)
    if ebits == 4:
        c = torch.where(x.view(torch.int32) < 0, c + 128, c)
    return c.to(torch.uint8), e.to(torch.uint8)


def _decode(codes, e, ebits):
    c = codes.to(torch.int64)
    top = (1 << (ebits + 3)) - 1
    mag = c & 127 if ebits == 4 else c
    bits = (mag.reshape(-1, _BLOCK) + (e.to(torch.int64) - ((1 << ebits) - 1))[:, None] * 8).reshape(-1) << 20
    x = torch.where(mag == 0, 0, bits).to(torch.int32).view(torch.float32)
    x = torch.where(mag == top, float("nan"), x)
    return torch.where(c > 127, -x, x) if ebits == 4 else x


def _pcg(v):
    """The PCG hash that seeds the environments' resets, of 32-bit words held in 64."""
    a = (v * 747796405 + 2891336453) & 0xFFFFFFFF
    w = (((a >> ((a >> 28) + 4)) ^ a) * 277803737) & 0xFFFFFFFF
    return (w >> 22) ^ w


def _rounding_bits(total, seed, step):
    key = _pcg(torch.tensor([(seed ^ (step * 0x9E3779B9)) & 0xFFFFFFFF], device="cuda"))
    return _pcg((torch.arange(total, device="cuda") ^ key) & 0xFFFFFFFF)


_LR, _BETAS, _EPS, _DECAY = 1e-3, (0.9, 0.999), 1e-8, 0.01


def _flat(tensors, sizes):
    return torch.cat([torch.nn.functional.pad(x.reshape(-1).float(), (0, -n % _BLOCK)) for x, n in zip(tensors, sizes)])


def _pieces(flat, s):
    return [flat[at:at + n] for at, n in zip(s["starts"], s["sizes"])]


def _plain_adamw(s):
    s["step"] += 1
    t, (b1, b2) = s["step"], _BETAS
    eight = s["case"]["bits"] == 8
    g = _flat(s["grads"], s["sizes"])
    m = _decode(s["m"], s["m_exp"], 4) if eight else s["m"]
    v = _decode(s["v"], s["v_exp"], 5) if eight else s["v"]
    m = m * b1 + g * (1.0 - b1)
    v = v * b2 + (g * g) * (1.0 - b2)
    denom = torch.sqrt(v) * (1.0 / math.sqrt(1.0 - b2 ** t)) + _EPS
    update = (m * (_LR / (1.0 - b1 ** t))) / denom
    torch._foreach_mul_(s["params"], 1.0 - _LR * _DECAY)
    torch._foreach_sub_(s["params"], _pieces(update, s))
    if s["copies"] is not None:
        torch._foreach_copy_(s["copies"], s["params"])
    if eight:
        rand = _rounding_bits(s["total"], s["seed"], t)
        s["m"], s["m_exp"] = _encode(m, rand & 0xFFFF, 4)
        s["v"], s["v_exp"] = _encode(v, rand >> 16, 5)
        m, v = _decode(s["m"], s["m_exp"], 4), _decode(s["v"], s["v_exp"], 5)
    else:
        s["m"], s["v"] = m, v
    return {"params": s["params"], "m": m, "v": v, "copies": s["copies"]}


_PLAIN = {"attend_step": _plain_attend_step, "attend_forward": _plain_attend_forward,
          "attend_backward": _plain_attend_backward, "ffn_forward": _plain_ffn_forward,
          "ffn_backward": _plain_ffn_backward, "adamw": _plain_adamw}


# ---- the framework's calls -----------------------------------------------------------------------

def _own_run(s):
    attention, ffn, adamw = _framework()
    op = s["case"]["op"]
    if op == "attend_step":
        out = attention.step(s["q"], s["k"], s["v"], s["decay"], s["state"], resets=s["resets"])
        return {"out": out, "state": s["state"]}
    if op == "attend_forward":
        out, state = attention.forward(s["q"], s["k"], s["v"], s["decay"], state=s["state"], resets=s["resets"])
        return {"out": out, "state": state}
    if op == "attend_backward":
        dq, dk, dv, dstate = attention.backward(s["grad"], s["q"], s["k"], s["v"], s["decay"], state=s["state"],
                                                resets=s["resets"], grad_state=s["grad_state"])
        return {"dq": dq, "dk": dk, "dv": dv, "dstate": dstate}
    if op == "ffn_forward":
        return ffn.forward(s["x"], s["w_gate"], s["w_up"], activation=s["case"]["act"])
    if op == "ffn_backward":
        dx, dwg, dwu = ffn.backward(s["grad"], s["x"], s["w_gate"], s["w_up"], activation=s["case"]["act"])
        return {"dx": dx, "dw_gate": dwg, "dw_up": dwu}
    if "moments" not in s:  # the user's optimizer state, made once of the tensors in hand
        s["moments"] = adamw.State(bits=s["case"]["bits"], sizes=tuple(s["sizes"]), m=s["m"], v=s["v"],
                                   m_exp=s.get("m_exp"), v_exp=s.get("v_exp"), step=s["step"], seed=s["seed"])
    state = s["moments"]
    adamw.step(s["params"], s["grads"], state, lr=_LR, betas=_BETAS, eps=_EPS, weight_decay=_DECAY, copies=s["copies"])
    m, v = adamw.moments(state)
    return {"params": s["params"], "m": m, "v": v, "copies": s["copies"]}


def run(state):
    return _own_run(state) if own else _PLAIN[state["case"]["op"]](state)


# ---- the definitions in 64 bits --------------------------------------------------------------------

def _exact_scan(x, a, b, decay, carry, resets, reverse):
    """The recurrence token by token."""
    t, n, h, d = x.shape
    g = decay.double()[:, None, None]
    state = torch.zeros((n, h, d, d), dtype=torch.float64, device=x.device) if carry is None else carry.double()
    out = torch.empty((t, n, h, d), dtype=torch.float64, device=x.device)
    keep = None if resets is None else (~resets).double()[:, :, None, None, None]
    for i in (range(t - 1, -1, -1) if reverse else range(t)):
        if not reverse:
            state = state * g if keep is None else state * g * keep[i]
        state = state + a[i].double()[..., :, None] * b[i].double()[..., None, :]
        out[i] = torch.einsum("nhd,nhde->nhe", x[i].double(), state)
        if reverse:
            state = state * g if keep is None else state * g * keep[i]
    return out, state


def _exact_adamw(s):
    (b1, b2), t = _BETAS, s["step"] + 1
    eight = s["case"]["bits"] == 8
    g = _flat(s["grads"], s["sizes"]).double()
    p = _flat(s["params"], s["sizes"]).double()
    m = (_decode(s["m"], s["m_exp"], 4) if eight else s["m"]).double()
    v = (_decode(s["v"], s["v_exp"], 5) if eight else s["v"]).double()
    m, v = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
    step = _LR * (m / (1 - b1 ** t)) / ((v / (1 - b2 ** t)).sqrt() + _EPS)
    p = p - _LR * _DECAY * p - step
    if eight:
        rand = _rounding_bits(s["total"], s["seed"], t)
        m, v = _exact_round(m, rand & 0xFFFF, 4), _exact_round(v, rand >> 16, 5)
    pieces = [x.clone() for x in _pieces(p, s)]
    return {"params": pieces, "m": m, "v": v, "copies": pieces if s["copies"] else None}


def _exact_round(x, rand, ebits):
    """The values that the 8-bit codes of x stand for, by arithmetic: an eighth of an octave is split at
    the random place rand / 65536."""
    mag = x.abs().reshape(-1, _BLOCK)
    mant, ex = torch.frexp(mag.amax(1))                 # mag = mant 2^ex, mant in [1/2, 1)
    e = ex - 1 + (mant * 2 > 1.75).to(ex.dtype)         # the block's octave, one up where seven eighths are passed
    e = torch.where(mag.amax(1) > 0, e, torch.full_like(e, -95)).clamp(min=-95)
    mant, ex = torch.frexp(mag)
    eighths = (mant * 2 - 1) * 8
    low = torch.floor(eighths)
    up = (eighths - low) + rand.reshape(-1, _BLOCK).double() / 65536.0 >= 1.0
    place = ((ex - 1 - e[:, None]).double() + (1 << ebits) - 1) * 8 + low + up.double()
    place = torch.where(mag > 0, place.clamp(min=1.0 if ebits == 5 else 0.0), torch.zeros_like(place))
    octave = torch.floor(place / 8)
    value = (1 + (place - 8 * octave) / 8) * torch.exp2(octave - ((1 << ebits) - 1) + e[:, None].double())
    value = torch.where(place >= 1, value, torch.zeros_like(value)).reshape(-1)
    return torch.where(x < 0, -value, value)


def exact(case, seed):
    s, op = prepare(case, seed), case["op"]
    if op == "attend_step":
        lift = {k: s[k][None] for k in ("q", "k", "v")}
        out, state = _exact_scan(lift["q"], lift["k"], lift["v"], s["decay"], s["state"],
                                 None if s["resets"] is None else s["resets"][None], False)
        return {"out": out[0] * case["d"] ** -0.5, "state": state}
    if op in ("attend_forward", "attend_backward"):
        if case["t"] * case["n"] * case["h"] * case["d"] ** 2 > 6e10 or case["t"] > 40000:
            return None
        scale = case["d"] ** -0.5
        q, k, v, r, g = s["q"], s["k"], s["v"], s["resets"], s["decay"]
        if op == "attend_forward":
            out, state = _exact_scan(q, k, v, g, s["state"], r, False)
            return {"out": out * scale, "state": state}
        gs = None if s["grad_state"] is None else s["grad_state"].double() / scale
        dq, _ = _exact_scan(s["grad"], v, k, g, None if s["state"] is None else s["state"].transpose(-1, -2), r, False)
        dv, carry = _exact_scan(k, q, s["grad"], g, gs, r, True)
        dk, _ = _exact_scan(v, s["grad"], q, g, None if gs is None else gs.transpose(-1, -2), r, True)
        return {"dq": dq * scale, "dk": dk * scale, "dv": dv * scale, "dstate": carry * scale}
    if op.startswith("ffn"):
        x, wg, wu = s["x"].double(), s["w_gate"].double(), s["w_up"].double()
        g, u = x @ wg, x @ wu
        if case["act"] == "silu":
            y, slope = g * torch.sigmoid(g), torch.sigmoid(g) + g * torch.sigmoid(g) * torch.sigmoid(-g)
        else:
            cdf = torch.special.ndtr(g)
            y, slope = g * cdf, cdf + g * torch.exp(-g * g / 2) / math.sqrt(2 * math.pi)
        if op == "ffn_forward":
            return y * u
        dy = s["grad"].double()
        dg, du = dy * u * slope, dy * y
        return {"dx": dg @ wg.t() + du @ wu.t(), "dw_gate": x.t() @ dg, "dw_up": x.t() @ du}
    return _exact_adamw(s)
