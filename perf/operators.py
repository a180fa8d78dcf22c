"""Cases of the sequence-layer operators: the short causal convolution and the selective scan, for
prompts and for single tokens, and the 8-bit matrix product with its quantiser.

``run`` computes a case in elementary torch operations (``own`` false) or through libcwg (``own``
true); ``exact`` computes it from the definition in 64 bits.
"""
from __future__ import annotations

import math
import os
import sys

import torch

own = False

FP8 = torch.float8_e4m3fn
FP8_MAX = 448.0
SCALE_MIN = 2.0 ** -126
GROUP = 128  # columns (and, for weights, rows) that share a scale


def _cwg():
    if "cwg" not in sys.modules:  # as any program, once
        sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(
            os.path.abspath(__file__))), "cache-aware-wino-implementation_b200"))
        import cwg  # noqa: F401
    return sys.modules["cwg"]


# ---- cases ------------------------------------------------------------------------
def listed():
    return [
        # a batch of prompts of mixed lengths through a wide layer's convolution
        dict(name="conv prompts bf16", op="conv", dtype="bf16", tokens=16384, seqs=12,
             channels=4096, width=4),
        # odd channel count and width: rows that are not 16-byte aligned
        dict(name="conv prompts fp32 odd", op="conv", dtype="fp32", tokens=1237, seqs=7,
             channels=1001, width=3),
        # one decoding step of a full serving batch
        dict(name="conv step bf16 x256", op="conv_step", dtype="bf16", seqs=256, channels=4096,
             width=4),
        # one decoding step of one sequence
        dict(name="conv step fp32 x1", op="conv_step", dtype="fp32", seqs=1, channels=2048,
             width=4),
        # one long prompt: all parallelism comes from channels, states and time
        dict(name="scan one long prompt bf16", op="scan", dtype="bf16", tokens=8192, seqs=1,
             channels=4096, groups=1, states=16, gate=True),
        # ragged prompts, several B/C groups, odd channel and state counts
        dict(name="scan prompts fp32 odd", op="scan", dtype="fp32", tokens=1531, seqs=9,
             channels=1002, groups=2, states=12, gate=False),
        # one decoding step of a full serving batch: the states are read and written
        dict(name="scan step bf16 x256", op="scan_step", dtype="bf16", seqs=256, channels=4096,
             groups=1, states=16, gate=True),
        # one decoding step of one sequence
        dict(name="scan step bf16 x1", op="scan_step", dtype="bf16", seqs=1, channels=2048,
             groups=1, states=16, gate=True),
        # a prompt's activations before a projection
        dict(name="quantize rows bf16", op="quantize", dtype="bf16", rows=8192, cols=4096,
             block_rows=1),
        # a weight matrix of odd size, blocks cut at both edges
        dict(name="quantize blocks fp32 odd", op="quantize", dtype="fp32", rows=1000, cols=1543,
             block_rows=128),
        # a decoding step's projection: few rows, the weights are streamed
        dict(name="matmul few rows", op="matmul", dtype="bf16", m=4, n=8192, k=4096, bias=False,
             relu=False),
        # a prompt's projection
        dict(name="matmul prompt", op="matmul", dtype="bf16", m=8192, n=8192, k=4096, bias=True,
             relu=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("conv", "conv_step", "scan", "scan_step", "quantize", "matmul"))
    dtype = rng.choice(("bf16", "fp32"))
    if op in ("conv", "conv_step"):
        channels = _log(rng, 64, 4096)
        if rng.random() < 0.6:  # most layers' channel counts are round
            channels = max(64, channels // 64 * 64)
        width = rng.choice((2, 3, 4))
        if op == "conv_step":
            return dict(op=op, dtype=dtype, seqs=_log(rng, 1, 512 if dtype == "bf16" else 256),
                        channels=channels, width=width)
        tokens = _log(rng, 1, 16384 if dtype == "bf16" else 8192)
        return dict(op=op, dtype=dtype, tokens=tokens, seqs=_log(rng, 1, 32), channels=channels,
                    width=width)
    if op in ("scan", "scan_step"):
        states = rng.choice((4, 8, 12, 16, 16, 16, 23, 32, 64))
        groups = rng.choice((1, 1, 2, 4))
        channels = groups * _log(rng, 16, 4096 // groups)
        if rng.random() < 0.6:
            channels = max(64 * groups, channels // (64 * groups) * 64 * groups)
        gate = rng.random() < 0.5
        if op == "scan_step":
            most = 256 * 4096 * 16 // (channels * states)
            return dict(op=op, dtype=dtype, seqs=_log(rng, 1, min(512, most)), channels=channels,
                        groups=groups, states=states, gate=gate)
        most = 8192 * 4096 * 16 // (channels * states)
        tokens = _log(rng, 1, min(8192 if dtype == "bf16" else 4096, most))
        return dict(op=op, dtype=dtype, tokens=tokens, seqs=_log(rng, 1, 24), channels=channels,
                    groups=groups, states=states, gate=gate)
    if op == "quantize":
        cols = _log(rng, 16, 8192)
        return dict(op=op, dtype=dtype, rows=_log(rng, 1, min(16384, 2 ** 24 // cols)), cols=cols,
                    block_rows=rng.choice((1, 128)))
    n, k = _log(rng, 32, 8192), _log(rng, 32, 8192)
    return dict(op=op, dtype=dtype, m=_log(rng, 1, min(8192, 2 ** 38 // (n * k))), n=n, k=k,
                bias=rng.random() < 0.5, relu=rng.random() < 0.5)


def work(case):
    c, es = case, 2 if case["dtype"] == "bf16" else 4
    op = c["op"]
    if op == "conv":
        elems = c["tokens"] * c["channels"]
        line = c["seqs"] * (c["width"] - 1) * c["channels"] * es
        return {"bytes": 2 * elems * es + 2 * line + 4 * c["channels"] * (c["width"] + 1),
                "flops": (2 * c["width"] + 5) * elems}
    if op == "conv_step":
        elems = c["seqs"] * c["channels"]
        return {"bytes": 2 * elems * es * c["width"] + 4 * c["channels"] * (c["width"] + 1),
                "flops": (2 * c["width"] + 5) * elems}
    if op in ("scan", "scan_step"):
        rows = c["tokens"] if op == "scan" else c["seqs"]
        elems = rows * c["channels"]
        bc = 2 * rows * c["groups"] * c["states"] * es
        states = 2 * 4 * c["seqs"] * c["channels"] * c["states"]
        weights = 4 * c["channels"] * (c["states"] + 2)
        return {"bytes": (3 + c["gate"]) * elems * es + bc + states + weights,
                "flops": elems * (7 * c["states"] + 12)}
    if op == "quantize":
        elems = c["rows"] * c["cols"]
        scales = -(-c["rows"] // c["block_rows"]) * -(-c["cols"] // GROUP)
        return {"bytes": elems * (es + 1) + 4 * scales, "flops": 3 * elems}
    m, n, k = c["m"], c["n"], c["k"]
    kb = -(-k // GROUP)
    return {"bytes": m * k + n * k + m * n * es + 4 * kb * (m + -(-n // GROUP)) +
            4 * n * c["bias"], "flops": 2 * m * n * k}


# ---- inputs -----------------------------------------------------------------------
def _lengths(total, seqs, gen):
    """`seqs` lengths that sum to `total`: ragged, some of them zero or one."""
    if seqs == 1:
        return [total]
    cuts = torch.randint(0, total + 1, (seqs - 1,), generator=gen).tolist()
    cuts = sorted(cuts)
    if seqs > 3:
        cuts[1] = cuts[0]                      # an empty sequence
        cuts[2] = min(total, cuts[1] + 1)      # and one of a single token
        cuts = sorted(cuts)
    return [b - a for a, b in zip([0] + cuts, cuts + [total])]


def _quantize(x, block_rows):
    """e4m3 values and scales of a matrix, as the framework's quantiser defines them."""
    rows, cols = x.shape
    kb, rb = -(-cols // GROUP), -(-rows // block_rows)
    x = torch.nn.functional.pad(x.float(), (0, kb * GROUP - cols, 0, rb * block_rows - rows))
    g = x.view(rb, block_rows, kb, GROUP)
    scale = (g.abs().amax(dim=(1, 3)) / FP8_MAX).clamp_min(SCALE_MIN)
    q = (g / scale[:, None, :, None]).to(FP8)
    return q.view(rb * block_rows, kb * GROUP)[:rows, :cols], scale


def prepare(case, seed):
    c = case
    host = torch.Generator().manual_seed(seed)
    gen = torch.Generator("cuda").manual_seed(seed)
    dt = torch.bfloat16 if c["dtype"] == "bf16" else torch.float32

    def normal(*shape, std=1.0, dtype=dt):
        return (torch.randn(*shape, generator=gen, device="cuda") * std).to(dtype)

    def uniform(*shape, lo, hi):
        return torch.rand(*shape, generator=gen, device="cuda") * (hi - lo) + lo

    s = dict(case=c)
    op = c["op"]
    if op in ("conv", "scan"):
        lens = _lengths(c["tokens"], c["seqs"], host)
        starts = torch.tensor([0] + lens).cumsum(0)
        s["starts"] = starts.to(torch.int32).cuda()
        s["resume"] = torch.randint(0, 2, (c["seqs"],), generator=host).to(torch.uint8).cuda()
    if op in ("conv", "conv_step", "scan", "scan_step"):
        lines = c["seqs"] + 3  # cache lines; the sequences hold some of them, in any order
        s["slots"] = torch.randperm(lines, generator=host)[:c["seqs"]].to(torch.int32).cuda()
        rows = c["tokens"] if op in ("conv", "scan") else c["seqs"]
        ch = c["channels"]
    if op in ("conv", "conv_step"):
        # x is the first half of a projection's rows, as the block's input projection writes it
        s["x"] = normal(rows, 2 * ch)[:, :ch]
        bound = 1 / math.sqrt(c["width"])
        s["w"] = uniform(ch, c["width"], lo=-bound, hi=bound)
        s["bias"] = uniform(ch, lo=-bound, hi=bound)
        s["state"] = normal(lines, c["width"] - 1, ch)
        s["y"] = torch.zeros(rows, ch, device="cuda", dtype=dt)
    elif op in ("scan", "scan_step"):
        g, n = c["groups"], c["states"]
        s["u"] = torch.nn.functional.silu(normal(rows, ch, dtype=torch.float32)).to(dt)
        s["dt"] = normal(rows, ch, std=0.5)
        proj = normal(rows, 2 * g * n)  # B and C as neighbouring columns of one projection
        s["B"], s["C"] = proj[:, :g * n], proj[:, g * n:]
        s["A"] = -torch.arange(1, n + 1, device="cuda").float().repeat(ch, 1)
        s["A"] *= uniform(ch, n, lo=0.8, hi=1.25)
        s["D"] = uniform(ch, lo=0.5, hi=1.5)
        step = torch.exp(uniform(ch, lo=math.log(1e-3), hi=math.log(1e-1)))
        s["dt_bias"] = step + torch.log(-torch.expm1(-step))  # softplus(dt_bias) = step
        s["z"] = normal(rows, 2 * ch)[:, ch:] if c["gate"] else None
        s["state"] = normal(lines, ch, n, std=0.1, dtype=torch.float32)
        s["y"] = torch.zeros(rows, ch, device="cuda", dtype=dt)
    elif op == "quantize":
        x = normal(c["rows"], c["cols"], dtype=torch.float32)
        x *= torch.exp(normal(c["rows"], 1, dtype=torch.float32))  # rows of unlike magnitude
        s["x"] = x.to(dt)
        ld = -(-c["cols"] // 16) * 16
        s["q"] = torch.zeros(c["rows"], ld, dtype=FP8, device="cuda")[:, :c["cols"]]
        s["scale"] = torch.zeros(-(-c["rows"] // c["block_rows"]), -(-c["cols"] // GROUP),
                                 device="cuda")
    else:
        m, n, k = c["m"], c["n"], c["k"]
        ld = -(-k // 16) * 16  # rows of a whole number of 16 bytes
        a, s["a_scale"] = _quantize(normal(m, k, dtype=torch.float32), 1)
        w, s["w_scale"] = _quantize(normal(n, k, std=1 / math.sqrt(k), dtype=torch.float32), 128)
        s["a"] = torch.zeros(m, ld, dtype=torch.uint8, device="cuda").view(FP8)[:, :k]
        s["w"] = torch.zeros(n, ld, dtype=torch.uint8, device="cuda").view(FP8)[:, :k]
        s["a"].copy_(a)
        s["w"].copy_(w)
        s["bias"] = uniform(n, lo=-0.1, hi=0.1) if c["bias"] else None
        s["y"] = torch.zeros(m, n, device="cuda", dtype=dt)
    return s


# ---- one pass ----------------------------------------------------------------------
def _own(s):
    cwg = _cwg()
    c = s["case"]
    op = c["op"]
    flags = cwg.BF16 if c["dtype"] == "bf16" else 0
    if op == "conv":
        cwg.conv1d_causal(s["x"], s["w"], s["bias"], s["y"], s["state"], s["starts"], s["slots"],
                          s["resume"], flags | cwg.SILU)
        return s["y"], s["state"]
    if op == "conv_step":
        cwg.conv1d_causal_step(s["x"], s["w"], s["bias"], s["y"], s["state"], s["slots"],
                               flags | cwg.SILU)
        return s["y"], s["state"]
    if op == "scan":
        need = cwg.ssm_workspace_bytes(c["tokens"], c["seqs"], c["channels"], c["states"])
        workspace = torch.empty(need, dtype=torch.uint8, device="cuda")
        cwg.ssm_scan(s["u"], s["dt"], s["A"], s["B"], s["C"], s["D"], s["dt_bias"], s["z"],
                     s["y"], s["state"], s["starts"], s["slots"], s["resume"], workspace,
                     flags | cwg.SOFTPLUS)
        return s["y"], s["state"]
    if op == "scan_step":
        cwg.ssm_step(s["u"], s["dt"], s["A"], s["B"], s["C"], s["D"], s["dt_bias"], s["z"],
                     s["y"], s["state"], s["slots"], flags | cwg.SOFTPLUS)
        return s["y"], s["state"]
    if op == "quantize":
        cwg.fp8_quantize(s["x"], s["q"], s["scale"], c["block_rows"], flags)
        return s["q"], s["scale"]
    if c["relu"]:
        flags |= cwg.RELU
    cwg.fp8_matmul(s["a"], s["a_scale"], s["w"], s["w_scale"], s["bias"], s["y"], flags)
    return s["y"]


def _silu(v):
    return v / (1 + torch.exp(-v))


def _softplus(v):
    return torch.where(v > 20, v, torch.log1p(torch.exp(v.clamp_max(20))))


def _sequence_of(s):
    """For every token: its sequence, and its place in it."""
    t = torch.arange(s["case"]["tokens"], device="cuda", dtype=torch.int32)
    seq = torch.searchsorted(s["starts"][1:], t, right=True)
    return seq, t - s["starts"][seq]


def _plain_conv(s):
    c = s["case"]
    k = c["width"]
    x, slots, state = s["x"].float(), s["slots"].long(), s["state"]
    seq, place = _sequence_of(s)
    line = state[slots].float() * s["resume"].float()[:, None, None]  # [seqs][k-1][channels]
    back = torch.arange(k, device="cuda") - (k - 1)                   # 0 is the token itself
    src = place[:, None] + back                                       # [tokens][k]
    t = torch.arange(c["tokens"], device="cuda")
    taps = torch.where((src >= 0)[:, :, None], x[(t[:, None] + back).clamp_min(0)],
                       line[seq[:, None], (src + k - 1).clamp(0, k - 2)])
    y = _silu((taps * s["w"].t()).sum(1) + s["bias"])
    lens = s["starts"][1:] - s["starts"][:-1]
    at = lens[:, None] + torch.arange(k - 1, device="cuda") - (k - 1)
    row = (s["starts"][1:, None] + torch.arange(k - 1, device="cuda") - (k - 1))
    state[slots] = torch.where((at >= 0)[:, :, None], x[row.clamp(0, c["tokens"] - 1).long()],
                               line.gather(1, (at + k - 1).clamp(0, k - 2).long()[:, :, None]
                                           .expand_as(line))).to(state.dtype)
    return y.to(s["y"].dtype), state


def _plain_conv_step(s):
    x, slots, state = s["x"].float(), s["slots"].long(), s["state"]
    taps = torch.cat((state[slots].float(), x[:, None]), 1)
    y = _silu((taps * s["w"].t()).sum(1) + s["bias"])
    state[slots] = taps[:, 1:].to(state.dtype)
    return y.to(s["y"].dtype), state


def _scan_inputs(s):
    """Decay and drive of every (row, channel, state), and C, D u and the gate's factor."""
    c = s["case"]
    per = c["channels"] // c["groups"]
    u = s["u"].float()
    step = _softplus(s["dt"].float() + s["dt_bias"])
    b, cc = (v.float().reshape(-1, c["groups"], 1, c["states"]) for v in (s["B"], s["C"]))
    decay = torch.exp(step[:, :, None] * s["A"])
    drive = ((step * u).view(-1, c["groups"], per, 1) * b).view_as(decay)
    return decay, drive, cc, u * s["D"]


def _scan_output(s, h, cc, skip):
    c = s["case"]
    y = (h.view(h.shape[0], c["groups"], -1, c["states"]) * cc).sum(-1).view_as(skip) + skip
    if s["z"] is not None:
        y = y * _silu(s["z"].float())
    return y.to(s["y"].dtype)


def _plain_scan(s):
    slots, state, starts = s["slots"].long(), s["state"], s["starts"].long()
    a, h, cc, skip = _scan_inputs(s)
    h0 = state[slots] * s["resume"].float()[:, None, None]
    some = starts[1:] > starts[:-1]
    first = starts[:-1][some]
    h[first] += a[first] * h0[some]
    a[first] = 0  # nothing crosses from one sequence into the next
    # h_t = a_t h_{t-1} + b_t by doubling: after the pass of distance d, row t holds the sum of
    # the last 2d rows' drives and the product of their decays
    d = 1
    while d < h.shape[0]:
        h = torch.cat((h[:d], h[d:] + a[d:] * h[:-d]))
        a = torch.cat((a[:d], a[d:] * a[:-d]))
        d *= 2
    state[slots] = torch.where(some[:, None, None], h[(starts[1:] - 1).clamp_min(0)], h0)
    return _scan_output(s, h, cc, skip), state


def _plain_scan_step(s):
    slots, state = s["slots"].long(), s["state"]
    a, b, cc, skip = _scan_inputs(s)
    h = a * state[slots] + b
    state[slots] = h
    return _scan_output(s, h, cc, skip), state


def _plain_matmul(s):
    def values(q, scale, block_rows):
        rows, cols = q.shape
        each = scale.repeat_interleave(block_rows, 0)[:rows].repeat_interleave(GROUP, 1)[:, :cols]
        return q.float() * each

    y = values(s["a"], s["a_scale"], 1) @ values(s["w"], s["w_scale"], 128).t()
    if s["bias"] is not None:
        y = y + s["bias"]
    if s["case"]["relu"]:
        y = y.clamp_min(0)
    return y.to(s["y"].dtype)


def run(state):
    if own:
        return _own(state)
    op = state["case"]["op"]
    if op == "conv":
        return _plain_conv(state)
    if op == "conv_step":
        return _plain_conv_step(state)
    if op == "scan":
        return _plain_scan(state)
    if op == "scan_step":
        return _plain_scan_step(state)
    if op == "quantize":
        return _quantize(state["x"], state["case"]["block_rows"])
    return _plain_matmul(state)


# ---- the definition in 64 bits -------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "quantize":
        return _exact_quantize(s)
    if op == "matmul":
        return _exact_matmul(s)
    steps = op.endswith("_step")
    starts = list(range(case["seqs"] + 1)) if steps else s["starts"].tolist()
    resume = [1] * case["seqs"] if steps else s["resume"].tolist()
    slots = s["slots"].tolist()
    one = _exact_conv if op.startswith("conv") else _exact_scan
    state = s["state"].double()
    y = torch.zeros(s["y"].shape, dtype=torch.float64, device="cuda")
    if steps:
        at = s["slots"].long()
        y, state[at] = one(s, state[at], slice(0, case["seqs"]), True)
        return y, state
    for i, slot in enumerate(slots):
        rows = slice(starts[i], starts[i + 1])
        before = state[slot] if resume[i] else torch.zeros_like(state[slot])
        y[rows], state[slot] = one(s, before, rows, False)
    return y, state


def _exact_conv(s, line, rows, steps):
    """One sequence's outputs and its new cache line; `steps`: one token of each of many."""
    x, w = s["x"][rows].double(), s["w"].double()
    k = w.shape[1]
    if steps:
        past = torch.cat((line, x[:, None]), 1)
        v = sum(past[:, j] * w[:, j] for j in range(k)) + s["bias"].double()
        return v * torch.sigmoid(v), past[:, 1:]
    past = torch.cat((line, x))
    v = sum(past[j:j + len(x)] * w[:, j] for j in range(k)) + s["bias"].double()
    return v * torch.sigmoid(v), past[len(x):]


def _exact_scan(s, h, rows, steps):
    u = s["u"][rows].double()
    delta = torch.nn.functional.softplus(s["dt"][rows].double() + s["dt_bias"].double(),
                                         threshold=60)
    case = s["case"]
    which = torch.arange(case["channels"], device="cuda") // (case["channels"] // case["groups"])
    b = s["B"][rows].double().unflatten(1, (case["groups"], case["states"]))
    c = s["C"][rows].double().unflatten(1, (case["groups"], case["states"]))
    a = s["A"].double()
    if steps:
        h = torch.exp(delta[:, :, None] * a) * h + (delta * u)[:, :, None] * b[:, which]
        y = torch.einsum("rcn,rcn->rc", h, c[:, which])
    else:
        y = torch.zeros_like(u)
        for t in range(len(u)):
            h = torch.exp(delta[t, :, None] * a) * h + (delta[t] * u[t])[:, None] * b[t, which]
            y[t] = (h * c[t, which]).sum(-1)
    y = y + u * s["D"].double()
    if s["z"] is not None:
        z = s["z"][rows].double()
        y = y * z * torch.sigmoid(z)
    return y, h


def _exact_quantize(s):
    """The scales in 64 bits; the 8-bit values have no value beyond their own rounding."""
    x, r = s["x"].double(), s["case"]["block_rows"]
    scale = torch.stack([torch.stack([g.abs().max() if r > 1 else g.abs().amax(1)
                                      for g in rows.split(GROUP, 1)], -1)
                         for rows in (x.split(r) if r > 1 else [x])])
    return None, (scale.reshape(s["scale"].shape) / FP8_MAX).clamp_min(SCALE_MIN)


def _exact_matmul(s):
    c = s["case"]
    a, w = s["a"].float().double(), s["w"].float().double()
    y = torch.zeros(c["m"], c["n"], dtype=torch.float64, device="cuda")
    for i, k in enumerate(range(0, c["k"], GROUP)):
        part = a[:, k:k + GROUP] @ w[:, k:k + GROUP].t()
        ws = s["w_scale"][:, i].double()[torch.arange(c["n"], device="cuda") // 128]
        y += part * s["a_scale"][:, i].double()[:, None] * ws
    if s["bias"] is not None:
        y += s["bias"].double()
    return torch.relu(y) if c["relu"] else y
