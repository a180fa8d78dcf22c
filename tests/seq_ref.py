"""The sequence layers and the 8-bit product in 64 bits, with bounds on what fp32 arithmetic
may add: plain loops over sequences and tokens, torch on the CPU.

u = 2^-24 is half a step of fp32.  expf, log1pf and ex2.approx are taken at 2 ulp (4 u) each,
every addition, product and division at u; an output rounded to bf16 adds 2^-8 of itself.
Each function returns (value, bound) pairs.
"""
import torch

U = 2.0 ** -24
F64 = torch.float64


def half_step(dtype):
    return 0.0 if dtype == torch.float32 else torch.finfo(dtype).eps / 2


def silu(v):
    return v * torch.sigmoid(v)


def silu_error(v, dtype):
    """Relative: exp (4 u), 1 + e (u), the division (u); for bf16 results the exponent's two
    roundings add 2 |v| u, and a reciprocal of 2 u with its product replaces the division."""
    return (8 + 2 * v.abs() if dtype == torch.bfloat16 else torch.full_like(v, 6)) * U


def act(v, err, kind, dtype):
    """An activation of values that carry an error, and its error: silu' stays below 1.1."""
    if kind == "silu":
        y = silu(v)
        return y, 1.1 * err + silu_error(v, dtype) * y.abs()
    if kind == "relu":
        return v.clamp_min(0), err
    return v, err


def rounded(y, err, dtype):
    """Plus the rounding to the output's type (of a value that may be `err` larger), and
    a little for results below the normal range."""
    return y, err + half_step(dtype) * (y.abs() + err) + 1e-37


def conv1d(x, w, bias, line, kind):
    """One sequence: x (T, C), line (K - 1, C) -> (y, bound), new line."""
    k = w.shape[1]
    past = torch.cat((line.to(F64), x.to(F64)))
    w, b = w.to(F64), torch.zeros(len(w), dtype=F64) if bias is None else bias.to(F64)
    v = b.expand(len(x), -1).clone()
    size = b.abs().expand(len(x), -1).clone()
    for j in range(k):
        v += past[j:j + len(x)] * w[:, j]
        size += (past[j:j + len(x)] * w[:, j]).abs()
    y, err = act(v, k * U * size, kind, x.dtype)
    return rounded(y, err, x.dtype), past[len(past) - (k - 1):]


def ssm(u, dt, A, B, C, D, dt_bias, z, h, softplus):
    """One sequence: u, dt, z (T, ch), B, C (T, groups, n), h (ch, n) -> (y, bound),
    (h, bound)."""
    dtype = u.dtype
    ch, n = A.shape
    of = torch.arange(ch) // (ch // B.shape[1])
    u, A, B, C = u.to(F64), A.to(F64), B.to(F64), C.to(F64)
    v = dt.to(F64) + (0 if dt_bias is None else dt_bias.to(F64))
    # dt + bias rounds once (log(1 + exp) is 1-Lipschitz); exp is off by (4 + 2 |v|) u of
    # itself, which moves log(1 + exp) by no more than that of itself (it is at least e / (1 +
    # e) times as large where e <= 1); reciprocal, series and sums add 8 u.  The larger of v
    # and 0 is exact: for v > 0 only log1p(e) <= 0.7 carries these
    if softplus:
        step = torch.nn.functional.softplus(v, threshold=60)
        small = torch.nn.functional.softplus(-v.abs(), threshold=60)
        dstep = U * v.abs() + (12 + 2 * v.abs()) * U * small + U * step
    else:
        step, dstep = v, U * v.abs()
    h = h.to(F64).clone()
    eh = torch.zeros_like(h)
    y, ey = torch.zeros_like(u), torch.zeros_like(u)
    for t in range(len(u)):
        d, dd = step[t, :, None], dstep[t, :, None]
        decay = torch.exp(d * A)
        # the exponent d A log2(e): A log2(e) and the product round (2 u of |d A|), d carries dd
        de = 4 * U + A.abs() * dd + 2 * U * (d * A).abs()
        drive = d * u[t, :, None] * B[t, of]
        ddrive = (dd * u[t, :, None] * B[t, of]).abs() + 2 * U * drive.abs()
        eh = decay * (eh + de * (h.abs() + eh)) + ddrive
        h = decay * h + drive
        eh = eh + U * (h.abs() + eh)
        y[t] = (h * C[t, of]).sum(-1)
        ey[t] = (eh * C[t, of].abs()).sum(-1) + (n + 3) * U * (h * C[t, of]).abs().sum(-1)
    if D is not None:
        y = y + D.to(F64) * u
        ey = ey + U * y.abs() + U * (D.to(F64) * u).abs()
    if z is not None:
        g = silu(z.to(F64))
        y, ey = y * g, ey * g.abs() + (U + silu_error(z.to(F64), dtype)) * (y * g).abs()
    return rounded(y, 1.01 * ey, dtype), (h, 1.01 * eh + 1e-37)


def quantize(x, block_rows):
    """Codes and scales as defined: fp32 division, e4m3 to nearest even."""
    rows, cols = x.shape
    kb, rb = -(-cols // 128), -(-rows // block_rows)
    p = torch.zeros(rb * block_rows, kb * 128)
    p[:rows, :cols] = x.float()
    g = p.view(rb, block_rows, kb, 128)
    scale = (g.abs().amax((1, 3)) / 448.0).clamp_min(2.0 ** -126)
    q = (g / scale[:, None, :, None]).to(torch.float8_e4m3fn)
    return q.view(rb * block_rows, kb * 128)[:rows, :cols], scale


def matmul(a, a_scale, w, w_scale, bias, relu, dtype):
    """(y, bound): the products of a block are exact; the tensor core's fp32 accumulation is
    taken at one ulp (2 u) of the block's absolute sum for each of its 128 / 32 steps; scale
    product, scaling and the sum over blocks round once each per block."""
    m, k = a.shape
    n = len(w)
    a, w = a.float().to(F64), w.float().to(F64)
    y, err, size = (torch.zeros(m, n, dtype=F64) for _ in range(3))
    col = torch.arange(n) // 128
    for i in range(-(-k // 128)):
        s = a_scale[:, i].to(F64)[:, None] * w_scale[:, i].to(F64)[col]
        part = a[:, i * 128:(i + 1) * 128] @ w[:, i * 128:(i + 1) * 128].t()
        full = a[:, i * 128:(i + 1) * 128].abs() @ w[:, i * 128:(i + 1) * 128].abs().t()
        y += s * part
        size += s.abs() * full
        err += s.abs() * full * 8 * U + 2 * U * (s * part).abs() + U * size
    if bias is not None:
        y = y + bias.to(F64)
        err = err + U * (y.abs() + err)
    if relu:
        y = y.clamp_min(0)
    return rounded(y, err, dtype)


def close(got, want, what):
    y, bound = want
    got = got.detach().cpu().to(F64)
    assert got.shape == y.shape, (what, got.shape, y.shape)
    assert torch.equal(got.isnan(), y.isnan()), f"{what}: NaN in other places"
    off = (got - y).abs()
    bad = ~(off <= bound) & ~y.isnan() & ~(got == y)
    if bad.any():
        i = tuple(bad.nonzero()[0].tolist())
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} outside the bound, first "
                             f"at {i}: {got[i].item()} for {y[i].item()}, bound {bound[i].item()}")
