"""Causal convolution, selective scan, 8-bit quantiser and product on the GPU, against plain
64-bit implementations (seq_ref.py) within bounds that count their roundings."""
import pytest
import torch

import cwg
import seq_ref as R

pytestmark = pytest.mark.gpu

DT = {"fp32": torch.float32, "bf16": torch.bfloat16}
GUARD = 7.25  # exact in both types


def gen(seed):
    return torch.Generator().manual_seed(seed)


def randn(g, *shape, dtype=torch.float32, std=1.0):
    return (torch.randn(*shape, generator=g) * std).to(dtype)


def wide(t, dev, left, right):
    """t as the columns left .. of a wider matrix of guard values, on the device."""
    m = torch.full((t.shape[0], left + t.shape[1] + right), GUARD, dtype=t.dtype, device=dev)
    v = m[:, left:left + t.shape[1]]
    v.copy_(t)
    return m, v


def offsets(lens):
    out = [0]
    for n in lens:
        out.append(out[-1] + n)
    return out


def put(v, dev):
    return None if v is None else v.to(dev)


# ---- causal convolution ---------------------------------------------------------------
LENS = [
    [1], [2], [40], [0], [0, 0, 5, 0], [1, 1, 1, 2, 3, 4], [31, 1, 0, 33, 2, 95],
    [32, 32, 64], [3, 29, 3, 200, 1], [700], [1] * 70,
]


def conv_case(dtype, lens, ch, width, kind, seed, bias=True, tail=3, slots="perm", pad=(0, 0)):
    g = gen(seed)
    dt = DT[dtype]
    starts = offsets(lens)
    T, n = starts[-1] + tail, len(lens)
    x = randn(g, T, ch, dtype=dt)
    w = randn(g, ch, width, std=0.6)
    b = randn(g, ch, std=0.3) if bias else None
    lines = n + 2
    state = randn(g, lines, width - 1, ch, dtype=dt)
    where = torch.randperm(lines, generator=g)[:n].to(torch.int32) if slots == "perm" else None
    resume = torch.randint(0, 2, (n,), generator=g).to(torch.uint8)
    return dict(x=x, w=w, bias=b, state=state, starts=starts, slots=where, resume=resume,
                kind=kind, dt=dt, pad=pad)


FLAG = {"silu": cwg.SILU, "relu": cwg.RELU, "none": 0}


def run_conv(c, dev):
    x = wide(c["x"], dev, *c["pad"])[1]
    ym, y = wide(torch.full_like(c["x"], GUARD), dev, *c["pad"])
    state = c["state"].to(dev)
    cwg.conv1d_causal(x, c["w"].to(dev), put(c["bias"], dev), y, state,
                      torch.tensor(c["starts"], dtype=torch.int32, device=dev),
                      put(c["slots"], dev), put(c["resume"], dev),
                      (cwg.BF16 if c["dt"] == torch.bfloat16 else 0) | FLAG[c["kind"]])
    cwg.device_status()
    return ym, y, state


def check_conv(c, dev):
    ym, y, state = run_conv(c, dev)
    want_state = c["state"].clone()
    for b in range(len(c["starts"]) - 1):
        s, e = c["starts"][b], c["starts"][b + 1]
        slot = b if c["slots"] is None else int(c["slots"][b])
        line = c["state"][slot] if c["resume"][b] else torch.zeros_like(c["state"][slot])
        want, new = R.conv1d(c["x"][s:e], c["w"], c["bias"], line, c["kind"])
        R.close(y[s:e], want, f"sequence {b}")
        want_state[slot] = new.to(c["dt"])
    assert torch.equal(state.cpu(), want_state)
    # rows of no sequence and the neighbouring columns are left as they were
    rest = ym.clone()
    rest[:c["starts"][-1], c["pad"][0]:c["pad"][0] + c["x"].shape[1]] = GUARD
    assert (rest == GUARD).all()


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("lens", LENS, ids=str)
def test_conv1d_sequences(cuda_dev, dtype, lens):
    check_conv(conv_case(dtype, lens, 96, 4, "silu", 1), cuda_dev)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("width", [2, 3, 4])
@pytest.mark.parametrize("ch,pad", [(1, (0, 0)), (7, (0, 0)), (40, (8, 8)), (40, (3, 0)),
                                    (264, (0, 16)), (521, (0, 0)), (1040, (0, 1))])
def test_conv1d_channels_and_strides(cuda_dev, dtype, width, ch, pad):
    kind = ("none", "relu", "silu")[(ch + width) % 3]
    check_conv(conv_case(dtype, [5, 0, 70, 1, 33], ch, width, kind, 2, bias=ch != 40, pad=pad,
                         slots="perm" if ch % 2 else None), cuda_dev)


def test_conv1d_without_cache_lines(cuda_dev):
    c = conv_case("bf16", [9, 40], 64, 4, "none", 3, tail=0)
    y = torch.empty_like(c["x"], device=cuda_dev)
    cwg.conv1d_causal(c["x"].to(cuda_dev), c["w"].to(cuda_dev), None, y, None,
                      torch.tensor(c["starts"], dtype=torch.int32, device=cuda_dev),
                      flags=cwg.BF16)
    for b, (s, e) in enumerate(((0, 9), (9, 49))):
        want, _ = R.conv1d(c["x"][s:e], c["w"], None, torch.zeros(3, 64), "none")
        R.close(y[s:e], want, f"sequence {b}")


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("n,ch,width", [(1, 2048, 4), (3, 7, 2), (17, 136, 3), (130, 72, 4),
                                        (5, 1, 4)])
def test_conv1d_step(cuda_dev, dtype, n, ch, width):
    c = conv_case(dtype, [1] * n, ch, width, "silu", 4, tail=0, pad=(8, 0))
    xs = wide(c["x"], cuda_dev, 8, 0)[1]
    y = torch.empty_like(c["x"], device=cuda_dev)
    state = c["state"].to(cuda_dev)
    slots = c["slots"].clone()
    slots[n // 2] = -1 if n > 1 else slots[0]  # a padding row: no line
    cwg.conv1d_causal_step(xs, c["w"].to(cuda_dev), c["bias"].to(cuda_dev), y, state,
                           slots.to(cuda_dev),
                           (cwg.BF16 if dtype == "bf16" else 0) | cwg.SILU)
    cwg.device_status()
    want_state = c["state"].clone()
    for i in range(n):
        slot = int(slots[i])
        line = c["state"][slot] if slot >= 0 else torch.zeros_like(c["state"][0])
        want, new = R.conv1d(c["x"][i:i + 1], c["w"], c["bias"], line, "silu")
        R.close(y[i:i + 1], want, f"row {i}")
        if slot >= 0:
            want_state[slot] = new.to(c["dt"])
    assert torch.equal(state.cpu(), want_state)


# ---- selective scan ----------------------------------------------------------------------
def ssm_case(dtype, lens, ch, groups, n, seed, gate=True, extras=True, pad=(0, 0), tail=2,
             slots="perm"):
    g = gen(seed)
    dt = DT[dtype]
    starts = offsets(lens)
    T, k = starts[-1] + tail, len(lens)
    c = dict(dt=dt, starts=starts, pad=pad, softplus=extras)
    c["u"] = randn(g, T, ch, dtype=dt)
    if extras:
        c["step"] = randn(g, T, ch, dtype=dt, std=0.7)
    else:
        c["step"] = (torch.rand(T, ch, generator=g) * 0.2).to(dt)
    c["B"], c["C"] = randn(g, T, groups * n, dtype=dt), randn(g, T, groups * n, dtype=dt)
    c["A"] = -torch.rand(ch, n, generator=g) * n - 0.05
    c["D"] = randn(g, ch) if extras else None
    c["bias"] = torch.rand(ch, generator=g) * 6 - 6 if extras else None
    c["z"] = randn(g, T, ch, dtype=dt) if gate else None
    c["state"] = randn(g, k + 2, ch, n)
    c["slots"] = torch.randperm(k + 2, generator=g)[:k].to(torch.int32) if slots else None
    c["resume"] = torch.randint(0, 2, (k,), generator=g).to(torch.uint8)
    return c


def run_ssm(c, dev, workspace=True, state=None):
    p = c["pad"]
    u, step, B, C = (wide(c[k], dev, *p)[1] for k in ("u", "step", "B", "C"))
    z = None if c["z"] is None else wide(c["z"], dev, *p)[1]
    ym, y = wide(torch.full_like(c["u"], GUARD), dev, *p)
    state = c["state"].to(dev) if state is None else state
    n = len(c["starts"]) - 1
    T, ch = c["u"].shape
    ws = None
    if workspace:
        ws = torch.empty(cwg.ssm_workspace_bytes(T, n, ch, c["A"].shape[1]), dtype=torch.uint8,
                         device=dev)
    cwg.ssm_scan(u, step, c["A"].to(dev), B, C, put(c["D"], dev), put(c["bias"], dev), z, y,
                 state, torch.tensor(c["starts"], dtype=torch.int32, device=dev),
                 put(c["slots"], dev), put(c["resume"], dev), ws,
                 (cwg.BF16 if c["dt"] == torch.bfloat16 else 0) |
                 (cwg.SOFTPLUS if c["softplus"] else 0))
    cwg.device_status()
    return ym, y, state


def ssm_want(c, rows, h):
    groups = c["B"].shape[1] // c["A"].shape[1]
    B, C = (c[k][rows].unflatten(1, (groups, -1)) for k in ("B", "C"))
    return R.ssm(c["u"][rows], c["step"][rows], c["A"], B, C, c["D"], c["bias"],
                 None if c["z"] is None else c["z"][rows], h, c["softplus"])


def check_ssm(c, dev, workspace=True):
    ym, y, state = run_ssm(c, dev, workspace)
    kept = torch.ones(len(state), dtype=torch.bool)
    for b in range(len(c["starts"]) - 1):
        s, e = c["starts"][b], c["starts"][b + 1]
        slot = b if c["slots"] is None else int(c["slots"][b])
        h = c["state"][slot] if c["resume"][b] else torch.zeros_like(c["state"][slot])
        want, new = ssm_want(c, slice(s, e), h)
        R.close(y[s:e], want, f"sequence {b}")
        R.close(state[slot], new, f"state of sequence {b}")
        kept[slot] = False
    assert torch.equal(state.cpu()[kept], c["state"][kept])
    rest = ym.clone()
    rest[:c["starts"][-1], c["pad"][0]:c["pad"][0] + c["u"].shape[1]] = GUARD
    assert (rest == GUARD).all()


@pytest.mark.parametrize("workspace", [True, False])
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("lens", LENS[:-1] + [[257, 0, 64]], ids=str)
def test_ssm_sequences(cuda_dev, dtype, lens, workspace):
    check_ssm(ssm_case(dtype, lens, 128, 1, 16, 5), cuda_dev, workspace)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("n", [1, 3, 4, 8, 12, 16, 23, 32, 64])
def test_ssm_states(cuda_dev, dtype, n):
    check_ssm(ssm_case(dtype, [37, 1, 70], 72, 1, n, 6, gate=n % 2 == 0, extras=n != 12),
              cuda_dev)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("ch,groups,pad", [(1, 1, (0, 0)), (6, 2, (0, 0)), (96, 3, (8, 8)),
                                           (130, 2, (1, 0)), (256, 4, (0, 8)), (201, 1, (0, 3))])
def test_ssm_channels_groups_and_strides(cuda_dev, dtype, ch, groups, pad):
    check_ssm(ssm_case(dtype, [33, 0, 65, 2], ch, groups, 16, 7, pad=pad,
                       slots="perm" if ch % 2 else None), cuda_dev)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_ssm_long_sequence(cuda_dev, dtype):
    check_ssm(ssm_case(dtype, [3000, 5], 64, 1, 16, 8), cuda_dev)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("lens,ch,groups,n,pad", [
    ([900, 0, 3500, 1, 800], 40, 1, 16, (0, 0)), ([1024, 1536], 128, 2, 16, (8, 8)),
    ([2600], 6, 2, 5, (0, 0)), ([1300, 1, 1800], 24, 1, 64, (0, 8)), ([256, 2000], 33, 1, 3, (0, 0)),
], ids=str)
def test_ssm_cut_sequences(cuda_dev, dtype, lens, ch, groups, n, pad):
    """Few channels and long sequences: cut into chunks of time when there is a workspace."""
    c = ssm_case(dtype, lens, ch, groups, n, 18, pad=pad)
    assert cwg.ssm_workspace_bytes(len(c["u"]), len(lens), ch, n) > 256
    check_ssm(c, cuda_dev)
    check_ssm(c, cuda_dev, workspace=False)


def test_ssm_cut_sequences_report_bad_indices(cuda_dev):
    for starts, slots in (([0, 1500, 1400, 3300], [0, 1, 2]), ([0, 900, 2000, 3300], [1, 1, 7])):
        c = ssm_case("bf16", [1100, 1100, 1100], 32, 1, 16, 19)
        c["starts"], c["slots"] = starts, torch.tensor(slots, dtype=torch.int32)
        with pytest.raises(cwg.CwgError) as e:
            run_ssm(c, cuda_dev)
        assert e.value.status == cwg.EINDEX
        cwg.device_status()


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("rows,ch,groups,n", [(1, 2048, 1, 16), (5, 6, 2, 12), (33, 264, 1, 64),
                                              (70, 128, 4, 4), (3, 70, 1, 23), (9, 64, 1, 8)])
def test_ssm_step(cuda_dev, dtype, rows, ch, groups, n):
    c = ssm_case(dtype, [1] * rows, ch, groups, n, 9, tail=0, gate=n != 4)
    dev = cuda_dev
    slots = c["slots"].clone()
    if rows > 1:
        slots[rows // 2] = -1
    state = c["state"].to(dev)
    y = torch.empty_like(c["u"], device=dev)
    cwg.ssm_step(c["u"].to(dev), c["step"].to(dev), c["A"].to(dev), c["B"].to(dev),
                 c["C"].to(dev), put(c["D"], dev), put(c["bias"], dev), put(c["z"], dev), y,
                 state, slots.to(dev),
                 (cwg.BF16 if dtype == "bf16" else 0) | cwg.SOFTPLUS)
    cwg.device_status()
    kept = torch.ones(len(state), dtype=torch.bool)
    for i in range(rows):
        slot = int(slots[i])
        h = c["state"][slot] if slot >= 0 else torch.zeros_like(c["state"][0])
        want, new = ssm_want(c, slice(i, i + 1), h)
        R.close(y[i:i + 1], want, f"row {i}")
        if slot >= 0:
            R.close(state[slot], new, f"state of row {i}")
            kept[slot] = False
    assert torch.equal(state.cpu()[kept], c["state"][kept])


# ---- indices in device memory -----------------------------------------------------------
def test_bad_indices_are_reported_and_stay_inside(cuda_dev):
    """A line out of range or given twice counts as no line, a sequence with bad offsets is
    left out; nothing outside the operands is touched, and the status says so."""
    dev = cuda_dev
    c = conv_case("fp32", [4, 40, 3, 6], 32, 4, "none", 10)
    c["slots"] = torch.tensor([1, 1, 99, 0], dtype=torch.int32)
    c["resume"] = torch.ones(4, dtype=torch.uint8)
    with pytest.raises(cwg.CwgError) as e:
        run_conv(c, dev)
    assert e.value.status == cwg.EINDEX
    cwg.device_status()  # cleared
    s = ssm_case("fp32", [4, 40, 3, 6], 32, 1, 16, 11)
    s["slots"], s["resume"] = c["slots"], c["resume"]
    with pytest.raises(cwg.CwgError) as e:
        run_ssm(s, dev)
    assert e.value.status == cwg.EINDEX
    for bad in ([0, 5, 3, 9], [0, 5, 60, 9], [-3, 5, 7, 9]):
        c = conv_case("bf16", [3, 3, 3], 32, 4, "none", 12)
        c["starts"] = bad
        with pytest.raises(cwg.CwgError) as e:
            run_conv(c, dev)
        assert e.value.status == cwg.EINDEX
        s = ssm_case("bf16", [3, 3, 3], 32, 1, 16, 13)
        s["starts"] = bad
        with pytest.raises(cwg.CwgError) as e:
            run_ssm(s, dev)
        assert e.value.status == cwg.EINDEX


def test_bad_lines_compute_as_no_line(cuda_dev):
    dev = cuda_dev
    s = ssm_case("fp32", [4, 40, 3, 6], 32, 1, 16, 14, tail=0)
    s["resume"] = torch.ones(4, dtype=torch.uint8)
    s["slots"] = torch.tensor([1, 1, 99, 0], dtype=torch.int32)
    T, ch = s["u"].shape
    y, state = torch.empty(T, ch, device=dev), s["state"].to(dev)
    cwg.ssm_scan(s["u"].to(dev), s["step"].to(dev), s["A"].to(dev), s["B"].to(dev),
                 s["C"].to(dev), s["D"].to(dev), s["bias"].to(dev), s["z"].to(dev), y, state,
                 torch.tensor(s["starts"], dtype=torch.int32, device=dev), s["slots"].to(dev),
                 s["resume"].to(dev), None, cwg.SOFTPLUS)
    with pytest.raises(cwg.CwgError):
        cwg.device_status()
    for b, slot in enumerate([1, -1, -1, 0]):
        rows = slice(s["starts"][b], s["starts"][b + 1])
        h = s["state"][slot] if slot >= 0 else torch.zeros_like(s["state"][0])
        want, new = ssm_want(s, rows, h)
        R.close(y[rows], want, f"sequence {b}")
        if slot >= 0:
            R.close(state[slot], new, f"state of sequence {b}")
    assert torch.equal(state[2:].cpu(), s["state"][2:])


# ---- 8-bit quantiser and product ---------------------------------------------------------
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("rows,cols,pad", [(1, 1, 0), (3, 128, 0), (130, 200, 8), (257, 333, 0),
                                           (64, 1024, 16), (5, 136, 3)])
def test_fp8_quantize(cuda_dev, dtype, block_rows, rows, cols, pad):
    g = gen(rows * cols)
    x = (torch.randn(rows, cols, generator=g) *
         torch.exp(4 * torch.randn(rows, 1, generator=g))).to(DT[dtype])
    if rows > 3:
        x[2] = 0
        x[3] *= 1e-30
    xd = wide(x, cuda_dev, pad, pad)[1]
    qm = torch.full((rows, cols + 16), 1.0, device=cuda_dev).to(torch.float8_e4m3fn)
    scale = torch.empty(-(-rows // block_rows), -(-cols // 128), device=cuda_dev)
    cwg.fp8_quantize(xd, qm[:, :cols], scale, block_rows, cwg.BF16 if dtype == "bf16" else 0)
    q, s = R.quantize(x, block_rows)
    assert torch.equal(scale.cpu(), s)
    assert torch.equal(qm[:, :cols].float().cpu(), q.float())
    assert (qm[:, cols:].float() == 1.0).all()


def test_fp8_quantize_rounds_as_the_division(cuda_dev):
    """Every bf16 magnitude of three binades under scales of many mantissas, among them
    quotients that lie between two codes, and groups near the ends of the range."""
    m = torch.arange(128, 512, dtype=torch.int32)
    x = (m << 16 | 0x3c000000).view(torch.float32)  # bf16 bit patterns as fp32
    rows = []
    for top in list(range(128, 256)) + [511]:
        big = torch.tensor((top << 16) | 0x3f000000, dtype=torch.int32).view(torch.float32)
        for part in x.split(127):
            rows.append(torch.cat((part, big.repeat(128 - len(part)))))
    x = torch.stack(rows)
    x = torch.cat((x, x * 2.0 ** -118, x * 2.0 ** 122, -x * 3.0 ** -40))
    q = torch.empty(x.shape, dtype=torch.float8_e4m3fn, device=cuda_dev)
    s = torch.empty(len(x), 1, device=cuda_dev)
    cwg.fp8_quantize(x.to(cuda_dev), q, s, 1)
    want, scale = R.quantize(x, 1)
    assert torch.equal(s.cpu(), scale) and torch.equal(q.float().cpu(), want.float())


def test_fp8_quantize_infinity_and_nan(cuda_dev):
    x = torch.ones(3, 256)
    x[0, 5], x[1, 130], x[2, 7] = float("inf"), float("nan"), -float("inf")
    q = torch.empty(3, 256, dtype=torch.float8_e4m3fn, device=cuda_dev)
    s = torch.empty(3, 2, device=cuda_dev)
    cwg.fp8_quantize(x.to(cuda_dev), q, s, 1)
    back = q.float().cpu().view(3, 2, 128) * s.cpu()[:, :, None]
    hurt = torch.tensor([[True, False], [False, True], [True, False]])
    assert back[hurt].isnan().all() and (back[~hurt] - 1).abs().max() <= 2.0 ** -4


def matmul_case(m, n, k, seed, dtype="fp32"):
    g = gen(seed)
    a, a_s = R.quantize(randn(g, m, k) * torch.exp(randn(g, m, 1)), 1)
    w, w_s = R.quantize(randn(g, n, k, std=k ** -0.5), 128)
    return a, a_s, w, w_s, randn(g, n, std=0.2)


def on_dev(q, dev):
    """e4m3 rows on 16-byte boundaries, with NaN behind every row's end."""
    ld = -(-q.shape[1] // 16) * 16
    t = torch.full((q.shape[0], ld), 0x7f, dtype=torch.uint8, device=dev).view(torch.float8_e4m3fn)
    t[:, :q.shape[1]].copy_(q)
    return t[:, :q.shape[1]]


def check_matmul(dev, m, n, k, dtype, relu, with_bias, seed=15, pad=(3, 2)):
    a, a_s, w, w_s, bias = matmul_case(m, n, k, seed)
    left, right = pad
    ym, y = wide(torch.zeros(m, n, dtype=DT[dtype]), dev, left, right)
    flags = (cwg.BF16 if dtype == "bf16" else 0) | (cwg.RELU if relu else 0)
    cwg.fp8_matmul(on_dev(a, dev), a_s.to(dev), on_dev(w, dev), w_s.to(dev),
                   bias.to(dev) if with_bias else None, y, flags)
    cwg.device_status()
    R.close(y, R.matmul(a, a_s, w, w_s, bias if with_bias else None, relu, DT[dtype]),
            f"{m}x{n}x{k}")
    assert (ym[:, :left] == GUARD).all() and (ym[:, left + n:] == GUARD).all()


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("m,n,k", [
    (1, 1, 1), (1, 128, 128), (1, 300, 100), (4, 1000, 4096), (16, 128, 640), (17, 257, 129),
    (33, 520, 1000), (64, 384, 256), (65, 130, 1543), (128, 128, 128), (200, 333, 700),
    (300, 512, 2048), (513, 640, 96),
])
def test_fp8_matmul(cuda_dev, dtype, m, n, k):
    check_matmul(cuda_dev, m, n, k, dtype, relu=(m + n) % 2 == 0, with_bias=m != 16)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("m,n,k", [(1300, 1700, 384), (2560, 1024, 129), (2600, 2304, 1000),
                                   (160, 9500, 100), (4864, 4300, 256)])
def test_fp8_matmul_pairs(cuda_dev, dtype, m, n, k):
    """Tiles of 256 x 256, more of them than pairs, cut at every edge."""
    check_matmul(cuda_dev, m, n, k, dtype, relu=dtype == "fp32", with_bias=True)
    check_matmul(cuda_dev, m, n, k, dtype, relu=False, with_bias=m % 3 == 0,
                 pad=(8, 24 - n % 8))


# ---- the Python mirror's checks ------------------------------------------------------------
def test_tensors_that_do_not_fit_are_named(cuda_dev):
    dev = cuda_dev
    x, y = torch.zeros(4, 64, device=dev), torch.zeros(4, 64, device=dev)
    w, st = torch.zeros(64, 4, device=dev), torch.zeros(5, 3, 64, device=dev)
    sl = torch.zeros(4, dtype=torch.int32, device=dev)
    for bad, what in (
        (dict(x=x.bfloat16()), "x is BFloat16"), (dict(x=x.t()), "x has strides"),
        (dict(y=y[:3]), "y has shape"), (dict(y=y.cpu()), "y is not on the call's device"),
        (dict(y=None), "y is missing"), (dict(w=w.double()), "w is Double"),
        (dict(y=torch.zeros(4, 128, device=dev)[:, ::2]), "y has strides"),
        (dict(x=x[:1].expand(4, 64)), "x has strides"), (dict(state=st[:, :2]), "state has shape"),
        (dict(state=st.transpose(0, 1).contiguous().transpose(0, 1)), "state is not contiguous"),
        (dict(slots=sl.long()), "slots is Long"), (dict(slots=sl[:2]), "slots has shape"),
        (dict(bias=w), "bias has shape"), (dict(x=3), "x is not a matrix"),
    ):
        a = dict(x=x, w=w, bias=None, y=y, state=st, slots=sl)
        a.update(bad)
        with pytest.raises(ValueError, match=what):
            cwg.conv1d_causal_step(**a)
    with pytest.raises(AttributeError):
        cwg.conv1d_causal_step(x, w, None, y, st, sl, 0, "stream")
    with pytest.raises(cwg.CwgError) as e:
        cwg.conv1d_causal_step(x, w, None, x, st, sl)
    assert e.value.status == cwg.EINVAL
    q = torch.zeros(4, 100, device=dev).to(torch.float8_e4m3fn)
    s1 = torch.zeros(4, 1, device=dev)
    with pytest.raises(cwg.CwgError) as e:  # rows that do not start on 16 bytes
        cwg.fp8_matmul(q, s1, q, s1[:1], None, torch.zeros(4, 4, device=dev))
    assert e.value.status == cwg.EINVAL


# ---- streams and graphs --------------------------------------------------------------------
def decode_calls(dev, seed=21):
    """A decoding step's calls on buffers of their own: quantise, product, convolution, scan."""
    g = gen(seed)
    n, ch, k = 5, 64, 200
    x = randn(g, n, k, dtype=torch.bfloat16).to(dev)
    q = on_dev(torch.zeros(n, k).to(torch.float8_e4m3fn), dev)
    s = torch.empty(n, 2, device=dev)
    w, w_s = R.quantize(randn(g, 2 * ch, k, std=0.1), 128)
    w, w_s = on_dev(w, dev), w_s.to(dev)
    xz = torch.empty(n, 2 * ch, dtype=torch.bfloat16, device=dev)
    cw, cb = randn(g, ch, 4).to(dev), randn(g, ch).to(dev)
    cst = randn(g, n, 3, ch, dtype=torch.bfloat16).to(dev)
    u = torch.empty(n, ch, dtype=torch.bfloat16, device=dev)
    dt, bc = (randn(g, n, m, dtype=torch.bfloat16).to(dev) for m in (ch, 32))
    A, D, db = -torch.rand(ch, 16, generator=g).to(dev), randn(g, ch).to(dev), randn(g, ch).to(dev)
    h, y = randn(g, n, ch, 16).to(dev), torch.empty_like(u)

    def calls():
        cwg.fp8_quantize(x, q, s, 1, cwg.BF16)
        cwg.fp8_matmul(q, s, w, w_s, None, xz, cwg.BF16)
        cwg.conv1d_causal_step(xz[:, :ch], cw, cb, u, cst, None, cwg.BF16 | cwg.SILU)
        cwg.ssm_step(u, dt, A, bc[:, :16], bc[:, 16:], D, db, xz[:, ch:], y, h, None,
                     cwg.BF16 | cwg.SOFTPLUS)
    return calls, (x, xz, cst, u, h, y)


def test_calls_follow_the_current_stream_and_replay(cuda_dev):
    """The same steps eagerly on a side stream, and captured there and replayed on another
    graph's heels, give what they give on the default stream, bit for bit."""
    plain, want = decode_calls(cuda_dev)
    for _ in range(3):
        plain()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    eager, got = decode_calls(cuda_dev)
    other, got2 = decode_calls(cuda_dev)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(20_000_000)  # what runs on the wrong stream would run too early
        got[0].mul_(2)
        got[0].div_(2)
        for _ in range(3):
            eager()
    side.synchronize()
    graph, graph2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        other()
    with torch.cuda.graph(graph2):
        other()
    graph.replay()
    graph2.replay()
    graph.replay()
    torch.cuda.synchronize()
    cwg.device_status()
    for a, b, c in zip(want, got, got2):
        assert torch.equal(a, b) and torch.equal(a, c)


# ---- the layers of a state space block, one after the other ----------------------------------
class Block:
    """Weights of a block and its calls, each checked against its 64-bit reference on the very
    inputs that it got: quantise, project to x and z, convolve, project to dt, B and C, scan with
    the gate z, project back."""

    def __init__(self, dev, d_model=136, ch=192, rank=24, n=16, lines=6, seed=31):
        g = gen(seed)
        self.dev, self.ch, self.rank, self.n = dev, ch, rank, n
        self.w = {}
        for name, out, k in (("in", 2 * ch, d_model), ("x", rank + 2 * n, ch), ("dt", ch, rank),
                             ("out", d_model, ch)):
            w = randn(g, out, k, std=k ** -0.5)
            q = on_dev(torch.zeros(out, k).to(torch.float8_e4m3fn), dev)
            s = torch.empty(-(-out // 128), -(-k // 128), device=dev)
            cwg.fp8_quantize(w.to(dev), q, s, 128)
            self.w[name] = (q, s)
        self.cw, self.cb = randn(g, ch, 4, std=0.4), randn(g, ch, std=0.1)
        self.A = -torch.arange(1.0, n + 1).repeat(ch, 1)
        self.D, self.db = torch.ones(ch), torch.rand(ch, generator=g) * 4 - 5
        self.conv = torch.zeros(lines, 3, ch, dtype=torch.bfloat16, device=dev)
        self.h = torch.zeros(lines, ch, n, device=dev)

    def project(self, name, x, bias=None):
        rows, k = x.shape
        q = on_dev(torch.zeros(rows, k).to(torch.float8_e4m3fn), self.dev)
        s = torch.empty(rows, -(-k // 128), device=self.dev)
        cwg.fp8_quantize(x, q, s, 1, cwg.BF16)
        want, scale = R.quantize(x.cpu(), 1)
        assert torch.equal(s.cpu(), scale) and torch.equal(q.float().cpu(), want.float())
        w, ws = self.w[name]
        y = torch.empty(rows, w.shape[0], dtype=torch.bfloat16, device=self.dev)
        cwg.fp8_matmul(q, s, w, ws, bias, y, cwg.BF16)
        R.close(y, R.matmul(q.cpu(), s.cpu(), w.cpu(), ws.cpu(), None, False, torch.bfloat16), name)
        return y

    def __call__(self, x, lens, slots, resume, step):
        dev, ch = self.dev, self.ch
        slots_d = torch.tensor(slots, dtype=torch.int32, device=dev)
        starts = offsets(lens)
        starts_d = torch.tensor(starts, dtype=torch.int32, device=dev)
        resume_d = torch.tensor(resume, dtype=torch.uint8, device=dev)
        xz = self.project("in", x)
        u = torch.empty(len(x), ch, dtype=torch.bfloat16, device=dev)
        conv, h = self.conv.cpu(), self.h.cpu()
        cw, cb = self.cw.to(dev), self.cb.to(dev)
        if step:
            cwg.conv1d_causal_step(xz[:, :ch], cw, cb, u, self.conv, slots_d, cwg.BF16 | cwg.SILU)
        else:
            cwg.conv1d_causal(xz[:, :ch], cw, cb, u, self.conv, starts_d, slots_d, resume_d,
                              cwg.BF16 | cwg.SILU)
        proj = self.project("x", u)
        r, n = self.rank, self.n
        dt = self.project("dt", proj[:, :r])
        y = torch.empty_like(u)
        args = (u, dt, self.A.to(dev), proj[:, r:r + n], proj[:, r + n:], self.D.to(dev),
                self.db.to(dev), xz[:, ch:], y, self.h)
        if step:
            cwg.ssm_step(*args, slots_d, cwg.BF16 | cwg.SOFTPLUS)
        else:
            ws = torch.empty(cwg.ssm_workspace_bytes(len(x), len(lens), ch, n),
                             dtype=torch.uint8, device=dev)
            cwg.ssm_scan(*args, starts_d, slots_d, resume_d, ws, cwg.BF16 | cwg.SOFTPLUS)
        cwg.device_status()
        for b, slot in enumerate(slots):
            rows = slice(starts[b], starts[b + 1])
            keep = 1 if resume[b] else 0
            want, line = R.conv1d(xz[rows, :ch].cpu(), self.cw, self.cb, conv[slot] * keep, "silu")
            R.close(u[rows], want, f"convolution {b}")
            assert torch.equal(self.conv[slot].cpu(), line.to(torch.bfloat16))
            p = proj[rows].cpu()
            want, state = R.ssm(u[rows].cpu(), dt[rows].cpu(), self.A, p[:, None, r:r + n],
                                p[:, None, r + n:], self.D, self.db, xz[rows, ch:].cpu(),
                                h[slot] * keep, True)
            R.close(y[rows], want, f"scan {b}")
            R.close(self.h[slot], state, f"state {b}")
        return self.project("out", y)


def test_block_prompts_then_steps(cuda_dev):
    g = gen(32)
    block = Block(cuda_dev)
    x = randn(g, 300, 136, dtype=torch.bfloat16).to(cuda_dev)
    out = block(x[:200], [70, 1, 129], [4, 0, 2], [0, 0, 0], step=False)
    assert out.shape == (200, 136) and out.isfinite().all()
    block(x[200:240], [30, 10], [4, 5], [1, 0], step=False)      # one goes on, one begins
    for i in range(3):
        y = block(x[240 + 4 * i:244 + 4 * i], [1] * 4, [2, 4, 5, 0], [1] * 4, step=True)
        assert y.isfinite().all()


def test_prompt_in_pieces_is_the_whole_prompt(cuda_dev):
    """A prompt cut at any place and resumed, and the same prompt token by token: the
    convolution gives the same bits, the scan stays within its bound."""
    c = conv_case("bf16", [90], 72, 4, "silu", 33, tail=0)
    c["resume"][:] = 1
    _, whole, line = run_conv(c, cuda_dev)
    for cuts in ([1], [2, 50], [89], [3, 4, 5, 40]):
        st, out = c["state"].to(cuda_dev), torch.empty_like(whole)
        for s, e in zip([0] + cuts, cuts + [90]):
            cwg.conv1d_causal(c["x"][s:e].to(cuda_dev), c["w"].to(cuda_dev), c["bias"].to(cuda_dev),
                              out[s:e], st, torch.tensor([0, e - s], dtype=torch.int32,
                                                         device=cuda_dev),
                              c["slots"].to(cuda_dev), c["resume"].to(cuda_dev),
                              cwg.BF16 | cwg.SILU)
        assert torch.equal(out, whole) and torch.equal(st, line)
    st, out = c["state"].to(cuda_dev), torch.empty_like(whole)
    for t in range(90):
        cwg.conv1d_causal_step(c["x"][t:t + 1].to(cuda_dev), c["w"].to(cuda_dev),
                               c["bias"].to(cuda_dev), out[t:t + 1], st, c["slots"].to(cuda_dev),
                               cwg.BF16 | cwg.SILU)
    assert torch.equal(out, whole) and torch.equal(st, line)

    s = ssm_case("fp32", [90], 40, 1, 16, 34, tail=0)
    h = s["state"][int(s["slots"][0])]
    want, end = ssm_want(s, slice(0, 90), h)
    dev = {k: put(s[k], cuda_dev) for k in ("u", "step", "A", "B", "C", "D", "bias", "z", "slots")}
    for cuts in ([1], [33, 64], list(range(1, 90))):
        st, out = s["state"].to(cuda_dev), torch.empty(90, 40, device=cuda_dev)
        for a, b in zip([0] + cuts, cuts + [90]):
            rows = [dev[k][a:b] for k in ("u", "step", "B", "C", "z")]
            call = (rows[0], rows[1], dev["A"], rows[2], rows[3], dev["D"], dev["bias"], rows[4],
                    out[a:b], st)
            if b - a == 1:
                cwg.ssm_step(*call, dev["slots"], cwg.SOFTPLUS)
            else:
                cwg.ssm_scan(*call, torch.tensor([0, b - a], dtype=torch.int32, device=cuda_dev),
                             dev["slots"], torch.ones(1, dtype=torch.uint8, device=cuda_dev), None,
                             cwg.SOFTPLUS)
        R.close(out, want, f"cuts {cuts[:3]}")
        R.close(st[int(s["slots"][0])], end, f"state, cuts {cuts[:3]}")


# ---- calls at the edges --------------------------------------------------------------------
def test_fresh_sequences_do_not_read_their_lines(cuda_dev):
    c = conv_case("fp32", [3, 1, 0, 40], 32, 4, "silu", 41)
    s = ssm_case("bf16", [3, 1, 0, 40], 32, 1, 16, 42)
    for case, check in ((c, check_conv), (s, check_ssm)):
        fresh = case["slots"][case["resume"] == 0].long()
        assert len(fresh)
        case["state"][fresh] = float("nan")
        case["state"][-1] = torch.where(torch.isnan(case["state"][-1]), 0.0, 1.0)
        check(case, cuda_dev)


def test_no_tokens_still_sets_the_lines(cuda_dev):
    c = conv_case("bf16", [0, 0], 40, 3, "none", 43, tail=0)
    c["resume"] = torch.tensor([0, 1], dtype=torch.uint8)
    check_conv(c, cuda_dev)
    s = ssm_case("fp32", [0, 0], 40, 1, 16, 44, tail=0)
    s["resume"] = c["resume"]
    check_ssm(s, cuda_dev)


def test_many_sequences(cuda_dev):
    """More sequences than the convolution keeps offsets of in shared memory."""
    lens = [1, 0, 3, 2, 9] * 330
    check_conv(conv_case("bf16", lens, 8, 4, "silu", 45), cuda_dev)
    s = ssm_case("fp32", lens[:1200], 8, 1, 4, 46)
    check_ssm(s, cuda_dev)


def test_ordinary_launches_give_the_same_bits(cuda_dev):
    a, got = decode_calls(cuda_dev)
    b, want = decode_calls(cuda_dev)
    orig = cwg.BF16
    a()
    try:
        cwg.BF16 = orig | cwg.NO_PDL
        b()
    finally:
        cwg.BF16 = orig
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(got, want))


def test_offsets_beyond_32_bits(cuda_dev):
    """Rows and cache lines more than 2^31 elements (and 2^32 bytes) from the first."""
    dev = cuda_dev
    ld, ch, rows = (1 << 28) + 8, 32, 18
    big = torch.empty(ld * (rows - 1) + 2 * ch, dtype=torch.bfloat16, device=dev)
    x, y = (big.as_strided((rows, ch), (ld, 1), off) for off in (0, ch))
    c = conv_case("bf16", [rows], ch, 4, "silu", 47, tail=0)
    lines = (1 << 31) // (3 * ch) + 3  # 4.3 GB
    state = torch.empty(lines, 3, ch, dtype=torch.bfloat16, device=dev)
    slot = torch.tensor([lines - 1], dtype=torch.int32, device=dev)
    one = torch.ones(1, dtype=torch.uint8, device=dev)
    starts = torch.tensor([0, rows], dtype=torch.int32, device=dev)
    x.copy_(c["x"])
    state[-1] = c["state"][0].to(dev)
    cwg.conv1d_causal(x, c["w"].to(dev), c["bias"].to(dev), y, state, starts, slot, one,
                      cwg.BF16 | cwg.SILU)
    want, line = R.conv1d(c["x"], c["w"], c["bias"], c["state"][0], "silu")
    R.close(y, want, "rows")
    assert torch.equal(state[-1].cpu(), line.to(torch.bfloat16))
    cwg.conv1d_causal_step(x[-1:], c["w"].to(dev), c["bias"].to(dev), y[-1:], state, slot,
                           cwg.BF16 | cwg.SILU)
    want, line = R.conv1d(c["x"][-1:], c["w"], c["bias"], line.to(torch.bfloat16), "silu")
    R.close(y[-1:], want, "step")
    del state

    s = ssm_case("bf16", [rows], ch, 1, 16, 48, tail=0)
    u = x
    u.copy_(s["u"])
    lines = (1 << 31) // (ch * 16) + 3  # 8.6 GB
    h = torch.empty(lines, ch, 16, device=dev)
    h[-1] = s["state"][0].to(dev)
    dv = {k: put(s[k], dev) for k in ("step", "A", "B", "C", "D", "bias", "z")}
    cwg.ssm_scan(u, dv["step"], dv["A"], dv["B"], dv["C"], dv["D"], dv["bias"], dv["z"], y, h,
                 starts, slot * 0 + lines - 1, one, None, cwg.BF16 | cwg.SOFTPLUS)
    want, end = ssm_want(s, slice(0, rows), s["state"][0])
    R.close(y, want, "scan")
    R.close(h[-1], end, "state")
    before = h[-1].cpu()
    cwg.ssm_step(u[-1:], dv["step"][-1:], dv["A"], dv["B"][-1:], dv["C"][-1:], dv["D"],
                 dv["bias"], dv["z"][-1:], y[-1:], h, slot * 0 + lines - 1,
                 cwg.BF16 | cwg.SOFTPLUS)
    want, end = ssm_want(s, slice(rows - 1, rows), before)
    R.close(y[-1:], want, "scan step")
    R.close(h[-1], end, "state after the step")
    del h

    q = torch.empty(rows, ch, dtype=torch.float8_e4m3fn, device=dev)
    sc = torch.empty(rows, 1, device=dev)
    cwg.fp8_quantize(x, q, sc, 1, cwg.BF16)
    want, scale = R.quantize(s["u"], 1)
    assert torch.equal(q.float().cpu(), want.float()) and torch.equal(sc.cpu(), scale)
    w, w_s = R.quantize(randn(gen(49), ch, ch), 128)
    cwg.fp8_matmul(q, sc, on_dev(w, dev), w_s.to(dev), None, y, cwg.BF16)
    R.close(y, R.matmul(want, scale, w, w_s, None, False, torch.bfloat16), "product")
    cwg.device_status()


def test_two_threads_at_once(cuda_dev):
    """Two host threads, each on a stream of its own, make the same calls as one."""
    import threading

    plain, want = decode_calls(cuda_dev)
    for _ in range(20):
        plain()
    torch.cuda.synchronize()
    runs = [decode_calls(cuda_dev) for _ in range(2)]
    torch.cuda.synchronize()
    errors = []

    def work(calls):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(20):
                    calls()
                torch.cuda.current_stream().synchronize()
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work, args=(c,)) for c, _ in runs]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors
    for _, got in runs:
        assert all(torch.equal(a, b) for a, b in zip(want, got))


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("pad", [(3, 2), (0, 0)])
@pytest.mark.parametrize("m,n,k", [
    (16, 1024, 4096), (9, 2048, 512), (20, 9000, 256),        # tiles of 16 and 32 rows
    (72, 2048, 2100), (128, 300, 1024), (90, 11008, 140),     # 32 rows, cut 4, 8 and 1 ways
    (250, 1000, 700), (130, 260, 3000), (1000, 384, 520),
    (40, 19000, 260), (700, 1000, 1100), (190, 4096, 520),    # 64 rows, cut 1, 2 and 2 ways
    (1100, 2048, 200), (100, 20000, 130),                     # 64 and 128 rows
    (400, 1600, 4100), (500, 3000, 4000),                     # 128 rows, cut 2 ways and not
    (1300, 2048, 260),                                        # pairs
])
def test_fp8_matmul_tiles(cuda_dev, dtype, pad, m, n, k):
    check_matmul(cuda_dev, m, n, k, dtype, relu=m % 3 == 0, with_bias=n % 3 != 0, pad=pad)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("left,right", [(2, 2), (1, 0), (4, 4), (8, 24)])
def test_fp8_matmul_pairs_row_alignment(cuda_dev, dtype, left, right):
    """Rows of y that are aligned to 16 bytes, to 4 and to an element."""
    n = 1690
    right += -(left + n + right) % (8 if left == 8 else 2)
    check_matmul(cuda_dev, 1540, n, 260, dtype, relu=left == 2, with_bias=left != 4,
                 pad=(left, right))


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("ch,groups,n", [(520, 1, 12), (514, 2, 20), (516, 2, 4), (330, 1, 23),
                                         (512, 1, 16), (128, 1, 60)])
def test_ssm_step_many_rows(cuda_dev, dtype, ch, groups, n):
    rows = 301
    c = ssm_case(dtype, [1] * rows, ch, groups, n, 51, tail=0)
    dev = cuda_dev
    state = c["state"].to(dev)
    y = torch.empty_like(c["u"], device=dev)
    cwg.ssm_step(*(put(c[k], dev) for k in ("u", "step", "A", "B", "C", "D", "bias", "z")), y,
                 state, put(c["slots"], dev), (cwg.BF16 if dtype == "bf16" else 0) | cwg.SOFTPLUS)
    cwg.device_status()
    for i in range(0, rows, 20):
        slot = int(c["slots"][i])
        want, new = ssm_want(c, slice(i, i + 1), c["state"][slot])
        R.close(y[i:i + 1], want, f"row {i}")
        R.close(state[slot], new, f"state of row {i}")


@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("cols", [384, 333])
def test_fp8_quantize_zeros_and_small_values(cuda_dev, block_rows, cols):
    x = torch.zeros(260, cols)
    x[1] = -0.0
    x[2, ::2] = 3e-39                      # denormal: the scale's lower bound
    x[3] = torch.linspace(-1e-35, 1e-35, cols)
    x[200:] = 0.5
    q = torch.empty(x.shape, dtype=torch.float8_e4m3fn, device=cuda_dev)
    want, scale = R.quantize(x, block_rows)
    s = torch.empty(scale.shape, device=cuda_dev)
    cwg.fp8_quantize(x.to(cuda_dev), q, s, block_rows)
    assert torch.equal(s.cpu(), scale) and torch.equal(q.float().cpu(), want.float())


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("lens,ch,n", [([384], 32, 16), ([400], 40, 16), ([1025], 7, 12),
                                       ([600], 1024, 4), ([300, 0, 900], 64, 23),
                                       ([0, 255, 257, 513], 16, 64)], ids=str)
def test_ssm_short_chunks(cuda_dev, dtype, lens, ch, n):
    check_ssm(ssm_case(dtype, lens, ch, 1, n, 53), cuda_dev)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("ch,groups,n,pad", [(2100, 1, 4, (0, 0)), (1504, 2, 16, (8, 8)),
                                             (640, 1, 23, (3, 0)), (512, 4, 64, (0, 0))])
def test_ssm_many_short_prompts(cuda_dev, dtype, ch, groups, n, pad):
    """Sequences of a tile on average, one of them of several."""
    check_ssm(ssm_case(dtype, [9, 0, 1, 150, 31, 33, 2, 64, 5, 7, 3, 4, 8], ch, groups, n, 54,
                       pad=pad), cuda_dev)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("cols", [384, 333])
def test_fp8_quantize_bytes(cuda_dev, dtype, block_rows, cols):
    """The codes themselves: zeros keep their sign, in groups of ordinary, tiny, huge and zero
    scale, and so do values that round to zero."""
    g = gen(55)
    x = torch.randn(260, cols, generator=g)
    x[:, ::5] = -0.0
    x[:, 1::5] = 0.0
    x[:, 2::15] *= 1e-8
    x[1] *= 1e-30
    x[2] *= 3e37
    x[3] = -0.0
    x[128:256] = -0.0
    x[130, 7] = 2.0 ** -120
    x = x.to(DT[dtype])
    q = torch.empty(x.shape, dtype=torch.float8_e4m3fn, device=cuda_dev)
    want, scale = R.quantize(x, block_rows)
    s = torch.empty(scale.shape, device=cuda_dev)
    cwg.fp8_quantize(x.to(cuda_dev), q, s, block_rows, cwg.BF16 if dtype == "bf16" else 0)
    assert torch.equal(s.cpu(), scale)
    assert torch.equal(q.view(torch.uint8).cpu(), want.contiguous().view(torch.uint8))


@pytest.mark.parametrize("groups", [1, 4])
def test_ssm_one_workspace_for_calls_of_many_sizes(cuda_dev, groups):
    """A workspace for the largest call serves every smaller one, cut or not, and is not left."""
    ch, n = 256, 16
    size = cwg.ssm_workspace_bytes(2100, 4, ch, n)
    whole = torch.full((size + 4096,), 0x5a, dtype=torch.uint8, device=cuda_dev)
    for lens in ([2100], [1500, 600], [600], [512], [384], [0, 1000, 900, 200], [70, 3]):
        c = ssm_case("bf16", lens, ch, groups, n, 56, tail=0)
        y, state = torch.empty_like(c["u"], device=cuda_dev), c["state"].to(cuda_dev)
        dv = {k: put(c[k], cuda_dev) for k in ("u", "step", "A", "B", "C", "D", "bias", "z")}
        cwg.ssm_scan(*dv.values(), y, state,
                     torch.tensor(c["starts"], dtype=torch.int32, device=cuda_dev),
                     c["slots"].to(cuda_dev), c["resume"].to(cuda_dev), whole[:size],
                     cwg.BF16 | cwg.SOFTPLUS)
        cwg.device_status()
        for b, slot in enumerate(c["slots"].tolist()):
            rows = slice(c["starts"][b], c["starts"][b + 1])
            h = c["state"][slot] if c["resume"][b] else torch.zeros_like(c["state"][slot])
            want, new = ssm_want(c, rows, h)
            R.close(y[rows], want, f"{lens}: sequence {b}")
            R.close(state[slot], new, f"{lens}: state of sequence {b}")
        assert (whole[size:] == 0x5a).all()


# ---- status and codes ----------------------------------------------------------------------
@pytest.mark.parametrize("default_stream", [False, True])
def test_device_status_waits_for_the_calls_that_it_reports(cuda_dev, default_stream):
    """Without a stream the status is that of torch's current stream, where the tensor calls
    run, and of the default one: a bad line behind other work on either is not missed."""
    dev = cuda_dev
    x, y, state = (torch.zeros(*shape, device=dev) for shape in ((2, 64), (2, 64), (2, 3, 64)))
    w, slots = torch.zeros(64, 4, device=dev), torch.tensor([0, 9], dtype=torch.int32, device=dev)
    cwg.conv1d_causal_step(x, w, None, y, state)  # a kernel's first launch may wait for the GPU
    cwg.device_status()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(torch.cuda.default_stream() if default_stream else side):
        torch.cuda._sleep(200_000_000)  # about 0.1 s
        cwg.conv1d_causal_step(x, w, None, y, state, slots)
    try:
        with torch.cuda.stream(side), pytest.raises(cwg.CwgError) as e:
            cwg.device_status()
        assert e.value.status == cwg.EINDEX
        cwg.device_status()  # cleared
    finally:
        torch.cuda.synchronize()
        cwg.lib().cwg_device_status(None)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_silu_of_large_negative_values(cuda_dev, dtype):
    """The convolution's activation and the scan's gate down to -100: within the stated error as
    far as results are above 1.1e-36, and next to zero beyond."""
    v = (-torch.arange(0, 1601) / 16).to(DT[dtype])  # exact in fp32, rounded once in bf16
    ch = len(v)
    x = v[None]
    w = torch.tensor([0.0, 1.0]).repeat(ch, 1)
    flags = cwg.BF16 if dtype == "bf16" else 0
    y, state = torch.empty_like(x, device=cuda_dev), torch.zeros(1, 1, ch, dtype=DT[dtype])
    cwg.conv1d_causal_step(x.to(cuda_dev), w.to(cuda_dev), None, y, state.to(cuda_dev), None,
                           flags | cwg.SILU)
    # decay 1, step 1, u B C = 1: the gate's argument is all that counts
    one, ab = torch.ones(1, ch, dtype=DT[dtype]), torch.ones(1, 1, dtype=DT[dtype])
    gated = torch.empty_like(y)
    cwg.ssm_step(one.to(cuda_dev), one.to(cuda_dev), torch.zeros(ch, 1, device=cuda_dev),
                 ab.to(cuda_dev), ab.to(cuda_dev), None, None, x.to(cuda_dev), gated,
                 torch.zeros(1, ch, 1, device=cuda_dev), None, flags)
    gated_prompt = torch.empty_like(y)
    cwg.ssm_scan(one.to(cuda_dev), one.to(cuda_dev), torch.zeros(ch, 1, device=cuda_dev),
                 ab.to(cuda_dev), ab.to(cuda_dev), None, None, x.to(cuda_dev), gated_prompt, None,
                 torch.tensor([0, 1], dtype=torch.int32, device=cuda_dev), flags=flags)
    z = x.to(torch.float64)
    want = R.silu(z)
    normal = z >= -87
    assert normal.sum() > 1300 and (~normal).sum() > 100
    bound = (R.silu_error(z, DT[dtype]) + R.U) * want.abs()
    bound = R.half_step(DT[dtype]) * (want.abs() + bound) + bound
    for got in (y, gated, gated_prompt):
        off = (got.cpu().to(torch.float64) - want).abs()
        assert (off <= torch.where(normal, bound, 1.5e-36)).all()


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("lens", [[5, 1], [37], [32, 64], [700]], ids=str)
def test_ssm_states_that_forget_at_once(cuda_dev, dtype, lens):
    """A = -infinity, or so large that A log2(e) is beyond fp32: exp(step A) is zero for every
    step, so a state is its last token's drive, wherever the last tile of 32 tokens ends."""
    ch, n = 40, 6
    c = ssm_case(dtype, lens, ch, 1, n, 57, gate=False, extras=False, tail=0)
    c["step"] = c["step"] + 0.125
    c["A"][:, 1::3], c["A"][:, 2::3] = -float("inf"), -3e38
    for workspace in (False, True):
        _, y, state = run_ssm(c, cuda_dev, workspace)
        for b, slot in enumerate(c["slots"].tolist()):
            t = c["starts"][b + 1] - 1
            drive = (c["step"][t].double() * c["u"][t].double())[:, None] * c["B"][t].double()
            off = (state[slot].cpu().double() - drive)[:, [1, 2, 4, 5]].abs()
            # step times u and the product with B round once each
            assert (off <= (2.1 * R.U * drive.abs() + 1e-37)[:, [1, 2, 4, 5]]).all()
            assert state[slot].isfinite().all()
        assert y.isfinite().all()


@pytest.mark.parametrize("tokens,ch", [(2100, 64), (700, 1100)])  # cut into chunks, and not
def test_captured_prompts_serve_changing_batches(cuda_dev, tokens, ch):
    """Prompts' calls captured once and replayed with other offsets, lines and inputs in the same
    tensors, a padded batch among them, give the bits of the same calls made eagerly."""
    dev, bf, n, lines = cuda_dev, torch.bfloat16, 6, 8
    g = gen(58)
    w, w_s = R.quantize(randn(g, 2 * ch, 136, std=0.1), 128)
    w, w_s = on_dev(w, dev), w_s.to(dev)
    cw, cb = randn(g, ch, 4).to(dev), randn(g, ch).to(dev)
    A, D = -torch.rand(ch, 16, generator=g).to(dev), randn(g, ch).to(dev)

    def buffers():
        x = torch.zeros(tokens, 136, dtype=bf, device=dev)
        q = on_dev(torch.zeros(tokens, 136).to(torch.float8_e4m3fn), dev)
        s = torch.empty(tokens, 2, device=dev)
        xz = torch.zeros(tokens, 2 * ch, dtype=bf, device=dev)
        bc = torch.zeros(tokens, 32, dtype=bf, device=dev)
        u, y = (torch.zeros(tokens, ch, dtype=bf, device=dev) for _ in range(2))
        conv = torch.zeros(lines, 3, ch, dtype=bf, device=dev)
        h = torch.zeros(lines, ch, 16, device=dev)
        starts = torch.zeros(n + 1, dtype=torch.int32, device=dev)
        slots = torch.full((n,), -1, dtype=torch.int32, device=dev)
        resume = torch.zeros(n, dtype=torch.uint8, device=dev)
        ws = torch.empty(cwg.ssm_workspace_bytes(tokens, n, ch, 16), dtype=torch.uint8, device=dev)

        def calls():
            cwg.fp8_quantize(x, q, s, 1, cwg.BF16)
            cwg.fp8_matmul(q, s, w, w_s, None, xz, cwg.BF16)
            cwg.conv1d_causal(xz[:, :ch], cw, cb, u, conv, starts, slots, resume,
                              cwg.BF16 | cwg.SILU)
            cwg.ssm_scan(u, xz[:, ch:], A, bc[:, :16], bc[:, 16:], D, None, xz[:, ch:], y, h,
                         starts, slots, resume, ws, cwg.BF16 | cwg.SOFTPLUS)
        return calls, (x, bc, starts, slots, resume), (xz, u, y, conv, h)

    eager, ins, want = buffers()
    captured, ins2, got = buffers()
    eager()
    captured()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured()
    batches = (([tokens], [3], [0]), ([tokens // 2, 1, tokens // 3], [3, 0, 7], [1, 0, 0]),
               ([], [], []), ([5, 0, 9, 64, 2, 33], [7, 1, 0, 3, 4, 5], [1, 1, 1, 1, 0, 0]))
    for lens, slot, keep in batches:
        pad = n - len(lens)
        data = (randn(g, tokens, 136, dtype=bf), randn(g, tokens, 32, dtype=bf),
                torch.tensor(offsets(lens) + [sum(lens)] * pad, dtype=torch.int32),
                torch.tensor(slot + [-1] * pad, dtype=torch.int32),
                torch.tensor(keep + [0] * pad, dtype=torch.uint8))
        for to in (ins, ins2):
            for a, b in zip(to, data):
                a.copy_(b)
        eager()
        graph.replay()
        torch.cuda.synchronize()
        cwg.device_status()
        for a, b in zip(want, got):
            assert torch.equal(a, b), lens
        assert want[2].isfinite().all()
