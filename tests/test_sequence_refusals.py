"""What the sequence layers and the 8-bit product refuse before any CUDA call, through the C
ABI (fake addresses: nothing is read) and through the Python mirror."""
import ctypes

import pytest
import torch

import cwg

X, W, Y, S, I = 0x10000, 0x20000, 0x400000, 0x800000, 0xC00000  # far apart, 16-byte aligned


def conv(**kw):
    a = dict(x=X, ldx=64, w=W, bias=None, y=Y, ldy=64, state=S, starts=I, slots=I, resume=None,
             tokens=10, n_seq=2, n_slots=4, channels=64, width=4, flags=0)
    a.update(kw)
    return cwg.lib().cwg_conv1d_causal(*a.values(), None)


def conv_step(**kw):
    a = dict(x=X, ldx=64, w=W, bias=None, y=Y, ldy=64, state=S, slots=I, n=3, n_slots=4,
             channels=64, width=4, flags=0)
    a.update(kw)
    return cwg.lib().cwg_conv1d_causal_step(*a.values(), None)


@pytest.mark.parametrize("kw,status", [
    (dict(x=None), cwg.EINVAL), (dict(y=None), cwg.EINVAL), (dict(w=None), cwg.EINVAL),
    (dict(starts=None), cwg.EINVAL), (dict(x=X + 2), cwg.EINVAL), (dict(w=W + 2), cwg.EINVAL),
    (dict(ldx=63), cwg.EINVAL), (dict(ldy=10), cwg.EINVAL), (dict(tokens=-1), cwg.EINVAL),
    (dict(tokens=(1 << 30) + 1), cwg.EINVAL), (dict(n_seq=-1), cwg.EINVAL),
    (dict(channels=0), cwg.EINVAL), (dict(width=1), cwg.EINVAL),
    (dict(width=5), cwg.EUNSUPPORTED), (dict(flags=cwg.SILU | cwg.RELU), cwg.EINVAL),
    (dict(flags=cwg.SOFTPLUS), cwg.EINVAL), (dict(flags=cwg.FORCE_TC), cwg.EINVAL),
    (dict(y=X), cwg.EINVAL),                            # in place
    (dict(y=X + 64 * 4, ldx=64), cwg.EINVAL),           # one row further
    (dict(ldx=96, ldy=96, y=X + 63 * 4), cwg.EINVAL),   # one shared column
    (dict(slots=None, n_slots=1), cwg.EINVAL),          # line b of too few lines
    (dict(n_slots=-1), cwg.EINVAL), (dict(state=S + 2), cwg.EINVAL),
    (dict(state=X), cwg.EINVAL), (dict(state=Y + 2556), cwg.EINVAL),  # lines among the rows
    (dict(state=Y - 4 * 3 * 64 * 4 + 4), cwg.EINVAL), (dict(state=X, n_slots=1 << 30), cwg.EINVAL),
    (dict(n_seq=0), cwg.OK), (dict(tokens=0, state=None), cwg.OK),
])
def test_conv1d_refuses(kw, status):
    assert conv(**kw) == status


@pytest.mark.parametrize("kw,status", [
    (dict(state=None), cwg.EINVAL), (dict(n=-1), cwg.EINVAL), (dict(n=0), cwg.OK),
    (dict(slots=None, n_slots=2), cwg.EINVAL), (dict(width=5), cwg.EUNSUPPORTED),
    (dict(y=X), cwg.EINVAL), (dict(ldx=8), cwg.EINVAL),
])
def test_conv1d_step_refuses(kw, status):
    assert conv_step(**kw) == status


def ssm(step=False, workspace=None, size=0, **kw):
    op = cwg.cwg_ssm(u=X, dt=X + 0x40000, B=X + 0x80000, C=X + 0xC0000, z=None, y=Y, ldu=64,
                     lddt=64, ldb=16, ldc=16, ldz=0, ldy=64, A=W, D=None, dt_bias=None, state=S,
                     starts=I, slots=I, resume=None, tokens=10, n_seq=2, n_slots=4, channels=64,
                     groups=1, states=16, flags=0)
    for k, v in kw.items():
        setattr(op, k, v)
    if step:
        return cwg.lib().cwg_ssm_step(ctypes.byref(op), None)
    return cwg.lib().cwg_ssm_scan(ctypes.byref(op), workspace, size, None)


@pytest.mark.parametrize("step", [False, True])
@pytest.mark.parametrize("kw", [
    dict(u=None), dict(dt=None), dict(A=None), dict(B=None), dict(C=None), dict(y=None),
    dict(ldu=63), dict(lddt=1), dict(ldb=15), dict(ldc=3), dict(ldy=0), dict(z=W, ldz=5),
    dict(channels=0), dict(groups=0), dict(groups=3), dict(states=0), dict(tokens=-1),
    dict(A=W + 1), dict(D=W + 2), dict(flags=cwg.SILU), dict(flags=cwg.RELU), dict(y=X),
    dict(B=Y, ldb=64), dict(slots=None, n_slots=1), dict(state=S + 1),
    dict(state=X), dict(state=X + 0x40000), dict(state=X + 0x80000 + 16), dict(state=X + 0xC0000),
    dict(state=Y + 4), dict(z=S + 16, ldz=64),
], ids=str)
def test_ssm_refuses(step, kw):
    assert ssm(step, **kw) == cwg.EINVAL


def test_ssm_refuses_and_accepts():
    assert ssm(states=65, ldb=65, ldc=65) == cwg.EUNSUPPORTED
    assert ssm(True, state=None) == cwg.EINVAL
    assert ssm(starts=None) == cwg.EINVAL
    assert ssm(n_seq=0) == cwg.OK and ssm(True, tokens=0) == cwg.OK
    assert ssm(tokens=0, state=None) == cwg.OK
    need = cwg.ssm_workspace_bytes(10, 2, 64, 16)
    assert need > 0
    assert ssm(workspace=0x1000001, size=1 << 30) == cwg.EINVAL  # misaligned
    assert ssm(workspace=0x1000000, size=need - 1) == cwg.EINVAL
    for bad in ((-1, 1, 64, 16), (10, -1, 64, 16), (10, 1, 0, 16), (10, 1, 64, 65)):
        assert cwg.ssm_workspace_bytes(*bad) == 0


def quantize(**kw):
    a = dict(x=X, ldx=200, q=Y, ldq=208, scale=S, lds=2, rows=3, cols=200, block_rows=1, flags=0)
    a.update(kw)
    return cwg.lib().cwg_fp8_quantize(*a.values(), None)


@pytest.mark.parametrize("kw,status", [
    (dict(x=None), cwg.EINVAL), (dict(q=None), cwg.EINVAL), (dict(scale=None), cwg.EINVAL),
    (dict(ldx=199), cwg.EINVAL), (dict(ldq=100), cwg.EINVAL), (dict(lds=1), cwg.EINVAL),
    (dict(block_rows=2), cwg.EINVAL), (dict(cols=0), cwg.EINVAL), (dict(rows=-1), cwg.EINVAL),
    (dict(flags=cwg.RELU), cwg.EINVAL), (dict(x=X + 1), cwg.EINVAL), (dict(rows=0), cwg.OK),
    (dict(q=X), cwg.EINVAL), (dict(scale=X + 64), cwg.EINVAL), (dict(scale=Y + 400), cwg.EINVAL),
    (dict(cols=(1 << 30) + 1, ldx=1 << 31), cwg.EINVAL),
])
def test_fp8_quantize_refuses(kw, status):
    assert quantize(**kw) == status


def matmul(**kw):
    a = dict(a=X, lda=208, a_scale=S, lda_scale=2, w=W, ldw=208, w_scale=S + 4096, ldw_scale=2,
             bias=None, y=Y, ldy=300, m=5, n=300, k=200, flags=0)
    a.update(kw)
    return cwg.lib().cwg_fp8_matmul(*a.values(), None)


@pytest.mark.parametrize("kw,status", [
    (dict(a=None), cwg.EINVAL), (dict(w=None), cwg.EINVAL), (dict(y=None), cwg.EINVAL),
    (dict(a_scale=None), cwg.EINVAL), (dict(w_scale=None), cwg.EINVAL),
    (dict(a=X + 8), cwg.EINVAL), (dict(w=W + 1), cwg.EINVAL), (dict(lda=200), cwg.EINVAL),
    (dict(ldw=204), cwg.EINVAL), (dict(lda=192), cwg.EINVAL), (dict(ldy=299), cwg.EINVAL),
    (dict(lda_scale=1), cwg.EINVAL), (dict(ldw_scale=1), cwg.EINVAL), (dict(m=-1), cwg.EINVAL),
    (dict(n=0), cwg.EINVAL), (dict(k=0), cwg.EINVAL), (dict(flags=cwg.SILU), cwg.EINVAL),
    (dict(bias=S + 2), cwg.EINVAL), (dict(m=0), cwg.OK), (dict(y=X), cwg.EINVAL),
    (dict(y=W + 16), cwg.EINVAL), (dict(y=S), cwg.EINVAL), (dict(m=(1 << 30) + 1), cwg.EINVAL),
])
def test_fp8_matmul_refuses(kw, status):
    assert matmul(**kw) == status


def test_python_mirror_names_the_wrong_argument():
    t = torch.zeros(4, 8)
    i = torch.zeros(2, dtype=torch.int32)
    w = torch.zeros(8, 4)
    with pytest.raises(ValueError, match="x is not on a CUDA device"):
        cwg.conv1d_causal(t, w, None, t, None, i)
    with pytest.raises(ValueError, match="x is not a matrix"):
        cwg.conv1d_causal_step(t[0], w, None, t, None)
    with pytest.raises(ValueError, match="u is not on a CUDA device"):
        cwg.ssm_scan(t, t, w, t, t, None, None, None, t, None, i)
    with pytest.raises(ValueError, match="u is not on a CUDA device"):
        cwg.ssm_step(t, t, w, t, t, None, None, None, t, None)
    with pytest.raises(ValueError, match="a is not on a CUDA device"):
        cwg.fp8_matmul(t, t, t, t, None, t)
    with pytest.raises(ValueError, match="x is not a matrix"):
        cwg.fp8_quantize(None, t, t, 1)
    with pytest.raises(TypeError):
        cwg.fp8_quantize(t, t, t, 1, "flags")


def test_strerror_of_bad_index():
    assert "index" in cwg.strerror(cwg.EINDEX)


def test_pair_kernel_votes_on_every_wait():
    """A bounded wait may give up for some lanes of a warp and not for others.  The pair
    product's warps run tcgen05 instructions and barriers behind their waits, which all lanes
    have to reach together, so every answer goes through a vote before it is used."""
    import os

    with open(os.path.join(cwg.HERE, "csrc", "cwg_fp8.cu")) as f:
        text = f.read()
    body = text[text.index("fp8_matmul_pair(const"):text.index("static int make_map")]
    waits = [s for s in body.split(";") if "mbar_wait(" in s]
    assert len(waits) >= 5
    for s in waits:
        assert "__all_sync(" in s, s


BIG = (1 << 30) + 1


def test_sizes_beyond_the_row_limit_are_refused():
    """Channels and sequences are bounded as rows are: index sums stay inside int."""
    assert conv(channels=BIG, ldx=BIG, ldy=BIG) == cwg.EINVAL
    assert conv(n_seq=BIG) == cwg.EINVAL
    assert conv(n_seq=BIG, slots=None, n_slots=BIG) == cwg.EINVAL
    assert conv_step(channels=(1 << 31) - 1, ldx=1 << 31, ldy=1 << 31) == cwg.EINVAL
    for step in (False, True):
        assert ssm(step, channels=BIG, ldu=BIG, lddt=BIG, ldy=BIG) == cwg.EINVAL
        assert ssm(step, channels=BIG, groups=BIG, states=1, ldu=BIG, lddt=BIG, ldy=BIG, ldb=BIG,
                   ldc=BIG) == cwg.EINVAL
    assert ssm(n_seq=BIG) == cwg.EINVAL


@pytest.mark.parametrize("size", [
    (10, 1, (1 << 31) - 1, 16), (10, 1, BIG, 16), (BIG, 1, 64, 16), ((1 << 31) - 1, 1, 64, 16),
    (10, BIG, 64, 16), (10, (1 << 31) - 1, (1 << 31) - 1, 64),
])
def test_workspace_query_beyond_the_limits(size):
    """In a process of its own: a query must answer 0, whatever it is asked."""
    import subprocess
    import sys

    code = f"import sys; sys.path.insert(0, {cwg.HERE!r}); import cwg; " \
           f"print(cwg.ssm_workspace_bytes{size})"
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stderr
    assert int(r.stdout) == 0


@pytest.mark.parametrize("size", [(1 << 30, 1, 64, 16), (1, 1 << 30, 64, 16), (1 << 30, 1, 1 << 30, 64)])
def test_workspace_query_at_the_limits(size):
    assert 0 < cwg.ssm_workspace_bytes(*size) < 1 << 40


# ---- operands that share bytes --------------------------------------------------------------
# conv(): x and y are 10 rows of 256 bytes, w 1024 bytes, state 4 lines of 768, 3 offsets
Y_END, S_END = Y + 10 * 256, S + 4 * 768


@pytest.mark.parametrize("kw", [
    dict(w=Y), dict(w=Y - 1020), dict(w=Y_END - 4), dict(bias=Y + 256), dict(bias=Y - 252),
    dict(starts=Y_END - 4), dict(starts=Y - 8), dict(slots=Y - 4), dict(slots=Y + 8),
    dict(resume=Y - 1), dict(resume=Y_END - 1),
    dict(w=S), dict(w=S - 1020), dict(bias=S_END - 4), dict(starts=S - 8), dict(slots=S_END - 4),
    dict(resume=S + 1), dict(resume=S - 1),
], ids=str)
def test_conv1d_refuses_outputs_over_dense_operands(kw):
    assert conv(**kw) == cwg.EINVAL


@pytest.mark.parametrize("kw", [dict(w=Y), dict(bias=Y + 4), dict(slots=Y + 3 * 256 - 4),
                                dict(w=S), dict(bias=S + 4), dict(slots=S_END - 4)], ids=str)
def test_conv1d_step_refuses_outputs_over_dense_operands(kw):
    assert conv_step(**kw) == cwg.EINVAL


def refused_by_arguments(status):
    """Whether a call ended in the checks; without a GPU the others end in a CUDA error."""
    return status in (cwg.EINVAL, cwg.EUNSUPPORTED)


@pytest.mark.skipif(torch.cuda.is_available(), reason="would read the fake addresses")
@pytest.mark.parametrize("call", [
    lambda: conv(), lambda: conv_step(), lambda: ssm(), lambda: ssm(True), lambda: quantize(),
    lambda: matmul(),
    # dense operands right before and behind y and the cache lines
    lambda: conv(w=Y - 1024, bias=Y_END, starts=S - 12, slots=S_END, resume=Y - 1026),
    # and between the columns that a wider matrix gives to y
    lambda: conv(ldy=128, bias=Y + 256, slots=Y + 504, starts=Y + 768, resume=Y + 1022),
    lambda: ssm(ldy=128, D=Y + 256, dt_bias=Y + 9 * 512 + 256, slots=Y + 504),
    # one row: the distance to the next says nothing
    lambda: conv(tokens=1, ldy=1 << 40, bias=Y + 256),
    # disjoint columns of one matrix, far apart rows
    lambda: conv(ldx=1 << 40, ldy=1 << 40, y=X + 256, state=None),
])
def test_operands_that_share_no_byte_pass_the_checks(call):
    assert not refused_by_arguments(call())


A_BYTES, H_END = 64 * 16 * 4, S + 4 * 64 * 16 * 4


@pytest.mark.parametrize("step", [False, True])
@pytest.mark.parametrize("kw", [
    dict(A=Y), dict(A=Y - A_BYTES + 4), dict(D=Y_END - 4), dict(dt_bias=Y - 252),
    dict(slots=Y - 4), dict(A=S), dict(A=H_END - 4), dict(D=S - 252), dict(dt_bias=S + 64),
    dict(slots=H_END - 4),
], ids=str)
def test_ssm_refuses_outputs_over_dense_operands(step, kw):
    assert ssm(step, **kw) == cwg.EINVAL


@pytest.mark.parametrize("kw", [dict(starts=Y - 8), dict(starts=Y_END - 4), dict(resume=Y - 1),
                                dict(starts=H_END - 4), dict(resume=S - 1)], ids=str)
def test_ssm_scan_refuses_outputs_over_offsets(kw):
    assert ssm(**kw) == cwg.EINVAL


# one sequence that is cut: 4096 rows of 64 channels, 16 states
LONG = dict(u=X, dt=X + 0x1000000, B=X + 0x2000000, C=X + 0x3000000, y=X + 0x4000000, z=X + 0x5000000,
            ldz=64, A=X + 0x6000000, D=X + 0x6010000, dt_bias=X + 0x6020000, starts=X + 0x6030000,
            slots=X + 0x6040000, resume=X + 0x6050000, state=X + 0x7000000, tokens=4096, n_seq=1)
WS = 0x20000000


@pytest.mark.parametrize("name,size", [
    ("u", 4096 * 256), ("dt", 4096 * 256), ("B", 4096 * 64), ("C", 4096 * 64), ("y", 4096 * 256),
    ("z", 4096 * 256), ("A", A_BYTES), ("D", 256), ("dt_bias", 256), ("starts", 8), ("slots", 4),
    ("resume", 1), ("state", 4 * A_BYTES)])
def test_ssm_refuses_a_workspace_over_an_operand(name, size):
    need = cwg.ssm_workspace_bytes(4096, 1, 64, 16)
    assert need > 256
    at = WS + 0x10000  # the operand begins inside the workspace, and ends inside it
    assert ssm(workspace=at - need + 256, size=need, **dict(LONG, **{name: at})) == cwg.EINVAL
    at = WS - size + (1 if name == "resume" else 4)
    assert ssm(workspace=WS, size=need, **dict(LONG, **{name: at})) == cwg.EINVAL


@pytest.mark.skipif(torch.cuda.is_available(), reason="would read the fake addresses")
def test_ssm_workspace_beside_the_operands_passes_the_checks():
    need = cwg.ssm_workspace_bytes(4096, 1, 64, 16)
    assert not refused_by_arguments(ssm(workspace=WS, size=need, **dict(LONG, D=WS - 256)))
    assert not refused_by_arguments(ssm(workspace=WS, size=need, **dict(LONG, D=WS + need)))


@pytest.mark.parametrize("kw", [dict(bias=Y), dict(bias=Y - 1196), dict(bias=Y + 4 * 1200 + 1196),
                                dict(bias=Y + 1204, ldy=400)], ids=str)
def test_fp8_matmul_refuses_a_bias_inside_y(kw):
    assert matmul(**kw) == cwg.EINVAL


def test_overlaps_of_far_apart_rows():
    """Row distances whose products with the rows pass 64 bits: (2^22 + 1) rows of fp32 at 2^40."""
    far, rows = 1 << 40, (1 << 22) + 1
    assert conv(tokens=rows, ldx=far, ldy=far, y=X + 4 * far, state=None) == cwg.EINVAL
    assert conv(tokens=rows, ldx=far, ldy=far, y=X + 4 * far + 252, state=None) == cwg.EINVAL
    assert conv(tokens=rows, ldx=far, ldy=far, x=X + 4 * far, y=X, state=None) == cwg.EINVAL
    assert conv(tokens=rows, ldy=far, bias=Y + 4 * far, state=None) == cwg.EINVAL
    assert quantize(rows=rows, ldx=far, q=X + 8 * far) == cwg.EINVAL
    assert matmul(m=4 * (rows - 1) + 1, lda=far, y=X + far) == cwg.EINVAL
    assert matmul(m=rows, ldy=far, bias=Y + (1 << 50)) == cwg.EINVAL


# ---- one workspace for calls of many sizes ----------------------------------------------------
def test_workspace_of_the_largest_call_serves_smaller_ones():
    """The query never falls where tokens or sequences grow: one workspace serves every call of
    at most as many."""
    tokens = (0, 1, 100, 255, 256, 383, 384, 511, 512, 513, 600, 767, 768, 1000, 1024, 1500, 2048,
              4095, 4096, 6127, 8192, 20000, 1 << 17, 1 << 30)
    seqs = (0, 1, 2, 3, 4, 7, 8, 16, 37, 74, 75, 1000, 1 << 30)
    for ch, n in ((1, 1), (64, 16), (219, 4), (1024, 16), (1184, 16), (2048, 64), (2368, 16),
                  (4096, 16), (40, 33), (600, 64)):
        size = [[cwg.ssm_workspace_bytes(t, s, ch, n) for s in seqs] for t in tokens]
        for i in range(len(tokens)):
            for j in range(len(seqs)):
                assert size[i][j] >= 256
                assert i == 0 or size[i][j] >= size[i - 1][j], (tokens[i], seqs[j], ch, n)
                assert j == 0 or size[i][j] >= size[i][j - 1], (tokens[i], seqs[j], ch, n)


@pytest.mark.skipif(torch.cuda.is_available(), reason="would read the fake addresses")
@pytest.mark.parametrize("largest,calls", [
    ((8192, 16), [(8192, 1), (8192, 2), (4096, 1), (600, 1), (512, 1), (384, 1), (10, 5)]),
    ((600, 1), [(513, 1), (512, 1), (511, 1), (385, 1), (1, 1)]),
    ((1024, 3), [(1024, 1), (1024, 2), (768, 2), (512, 2)]),
])
def test_calls_accept_the_largest_ones_workspace(largest, calls):
    size = cwg.ssm_workspace_bytes(*largest, 1024, 16)
    for tokens, n in calls:
        for groups in (1, 2, 64):
            op = dict(LONG, tokens=tokens, n_seq=n, channels=1024, groups=groups, ldu=1024,
                      lddt=1024, ldz=1024, ldy=1024, ldb=16 * groups, ldc=16 * groups,
                      **{k: X + (i << 28) for i, k in enumerate(("u", "dt", "B", "C", "y", "z"))},
                      state=X + (6 << 28), n_slots=16)
            op.update({k: X + (7 << 28) + (i << 20) for i, k in enumerate(
                ("A", "D", "dt_bias", "starts", "slots", "resume"))})
            assert not refused_by_arguments(ssm(workspace=8 << 28, size=size, **op)), (tokens, n)
