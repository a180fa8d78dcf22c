"""ctypes binding of libcwg (include/cwg.h) -- the Python side of the C ABI.

This module only forwards to the compiled library: there is no CPU or PyTorch
fallback anywhere.  If ``lib/libcwg.so`` is missing, importing succeeds but the
first call raises ``RuntimeError`` telling the user to build it.

Device-pointer calls take ``torch`` tensors (used here purely as device-memory
and stream plumbing) or raw integer addresses; host-pointer calls take numpy
arrays.
"""
from __future__ import annotations

import ctypes
import os
import sys
from dataclasses import dataclass

import numpy as np

HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.environ.get("CWG_LIB") or os.path.join(HERE, "lib", "libcwg.so")
HEADER = os.path.join(os.path.dirname(HERE), "include", "cwg.h")

# status codes and flags (include/cwg.h)
OK, EINVAL, EUNSUPPORTED, ECUDA, ETIMEOUT, ENOMEM, ENODEV, ERANGE = 0, -1, -2, -3, -4, -5, -6, -7
EINDEX = -8
RELU, BF16, FORCE_FFMA, FORCE_TC, TC_SINGLE, TC_FULL16 = 0x1, 0x2, 0x10, 0x20, 0x40, 0x80
TC_NOPAIR, NO_SPLIT, TC_X3, NO_PDL = 0x100, 0x200, 0x400, 0x800
SILU, SOFTPLUS = 0x1000, 0x2000
PATH_FFMA, PATH_TC = 1, 2
ORDER_GRID, ORDER_RUNS, ORDER_ROUND = 0, 1, 2  # cwg_choice.order

EXPORTED = (
    "fused_winograd_f23", "cwg_tiles_fused", "cwg_last_status", "cwg_weight_bytes",
    "cwg_weight_transform", "cwg_weight_import", "cwg_conv3x3_fused",
    "cwg_host_workspace_bytes", "cwg_conv3x3_fused_host", "cwg_select", "cwg_strerror",
    "cwg_last_cuda_error", "cwg_device_status", "cwg_launch_count", "cwg_version",
    "cwg_nonfused_workspace_bytes", "cwg_conv3x3_nonfused", "cwg_selftest_wait_timeout",
    "cwg_conv1d_causal", "cwg_conv1d_causal_step", "cwg_ssm_workspace_bytes", "cwg_ssm_scan",
    "cwg_ssm_step", "cwg_fp8_quantize", "cwg_fp8_matmul",
)


class CwgError(RuntimeError):
    """A libcwg call returned a negative status."""

    def __init__(self, status: int, what: str):
        self.status = status
        super().__init__(f"{what}: {strerror(status)} (status {status})")


class cwg_choice(ctypes.Structure):
    _fields_ = [
        ("m", ctypes.c_int), ("path", ctypes.c_int), ("tiles_per_cta", ctypes.c_int),
        ("cout_per_cta", ctypes.c_int), ("cin_chunk", ctypes.c_int), ("threads", ctypes.c_int),
        ("smem_bytes", ctypes.c_int), ("tmem_cols", ctypes.c_int), ("ctas", ctypes.c_longlong),
        ("gemm_flops", ctypes.c_double), ("alg_bytes", ctypes.c_double),
        ("mma_products", ctypes.c_int), ("ctas_launched", ctypes.c_longlong),
        ("order", ctypes.c_int),
    ]


class cwg_ssm(ctypes.Structure):
    _fields_ = (
        [(f, ctypes.c_void_p) for f in ("u", "dt", "B", "C", "z", "y")] +
        [(f, ctypes.c_longlong) for f in ("ldu", "lddt", "ldb", "ldc", "ldz", "ldy")] +
        [(f, ctypes.c_void_p) for f in ("A", "D", "dt_bias", "state", "starts", "slots",
                                        "resume")] +
        [(f, ctypes.c_int) for f in ("tokens", "n_seq", "n_slots", "channels", "groups",
                                     "states")] +
        [("flags", ctypes.c_uint)])


@dataclass
class Choice:
    m: int
    path: int
    tiles_per_cta: int
    cout_per_cta: int
    cin_chunk: int
    threads: int
    smem_bytes: int
    tmem_cols: int
    ctas: int
    gemm_flops: float
    alg_bytes: float
    mma_products: int
    ctas_launched: int
    order: int

    @property
    def path_name(self) -> str:
        return {PATH_FFMA: "ffma", PATH_TC: "tcgen05"}.get(self.path, "?")

    @property
    def order_name(self) -> str:
        return {ORDER_GRID: "one unit per CTA pair", ORDER_RUNS: "persistent pairs, equal tile runs",
                ORDER_ROUND: "persistent pairs, round robin"}.get(self.order, "?")


_lib = None


def lib() -> ctypes.CDLL:
    """Loads libcwg.so once; raises if it has not been built."""
    global _lib
    if _lib is not None:
        return _lib
    if not os.path.exists(LIB_PATH):
        raise RuntimeError(
            f"libcwg.so not found at {LIB_PATH}: build it with "
            "`python -c 'import __graft_entry__ as g; g.build()'` (no CPU fallback exists)")
    L = ctypes.CDLL(LIB_PATH)
    vp, i, u, sz = ctypes.c_void_p, ctypes.c_int, ctypes.c_uint, ctypes.c_size_t
    fp = ctypes.POINTER(ctypes.c_float)
    L.fused_winograd_f23.argtypes = [fp, fp, fp, i, i]
    L.fused_winograd_f23.restype = None
    L.cwg_tiles_fused.argtypes = [fp, fp, fp, i, i, i, i]
    L.cwg_tiles_fused.restype = i
    L.cwg_last_status.argtypes = []
    L.cwg_last_status.restype = i
    L.cwg_weight_bytes.argtypes = [i, i, i, u]
    L.cwg_weight_bytes.restype = sz
    L.cwg_weight_transform.argtypes = [vp, vp, i, i, i, u, vp]
    L.cwg_weight_transform.restype = i
    L.cwg_weight_import.argtypes = [vp, vp, i, i, i, u, vp]
    L.cwg_weight_import.restype = i
    L.cwg_conv3x3_fused.argtypes = [vp, vp, vp, vp, i, i, i, i, i, i, u, vp]
    L.cwg_conv3x3_fused.restype = i
    L.cwg_host_workspace_bytes.argtypes = [i, i, i, i, i, u]
    L.cwg_host_workspace_bytes.restype = sz
    L.cwg_conv3x3_fused_host.argtypes = [vp, vp, vp, vp, vp, sz, i, i, i, i, i, i, u, vp]
    L.cwg_conv3x3_fused_host.restype = i
    L.cwg_select.argtypes = [i, i, i, i, i, i, u, ctypes.POINTER(cwg_choice)]
    L.cwg_select.restype = i
    L.cwg_strerror.argtypes = [i]
    L.cwg_strerror.restype = ctypes.c_char_p
    L.cwg_last_cuda_error.argtypes = []
    L.cwg_last_cuda_error.restype = i
    L.cwg_device_status.argtypes = [vp]
    L.cwg_device_status.restype = i
    L.cwg_launch_count.argtypes = []
    L.cwg_launch_count.restype = ctypes.c_longlong
    L.cwg_version.argtypes = []
    L.cwg_version.restype = ctypes.c_char_p
    L.cwg_selftest_wait_timeout.argtypes = [vp]
    L.cwg_selftest_wait_timeout.restype = i
    L.cwg_nonfused_workspace_bytes.argtypes = [i, i, i, i, i, i]
    L.cwg_nonfused_workspace_bytes.restype = sz
    L.cwg_conv3x3_nonfused.argtypes = [vp, vp, vp, vp, vp, sz, i, i, i, i, i, i, u, vp]
    L.cwg_conv3x3_nonfused.restype = i
    ll = ctypes.c_longlong
    L.cwg_conv1d_causal.argtypes = [vp, ll, vp, vp, vp, ll, vp, vp, vp, vp, i, i, i, i, i, u, vp]
    L.cwg_conv1d_causal.restype = i
    L.cwg_conv1d_causal_step.argtypes = [vp, ll, vp, vp, vp, ll, vp, vp, i, i, i, i, u, vp]
    L.cwg_conv1d_causal_step.restype = i
    L.cwg_ssm_workspace_bytes.argtypes = [i, i, i, i]
    L.cwg_ssm_workspace_bytes.restype = sz
    L.cwg_ssm_scan.argtypes = [ctypes.POINTER(cwg_ssm), vp, sz, vp]
    L.cwg_ssm_scan.restype = i
    L.cwg_ssm_step.argtypes = [ctypes.POINTER(cwg_ssm), vp]
    L.cwg_ssm_step.restype = i
    L.cwg_fp8_quantize.argtypes = [vp, ll, vp, ll, vp, ll, i, i, i, u, vp]
    L.cwg_fp8_quantize.restype = i
    L.cwg_fp8_matmul.argtypes = [vp, ll, vp, ll, vp, ll, vp, ll, vp, vp, ll, i, i, i, u, vp]
    L.cwg_fp8_matmul.restype = i
    _lib = L
    return L


def strerror(status: int) -> str:
    try:
        return lib().cwg_strerror(int(status)).decode()
    except RuntimeError:
        return f"status {status}"


def _check(status: int, what: str) -> None:
    if status != OK:
        if status == ECUDA:
            what = f"{what} (cudaError {lib().cwg_last_cuda_error()})"
        raise CwgError(status, what)


def _ptr(t) -> int | None:
    """Device address of a torch tensor (or an int address, or None)."""
    if t is None:
        return None
    if isinstance(t, int):
        return t
    return int(t.data_ptr())


def _stream(stream) -> int | None:
    if stream is None:
        return None
    if isinstance(stream, int):
        return stream
    return int(stream.cuda_stream)


# ---- selector -----------------------------------------------------------------
def select(n: int, c_in: int, c_out: int, h: int, w: int, m: int = 0, flags: int = 0) -> Choice:
    """Tile/kernel choice for a layer (replaces CacheAdaptiveAutotiler.select_best_tile)."""
    out = cwg_choice()
    _check(lib().cwg_select(n, c_in, c_out, h, w, m, flags, ctypes.byref(out)), "cwg_select")
    return Choice(*(getattr(out, f) for f, _ in cwg_choice._fields_))


def weight_bytes(c_in: int, c_out: int, m: int = 0, flags: int = 0) -> int:
    return int(lib().cwg_weight_bytes(c_in, c_out, m, flags))


# ---- device-pointer layer API -----------------------------------------------------
def weight_transform(g, U, c_in: int, c_out: int, m: int = 0, flags: int = 0, stream=None):
    _check(lib().cwg_weight_transform(_ptr(g), _ptr(U), c_in, c_out, m, flags, _stream(stream)),
           "cwg_weight_transform")


def weight_import(U_ref, U, c_in: int, c_out: int, m: int, flags: int = 0, stream=None):
    _check(lib().cwg_weight_import(_ptr(U_ref), _ptr(U), c_in, c_out, m, flags,
                                   _stream(stream)), "cwg_weight_import")


def conv3x3_fused(x, U, bias, y, n: int, c_in: int, c_out: int, h: int, w: int, m: int = 0,
                  flags: int = 0, stream=None) -> None:
    _check(lib().cwg_conv3x3_fused(_ptr(x), _ptr(U), _ptr(bias), _ptr(y), n, c_in, c_out, h, w,
                                   m, flags, _stream(stream)), "cwg_conv3x3_fused")


def nonfused_workspace_bytes(n, c_in, c_out, h, w, m) -> int:
    return int(lib().cwg_nonfused_workspace_bytes(n, c_in, c_out, h, w, m))


def conv3x3_nonfused(x, U, bias, y, workspace, workspace_bytes: int, n: int, c_in: int,
                     c_out: int, h: int, w: int, m: int, flags: int = 0, stream=None) -> None:
    """Non-fused ablation: three passes over HBM (fp32; U from weight_transform with
    FORCE_FFMA)."""
    _check(lib().cwg_conv3x3_nonfused(_ptr(x), _ptr(U), _ptr(bias), _ptr(y), _ptr(workspace),
                                      workspace_bytes, n, c_in, c_out, h, w, m, flags,
                                      _stream(stream)), "cwg_conv3x3_nonfused")


def host_workspace_bytes(n, c_in, c_out, h, w, flags=0) -> int:
    return int(lib().cwg_host_workspace_bytes(n, c_in, c_out, h, w, flags))


def conv3x3_fused_host(x_host: int, U, bias, y_host: int, workspace, workspace_bytes: int,
                       n, c_in, c_out, h, w, m=0, flags=0, stream=None) -> None:
    _check(lib().cwg_conv3x3_fused_host(_ptr(x_host), _ptr(U), _ptr(bias), _ptr(y_host),
                                        _ptr(workspace), workspace_bytes, n, c_in, c_out, h, w,
                                        m, flags, _stream(stream)), "cwg_conv3x3_fused_host")


def device_status(stream=None) -> None:
    """Raises CwgError(ETIMEOUT) if a bounded device wait gave up since the last check,
    CwgError(ERANGE) if an fp16 tensor-core operand overflowed, or CwgError(EINDEX) if a
    sequence layer met a bad offset or cache line.  Waits for `stream`, whose calls it then
    reports; without one for both streams that calls without one run on: the default stream and
    torch's current stream.  Calls on other streams may still be running."""
    streams = [_stream(stream)]
    torch = sys.modules.get("torch")
    if stream is None and torch is not None and torch.cuda.is_initialized():
        current = torch.cuda.current_stream().cuda_stream
        if current:
            streams.append(current)
    # the codes of failures grow with their weight: ECUDA, ETIMEOUT, ERANGE, EINDEX
    bad = [st for st in [lib().cwg_device_status(s) for s in streams] if st != OK]
    if bad:
        _check(max(bad), "device status")


def selftest_wait_timeout(stream=None) -> None:
    """Launches a kernel whose bounded wait runs out; the next device_status() raises
    CwgError(ETIMEOUT)."""
    _check(lib().cwg_selftest_wait_timeout(_stream(stream)), "cwg_selftest_wait_timeout")


def launch_count() -> int:
    return int(lib().cwg_launch_count())


def version() -> str:
    return lib().cwg_version().decode()


# ---- sequence layers and the 8-bit matrix product ---------------------------------
# These take torch tensors: sizes and row distances come from the tensors (a column range
# of a wider matrix is passed as it is), and every tensor is checked before the call, since
# a wrong type, device or size would otherwise only show as wrong memory accesses.
# ValueError names the argument; what the library itself refuses is a CwgError.  Without a
# stream a call runs on torch's current stream, as an operator of torch's on the same tensors
# would (the calls above, which take addresses, run on the default stream then).  The checks
# are compiled (csrc/cwg_torch.cpp): a decoding step's kernels are shorter than they would
# take in Python.
_torch_ext = None


def _ext():
    """Loads lib/cwg_torch.so once and gives it libcwg's entry points."""
    global _torch_ext
    if _torch_ext is None:
        import importlib.util

        import torch  # noqa: F401  (its libraries are the module's)

        path = os.path.join(HERE, "lib", "cwg_torch.so")
        if not os.path.exists(path):
            raise RuntimeError(f"cwg_torch.so not found at {path}: build it with "
                               "`python -c 'import __graft_entry__ as g; g.build()'`")
        spec = importlib.util.spec_from_file_location("cwg_torch", path)
        mod = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(mod)
        L = lib()
        mod.bind(*(ctypes.cast(f, ctypes.c_void_p).value for f in (
            L.cwg_conv1d_causal, L.cwg_conv1d_causal_step, L.cwg_ssm_scan, L.cwg_ssm_step,
            L.cwg_fp8_quantize, L.cwg_fp8_matmul)))
        _torch_ext = mod
    return _torch_ext


def conv1d_causal(x, w, bias, y, state, starts, slots=None, resume=None, flags: int = 0,
                  stream=None) -> None:
    """Causal convolution of packed prompts: x and y (tokens, channels), w (channels, width),
    bias (channels,) or None, state (lines, width - 1, channels) or None, starts (sequences + 1,)
    int32, slots (sequences,) int32 or None, resume (sequences,) uint8 or None.  `state` is
    updated in place.  flags: BF16, SILU or RELU."""
    st = (_torch_ext or _ext()).conv1d_causal(x, w, bias, y, state, starts, slots, resume, flags,
                                              stream)
    if st:
        _check(st, "cwg_conv1d_causal")


def conv1d_causal_step(x, w, bias, y, state, slots=None, flags: int = 0, stream=None) -> None:
    """One token of each sequence: x and y (sequences, channels), the rest as for
    conv1d_causal.  `state` is updated in place."""
    st = (_torch_ext or _ext()).conv1d_causal_step(x, w, bias, y, state, slots, flags, stream)
    if st:
        _check(st, "cwg_conv1d_causal_step")


def ssm_workspace_bytes(tokens: int, n_seq: int, channels: int, states: int) -> int:
    """Bytes that serve every scan of at most `tokens` tokens in at most `n_seq` sequences."""
    return int(lib().cwg_ssm_workspace_bytes(tokens, n_seq, channels, states))


def ssm_scan(u, dt, A, B, C, D, dt_bias, z, y, state, starts, slots=None, resume=None,
             workspace=None, flags: int = 0, stream=None) -> None:
    """Selective scan of packed prompts: u, dt, z (or None) and y (tokens, channels), A
    (channels, states), B and C (tokens, groups * states), D and dt_bias (channels,) or None,
    state (lines, channels, states) fp32 or None, starts, slots and resume as for
    conv1d_causal.  workspace: uint8, ssm_workspace_bytes(...) of them, or None (sequences are
    then never cut).  `state` is updated in place.  flags: BF16, SOFTPLUS."""
    st = (_torch_ext or _ext()).ssm_scan(u, dt, A, B, C, D, dt_bias, z, y, state, starts, slots,
                                         resume, workspace, flags, stream)
    if st:
        _check(st, "cwg_ssm_scan")


def ssm_step(u, dt, A, B, C, D, dt_bias, z, y, state, slots=None, flags: int = 0,
             stream=None) -> None:
    """One token of each sequence: rows are sequences, the rest as for ssm_scan.  `state` is
    updated in place."""
    st = (_torch_ext or _ext()).ssm_step(u, dt, A, B, C, D, dt_bias, z, y, state, slots, flags,
                                         stream)
    if st:
        _check(st, "cwg_ssm_step")


def fp8_quantize(x, q, scale, block_rows: int, flags: int = 0, stream=None) -> None:
    """e4m3 values q (rows, cols) and scales (ceil(rows / block_rows), ceil(cols / 128)) of x
    (rows, cols), per block_rows (1 or 128) x 128 elements.  flags: BF16."""
    st = (_torch_ext or _ext()).fp8_quantize(x, q, scale, block_rows, flags, stream)
    if st:
        _check(st, "cwg_fp8_quantize")


def fp8_matmul(a, a_scale, w, w_scale, bias, y, flags: int = 0, stream=None) -> None:
    """y (m, n) = a (m, k) w (n, k)^T + bias, a and w e4m3 with the scales that fp8_quantize
    gives them with block_rows 1 and 128; rows of a and w start on 16-byte boundaries.
    flags: BF16 (y), RELU."""
    st = (_torch_ext or _ext()).fp8_matmul(a, a_scale, w, w_scale, bias, y, flags, stream)
    if st:
        _check(st, "cwg_fp8_matmul")


# ---- host-pointer per-tile API ----------------------------------------------------
def _f32c(a) -> np.ndarray:
    return np.ascontiguousarray(a, dtype=np.float32)


def tiles_fused(tiles: np.ndarray, U: np.ndarray) -> np.ndarray:
    """Per-tile fused Winograd on the GPU: tiles (T, C_in, td, td), U (C_out, C_in, td, td)
    -> (T, C_out, td-2, td-2); td in {4, 6, 8}."""
    tiles = _f32c(tiles)
    U = _f32c(U)
    if tiles.ndim != 4 or U.ndim != 4:
        raise ValueError("tiles must be (T, C_in, td, td) and U (C_out, C_in, td, td)")
    nt, c_in, td, td2 = tiles.shape
    c_out = U.shape[0]
    if td != td2 or U.shape[1:] != (c_in, td, td):
        raise ValueError(f"shape mismatch: tiles {tiles.shape}, U {U.shape}")
    m = td - 2
    out = np.empty((nt, c_out, max(m, 0), max(m, 0)), np.float32)
    fp = ctypes.POINTER(ctypes.c_float)
    st = lib().cwg_tiles_fused(tiles.ctypes.data_as(fp), U.ctypes.data_as(fp),
                               out.ctypes.data_as(fp), nt, c_in, c_out, td)
    if st == EINVAL and td not in (4, 6, 8):
        raise ValueError(f"Unsupported tile dimension td={td}. Supported: [4, 6, 8]")
    _check(st, "cwg_tiles_fused")
    return out


def fused_winograd_f23(input_tile: np.ndarray, U: np.ndarray) -> np.ndarray:
    """The reference's C entry point (fused_winograd.c:103) called through ctypes:
    input (C_in, 4, 4), U (C_out, C_in, 4, 4) -> (C_out, 2, 2)."""
    inp = _f32c(input_tile)
    U = _f32c(U)
    c_in, c_out = inp.shape[0], U.shape[0]
    out = np.empty((c_out, 2, 2), np.float32)
    fp = ctypes.POINTER(ctypes.c_float)
    lib().fused_winograd_f23(inp.ctypes.data_as(fp), U.ctypes.data_as(fp),
                             out.ctypes.data_as(fp), c_in, c_out)
    _check(lib().cwg_last_status(), "fused_winograd_f23")
    return out
