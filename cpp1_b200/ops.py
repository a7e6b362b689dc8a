"""Tensor-level API over libsmm: each function takes torch CUDA tensors
(row-major fp32, contiguous; the state-space operators and the 4-bit product also
bf16 and strided rows), calls one C ABI entry point on the current
stream, and returns the output tensor.

Storage conventions follow the reference DSL (src/dsl/layout_functions.py):
packed upper / symmetric operands are the row-major upper triangle
(``torch.triu_indices`` order), diagonals are length-N vectors and Toeplitz
matrices are their 2N-1 generator with ``T[i][j] = g[(N-1) + (j-i)]``.
"""
from __future__ import annotations

import math
from typing import Optional

import torch

from . import _lib

_ws_cache = {}


def _stream_ptr(stream: Optional[torch.cuda.Stream]) -> Optional[int]:
    s = stream if stream is not None else torch.cuda.current_stream()
    return s.cuda_stream or None


def _ptr(t: torch.Tensor) -> int:
    return t.data_ptr()


def _check_f32(name: str, t: torch.Tensor, numel: Optional[int] = None) -> torch.Tensor:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor")
    if t.dtype != torch.float32:
        raise TypeError(f"{name} must be float32, got {t.dtype}")
    if not t.is_contiguous():
        t = t.contiguous()
    if numel is not None and t.numel() != numel:
        raise ValueError(f"{name} has {t.numel()} elements, expected {numel}")
    return t


def _mode(mode: str) -> int:
    try:
        return _lib.MODES[mode]
    except KeyError:
        raise ValueError(f"unknown mode {mode!r}; expected one of {sorted(_lib.MODES)}") from None


def workspace(nbytes: int, device: torch.device) -> Optional[torch.Tensor]:
    """A cached device buffer of at least nbytes (grown on demand)."""
    if nbytes <= 0:
        return None
    key = device.index if device.index is not None else torch.cuda.current_device()
    buf = _ws_cache.get(key)
    if buf is None or buf.numel() < nbytes:
        buf = torch.empty(nbytes, dtype=torch.uint8, device=device)
        _ws_cache[key] = buf
    return buf


def _ws_args(nbytes: int, device: torch.device):
    buf = workspace(nbytes, device)
    return (buf.data_ptr(), buf.numel()) if buf is not None else (None, 0)


def _out(out: Optional[torch.Tensor], shape, like: torch.Tensor) -> torch.Tensor:
    if out is None:
        return torch.empty(shape, dtype=torch.float32, device=like.device)
    out = _check_f32("out", out)
    if tuple(out.shape) != tuple(shape) and out.numel() != int(torch.tensor(shape).prod()):
        raise ValueError(f"out has shape {tuple(out.shape)}, expected {tuple(shape)}")
    return out


def diag_rows(d: torch.Tensor, B: torch.Tensor, out: Optional[torch.Tensor] = None, stream=None) -> torch.Tensor:
    """C = diag(d) @ B (row scale), bit-exact single fp32 multiply."""
    B = _check_f32("B", B)
    M, N = B.shape
    d = _check_f32("d", d, M)
    C = _out(out, (M, N), B)
    _lib.check(_lib.load().smm_diag_rows(_ptr(d), _ptr(B), _ptr(C), M, N, _stream_ptr(stream)), "smm_diag_rows")
    return C


def diag_cols(A: torch.Tensor, b: torch.Tensor, out: Optional[torch.Tensor] = None, stream=None) -> torch.Tensor:
    """C = A @ diag(b) (column scale)."""
    A = _check_f32("A", A)
    M, N = A.shape
    b = _check_f32("b", b, N)
    C = _out(out, (M, N), A)
    _lib.check(_lib.load().smm_diag_cols(_ptr(A), _ptr(b), _ptr(C), M, N, _stream_ptr(stream)), "smm_diag_cols")
    return C


def gemm(A: torch.Tensor, B: torch.Tensor, mode: str = "3xtf32", out: Optional[torch.Tensor] = None,
         stream=None) -> torch.Tensor:
    """C = A @ B."""
    A = _check_f32("A", A)
    B = _check_f32("B", B)
    M, K = A.shape
    K2, N = B.shape
    if K != K2:
        raise ValueError(f"inner dimensions differ: {K} vs {K2}")
    m = _mode(mode)
    L = _lib.load()
    ws, wsb = _ws_args(L.smm_gemm_workspace_size(M, N, K, m), A.device)
    C = _out(out, (M, N), A)
    _lib.check(L.smm_gemm(_ptr(A), _ptr(B), _ptr(C), M, N, K, m, ws, wsb, _stream_ptr(stream)), "smm_gemm")
    return C


def upper_left(U: torch.Tensor, B: torch.Tensor, packed: bool = True, mode: str = "3xtf32",
               out: Optional[torch.Tensor] = None, stream=None) -> torch.Tensor:
    """C = U @ B with U upper triangular, packed (N(N+1)/2) or dense N x N
    with exact zeros below the diagonal."""
    B = _check_f32("B", B)
    N, ncols = B.shape
    U = _check_f32("U", U, N * (N + 1) // 2 if packed else N * N)
    fmt = _lib.FMT_PACKED if packed else _lib.FMT_DENSE
    m = _mode(mode)
    L = _lib.load()
    ws, wsb = _ws_args(L.smm_upper_left_workspace_size(N, ncols, fmt, m), B.device)
    C = _out(out, (N, ncols), B)
    _lib.check(L.smm_upper_left(_ptr(U), fmt, _ptr(B), _ptr(C), N, ncols, m, ws, wsb, _stream_ptr(stream)),
               "smm_upper_left")
    return C


def toeplitz_left(g: torch.Tensor, B: torch.Tensor, mode: str = "3xtf32", out: Optional[torch.Tensor] = None,
                  stream=None) -> torch.Tensor:
    """C = T @ B, T the Toeplitz matrix of generator g (2N-1)."""
    B = _check_f32("B", B)
    N, ncols = B.shape
    g = _check_f32("g", g, 2 * N - 1)
    m = _mode(mode)
    L = _lib.load()
    ws, wsb = _ws_args(L.smm_toeplitz_left_workspace_size(N, ncols, m), B.device)
    C = _out(out, (N, ncols), B)
    _lib.check(L.smm_toeplitz_left(_ptr(g), _ptr(B), _ptr(C), N, ncols, m, ws, wsb, _stream_ptr(stream)),
               "smm_toeplitz_left")
    return C


def symm_left(S: torch.Tensor, B: torch.Tensor, mode: str = "3xtf32", out: Optional[torch.Tensor] = None,
              stream=None) -> torch.Tensor:
    """C = S @ B, S symmetric given packed upper."""
    B = _check_f32("B", B)
    N, ncols = B.shape
    S = _check_f32("S", S, N * (N + 1) // 2)
    m = _mode(mode)
    L = _lib.load()
    ws, wsb = _ws_args(L.smm_symm_left_workspace_size(N, ncols, m), B.device)
    C = _out(out, (N, ncols), B)
    _lib.check(L.smm_symm_left(_ptr(S), _ptr(B), _ptr(C), N, ncols, m, ws, wsb, _stream_ptr(stream)),
               "smm_symm_left")
    return C


def symm_sandwich(A: torch.Tensor, S: torch.Tensor, B: torch.Tensor, mode: str = "3xtf32",
                  out: Optional[torch.Tensor] = None, stream=None) -> torch.Tensor:
    """C = A @ S @ B, S symmetric given packed upper, all N x N."""
    A = _check_f32("A", A)
    N = A.shape[0]
    if tuple(A.shape) != (N, N):
        raise ValueError("A must be square")
    B = _check_f32("B", B, N * N)
    S = _check_f32("S", S, N * (N + 1) // 2)
    m = _mode(mode)
    L = _lib.load()
    ws, wsb = _ws_args(L.smm_symm_sandwich_workspace_size(N, m), A.device)
    C = _out(out, (N, N), A)
    _lib.check(L.smm_symm_sandwich(_ptr(A), _ptr(S), _ptr(B), _ptr(C), N, m, ws, wsb, _stream_ptr(stream)),
               "smm_symm_sandwich")
    return C


def _gen_x_struct(entry: str, A: torch.Tensor, X: torch.Tensor, mode: str, out, stream) -> torch.Tensor:
    A = _check_f32("A", A)
    M, N = A.shape
    X = _check_f32("packed operand", X, N * (N + 1) // 2)
    m = _mode(mode)
    L = _lib.load()
    ws, wsb = _ws_args(L.smm_gen_x_struct_workspace_size(M, N, m), A.device)
    C = _out(out, (M, N), A)
    _lib.check(getattr(L, entry)(_ptr(A), _ptr(X), _ptr(C), M, N, m, ws, wsb, _stream_ptr(stream)), entry)
    return C


def gen_x_upper(A: torch.Tensor, U: torch.Tensor, mode: str = "3xtf32", out: Optional[torch.Tensor] = None,
                stream=None) -> torch.Tensor:
    """C = A @ U, U upper triangular given packed (right side)."""
    return _gen_x_struct("smm_gen_x_upper", A, U, mode, out, stream)


def gen_x_symm(A: torch.Tensor, S: torch.Tensor, mode: str = "3xtf32", out: Optional[torch.Tensor] = None,
               stream=None) -> torch.Tensor:
    """C = A @ S, S symmetric given packed upper (right side)."""
    return _gen_x_struct("smm_gen_x_symm", A, S, mode, out, stream)


def gen_x_lower(A: torch.Tensor, Lp: torch.Tensor, mode: str = "3xtf32", out: Optional[torch.Tensor] = None,
                stream=None) -> torch.Tensor:
    """C = A @ L with L lower triangular given packed lower (i(i+1)/2 + j)."""
    return _gen_x_struct("smm_gen_x_lower", A, Lp, mode, out, stream)


def gen_x_toeplitz(A: torch.Tensor, g: torch.Tensor, N: Optional[int] = None, mode: str = "3xtf32",
                   out: Optional[torch.Tensor] = None, stream=None) -> torch.Tensor:
    """C = A @ T with T (K x N) the Toeplitz matrix of generator g (K + N - 1),
    T[k][n] = g[(K-1) + (n-k)]; N defaults to K (square T, 2K - 1 generator)."""
    A = _check_f32("A", A)
    M, K = A.shape
    N = K if N is None else N
    g = _check_f32("g", g, K + N - 1)
    m = _mode(mode)
    L = _lib.load()
    ws, wsb = _ws_args(L.smm_gen_x_toeplitz_workspace_size(M, N, K, m), A.device)
    C = _out(out, (M, N), A)
    _lib.check(L.smm_gen_x_toeplitz(_ptr(A), _ptr(g), _ptr(C), M, N, K, m, ws, wsb, _stream_ptr(stream)),
               "smm_gen_x_toeplitz")
    return C


def _packed_order(name: str, t: torch.Tensor) -> int:
    p = t.numel()
    N = int((-1 + (1 + 8 * p) ** 0.5) // 2)
    if N * (N + 1) // 2 != p:
        raise ValueError(f"{name} has {p} elements, not a packed triangle")
    return N


def lower_left(Lp: torch.Tensor, B: torch.Tensor, mode: str = "3xtf32", out: Optional[torch.Tensor] = None,
               stream=None) -> torch.Tensor:
    """C = L @ B with L lower triangular given packed lower."""
    B = _check_f32("B", B)
    N, ncols = B.shape
    Lp = _check_f32("L", Lp, N * (N + 1) // 2)
    m = _mode(mode)
    L = _lib.load()
    ws, wsb = _ws_args(L.smm_lower_left_workspace_size(N, ncols, m), B.device)
    C = _out(out, (N, ncols), B)
    _lib.check(L.smm_lower_left(_ptr(Lp), _ptr(B), _ptr(C), N, ncols, m, ws, wsb, _stream_ptr(stream)),
               "smm_lower_left")
    return C


def lower_x_lower(L1: torch.Tensor, L2: torch.Tensor, mode: str = "3xtf32", out: Optional[torch.Tensor] = None,
                  stream=None) -> torch.Tensor:
    """C = L1 @ L2, both lower triangular given packed lower."""
    L1 = _check_f32("L1", L1)
    N = _packed_order("L1", L1)
    L2 = _check_f32("L2", L2, L1.numel())
    C = _out(out, (N, N), L1)
    m = _mode(mode)
    L = _lib.load()
    ws, wsb = _ws_args(L.smm_lower_x_lower_workspace_size(N, m), L1.device)
    _lib.check(L.smm_lower_x_lower_ws(_ptr(L1), _ptr(L2), _ptr(C), N, m, ws, wsb, _stream_ptr(stream)),
               "smm_lower_x_lower")
    return C


def symm_x_symm(S1: torch.Tensor, S2: torch.Tensor, mode: str = "3xtf32", out: Optional[torch.Tensor] = None,
                stream=None) -> torch.Tensor:
    """C = S1 @ S2, both symmetric given packed upper."""
    S1 = _check_f32("S1", S1)
    p = S1.numel()
    N = int((-1 + (1 + 8 * p) ** 0.5) // 2)
    if N * (N + 1) // 2 != p:
        raise ValueError(f"S1 has {p} elements, not a packed triangle")
    S2 = _check_f32("S2", S2, p)
    C = _out(out, (N, N), S1)
    m = _mode(mode)
    L = _lib.load()
    ws, wsb = _ws_args(L.smm_symm_x_symm_workspace_size(N, m), S1.device)
    _lib.check(L.smm_symm_x_symm_ws(_ptr(S1), _ptr(S2), _ptr(C), N, m, ws, wsb, _stream_ptr(stream)),
               "smm_symm_x_symm")
    return C


# ---------------------------------------------------------------- elementwise / converters
def _struct(fmt: str) -> int:
    try:
        return _lib.STRUCTS[fmt]
    except KeyError:
        raise ValueError(f"unknown structure {fmt!r}; expected one of {sorted(_lib.STRUCTS)}") from None


def struct_numel(fmt: str, N: int) -> int:
    """Storage size of an order-N structured matrix."""
    _struct(fmt)
    return {"upper": N * (N + 1) // 2, "lower": N * (N + 1) // 2, "symm": N * (N + 1) // 2, "diag": N,
            "toeplitz": max(2 * N - 1, 0)}[fmt]


def add(A: torch.Tensor, B: torch.Tensor, out: Optional[torch.Tensor] = None, stream=None) -> torch.Tensor:
    """C = A + B elementwise over the storage of two operands of the same
    structure (flat, any shape with equal element counts)."""
    A = _check_f32("A", A)
    B = _check_f32("B", B, A.numel())
    C = _out(out, tuple(A.shape), A)
    _lib.check(_lib.load().smm_add(_ptr(A), _ptr(B), _ptr(C), A.numel(), _stream_ptr(stream)), "smm_add")
    return C


def add_struct(A: torch.Tensor, S: torch.Tensor, fmt: str, out: Optional[torch.Tensor] = None,
               stream=None) -> torch.Tensor:
    """C = A + S with A dense N x N and S structured (fmt: upper, lower, symm,
    diag, toeplitz) in its packed storage."""
    A = _check_f32("A", A)
    N = int(round(A.numel() ** 0.5))
    if N * N != A.numel():
        raise ValueError(f"A has {A.numel()} elements, not a square matrix")
    S = _check_f32("S", S, struct_numel(fmt, N))
    C = _out(out, (N, N), A)
    _lib.check(_lib.load().smm_add_struct(_ptr(A), _ptr(S), _struct(fmt), _ptr(C), N, _stream_ptr(stream)),
               "smm_add_struct")
    return C


def unpack(S: torch.Tensor, fmt: str, N: int, out: Optional[torch.Tensor] = None, stream=None) -> torch.Tensor:
    """Dense N x N matrix of the structured storage S."""
    S = _check_f32("S", S, struct_numel(fmt, N))
    D = _out(out, (N, N), S)
    _lib.check(_lib.load().smm_unpack(_ptr(S), _struct(fmt), _ptr(D), N, _stream_ptr(stream)), "smm_unpack")
    return D


def pack(D: torch.Tensor, fmt: str, out: Optional[torch.Tensor] = None, stream=None) -> torch.Tensor:
    """Packed upper (fmt upper or symm) or lower triangle of the dense square D."""
    D = _check_f32("D", D)
    N = int(round(D.numel() ** 0.5))
    if N * N != D.numel():
        raise ValueError(f"D has {D.numel()} elements, not a square matrix")
    P = _out(out, (N * (N + 1) // 2,), D)
    _lib.check(_lib.load().smm_pack(_ptr(D), _struct(fmt), _ptr(P), N, _stream_ptr(stream)), "smm_pack")
    return P


def toeplitz_compact(T: torch.Tensor, out: Optional[torch.Tensor] = None, stream=None) -> torch.Tensor:
    """Generator (rows + cols - 1) of the Toeplitz matrix T (2-D)."""
    if T.dim() != 2:
        raise ValueError("T must be 2-D")
    T = _check_f32("T", T)
    rows, cols = T.shape
    g = _out(out, (max(rows + cols - 1, 0),), T)
    _lib.check(_lib.load().smm_toeplitz_compact(_ptr(T), _ptr(g), rows, cols, _stream_ptr(stream)),
               "smm_toeplitz_compact")
    return g


def device_status(stream=None) -> None:
    """Raise SmmError(SMM_ERR_DEVICE_TIMEOUT) if a kernel gave up a bounded wait."""
    _lib.check(_lib.load().smm_device_status(_stream_ptr(stream)), "smm_device_status")


def launch_count() -> int:
    return int(_lib.load().smm_launch_count())


# ---------------------------------------------------------------- state-space blocks
_DTYPES = {torch.float32: _lib.DTYPE_F32, torch.bfloat16: _lib.DTYPE_BF16}
_ACTS = {None: 0, "silu": 1}


def _check_seq(name: str, t: torch.Tensor, like: torch.Tensor, dtype, shape) -> torch.Tensor:
    """A tensor of this type and shape on like's device."""
    try:
        if t.dtype is dtype and t.shape == shape and t.device == like.device:
            return t
    except AttributeError:
        pass
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if t.device != like.device:
        raise ValueError(f"{name} is on {t.device}, expected {like.device}")
    if t.dtype != dtype:
        raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
    raise ValueError(f"{name} has shape {tuple(t.shape)}, expected {tuple(shape)}")


def _dims(name: str, t: torch.Tensor, dims: int):
    """The shape of a tensor of so many dimensions."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    shape = t.shape
    if len(shape) != dims:
        raise ValueError(f"{name} has shape {tuple(shape)}, expected {dims} dimensions")
    if max(shape) > 0x7FFFFFFF:
        raise ValueError(f"{name} has shape {tuple(shape)}, a dimension beyond 31 bits")
    return shape


def _x_dtype(x: torch.Tensor) -> int:
    try:
        return _DTYPES[x.dtype]
    except KeyError:
        raise TypeError(f"x must be float32 or bfloat16, got {x.dtype}") from None


def _row_stride(t: torch.Tensor, width: int) -> Optional[int]:
    """The distance of t's rows (its first dimension), or None where the elements of
    a row are not contiguous or rows overlap.  Dimensions of size one may have any stride."""
    if t.is_contiguous():
        return width
    shape, stride, w = t.shape, t.stride(), 1
    for i in range(len(shape) - 1, 0, -1):
        if shape[i] != 1 and stride[i] != w:
            return None
        w *= shape[i]
    if shape[0] <= 1:
        return width
    return stride[0] if stride[0] >= width else None


def _rows(t: torch.Tensor, width: int):
    """t with contiguous rows (copied if it is laid out otherwise), and the row stride."""
    ld = _row_stride(t, width)
    return (t, ld) if ld is not None else (t.contiguous(), width)


def _seq_out(out: Optional[torch.Tensor], x: torch.Tensor, shape, width: int):
    if out is None:
        return x.new_empty(shape), width
    _check_seq("out", out, x, x.dtype, shape)
    ld = _row_stride(out, width)
    if ld is None:
        raise ValueError("out must have contiguous rows that do not overlap")
    return out, ld


def _states(x, dtype, entry, state, state_out):
    """The checked pair of state tensors (in place without state_out) and their number of entries."""
    n = None
    for name, t in (("state", state), ("state_out", state_out)):
        if t is not None:
            m = _dims(name, t, 1 + len(entry))[0]
            _check_seq(name, t, x, dtype, (m, *entry))
            if not t.is_contiguous():
                raise ValueError(f"{name} must be contiguous")
            if n is not None and n != m:
                raise ValueError(f"state has {n} entries, state_out {m}")
            n = m
    return state, state if state_out is None else state_out, n or 0


def _check_index(name: str, t: Optional[torch.Tensor], like: torch.Tensor, n: Optional[int]) -> None:
    if t is not None:
        _check_seq(name, t, like, torch.int32, _dims(name, t, 1) if n is None else (n,))


def _opt(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


def _vec(t: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    return t if t is None or t.is_contiguous() else t.contiguous()


# A small call's time is the host's: the stream's handle without a Stream object.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream",
                      lambda index: torch.cuda.current_stream(index).cuda_stream)


def _on(x: torch.Tensor, stream: Optional[torch.cuda.Stream], call):
    """call(stream pointer) with x's device current.  Whatever call allocates and copies belongs
    to the stream that its kernels run on, so nothing is copied outside of it."""
    if not x.is_cuda:
        raise ValueError("x must be a CUDA tensor")
    index = x.device.index
    if stream is not None:
        if stream.device != x.device:
            raise ValueError(f"stream is on {stream.device}, x on {x.device}")
        with torch.cuda.stream(stream):
            return call(stream.cuda_stream or None)
    if index == torch.cuda.current_device():
        return call(_raw_stream(index) or None)
    with torch.cuda.device(index):
        return call(_raw_stream(index) or None)


def _sequences(offsets, x) -> int:
    if offsets is None:
        return 1
    _check_index("offsets", offsets, x, None)
    if offsets.shape[0] < 1:
        raise ValueError("offsets must have at least one element")
    return offsets.shape[0] - 1


def _conv_args(x, weight, bias, activation):
    """Checks shared by the convolution and its step; returns (rows, channels, width, dtype, act)."""
    rows, channels = _dims("x", x, 2)
    ty = _x_dtype(x)
    width = _dims("weight", weight, 2)[1]
    _check_seq("weight", weight, x, x.dtype, (channels, width))
    if not 2 <= width <= 8:
        raise ValueError(f"weight has {width} taps, expected 2 to 8")
    if bias is not None:
        _check_seq("bias", bias, x, x.dtype, (channels,))
    try:
        return rows, channels, width, ty, _ACTS[activation]
    except (KeyError, TypeError):
        raise ValueError(f"unknown activation {activation!r}; expected None or 'silu'") from None


def causal_conv(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, *,
                offsets: Optional[torch.Tensor] = None, state: Optional[torch.Tensor] = None,
                state_out: Optional[torch.Tensor] = None, slots: Optional[torch.Tensor] = None,
                activation: Optional[str] = "silu", out: Optional[torch.Tensor] = None, stream=None) -> torch.Tensor:
    """y[t, c] = act(bias[c] + sum_j weight[c, j] x[t-W+1+j, c]): a banded
    lower-triangular Toeplitz matrix per channel, over packed sequences.

    x (tokens, channels) float32 or bfloat16; weight (channels, W), W in 2..8,
    and bias (channels) of the same type.  Sequence s is the rows
    [offsets[s], offsets[s+1]) (int32, not decreasing; None: all rows are one sequence).  state (entries,
    channels, W-1), of x's type, holds the rows before each sequence, oldest first
    (None: zeros), and state_out receives the rows that each one ends with (None:
    state is updated in place).  Sequence s uses entry slots[s] (int32; None: s;
    negative: no state); no two may share one.  Rows outside every sequence are
    left as they are in `out`, and have no defined values without it.  `out` may be columns of
    the matrix whose other columns are inputs."""
    tokens, channels, width, ty, act = _conv_args(x, weight, bias, activation)
    state, state_out, entries = _states(x, x.dtype, (channels, width - 1), state, state_out)
    nseq = _sequences(offsets, x)
    _check_index("slots", slots, x, nseq)

    def call(st):
        xr, ldx = _rows(x, channels)
        w, b, off, sl = _vec(weight), _vec(bias), _vec(offsets), _vec(slots)
        y, ldy = _seq_out(out, x, (tokens, channels), channels)
        _lib.check(_lib.load().smm_causal_conv(
            xr.data_ptr(), w.data_ptr(), _opt(b), _opt(off), _opt(state), _opt(state_out), _opt(sl),
            y.data_ptr(), tokens, channels, width, nseq, entries, ldx, ldy, ty, act, st), "smm_causal_conv")
        return y
    return _on(x, stream, call)


def causal_conv_step(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, *,
                     state: torch.Tensor, state_out: Optional[torch.Tensor] = None,
                     slots: Optional[torch.Tensor] = None, activation: Optional[str] = "silu",
                     out: Optional[torch.Tensor] = None, stream=None) -> torch.Tensor:
    """causal_conv for one new token of each sequence: row b of x (batch,
    channels) continues the state at entry slots[b] (None: b), which is updated in
    place unless state_out is given.  A row with a negative slot starts from zero and leaves no state."""
    batch, channels, width, ty, act = _conv_args(x, weight, bias, activation)
    if state is None:
        raise TypeError("state must be a torch.Tensor")
    state, state_out, entries = _states(x, x.dtype, (channels, width - 1), state, state_out)
    _check_index("slots", slots, x, batch)

    def call(st):
        xr, ldx = _rows(x, channels)
        w, b, sl = _vec(weight), _vec(bias), _vec(slots)
        y, ldy = _seq_out(out, x, (batch, channels), channels)
        _lib.check(_lib.load().smm_causal_conv_step(
            xr.data_ptr(), w.data_ptr(), _opt(b), state.data_ptr(), state_out.data_ptr(), _opt(sl), y.data_ptr(),
            batch, channels, width, entries, ldx, ldy, ty, act, st), "smm_causal_conv_step")
        return y
    return _on(x, stream, call)


def _scan_args(x, dt, A, B, C, D, z, dt_bias):
    """Checks shared by the scan and the step; returns (rows, heads, dim, groups, state_dim, dtype, dt's dtype)."""
    t, heads, dim = _dims("x", x, 3)
    ty = _x_dtype(x)
    if not isinstance(dt, torch.Tensor):
        raise TypeError("dt must be a torch.Tensor")
    if dt.dtype is not x.dtype and dt.dtype is not torch.float32:
        raise TypeError(f"dt must be {x.dtype} or float32, got {dt.dtype}")
    _check_seq("dt", dt, x, dt.dtype, (t, heads))
    _check_seq("A", A, x, torch.float32, (heads,))
    _, groups, n = shape = _dims("B", B, 3)
    _check_seq("B", B, x, x.dtype, (t, groups, n))
    _check_seq("C", C, x, x.dtype, shape)
    if not (1 <= dim <= 256 and 1 <= n <= 256):
        raise ValueError(f"head dim {dim} and state dim {n} must be 1 to 256")
    if groups < 1 or heads % groups:
        raise ValueError(f"{heads} heads do not divide into {groups} groups")
    if D is not None:
        _check_seq("D", D, x, torch.float32, (heads,))
    if dt_bias is not None:
        _check_seq("dt_bias", dt_bias, x, torch.float32, (heads,))
    if z is not None:
        _check_seq("z", z, x, x.dtype, (t, heads, dim))
    return t, heads, dim, groups, n, ty, _DTYPES[dt.dtype]


def selective_scan(x: torch.Tensor, dt: torch.Tensor, A: torch.Tensor, B: torch.Tensor, C: torch.Tensor, *,
                   D: Optional[torch.Tensor] = None, z: Optional[torch.Tensor] = None,
                   dt_bias: Optional[torch.Tensor] = None, dt_softplus: bool = False,
                   offsets: Optional[torch.Tensor] = None, state: Optional[torch.Tensor] = None,
                   state_out: Optional[torch.Tensor] = None, slots: Optional[torch.Tensor] = None,
                   out: Optional[torch.Tensor] = None, stream=None) -> torch.Tensor:
    """Selective state space scan over packed sequences: per head a
    lower-triangular semiseparable matrix times x.  With d = dt + dt_bias (through
    softplus if dt_softplus) and g the head's group,

        S_t = exp(d_t A_h) S_{t-1} + d_t x_t (outer) B_t,g
        y_t = (S_t C_t,g + D_h x_t) * silu(z_t)

    x, z, y (tokens, heads, dim) and B, C (tokens, groups, state_dim) float32 or
    bfloat16, dt (tokens, heads) of the same type or float32; A (one decay rate a head), D, dt_bias
    (heads) float32.  dim and state_dim are 1 to 256.  Rows may be strided (x, B and
    C columns of one matrix).  Sums, decays and states are float32; longer bfloat16 prompts go through
    the tensor cores, where scores and states enter products as two bfloat16 terms (2^-17 relative).

    offsets, slots, out, state (entries, heads, dim, state_dim; float32) and state_out are as in causal_conv.
    What depends on a non-finite input is not finite (NaN at times where an infinity would do); the
    tokens before it do not depend on it."""
    tokens, heads, dim, groups, n, ty, dty = _scan_args(x, dt, A, B, C, D, z, dt_bias)
    state, state_out, entries = _states(x, torch.float32, (heads, dim, n), state, state_out)
    nseq = _sequences(offsets, x)
    _check_index("slots", slots, x, nseq)

    def call(st):
        L = _lib.load()
        wx, wb = heads * dim, groups * n
        (xr, ldx), (dr, ldd), (br, ldb), (cr, ldc) = _rows(x, wx), _rows(dt, heads), _rows(B, wb), _rows(C, wb)
        zr, ldz = (None, 0) if z is None else _rows(z, wx)
        a, dd, db, off, sl = _vec(A), _vec(D), _vec(dt_bias), _vec(offsets), _vec(slots)
        y, ldy = _seq_out(out, x, (tokens, heads, dim), wx)
        nws = L.smm_selective_scan_workspace_size(tokens, nseq, heads, dim, groups, n, ty)
        # of this call alone: streams and captured graphs share nothing
        ws = torch.empty(nws, dtype=torch.uint8, device=x.device) if nws else None
        _lib.check(L.smm_selective_scan(
            xr.data_ptr(), dr.data_ptr(), a.data_ptr(), br.data_ptr(), cr.data_ptr(), _opt(dd), _opt(zr), _opt(db),
            _opt(off), _opt(state), _opt(state_out), _opt(sl), y.data_ptr(), tokens, nseq, entries, heads, dim,
            groups, n, ldx, ldd, ldb, ldc, ldz, ldy, ty, dty, 1 if dt_softplus else 0, _opt(ws), nws, st),
            "smm_selective_scan")
        return y
    return _on(x, stream, call)


def selective_step(x: torch.Tensor, dt: torch.Tensor, A: torch.Tensor, B: torch.Tensor, C: torch.Tensor, *,
                   state: torch.Tensor, D: Optional[torch.Tensor] = None, z: Optional[torch.Tensor] = None,
                   dt_bias: Optional[torch.Tensor] = None, dt_softplus: bool = False,
                   state_out: Optional[torch.Tensor] = None, slots: Optional[torch.Tensor] = None,
                   out: Optional[torch.Tensor] = None, stream=None) -> torch.Tensor:
    """selective_scan for one new token of each sequence: row b of x (batch,
    heads, dim) continues the state at entry slots[b] (None: b), which is updated
    in place unless state_out is given.  A row with a negative slot starts from
    zero and leaves no state."""
    batch, heads, dim, groups, n, ty, dty = _scan_args(x, dt, A, B, C, D, z, dt_bias)
    if state is None:
        raise TypeError("state must be a torch.Tensor")
    state, state_out, entries = _states(x, torch.float32, (heads, dim, n), state, state_out)
    _check_index("slots", slots, x, batch)

    def call(st):
        wx, wb = heads * dim, groups * n
        (xr, ldx), (dr, ldd), (br, ldb), (cr, ldc) = _rows(x, wx), _rows(dt, heads), _rows(B, wb), _rows(C, wb)
        zr, ldz = (None, 0) if z is None else _rows(z, wx)
        a, dd, db, sl = _vec(A), _vec(D), _vec(dt_bias), _vec(slots)
        y, ldy = _seq_out(out, x, (batch, heads, dim), wx)
        _lib.check(_lib.load().smm_selective_step(
            xr.data_ptr(), dr.data_ptr(), a.data_ptr(), br.data_ptr(), cr.data_ptr(), _opt(dd), _opt(zr), _opt(db),
            state.data_ptr(), state_out.data_ptr(), _opt(sl), y.data_ptr(), batch, entries, heads, dim, groups, n,
            ldx, ldd, ldb, ldc, ldz, ldy, ty, dty, 1 if dt_softplus else 0, st), "smm_selective_step")
        return y
    return _on(x, stream, call)


def q4_matvec(q: torch.Tensor, scales: torch.Tensor, x: torch.Tensor, zeros: Optional[torch.Tensor] = None, *,
              out: Optional[torch.Tensor] = None, stream=None) -> torch.Tensor:
    """y = x W^T for a few rows x (batch, cols) and W held in 4 bits:
    W[r, k] = (code[r, k] - zero[r, k // group]) * scales[r, k // group].

    q (rows, cols/2) uint8 holds code 2i of a row in the low half of byte i; scales
    (rows, cols/group), of x's type or float32, and zeros (same shape, uint8, 0..127; None:
    8 everywhere) give the group, a multiple of 32.  x float32 or bfloat16; products are
    exact and sums float32 in both (over x times codes, before the scale).  Returns (batch, rows).

    For a few rows: at most 65535, and q is read again for every 8 or 16 of them."""
    batch, cols = _dims("x", x, 2)
    ty = _x_dtype(x)
    if cols % 2:
        raise ValueError(f"x has an odd number of columns, {cols}")
    rows = _dims("q", q, 2)[0]
    _check_seq("q", q, x, torch.uint8, (rows, cols // 2))
    _, groups = shape = _dims("scales", scales, 2)
    if scales.dtype is not x.dtype and scales.dtype is not torch.float32:
        raise TypeError(f"scales must be {x.dtype} or float32, got {scales.dtype}")
    _check_seq("scales", scales, x, scales.dtype, (rows, groups))
    if groups < 1 or cols % groups or (cols // groups) % 32 or cols == 0:
        raise ValueError(f"{cols} columns do not divide into {groups} groups of a multiple of 32")
    if zeros is not None:
        _check_seq("zeros", zeros, x, torch.uint8, shape)

    def call(st):
        xr, ldx = _rows(x, cols)
        if xr.data_ptr() % 16 or (batch > 1 and ldx * xr.element_size() % 16):
            xr, ldx = xr.clone(memory_format=torch.contiguous_format), cols
        qc, sc, zc = _vec(q), _vec(scales), _vec(zeros)
        if qc.data_ptr() % 16:
            qc = qc.clone()
        y, ldy = _seq_out(out, x, (batch, rows), rows)
        _lib.check(_lib.load().smm_q4_matvec(
            qc.data_ptr(), sc.data_ptr(), _opt(zc), xr.data_ptr(), y.data_ptr(), batch, rows, cols, cols // groups, ldx,
            ldy, ty, _DTYPES[scales.dtype], st), "smm_q4_matvec")
        return y
    return _on(x, stream, call)


# ---------------------------------------------------------------- host buffers
def _check_host(name: str, t: torch.Tensor, numel: Optional[int] = None) -> torch.Tensor:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if t.is_cuda:
        raise ValueError(f"{name} must be a host (CPU) tensor")
    if t.dtype != torch.float32:
        raise TypeError(f"{name} must be float32, got {t.dtype}")
    if not t.is_contiguous():
        t = t.contiguous()
    if numel is not None and t.numel() != numel:
        raise ValueError(f"{name} has {t.numel()} elements, expected {numel}")
    return t


def host_product(op: str, *inputs: torch.Tensor, mode: str = "3xtf32",
                 out: Optional[torch.Tensor] = None, toeplitz_cols: Optional[int] = None) -> torch.Tensor:
    """C = the product ``op`` of HOST tensors through the smm_*_host entry
    points: the left operand(s) cross PCIe once, B streams through in column
    chunks whose copies overlap the products (pinned tensors overlap; pageable
    ones work synchronously).  Synchronous; C is a host tensor (pinned unless
    ``out`` is given).

    op: "gemm" (A, B), "upper" (U_packed, B), "symm" (S_packed, B),
    "toeplitz" (g, B), "sandwich" (A, S_packed, B); the right-side
    orientation of the reference's CPU drivers: "gen_x_upper" (A, U_packed),
    "gen_x_symm" (A, S_packed), "gen_x_toeplitz" (A, g; T square unless
    ``toeplitz_cols`` is given), "diag_cols" (A, b)."""
    arity = {"gemm": 2, "upper": 2, "symm": 2, "toeplitz": 2, "sandwich": 3, "gen_x_upper": 2, "gen_x_symm": 2,
             "gen_x_toeplitz": 2, "diag_cols": 2}
    if op not in arity:
        raise ValueError(f"unknown host product {op!r}; expected one of {sorted(arity)}")
    if len(inputs) != arity[op]:
        raise ValueError(f"host product {op!r} takes {arity[op]} inputs, got {len(inputs)}")
    m = _mode(mode)
    L = _lib.load()
    if op == "gemm":
        A, B = _check_host("A", inputs[0]), _check_host("B", inputs[1])
        (M, K), (K2, N) = A.shape, B.shape
        if K != K2:
            raise ValueError(f"inner dimensions differ: {K} vs {K2}")
        shape = (M, N)
        size = L.smm_gemm_host_workspace_size(M, N, K, m)
        call = lambda C, ws, wsb: L.smm_gemm_host(A.data_ptr(), B.data_ptr(), C.data_ptr(), M, N, K, m, ws, wsb)
    elif op in ("upper", "symm", "toeplitz"):
        B = _check_host("B", inputs[1])
        N, ncols = B.shape
        X = _check_host("left operand", inputs[0], 2 * N - 1 if op == "toeplitz" else N * (N + 1) // 2)
        shape = (N, ncols)
        size = getattr(L, f"smm_{op}_left_host_workspace_size")(N, ncols, m)
        fn = getattr(L, f"smm_{op}_left_host")
        call = lambda C, ws, wsb: fn(X.data_ptr(), B.data_ptr(), C.data_ptr(), N, ncols, m, ws, wsb)
    elif op == "sandwich":
        A = _check_host("A", inputs[0])
        N = A.shape[0]
        if tuple(A.shape) != (N, N):
            raise ValueError("A must be square")
        S = _check_host("S", inputs[1], N * (N + 1) // 2)
        B = _check_host("B", inputs[2], N * N)
        shape = (N, N)
        size = L.smm_symm_sandwich_host_workspace_size(N, m)
        call = lambda C, ws, wsb: L.smm_symm_sandwich_host(A.data_ptr(), S.data_ptr(), B.data_ptr(), C.data_ptr(),
                                                           N, m, ws, wsb)
    elif op in ("gen_x_upper", "gen_x_symm"):
        A = _check_host("A", inputs[0])
        M, N = A.shape
        X = _check_host("right operand", inputs[1], N * (N + 1) // 2)
        shape = (M, N)
        size = getattr(L, f"smm_{op}_host_workspace_size")(M, N, m)
        fn = getattr(L, f"smm_{op}_host")
        call = lambda C, ws, wsb: fn(A.data_ptr(), X.data_ptr(), C.data_ptr(), M, N, m, ws, wsb)
    elif op == "gen_x_toeplitz":
        A = _check_host("A", inputs[0])
        M, K = A.shape
        N = K if toeplitz_cols is None else toeplitz_cols
        g = _check_host("g", inputs[1], K + N - 1)
        shape = (M, N)
        size = L.smm_gen_x_toeplitz_host_workspace_size(M, N, K, m)
        call = lambda C, ws, wsb: L.smm_gen_x_toeplitz_host(A.data_ptr(), g.data_ptr(), C.data_ptr(), M, N, K, m,
                                                            ws, wsb)
    elif op == "diag_cols":
        A = _check_host("A", inputs[0])
        M, N = A.shape
        b = _check_host("b", inputs[1], N)
        shape = (M, N)
        size = L.smm_diag_cols_host_workspace_size(M, N)
        call = lambda C, ws, wsb: L.smm_diag_cols_host(A.data_ptr(), b.data_ptr(), C.data_ptr(), M, N, ws, wsb)
    if out is None:
        C = torch.empty(shape, dtype=torch.float32, pin_memory=True)
    else:
        C = _check_host("out", out, shape[0] * shape[1])
    ws, wsb = _ws_args(size, torch.device("cuda", torch.cuda.current_device()))
    # the entry points run on internal streams: finish work that may still
    # use the shared workspace
    torch.cuda.current_stream().synchronize()
    _lib.check(call(C, ws, wsb), f"host product {op}")
    return C
