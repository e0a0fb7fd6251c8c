"""Host layer of the expert-layer operators: FP8 products grouped by expert, their gradients, the row quantiser that makes
their operands, and products of 4-bit weights with a few vectors.

Layouts and formats are those of the dense operator (GEMM/include/gemm.cuh:12-55): operands row-major, ``b`` as rows of
the contraction index.  The reference has one weight matrix per product and no weights below eight bits, so these
operators have no counterpart there.  Everything is checked here before the call (the C ABI sees only pointers); calls
are enqueued on the current stream of the tensors' device.  Outputs must not share memory with inputs.
"""
from __future__ import annotations

import ctypes

import torch

from . import _cabi
from ._cabi import E4M3, E5M2, KERNEL_AUTO, Options

F8 = {torch.float8_e4m3fn: E4M3, torch.float8_e5m2: E5M2}
OUT = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2, torch.float8_e4m3fn: 3, torch.float8_e5m2: 4}
HALF = {torch.bfloat16: 1, torch.float16: 2}
WIDE = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
F32, INT32, U8 = (torch.float32,), (torch.int32,), (torch.uint8,)
_EPILOGUE_BYTES, _OPTIONS_BYTES = ctypes.sizeof(_cabi.EpilogueDesc), ctypes.sizeof(Options)
ACTIVATIONS = {"none": 0, "relu": 1, "gelu": 2, "gelu_tanh": 3}


def _matrix(name: str, t: torch.Tensor, dtypes, shape) -> int:
    """Checks type, shape and layout of a matrix (or of one per expert) and returns its row pitch in elements."""
    if t.dtype not in dtypes:
        raise TypeError(f"{name} has type {t.dtype}, expected one of {', '.join(str(d) for d in dtypes)}")
    if t.shape != shape:
        raise ValueError(f"{name} must be {list(shape)}, got {list(t.shape)}")
    cols, rows = shape[-1], shape[-2]
    if t.is_contiguous():
        return cols
    if cols > 1 and t.stride(-1) != 1:
        raise ValueError(f"{name}: the last dimension must be contiguous, got strides {t.stride()}")
    pitch = t.stride(-2) if rows > 1 else cols
    if pitch < cols:
        raise ValueError(f"{name}: rows overlap (pitch {pitch}, {cols} columns)")
    if len(shape) == 3 and shape[0] > 1 and t.stride(0) < (rows - 1) * pitch + cols:
        raise ValueError(f"{name}: matrices overlap (pitch {t.stride(0)})")
    return pitch


def _stride(t: torch.Tensor, pitch: int) -> int:
    return t.stride(0) if t.shape[0] > 1 else t.shape[1] * pitch


def _vector(name: str, t: torch.Tensor, dtypes, shape) -> None:
    if t.dtype not in dtypes or t.shape != shape or not t.is_contiguous():
        raise TypeError(f"{name} must be contiguous {list(shape)} of {', '.join(str(d) for d in dtypes)}, got {t.dtype} {list(t.shape)}")


def _device(first: torch.Tensor, *others) -> torch.device:
    device = first.device
    if device.type != "cuda":
        raise ValueError("the operators take CUDA tensors (device pointers)")
    for t in others:
        if t is not None and t.device != device:
            raise ValueError(f"all tensors must live on one device, got {device} and {t.device}")
    return device


def _call(device: torch.device, what: str, function, *args) -> None:
    """Enqueues the call on the device's current stream, with that device current."""
    stream = torch.cuda.current_stream(device).cuda_stream
    if torch.cuda.current_device() == device.index:
        code = function(*args, stream)
    else:
        with torch.cuda.device(device):
            code = function(*args, stream)
    if code:
        _cabi.check(code, what)


def quantize_rows(x: torch.Tensor, q: torch.Tensor, scale: torch.Tensor, *, rows: torch.Tensor | None = None):
    """Rows of bfloat16 / float16 to FP8 rows ``q`` with one float32 ``scale`` each, so that q * scale is the row again.

    scale = m / top with m the largest finite magnitude of the row (at least 2^-80) and top = 448 (e4m3) or 57344 (e5m2);
    q is the nearest FP8 value to x / m * top.  Infinities saturate, a NaN stays one.  ``rows`` (int32) gathers: row r of q
    comes from row rows[r] of x, which may repeat; an index outside x gives a row of zeros.  Returns (q, scale).
    """
    if x.dim() != 2 or q.dim() != 2:
        raise ValueError("x and q are matrices")
    count, k = q.shape
    if x.shape[1] != k or (rows is None and count != x.shape[0]):
        raise ValueError(f"q must have x's rows and columns (rows as `rows` says), got {list(q.shape)} for {list(x.shape)}")
    ldx = _matrix("x", x, HALF, x.shape)
    ldq = _matrix("q", q, F8, q.shape)
    _vector("scale", scale, F32, (count,))
    if rows is not None:
        _vector("rows", rows, INT32, (count,))
    device = _device(q, x, scale, rows)
    _call(device, "quantize_rows", _cabi.lib().b200fp8_quantize_rows, x.shape[0], count, k, x.data_ptr(), HALF[x.dtype], ldx,
          None if rows is None else rows.data_ptr(), q.data_ptr(), F8[q.dtype], ldq, scale.data_ptr())
    return q, scale


def _grouped(what, a, b, d, ends, cols, *, alpha, beta, a_scale, b_scale, d_scale, amax_d, bias=None, a_row_scale=None,
             b_row_scale=None, activation=0, kernel=KERNEL_AUTO, max_ctas=0):
    """The part of the three products that comes behind their shape checks: epilogue, options, call."""
    experts = ends.shape[0]
    _vector("ends", ends, INT32, (experts,))
    for name, t in (("a_scale", a_scale), ("b_scale", b_scale), ("d_scale", d_scale), ("amax_d", amax_d)):
        if t is not None and (t.dtype != torch.float32 or t.numel() != 1):
            raise TypeError(f"{name} is a one-element float32 tensor")
    if bias is not None:
        _vector("bias", bias, WIDE, (experts, cols))
    if a_row_scale is not None:
        _vector("a_row_scale", a_row_scale, F32, (a.shape[0],))
    if b_row_scale is not None:
        _vector("b_row_scale", b_row_scale, F32, (experts, cols))
    if isinstance(activation, str):
        if activation not in ACTIVATIONS:
            raise ValueError(f"activation is one of {sorted(ACTIVATIONS)}")
        activation = ACTIVATIONS[activation]
    elif activation not in ACTIVATIONS.values():
        raise ValueError("unknown activation")
    device = _device(d, a, b, ends, a_scale, b_scale, d_scale, amax_d, bias, a_row_scale, b_row_scale)
    ptr = lambda t: None if t is None else t.data_ptr()
    ep = _cabi.EpilogueDesc(_EPILOGUE_BYTES, alpha, beta, ptr(a_scale), ptr(b_scale), ptr(d_scale), ptr(amax_d), ptr(bias),
                            0 if bias is None else WIDE[bias.dtype], activation, ptr(a_row_scale), ptr(b_row_scale))
    opt = None if kernel == KERNEL_AUTO and not max_ctas else ctypes.byref(Options(_OPTIONS_BYTES, 0, kernel, 0, max_ctas))
    lda = _matrix("a", a, F8, a.shape)
    ldb = _matrix("b", b, F8, b.shape)
    ldd = _matrix("d", d, OUT, d.shape)
    if what == "gemm_grouped_wgrad":
        tail = (ldb, d.data_ptr(), OUT[d.dtype], ldd, _stride(d, ldd))
        n, k = d.shape[1:]
    else:
        tail = (ldb, _stride(b, ldb), d.data_ptr(), OUT[d.dtype], ldd)
        n, k = b.shape[1:]
    if experts == 0 or n == 0 or k == 0:
        return d
    _call(device, what, getattr(_cabi.lib(), "b200fp8_" + what), experts, a.shape[0], k, n, ends.data_ptr(), a.data_ptr(), F8[a.dtype], lda,
          b.data_ptr(), F8[b.dtype], *tail, ctypes.byref(ep), opt)
    return d


def gemm_grouped(a: torch.Tensor, b: torch.Tensor, d: torch.Tensor, ends: torch.Tensor, *, alpha: float = 1.0, beta: float = 0.0,
                 a_scale=None, b_scale=None, d_scale=None, amax_d=None, bias=None, a_row_scale=None, b_row_scale=None,
                 activation: str | int = 0, kernel: int = KERNEL_AUTO, max_ctas: int = 0):
    """The experts' products: d[r] = ep(b[e] a[r]) for the rows r of group e.

    a [rows][K] and b [experts][N][K] are FP8, d [rows][N] is float32, bfloat16, float16 or FP8; ``ends`` (int32, on the
    device) holds each group's end, the first group starts at row 0, groups may be empty, and rows of no group are left as
    they were.  The epilogue is that of ``gemm_epilogue`` with ``b_row_scale`` and ``bias`` as [experts][N]:
    act(alpha * a_scale * b_scale * a_row_scale[r] * b_row_scale[e][n] * sum + beta * d + bias[e][n]), times d_scale.
    K must be a multiple of 16.  Returns d.
    """
    if a.dim() != 2 or b.dim() != 3 or d.dim() != 2 or ends.dim() != 1 or b.shape[0] != ends.shape[0] or b.shape[2] != a.shape[1] \
            or d.shape != (a.shape[0], b.shape[1]):
        raise ValueError(f"a [rows][K], b [experts][N][K], d [rows][N], ends [experts]: got {list(a.shape)}, {list(b.shape)}, "
                         f"{list(d.shape)}, {list(ends.shape)}")
    return _grouped("gemm_grouped", a, b, d, ends, b.shape[1], alpha=alpha, beta=beta, a_scale=a_scale, b_scale=b_scale, d_scale=d_scale,
                    amax_d=amax_d, bias=bias, a_row_scale=a_row_scale, b_row_scale=b_row_scale, activation=activation, kernel=kernel,
                    max_ctas=max_ctas)


def gemm_grouped_dgrad(a: torch.Tensor, b: torch.Tensor, d: torch.Tensor, ends: torch.Tensor, *, alpha: float = 1.0, beta: float = 0.0,
                       a_scale=None, b_scale=None, d_scale=None, amax_d=None, bias=None, a_row_scale=None, b_row_scale=None,
                       activation: str | int = 0, kernel: int = KERNEL_AUTO, max_ctas: int = 0):
    """The gradient of ``gemm_grouped`` by its rows: d[r] = ep(b[e]^T a[r]), with a [rows][N] the gradient of the output, the
    weights b [experts][N][K] as the forward pass has them, and d [rows][K].  Epilogue as there, vectors of [experts][K].
    N and K must be multiples of 16."""
    if a.dim() != 2 or b.dim() != 3 or d.dim() != 2 or ends.dim() != 1 or b.shape[0] != ends.shape[0] or b.shape[1] != a.shape[1] \
            or d.shape != (a.shape[0], b.shape[2]):
        raise ValueError(f"a [rows][N], b [experts][N][K], d [rows][K], ends [experts]: got {list(a.shape)}, {list(b.shape)}, "
                         f"{list(d.shape)}, {list(ends.shape)}")
    return _grouped("gemm_grouped_dgrad", a, b, d, ends, b.shape[2], alpha=alpha, beta=beta, a_scale=a_scale, b_scale=b_scale, d_scale=d_scale,
                    amax_d=amax_d, bias=bias, a_row_scale=a_row_scale, b_row_scale=b_row_scale, activation=activation, kernel=kernel,
                    max_ctas=max_ctas)


def gemm_grouped_wgrad(a: torch.Tensor, b: torch.Tensor, d: torch.Tensor, ends: torch.Tensor, *, alpha: float = 1.0, beta: float = 0.0,
                       a_scale=None, b_scale=None, d_scale=None, amax_d=None, kernel: int = KERNEL_AUTO, max_ctas: int = 0):
    """The gradient of ``gemm_grouped`` by its weights: d[e] = alpha * a_scale * b_scale * sum over the rows r of group e of
    a[r]^T b[r], plus beta * d[e]; a [rows][N] is the gradient of the output, b [rows][K] the forward pass's input, d
    [experts][N][K].  An empty group gives beta * d[e] (zeros for beta = 0).  N and K must be multiples of 16."""
    if a.dim() != 2 or b.dim() != 2 or d.dim() != 3 or ends.dim() != 1 or a.shape[0] != b.shape[0] \
            or d.shape != (ends.shape[0], a.shape[1], b.shape[1]):
        raise ValueError(f"a [rows][N], b [rows][K], d [experts][N][K], ends [experts]: got {list(a.shape)}, {list(b.shape)}, "
                         f"{list(d.shape)}, {list(ends.shape)}")
    return _grouped("gemm_grouped_wgrad", a, b, d, ends, b.shape[1], alpha=alpha, beta=beta, a_scale=a_scale, b_scale=b_scale, d_scale=d_scale,
                    amax_d=amax_d, kernel=kernel, max_ctas=max_ctas)


def _w4(codes, scales, x, y, zeros, lead):
    """Shapes and layouts that both 4-bit products check; returns (n, k, group, pitches)."""
    n, half = codes.shape[-2:]
    k, groups = 2 * half, scales.shape[-1]
    if groups == 0 or k % groups or k // groups not in (32, 64, 128):
        raise ValueError(f"scales has one value per row and group of 32, 64 or 128: got {groups} for K = {k}")
    pitch = (_matrix("codes", codes, U8, (*lead, n, half)), _matrix("scales", scales, WIDE, (*lead, n, groups)),
             0 if zeros is None else _matrix("zeros", zeros, U8, (*lead, n, groups)),
             _matrix("x", x, HALF, (x.shape[0], k)), _matrix("y", y, (x.dtype, torch.float32), (y.shape[0], n)))
    return n, k, k // groups, pitch


def gemv_w4(codes: torch.Tensor, scales: torch.Tensor, x: torch.Tensor, y: torch.Tensor, *, zeros: torch.Tensor | None = None):
    """y[m] = W x[m] for a matrix of 4-bit weights W[n][k] = scales[n][k // group] * (codes[n][k] - zeros[n][k // group]).

    codes is uint8 [N][K/2], two codes to a byte with the even k in the low half; scales [N][K/group] is float32, bfloat16 or
    float16 and says the group size (32, 64 or 128); zeros is uint8 of the same shape, or None for 8.  x [M][K] is bfloat16 or
    float16, y [M][N] has its type or float32.  Made for a few vectors.  Returns y.
    """
    if codes.dim() != 2 or scales.dim() != 2 or x.dim() != 2 or y.dim() != 2 or x.shape[0] != y.shape[0]:
        raise ValueError("codes [N][K/2], scales [N][K/group], x [M][K], y [M][N]")
    n, k, group, ld = _w4(codes, scales, x, y, zeros, ())
    device = _device(y, codes, scales, x, zeros)
    _call(device, "gemv_w4", _cabi.lib().b200fp8_gemv_w4, x.shape[0], k, n, group, codes.data_ptr(), ld[0], scales.data_ptr(),
          WIDE[scales.dtype], ld[1], None if zeros is None else zeros.data_ptr(), ld[2], x.data_ptr(), HALF[x.dtype], ld[3],
          y.data_ptr(), WIDE[y.dtype], ld[4])
    return y


def gemv_w4_experts(codes: torch.Tensor, scales: torch.Tensor, x: torch.Tensor, y: torch.Tensor, expert: torch.Tensor, *,
                    zeros: torch.Tensor | None = None):
    """The experts' products of a few tokens with 4-bit weights: y[r] = W[expert[r]] x[r // (rows / tokens)].

    codes [experts][N][K/2], scales and zeros [experts][N][K/group] as in ``gemv_w4``; x [tokens][K]; y [rows][N] with rows a
    multiple of tokens (the experts of a token follow one another), at most 4096; ``expert`` int32 [rows] on the device.  A
    row whose expert is not one of the experts (for instance -1) is left as it was.  Returns y.
    """
    if codes.dim() != 3 or scales.dim() != 3 or x.dim() != 2 or y.dim() != 2:
        raise ValueError("codes [experts][N][K/2], scales [experts][N][K/group], x [tokens][K], y [rows][N]")
    tokens, rows, experts = x.shape[0], y.shape[0], codes.shape[0]
    if (rows % tokens if tokens else rows):
        raise ValueError(f"y's rows ({rows}) must be a multiple of x's ({tokens})")
    _vector("expert", expert, INT32, (rows,))
    n, k, group, ld = _w4(codes, scales, x, y, zeros, (experts,))
    device = _device(y, codes, scales, x, expert, zeros)
    _call(device, "gemv_w4_experts", _cabi.lib().b200fp8_gemv_w4_experts, tokens, rows, experts, k, n, group, codes.data_ptr(), ld[0],
          _stride(codes, ld[0]), scales.data_ptr(), WIDE[scales.dtype], ld[1], _stride(scales, ld[1]),
          None if zeros is None else zeros.data_ptr(), ld[2], 0 if zeros is None else _stride(zeros, ld[2]), expert.data_ptr(),
          x.data_ptr(), HALF[x.dtype], ld[3], y.data_ptr(), WIDE[y.dtype], ld[4])
    return y
