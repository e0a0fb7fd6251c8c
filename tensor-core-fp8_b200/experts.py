"""Host layer of the expert-layer operators: FP8 products grouped by expert, their gradients, the row quantiser that makes
their operands, and products of 4-bit weights with a few vectors.

Layouts and formats are those of the dense operator (GEMM/include/gemm.cuh:12-55): operands row-major, ``b`` as rows of
the contraction index.  The reference has one weight matrix per product and no weights below eight bits, so these
operators have no counterpart there.  Everything is checked here before the call (the C ABI sees only pointers); calls
are enqueued on the current stream of the tensors' device.  Outputs must not share memory with inputs.

A decode step's kernels run for a few microseconds, so the checks are written to cost little: each asks a tensor once for
what it needs and looks closer only where that is not the plain contiguous case.
"""
from __future__ import annotations

import ctypes
import struct

import torch

from . import _cabi
from ._cabi import E4M3, E5M2, KERNEL_AUTO, Options

F8 = {torch.float8_e4m3fn: E4M3, torch.float8_e5m2: E5M2}
OUT = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2, torch.float8_e4m3fn: 3, torch.float8_e5m2: 4}
HALF = {torch.bfloat16: 1, torch.float16: 2}
WIDE = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
F32, INT32, U8 = {torch.float32: 0}, {torch.int32: 0}, {torch.uint8: 0}
ACTIVATIONS = {"none": 0, "relu": 1, "gelu": 2, "gelu_tanh": 3}

_EPILOGUE = struct.Struct("@iffPPPPPiiPP")          # b200fp8_epilogue of include/b200fp8.h
_EPILOGUE_BYTES = ctypes.sizeof(_cabi.EpilogueDesc)
assert _EPILOGUE.size == _EPILOGUE_BYTES
_functions: dict = {}


def _pitch(name: str, t: torch.Tensor, dtypes, cols: int) -> int:
    """Type and layout of a matrix of `cols` columns (or of one per expert); returns its row pitch in elements."""
    if t.dtype in dtypes and t.is_contiguous():
        return cols
    if t.dtype not in dtypes:
        raise TypeError(f"{name} has type {t.dtype}, expected one of {', '.join(str(d) for d in dtypes)}")
    rows = t.shape[-2]
    if cols > 1 and t.stride(-1) != 1:
        raise ValueError(f"{name}: the last dimension must be contiguous, got strides {t.stride()}")
    pitch = t.stride(-2) if rows > 1 else cols
    if pitch < cols:
        raise ValueError(f"{name}: rows overlap (pitch {pitch}, {cols} columns)")
    if t.dim() == 3 and t.shape[0] > 1 and t.stride(0) < (rows - 1) * pitch + cols:
        raise ValueError(f"{name}: matrices overlap (pitch {t.stride(0)})")
    return pitch


def _stride(t: torch.Tensor, matrices: int, rows: int, pitch: int) -> int:
    """Pitch from one expert's matrix to the next."""
    return t.stride()[0] if matrices > 1 else rows * pitch


def _vector(name: str, t: torch.Tensor, dtypes, *shape: int) -> int:
    """Checks a contiguous tensor of this shape and returns its address."""
    if t.dtype not in dtypes or t.shape != shape or not t.is_contiguous():
        raise TypeError(f"{name} must be contiguous {list(shape)} of {', '.join(str(d) for d in dtypes)}, got {t.dtype} {list(t.shape)}")
    return t.data_ptr()


def _device(first: torch.Tensor, *others) -> int:
    device = first.get_device()
    if device < 0:
        raise ValueError("the operators take CUDA tensors (device pointers)")
    for t in others:
        if t is not None and t.get_device() != device:
            raise ValueError(f"all tensors must live on one device, got {first.device} and {t.device}")
    return device


def _call(device: int, what: str, *args) -> None:
    """Enqueues the call on the device's current stream, with that device current."""
    function = _functions.get(what)
    if function is None:
        function = _functions[what] = getattr(_cabi.lib(), "b200fp8_" + what)
    if torch.cuda.current_device() == device:
        code = function(*args, torch._C._cuda_getCurrentRawStream(device))
    else:
        with torch.cuda.device(device):
            code = function(*args, torch._C._cuda_getCurrentRawStream(device))
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
    source, k = x.shape
    count, columns = q.shape
    if columns != k or (rows is None and count != source):
        raise ValueError(f"q must have x's rows and columns (rows as `rows` says), got {list(q.shape)} for {list(x.shape)}")
    ldx, ldq = _pitch("x", x, HALF, k), _pitch("q", q, F8, k)
    at = _vector("scale", scale, F32, count)
    index = None if rows is None else _vector("rows", rows, INT32, count)
    _call(_device(q, x, scale, rows), "quantize_rows", source, count, k, x.data_ptr(), HALF[x.dtype], ldx, index, q.data_ptr(),
          F8[q.dtype], ldq, at)
    return q, scale


def _one(name: str, t) -> int:
    """Address of an optional one-element float32 tensor."""
    if t is None:
        return 0
    if t.dtype != torch.float32 or t.numel() != 1:
        raise TypeError(f"{name} is a one-element float32 tensor")
    return t.data_ptr()


def _grouped(what, a, b, d, ends, experts, rows, n, k, a_cols, cols, alpha, beta, a_scale, b_scale, d_scale, amax_d, bias, a_row_scale, b_row_scale,
             activation, kernel, max_ctas):
    """The part of the three products that comes behind their shape checks: epilogue, options, call."""
    first_row = _vector("ends", ends, INT32, experts)
    if activation.__class__ is str:
        if activation not in ACTIVATIONS:
            raise ValueError(f"activation is one of {sorted(ACTIVATIONS)}")
        activation = ACTIVATIONS[activation]
    elif activation not in (0, 1, 2, 3):
        raise ValueError("unknown activation")
    ep = _EPILOGUE.pack(_EPILOGUE_BYTES, alpha, beta, _one("a_scale", a_scale), _one("b_scale", b_scale), _one("d_scale", d_scale),
                        _one("amax_d", amax_d), 0 if bias is None else _vector("bias", bias, WIDE, experts, cols),
                        0 if bias is None else WIDE[bias.dtype], activation,
                        0 if a_row_scale is None else _vector("a_row_scale", a_row_scale, F32, rows),
                        0 if b_row_scale is None else _vector("b_row_scale", b_row_scale, F32, experts, cols))
    opt = None if kernel == KERNEL_AUTO and not max_ctas else ctypes.byref(Options(ctypes.sizeof(Options), 0, kernel, 0, max_ctas))
    lda, ldb, ldd = _pitch("a", a, F8, a_cols), _pitch("b", b, F8, k), _pitch("d", d, OUT, cols)
    device = _device(d, a, b, ends, a_scale, b_scale, d_scale, amax_d, bias, a_row_scale, b_row_scale)
    if experts == 0 or n == 0 or k == 0:
        if experts and rows and cols and what != "gemm_grouped_wgrad":
            raise ValueError(f"{what}: the contraction has no extent, a is {list(a.shape)}")
        if amax_d is not None:
            amax_d.zero_()
        return d
    if what == "gemm_grouped_wgrad":
        _call(device, what, experts, rows, k, n, first_row, a.data_ptr(), F8[a.dtype], lda, b.data_ptr(), F8[b.dtype], ldb, d.data_ptr(),
              OUT[d.dtype], ldd, _stride(d, experts, n, ldd), ep, opt)
    else:
        _call(device, what, experts, rows, k, n, first_row, a.data_ptr(), F8[a.dtype], lda, b.data_ptr(), F8[b.dtype], ldb,
              _stride(b, experts, n, ldb), d.data_ptr(), OUT[d.dtype], ldd, ep, opt)
    return d


def _shapes(a, b, d, ends, wanted):
    raise ValueError(f"{wanted}, ends [experts]: got {list(a.shape)}, {list(b.shape)}, {list(d.shape)}, {list(ends.shape)}")


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
    if a.dim() != 2 or b.dim() != 3 or d.dim() != 2 or ends.dim() != 1:
        _shapes(a, b, d, ends, "a [rows][K], b [experts][N][K], d [rows][N]")
    rows, k = a.shape
    experts, n, depth = b.shape
    if depth != k or d.shape != (rows, n) or ends.shape[0] != experts:
        _shapes(a, b, d, ends, "a [rows][K], b [experts][N][K], d [rows][N]")
    return _grouped("gemm_grouped", a, b, d, ends, experts, rows, n, k, k, n, alpha, beta, a_scale, b_scale, d_scale, amax_d, bias, a_row_scale,
                    b_row_scale, activation, kernel, max_ctas)


def gemm_grouped_dgrad(a: torch.Tensor, b: torch.Tensor, d: torch.Tensor, ends: torch.Tensor, *, alpha: float = 1.0, beta: float = 0.0,
                       a_scale=None, b_scale=None, d_scale=None, amax_d=None, bias=None, a_row_scale=None, b_row_scale=None,
                       activation: str | int = 0, kernel: int = KERNEL_AUTO, max_ctas: int = 0):
    """The gradient of ``gemm_grouped`` by its rows: d[r] = ep(b[e]^T a[r]), with a [rows][N] the gradient of the output, the
    weights b [experts][N][K] as the forward pass has them, and d [rows][K].  Epilogue as there, vectors of [experts][K].
    The forward pass's ``b_row_scale`` lies along the sum over N: multiply it into the gradient before that is quantised.
    N and K must be multiples of 16."""
    if a.dim() != 2 or b.dim() != 3 or d.dim() != 2 or ends.dim() != 1:
        _shapes(a, b, d, ends, "a [rows][N], b [experts][N][K], d [rows][K]")
    rows, n = a.shape
    experts, depth, k = b.shape
    if depth != n or d.shape != (rows, k) or ends.shape[0] != experts:
        _shapes(a, b, d, ends, "a [rows][N], b [experts][N][K], d [rows][K]")
    return _grouped("gemm_grouped_dgrad", a, b, d, ends, experts, rows, n, k, n, k, alpha, beta, a_scale, b_scale, d_scale, amax_d, bias, a_row_scale,
                    b_row_scale, activation, kernel, max_ctas)


def gemm_grouped_wgrad(a: torch.Tensor, b: torch.Tensor, d: torch.Tensor, ends: torch.Tensor, *, alpha: float = 1.0, beta: float = 0.0,
                       a_scale=None, b_scale=None, d_scale=None, amax_d=None, kernel: int = KERNEL_AUTO, max_ctas: int = 0):
    """The gradient of ``gemm_grouped`` by its weights: d[e] = alpha * a_scale * b_scale * sum over the rows r of group e of
    a[r]^T b[r], plus beta * d[e]; a [rows][N] is the gradient of the output, b [rows][K] the forward pass's input, d
    [experts][N][K].  An empty group gives beta * d[e] (zeros for beta = 0).  The operands have one scale each: the forward
    pass's ``a_row_scale`` lies along the sum over the rows, multiply it into the gradient before that is quantised.  N and K must be
    multiples of 16."""
    if a.dim() != 2 or b.dim() != 2 or d.dim() != 3 or ends.dim() != 1:
        _shapes(a, b, d, ends, "a [rows][N], b [rows][K], d [experts][N][K]")
    experts, n, k = d.shape
    rows, a_cols = a.shape
    if b.shape != (rows, k) or a_cols != n or ends.shape[0] != experts:
        _shapes(a, b, d, ends, "a [rows][N], b [rows][K], d [experts][N][K]")
    return _grouped("gemm_grouped_wgrad", a, b, d, ends, experts, rows, n, k, n, k, alpha, beta, a_scale, b_scale, d_scale, amax_d, None, None, None, 0,
                    kernel, max_ctas)


def _w4_group(k: int, groups: int) -> int:
    """The group size that the number of scales of a row says."""
    for group in (128, 64, 32):
        if group * groups == k and groups:
            return group
    raise ValueError(f"scales (and zeros) have one value per row and group of 32, 64 or 128 of K: got {groups} groups for K = {k}")


def gemv_w4(codes: torch.Tensor, scales: torch.Tensor, x: torch.Tensor, y: torch.Tensor, *, zeros: torch.Tensor | None = None):
    """y[m] = W x[m] for a matrix of 4-bit weights W[n][k] = scales[n][k // group] * (codes[n][k] - zeros[n][k // group]).

    codes is uint8 [N][K/2], two codes to a byte with the even k in the low half; scales [N][K/group] is float32, bfloat16 or
    float16, finite and below 2^100, and says the group size (32, 64 or 128); zeros is uint8 of the same shape, or None for 8.
    x [M][K] is bfloat16 or float16, y [M][N] has its type or float32.  Products are exact and sums float32, whatever the spread of
    x.  Made for a few vectors.  Returns y.
    """
    if codes.dim() != 2 or scales.dim() != 2 or x.dim() != 2 or y.dim() != 2:
        raise ValueError("codes [N][K/2], scales [N][K/group], x [M][K], y [M][N]")
    n, half = codes.shape
    m, k = x.shape
    lines, groups = scales.shape
    if k != 2 * half or lines != n or y.shape != (m, n) or (zeros is not None and zeros.shape != (n, groups)):
        raise ValueError(f"codes [N][K/2], scales and zeros [N][K/group], x [M][K], y [M][N]: got {list(codes.shape)}, {list(scales.shape)}, "
                         f"{list(x.shape)}, {list(y.shape)}")
    group = _w4_group(k, groups)
    ldc, lds, ldx, ldy = _pitch("codes", codes, U8, half), _pitch("scales", scales, WIDE, groups), _pitch("x", x, HALF, k), _pitch("y", y, WIDE, n)
    if y.dtype != x.dtype and y.dtype != torch.float32:
        raise TypeError(f"y has x's type or float32, got {y.dtype} and {x.dtype}")
    device = _device(y, codes, scales, x, zeros)
    if zeros is None:
        z, ldz = None, 0
    else:
        ldz, z = _pitch("zeros", zeros, U8, groups), zeros.data_ptr()
    _call(device, "gemv_w4", m, k, n, group, codes.data_ptr(), ldc, scales.data_ptr(), WIDE[scales.dtype], lds, z, ldz, x.data_ptr(),
          HALF[x.dtype], ldx, y.data_ptr(), WIDE[y.dtype], ldy)
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
    experts, n, half = codes.shape
    tokens, k = x.shape
    rows, columns = y.shape
    matrices, lines, groups = scales.shape
    if k != 2 * half or columns != n or matrices != experts or lines != n or (rows % tokens if tokens else rows) or \
            (zeros is not None and zeros.shape != (experts, n, groups)):
        raise ValueError(f"codes [experts][N][K/2], scales and zeros [experts][N][K/group], x [tokens][K], y [rows][N], rows a multiple of "
                         f"tokens: got {list(codes.shape)}, {list(scales.shape)}, {list(x.shape)}, {list(y.shape)}")
    group = _w4_group(k, groups)
    ids = _vector("expert", expert, INT32, rows)
    ldc, lds, ldx, ldy = _pitch("codes", codes, U8, half), _pitch("scales", scales, WIDE, groups), _pitch("x", x, HALF, k), _pitch("y", y, WIDE, n)
    if y.dtype != x.dtype and y.dtype != torch.float32:
        raise TypeError(f"y has x's type or float32, got {y.dtype} and {x.dtype}")
    device = _device(y, codes, scales, x, expert, zeros)
    if zeros is None:
        z, ldz, stride_z = None, 0, 0
    else:
        ldz, z = _pitch("zeros", zeros, U8, groups), zeros.data_ptr()
        stride_z = _stride(zeros, experts, n, ldz)
    _call(device, "gemv_w4_experts", tokens, rows, experts, k, n, group, codes.data_ptr(), ldc, _stride(codes, experts, n, ldc), scales.data_ptr(),
          WIDE[scales.dtype], lds, _stride(scales, experts, n, lds), z, ldz, stride_z, ids, x.data_ptr(), HALF[x.dtype], ldx, y.data_ptr(),
          WIDE[y.dtype], ldy)
    return y
