"""Refusals of the expert-layer entry points: bad arguments come back as errors before anything touches a device."""
import ctypes

import pytest
import torch

from __graft_entry__ import load_package


@pytest.fixture(scope="module")
def pkg():
    return load_package()


INVALID = 1                                   # cudaErrorInvalidValue
P = ctypes.c_void_p(0x10000)                  # never dereferenced: the checks come first
ODD = ctypes.c_void_p(0x10001)


def change(args, **kw):
    return {**args, **kw}


GROUPED = dict(experts=4, rows=64, k=128, n=256, ends=P, a=P, a_dtype=0, lda=256, b=P, b_dtype=0, ldb=128, stride_b=256 * 128, d=P,
               d_dtype=1, ldd=256, epilogue=None, options=None)


@pytest.mark.parametrize("entry", ["b200fp8_gemm_grouped", "b200fp8_gemm_grouped_dgrad", "b200fp8_gemm_grouped_wgrad"])
@pytest.mark.parametrize("bad", [dict(experts=-1), dict(rows=-1), dict(k=0), dict(n=0), dict(k=-16), dict(ends=None), dict(ends=ODD),
                                 dict(a=None), dict(a=ODD), dict(b=None), dict(b=ODD), dict(d=None), dict(d=ODD), dict(a_dtype=2),
                                 dict(b_dtype=-1), dict(d_dtype=5), dict(d_dtype=-1), dict(k=120), dict(lda=250), dict(ldb=136), dict(ldb=64),
                                 dict(ldd=64), dict(experts=1 << 17), dict(rows=(1 << 30) + 1), dict(k=(1 << 30) + 16, lda=1 << 31, ldb=1 << 31, stride_b=1 << 38),
                                 dict(n=(1 << 30) + 16, lda=1 << 31, ldd=1 << 31, stride_b=1 << 38), dict(lda=1 << 62), dict(epilogue="size"),
                                 dict(epilogue="activation"), dict(options="size"), dict(options="depth"), dict(options="split"),
                                 dict(options="kernel"), dict(options="ctas")])
def test_grouped_products_refuse(pkg, entry, bad):
    if "lda" in bad and bad["lda"] == 250:
        bad = dict(lda=120)
    call = dict(GROUPED, lda=128 if entry == "b200fp8_gemm_grouped" else 256)
    call.update(bad)
    if call["epilogue"] is not None:
        size = ctypes.sizeof(pkg._cabi.EpilogueDesc)
        call["epilogue"] = ctypes.byref(pkg._cabi.EpilogueDesc(7 if bad["epilogue"] == "size" else size, 1.0, 0.0, None, None, None, None, None, 0, 9))
    if call["options"] is not None:
        fields = {"size": (3, 0, 0, 0, 0), "depth": (20, 2, 0, 0, 0), "split": (20, 0, 0, 2, 0), "kernel": (20, 0, 4, 0, 0), "ctas": (20, 0, 0, 0, -1)}
        call["options"] = ctypes.byref(pkg._cabi.Options(*fields[bad["options"]]))
    c = call
    head = (c["experts"], c["rows"], c["k"], c["n"], c["ends"], c["a"], c["a_dtype"], c["lda"], c["b"], c["b_dtype"], c["ldb"])
    tail = (c["epilogue"], c["options"], None)
    if entry.endswith("wgrad"):
        args = head + (c["d"], c["d_dtype"], c["ldd"], 256 * 256) + tail
    else:
        args = head + (c["stride_b"], c["d"], c["d_dtype"], c["ldd"]) + tail
    assert getattr(pkg._cabi.lib(), entry)(*args) == INVALID


def test_grouped_products_refuse_what_only_one_of_them_refuses(pkg):
    lib, size = pkg._cabi.lib(), ctypes.sizeof(pkg._cabi.EpilogueDesc)
    # matrices of the experts that overlap, and a pitch between them that TMA cannot take
    for stride in (255 * 128, 256 * 128 + 8):
        assert lib.b200fp8_gemm_grouped(4, 64, 128, 256, P, P, 0, 128, P, 0, 128, stride, P, 1, 256, None, None, None) == INVALID
        assert lib.b200fp8_gemm_grouped_dgrad(4, 64, 128, 256, P, P, 0, 256, P, 0, 128, stride, P, 1, 128, None, None, None) == INVALID
    assert lib.b200fp8_gemm_grouped_wgrad(4, 64, 128, 256, P, P, 0, 256, P, 0, 128, P, 0, 128, 255 * 128, None, None, None) == INVALID
    # N is a contiguous extent in the backward products only
    assert lib.b200fp8_gemm_grouped_dgrad(4, 64, 128, 250, P, P, 0, 256, P, 0, 128, 1 << 20, P, 1, 128, None, None, None) == INVALID
    assert lib.b200fp8_gemm_grouped_wgrad(4, 64, 128, 250, P, P, 0, 256, P, 0, 128, P, 0, 128, 1 << 20, None, None, None) == INVALID
    # scales of rows, a bias or an activation inside a sum over the rows
    for field in (dict(bias=0x10000), dict(activation=1), dict(a_row_scale=0x10000), dict(b_row_scale=0x10000)):
        ep = pkg._cabi.EpilogueDesc(size, 1.0, 0.0)
        for key, value in field.items():
            setattr(ep, key, value)
        assert lib.b200fp8_gemm_grouped_wgrad(4, 64, 128, 256, P, P, 0, 256, P, 0, 128, P, 0, 128, 256 * 128, ctypes.byref(ep), None, None) == INVALID


@pytest.mark.parametrize("field", ["a_scale", "b_scale", "d_scale", "amax_d", "a_row_scale", "b_row_scale", "bias"])
def test_grouped_products_refuse_misaligned_epilogue_vectors(pkg, field):
    ep = pkg._cabi.EpilogueDesc(ctypes.sizeof(pkg._cabi.EpilogueDesc), 1.0, 0.0)
    setattr(ep, field, 0x10002)
    assert pkg._cabi.lib().b200fp8_gemm_grouped(4, 64, 128, 256, P, P, 0, 128, P, 0, 128, 256 * 128, P, 1, 256, ctypes.byref(ep), None, None) == INVALID


@pytest.mark.parametrize("bad", [dict(source=-1), dict(rows=-1), dict(k=-1), dict(k=(1 << 30) + 1, ldx=1 << 31, ldq=1 << 31), dict(x_dtype=0), dict(x_dtype=3), dict(q_dtype=2), dict(ldx=63),
                                 dict(ldq=63), dict(rows=11), dict(scale=None), dict(scale=ODD), dict(x=None), dict(x=ODD), dict(q=None),
                                 dict(index=ODD)])
def test_quantize_rows_refuses(pkg, bad):
    c = dict(source=10, rows=10, k=64, x=P, x_dtype=1, ldx=64, index=None, q=P, q_dtype=0, ldq=64, scale=P)
    c.update(bad)
    assert pkg._cabi.lib().b200fp8_quantize_rows(*(c[key] for key in ("source", "rows", "k", "x", "x_dtype", "ldx", "index", "q", "q_dtype", "ldq",
                                                                      "scale")), None) == INVALID


W4 = dict(m=2, k=256, n=64, group=64, codes=P, code_ld=128, scales=P, scale_dtype=1, scale_ld=4, zeros=P, zero_ld=4, x=P, x_dtype=1, ldx=256, y=P,
          y_dtype=1, ldy=64)


@pytest.mark.parametrize("bad", [dict(m=-1), dict(k=-64), dict(k=0), dict(n=-1), dict(n=(1 << 23) + 1, ldy=1 << 24), dict(group=0), dict(group=48), dict(group=256), dict(k=224), dict(codes=None),
                                 dict(codes=ODD), dict(code_ld=112), dict(code_ld=136), dict(scales=None), dict(scales=ODD), dict(scale_dtype=3),
                                 dict(scale_ld=3), dict(zero_ld=3), dict(x=None), dict(x=ODD), dict(x_dtype=0), dict(ldx=248), dict(ldx=260),
                                 dict(y=None), dict(y=ODD), dict(y_dtype=2), dict(ldy=63)])
def test_w4_products_refuse(pkg, bad):
    c = dict(W4)
    c.update(bad)
    lib = pkg._cabi.lib()
    assert lib.b200fp8_gemv_w4(*(c[key] for key in W4), None) == INVALID
    args = (c["m"], c["m"], 3, c["k"], c["n"], c["group"], c["codes"], c["code_ld"], 64 * 128, c["scales"], c["scale_dtype"], c["scale_ld"], 256,
            c["zeros"], c["zero_ld"], 256, P, c["x"], c["x_dtype"], c["ldx"], c["y"], c["y_dtype"], c["ldy"], None)
    assert lib.b200fp8_gemv_w4_experts(*args) == INVALID


@pytest.mark.parametrize("change", [{0: -1}, {1: -2}, {2: -1}, {1: 5}, {0: 0}, {1: 4098}, {2: 4097}, {8: 63 * 128}, {8: 64 * 128 + 8}, {12: 255}, {15: 255},
                                    {16: None}, {16: ODD}])
def test_w4_by_expert_refuses(pkg, change):
    args = [2, 4, 3, 256, 64, 64, P, 128, 64 * 128, P, 1, 4, 256, P, 4, 256, P, P, 1, 256, P, 1, 64, None]
    for at, value in change.items():
        args[at] = value
    assert pkg._cabi.lib().b200fp8_gemv_w4_experts(*args) == INVALID


def test_one_experts_stride_is_not_read(pkg):
    """The pitch from one expert's matrix to the next says nothing where there is one expert (calls without rows: nothing is launched)."""
    lib = pkg._cabi.lib()
    for stride in (7, -16, 1 << 60):
        assert lib.b200fp8_gemm_grouped(1, 0, 128, 256, P, P, 0, 128, P, 0, 128, stride, P, 1, 256, None, None, None) != INVALID
        assert lib.b200fp8_gemm_grouped_dgrad(1, 0, 128, 256, P, P, 0, 256, P, 0, 128, stride, P, 1, 128, None, None, None) != INVALID
        assert lib.b200fp8_gemv_w4_experts(0, 0, 1, 64, 64, 64, P, 32, stride, P, 1, 1, stride, P, 1, stride, None, P, 1, 64, P, 1, 64, None) == 0
    # with two it does, and a pitch between rows that overflows does not slip through
    assert lib.b200fp8_gemm_grouped(2, 0, 128, 256, P, P, 0, 128, P, 0, 128, 7, P, 1, 256, None, None, None) == INVALID
    assert lib.b200fp8_gemm_grouped(2, 0, 128, 1 << 30, P, P, 0, 128, P, 0, 1 << 38, 1 << 38, P, 1, 1 << 30, None, None, None) == INVALID
    assert lib.b200fp8_gemv_w4_experts(0, 0, 2, 64, 65, 64, P, 32, 2080, P, 1, 1 << 58, 64, P, 1, 65, None, P, 1, 64, P, 1, 65, None) == INVALID


def test_empty_calls_do_nothing(pkg):
    lib = pkg._cabi.lib()
    assert lib.b200fp8_quantize_rows(0, 0, 64, None, 1, 64, None, None, 0, 64, None, None) == 0
    assert lib.b200fp8_gemv_w4(0, 64, 64, 64, None, 32, None, 1, 1, None, 0, None, 1, 64, None, 1, 64, None) == 0
    assert lib.b200fp8_gemv_w4_experts(0, 0, 4, 64, 64, 64, P, 32, 2048, P, 1, 1, 64, None, 0, 0, None, P, 1, 64, P, 1, 64, None) == 0


def f8(*shape):
    return torch.empty(shape, dtype=torch.uint8).view(torch.float8_e4m3fn)


def test_python_layer_proves_shapes_and_types_first(pkg):
    g = pkg.gemm
    ends = torch.zeros(3, dtype=torch.int32)
    a, b, d = f8(8, 32), f8(3, 16, 32), torch.empty(8, 16)
    for args in ((a, b, torch.empty(8, 15), ends), (a, b, d, ends[:2]), (f8(8, 16), b, d, ends), (a, b[0], d, ends), (a, b, torch.empty(7, 16), ends)):
        with pytest.raises(ValueError):
            g.gemm_grouped(*args)
    with pytest.raises(TypeError):
        g.gemm_grouped(a, b, d, ends.long())
    with pytest.raises(ValueError):
        g.gemm_grouped(a, b, d, ends)                                          # host tensors
    with pytest.raises(TypeError):
        g.gemm_grouped(a, b, d, ends, bias=torch.empty(16))                    # one bias row per expert
    with pytest.raises(TypeError):
        g.gemm_grouped(a, b, d, ends, a_row_scale=torch.empty(7))
    with pytest.raises(ValueError):
        g.gemm_grouped(a, b, d, ends, activation="swish")
    with pytest.raises(ValueError):
        g.gemm_grouped_dgrad(f8(8, 16), b, torch.empty(8, 16), ends)           # d has K columns
    with pytest.raises(ValueError):
        g.gemm_grouped_wgrad(f8(8, 16), a, torch.empty(3, 32, 16), ends)       # d is [experts][N][K]
    with pytest.raises(ValueError):
        g.quantize_rows(torch.empty(4, 32, dtype=torch.bfloat16), f8(5, 32), torch.empty(5))
    with pytest.raises(TypeError):
        g.quantize_rows(torch.empty(4, 32), f8(4, 32), torch.empty(4))         # FP32 rows
    with pytest.raises(TypeError):
        g.quantize_rows(torch.empty(4, 32, dtype=torch.bfloat16), f8(4, 32), torch.empty(4, dtype=torch.float64))
    with pytest.raises(ValueError):
        g.quantize_rows(torch.empty(32, 4, dtype=torch.bfloat16).t(), f8(4, 32), torch.empty(4))
    codes, x = torch.empty(16, 64, dtype=torch.uint8), torch.empty(2, 128, dtype=torch.bfloat16)
    y = torch.empty(2, 16, dtype=torch.bfloat16)
    for scales in (torch.empty(16, 8), torch.empty(16, 0), torch.empty(15, 1)):
        with pytest.raises(ValueError):
            g.gemv_w4(codes, scales, x, y)
    with pytest.raises(TypeError):
        g.gemv_w4(codes, torch.empty(16, 2), x, y.half())
    with pytest.raises(ValueError):
        g.gemv_w4(codes, torch.empty(16, 2), x, y, zeros=torch.empty(16, 1, dtype=torch.uint8))
    with pytest.raises(ValueError):
        g.gemv_w4_experts(codes[None], torch.empty(1, 16, 2), x, torch.empty(3, 16, dtype=torch.bfloat16), torch.zeros(3, dtype=torch.int32))
    with pytest.raises(TypeError):
        g.gemv_w4_experts(codes[None], torch.empty(1, 16, 2), x, y, torch.zeros(2, dtype=torch.int64))


def test_python_layer_refuses_rows_and_matrices_that_overlap(pkg):
    e, one = pkg.experts, {torch.float32: 0}
    with pytest.raises(ValueError):
        e._pitch("t", torch.empty(4, 8).as_strided((4, 8), (4, 1)), one, 8)            # rows that overlap
    with pytest.raises(ValueError):
        e._pitch("t", torch.empty(100).as_strided((2, 4, 8), (24, 8, 1)), one, 8)      # matrices that overlap
    assert e._pitch("t", torch.empty(4, 16)[:, :8], one, 8) == 16 and e._pitch("t", torch.empty(1, 16)[:, :8], one, 8) == 8
