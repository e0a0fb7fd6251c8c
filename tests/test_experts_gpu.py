"""GPU tests of the expert-layer operators against plain implementations in 64 bits.

Tolerances, before any run: products of FP8 values are exact in FP32; a sum of K of them is formed by K / 32 tensor-core
steps (and a handful of alignments inside one), each of which loses less than one FP32 step (2^-23) of the partial sum's
bound, sum |a b|.  So a product is within (K / 32 + 8) * 2^-23 * S of the exact one, S = sum |a b|, times the scales; the
16-bit products of the 4-bit weights likewise with steps of 16.  The epilogue adds a few FP32 roundings (2^-22 of its
terms' magnitudes), GELU 2e-6 relative / 1e-6 absolute of |t|, and the output's rounding is half a step of its type.
FP8 outputs and the quantiser are compared value for value (or within one rounding of the two ends of the tolerance)."""
import math
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

from __graft_entry__ import load_package

pytestmark = pytest.mark.gpu

E4, E5 = torch.float8_e4m3fn, torch.float8_e5m2
TOP = {E4: 448.0, E5: 57344.0}


@pytest.fixture(scope="module")
def g():
    assert torch.cuda.is_available()
    pkg = load_package()
    pkg._cabi.lib()          # the library must be present: there is no fallback
    torch.cuda.set_device(0)
    return pkg.gemm


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def fp8(shape, dtype, seed, spread=20.0):
    return (torch.randn(shape, generator=gen(seed), device="cuda") * spread).clamp(-400, 400).to(dtype)


def bytes_of(t):
    return t.contiguous().view(torch.uint8)


def done(g):
    torch.cuda.synchronize()
    assert g.device_status() == 0


# ---- the row quantiser ---------------------------------------------------------------------------------------------


def nearest8(v, dtype):
    """The nearest 8-bit value in 64 bits, ties to even, saturating; NaN stays."""
    fraction, lowest = (3, -6) if dtype == E4 else (2, -14)
    _, up = torch.frexp(v)
    step = torch.exp2((up - 1).clamp_min(lowest).double() - fraction)
    return (torch.round(v / step) * step).clamp(-TOP[dtype], TOP[dtype])


def quantized(x, dtype, rows=None):
    v = x.double()
    if rows is not None and x.shape[0] == 0:
        v = v.new_zeros((rows.shape[0], x.shape[1]))
    elif rows is not None:
        ok = (rows >= 0) & (rows < x.shape[0])
        v = torch.where(ok[:, None], v[rows.long().clamp(0, x.shape[0] - 1)], 0.0)
    finite = torch.where(torch.isfinite(v), v.abs(), 0.0)
    m = (finite.amax(1) if v.shape[1] else torch.zeros(v.shape[0], dtype=torch.float64, device=v.device)).clamp_min(2.0 ** -80)
    big = torch.isinf(v)
    # the product by `top` is exact, so the one rounding of the division cannot move a tie (x / m first could)
    q = nearest8(torch.where(big, 0.0, v) * TOP[dtype] / m[:, None], dtype)
    return torch.where(big, torch.sign(v) * TOP[dtype], q), (m / TOP[dtype]).float()


def check_quantized(g, x, dtype, rows=None, q=None):
    count = x.shape[0] if rows is None else rows.shape[0]
    if q is None:
        q = torch.full((count, x.shape[1]), 0x55, dtype=torch.uint8, device="cuda").view(dtype)
    scale = torch.full((count,), float("nan"), device="cuda")
    got = g.quantize_rows(x, q, scale, rows=rows)
    done(g)
    assert got[0] is q and got[1] is scale
    want, want_scale = quantized(x, dtype, rows)
    assert torch.equal(scale, want_scale)
    have = q.double()
    same = (have == want) | (torch.isnan(have) & torch.isnan(want))
    assert same.all(), (torch.nonzero(~same)[:4], have[~same][:4], want[~same][:4])


@pytest.mark.parametrize("dtype", [E4, E5])
@pytest.mark.parametrize("source", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,k", [(1, 1), (3, 7), (5, 16), (2, 8), (1, 8192), (130, 1000), (64, 1024), (7, 20000), (4, 65544), (9, 264), (300, 4096)])
def test_quantize_rows_every_value(g, dtype, source, rows, k):
    x = (torch.randn((rows, k), generator=gen(rows + k), device="cuda") * torch.exp2(torch.randint(-6, 6, (rows, 1), device="cuda", generator=gen(1)).float())).to(source)
    check_quantized(g, x, dtype)


@pytest.mark.parametrize("dtype", [E4, E5])
@pytest.mark.parametrize("source", [torch.bfloat16, torch.float16])
def test_quantize_rows_special_values_and_ties(g, dtype, source):
    inf, nan = float("inf"), float("nan")
    big = torch.finfo(source).max
    tiny = torch.finfo(source).smallest_normal
    k = 512
    x = torch.zeros((10, k), device="cuda")
    x[1, :4] = torch.tensor([inf, -inf, nan, 3.0], device="cuda")             # one finite value decides the scale
    x[2, 5] = nan                                                             # no finite value but zeros
    x[3, :6] = torch.tensor([big, -big, big / 2, 1.0, big / 1024, inf], device="cuda")
    x[4, :5] = torch.tensor([tiny, -tiny / 2, tiny / 128, tiny / 4, 0.0], device="cuda")
    x[5, :k] = torch.arange(k, device="cuda") - 63                            # with 448 as the maximum: every tie of whole numbers
    x[6, :k] = (torch.arange(k, device="cuda") - 63) / 512                    # the same ones, smaller
    x[7, 0], x[7, 1] = 2.0 ** -15, -0.0
    x[8] = inf
    x[9, :] = torch.linspace(-7, 7, k, device="cuda")
    check_quantized(g, x.to(source), dtype)
    # every 16-bit number as a row's member, next to a few maxima
    bits = torch.arange(65536, dtype=torch.int32, device="cuda").to(torch.int16).view(source)
    rows = torch.stack([bits.roll(i) for i in range(3)])
    rows[1] = torch.where(rows[1].abs() <= 448, rows[1], 0.0)
    rows[2] = torch.where(rows[2].abs() <= 1.7, rows[2], 0.0)
    check_quantized(g, rows, dtype)


@pytest.mark.parametrize("dtype", [E4, E5])
@pytest.mark.parametrize("pad", [0, 7])
@pytest.mark.parametrize("exponent", [-80, -79, -76, -70, -30, -1, 0, 1, 100])
def test_quantize_rows_ties_of_small_and_large_rows(g, dtype, pad, exponent):
    """Every BF16 maximum of one exponent with every number down to 2^-34 of it, both ways of reading a row."""
    below = torch.arange((exponent + 127 - 34) << 7, (exponent + 128) << 7, dtype=torch.int32, device="cuda")
    top = below[-128:]
    x = torch.where(below[None] <= top[:, None], below[None], 0).to(torch.int16).view(torch.bfloat16)
    x[:, ::3] = -x[:, ::3]
    check_quantized(g, torch.nn.functional.pad(x, (0, pad)), dtype)


@pytest.mark.parametrize("dtype,source", [(E4, torch.bfloat16), (E5, torch.float16)])
@pytest.mark.parametrize("rows,k", [(1301, 1024), (1301, 1032), (1301, 2048), (1301, 2056), (1301, 3064), (1301, 3080), (1100, 1032), (33, 2056), (33, 4104),
                                    (33, 6144), (33, 6152), (33, 8200), (33, 12288), (33, 12296), (33, 16384)])
def test_quantize_rows_every_form(g, dtype, source, rows, k):
    """Row lengths at both ends of every form, with gathered and padding rows, infinities and NaNs in the first and last pieces."""
    x = torch.randn((rows, k), generator=gen(k), device="cuda").to(source)
    x[3, k - 1], x[4, 0], x[5, k - 8], x[6] = float("inf"), float("nan"), -float("inf"), float("inf")
    check_quantized(g, x, dtype)
    index = torch.randint(0, rows, (rows,), generator=gen(2), device="cuda", dtype=torch.int32)
    index[0], index[-1], index[7:11] = -1, rows, torch.tensor([3, 4, 5, 6], device="cuda")
    buf = torch.full((rows, k + 24), 0x33, dtype=torch.uint8, device="cuda").view(dtype)
    check_quantized(g, x, dtype, index, buf[:, :k])
    assert (bytes_of(buf[:, k:]) == 0x33).all()


def test_quantize_rows_gathers_with_strides_and_padding(g):
    wide = torch.randn((40, 1000), generator=gen(3), device="cuda").to(torch.bfloat16)
    for lo, k in ((0, 512), (8, 512), (3, 512), (16, 333)):
        x = wide[:, lo:lo + k]
        rows = torch.tensor([0, 39, 39, -1, 7, 40, 2 ** 31 - 1, -2 ** 31, 7, 12, 0], dtype=torch.int32, device="cuda")
        for pitch in (k, k + 16, k + 3):
            buf = torch.full((len(rows), pitch), 0x33, dtype=torch.uint8, device="cuda").view(E4)
            check_quantized(g, x, E4, rows, buf[:, :k])
            assert (bytes_of(buf[:, k:]) == 0x33).all()
        check_quantized(g, x, E5)
    empty = torch.empty((0, 64), dtype=torch.bfloat16, device="cuda")
    none = torch.full((3,), -1, dtype=torch.int32, device="cuda")
    check_quantized(g, empty, E4, none)                                       # nothing to take rows from: zeros
    check_quantized(g, torch.empty((4, 0), dtype=torch.float16, device="cuda"), E5)


# ---- products grouped by expert --------------------------------------------------------------------------------------


KERNELS = [0, 1, 2, 3, 7]      # automatic, one CTA with 256-, 128-row tiles, a pair, one CTA with 64-row tiles


SIZES = {
    "one": [1], "few": [3, 0, 1, 17, 0, 40], "skewed": [0, 700, 2, 0, 129, 128, 127, 31, 33, 0, 1, 255], "all_empty": [0, 0, 0],
    "many": [(i * 7) % 19 for i in range(70)], "even": [256, 256, 512],
}


def ends_of(sizes):
    return torch.tensor(np.cumsum(sizes), dtype=torch.int32, device="cuda")


def spans(sizes):
    at = 0
    for e, n in enumerate(sizes):
        yield e, at, at + n
        at += n


def product64(kind, a, b, sizes, d_shape):
    """(sum, sum of magnitudes) of the three products, rows of no group as NaN."""
    t = torch.full(d_shape, float("nan"), dtype=torch.float64, device="cuda")
    s = torch.zeros(d_shape, dtype=torch.float64, device="cuda")
    for e, lo, hi in spans(sizes):
        x = a[lo:hi].double()
        if kind == "wgrad":
            y = b[lo:hi].double()
            t[e], s[e] = x.T @ y, x.abs().T @ y.abs()
        else:
            w = b[e].double().T if kind == "forward" else b[e].double()
            t[lo:hi], s[lo:hi] = x @ w, x.abs() @ w.abs()
    return t, s


def close(got, want, tol, dtype):
    ok = ~torch.isnan(want)
    err = (got.double() - want).abs()
    bound = tol + half_step(dtype) * (want.abs() + tol) + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    bad = ok & ~(err <= bound)
    assert not bad.any(), (int(bad.sum()), torch.nonzero(bad)[:4], got[bad][:4], want[bad][:4], bound[bad][:4])


def steps(k):
    return (k / 32 + 8) * 2.0 ** -23


def operands(kind, sizes, slack, n, k, da, db, seed):
    rows, e = sum(sizes) + slack, len(sizes)
    a = fp8((rows, k if kind == "forward" else n), da, seed)
    b = fp8((rows, k) if kind == "wgrad" else (e, n, k), db, seed + 1)
    shape = {"forward": (rows, n), "dgrad": (rows, k), "wgrad": (e, n, k)}[kind]
    return a, b, shape


def call(g, kind):
    f = {"forward": g.gemm_grouped, "dgrad": g.gemm_grouped_dgrad, "wgrad": g.gemm_grouped_wgrad}[kind]
    # wgrad has no 64-row tiles
    return f if kind != "wgrad" else lambda *args, kernel=0, **kw: f(*args, kernel=0 if kernel == 7 else kernel, **kw)


def deepest(kind, sizes, n, k):
    return {"forward": k, "dgrad": n, "wgrad": max(sizes)}[kind]


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("kind", ["forward", "dgrad", "wgrad"])
@pytest.mark.parametrize("sizes", list(SIZES))
@pytest.mark.parametrize("n,k", [(256, 128), (528, 400), (16, 1040), (1040, 16), (144, 272)])
def test_grouped_products_plain(g, kernel, kind, sizes, n, k):
    sizes, slack = SIZES[sizes], 5
    a, b, shape = operands(kind, sizes, slack, n, k, E5 if kind != "forward" else E4, E4, 7 * n + k)
    d = torch.full(shape, 77.0, device="cuda")
    assert call(g, kind)(a, b, d, ends_of(sizes), kernel=kernel) is d
    done(g)
    t, s = product64(kind, a, b, sizes, shape)
    close(d, t, steps(deepest(kind, sizes, n, k)) * s, torch.float32)
    if kind != "wgrad":
        assert (d[sum(sizes):] == 77.0).all()                # rows of no group are left as they were


@pytest.mark.parametrize("da", [E4, E5])
@pytest.mark.parametrize("db", [E4, E5])
@pytest.mark.parametrize("kind", ["forward", "dgrad", "wgrad"])
@pytest.mark.parametrize("out", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("kernel", KERNELS)
def test_grouped_products_types(g, da, db, kind, out, kernel):
    sizes, n, k = [130, 0, 300, 1], 272, 304
    a, b, shape = operands(kind, sizes, 0, n, k, da, db, 5)
    d = torch.zeros(shape, dtype=out, device="cuda")
    call(g, kind)(a, b, d, ends_of(sizes), alpha=2.0 ** -6, kernel=kernel)
    done(g)
    t, s = product64(kind, a, b, sizes, shape)
    close(d, t / 64, steps(304) * s / 64, out)


@pytest.mark.parametrize("n", [1, 7, 33, 129, 250, 515])
@pytest.mark.parametrize("out", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("kernel", KERNELS)
def test_grouped_forward_takes_any_number_of_columns(g, n, out, kernel):
    sizes, k = [3, 140, 0, 64], 144
    a, b, shape = operands("forward", sizes, 2, n, k, E4, E4, n)
    buf = torch.full((shape[0], n + 3), 9.0, dtype=out, device="cuda")        # a pitch that no fast path takes
    d = buf[:, :n]
    g.gemm_grouped(a, b, d, ends_of(sizes), alpha=0.125, kernel=kernel)
    done(g)
    t, s = product64("forward", a, b, sizes, shape)
    close(d, t / 8, steps(k) * s / 8, out)
    assert (buf[:, n:] == 9.0).all() and (buf[sum(sizes):] == 9.0).all()


@pytest.mark.parametrize("kind", ["forward", "dgrad", "wgrad"])
@pytest.mark.parametrize("kernel", KERNELS)
def test_grouped_products_strides(g, kind, kernel):
    sizes, n, k = [70, 0, 33, 200], 160, 208
    a, b, shape = operands(kind, sizes, 4, n, k, E4, E4, 3)
    def spread(t, pad, more=0):                       # the same values in a buffer with gaps behind rows and matrices
        big = torch.full((*t.shape[:-2], t.shape[-2] + more, t.shape[-1] + pad), 0x7F, dtype=torch.uint8, device="cuda")
        view = big.view(t.dtype)[..., :t.shape[-2], :t.shape[-1]]
        view.copy_(t)
        return view
    a2, b2 = spread(a, 48), spread(b, 32, 3 if kind != "wgrad" else 0)
    buf = torch.full((*shape[:-2], shape[-2] + (2 if kind == "wgrad" else 0), shape[-1] + 8), 5.0, device="cuda")
    d2 = buf[..., :shape[-2], :shape[-1]]
    d = torch.full(shape, 5.0, device="cuda")
    call(g, kind)(a, b, d, ends_of(sizes), kernel=kernel)
    call(g, kind)(a2, b2, d2, ends_of(sizes), kernel=kernel)
    done(g)
    assert torch.equal(d, d2)
    assert (buf[..., shape[-1]:] == 5.0).all() and (buf[..., shape[-2]:, :] == 5.0).all()


def activation64(t, name):
    if name == "relu":
        return t.clamp_min(0)
    if name == "gelu":
        return 0.5 * t * (1 + torch.erf(t / math.sqrt(2)))
    if name == "gelu_tanh":
        return 0.5 * t * (1 + torch.tanh(math.sqrt(2 / math.pi) * (t + 0.044715 * t ** 3)))
    return t


@pytest.mark.parametrize("kind", ["forward", "dgrad"])
@pytest.mark.parametrize("act", ["none", "relu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("out", [torch.float32, torch.bfloat16, E4, E5])
@pytest.mark.parametrize("kernel", KERNELS)
def test_grouped_epilogue(g, kind, act, out, kernel):
    sizes, n, k = [65, 0, 300, 31], 272, 240
    a, b, shape = operands(kind, sizes, 6, n, k, E4, E4, 11)
    rows, cols = shape
    one = lambda v: torch.tensor([v], device="cuda")
    ra = torch.rand(rows, generator=gen(1), device="cuda") + 0.5
    rb = torch.rand((4, cols), generator=gen(2), device="cuda") * 0.01 + 1e-3
    bias = torch.randn((4, cols), generator=gen(3), device="cuda").to(torch.bfloat16)
    old = (torch.randn(shape, generator=gen(4), device="cuda") * 3).to(out)
    d, amax = old.clone(), one(1e9)
    sd = 4.0
    call(g, kind)(a, b, d, ends_of(sizes), alpha=0.5, beta=0.25, a_scale=one(0.5), b_scale=one(0.25), d_scale=one(sd), amax_d=amax, bias=bias,
                  a_row_scale=ra, b_row_scale=rb, activation=act, kernel=kernel)
    done(g)
    t, s = product64(kind, a, b, sizes, shape)
    of = torch.cat([torch.full((hi - lo,), e, device="cuda") for e, lo, hi in spans(sizes)] + [torch.zeros(6, device="cuda")]).long()
    scale = 0.0625 * ra.double()[:, None] * rb.double()[of]
    pre = t * scale + 0.25 * old.double() + bias.double()[of]
    parts = s * scale + 0.25 * old.double().abs() + bias.double()[of].abs()
    want = activation64(pre, act)
    tol = 1.2 * (s * scale * steps(max(n, k)) + 2.0 ** -21 * parts) + (2e-6 * pre.abs() if act.startswith("gelu") else 0)
    if out in TOP:
        lo, hi = (nearest8((sd * (want + sign * tol)), out) for sign in (-1, 1))
        have = d.double()
        good = ((have >= lo) & (have <= hi)) | torch.isnan(want)
        assert good.all(), int((~good).sum())
    else:
        close(d, sd * want, sd * tol, out)
    used = sum(sizes)
    assert torch.equal(bytes_of(d[used:]), bytes_of(old[used:]))
    top = want[:used].abs().max().item()
    assert abs(amax.item() - top) <= tol[:used].max().item() + 2.0 ** -22 * top


@pytest.mark.parametrize("kernel", KERNELS[:4])
@pytest.mark.parametrize("out", [torch.float32, torch.bfloat16])
def test_wgrad_adds_to_what_is_there(g, kernel, out):
    sizes, n, k = [40, 0, 257, 3], 144, 272
    a, b, shape = operands("wgrad", sizes, 9, n, k, E5, E4, 2)
    old = torch.randn(shape, generator=gen(4), device="cuda").to(out)
    one = lambda v: torch.tensor([v], device="cuda")
    d, amax = old.clone(), one(-1.0)
    g.gemm_grouped_wgrad(a, b, d, ends_of(sizes), alpha=0.5, beta=2.0, a_scale=one(0.125), b_scale=one(0.25), d_scale=one(0.5), amax_d=amax, kernel=kernel)
    done(g)
    t, s = product64("wgrad", a, b, sizes, shape)
    f = 0.5 * 0.125 * 0.25
    want = f * t + 2 * old.double()
    tol = f * s * steps(257) + 2.0 ** -21 * (f * s + 2 * old.double().abs())
    close(d, 0.5 * want, 0.5 * tol, out)
    assert abs(amax.item() - want.abs().max().item()) <= tol.max().item()
    assert torch.equal(d[1], old[1])                                          # the empty group: beta * d_scale = 1


@pytest.mark.parametrize("kind", ["forward", "dgrad", "wgrad"])
@pytest.mark.parametrize("kernel", KERNELS)
def test_other_groups_infinities_and_nans_stay_out(g, kind, kernel):
    """Every second group and the rows behind the last one hold NaN and infinities: the other groups' results are those of
    clean operands, bit for bit."""
    sizes, n, k, slack = [33, 5, 127, 128, 1, 64, 31, 300, 95], 272, 144, 40
    a, b, shape = operands(kind, sizes, slack, n, k, E5, E5, 21)
    bad_a, bad_b = a.clone(), b.clone()
    dirty = [(lo, hi) for e, lo, hi in spans(sizes) if e % 2] + [(sum(sizes), sum(sizes) + slack)]
    for i, (lo, hi) in enumerate(dirty):
        bytes_of_view = bad_a.view(torch.uint8)
        bytes_of_view[lo:hi] = (0x7F, 0x7C, 0xFC)[i % 3]                      # NaN, inf, -inf of e5m2
        if kind == "wgrad":
            bad_b.view(torch.uint8)[lo:hi] = (0x7C, 0x7F, 0xFF)[i % 3]
    d, want = torch.zeros(shape, device="cuda"), torch.zeros(shape, device="cuda")
    call(g, kind)(a, b, want, ends_of(sizes), kernel=kernel)
    call(g, kind)(bad_a, bad_b, d, ends_of(sizes), kernel=kernel)
    done(g)
    for e, lo, hi in spans(sizes):
        if e % 2 == 0:
            part = (slice(e, e + 1) if kind == "wgrad" else slice(lo, hi))
            assert torch.equal(d[part], want[part]), e
            assert torch.isfinite(d[part]).all()


@pytest.mark.parametrize("kind", ["forward", "dgrad", "wgrad"])
@pytest.mark.parametrize("kernel", KERNELS[1:])
def test_ends_are_clamped(g, kind, kernel):
    """Ends that fall or leave [0, rows] mean what their clamped running maximum means."""
    rows, n, k = 300, 144, 272
    a, b, shape = operands(kind, [rows - 20, 10, 0, 0, 10], 0, n, k, E4, E4, 4)
    ends = torch.tensor([-5, 120, 60, 2 ** 31 - 1, 250], dtype=torch.int32, device="cuda")
    clean = torch.tensor([0, 120, 120, 300, 300], dtype=torch.int32, device="cuda")
    d, want = torch.full(shape, 3.0, device="cuda"), torch.full(shape, 3.0, device="cuda")
    call(g, kind)(a, b, d, ends, kernel=kernel)
    call(g, kind)(a, b, want, clean, kernel=kernel)
    done(g)
    assert torch.equal(d, want)


def test_grouped_products_without_rows_or_experts(g):
    none = torch.empty(0, dtype=torch.int32, device="cuda")
    g.gemm_grouped(fp8((8, 32), E4, 1), fp8((0, 16, 32), E4, 1), torch.ones(8, 16, device="cuda"), none)
    d = torch.ones(3, 32, 16, device="cuda")
    zero = torch.zeros(3, dtype=torch.int32, device="cuda")
    g.gemm_grouped_wgrad(fp8((0, 32), E4, 1), fp8((0, 16), E4, 1), d, zero)
    done(g)
    assert not d.any()
    g.gemm_grouped(fp8((0, 32), E4, 1), fp8((3, 16, 32), E4, 1), torch.ones(0, 16, device="cuda"), zero)
    done(g)


def test_grouped_forward_is_the_dense_operator_group_by_group(g):
    """The same kernel shape on each group's rows: same sums, same order, same bits."""
    sizes, n, k = [200, 1, 0, 640], 512, 1024
    a, b, shape = operands("forward", sizes, 0, n, k, E4, E4, 6)
    for kernel in (1, 2, 3, 7):
        d = torch.zeros(shape, device="cuda")
        g.gemm_grouped(a, b, d, ends_of(sizes), kernel=kernel)
        for e, lo, hi in spans(sizes):
            if hi > lo:
                want = g.gemm_ex(a[lo:hi], b[e], kernel=kernel)
                assert torch.equal(d[lo:hi], want), (kernel, e)
    done(g)


@pytest.mark.parametrize("kind", ["forward", "dgrad", "wgrad"])
@pytest.mark.parametrize("max_ctas", [1, 3, 40])
def test_grouped_products_do_not_depend_on_the_grid_or_the_run(g, kind, max_ctas):
    """A thousand groups, most of them small or empty, on few CTAs and on all: the same bits every time."""
    rng = np.random.RandomState(5)
    sizes = [int(v) for v in rng.poisson(1.5, 1000) * (rng.rand(1000) < 0.7)]
    sizes[500] = 900
    n, k = 80, 96
    a, b, shape = operands(kind, sizes, 3, n, k, E4, E4, 8)
    want = torch.full(shape, 2.0, dtype=torch.bfloat16, device="cuda")
    call(g, kind)(a, b, want, ends_of(sizes), alpha=0.01)
    for kernel in KERNELS:
        d = torch.full(shape, 2.0, dtype=torch.bfloat16, device="cuda")
        call(g, kind)(a, b, d, ends_of(sizes), alpha=0.01, kernel=kernel, max_ctas=max_ctas)
        assert torch.equal(d, want), kernel
    done(g)
    t, s = product64(kind, a, b, sizes, shape)
    close(want, t * 0.01, steps(900) * s * 0.01 + 2.0 ** -23 * s * 0.01, torch.bfloat16)


@pytest.mark.parametrize("bias_dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("out", [torch.float16, torch.float32, E4])
def test_grouped_bias_types_and_one_vector_at_a_time(g, bias_dtype, out):
    sizes, n, k = [20, 0, 70], 136, 64
    a, b, shape = operands("forward", sizes, 1, n, k, E4, E4, 2)
    bias = torch.randn((3, n), generator=gen(3), device="cuda").to(bias_dtype)
    rb = torch.rand((3, n), generator=gen(2), device="cuda") * 0.001
    t, s = product64("forward", a, b, sizes, shape)
    of = torch.cat([torch.full((hi - lo,), e, device="cuda") for e, lo, hi in spans(sizes)] + [torch.zeros(1, device="cuda")]).long()
    for kw, want, scale in (({"bias": bias}, t / 1024 + bias.double()[of], 1 / 1024), ({"b_row_scale": rb}, t / 1024 * rb.double()[of], rb.double()[of] / 1024)):
        d = torch.zeros(shape, device="cuda").to(out)
        g.gemm_grouped(a, b, d, ends_of(sizes), alpha=1 / 1024, **kw)
        done(g)
        tol = steps(k) * s * scale + 2.0 ** -22 * torch.nan_to_num(want).abs()
        if out in TOP:
            lo, hi = (nearest8(want + sign * tol, out) for sign in (-1, 1))
            have = d.double()
            assert (((have >= lo) & (have <= hi)) | torch.isnan(want)).all()
        else:
            close(d, want, tol, out)


@pytest.mark.parametrize("kind", ["forward", "dgrad", "wgrad"])
@pytest.mark.parametrize("out", [E4, E5])
def test_grouped_8_bit_outputs_are_the_rounded_wide_ones(g, kind, out):
    """Every alignment of an 8-bit output: the bytes are those of the FP32 output rounded, and nothing beside them is written."""
    sizes, n, k = [37, 0, 64, 101], 80, 144
    a, b, shape = operands(kind, sizes, 3, n, k, E5 if kind != "forward" else E4, E4, 5)
    widths = {"forward": (n, n - 4, n - 1, n - 6), "dgrad": (k,), "wgrad": (k,)}[kind]
    for cols in widths:
        w = b[:, :cols].contiguous() if cols != b.shape[1] and kind == "forward" else b
        wide = torch.zeros((*shape[:-1], cols), device="cuda")
        call(g, kind)(a, w, wide, ends_of(sizes), alpha=2.0 ** -4)
        for pitch, at in ((cols, 0), (cols + 8, 4), (cols + 4, 1), (cols + 5, 0)):
            buf = torch.full((*shape[:-1], pitch), 0x33, dtype=torch.uint8, device="cuda")
            d = buf.view(out)[..., at:at + cols]
            call(g, kind)(a, w, d, ends_of(sizes), alpha=2.0 ** -4)
            done(g)
            want = torch.full_like(buf, 0x33)
            rounded = bytes_of(nearest8(wide.double(), out).float().to(out))
            if kind != "wgrad":
                rounded[sum(sizes):] = 0x33
            want[..., at:at + cols] = rounded
            assert torch.equal(buf & 0x7F, want & 0x7F) and torch.equal(buf.view(out).float(), want.view(out).float())


@pytest.mark.parametrize("out", [E4, E5])
def test_wgrad_to_fp8(g, out):
    sizes, n, k = [33, 0, 200], 48, 112
    a, b, shape = operands("wgrad", sizes, 0, n, k, E5, E4, 2)
    d = torch.ones(shape, device="cuda").to(out)
    g.gemm_grouped_wgrad(a, b, d, ends_of(sizes), alpha=2.0 ** -7, d_scale=torch.tensor([0.5], device="cuda"))
    done(g)
    t, s = product64("wgrad", a, b, sizes, shape)
    lo, hi = (nearest8((t + sign * steps(200) * s) * 2.0 ** -8, out) for sign in (-1, 1))
    have = d.double()
    assert ((have >= lo) & (have <= hi)).all()
    assert not d[1].float().any()


@pytest.mark.parametrize("kind", ["dgrad", "wgrad"])
def test_grouped_gradients_against_differences(g, kind):
    """A gradient's elements against the change of a scalar function of the forward product along FP8-exact steps."""
    sizes, n, k = [20, 0, 45, 7], 48, 64
    rows, e = sum(sizes), len(sizes)
    x = torch.randint(-4, 5, (rows, k), generator=gen(1), device="cuda").float()
    w = torch.randint(-4, 5, (e, n, k), generator=gen(2), device="cuda").float()
    dy = torch.randint(-4, 5, (rows, n), generator=gen(3), device="cuda").float()
    ends = ends_of(sizes)

    def loss(x, w):
        d = torch.zeros(rows, n, device="cuda")
        g.gemm_grouped(x.to(E4), w.to(E4), d, ends)
        return (d.double() * dy.double()).sum().item()

    # whole numbers: every product and sum is exact, so the central difference of the bilinear form is exact too
    if kind == "dgrad":
        grad = torch.zeros(rows, k, device="cuda")
        g.gemm_grouped_dgrad(dy.to(E5), w.to(E4), grad, ends)
        for at in ((0, 0), (19, 63), (20, 5), (64, 40), (71, 63)):
            up, down = x.clone(), x.clone()
            up[at] += 1
            down[at] -= 1
            assert grad[at].item() == (loss(up, w) - loss(down, w)) / 2
    else:
        grad = torch.full((e, n, k), float("nan"), device="cuda")
        g.gemm_grouped_wgrad(dy.to(E5), x.to(E4), grad, ends)
        for at in ((0, 0, 0), (0, 47, 63), (1, 3, 3), (2, 10, 20), (3, 47, 0)):
            up, down = w.clone(), w.clone()
            up[at] += 1
            down[at] -= 1
            assert grad[at].item() == (loss(x, up) - loss(x, down)) / 2
    done(g)


@pytest.mark.parametrize("kind", ["forward", "dgrad", "wgrad"])
@pytest.mark.parametrize("out", [torch.float32, torch.bfloat16, torch.float16, E4, E5])
def test_grouped_accumulation_at_every_alignment(g, kind, out):
    """beta * D with rows at any place of a wider buffer: what D held counts once, and nothing beside it changes."""
    sizes, n, k = [37, 0, 64, 101], 144, 160
    a, b, shape = operands(kind, sizes, 3, n, k, E5 if kind != "forward" else E4, E4, 5)
    cols = shape[-1]
    old = torch.randint(-8, 9, shape, generator=gen(7), device="cuda").float().to(out)
    t, s = product64(kind, a, b, sizes, shape)
    want, tol = t / 64 + 0.5 * old.double(), 1.2 * s / 64 * steps(max(n, k)) + 2.0 ** -22 * (s / 64 + old.double().abs())
    if kind != "wgrad":
        want[sum(sizes):] = old[sum(sizes):].double()
    first = None
    for pitch, at in ((cols, 0), (cols + 16, 8), (cols + 5, 3), (cols + 3, 0)):
        buf = torch.full((*shape[:-1], pitch), 3.0, device="cuda").to(out)
        d = buf[..., at:at + cols]
        d.copy_(old)
        call(g, kind)(a, b, d, ends_of(sizes), alpha=1 / 64, beta=0.5)
        done(g)
        if out in TOP:
            lo, hi = (nearest8(want + sign * tol, out) for sign in (-1, 1))
            assert ((d.double() >= lo) & (d.double() <= hi)).all()
        else:
            close(d, want, tol, out)
        first = d.clone() if first is None else first
        assert torch.equal(bytes_of(d), bytes_of(first))
        assert (buf[..., :at].float() == 3.0).all() and (buf[..., at + cols:].float() == 3.0).all()


@pytest.mark.parametrize("out", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n", [1, 17, 33, 129, 250, 515])
def test_grouped_products_of_any_number_of_columns(g, out, n):
    sizes, k = [65, 0, 300, 31, 1], 208
    a, b, shape = operands("forward", sizes, 2, n, k, E4, E4, n)
    buf = torch.full((shape[0] + 1, n), 3.0, device="cuda").to(out)
    d, bias = buf[:-1], torch.randn((5, n), generator=gen(3), device="cuda")
    g.gemm_grouped(a, b, d, ends_of(sizes), alpha=1 / 64, bias=bias)
    done(g)
    t, s = product64("forward", a, b, sizes, shape)
    used = sum(sizes)
    of = torch.cat([torch.full((hi - lo,), e, device="cuda") for e, lo, hi in spans(sizes)]).long()
    want = t[:used] / 64 + bias.double()[of]
    close(d[:used], want, steps(k) * s[:used] / 64 + 2.0 ** -23 * (s[:used] / 64 + bias.double()[of].abs()), out)
    assert (buf[used:].float() == 3.0).all()


def test_grouped_products_without_extent(g):
    """An empty contraction is refused, not skipped; what has no output at all still sets the maximum to zero."""
    ends = ends_of([4, 4])
    e8 = lambda *shape: torch.empty(shape, dtype=torch.uint8, device="cuda").view(E4)
    amax = torch.full((1,), 7.0, device="cuda")
    with pytest.raises(ValueError):
        g.gemm_grouped(e8(8, 0), e8(2, 16, 0), torch.empty((8, 16), device="cuda"), ends)
    with pytest.raises(ValueError):
        g.gemm_grouped_dgrad(e8(8, 0), e8(2, 0, 16), torch.empty((8, 16), device="cuda"), ends)
    g.gemm_grouped(e8(8, 16), e8(2, 0, 16), torch.empty((8, 0), device="cuda"), ends, amax_d=amax)
    assert amax.item() == 0.0
    amax.fill_(7.0)
    g.gemm_grouped(e8(0, 16), e8(2, 16, 16), torch.empty((0, 16), device="cuda"), ends_of([0, 0]), amax_d=amax)
    assert amax.item() == 0.0
    d = torch.full((2, 16, 16), 3.0, device="cuda")
    g.gemm_grouped_wgrad(e8(0, 16), e8(0, 16), d, ends_of([0, 0]), beta=2.0)
    done(g)
    assert (d == 6.0).all()


@pytest.mark.parametrize("stride", [7, -16, 1 << 60])
def test_one_experts_stride_is_not_read(g, stride):
    n, k, rows = 48, 64, 70
    lib, stream = g._cabi.lib(), torch.cuda.current_stream().cuda_stream
    a, b, dy = fp8((rows, k), E4, 1), fp8((1, n, k), E4, 2), fp8((rows, n), E5, 3)
    ends = ends_of([rows])
    y, dx, dw = torch.empty((rows, n), device="cuda"), torch.empty((rows, k), device="cuda"), torch.empty((1, n, k), device="cuda")
    at = lambda t: t.data_ptr()
    assert lib.b200fp8_gemm_grouped(1, rows, k, n, at(ends), at(a), 0, k, at(b), 0, k, stride, at(y), 0, n, None, None, stream) == 0
    assert lib.b200fp8_gemm_grouped_dgrad(1, rows, k, n, at(ends), at(dy), 1, n, at(b), 0, k, stride, at(dx), 0, k, None, None, stream) == 0
    assert lib.b200fp8_gemm_grouped_wgrad(1, rows, k, n, at(ends), at(dy), 1, n, at(a), 0, k, at(dw), 0, k, stride, None, None, stream) == 0
    done(g)
    assert torch.equal(y, g.gemm_grouped(a, b, torch.empty_like(y), ends)) and torch.equal(dx, g.gemm_grouped_dgrad(dy, b, torch.empty_like(dx), ends))
    assert torch.equal(dw, g.gemm_grouped_wgrad(dy, a, torch.empty_like(dw), ends))
    codes, scales, z = weights((1,), n, k, 64, torch.float16, 4, True)
    x = torch.randn((2, k), generator=gen(9), device="cuda").half()
    expert, out = torch.zeros(2, dtype=torch.int32, device="cuda"), torch.empty((2, n), device="cuda")
    assert lib.b200fp8_gemv_w4_experts(2, 2, 1, k, n, 64, at(codes), k // 2, stride, at(scales), 2, 1, stride, at(z), 1, stride, at(expert), at(x), 2, k,
                                       at(out), 0, n, stream) == 0
    done(g)
    assert torch.equal(out, g.gemv_w4_experts(codes, scales, x, torch.empty_like(out), expert, zeros=z))


# ---- 4-bit weights ---------------------------------------------------------------------------------------------------


def weights(lead, n, k, group, x_dtype, seed, zeros):
    codes = torch.randint(0, 256, (*lead, n, k // 2), generator=gen(seed), device="cuda", dtype=torch.uint8)
    scales = (torch.rand((*lead, n, k // group), generator=gen(seed + 1), device="cuda") * 0.1 + 0.01).to(x_dtype)
    z = torch.randint(0, 16, (*lead, n, k // group), generator=gen(seed + 2), device="cuda", dtype=torch.uint8) if zeros else None
    return codes, scales, z


def weights64(codes, scales, zeros):
    q = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).double().unflatten(-1, (scales.shape[-1], -1))
    z = 8.0 if zeros is None else (zeros & 15).double()[..., None]
    return ((q - z) * scales.double()[..., None]).flatten(-2)


def w4_close(y, w, x, k, dtype):
    want, s = x.double() @ w.T, x.double().abs() @ w.abs().T
    # 16 of K per step, plus one FP32 product and sum per group
    close(y, want, (k / 16 + k / 32 + 8) * 2.0 ** -23 * s, dtype)


@pytest.mark.parametrize("x_dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("m", [1, 2, 3, 5, 6, 8, 9, 17, 40])
@pytest.mark.parametrize("n,blocks", [(1, 1), (16, 2), (130, 3), (1000, 8), (515, 17)])
def test_w4_products(g, x_dtype, group, zeros, m, n, blocks):
    k = group * blocks
    codes, scales, z = weights((), n, k, group, x_dtype, n + m, zeros)
    x = torch.randn((m, k), generator=gen(9), device="cuda").to(x_dtype)
    for y_dtype in (x_dtype, torch.float32):
        y = torch.full((m, n), float("nan"), dtype=y_dtype, device="cuda")
        assert g.gemv_w4(codes, scales, x, y, zeros=z) is y
        done(g)
        w4_close(y, weights64(codes, scales, z), x, k, y_dtype)


@pytest.mark.parametrize("scale_dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n,k,group,m", [(8192, 8192, 128, 1), (4100, 14336, 64, 8), (300, 32768, 128, 3), (28672, 1024, 32, 2)])
def test_w4_products_of_real_size(g, scale_dtype, n, k, group, m):
    codes, scales, z = weights((), n, k, group, scale_dtype, 3, True)
    x = torch.randn((m, k), generator=gen(9), device="cuda").to(torch.bfloat16)
    y = torch.empty((m, n), device="cuda")
    g.gemv_w4(codes, scales, x, y, zeros=z)
    done(g)
    w4_close(y, weights64(codes, scales, z), x, k, torch.float32)


def test_w4_strides_and_canaries(g):
    n, k, group, m = 133, 384, 64, 5
    codes, scales, z = weights((), n, k, group, torch.float16, 1, True)
    x = torch.randn((m, k), generator=gen(9), device="cuda").half()
    def wide(t, pad):
        big = torch.full((t.shape[0], t.shape[1] + pad), 127, dtype=torch.uint8, device="cuda").to(t.dtype) if t.dtype != torch.uint8 else \
            torch.full((t.shape[0], t.shape[1] + pad), 0xFF, dtype=torch.uint8, device="cuda")
        big[:, :t.shape[1]] = t
        return big[:, :t.shape[1]]
    xs = wide(x, 8)
    xs._base[:, k:] = float("nan")
    buf = torch.full((m, n + 5), 9.0, dtype=torch.float16, device="cuda")
    g.gemv_w4(wide(codes, 16), wide(scales, 3), xs, buf[:, :n], zeros=wide(z, 5))
    done(g)
    w4_close(buf[:, :n], weights64(codes, scales, z), x, k, torch.float16)
    assert (buf[:, n:] == 9.0).all()


def test_w4_special_values(g):
    """Codes and zero points at their ends are exact; an infinity or NaN in one vector stays in its row of y."""
    n, k, group = 32, 256, 32
    codes = torch.full((n, k // 2), 0xFF, dtype=torch.uint8, device="cuda")
    codes[1::2] = 0x00
    z = torch.full((n, k // group), 0xF0, dtype=torch.uint8, device="cuda")   # only the low four bits count
    scales = torch.ones((n, k // group), dtype=torch.float16, device="cuda")
    x = torch.ones((3, k), dtype=torch.float16, device="cuda")
    x[1, 7], x[2, 255] = float("inf"), float("nan")
    y = torch.zeros((3, n), dtype=torch.float32, device="cuda")
    g.gemv_w4(codes, scales, x, y, zeros=z)
    done(g)
    assert (y[0, ::2] == 15.0 * k).all() and (y[0, 1::2] == 0).all()
    assert torch.isinf(y[1, ::2]).all() and torch.isnan(y[2]).all()


@pytest.mark.parametrize("x_dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m", [1, 4, 7])
def test_w4_infinities_and_nans_add_what_their_weights_say(g, x_dtype, m):
    """inf and NaN in x times a weight of either sign or zero, in several vectors and blocks of K."""
    n, k, group = 48, 2304, 64
    codes, scales, z = weights((), n, k, group, torch.float16, 1, True)
    x = torch.randn((m, k), generator=gen(9), device="cuda").to(x_dtype)
    inf = float("inf")
    x[0, 3], x[m - 1, 2303] = inf, -inf
    x[m // 2, 700] = inf
    y = torch.zeros((m, n), device="cuda")
    g.gemv_w4(codes, scales, x, y, zeros=z)
    done(g)
    w = weights64(codes, scales, z)
    want = (x.double()[:, None, :] * w[None]).sum(-1)
    assert torch.equal(torch.isnan(y), torch.isnan(want)) and torch.equal(torch.isinf(y), torch.isinf(want))
    assert torch.equal(torch.sign(y[torch.isinf(y)]).double(), torch.sign(want[torch.isinf(want)]))


@pytest.mark.parametrize("x_dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m", [1, 5, 8])
def test_w4_vectors_of_any_size(g, x_dtype, m):
    """Very large, very small and very uneven vectors: the scaling per vector and 256 of K loses nothing that FP32 sums keep."""
    n, k, group = 64, 1024, 32
    codes, scales, z = weights((), n, k, group, torch.float32, 1, True)
    x = torch.randn((m, k), generator=gen(9), device="cuda").double()
    e = 100.0 if x_dtype == torch.bfloat16 else 12.0
    x *= torch.exp2(torch.linspace(-e, e, m, device="cuda").double().round())[:, None] if m > 1 else 2.0 ** e
    x[:, 256:512] *= 2.0 ** -20
    x[:, 512:768] = 0
    x = x.to(x_dtype)
    y = torch.zeros((m, n), device="cuda")
    g.gemv_w4(codes, scales, x, y, zeros=z)
    done(g)
    w, v = weights64(codes, scales, z), x.double()
    # on top of the sums' bound, a scaled element is off by at most 2^-23 of the largest of its 256: FP16's subnormals by far
    # less, the integers' last bit by half of it
    blocks = v.abs().unflatten(1, (-1, 256)).amax(-1, keepdim=True).expand(-1, -1, 256).flatten(1)
    s = v.abs() @ w.abs().T
    tol = (k / 16 + k / 32 + 8) * 2.0 ** -23 * s + 2.0 ** -23 * (blocks @ w.abs().T)
    close(y, v @ w.T, tol, torch.float32)


@pytest.mark.parametrize("x_dtype,outliers", [(torch.float16, (1e3, 6e4)), (torch.bfloat16, (1e3, 6e4, 2.0 ** 20, 2.0 ** 60, 2.0 ** 120))])
@pytest.mark.parametrize("group,zeros", [(32, True), (64, False), (128, True)])
@pytest.mark.parametrize("m,n,k", [(1, 64, 4096), (2, 64, 4096), (3, 64, 4096), (8, 64, 4096), (16, 64, 4096), (1, 20001, 8320), (2, 20001, 8320)])
def test_w4_small_numbers_beside_a_large_one(g, x_dtype, outliers, group, zeros, m, n, k):
    """One large element among small ones, with a weight of zero in every second row: the row's sum is that of the small ones."""
    codes, scales, z = weights((), n, k, group, torch.float32, 1, zeros)
    x = torch.randn((m, k), generator=gen(9), device="cuda") * 0.01
    for i, size in enumerate(outliers):
        at = 700 * i + 37
        x[i % min(m, 2)::2, at] = size                                        # every second vector
        none = 8 if z is None else z[::2, at // group]
        codes[::2, at // 2] = codes[::2, at // 2] & 15 | none << 4            # odd places: the high half
    x = x.to(x_dtype)
    w = weights64(codes, scales, z)
    y = torch.full((m, n), float("nan"), device="cuda")
    g.gemv_w4(codes, scales, x, y, zeros=z)
    done(g)
    w4_close(y, w, x, k, torch.float32)
    if n > 64:
        return
    # by expert, every token with two of four
    ids = torch.tensor([(3 * t + j) % 4 for t in range(m) for j in range(2)], dtype=torch.int32, device="cuda")
    four = lambda t: None if t is None else torch.stack([t] * 4)
    y2 = torch.full((2 * m, n), float("nan"), device="cuda")
    g.gemv_w4_experts(four(codes), four(scales), x, y2, ids, zeros=four(z))
    done(g)
    w4_close(y2, w, x.repeat_interleave(2, 0), k, torch.float32)


@pytest.mark.parametrize("x_dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("scale_dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("group,zeros", [(32, False), (64, True), (128, False), (128, True)])
@pytest.mark.parametrize("m", [1, 2])
@pytest.mark.parametrize("n,k", [(4100, 8320), (515, 65664), (40001, 896)])
def test_w4_one_or_two_vectors_of_large_weights(g, x_dtype, scale_dtype, group, zeros, m, n, k):
    """Sizes beyond the border to the integer form, with odd ends of N and K and every spread of x: blocks of whole numbers, of wide
    range, of zeros, of subnormal numbers, beside an infinity and a NaN in rows of their own further down."""
    codes, scales, z = weights((), n, k, group, scale_dtype, 2, zeros)
    x = torch.randn((m, k), generator=gen(9), device="cuda")
    x[:, 256:300] *= 1e-7                                                     # more than FP16 or 30 bits hold
    x[:, 300:330] = 0
    x[-1, 512:768] = 0
    x[0, 800:1024 if k > 900 else 896] *= 2.0 ** (-24 if x_dtype == torch.float16 else -133)
    x = x.to(x_dtype)
    w = weights64(codes, scales, z)
    for y_dtype in (x_dtype, torch.float32):
        y = torch.full((m, n), float("nan"), dtype=y_dtype, device="cuda")
        g.gemv_w4(codes, scales, x, y, zeros=z)
        done(g)
        w4_close(y, w, x, k, y_dtype)
    first = y.clone()
    g.gemv_w4(codes, scales, x, y, zeros=z)
    assert torch.equal(y, first)
    x[0, 5], x[0, k - 1], x[m - 1, 520] = float("inf"), float("inf"), -float("inf") if m == 1 else float("nan")
    g.gemv_w4(codes, scales, x, y, zeros=z)
    done(g)
    want = torch.stack([(row * w[:, [5, 520, k - 1]]).sum(-1) for row in x.double()[:, [5, 520, k - 1]]])
    assert torch.equal(torch.isnan(y), torch.isnan(want)) and torch.equal(torch.isinf(y), torch.isinf(want))
    assert torch.equal(torch.sign(y[torch.isinf(y)]).double(), torch.sign(want[torch.isinf(want)]))


def test_w4_of_large_weights_replayed_on_two_streams(g):
    """Two captured calls at once, replayed with other vectors than the captured ones: narrow, wide in some blocks, infinite."""
    n, k, group = 4100, 8320, 64
    graphs, streams, states = [], [torch.cuda.Stream() for _ in range(2)], []
    for i, stream in enumerate(streams):
        codes, scales, z = weights((), n, k, group, torch.float16, 5 + i, True)
        x, y = torch.ones((1 + i, k), dtype=torch.bfloat16, device="cuda"), torch.empty((1 + i, n), device="cuda")
        g.gemv_w4(codes, scales, x, y, zeros=z)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            for _ in range(20):
                g.gemv_w4(codes, scales, x, y, zeros=z)
        graphs.append(graph)
        states.append((codes, scales, z, x, y))
    for at, value in ((0, 0.0), (300, 1e6), (5000, 1e30), (77, float("inf"))):
        for i, (codes, scales, z, x, y) in enumerate(states):
            x.copy_(torch.randn(x.shape, generator=gen(at + i), device="cuda"))
            x[-1, at] = value
            y.fill_(float("nan"))
        torch.cuda.synchronize()
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        done(g)
        for codes, scales, z, x, y in states:
            w = weights64(codes, scales, z)
            if math.isinf(value):
                assert not torch.isfinite(y[-1]).any()
                x, y = x[:-1], y[:-1]
            w4_close(y, w, x, k, torch.float32)


@pytest.mark.parametrize("x_dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("group,zeros", [(64, True), (128, False)])
@pytest.mark.parametrize("tokens,top_k,experts,n,k", [(1, 8, 9, 1000, 8320), (2, 4, 40, 515, 8320), (2, 12, 3, 700, 32896)])
def test_w4_by_expert_of_large_weights(g, x_dtype, group, zeros, tokens, top_k, experts, n, k):
    """One or two tokens beyond the border to the integer form: several rows of one expert, padding rows, strided weights."""
    rows = tokens * top_k
    codes, scales, z = weights((experts,), n, k, group, torch.float16, n, zeros)
    wide = torch.full((experts, n + 1, k // 2 + 16), 255, dtype=torch.uint8, device="cuda")
    wide[:, :n, :k // 2] = codes
    x = torch.randn((tokens, k), generator=gen(9), device="cuda")
    x[0, 300] = 3e4                                                           # a block as floats
    x = x.to(x_dtype)
    expert = torch.randint(0, experts, (rows,), generator=gen(5), device="cuda", dtype=torch.int32)
    expert[1], expert[3], expert[4] = -1, expert[2], expert[2]
    buf = torch.full((rows, n + 3), 5.0, device="cuda")
    y = buf[:, :n]
    g.gemv_w4_experts(wide[:, :n, :k // 2], scales, x, y, expert, zeros=z)
    done(g)
    assert (buf[:, n:] == 5.0).all() and (buf[1] == 5.0).all()
    for r, e in enumerate(expert.tolist()):
        if e >= 0:
            w4_close(y[r:r + 1], weights64(codes[e], scales[e], None if z is None else z[e]), x[r // top_k:r // top_k + 1], k, torch.float32)


@pytest.mark.parametrize("x_dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("group,zeros", [(32, True), (64, False), (128, True)])
@pytest.mark.parametrize("tokens,top_k,experts,n,blocks", [(1, 1, 1, 16, 1), (1, 4, 64, 1000, 4), (16, 8, 64, 130, 3), (5, 2, 3, 515, 2), (33, 2, 2, 64, 2),
                                                           (128, 1, 40, 33, 1), (3, 1, 1000, 48, 2)])
def test_w4_by_expert(g, x_dtype, group, zeros, tokens, top_k, experts, n, blocks):
    k, rows = group * blocks, tokens * top_k
    codes, scales, z = weights((experts,), n, k, group, x_dtype, n, zeros)
    x = torch.randn((tokens, k), generator=gen(9), device="cuda").to(x_dtype)
    expert = torch.randint(0, experts, (rows,), generator=gen(5), device="cuda", dtype=torch.int32)
    if rows > 3:                                              # padding rows, and one expert for all the rest of a few
        expert[1], expert[2], expert[-1] = -1, experts, 2 ** 31 - 1
    y = torch.full((rows, n), 5.0, dtype=x_dtype, device="cuda")
    assert g.gemv_w4_experts(codes, scales, x, y, expert, zeros=z) is y
    done(g)
    for r, e in enumerate(expert.tolist()):
        if 0 <= e < experts:
            w4_close(y[r:r + 1], weights64(codes[e], scales[e], None if z is None else z[e]), x[r // top_k:r // top_k + 1], k, x_dtype)
        else:
            assert (y[r] == 5.0).all()


@pytest.mark.parametrize("x_dtype,scale_dtype", [(torch.bfloat16, torch.float32), (torch.float16, torch.float16)])
@pytest.mark.parametrize("group,zeros", [(32, True), (64, False), (128, True)])
@pytest.mark.parametrize("experts,n,k", [(64, 700, 1408), (64, 1000, 256), (160, 17, 640)])
def test_w4_by_expert_with_more_blocks_than_fit(g, x_dtype, scale_dtype, group, zeros, experts, n, k):
    """The form with 32 rows per warp: with K parted and whole, experts with more than eight rows, odd ends of N and K."""
    tokens, top_k = 20, 8
    rows = tokens * top_k
    codes, scales, z = weights((experts,), n, k, group, scale_dtype, n, zeros)
    x = torch.randn((tokens, k), generator=gen(9), device="cuda").to(x_dtype)
    x[3, 7], x[4] = float("inf"), 0.0
    expert = torch.randint(0, experts, (rows,), generator=gen(5), device="cuda", dtype=torch.int32)
    expert[5::14], expert[2] = 3, -1                          # a dozen for one expert, and a padding row
    y = torch.full((rows, n), 5.0, dtype=x_dtype, device="cuda")
    g.gemv_w4_experts(codes, scales, x, y, expert, zeros=z)
    done(g)
    for r, e in enumerate(expert.tolist()):
        if e < 0:
            assert (y[r] == 5.0).all()
        elif r // top_k == 3:                                 # infinity times a weight: its sign, or NaN for a weight of zero
            assert torch.equal(torch.nan_to_num(y[r].double(), nan=9.0, posinf=1.0, neginf=-1.0),
                               torch.nan_to_num(x[3, 7].double() * weights64(codes[e], scales[e], None if z is None else z[e])[:, 7], nan=9.0, posinf=1.0, neginf=-1.0))
        else:
            w4_close(y[r:r + 1], weights64(codes[e], scales[e], None if z is None else z[e]), x[r // top_k:r // top_k + 1], k, x_dtype)


@pytest.mark.parametrize("m", [4, 8])
def test_w4_of_many_outputs(g, m):
    n, k, group = 40001, 320, 64
    codes, scales, z = weights((), n, k, group, torch.bfloat16, 3, True)
    x = torch.randn((m, k), generator=gen(9), device="cuda").half()
    y = torch.empty((m, n), device="cuda")
    g.gemv_w4(codes, scales, x, y, zeros=z)
    done(g)
    w4_close(y, weights64(codes, scales, z), x, k, torch.float32)


@pytest.mark.parametrize("tokens", [1, 3, 20])
def test_w4_by_expert_strides_and_repeats(g, tokens):
    """Experts' matrices inside wider buffers; a token that names one expert twice; the same bits on every run."""
    experts, n, k, group, top_k = 5, 70, 512, 64, 3
    codes, scales, z = weights((experts,), n, k, group, torch.float32, 4, True)
    def wide(t, rows, cols):
        big = torch.full((experts, n + rows, t.shape[-1] + cols), 255, dtype=torch.uint8, device="cuda").to(t.dtype)
        big[:, :n, :t.shape[-1]] = t
        return big[:, :n, :t.shape[-1]]
    x = torch.randn((tokens, k), generator=gen(9), device="cuda").half()
    expert = torch.randint(0, experts, (tokens * top_k,), generator=gen(5), device="cuda", dtype=torch.int32)
    expert[1] = expert[0]
    buf = torch.full((tokens * top_k, n + 2), 5.0, dtype=torch.float16, device="cuda")
    y = buf[:, :n]
    g.gemv_w4_experts(wide(codes, 2, 16), wide(scales, 1, 3), x, y, expert, zeros=wide(z, 3, 5))
    first = y.clone()
    for _ in range(5):
        g.gemv_w4_experts(codes, scales, x, y, expert, zeros=z)
        assert torch.equal(y, first)
    done(g)
    assert torch.equal(y[0], y[1]) and (buf[:, n:] == 5.0).all()
    for r, e in enumerate(expert.tolist()):
        w4_close(y[r:r + 1], weights64(codes[e], scales[e], z[e]), x[r // top_k:r // top_k + 1], k, torch.float16)


def test_w4_by_expert_at_its_limits(g):
    tokens, experts, n, k, group = 4096, 4096, 16, 32, 32
    codes, scales, _ = weights((experts,), n, k, group, torch.float16, 1, False)
    x = torch.randn((tokens, k), generator=gen(9), device="cuda").half()
    w = weights64(codes, scales, None)
    for expert in (torch.arange(tokens, device="cuda").flip(0), torch.full((tokens,), 4095, device="cuda"), torch.full((tokens,), -1, device="cuda")):
        y = torch.full((tokens, n), 5.0, device="cuda")
        g.gemv_w4_experts(codes, scales, x, y, expert.to(torch.int32))
        done(g)
        if expert[0] < 0:
            assert (y == 5.0).all()
        else:
            want = torch.einsum("tnk,tk->tn", w[expert], x.double())
            s = torch.einsum("tnk,tk->tn", w[expert].abs(), x.double().abs())
            close(y, want, 11 * 2.0 ** -23 * s, torch.float32)


# ---- together, as a layer ------------------------------------------------------------------------------------------------


def route(tokens, top_k, experts, seed):
    """Token rows in expert order: (source rows, ends, expert of each row)."""
    chosen = torch.rand((tokens, experts), generator=gen(seed), device="cuda").topk(top_k, dim=1).indices.reshape(-1)
    order = torch.argsort(chosen, stable=True)
    ends = torch.cumsum(torch.bincount(chosen, minlength=experts), 0).to(torch.int32)
    return (order // top_k).to(torch.int32), ends, chosen[order].to(torch.int32), chosen, order


def layer(g, x, w1, w2, s1, s2, rows, ends, bufs):
    q1, a1, h, q2, a2, y = bufs
    g.quantize_rows(x, q1, a1, rows=rows)
    g.gemm_grouped(q1, w1, h, ends, a_row_scale=a1, b_row_scale=s1, activation="gelu_tanh")
    g.quantize_rows(h, q2, a2)
    g.gemm_grouped(q2, w2, y, ends, a_row_scale=a2, b_row_scale=s2)
    return y


def layer_buffers(rows, hidden, inner):
    return (torch.empty((rows, hidden), dtype=torch.uint8, device="cuda").view(E4), torch.empty(rows, device="cuda"),
            torch.empty((rows, inner), dtype=torch.bfloat16, device="cuda"), torch.empty((rows, inner), dtype=torch.uint8, device="cuda").view(E4),
            torch.empty(rows, device="cuda"), torch.empty((rows, hidden), dtype=torch.bfloat16, device="cuda"))


@pytest.mark.parametrize("tokens", [1, 5, 64, 700])
def test_expert_layer_runs_together_and_in_a_graph(g, tokens):
    hidden, inner, experts, top_k = 512, 768, 6, 2
    w1, w2 = fp8((experts, inner, hidden), E4, 1), fp8((experts, hidden, inner), E4, 2)
    s1, s2 = (torch.full((experts, n), 0.002, device="cuda") for n in (inner, hidden))
    x = torch.randn((tokens, hidden), generator=gen(3), device="cuda").to(torch.bfloat16)
    rows, ends, of_row, _, _ = route(tokens, top_k, experts, 4)
    bufs = layer_buffers(tokens * top_k, hidden, inner)
    y = layer(g, x, w1, w2, s1, s2, rows, ends, bufs).clone()
    done(g)
    # step by step in 64 bits from the stored intermediate values, so that each tolerance is one operator's
    q1, a1, h, q2, a2, _ = bufs
    want, _ = quantized(x, E4, rows)
    assert torch.equal(q1.double(), want)
    for e in range(experts):
        mine = of_row == e
        t, s = q1[mine].double() @ w1[e].double().T * a1[mine].double()[:, None] * 0.002, None
        s = (q1[mine].double().abs() @ w1[e].double().abs().T) * a1[mine].double()[:, None] * 0.002
        close(h[mine], activation64(t, "gelu_tanh"), 1.2 * s * (steps(hidden) + 2.0 ** -21) + 2e-6 * t.abs(), torch.bfloat16)
        t = q2[mine].double() @ w2[e].double().T * a2[mine].double()[:, None] * 0.002
        s = (q2[mine].double().abs() @ w2[e].double().abs().T) * a2[mine].double()[:, None] * 0.002
        close(y[mine], t, s * (steps(inner) + 2.0 ** -21), torch.bfloat16)
    assert torch.equal(q2.double(), quantized(h, E4)[0])
    # captured once, replayed with other tokens and another routing written into the same tensors
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        layer(g, x, w1, w2, s1, s2, rows, ends, bufs)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(bufs[-1], y)
    x2 = torch.randn((tokens, hidden), generator=gen(30), device="cuda").to(torch.bfloat16)
    rows2, ends2, _, _, _ = route(tokens, top_k, experts, 40)
    x.copy_(x2), rows.copy_(rows2), ends.copy_(ends2)
    graph.replay()
    torch.cuda.synchronize()
    eager = layer(g, x2, w1, w2, s1, s2, rows2, ends2, layer_buffers(tokens * top_k, hidden, inner))
    done(g)
    assert torch.equal(bufs[-1], eager)


def test_training_step_of_a_layer(g):
    """Forward, both gradients: the three products share the FP8 tensors; gradients against 64 bits from the same tensors."""
    hidden, inner, experts, tokens = 256, 384, 5, 333
    rows, ends, of_row, _, _ = route(tokens, 2, experts, 6)
    count = tokens * 2
    x8, dy8 = fp8((count, hidden), E4, 1), fp8((count, inner), E5, 2)
    w = fp8((experts, inner, hidden), E4, 3)
    sx, sdy = torch.tensor([0.01], device="cuda"), torch.tensor([0.003], device="cuda")
    y = torch.zeros((count, inner), device="cuda")
    dx, dw = torch.zeros((count, hidden), device="cuda"), torch.ones((experts, inner, hidden), device="cuda")
    g.gemm_grouped(x8, w, y, ends, a_scale=sx)
    g.gemm_grouped_dgrad(dy8, w, dx, ends, a_scale=sdy)
    g.gemm_grouped_wgrad(dy8, x8, dw, ends, a_scale=sdy, b_scale=sx, beta=1.0)
    done(g)
    sizes = torch.diff(ends, prepend=ends.new_zeros(1)).tolist()
    for kind, got, a, b, f, old in (("forward", y, x8, w, sx, 0), ("dgrad", dx, dy8, w, sdy, 0), ("wgrad", dw, dy8, x8, sx.double() * sdy.double(), 1)):
        t, s = product64(kind, a, b, sizes, got.shape)
        f = f.double()
        close(got, t * f + old, (steps(max(hidden, inner, max(sizes))) + 2.0 ** -21) * s * f + 2.0 ** -22, torch.float32)


def test_documented_training_step_with_scales_of_rows_and_columns(g):
    """The lines that the integration guide gives, run as they stand: gradients of the product with a scale per row and per
    output channel.  dq * dq_scale is within half an E5M2 step (2^-3 of the value, at least 2^-17 of the scale) and a BF16
    rounding (2^-8, here 2^-7 with the products of both) of dh * w1_scale; dr without the latter; the sums add FP32's roundings."""
    text = open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "INTEGRATION.md")).read()
    lines = text[text.index("# a layer of experts"):text.index("# few tokens")]
    hidden, inner, experts, tokens = 256, 320, 5, 300
    source_row, ends, expert_of_row, _, _ = route(tokens, 2, experts, 6)
    rows, expert_of_row = 2 * tokens, expert_of_row.long()
    power = lambda shape, seed: torch.exp2(torch.randint(-4, 5, shape, generator=gen(seed), device="cuda").float())
    x = (torch.randn((tokens, hidden), generator=gen(1), device="cuda") * power((tokens, 1), 2)).to(torch.bfloat16)
    w1, w1_scale = fp8((experts, inner, hidden), E4, 3), power((experts, inner), 4) * (1 / 48 + torch.rand((experts, inner), generator=gen(5), device="cuda") / 48)
    b1 = torch.zeros((experts, inner), device="cuda")
    q, row_scale = torch.empty((rows, hidden), dtype=torch.uint8, device="cuda").view(E4), torch.empty(rows, device="cuda")
    h, dh = torch.empty((rows, inner), dtype=torch.bfloat16, device="cuda"), torch.randn((rows, inner), generator=gen(7), device="cuda").to(torch.bfloat16)
    dq, dq_scale = torch.empty((rows, inner), dtype=torch.uint8, device="cuda").view(E5), torch.empty(rows, device="cuda")
    dx, dw1 = torch.empty((rows, hidden), device="cuda"), torch.empty((experts, inner, hidden), device="cuda")
    names = dict(locals(), torch=torch)
    exec(lines, names)
    done(g)
    real_w = w1.double() * w1_scale.double()[..., None]
    real_x = q.double() * row_scale.double()[:, None]
    for e, lo, hi in spans(torch.diff(ends, prepend=ends.new_zeros(1)).tolist()):
        grad = dh[lo:hi].double()
        folded = grad * w1_scale[e].double()
        off = (2.0 ** -3 + 2.0 ** -7) * folded.abs() + 2.0 ** -17 * dq_scale[lo:hi, None].double()
        want, s = grad @ real_w[e], folded.abs() @ w1[e].double().abs()
        assert ((dx[lo:hi].double() - want).abs() <= off @ w1[e].double().abs() + 2 * (steps(inner) + 2.0 ** -21) * s).all()
        folded = grad * row_scale[lo:hi, None].double()
        off = (2.0 ** -3 + 2.0 ** -20) * folded.abs() + 2.0 ** -17 * names["dr_scale"].double()
        want, s = grad.T @ real_x[lo:hi], folded.abs().T @ q[lo:hi].double().abs()
        assert ((dw1[e].double() - want).abs() <= off.T @ q[lo:hi].double().abs() + 2 * (steps(hi - lo) + 2.0 ** -21) * s).all()


@pytest.mark.parametrize("tokens", [1, 6])
def test_decode_step_with_four_bit_experts(g, tokens):
    hidden, inner, experts, top_k = 512, 640, 16, 4
    c1, s1, z1 = weights((experts,), inner, hidden, 64, torch.bfloat16, 1, True)
    c2, s2, _ = weights((experts,), hidden, inner, 128, torch.bfloat16, 2, False)
    x = torch.randn((tokens, hidden), generator=gen(3), device="cuda").to(torch.bfloat16)
    _, _, _, chosen, _ = route(tokens, top_k, experts, 8)
    expert = chosen.to(torch.int32)
    h = torch.empty((tokens * top_k, inner), dtype=torch.bfloat16, device="cuda")
    y = torch.empty((tokens * top_k, hidden), dtype=torch.bfloat16, device="cuda")

    def step():
        g.gemv_w4_experts(c1, s1, x, h, expert, zeros=z1)
        g.gemv_w4_experts(c2, s2, h, y, expert)

    step()
    done(g)
    for r, e in enumerate(expert.tolist()):
        w4_close(h[r:r + 1], weights64(c1[e], s1[e], z1[e]), x[r // top_k:r // top_k + 1], hidden, torch.bfloat16)
        w4_close(y[r:r + 1], weights64(c2[e], s2[e], None), h[r:r + 1], inner, torch.bfloat16)
    first = y.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    y.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, first)


def test_two_streams_at_once(g):
    """The same operators on two streams together: nothing is shared between calls."""
    sizes, n, k = [500, 3, 0, 900], 512, 512
    a, b, shape = operands("forward", sizes, 0, n, k, E4, E4, 1)
    ends = ends_of(sizes)
    codes, scales, _ = weights((), 4096, 2048, 128, torch.bfloat16, 1, False)
    x = torch.randn((2, 2048), generator=gen(1), device="cuda").to(torch.bfloat16)
    want, want_w, want_y = torch.zeros(shape, device="cuda"), torch.zeros((4, n, k), device="cuda"), torch.zeros((2, 4096), device="cuda")
    dy = fp8((sum(sizes), n), E5, 3)
    g.gemm_grouped(a, b, want, ends)
    g.gemm_grouped_wgrad(dy, a, want_w, ends)
    g.gemv_w4(codes, scales, x, want_y)
    done(g)
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for _ in range(6):
        for s in streams:
            with torch.cuda.stream(s):
                d, w, y = torch.zeros(shape, device="cuda"), torch.zeros((4, n, k), device="cuda"), torch.zeros((2, 4096), device="cuda")
                g.gemm_grouped(a, b, d, ends)
                g.gemm_grouped_wgrad(dy, a, w, ends)
                g.gemv_w4(codes, scales, x, y)
                outs.append((d, w, y))
    done(g)
    for d, w, y in outs:
        assert torch.equal(d, want) and torch.equal(w, want_w) and torch.equal(y, want_y)


def test_offsets_beyond_32_bits(g):
    """Weights of more than 2^31 elements: the last expert's matrix is reached by 64-bit offsets."""
    experts, n, k = 40, 8192, 8192
    b = torch.zeros((experts, n, k), dtype=torch.uint8, device="cuda").view(E4)
    b[-1] = fp8((n, k), E4, 1)
    a = fp8((3, k), E4, 2)
    ends = torch.tensor([0] * (experts - 1) + [3], dtype=torch.int32, device="cuda")
    d = torch.zeros((3, n), device="cuda")
    g.gemm_grouped(a, b, d, ends)
    dx = torch.zeros((3, k), device="cuda")
    dy = fp8((3, n), E5, 3)
    g.gemm_grouped_dgrad(dy, b, dx, ends)
    done(g)
    for kind, got, left in (("forward", d, a), ("dgrad", dx, dy)):
        w = b[-1].double()
        w = w.T if kind == "forward" else w
        close(got, left.double() @ w, steps(8192) * (left.double().abs() @ w.abs()), torch.float32)
    del b
    codes = torch.zeros((160, n, k // 2), dtype=torch.uint8, device="cuda")
    codes[-1] = torch.randint(0, 256, (n, k // 2), generator=gen(5), device="cuda", dtype=torch.uint8)
    scales = torch.ones((160, n, k // 128), dtype=torch.bfloat16, device="cuda")
    x = torch.randn((1, k), generator=gen(6), device="cuda").to(torch.bfloat16)
    y = torch.zeros((1, n), device="cuda")
    g.gemv_w4_experts(codes, scales, x, y, torch.tensor([159], dtype=torch.int32, device="cuda"))
    done(g)
    w4_close(y, weights64(codes[-1], scales[-1], None), x, k, torch.float32)


# ---- a wait that runs out ---------------------------------------------------------------------------------------------


CHILD = r"""
import sys, time
sys.path[:0] = [%r, %r]
import torch
import test_experts_gpu as T
from __graft_entry__ import load_package
g = load_package().gemm
torch.cuda.set_device(0)


def run(k):
    a, b, shape = T.operands("forward", [300, 700], 0, 512, k, T.E4, T.E4, 1)
    ends = T.ends_of([300, 700])
    for kernel in (2, 3):
        yield lambda: g.gemm_grouped(a, b, torch.zeros(shape, device="cuda"), ends, kernel=kernel), (101, 102, 103)
    # wgrad contracts over the rows: 300 and 700 of them, or 100 and 200 where no block may be left out
    few = T.ends_of([300, 700] if k > 256 else [100, 200])
    for kernel in (1, 3):
        yield lambda: g.gemm_grouped_wgrad(a, a, torch.zeros((2, k, k), device="cuda"), few, kernel=kernel), (101, 102, 103)
    codes, scales, z = T.weights((), 512, 4 * k, 128, torch.float32, 1, True)
    for m in (1, 8):
        x = torch.ones((m, 4 * k), dtype=torch.bfloat16, device="cuda")
        yield lambda: g.gemv_w4(codes, scales, x, torch.zeros((m, 512), device="cuda"), zeros=z), (106,)


for call, codes in run(2048):
    t0 = time.time()
    call()
    torch.cuda.synchronize()                      # must return: no hang, no CUDA error
    status, seconds = g.device_status(reset=True), time.time() - t0
    print("status", status, "seconds", round(seconds, 2), flush=True)
    assert status in codes and seconds < 60, (status, seconds)
for call, codes in run(256):                      # the context is intact: problems without a third block run through
    call()
    torch.cuda.synchronize()
    assert g.device_status() == 0
print("OK")
"""


def test_an_expired_wait_ends_the_kernels_with_a_status():
    here = os.path.dirname(os.path.abspath(__file__))
    res = subprocess.run([sys.executable, "-c", CHILD % (os.path.dirname(here), here)], env=dict(os.environ, B200FP8_DEBUG="512"), capture_output=True,
                         text=True, timeout=600)
    assert res.returncode == 0, res.stdout + res.stderr
    assert "OK" in res.stdout
