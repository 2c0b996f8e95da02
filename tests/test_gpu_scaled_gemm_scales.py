"""The block-scaled GEMM over the whole range of float32 scales: wherever sA sB d is a float32, it comes
out within the bound of an ordinary product, whichever operand holds which scale and whichever is the
row side of the tile."""
import numpy as np
import pytest

import block_util as bu
import gpu_util as gu
from ccglib_b200 import capi
from test_gpu_scaled_gemm import _check, _run, _values

pytestmark = pytest.mark.gpu

E4M3, E5M2, F32 = capi.FLOAT8E4M3, capi.FLOAT8E5M2, capi.FLOAT32
K = 256  # two blocks: two roundings of at most 2^-150 each where the sums are subnormal
# tiles of 64 columns, of 64 and of 16 columns with B or A as the row side (128 columns: at the end)
SHAPES = [(130, 140), (40, 200), (200, 40), (9, 150), (150, 9), (200, 260)]
FORMS = [(1, 1), (1, 128), (128, 1), (128, 128)]


def _operands(rng, m, n, code, top, k=K):
    """Values over the format up to `top` of its largest."""
    import torch

    out = []
    for rows in (m, n):
        v = rng.standard_normal((1, 2, rows, k)) * bu.FMAX[code] / 4 * top
        out.append(torch.from_numpy(bu.round_fp8(np.clip(v, -bu.FMAX[code], bu.FMAX[code]), code))
                   .float().to(bu.torch_type(code)))
    return out


def _scales(rows, g, exponent, rng):
    """2^exponent times 1 .. 2; `exponent` a number or (low, high)."""
    import torch

    shape = (1, 2, bu.ceil(rows, g))
    e = rng.integers(*exponent, shape) if isinstance(exponent, tuple) else np.full(shape, exponent)
    return torch.from_numpy((np.exp2(e.astype(np.float64)) * rng.uniform(1, 1.99, shape)).astype(np.float32))


def _compare(m, n, a, sa, ga, b, sb, gb, code, k=K):
    plan = capi.ScaledGemmPlan(1, m, n, k, code, code, F32, ga, gb)
    want, s_re, s_im = bu.scaled_product(_values(a, k), sa.numpy(), ga, _values(b, k), sb.numpy(), gb)
    largest = max(abs(want.real).max(), abs(want.imag).max())
    assert 2.0 ** -140 < largest < 2.0 ** 127  # the case asks for float32 values
    _check(_run(plan, a, sa, b, sb, (1, 2, m, n), F32), want, s_re, s_im, k, F32)


@pytest.mark.parametrize("code, top, ea, eb", [
    (E5M2, 1, -76, -76),       # the product of the scales vanishes
    (E4M3, 1, -66, -69),       # ... is subnormal
    (E4M3, 1, -126, -19),      # a block at the quantiser's floor against an ordinary one
    (E4M3, 1, -18, -126),
    (E5M2, 1, -126, -1),
    (E5M2, 1, -140, 30),       # a subnormal scale
    (E5M2, 1, 30, -140),
    (E4M3, 2.0 ** -15, 64, 63),   # the product overflows, the sums do not
    (E4M3, 2.0 ** -15, 63, 64),
    (E4M3, 1, 120, -110),      # one way round overflows, the other vanishes
    (E4M3, 1, -110, 120),
    (E4M3, 1, 90, -126),
    (E4M3, 1, (-126, 45), (-126, 45)),  # everything in one tile
    (E5M2, 1, (-126, 40), (-149, 40)),
    (E5M2, 1, (-63, 40), (-126, -62)),
])
@pytest.mark.parametrize("m, n", SHAPES)
def test_range_of_scales(m, n, code, top, ea, eb):
    rng = np.random.default_rng(31)
    a, b = _operands(rng, m, n, code, top)
    for ga, gb in FORMS:
        _compare(m, n, a, _scales(m, ga, ea, rng), ga, b, _scales(n, gb, eb, rng), gb, code)


@pytest.mark.parametrize("ea, eb", [
    ((-126, -126, -126, -3, -126), (-3, -126, -3, -3, -3)),    # faint first, then ordinary
    ((-3, -3, -126, -3, -126), (-3, -126, -126, -3, -3)),      # ordinary first
    ((-126, 12, -126, 40, -126), (-3, 12, -126, -20, -3)),     # past what lifted sums hold
    ((-126, 70, -126, -140, -3), (-3, -60, -126, -3, -3)),     # past float32's middle at either end
    ((-126, -70, -126, -90, -126), (-9, -20, -126, -9, -9)),   # faint throughout
])
@pytest.mark.parametrize("code", [E4M3, E5M2])
@pytest.mark.parametrize("m, n", SHAPES)
def test_scales_that_change_along_k(m, n, code, ea, eb):
    """Every second row (column, block of rows) goes through the exponents, the others stay at 2^-3."""
    import torch

    rng = np.random.default_rng(35)
    k = 128 * len(ea) - 60
    a, b = _operands(rng, m, n, code, 1, 128 * len(ea))
    a, b = a[..., :k].contiguous(), b[..., :k].contiguous()
    pad = capi.operand_pitch(k) - k
    a, b = (torch.nn.functional.pad(x.view(torch.uint8), (0, pad)).view(x.dtype) for x in (a, b))
    for ga, gb in FORMS:
        scales = []
        for rows, g, e in ((m, ga, ea), (n, gb, eb)):
            x = np.full((1, len(e), bu.ceil(rows, g)), -3.0)
            x[:, :, ::2] = np.array(e, np.float64)[None, :, None]
            scales.append(torch.from_numpy((np.exp2(x) * rng.uniform(1, 1.99, x.shape)).astype(np.float32)))
        _compare(m, n, a, scales[0], ga, b, scales[1], gb, code, k)


@pytest.mark.parametrize("m, n", SHAPES)
def test_zero_sums_stay_zero(m, n):
    """Scales at and beyond the borders of the ranges, their product an infinity in float32."""
    import torch

    rng = np.random.default_rng(32)
    a, b = _operands(rng, m, n, E4M3, 1)
    a.view(torch.uint8)[:] = 0
    for s in (2.0 ** 63, 2.0 ** 64, 1.8446744e19, 3e38):
        for ga, gb in FORMS:
            sa, sb = (torch.full((1, 2, bu.ceil(r, g)), s) for r, g in ((m, ga), (n, gb)))
            plan = capi.ScaledGemmPlan(1, m, n, K, E4M3, E4M3, F32, ga, gb)
            assert not _run(plan, a, sa, b, sb, (1, 2, m, n), F32).any()


@pytest.mark.parametrize("m, n", SHAPES)
@pytest.mark.parametrize("ea, eb", [(-126, -126), (-126, -3), (-70, -126), (0, 0), (-140, -130)])
def test_infinite_sums_stay_infinite(m, n, ea, eb):
    """However small the scales: an infinity does not meet a factor that has become zero."""
    import torch

    rng = np.random.default_rng(33)
    a, b = _operands(rng, m, n, E5M2, 1)
    a.view(torch.uint8)[0, 0, 3, 5] = 0x7C
    b.view(torch.uint8)[0, :, :, 5] = 0x3C  # ones: no product of the infinity is a NaN
    for ga, gb in FORMS:
        sa, sb = _scales(m, ga, ea, rng), _scales(n, gb, eb, rng)
        plan = capi.ScaledGemmPlan(1, m, n, K, E5M2, E5M2, F32, ga, gb)
        c = _run(plan, a, sa, b, sb, (1, 2, m, n), F32)
        assert (c[:, :, 3] == float("inf")).all()
        assert torch.isfinite(c[:, :, :3]).all() and torch.isfinite(c[:, :, 4:]).all()


def test_silent_and_faint_rows_of_the_quantiser():
    """Samples down to 1e-38, quantised and multiplied with weights of 1e-30 .. 1: rows whose scale is at
    the quantiser's floor, rows near it and silent rows beside ordinary ones."""
    import torch

    rng = np.random.default_rng(34)
    m, n = 200, 150
    level = np.exp2(rng.uniform(-126, 3, (1, 1, m, 1)))
    level[:, :, ::7] = 0
    x = torch.from_numpy(rng.standard_normal((1, 2, m, K)) * level).float()
    w = torch.from_numpy(rng.standard_normal((1, 2, n, K)) * np.exp2(rng.uniform(-100, 40, (1, 1, n, 1)))).float()
    q, s = [], []
    for v, rows in ((x, m), (w, n)):
        d = v.cuda()
        q.append(torch.empty((1, 2, rows, K), dtype=torch.uint8, device="cuda"))
        s.append(torch.empty((1, 2, rows), device="cuda"))
        capi.quantize(1, rows, K, F32, E4M3, d.data_ptr(), q[-1].data_ptr(), s[-1].data_ptr(),
                      gu.stream_handle())
        torch.cuda.synchronize()
    a, b = (t.cpu().view(torch.float8_e4m3fn) for t in q)
    sa, sb = (t.cpu() for t in s)
    assert (sa == 2.0 ** -126).any() and (sa > 2.0 ** -126).any()
    _compare(m, n, a, sa, 1, b, sb, 1, E4M3)


@pytest.mark.parametrize("runs", ["0", "1"])
def test_wide_tiles(runs, monkeypatch):
    """All of the above on tiles of 128 columns."""
    monkeypatch.setenv("CCGLIB_B200_SCALED_BN", "128")
    monkeypatch.setenv("CCGLIB_B200_SCALED_RUNS", runs)
    m, n = 200, 260
    assert capi.ScaledGemmPlan(1, m, n, K, E4M3, E4M3, F32, 1, 1).tile["bn"] == 128
    for test, names in ((test_range_of_scales, "code, top, ea, eb"), (test_infinite_sums_stay_infinite, "ea, eb"),
                        (test_scales_that_change_along_k, "code"), (test_scales_that_change_along_k, "ea, eb")):
        for mark in test.pytestmark:
            if mark.args[0] != names:
                continue
            for values in mark.args[1]:
                values = values if isinstance(values, tuple) else (values,)
                kw = dict(zip(names.split(", "), values))
                if test is test_scales_that_change_along_k:
                    kw = {"code": E4M3, "ea": (-126, -3, -126, 40, -126), "eb": (-3, 12, -126, -20, -3), **kw}
                test(m, n, **kw)
    test_zero_sums_stay_zero(m, n)
    test_silent_and_faint_rows_of_the_quantiser()
