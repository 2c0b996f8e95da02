"""Newton-Schulz orthogonalisation against the iteration in 64 bits."""
import numpy as np
import pytest

import block_util as bu
import gpu_util as gu
from ccglib_b200 import capi

pytestmark = pytest.mark.gpu

F16, BF16, F32 = capi.FLOAT16, capi.BFLOAT16, capi.FLOAT32
QUINTIC, CONVERGENT = (3.4445, -4.7750, 2.0315), (1.875, -1.25, 0.375)
U16 = 2.0 ** -11  # half a step of float16, relative
ETA16 = 2.0 ** -25  # and absolute below its normal range
GUARD = 64


def _f16(z):
    return (z.real.astype(np.float16).astype(np.float64)
            + 1j * z.imag.astype(np.float16).astype(np.float64))


def _fro(z):
    return float(np.linalg.norm(z))


def _iterate(x, steps, coefficients):
    """x complex128 n x l, n <= l -> (exact result, bound on the Frobenius error, result with the
    declared float16 roundings of the iterates in otherwise 64-bit arithmetic).

    The bound is first order, in Frobenius norms, times 1.1 for the rest.  A step maps singular values by
    f(s) = s (a + b s^2 + c s^4); an error of its argument grows by at most max |f'| over the
    singular values' range (divided differences of f are values of f').  A step's own errors:
    S, P and X' are rounded to float16 (U16 relative or ETA16 absolute per real value), and every
    float32 sum of 2K products taken 16 at a time by MMAs may lose a unit (2^-23) of the running sum each
    time: (K / 8 + 8) 2^-23 of the sum of absolute products."""
    a, b, c = coefficients
    n, l = x.shape
    scale = 2.0 ** round(0.5 * np.log2(np.float32(l)))
    x = x / _fro(x)
    emu = _f16(x * scale)
    err = U16 * _fro(x) + ETA16 / scale * np.sqrt(2.0 * n * l)
    for _ in range(steps):
        s = x @ x.conj().T
        p = b * s + c * (s @ s)
        top = np.linalg.norm(x, 2)
        t = np.linspace(0, 1.05 * top, 2001)
        growth = np.abs(a + 3 * b * t ** 2 + 5 * c * t ** 4).max()
        acc_l, acc_n = (l / 8 + 8) * 2.0 ** -23, (n / 8 + 8) * 2.0 ** -23
        d_s = U16 * _fro(s) + ETA16 * np.sqrt(2.0) * n + acc_l * _fro(np.abs(x) @ np.abs(x).T) * 2
        d_p = ((abs(b) + 2 * abs(c) * np.linalg.norm(s, 2)) * d_s + U16 * _fro(p)
               + ETA16 * np.sqrt(2.0) * n + acc_n * abs(c) * _fro(np.abs(s) @ np.abs(s)) * 2)
        new = a * x + p @ x
        own = (d_p * top + U16 * _fro(new) + ETA16 / scale * np.sqrt(2.0 * n * l)
               + acc_n * _fro(np.abs(p) @ np.abs(x)) * 2)
        err = growth * err + own
        x = new
        s = _f16(emu @ emu.conj().T / scale ** 2)
        p = _f16(b * s + c * (s @ s))
        emu = _f16(a * emu + p @ emu)
    return x, 1.1 * err, emu / scale


def _run(plan, x, type_in, type_out, axis, stream=None, in_place=False):
    """x: planar CPU tensor [batch][2][m][n] -> planar output, guards checked."""
    import torch

    batch, _, m, n = x.shape
    d_in = bu.lay_out(x, axis, capi.ROW_MAJOR).cuda()
    size = batch * 2 * m * n
    buf = torch.full((size + 2 * GUARD,), 7.0, dtype=bu.torch_type(type_out), device="cuda")
    out = buf[GUARD:GUARD + size].view(batch, 2, m, n)
    if in_place:
        out.copy_(d_in)
        d_in = out
    plan.run(d_in.data_ptr(), out.data_ptr(), gu.stream_handle() if stream is None else stream)
    torch.cuda.synchronize()
    gu.check_device_status()
    assert (buf[:GUARD] == 7).all() and (buf[-GUARD:] == 7).all(), "wrote outside the output"
    return out.clone()


def _input(rng, batch, m, n, type_in, strong=True):
    import torch

    x = rng.standard_normal((batch, 2, m, n))
    if strong:
        x += rng.standard_normal((batch, 2, m, 1)) * rng.standard_normal((batch, 1, 1, n))
    x *= np.exp(rng.uniform(-4, 4, (batch, 1, 1, 1)))
    return torch.from_numpy(x).to(bu.torch_type(type_in))


def _complex(x):
    v = x.double().cpu().numpy()
    return v[:, 0] + 1j * v[:, 1]


def _check(x, got, steps, coefficients, type_out):
    u = 2.0 ** -8 if type_out == BF16 else 2.0 ** -11
    for xi, gi in zip(_complex(x), _complex(got)):
        tall = xi.shape[0] > xi.shape[1]
        want, bound, emu = _iterate(xi.T if tall else xi, steps, coefficients)
        gi = gi.T if tall else gi
        bound += u * _fro(want) + 2.0 ** -24 * np.sqrt(want.size)
        assert _fro(gi - want) <= bound, "error %g, bound %g" % (_fro(gi - want), bound)
        # Small matrices stay in float32 to the end.  In the others float32 sums flip some of the
        # declared roundings, and that is all that is added to them.
        assert min(_fro(gi - emu), _fro(gi - want)) <= (0.5 * _fro(emu - want)
                                                        + 2 * u * _fro(want) / np.sqrt(3))


SHAPES = [(1, 1, 1), (3, 1, 7), (2, 9, 1), (2, 2, 2), (3, 5, 33), (2, 33, 70), (2, 70, 33),
          (1, 64, 64), (2, 100, 72), (1, 128, 256), (1, 129, 300), (1, 300, 130), (1, 257, 257)]


@pytest.mark.parametrize("steps, coefficients", [(1, QUINTIC), (5, QUINTIC), (8, CONVERGENT)])
@pytest.mark.parametrize("batch, m, n", SHAPES)
def test_shapes(batch, m, n, steps, coefficients):
    rng = np.random.default_rng(11)
    x = _input(rng, batch, m, n, F32)
    plan = capi.OrthogonalizePlan(batch, m, n, F32, F16, steps, coefficients)
    _check(x, _run(plan, x, F32, F16, capi.PLANAR), steps, coefficients, F16)


@pytest.mark.parametrize("form", ["0", "1", "2", "4", "8"])
def test_every_form_of_small_matrices(form, monkeypatch):
    """Three launches per step, or one with 1 .. 8 CTAs per matrix (the plan's choice by hand)."""
    rng = np.random.default_rng(18)
    monkeypatch.setenv("CCGLIB_B200_ORTH_SMALL", form)
    for batch, m, n in ((3, 4, 8), (2, 9, 200), (5, 200, 33), (2, 31, 90), (300, 8, 12), (2, 3, 5000)):
        x = _input(rng, batch, m, n, F16)
        plan = capi.OrthogonalizePlan(batch, m, n, F16, F16, 4, QUINTIC)
        got = _run(plan, x, F16, F16, capi.PLANAR)
        _check(x[-3:], got[-3:], 4, QUINTIC, F16)
        import torch

        assert torch.equal(_run(plan, x, F16, F16, capi.PLANAR, in_place=True), got)


@pytest.mark.parametrize("split", ["1", "2", "4"])
def test_every_split_of_large_matrices(split, monkeypatch):
    """CTAs that share the K of a tile (the plan's choice by hand)."""
    rng = np.random.default_rng(19)
    monkeypatch.setenv("CCGLIB_B200_ORTH_SPLIT", split)
    for batch, m, n in ((1, 150, 600), (1, 600, 150), (2, 260, 260)):
        x = _input(rng, batch, m, n, BF16)
        plan = capi.OrthogonalizePlan(batch, m, n, BF16, BF16, 3, QUINTIC)
        _check(x, _run(plan, x, BF16, BF16, capi.PLANAR), 3, QUINTIC, BF16)


@pytest.mark.parametrize("type_out", [F16, BF16])
@pytest.mark.parametrize("axis", [capi.PLANAR, capi.INTERLEAVED])
@pytest.mark.parametrize("type_in", [F16, BF16, F32])
def test_types_and_layouts(type_in, axis, type_out):
    rng = np.random.default_rng(12)
    for batch, m, n in ((2, 40, 72), (2, 75, 41), (1, 200, 136), (1, 136, 200)):
        x = _input(rng, batch, m, n, type_in)
        plan = capi.OrthogonalizePlan(batch, m, n, type_in, type_out, 3, QUINTIC, axis)
        _check(x, _run(plan, x, type_in, type_out, axis), 3, QUINTIC, type_out)


def test_rows_become_orthonormal():
    rng = np.random.default_rng(13)
    for m, n in ((24, 300), (300, 24), (160, 512)):
        x = _input(rng, 2, m, n, F32)
        plan = capi.OrthogonalizePlan(2, m, n, F32, F16, 14, CONVERGENT)
        for y in _complex(_run(plan, x, F32, F16, capi.PLANAR)):
            g = y @ y.conj().T if m <= n else y.conj().T @ y
            # entries of y are off by a few float16 steps; rows have unit norm
            assert np.abs(g - np.eye(len(g))).max() < 16 * U16


def test_scale_does_not_matter():
    """The norm is taken in float64: no input overflows or vanishes in it."""
    import torch

    rng = np.random.default_rng(14)
    x = torch.from_numpy(rng.standard_normal((1, 2, 20, 50))).float()
    plan = capi.OrthogonalizePlan(1, 20, 50, F32, F16)
    want = _run(plan, x, F32, F16, capi.PLANAR)
    for e in (-100, -60, 60, 120):
        assert torch.equal(_run(plan, x * 2.0 ** e, F32, F16, capi.PLANAR), want)


@pytest.mark.parametrize("m, n", [(20, 50), (140, 136)])
def test_zero_and_nan_stay_in_their_matrix(m, n):
    import torch

    rng = np.random.default_rng(15)
    x = _input(rng, 4, m, n, F32)
    plan = capi.OrthogonalizePlan(4, m, n, F32, F16)
    clean = _run(plan, x, F32, F16, capi.PLANAR)
    y = x.clone()
    y[1] = 0
    y[2, 1, 3, 4] = float("nan")
    y[3, 0, 0, 0] = float("inf")
    got = _run(plan, y, F32, F16, capi.PLANAR)
    assert torch.equal(got[0], clean[0])
    assert not got[1].any()
    assert torch.isnan(got[2]).all() and torch.isnan(got[3]).all()
    assert torch.equal(_run(plan, x, F32, F16, capi.PLANAR), clean)  # nothing left behind


def test_same_bits_in_place_on_a_side_stream_and_from_a_graph():
    import torch

    rng = np.random.default_rng(16)
    for m, n in ((30, 60), (200, 264)):
        x = _input(rng, 2, m, n, F16)
        plan = capi.OrthogonalizePlan(2, m, n, F16, F16)
        first = _run(plan, x, F16, F16, capi.PLANAR)
        assert torch.equal(_run(plan, x, F16, F16, capi.PLANAR, in_place=True), first)
        side = torch.cuda.Stream()
        assert torch.equal(_run(plan, x, F16, F16, capi.PLANAR, stream=side.cuda_stream), first)
        d_in, out = x.cuda(), torch.zeros_like(first)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            plan.run(d_in.data_ptr(), out.data_ptr(), gu.stream_handle())
        for _ in range(3):
            out.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, first)


def test_buffers_aligned_to_their_elements_only():
    import torch

    rng = np.random.default_rng(22)
    for m, n in ((40, 72), (200, 136)):
        x = _input(rng, 1, m, n, F16)
        plan = capi.OrthogonalizePlan(1, m, n, F16, F16, 3)
        want = _run(plan, x, F16, F16, capi.PLANAR)
        d_in = torch.zeros(2 * m * n + 8, dtype=torch.float16, device="cuda")
        out = torch.zeros(2 * m * n + 8, dtype=torch.float16, device="cuda")
        d_in[1:1 + 2 * m * n] = x.cuda().reshape(-1)
        plan.run(d_in.data_ptr() + 2, out.data_ptr() + 2, gu.stream_handle())
        torch.cuda.synchronize()
        assert torch.equal(out[1:1 + 2 * m * n].view(want.shape), want)
        assert out[0] == 0 and not out[1 + 2 * m * n:].any()


def test_weights_orthogonalised_quantised_and_multiplied():
    """The operators as they are used together: an orthonormal set of weights, quantised with one
    scale per 128 x 128 block, applied to samples quantised with one scale per row and block."""
    import torch

    rng = np.random.default_rng(17)
    beams, antennas, samples = 40, 300, 500
    e4 = capi.FLOAT8E4M3
    w = _input(rng, 1, beams, antennas, F32)
    x = torch.from_numpy(rng.standard_normal((1, 2, samples, antennas))).float()
    stream = gu.stream_handle()
    d_w, d_x = w.cuda(), x.cuda()
    ortho = torch.empty((1, 2, beams, antennas), dtype=torch.float16, device="cuda")
    plan = capi.OrthogonalizePlan(1, beams, antennas, F32, F16, 12, CONVERGENT)
    plan.run(d_w.data_ptr(), ortho.data_ptr(), stream)
    pitch, kb = capi.operand_pitch(antennas), bu.ceil(antennas, 128)
    qw = torch.empty((1, 2, beams, pitch), dtype=torch.uint8, device="cuda")
    qx = torch.empty((1, 2, samples, pitch), dtype=torch.uint8, device="cuda")
    sw = torch.empty((1, kb, 1), device="cuda")
    sx = torch.empty((1, kb, samples), device="cuda")
    capi.quantize(1, beams, antennas, F16, e4, ortho.data_ptr(), qw.data_ptr(), sw.data_ptr(), stream,
                  block_rows=128)
    capi.quantize(1, samples, antennas, F32, e4, d_x.data_ptr(), qx.data_ptr(), sx.data_ptr(), stream)
    gemm = capi.ScaledGemmPlan(1, beams, samples, antennas, e4, e4, F32, a_block_rows=128,
                               b_block_rows=1)
    c = torch.empty((1, 2, beams, samples), device="cuda")
    gemm.run(qw.data_ptr(), sw.data_ptr(), qx.data_ptr(), sx.data_ptr(), c.data_ptr(), stream)
    torch.cuda.synchronize()
    gu.check_device_status()
    u, _, vh = np.linalg.svd(_complex(w)[0], full_matrices=False)
    want = (u @ vh) @ _complex(x)[0].T
    got = _complex(c)[0]
    # e4m3 rounds either operand by at most 2^-4, rms about 2^-4 / sqrt(3) over a binade's lower end
    assert _fro(got - want) <= 2 * 2.0 ** -4 / np.sqrt(3) * _fro(want)
