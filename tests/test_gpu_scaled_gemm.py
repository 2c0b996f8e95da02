"""Block-scaled fp8 complex GEMM against a 64-bit product of the same fp8 values and scales."""
import numpy as np
import pytest

import block_util as bu
import gpu_util as gu
from ccglib_b200 import capi

pytestmark = pytest.mark.gpu

E4M3, E5M2 = capi.FLOAT8E4M3, capi.FLOAT8E5M2
F16, BF16, F32 = capi.FLOAT16, capi.BFLOAT16, capi.FLOAT32
PLANAR, INTER, ROW, COL = capi.PLANAR, capi.INTERLEAVED, capi.ROW_MAJOR, capi.COL_MAJOR
GUARD = 128


def _values(q, k):
    return q[..., :k].float().numpy().astype(np.float64)


def _run(plan, a, sa, b, sb, shape, type_out, c0=None, stream=None):
    import torch

    d = [t.cuda() for t in (a, sa, b, sb)]
    n = int(np.prod(shape))
    buf = torch.full((n + 2 * GUARD,), 77.0, dtype=bu.torch_type(type_out), device="cuda")
    c = buf[GUARD:GUARD + n].view(shape)
    if c0 is not None:
        c.copy_(c0)
    plan.run(*[t.data_ptr() for t in d], c.data_ptr(),
             gu.stream_handle() if stream is None else stream)
    torch.cuda.synchronize()
    gu.check_device_status()
    assert (buf[:GUARD] == 77).all() and (buf[-GUARD:] == 77).all(), "wrote outside C"
    return c.clone()


def _check(c, want, s_re, s_im, k, type_out):
    got = c.double().cpu().numpy()
    for i, (w, s) in enumerate(((want.real, s_re), (want.imag, s_im))):
        err, tol = np.abs(got[:, i] - w), bu.product_tolerance(w, s, k, type_out)
        assert (err <= tol).all(), "%d values off, worst %g of its tolerance" % (
            int((err > tol).sum()), float((err / tol).max()))


def _case(seed, batch, m, n, k, ta, tb, type_out, ga, gb, axis=PLANAR, order=ROW, **kw):
    rng = np.random.default_rng(seed)
    a, sa = bu.random_operand(rng, batch, m, k, ta, ga)
    b, sb = bu.random_operand(rng, batch, n, k, tb, gb)
    plan = capi.ScaledGemmPlan(batch, m, n, k, ta, tb, type_out, ga, gb, axis, order, **kw)
    want, s_re, s_im = bu.scaled_product(_values(a, k), sa.numpy(), ga, _values(b, k), sb.numpy(), gb)
    c = _run(plan, a, sa, b, sb, bu.c_shape(batch, m, n, axis, order), type_out)
    _check(bu.canonical_c(c, axis, order), want, s_re, s_im, k, type_out)
    return plan.tile


SHAPES = [(1, 1, 1, 1), (1, 1, 1, 5), (2, 1, 300, 128), (1, 300, 1, 129), (3, 5, 7, 300),
          (1, 16, 200, 512), (2, 17, 130, 400), (1, 33, 129, 1000), (1, 64, 65, 127),
          (1, 65, 64, 130), (2, 128, 128, 256), (1, 129, 257, 640), (3, 200, 100, 1111),
          (1, 512, 300, 2048)]


@pytest.mark.parametrize("ga, gb", [(1, 1), (1, 128), (128, 1), (128, 128)])
@pytest.mark.parametrize("batch, m, n, k", SHAPES)
def test_shapes_and_block_forms(batch, m, n, k, ga, gb):
    _case(1, batch, m, n, k, E4M3, E4M3, F32, ga, gb)


@pytest.mark.parametrize("ta, tb", [(E4M3, E5M2), (E5M2, E4M3), (E5M2, E5M2)])
@pytest.mark.parametrize("m, n", [(9, 200), (200, 9), (150, 260)])
def test_types(ta, tb, m, n):
    _case(2, 2, m, n, 390, ta, tb, F32, 1, 128)


@pytest.mark.parametrize("order", [ROW, COL])
@pytest.mark.parametrize("axis", [PLANAR, INTER])
@pytest.mark.parametrize("type_out", [F32, F16, BF16])
def test_output_layouts(type_out, axis, order):
    # aligned and odd row lengths, row side either operand, every tile width
    for m, n in ((256, 256), (130, 136), (131, 133), (8, 264), (264, 8), (50, 300), (300, 31)):
        _case(3, 2, m, n, 256, E4M3, E4M3, type_out, 1, 1, axis, order)


@pytest.mark.parametrize("order", [ROW, COL])
@pytest.mark.parametrize("axis", [PLANAR, INTER])
@pytest.mark.parametrize("type_out, m, n", [(F32, 200, 144), (F16, 200, 144), (BF16, 7, 133), (F32, 133, 7)])
def test_alpha_beta(type_out, m, n, axis, order):
    import torch

    rng = np.random.default_rng(4)
    batch, k, alpha, beta = 2, 300, (0.5, -0.25), (-1.5, 2.0)
    a, sa = bu.random_operand(rng, batch, m, k, E4M3, 1)
    b, sb = bu.random_operand(rng, batch, n, k, E4M3, 128)
    want, s_re, s_im = bu.scaled_product(_values(a, k), sa.numpy(), 1, _values(b, k), sb.numpy(), 128)
    shape = bu.c_shape(batch, m, n, axis, order)
    c0 = torch.from_numpy(rng.standard_normal(shape)).to(bu.torch_type(type_out))
    plan = capi.ScaledGemmPlan(batch, m, n, k, E4M3, E4M3, type_out, 1, 128, axis, order, alpha=alpha,
                               beta=beta)
    c = bu.canonical_c(_run(plan, a, sa, b, sb, shape, type_out, c0), axis, order)
    old = bu.canonical_c(c0, axis, order).double().numpy()
    old = old[:, 0] + 1j * old[:, 1]
    full = complex(*alpha) * want + complex(*beta) * old
    # the bound of the product, times |alpha|_1, and four roundings of terms below S_all
    mag = np.abs(old.real) + np.abs(old.imag)
    s_all = (abs(alpha[0]) + abs(alpha[1])) * (s_re + s_im) + (abs(beta[0]) + abs(beta[1])) * mag
    _check(c, full, s_all, s_all, k, type_out)


def test_nan_and_infinity_reach_only_their_row_and_column():
    import torch

    rng = np.random.default_rng(5)
    m, n, k = 140, 150, 300
    a, sa = bu.random_operand(rng, 1, m, k, E4M3, 1)
    b, sb = bu.random_operand(rng, 1, n, k, E5M2, 1)
    a.view(torch.uint8)[0, 0, 3, 299] = 0x7F  # NaN
    b.view(torch.uint8)[0, 1, 149, 0] = 0x7C  # infinity
    plan = capi.ScaledGemmPlan(1, m, n, k, E4M3, E5M2, F32, 1, 1)
    c = _run(plan, a, sa, b, sb, (1, 2, m, n), F32).cpu().numpy()
    assert np.isnan(c[:, :, 3]).all()
    assert not np.isfinite(c[:, :, :, 149]).any()
    c[:, :, 3] = 0
    c[:, :, :, 149] = 0
    assert np.isfinite(c).all()


def test_extreme_scales_do_not_overflow_on_the_way():
    """A silent block (scale 2^-126, zeros) against one whose scale is huge, and scales whose product
    leaves float32 although the scaled sums do not."""
    import torch

    rng = np.random.default_rng(6)
    m, n, k = 130, 140, 256
    a, sa = bu.random_operand(rng, 1, m, k, E4M3, 1)
    b, sb = bu.random_operand(rng, 1, n, k, E4M3, 1)
    a.view(torch.uint8)[0, :, 5, :128] = 0
    sa[0, 0, :] = 2.0 ** -126
    sb[0, 0, :] = 2.0 ** 110
    sa[0, 1, :] = 2.0 ** -100
    sb[0, 1, :] = 2.0 ** 80
    want, s_re, s_im = bu.scaled_product(_values(a, k), sa.numpy(), 1, _values(b, k), sb.numpy(), 1)
    plan = capi.ScaledGemmPlan(1, m, n, k, E4M3, E4M3, F32, 1, 1)
    c = _run(plan, a, sa, b, sb, (1, 2, m, n), F32)
    _check(c, want, s_re, s_im, k, F32)
    a.view(torch.uint8)[0] = 0
    sa[:] = 1e38
    sb[:] = 1e38
    assert not _run(plan, a, sa, b, sb, (1, 2, m, n), F32).any()


def test_zero_beta_does_not_read_c():
    import torch

    rng = np.random.default_rng(7)
    m, n, k = 128, 128, 128
    a, sa = bu.random_operand(rng, 1, m, k, E4M3, 1)
    b, sb = bu.random_operand(rng, 1, n, k, E4M3, 1)
    plan = capi.ScaledGemmPlan(1, m, n, k, E4M3, E4M3, F32, 1, 1)
    c = _run(plan, a, sa, b, sb, (1, 2, m, n), F32, c0=torch.full((1, 2, m, n), float("nan")))
    assert torch.isfinite(c).all()


def test_same_bits_from_run_to_run_and_from_a_graph():
    """Shared tiles are added in the order of k whoever comes last; the workspace is clean again
    after every run."""
    import torch

    rng = np.random.default_rng(8)
    for batch, m, n, k in ((1, 1, 2000, 4096), (1, 300, 300, 4096), (2, 12, 700, 8192)):
        plan = capi.ScaledGemmPlan(batch, m, n, k, E4M3, E4M3, F32, 1, 128)
        assert plan.tile["runs"] > 0 and plan.scratch_bytes > 0
        a, sa = bu.random_operand(rng, batch, m, k, E4M3, 1)
        b, sb = bu.random_operand(rng, batch, n, k, E4M3, 128)
        shape = (batch, 2, m, n)
        first = _run(plan, a, sa, b, sb, shape, F32)
        for _ in range(5):
            assert torch.equal(_run(plan, a, sa, b, sb, shape, F32), first)
        d = [t.cuda() for t in (a, sa, b, sb)]
        c = torch.zeros(shape, device="cuda")
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            plan.run(*[t.data_ptr() for t in d], c.data_ptr(), gu.stream_handle())
        for _ in range(3):
            c.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(c, first)
        gu.check_device_status()


def test_two_plans_on_two_streams():
    import torch

    rng = np.random.default_rng(9)
    m, n, k = 40, 900, 4096
    a, sa = bu.random_operand(rng, 1, m, k, E4M3, 1)
    b, sb = bu.random_operand(rng, 1, n, k, E4M3, 1)
    plans = [capi.ScaledGemmPlan(1, m, n, k, E4M3, E4M3, F32, 1, 1) for _ in range(2)]
    want = _run(plans[0], a, sa, b, sb, (1, 2, m, n), F32)
    d = [t.cuda() for t in (a, sa, b, sb)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    out = [torch.zeros((8, 2, m, n), device="cuda") for _ in range(2)]
    torch.cuda.synchronize()
    for i in range(8):
        for plan, stream, c in zip(plans, streams, out):
            plan.run(*[t.data_ptr() for t in d], c[i].data_ptr(), stream.cuda_stream)
    torch.cuda.synchronize()
    for c in out:
        for i in range(8):
            assert torch.equal(c[i:i + 1], want)


def test_quantise_and_multiply():
    """Both operators as they are used: float samples in, C out, against the 64-bit product of the
    samples; what the quantiser rounds is counted in."""
    import torch

    rng = np.random.default_rng(10)
    batch, m, n, k = 2, 70, 200, 700
    x = torch.from_numpy(rng.standard_normal((batch, 2, m, k)) * np.exp(rng.uniform(-6, 6, (batch, 1, m, 1)))).float()
    w = torch.from_numpy(rng.standard_normal((batch, 2, n, k))).to(torch.bfloat16)
    pitch, kb = capi.operand_pitch(k), bu.ceil(k, 128)
    q = [torch.empty((batch, 2, r, pitch), dtype=torch.uint8, device="cuda") for r in (m, n)]
    s = [torch.empty((batch, kb, r), device="cuda") for r in (m, bu.ceil(n, 128))]
    d_x = bu.lay_out(x, INTER, ROW).cuda()
    d_w = bu.lay_out(w, PLANAR, COL).cuda()
    stream = gu.stream_handle()
    capi.quantize(batch, m, k, F32, E4M3, d_x.data_ptr(), q[0].data_ptr(), s[0].data_ptr(), stream,
                  input_complex_axis=INTER)
    capi.quantize(batch, n, k, BF16, E4M3, d_w.data_ptr(), q[1].data_ptr(), s[1].data_ptr(), stream,
                  input_mem_order=COL, block_rows=128)
    plan = capi.ScaledGemmPlan(batch, m, n, k, E4M3, E4M3, F32)
    c = torch.empty((batch, 2, m, n), device="cuda")
    plan.run(q[0].data_ptr(), s[0].data_ptr(), q[1].data_ptr(), s[1].data_ptr(), c.data_ptr(), stream)
    torch.cuda.synchronize()
    xv, wv = x.double().numpy(), w.double().numpy()
    one = np.ones((batch, kb, m), np.float32)
    want, s_re, s_im = bu.scaled_product(xv, one, 1, wv, np.ones((batch, kb, n), np.float32), 1)
    got = c.double().cpu().numpy()
    # e4m3 rounds by half a step (2^-4 relative, or 2^-10 of the scale when subnormal): each product
    # is off by at most 2 * 2^-4 + 2^-8 of its size plus the subnormal part
    sx = bu.per_element(s[0].cpu().numpy().astype(np.float64), 1, m, k)
    sw = bu.per_element(s[1].cpu().numpy().astype(np.float64), 128, n, k)
    ax, aw = np.abs(xv).sum(1), np.abs(wv).sum(1)
    sub = 2.0 ** -10 * (np.einsum("bmk,bnk->bmn", sx, aw) + np.einsum("bmk,bnk->bmn", ax, sw)) * 1.1
    for i, (v, mag) in enumerate(((want.real, s_re), (want.imag, s_im))):
        bound = (2 * 2.0 ** -4 + 2.0 ** -8) * mag + 2 * sub + bu.product_tolerance(v, mag, k, F32)
        assert (np.abs(got[:, i] - v) <= bound).all()
        rms = np.sqrt(np.mean((got[:, i] - v) ** 2) / np.mean(v ** 2))
        assert rms < 2 * 2.0 ** -4


def test_backward_products():
    """Gradients of a real loss L = Re sum conj(G) C of C = A B^T: dA = G conj(B), dB = G^T conj(A), from
    the same two operators with the operands quantised along their other axis.  Against the formula in
    64 bits on the dequantised operands, and the formula against differences of L."""
    import torch

    rng = np.random.default_rng(21)
    m, n, k = 90, 140, 200
    a, b = (torch.from_numpy(rng.standard_normal((1, 2, r, k))).float() for r in (m, n))
    g = torch.from_numpy(rng.standard_normal((1, 2, m, n))).float()

    def quantised(x, rows, kk, code, order, conjugate):
        """-> (tensors for the GEMM, complex values [rows][kk] that they stand for)"""
        d_in = x.cuda()
        q = torch.empty((1, 2, rows, capi.operand_pitch(kk)), dtype=torch.uint8, device="cuda")
        s = torch.empty((1, bu.ceil(kk, 128), rows), device="cuda")
        capi.quantize(1, rows, kk, F32, code, d_in.data_ptr(), q.data_ptr(), s.data_ptr(),
                      gu.stream_handle(), input_mem_order=order, conjugate=conjugate)
        v = q.view(bu.torch_type(code))[..., :kk].double().cpu().numpy()
        return (q, s), v, s.cpu().numpy()

    def product(x, xv, xs, y, yv, ys, rows, cols, kk, ta):
        plan = capi.ScaledGemmPlan(1, rows, cols, kk, ta, E4M3, F32, 1, 1)
        c = torch.empty((1, 2, rows, cols), device="cuda")
        plan.run(x[0].data_ptr(), x[1].data_ptr(), y[0].data_ptr(), y[1].data_ptr(), c.data_ptr(),
                 gu.stream_handle())
        torch.cuda.synchronize()
        want, s_re, s_im = bu.scaled_product(xv, xs, 1, yv, ys, 1)
        _check(c, want, s_re, s_im, kk, F32)
        got = c.double().cpu().numpy()
        return got[0, 0] + 1j * got[0, 1]

    # dA [m][k]: over n.  B is [n][k]: for rows of k it is col-major.
    d_a = product(*quantised(g, m, n, E5M2, ROW, False), *quantised(b, k, n, E4M3, COL, True),
                  m, k, n, E5M2)
    # dB [n][k]: over m
    d_b = product(*quantised(g, n, m, E5M2, COL, False), *quantised(a, k, m, E4M3, COL, True),
                  n, k, m, E5M2)
    av, bv, gv = ((x[0, 0] + 1j * x[0, 1]).numpy().astype(np.complex128) for x in (a, b, g))
    exact_a, exact_b = gv @ bv.conj(), gv.T @ av.conj()
    # e5m2 rounds by at most 2^-3, e4m3 by 2^-4; errors of the terms are independent
    for got, want in ((d_a, exact_a), (d_b, exact_b)):
        assert np.linalg.norm(got - want) <= (2.0 ** -3 + 2.0 ** -4) * np.linalg.norm(want)

    def loss(x, y):
        return float(np.sum(gv.conj() * (x @ y.T)).real)

    # L is linear in either operand: differences are exact up to rounding
    for _ in range(3):
        e = rng.standard_normal((m, k)) + 1j * rng.standard_normal((m, k))
        f = rng.standard_normal((n, k)) + 1j * rng.standard_normal((n, k))
        da = (loss(av + e, bv) - loss(av - e, bv)) / 2
        db = (loss(av, bv + f) - loss(av, bv - f)) / 2
        assert abs(da - np.sum(exact_a.conj() * e).real) <= 1e-9 * np.linalg.norm(exact_a) * np.linalg.norm(e)
        assert abs(db - np.sum(exact_b.conj() * f).real) <= 1e-9 * np.linalg.norm(exact_b) * np.linalg.norm(f)
