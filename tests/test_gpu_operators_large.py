"""Arrays whose element offsets pass 32 bits: the quantiser, the scaled GEMM and the orthogonalisation at a
size where only 64-bit offsets reach the end, checked at both ends."""
import numpy as np
import pytest

import block_util as bu
import gpu_util as gu
from ccglib_b200 import capi

pytestmark = pytest.mark.gpu

E4M3, F16, F32 = capi.FLOAT8E4M3, capi.FLOAT16, capi.FLOAT32


def _free():
    import torch

    torch.cuda.empty_cache()


@pytest.mark.parametrize("order", [capi.ROW_MAJOR, capi.COL_MAJOR])
def test_quantize(order):
    import torch

    rows, k = 33000, 66048  # 4.36e9 values
    gen = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn((1, 2, 1, 66048), generator=gen, device="cuda").half()
    shape = (1, 2, rows, k) if order == capi.ROW_MAJOR else (1, 2, k, rows)
    d_in = torch.zeros(shape, dtype=torch.float16, device="cuda")
    # only the last 130 rows are not silent
    last = x.expand(1, 2, 130, k).clone() * torch.arange(1, 131, device="cuda").half()[:, None]
    if order == capi.ROW_MAJOR:
        d_in[:, :, -130:] = last
    else:
        d_in[:, :, :, -130:] = last.transpose(2, 3)
    q = torch.full((1, 2, rows, k), 0x5A, dtype=torch.uint8, device="cuda")
    s = torch.empty((1, k // 128, rows), device="cuda")
    capi.quantize(1, rows, k, F16, E4M3, d_in.data_ptr(), q.data_ptr(), s.data_ptr(),
                  gu.stream_handle(), input_mem_order=order)
    del d_in
    want, want_scale = bu.quantize(last.float().cpu().numpy(), E4M3, 1)
    got = q[:, :, -130:].contiguous().view(torch.float8_e4m3fn).double().cpu().numpy()
    np.testing.assert_array_equal(got, want)
    np.testing.assert_array_equal(s[:, :, -130:].cpu().numpy(), want_scale)
    assert not (q[:, :, :-130] & 0x7F).any() and (s[:, :, :-130] == 2.0 ** -126).all()
    del q, s
    _free()


@pytest.mark.parametrize("axis, order", [(capi.PLANAR, capi.ROW_MAJOR), (capi.INTERLEAVED, capi.COL_MAJOR)])
def test_scaled_gemm(axis, order):
    import torch

    m, n, k = 46400, 46337, 40  # 4.3e9 values of C
    rng = np.random.default_rng(2)
    a, sa = bu.random_operand(rng, 1, m, k, E4M3, 1)
    b, sb = bu.random_operand(rng, 1, n, k, E4M3, 128)
    d = [t.cuda() for t in (a, sa, b, sb)]
    c = torch.full(bu.c_shape(1, m, n, axis, order), 7.0, device="cuda")
    plan = capi.ScaledGemmPlan(1, m, n, k, E4M3, E4M3, F32, 1, 128, axis, order)
    plan.run(*[t.data_ptr() for t in d], c.data_ptr(), gu.stream_handle())
    torch.cuda.synchronize()
    gu.check_device_status()
    if axis == capi.INTERLEAVED:
        c = c.permute(0, 3, 1, 2)
    if order == capi.COL_MAJOR:
        c = c.transpose(2, 3)
    av, bv = (t[..., :k].float().numpy().astype(np.float64) for t in (a, b))
    for rows in (slice(0, 40), slice(m - 40, m)):
        want, s_re, s_im = bu.scaled_product(av[:, :, rows], sa.numpy()[:, :, rows], 1, bv, sb.numpy(), 128)
        got = c[:, :, rows].double().cpu().numpy()
        for i, (w, s) in enumerate(((want.real, s_re), (want.imag, s_im))):
            assert (np.abs(got[:, i] - w) <= bu.product_tolerance(w, s, k, F32)).all()
    del c, d
    _free()


def test_orthogonalize():
    """Rows far apart of a tall matrix that is zero in between: as if the zero rows were not there."""
    import torch

    m, n = 4200000, 1040 // 2  # 4.37e9 values
    rng = np.random.default_rng(3)
    x = torch.from_numpy(rng.standard_normal((1, 2, 2 * n, n))).half().cuda()
    small = torch.empty((1, 2, 2 * n, n), dtype=torch.float16, device="cuda")
    plan = capi.OrthogonalizePlan(1, 2 * n, n, F16, F16, 2)
    plan.run(x.data_ptr(), small.data_ptr(), gu.stream_handle())
    d_in = torch.zeros((1, 2, m, n), dtype=torch.float16, device="cuda")
    d_in[:, :, :n], d_in[:, :, -n:] = x[:, :, :n], x[:, :, n:]
    plan = capi.OrthogonalizePlan(1, m, n, F16, F16, 2)
    plan.run(d_in.data_ptr(), d_in.data_ptr(), gu.stream_handle())
    torch.cuda.synchronize()
    gu.check_device_status()
    got = torch.cat((d_in[:, :, :n], d_in[:, :, -n:]), 2).double()
    # The two differ by their scaling (a power of two each), which changes what falls below float16's normal
    # range, and by the order of float32 sums: far less than two steps' float16 roundings, a few 2^-11.
    assert (got - small.double()).norm() <= 8 * 2.0 ** -11 * small.double().norm()
    assert not d_in[:, :, n:-n].any()
    del d_in, plan
    _free()
