"""Block quantiser against its definition: scales and fp8 values are equal bit for bit (every step is
one correctly rounded float32 operation), padding is zero, nothing outside is written."""
import numpy as np
import pytest

import block_util as bu
import gpu_util as gu
from ccglib_b200 import capi

pytestmark = pytest.mark.gpu

E4M3, E5M2 = capi.FLOAT8E4M3, capi.FLOAT8E5M2
F16, BF16, F32 = capi.FLOAT16, capi.BFLOAT16, capi.FLOAT32
GUARD = 64


def _signal(rng, batch, rows, k, type_in):
    import torch

    x = rng.standard_normal((batch, 2, rows, k)) * np.exp(rng.uniform(-3, 3, (batch, 1, rows, 1)))
    if rows > 2:
        x[:, :, rows // 2] = 0  # a silent row
    return torch.from_numpy(x).to(bu.torch_type(type_in))


def _run(x, type_in, type_out, axis, order, block_rows, stream=None):
    """x: planar CPU tensor -> (fp8 values with padding float64, scales), guards checked."""
    import torch

    batch, _, rows, k = x.shape
    pitch = capi.operand_pitch(k)
    d_in = bu.lay_out(x, axis, order).cuda()
    nq = batch * 2 * rows * pitch
    q = torch.full((nq + 2 * GUARD,), 0x5A, dtype=torch.uint8, device="cuda")
    ns = batch * bu.ceil(k, 128) * bu.ceil(rows, block_rows)
    s = torch.full((ns + 2,), -7.0, dtype=torch.float32, device="cuda")
    capi.quantize(batch, rows, k, type_in, type_out, d_in.data_ptr(), q.data_ptr() + GUARD,
                  s.data_ptr() + 4, gu.stream_handle() if stream is None else stream,
                  input_complex_axis=axis, input_mem_order=order, block_rows=block_rows)
    torch.cuda.synchronize()
    assert (q[:GUARD] == 0x5A).all() and (q[-GUARD:] == 0x5A).all() and s[0] == -7 and s[-1] == -7
    v = q[GUARD:-GUARD].view(bu.torch_type(type_out)).double().cpu().numpy()
    return (v.reshape(batch, 2, rows, pitch),
            s[1:-1].cpu().numpy().reshape(batch, bu.ceil(k, 128), bu.ceil(rows, block_rows)))


def _check(x, type_out, block_rows, got, scale):
    want, want_scale = bu.quantize(x.float().numpy(), type_out, block_rows)
    np.testing.assert_array_equal(scale, want_scale)
    np.testing.assert_array_equal(got[..., :x.shape[3]], want)
    assert not got[..., x.shape[3]:].any()


SHAPES = [(1, 1, 1), (2, 3, 5), (1, 4, 128), (3, 129, 130), (2, 127, 260), (1, 300, 1000),
          (5, 33, 16), (1, 1, 4099), (1, 1000, 3)]


@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("order", [capi.ROW_MAJOR, capi.COL_MAJOR])
@pytest.mark.parametrize("axis", [capi.PLANAR, capi.INTERLEAVED])
@pytest.mark.parametrize("type_in", [F16, BF16, F32])
def test_matches_definition(type_in, axis, order, block_rows):
    rng = np.random.default_rng(7)
    for i, (batch, rows, k) in enumerate(SHAPES):
        type_out = E4M3 if i % 2 else E5M2
        x = _signal(rng, batch, rows, k, type_in)
        got, scale = _run(x, type_in, type_out, axis, order, block_rows)
        _check(x, type_out, block_rows, got, scale)


@pytest.mark.parametrize("order", [capi.ROW_MAJOR, capi.COL_MAJOR])
@pytest.mark.parametrize("type_out", [E4M3, E5M2])
def test_special_values(type_out, order):
    """NaN and infinities stay out of the maximum; tiny and huge blocks keep a finite factor."""
    import torch

    rng = np.random.default_rng(8)
    x = rng.standard_normal((1, 2, 8, 256)).astype(np.float32)
    x[0, 0, 0, 3], x[0, 1, 0, 4], x[0, 0, 1, 130] = np.nan, np.inf, -np.inf
    x[0, :, 2] = np.nan
    x[0, :, 3] = np.inf
    x[0, :, 4] *= np.float32(1e-40)  # denormal
    x[0, :, 5] *= np.float32(5e37)
    x[0, :, 6] = np.float32(np.finfo(np.float32).max)
    x[0, :, 7] = np.float32(1e-45)
    x = torch.from_numpy(x)
    for block_rows in (1, 128):
        got, scale = _run(x, F32, type_out, capi.PLANAR, order, block_rows)
        _check(x, type_out, block_rows, got, scale)
        assert np.isfinite(scale).all() and (scale > 0).all()


def test_ties_round_to_even():
    """Values halfway between two fp8 values: an amax of FMAX makes the scale exactly one."""
    import torch

    for code in (E4M3, E5M2):
        q = np.unique(bu.round_fp8(np.linspace(0, bu.FMAX[code], 4001), code))
        mid = (q[1:] + q[:-1]) / 2
        k = len(mid) + 1
        x = np.zeros((1, 2, 2, 128 * bu.ceil(k, 127)), np.float32)
        for i in range(0, len(mid), 127):
            x[0, 0, 0, i // 127 * 128:][: len(mid[i:i + 127])] = mid[i:i + 127]
        x[0, 1, 0, ::128] = bu.FMAX[code]
        x[0, :, 1] = -x[0, :, 0]
        x = torch.from_numpy(x)
        got, scale = _run(x, F32, code, capi.PLANAR, capi.ROW_MAJOR, 1)
        assert (scale == 1).all()
        _check(x, code, 1, got, scale)


@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("order", [capi.ROW_MAJOR, capi.COL_MAJOR])
def test_conjugate_is_the_same_with_the_other_sign(order, block_rows):
    import torch

    rng = np.random.default_rng(20)
    batch, rows, k = 2, 70, 300
    x = _signal(rng, batch, rows, k, F32)
    d_in = bu.lay_out(x, capi.PLANAR, order).cuda()
    got = []
    for conjugate in (False, True):
        q = torch.empty((batch, 2, rows, capi.operand_pitch(k)), dtype=torch.uint8, device="cuda")
        s = torch.empty((batch, 3, bu.ceil(rows, block_rows)), device="cuda")
        capi.quantize(batch, rows, k, F32, E4M3, d_in.data_ptr(), q.data_ptr(), s.data_ptr(),
                      gu.stream_handle(), input_mem_order=order, block_rows=block_rows,
                      conjugate=conjugate)
        got.append((q.view(torch.float8_e4m3fn).float(), s))
    assert torch.equal(got[0][1], got[1][1])
    assert torch.equal(got[0][0][:, 0], got[1][0][:, 0])
    assert torch.equal(got[0][0][:, 1], -got[1][0][:, 1])


def test_side_stream_and_replayed_graph():
    import torch

    rng = np.random.default_rng(9)
    x = _signal(rng, 2, 200, 384, F16)
    side = torch.cuda.Stream()
    got, scale = _run(x, F16, E4M3, capi.PLANAR, capi.ROW_MAJOR, 1, stream=side.cuda_stream)
    _check(x, E4M3, 1, got, scale)
    d_in = x.cuda()
    q = torch.zeros(2 * 2 * 200 * 384, dtype=torch.uint8, device="cuda")
    s = torch.zeros(2 * 3 * 200, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        capi.quantize(2, 200, 384, F16, E4M3, d_in.data_ptr(), q.data_ptr(), s.data_ptr(),
                      gu.stream_handle())
    x2 = _signal(rng, 2, 200, 384, F16)
    d_in.copy_(x2)
    graph.replay()
    torch.cuda.synchronize()
    _check(x2, E4M3, 1, q.view(torch.float8_e4m3fn).double().cpu().numpy().reshape(2, 2, 200, 384),
           s.cpu().numpy().reshape(2, 3, 200))


def test_more_blocks_than_the_grid_holds():
    """Every kernel form walks its items in a loop: compare with the same rows in small calls."""
    import torch

    batch, rows, k = 2, 5000, 1408
    gen = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn((batch, 2, rows, k), generator=gen, device="cuda").half()
    for order, block_rows in ((capi.ROW_MAJOR, 1), (capi.ROW_MAJOR, 128), (capi.COL_MAJOR, 1),
                              (capi.COL_MAJOR, 128)):
        d_in = bu.lay_out(x, capi.PLANAR, order)
        q = torch.empty((batch, 2, rows, k), dtype=torch.uint8, device="cuda")
        s = torch.empty((batch, k // 128, bu.ceil(rows, block_rows)), device="cuda")
        capi.quantize(batch, rows, k, F16, E4M3, d_in.data_ptr(), q.data_ptr(), s.data_ptr(),
                      gu.stream_handle(), input_mem_order=order, block_rows=block_rows)
        for r0, r1 in ((0, 128), (2560, 2688), (4992, 5000)):
            part = x[1:2, :, r0:r1].cpu()
            want, want_scale = bu.quantize(part.float().numpy(), E4M3, block_rows)
            got = q[1:2, :, r0:r1].contiguous().view(torch.float8_e4m3fn).double().cpu().numpy()
            np.testing.assert_array_equal(got, want)
            b0, b1 = r0 // block_rows, bu.ceil(r1, block_rows)
            np.testing.assert_array_equal(s[1:2, :, b0:b1].cpu().numpy(), want_scale)
