"""The quantiser refuses arrays that overlap, before CUDA is touched."""
import pytest

from ccglib_b200 import capi

F32, F16, E4M3 = capi.FLOAT32, capi.FLOAT16, capi.FLOAT8E4M3
# 3 matrices of 5 x 40: 4800 bytes of float32, 1440 bytes of fp8 (pitch 48), 15 scales of 60 bytes
IN, OUT, SCALE = 1 << 20, 1 << 21, 1 << 22


@pytest.mark.parametrize("d_in, d_out, d_scale", [
    (IN, IN, SCALE),              # in place
    (IN, IN + 4784, SCALE),       # the input's last bytes
    (IN, IN - 1424, SCALE),       # the output's last bytes
    (IN, OUT, IN + 4796),
    (IN, OUT, IN - 56),
    (IN, OUT, OUT + 1436),
    (IN, OUT, OUT - 56),
])
def test_quantize_refuses_overlap(d_in, d_out, d_scale):
    with pytest.raises(capi.Error) as err:
        capi.quantize(3, 5, 40, F32, E4M3, d_in, d_out, d_scale)
    assert err.value.status == capi.INVALID_ARGUMENT and "overlap" in str(err.value)


gpu = pytest.mark.gpu


@gpu
def test_quantize_takes_neighbours():
    import torch

    buf = torch.zeros(1 << 14, dtype=torch.uint8, device="cuda")
    buf[:4800] = torch.randn(1200, device="cuda").view(torch.uint8)
    base = buf.data_ptr()
    capi.quantize(3, 5, 40, F32, E4M3, base, base + 4800, base + 4800 + 1440)
    torch.cuda.synchronize()
    scales = buf[6240:6300].view(torch.float32)
    amax = buf[:4800].view(torch.float32).view(3, 2, 5, 40).abs().amax(dim=(1, 3)).flatten()
    # (by a tensor on the CPU: torch may multiply by the reciprocal of a number)
    want = amax.cpu() / torch.full((15,), 448.0)
    assert torch.equal(scales.cpu(), want) and buf[4800:6240].any() and not buf[6300:].any()


@gpu
def test_scaled_gemm_refuses_overlap():
    import torch

    m, n, k = 40, 50, 256
    plan = capi.ScaledGemmPlan(1, m, n, k, E4M3, E4M3, F16, 1, 1)
    sizes = {"a": 2 * m * k, "sa": 4 * 2 * m, "b": 2 * n * k, "sb": 4 * 2 * n}
    buf = torch.zeros(1 << 18, dtype=torch.uint8, device="cuda")
    at, where = buf.data_ptr() + (1 << 15), {}
    for name, size in sizes.items():
        where[name] = at
        at += -(-size // 16) * 16 + (1 << 13)  # gaps wider than C
    c_bytes = 2 * 2 * m * n
    args = [where[name] for name in sizes]
    for name, size in sizes.items():
        for c in (where[name], where[name] + size - 2, where[name] - c_bytes + 2):
            with pytest.raises(capi.Error) as err:
                plan.run(*args, c)
            assert err.value.status == capi.INVALID_ARGUMENT and "overlap" in str(err.value)
        plan.run(*args, where[name] - c_bytes)  # right in front is no overlap
    torch.cuda.synchronize()
    assert capi.device_status() == 0
