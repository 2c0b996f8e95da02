"""Bounded waits of kernels that are set up while the kernel before them still runs: the time that one takes
is not part of their own limit."""
import numpy as np
import pytest

import block_util as bu
import gpu_util as gu
from ccglib_b200 import capi

pytestmark = pytest.mark.gpu

E4M3, F32 = capi.FLOAT8E4M3, capi.FLOAT32


@pytest.mark.parametrize("m, n", [(200, 260), (30, 300)])
def test_limit_shorter_than_the_kernel_before(m, n, monkeypatch):
    """A product of a few tiles and a long K leaves most SMs free, where the next one is set up at once.
    Its limit (0.2 ms at least) is far above any of its own waits and far below the run time of the
    first."""
    import torch

    k_long, k, limit = 1 << 19, 384, 400_000
    long_a, long_b = (torch.full((1, 2, r, k_long), 0x38, dtype=torch.uint8, device="cuda") for r in (128, 128))
    ones = torch.ones((1, k_long // 128, 128), device="cuda")
    long_c = torch.empty((1, 2, 128, 128), device="cuda")
    monkeypatch.setenv("CCGLIB_B200_SCALED_RUNS", "0")
    before = capi.ScaledGemmPlan(1, 128, 128, k_long, E4M3, E4M3, F32, 1, 1)
    assert before.tile["runs"] == 0
    monkeypatch.setenv("CCGLIB_B200_WAIT_CYCLES", str(limit))
    plan = capi.ScaledGemmPlan(1, m, n, k, E4M3, E4M3, F32, 1, 128)
    rng = np.random.default_rng(41)
    a, sa = bu.random_operand(rng, 1, m, k, E4M3, 1)
    b, sb = bu.random_operand(rng, 1, n, k, E4M3, 128)
    d = [t.cuda() for t in (a, sa, b, sb)]
    c, want = (torch.full((1, 2, m, n), 7.0, device="cuda") for _ in range(2))
    stream = gu.stream_handle()
    plan.run(*[t.data_ptr() for t in d], want.data_ptr(), stream)
    torch.cuda.synchronize()
    gu.check_device_status()
    start, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    start.record()
    before.run(long_a.data_ptr(), ones.data_ptr(), long_b.data_ptr(), ones.data_ptr(), long_c.data_ptr(), stream)
    plan.run(*[t.data_ptr() for t in d], c.data_ptr(), stream)
    end.record()
    torch.cuda.synchronize()
    gu.check_device_status()
    assert start.elapsed_time(end) > 4 * limit / 1.0e6  # the SM clock is above 1 GHz: 4 limits or more
    assert torch.equal(c, want)
    # 1.0 x 1.0 summed: Re = k - k, Im = 2 k, exact in float32
    assert not long_c[:, 0].any() and (long_c[:, 1] == 2 * k_long).all()


def test_limit_shorter_than_a_long_tile(monkeypatch):
    """The sums of a tile take as long as its K: that is not a wait that has gone wrong."""
    import torch

    monkeypatch.setenv("CCGLIB_B200_ORTH_SMALL", "0")
    rng = np.random.default_rng(42)
    x = torch.from_numpy(rng.standard_normal((1, 2, 300_000, 48))).float().cuda()
    out = [torch.empty((1, 2, 300_000, 48), dtype=torch.float16, device="cuda") for _ in range(2)]
    for i, limit in enumerate(("", "400000")):
        monkeypatch.setenv("CCGLIB_B200_WAIT_CYCLES", limit)
        plan = capi.OrthogonalizePlan(1, 300_000, 48, F32, capi.FLOAT16, 2)
        plan.run(x.data_ptr(), out[i].data_ptr(), gu.stream_handle())
        torch.cuda.synchronize()
        gu.check_device_status()
    assert torch.equal(*out) and out[0].any()
