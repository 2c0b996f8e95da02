"""Overlapping input and output of the orthogonalisation: only the same planar array of the output's type may
be both; everything else is refused before anything runs."""
import pytest

import gpu_util as gu
from ccglib_b200 import capi

pytestmark = pytest.mark.gpu

F16, BF16, F32 = capi.FLOAT16, capi.BFLOAT16, capi.FLOAT32


# in one launch (a CTA or a cluster per matrix) and in three launches per step
@pytest.mark.parametrize("batch, m, n", [(300, 8, 12), (3, 20, 200), (2, 130, 140)])
@pytest.mark.parametrize("type_in, type_out, axis, offset", [
    (F32, F16, capi.PLANAR, 0),         # the output of a matrix lies on the input of others
    (F32, BF16, capi.INTERLEAVED, 0),
    (F16, F16, capi.INTERLEAVED, 0),    # another layout
    (F16, BF16, capi.PLANAR, 0),        # another type
    (F16, F16, capi.PLANAR, 2),         # shifted by a value
    (F16, F16, capi.PLANAR, -2),
    (F32, F16, capi.PLANAR, 4),
])
def test_refused(batch, m, n, type_in, type_out, axis, offset):
    import torch

    plan = capi.OrthogonalizePlan(batch, m, n, type_in, type_out, 2, input_complex_axis=axis)
    before = torch.randn(batch * 2 * m * n + 64, device="cuda")
    x = before.clone()
    with pytest.raises(capi.Error) as err:
        plan.run(x.data_ptr() + 64, x.data_ptr() + 64 + offset, gu.stream_handle())
    assert err.value.status == capi.INVALID_ARGUMENT and "overlap" in str(err.value)
    torch.cuda.synchronize()
    assert torch.equal(x, before)


@pytest.mark.parametrize("type_in", [F16, F32])
def test_neighbours_are_no_overlap(type_in):
    """Output right behind the input, and right in front of it."""
    import torch

    batch, m, n = 2, 16, 24
    size, width = batch * 2 * m * n, 4 if type_in == F32 else 2
    dtype = torch.float32 if type_in == F32 else torch.float16
    x = torch.randn(size, device="cuda").to(dtype)
    plan = capi.OrthogonalizePlan(batch, m, n, type_in, F16, 2)
    want = torch.empty(size, dtype=torch.float16, device="cuda")
    plan.run(x.data_ptr(), want.data_ptr(), gu.stream_handle())
    for first in ("input", "output"):
        buf = torch.zeros(size * (width + 2), dtype=torch.uint8, device="cuda")
        at_in, at_out = (0, size * width) if first == "input" else (size * 2, 0)
        buf[at_in:at_in + size * width] = x.view(torch.uint8)
        plan.run(buf.data_ptr() + at_in, buf.data_ptr() + at_out, gu.stream_handle())
        torch.cuda.synchronize()
        assert torch.equal(buf[at_out:at_out + size * 2].view(torch.float16), want)
        assert torch.equal(buf[at_in:at_in + size * width], x.view(torch.uint8))
