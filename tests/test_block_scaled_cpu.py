"""Refusals of the block quantiser and the block-scaled GEMM: found before CUDA is touched."""
import pytest

from ccglib_b200 import capi

E4M3, F16, F32 = capi.FLOAT8E4M3, capi.FLOAT16, capi.FLOAT32


def _status(call, *args, **kw):
    with pytest.raises(capi.Error) as err:
        call(*args, **kw)
    return err.value.status, str(err.value)


@pytest.mark.parametrize("args, kw, status, text", [
    ((0, 1, 1, F16, E4M3, 256, 512, 768), {}, capi.INVALID_ARGUMENT, "positive"),
    ((1, 0, 1, F16, E4M3, 256, 512, 768), {}, capi.INVALID_ARGUMENT, "positive"),
    ((1, 1, 0, F16, E4M3, 256, 512, 768), {}, capi.INVALID_ARGUMENT, "positive"),
    ((1, 1 << 31, 1, F16, E4M3, 256, 512, 768), {}, capi.INVALID_ARGUMENT, "too large"),
    ((1 << 29, 1 << 30, 1 << 30, F16, E4M3, 256, 512, 768), {}, capi.INVALID_ARGUMENT, "too large"),
    ((1, 1, 1, E4M3, E4M3, 256, 512, 768), {}, capi.UNSUPPORTED, "input must be"),
    ((1, 1, 1, F16, F16, 256, 512, 768), {}, capi.UNSUPPORTED, "output must be"),
    ((1, 1, 1, F16, E4M3, 256, 512, 768), {"block_rows": 64}, capi.INVALID_ARGUMENT, "1 or 128 rows"),
    ((1, 1, 1, F16, E4M3, 256, 512, 768), {"input_complex_axis": 2}, capi.INVALID_ARGUMENT, "axis"),
    ((1, 1, 1, F16, E4M3, 256, 512, 768), {"input_mem_order": 2}, capi.INVALID_ARGUMENT, "order"),
    ((1, 1, 1, F16, E4M3, 256, 512, 768), {"conjugate": 2}, capi.INVALID_ARGUMENT, "conjugate"),
    ((1, 1, 1, F16, E4M3, 0, 512, 768), {}, capi.INVALID_ARGUMENT, "null"),
    ((1, 1, 1, F16, E4M3, 256, 0, 768), {}, capi.INVALID_ARGUMENT, "null"),
    ((1, 1, 1, F16, E4M3, 256, 512, 0), {}, capi.INVALID_ARGUMENT, "null"),
    ((1, 1, 1, F16, E4M3, 258, 512, 768), {}, capi.INVALID_ARGUMENT, "aligned"),
    ((1, 1, 1, F16, E4M3, 256, 520, 768), {}, capi.INVALID_ARGUMENT, "aligned"),
    ((1, 1, 1, F16, E4M3, 256, 512, 770), {}, capi.INVALID_ARGUMENT, "aligned"),
])
def test_quantize_refuses(args, kw, status, text):
    got, message = _status(capi.quantize, *args, **kw)
    assert got == status and text in message


@pytest.mark.parametrize("args, kw, status, text", [
    ((0, 1, 1, 1, E4M3, E4M3, F32), {}, capi.INVALID_ARGUMENT, "positive"),
    ((1, 0, 1, 1, E4M3, E4M3, F32), {}, capi.INVALID_ARGUMENT, "positive"),
    ((1, 1, 0, 1, E4M3, E4M3, F32), {}, capi.INVALID_ARGUMENT, "positive"),
    ((1, 1, 1, 0, E4M3, E4M3, F32), {}, capi.INVALID_ARGUMENT, "positive"),
    ((1, 1 << 30, 1, 1, E4M3, E4M3, F32), {}, capi.INVALID_ARGUMENT, "too large"),
    ((1, 1, 1, 1 << 31, E4M3, E4M3, F32), {}, capi.INVALID_ARGUMENT, "too large"),
    ((1, 1, 1, 1, F16, E4M3, F32), {}, capi.UNSUPPORTED, "A and B must be"),
    ((1, 1, 1, 1, E4M3, F16, F32), {}, capi.UNSUPPORTED, "A and B must be"),
    ((1, 1, 1, 1, E4M3, E4M3, capi.INT32), {}, capi.UNSUPPORTED, "output must be"),
    ((1, 1, 1, 1, E4M3, E4M3, F32), {"a_block_rows": 2}, capi.INVALID_ARGUMENT, "1 or 128 rows"),
    ((1, 1, 1, 1, E4M3, E4M3, F32), {"b_block_rows": 0}, capi.INVALID_ARGUMENT, "1 or 128 rows"),
    ((1, 1, 1, 1, E4M3, E4M3, F32), {"c_complex_axis": 3}, capi.INVALID_ARGUMENT, "axis"),
    ((1, 1, 1, 1, E4M3, E4M3, F32), {"c_mem_order": -1}, capi.INVALID_ARGUMENT, "order"),
])
def test_scaled_gemm_plan_refuses(args, kw, status, text):
    got, message = _status(capi.ScaledGemmPlan, *args, **kw)
    assert got == status and text in message


def test_operand_pitch():
    assert [capi.operand_pitch(k) for k in (1, 16, 17, 128, 1990)] == [16, 16, 32, 128, 2000]


@pytest.mark.parametrize("args, kw, status, text", [
    ((0, 4, 4, F16, F16), {}, capi.INVALID_ARGUMENT, "positive"),
    ((1, 0, 4, F16, F16), {}, capi.INVALID_ARGUMENT, "positive"),
    ((1, 4, 0, F16, F16), {}, capi.INVALID_ARGUMENT, "positive"),
    ((1, 1 << 30, 4, F16, F16), {}, capi.INVALID_ARGUMENT, "too large"),
    ((1 << 29, 1 << 20, 1 << 20, F16, F16), {}, capi.INVALID_ARGUMENT, "too large"),
    ((1, 4, 4, E4M3, F16), {}, capi.UNSUPPORTED, "input must be"),
    ((1, 4, 4, F16, F32), {}, capi.UNSUPPORTED, "output must be"),
    ((1, 4, 4, F16, F16), {"steps": 0}, capi.INVALID_ARGUMENT, "steps"),
    ((1, 4, 4, F16, F16), {"steps": 1001}, capi.INVALID_ARGUMENT, "steps"),
    ((1, 4, 4, F16, F16), {"coefficients": (1.0, float("nan"), 0.0)}, capi.INVALID_ARGUMENT, "finite"),
    ((1, 4, 4, F16, F16), {"input_complex_axis": 5}, capi.INVALID_ARGUMENT, "axis"),
])
def test_orthogonalize_plan_refuses(args, kw, status, text):
    got, message = _status(capi.OrthogonalizePlan, *args, **kw)
    assert got == status and text in message
