"""Every form of the block-scaled GEMM by hand: tiles of 64 and 128 columns, whole tiles and blocks dealt
out in equal runs, over K longer than the stages and more tiles than one per CTA."""
import numpy as np
import pytest

import block_util as bu
import gpu_util as gu
from ccglib_b200 import capi
from test_gpu_scaled_gemm import _check, _run, _values

pytestmark = pytest.mark.gpu

E4M3, E5M2 = capi.FLOAT8E4M3, capi.FLOAT8E5M2
F16, BF16, F32 = capi.FLOAT16, capi.BFLOAT16, capi.FLOAT32
PLANAR, INTER, ROW, COL = capi.PLANAR, capi.INTERLEAVED, capi.ROW_MAJOR, capi.COL_MAJOR


@pytest.fixture(params=[(64, 0), (64, 1), (128, 0), (128, 1)], ids=["64", "64-runs", "128", "128-runs"])
def form(request, monkeypatch):
    bn, runs = request.param
    monkeypatch.setenv("CCGLIB_B200_SCALED_BN", str(bn))
    monkeypatch.setenv("CCGLIB_B200_SCALED_RUNS", str(runs))
    return bn, runs


def _case(form, seed, batch, m, n, k, ta, tb, type_out, ga, gb, axis=PLANAR, order=ROW, c0=None, alpha=(1.0, 0.0),
          beta=(0.0, 0.0)):
    rng = np.random.default_rng(seed)
    a, sa = bu.random_operand(rng, batch, m, k, ta, ga)
    b, sb = bu.random_operand(rng, batch, n, k, tb, gb)
    # float16 holds the result: the scales' largest product times a block's sums of at most 2^26 .. 2^40
    if type_out == F16:
        sb = sb * np.float32(2.0 ** -8)
    plan = capi.ScaledGemmPlan(batch, m, n, k, ta, tb, type_out, ga, gb, axis, order, alpha=alpha, beta=beta)
    assert plan.tile["bn"] == form[0] and (plan.tile["runs"] > 0) == bool(form[1])
    want, s_re, s_im = bu.scaled_product(_values(a, k), sa.numpy(), ga, _values(b, k), sb.numpy(), gb)
    shape = bu.c_shape(batch, m, n, axis, order)
    if beta != (0.0, 0.0):
        import torch

        c0 = torch.from_numpy(rng.standard_normal(shape)).to(bu.torch_type(type_out))
        old = bu.canonical_c(c0, axis, order).double().numpy()
        old = old[:, 0] + 1j * old[:, 1]
        want = complex(*alpha) * want + complex(*beta) * old
        mag = np.abs(old.real) + np.abs(old.imag)
        s_re = s_im = (abs(alpha[0]) + abs(alpha[1])) * (s_re + s_im) + (abs(beta[0]) + abs(beta[1])) * mag
    c = _run(plan, a, sa, b, sb, shape, type_out, c0)
    _check(bu.canonical_c(c, axis, order), want, s_re, s_im, k, type_out)


@pytest.mark.parametrize("ga, gb", [(1, 1), (1, 128), (128, 1), (128, 128)])
@pytest.mark.parametrize("m, n, k", [(300, 264, 1024), (261, 300, 1500), (70, 650, 1000), (650, 70, 1000)])
def test_block_forms(form, m, n, k, ga, gb):
    _case(form, 51, 2, m, n, k, E4M3, E4M3, F32, ga, gb)


@pytest.mark.parametrize("order", [ROW, COL])
@pytest.mark.parametrize("axis", [PLANAR, INTER])
@pytest.mark.parametrize("type_out", [F32, F16, BF16])
def test_outputs(form, type_out, axis, order):
    # aligned rows (through the TMA unit where row-major) and odd ones
    for m, n in ((256, 264), (203, 133)):
        _case(form, 52, 1, m, n, 1100, E4M3, E4M3, type_out, 1, 1, axis, order)


@pytest.mark.parametrize("ta, tb", [(E4M3, E5M2), (E5M2, E4M3), (E5M2, E5M2)])
def test_types(form, ta, tb):
    _case(form, 53, 2, 150, 260, 1000, ta, tb, F32, 1, 128)


@pytest.mark.parametrize("type_out, axis, order", [(F32, PLANAR, ROW), (BF16, INTER, ROW), (F16, INTER, COL)])
def test_alpha_beta(form, type_out, axis, order):
    for n in (264, 263):
        _case(form, 54, 1, 140, n, 900, E4M3, E4M3, type_out, 1, 128, axis, order, alpha=(0.5, -0.25),
              beta=(-1.5, 2.0))


@pytest.mark.parametrize("gb", [1, 128])
def test_several_tiles_per_cta(form, gb):
    """More tiles than SMs (equal runs are for at most four per SM): accumulators, stages and staging tiles go on from one to the next."""
    _case(form, 55, 15, 512, 513, 1040, E4M3, E4M3, BF16, 1, gb)
    _case(form, 56, 15, 512, 512, 400, E4M3, E4M3, F32, 1, gb)


@pytest.mark.parametrize("k", [1, 128, 129, 256, 384, 512])
def test_short_k_and_many_tiles(k, monkeypatch):
    for bn in (64, 128):
        monkeypatch.setenv("CCGLIB_B200_SCALED_BN", str(bn))
        monkeypatch.setenv("CCGLIB_B200_SCALED_RUNS", "0")
        _case((bn, 0), 57, 40, 400, 260, k, E4M3, E4M3, F32, 1, 128)
