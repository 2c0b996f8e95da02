"""Orthogonalisation of large wide matrices and of matrices with weak directions, against the iteration in
64 bits with the bound of test_gpu_orthogonalize.py."""
import numpy as np
import pytest

import block_util as bu
from ccglib_b200 import capi
from test_gpu_orthogonalize import CONVERGENT, QUINTIC, _check, _complex, _fro, _input, _iterate, _run

pytestmark = pytest.mark.gpu

F16, BF16, F32 = capi.FLOAT16, capi.BFLOAT16, capi.FLOAT32


@pytest.mark.parametrize("m, n", [(600, 4000), (520, 1111), (1024, 1500), (4000, 600), (1111, 520)])
@pytest.mark.parametrize("type_in, type_out, coefficients, steps", [(F32, F16, QUINTIC, 3), (BF16, BF16, CONVERGENT, 2)])
def test_large(m, n, type_in, type_out, coefficients, steps):
    """Wide ones contract over K-contiguous rows in S and read X with N as the other axis in the update."""
    rng = np.random.default_rng(61)
    x = _input(rng, 1, m, n, type_in)
    plan = capi.OrthogonalizePlan(1, m, n, type_in, type_out, steps, coefficients)
    _check(x, _run(plan, x, type_in, type_out, capi.PLANAR), steps, coefficients, type_out)


def _with_singular_values(rng, m, n, s):
    import torch

    def basis(rows):
        q, _ = np.linalg.qr(rng.standard_normal((rows, len(s))) + 1j * rng.standard_normal((rows, len(s))))
        return q

    x = (basis(m) * s) @ basis(n).conj().T
    return torch.from_numpy(np.stack((x.real, x.imag))[None]).float()


@pytest.mark.parametrize("steps, coefficients", [(5, QUINTIC), (8, QUINTIC), (8, CONVERGENT)])
@pytest.mark.parametrize("m, n", [(24, 60), (60, 24), (130, 300), (300, 130)])
def test_weak_directions(m, n, steps, coefficients):
    """Singular values over five decades: within the bound, which grows with what the steps make of the
    float16 roundings of X, and not worse than those roundings in directions that are strong enough."""
    rng = np.random.default_rng(62)
    r = min(m, n)
    x = _with_singular_values(rng, m, n, np.geomspace(1, 1e-5, r))
    plan = capi.OrthogonalizePlan(1, m, n, F32, F16, steps, coefficients)
    got = _run(plan, x, F32, F16, capi.PLANAR)
    xi, gi = _complex(x)[0], _complex(got)[0]
    if m > n:
        xi, gi = xi.T, gi.T
    want, bound, _ = _iterate(xi, steps, coefficients)
    assert _fro(gi - want) <= bound + 2.0 ** -11 * _fro(want) + 2.0 ** -24 * np.sqrt(want.size)


@pytest.mark.parametrize("m, n", [(40, 300), (200, 1024), (1024, 200), (160, 160)])
@pytest.mark.parametrize("decades", [3, 5])
def test_rows_of_different_levels(m, n, decades):
    """Antennas with gains over several decades: faint rows keep their bits beside strong ones (a row's
    error is measured against that row)."""
    import torch

    rng = np.random.default_rng(66)
    gain = 10.0 ** -np.linspace(0, decades, min(m, n))
    gain = gain[:, None] if m <= n else gain[None, :]
    x = torch.from_numpy(rng.standard_normal((1, 2, m, n)) * gain).float()
    plan = capi.OrthogonalizePlan(1, m, n, F32, BF16, 3, CONVERGENT)  # (bfloat16: faint rows of the result too)
    xi, gi = (_complex(v)[0] for v in (x, _run(plan, x, F32, BF16, capi.PLANAR)))
    u, s, v = np.linalg.svd(xi, full_matrices=False)
    s /= _fro(xi)
    for _ in range(3):
        s = s * (CONVERGENT[0] + CONVERGENT[1] * s ** 2 + CONVERGENT[2] * s ** 4)
    want = (u * s) @ v
    if m > n:
        want, gi = want.T, gi.T
    error = np.linalg.norm(gi - want, axis=1) / np.linalg.norm(want, axis=1)
    # half a step of bfloat16 at most, rms 1 / sqrt(3) of that; entries of one row differ little, so a row of n
    # has rms within 10 % of the expected one; the iteration may add a fifth of it
    assert (error <= 1.1 * 1.02 * 2.0 ** -8 / np.sqrt(3)).all(), error.max()


@pytest.mark.parametrize("m, n", [(24, 60), (130, 300)])
def test_rank_deficient(m, n):
    """Directions that are not there stay out: rank 5, the rest rounding noise below float16's of X."""
    rng = np.random.default_rng(63)
    s = np.array([1, 0.8, 0.5, 0.3, 0.2])
    x = _with_singular_values(rng, m, n, s)
    plan = capi.OrthogonalizePlan(1, m, n, F32, F16, 4, CONVERGENT)
    got = _complex(_run(plan, x, F32, F16, capi.PLANAR))[0]
    want, bound, _ = _iterate(_complex(x)[0], 4, CONVERGENT)
    assert _fro(got - want) <= bound + 2.0 ** -11 * _fro(want) + 2.0 ** -24 * np.sqrt(want.size)


@pytest.mark.parametrize("coefficients", [
    (1.5, -0.5, 0.0),       # third order: no square
    (1.5, -0.5, 0.001),     # its square would cancel
    (1.0, 0.0, 0.0),        # the matrix over its norm
    (2.0, -1.5, 0.5), (3.0, -3.2, 1.2), (0.5, 0.25, -0.125), (0.0, 0.0, 1.0),
    (20.0, -160.0, 300.0),  # entries of P far above one
])
@pytest.mark.parametrize("m, n", [(24, 60), (130, 300), (300, 130), (200, 200)])
def test_coefficients(m, n, coefficients):
    """Every way in which a I + b S + c S^2 is computed."""
    rng = np.random.default_rng(64)
    # (the last map would take three steps past float32: its results are no float16 either way)
    for steps in (1, 3) if coefficients[0] < 20 else (1,):
        x = _input(rng, 2, m, n, F32)
        plan = capi.OrthogonalizePlan(2, m, n, F32, F16, steps, coefficients)
        _check(x, _run(plan, x, F32, F16, capi.PLANAR), steps, coefficients, F16)


# A rounding is off by at most half a step, 2^-11 (float16) or 2^-8 (bfloat16) of the value, and evenly
# distributed up to that: rms at most 1 / sqrt(3) of it, relative to the Frobenius norm.  10 % on top are for the
# iteration, whose iterates have about 20 bits: roundings of 2^-21 in X, S and P, which eight steps
# multiply by less than 20 (single float16 iterates, 2^-12, end at 3.8e-3 at most), are 1e-5, and add to the
# output's as squares.
@pytest.mark.parametrize("type_in, type_out, half_step", [(F32, F16, 2.0 ** -11), (F16, F16, 2.0 ** -11),
                                                          (F32, BF16, 2.0 ** -8)])
@pytest.mark.parametrize("batch, m, n, steps, coefficients", [
    (1, 256, 1024, 8, CONVERGENT), (2, 1024, 256, 8, CONVERGENT), (1, 256, 256, 5, QUINTIC),
    (1, 400, 420, 8, QUINTIC), (1, 200, 2000, 8, QUINTIC), (3, 40, 72, 8, QUINTIC)])
def test_the_output_rounding_is_what_is_lost(batch, m, n, steps, coefficients, type_in, type_out, half_step):
    """The result is as near as its type allows, in every form, whatever the input's type."""
    rng = np.random.default_rng(65)
    x = _input(rng, batch, m, n, type_in)
    plan = capi.OrthogonalizePlan(batch, m, n, type_in, type_out, steps, coefficients)
    for xi, gi in zip(_complex(x), _complex(_run(plan, x, type_in, type_out, capi.PLANAR))):
        u, s, v = np.linalg.svd(xi, full_matrices=False)
        s /= _fro(xi)
        for _ in range(steps):
            s = s * (coefficients[0] + coefficients[1] * s ** 2 + coefficients[2] * s ** 4)
        want = (u * s) @ v
        assert _fro(gi - want) <= 1.1 * half_step / np.sqrt(3) * _fro(want)
