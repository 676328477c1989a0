"""Values at the ends of f32's range in the operators of a step's rest."""
import numpy as np
import pytest

import step_oracle as so
from test_gpu_moe import Layer

pytestmark = pytest.mark.gpu

STEP = 2.0**-149  # f32's smallest


# ------------------------------------------------------------------ experts

def check_small(m, x, got, residual=None):
    """step_oracle.moe's bound, and f32's steps at its lower end.  Of h: its
    rounding, half a step, and the product's with gate or up half a step off, less
    than half a step for |gate|, |up| < 0.4: a step times the weights of down.  Of y:
    at most eight sums or 32 weighted products, each rounded twice: 32 steps."""
    y, ids, p = got
    want, bound, we, wp = so.moe(x, m.router, m.gate, m.up, m.down, m.k, m.normalise, residual)
    assert np.array_equal(ids, we)
    assert np.all(np.abs(p - wp) <= 4 * so.H * wp + STEP)
    down = np.abs(so.weights(*m.down)).sum(2)  # [experts, dim]
    bound = bound + STEP * ((wp[..., None] * down[we]).sum(1) + 32)
    d = np.abs(y - want)
    assert np.all(d <= bound), (float(d.max()), float((d / bound).max()))


@pytest.mark.parametrize("dim,hidden", [(256, 128), (96, 160), (512, 576)])
@pytest.mark.parametrize("size", [-45, -57, -60, -100, -114, -122, -126, -147])
@pytest.mark.parametrize("rows", [1, 6, 30, 170])
def test_rows_of_small_values(ctx, rng, rows, size, dim, hidden):
    """x, or h that is its square, down to the smallest values there are, beside
    ordinary rows."""
    m = Layer(ctx, rng, dim, hidden, 16, 4)
    x = rng.standard_normal((rows, dim)) * 2.0**size
    x[1::3] = rng.standard_normal((len(x[1::3]), dim))
    x = x.astype(np.float32)
    x[0, :2] = 2.0**size, 0.0
    check_small(m, x, m.run(x))
    res = rng.standard_normal((rows, dim)).astype(np.float32)
    check_small(m, x, m.run(x, res), res)


@pytest.mark.parametrize("hidden", [128, 96])
@pytest.mark.parametrize("rows,n", [(1, 500), (40, 500), (100, 500), (300, 70)])
def test_small_rows_under_small_weights(ctx, rng, rows, n, hidden):
    """h near f32's lower end, large matrices behind it, and p of 1 / n."""
    m = Layer(ctx, rng, 64, hidden, n, 3, normalise=False)
    m.down = so.q4(rng, n, 64, hidden, scale=90.0)
    m.upload()
    for size in (-56, -60, -62):
        x = (rng.standard_normal((rows, 64)) * 2.0**size).astype(np.float32)
        check_small(m, x, m.run(x))
