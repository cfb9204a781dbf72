"""8-bit moments over many steps (the 64-bit restatement in oracle/lowbit_oracle.py, on the CPU): no single update is
far larger than f32 moments give, however the gradients of a block are spread."""
import numpy as np
import pytest

from oracle import lowbit_oracle as Q

B1, B2, EPS, T = 0.9, 0.999, 1e-8, 60
# The largest update, in units of lr.  With f(t) = sqrt(1 - b2^t) / (1 - b1^t) <= 0.317 for t <= 100 an update is f |m'| / sqrt(v').
# A moment at m's least code, 2^-9 2^km, beside a root at its least, 2^-10 2^kr: 2^km < 2 max|m| / 448 and 2^kr >= max r / 496, so their ratio
# is under 4.43 max|m| / max r <= 4.43 (1 - b1) / sqrt(1 - b2) = 14.1, an update of 4.5.  What larger codes hold is off by at most 1/8 (m) and 1/16
# (r): 1.2 of f32's 1.2.  The present gradient alone: 1 at most, at t = 1, and 0.317 0.1 / sqrt(0.001) = 1 later.
BOUND = 6.4


def gradients(n, sigma, active, seed):
    """Sizes log-normal of width sigma, a share `active` of them nonzero at a time."""
    rng = np.random.default_rng(seed)
    scale = 1e-3 * np.exp(sigma * rng.standard_normal(n))
    while True:
        yield (scale * rng.standard_normal(n) * (rng.random(n) < active)).astype(np.float32).astype(np.float64)


@pytest.mark.parametrize("sigma,active", [(1, 1), (1, 0.05), (2, 0.05), (3, 1), (3, 0.05), (4, 0.02)])
def test_updates_stay_bounded(sigma, active):
    n = 16384
    m, r, worst = np.zeros(n), np.zeros(n), 0.0
    for t, g in zip(range(1, T + 1), gradients(n, sigma, active, seed=1)):
        step, m, v = Q.adamw(np.zeros(n), g, m, r * r, t, 1.0, (B1, B2), EPS, 0.0)
        worst = max(worst, np.abs(step).max())
        w = Q.draws16(n, 0, t, 7)
        sm, sv = Q.scales8(np.abs(m), True), Q.scales8(np.sqrt(v), False)
        cm, cv = Q.round8(m, w, sm, True)[0], Q.round8(v, w, sv, False)[0]
        assert ((cv > 0) == (v > 0)).all()
        m, r = Q.values8(cm, sm, True), Q.values8(cv, sv, False)
    assert worst <= BOUND, worst
