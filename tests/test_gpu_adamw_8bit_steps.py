"""The AdamW kernel's 8-bit moments over many steps (csrc/adamw.hip, llp_optim)."""
import pytest
import torch

from oracle import lowbit_oracle as Q
from test_adamw_8bit_steps import B1, B2, BOUND, EPS, T, gradients

pytestmark = pytest.mark.gpu

DEV = "cuda"


@pytest.fixture(scope="module", autouse=True)
def _lib():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    import llp_hip
    llp_hip.lib()


@pytest.mark.parametrize("sigma,active", [(1, 1), (2, 0.05), (3, 1), (3, 0.05), (4, 0.02)])
def test_updates_stay_bounded(sigma, active):
    """As on the CPU, where the bound is derived; a positive second moment never reads back as 0."""
    import llp_optim
    n = 131072 + 45
    p, g = torch.zeros(n, device=DEV), torch.zeros(n, device=DEV)
    (m, ms), (v, vs) = llp_optim.AdamWTable.state8(n, DEV), llp_optim.AdamWTable.state8(n, DEV)
    tab = llp_optim.AdamWTable([p], [g], [m], [v], [ms], [vs])
    ctr, seen = torch.zeros(1, dtype=torch.int64, device=DEV), torch.zeros(n, dtype=torch.bool, device=DEV)
    for t, x in zip(range(T), gradients(n, sigma, active, seed=2)):
        p.zero_(), g.copy_(torch.from_numpy(x)), ctr.fill_(t)
        tab.step(ctr, lr=1.0, betas=(B1, B2), eps=EPS, weight_decay=0.0, seed=7)
        seen |= g != 0
        assert float(p.abs().max()) <= BOUND, t
        assert torch.equal(v > 0, seen)
