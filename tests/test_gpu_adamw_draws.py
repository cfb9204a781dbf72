"""The AdamW kernel's stochastic rounding, draw by draw (csrc/adamw.hip, llp_optim)."""
import numpy as np
import pytest
import torch

from oracle import lowbit_oracle as Q

pytestmark = pytest.mark.gpu

DEV = "cuda"
B1, B2 = 0.9, 0.999


@pytest.fixture(scope="module", autouse=True)
def _lib():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    import llp_hip
    llp_hip.lib()


def test_every_draw_is_decided_exactly():
    """From the f32 moments m', v' (elementary f32 operations, each rounded once) the codes are those that exact arithmetic
    picks.  Above 2^-6 scales m's draw adds into the bits below its code: exact.  Below, 2^-6 is added first, off by 2^-30 of
    codes 2^-9 apart: 2^-21 of their distance.  The second moment's share is of a difference rounded once: 2^-24."""
    import llp_optim
    n, step, seed = 1 << 18, 40, 0xABCDEF
    gen = torch.Generator().manual_seed(21)
    size = 1e-3 * torch.exp(torch.randn(n, generator=gen))
    g = torch.randn(n, generator=gen) * size
    m0, r0 = (0.3 * torch.randn(n, generator=gen) * size).double().numpy(), size.double().numpy()
    sm, sr = Q.scales8(np.abs(m0), True), Q.scales8(r0, False)
    cm, cr = (Q.round8(x, np.full(n, 0x8000), s, signed)[0] for x, s, signed in ((m0, sm, True), (r0 * r0, sr, False)))
    st = [torch.from_numpy(a.copy()).to(DEV) for a in (cm, cr, sm, sr)]
    llp_optim.AdamWTable([torch.zeros(n, device=DEV)], [g.to(DEV)], [st[0]], [st[1]], [st[2]], [st[3]]).step(
        torch.full((1,), step, dtype=torch.int64, device=DEV), betas=(B1, B2), seed=seed)
    got_m, got_r, got_sm, got_sr = (t.cpu().numpy() for t in st)
    f = np.float32
    m, r = Q.values8(cm, sm, True).astype(f), Q.values8(cr, sr, False).astype(f)
    gn = g.numpy()
    m = f(B1) * m + f(1 - B1) * gn
    v = f(B2) * (r * r) + (f(1 - B2) * gn) * gn
    assert m.dtype == v.dtype == f
    m, v = m.astype(np.float64), v.astype(np.float64)
    w = Q.draws16(n, 0, step + 1, seed)
    assert np.array_equal(got_sm, Q.scales8(np.abs(m), True))
    assert np.array_equal(got_sr, Q.scales8(np.sqrt(v).astype(f), False))
    want, room = Q.round8(m, w, got_sm, True)
    low = np.abs(m) < 2.0 ** -6 * np.exp2(np.repeat(got_sm.astype(np.float64) - 127, 32))
    sure = ~low | (room > 2.0 ** -20)
    assert np.array_equal(np.where(want & 127, want, 0)[sure], np.where(got_m & 127, got_m, 0)[sure])
    want, room = Q.round8(v, w, got_sr, False)
    assert np.array_equal(want[room > 2.0 ** -22], got_r[room > 2.0 ** -22])
