"""AdamW over a tensor of more than 2^31 elements: slices on either side of the places where offsets pass 31 and 32 bits.

Tolerances as in tests/test_gpu_adamw.py (u = 2^-24): p' 3 u |p| + 24 u of the update's terms, a bf16 param or copy half a step of
2^-8 more; an 8-bit moment within one code (32 scales for m, 16 for the root of v)."""
import numpy as np
import pytest
import torch

from oracle import lowbit_oracle as Q

pytestmark = pytest.mark.gpu

DEV, U = "cuda", 2.0 ** -24
HYPER = dict(lr=0.01, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.05)


@pytest.fixture(scope="module", autouse=True)
def _lib():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    import llp_hip
    llp_hip.lib()


def _f64(t):
    return t.detach().float().cpu().numpy().astype(np.float64)


def test_offsets_past_32_bits():
    import llp_optim
    n = (1 << 31) + 2085
    g = torch.Generator(device=DEV).manual_seed(1)
    p = torch.empty(n, device=DEV).normal_(generator=g)
    grad = torch.empty(n, dtype=torch.bfloat16, device=DEV).normal_(generator=g).mul_(1e-3)
    (m, ms), (v, vs) = llp_optim.AdamWTable.state8(n, DEV), llp_optim.AdamWTable.state8(n, DEV)
    copy = torch.zeros(n, dtype=torch.bfloat16, device=DEV)
    vals = {k: [torch.zeros(n, dtype=torch.bfloat16, device=DEV)] for k in ("exp_avg", "exp_avg_sq")}
    tab = llp_optim.AdamWTable([p], [grad], [m], [v], [ms], [vs], copies=[copy], values=vals)
    at = [slice(0, 4096)] + [slice((1 << b) - 2048, (1 << b) + 2048) for b in (29, 30)] + [slice((1 << 31) - 2048, n)]
    ctr, seed = torch.zeros(1, dtype=torch.int64, device=DEV), 9
    for t in range(2):
        ctr.fill_(t)
        before = [(_f64(p[s]), _f64(grad[s]), m[s].cpu().numpy(), ms[s.start // 32:-(-s.stop // 32)].cpu().numpy(),
                   v[s].cpu().numpy(), vs[s.start // 32:-(-s.stop // 32)].cpu().numpy()) for s in at]
        tab.step(ctr, seed=seed, **HYPER)
        tab.values()
        for s, (p0, g0, m0, ms0, v0, vs0) in zip(at, before):
            m0, r0 = Q.values8(m0, ms0, True), Q.values8(v0, vs0, False)
            rp, rm, rv = Q.adamw(p0, g0, m0, r0 * r0, t + 1, HYPER["lr"], HYPER["betas"], HYPER["eps"], HYPER["weight_decay"])
            terms = 0.9 * np.abs(m0) + 0.1 * np.abs(g0)
            upd = HYPER["lr"] / (1 - 0.9 ** (t + 1)) * terms / (np.sqrt(rv) / np.sqrt(1 - 0.999 ** (t + 1)) + 1e-8)
            tol = 3 * U * np.abs(p0) + 24 * U * upd
            assert (np.abs(_f64(p[s]) - rp) <= tol).all()
            assert torch.equal(copy[s], p[s].bfloat16())
            for x, codes, scales, signed, val in ((rm, m, ms, True, vals["exp_avg"][0]), (np.sqrt(rv), v, vs, False, vals["exp_avg_sq"][0])):
                b = scales[s.start // 32:-(-s.stop // 32)].cpu().numpy()
                got = Q.values8(codes[s].cpu().numpy(), b, signed)
                f = np.repeat(np.exp2(b.astype(np.float64) - 127), 32)[:got.size]
                assert (np.abs(got - x) <= (32 if signed else 16) * f * (1 + 1e-5)).all()
                want = torch.from_numpy(got if signed else got * got).float().bfloat16()
                assert torch.equal(val[s].cpu(), want)
    # the draws of far elements are their own: not those of the elements 2^31 before
    assert not torch.equal(m[(1 << 31):(1 << 31) + 2048], m[:2048])
