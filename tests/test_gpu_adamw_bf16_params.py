"""AdamW on bf16 params: their working copies, and 8-bit moments beside them (csrc/adamw.hip, llp_optim)."""
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"


@pytest.fixture(scope="module", autouse=True)
def _lib():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    import llp_hip
    llp_hip.lib()


def _table(p, g, bits, **kw):
    import llp_optim
    n = p.numel()
    if bits == 32:
        m, v = [torch.zeros(n, device=DEV)], [torch.zeros(n, device=DEV)]
    else:
        (m, ms), (v, vs) = llp_optim.AdamWTable.state8(n, DEV), llp_optim.AdamWTable.state8(n, DEV)
        m, v, kw = [m], [v], dict(kw, exp_avg_scale=[ms], exp_avg_sq_scale=[vs])
    return llp_optim.AdamWTable([p], [g], m, v, **kw), [*m, *v, *kw.get("exp_avg_scale", []), *kw.get("exp_avg_sq_scale", [])]


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("ld", [0, 57])
def test_copies_hold_the_param(bits, dtype, ld):
    g = torch.Generator(device=DEV).manual_seed(1)
    p = torch.randn(70, 45, generator=g, device=DEV).bfloat16()
    copy = torch.zeros(70, ld or 45, dtype=dtype, device=DEV)
    copy_t = torch.zeros(45, 70, dtype=dtype, device=DEV)
    tab, _ = _table(p, torch.randn(70, 45, generator=g, device=DEV), bits, copies=[(copy, ld) if ld else copy], copies_t=[copy_t])
    before = p.clone()
    tab.step(torch.zeros(1, dtype=torch.int64, device=DEV), lr=0.01)
    assert not torch.equal(p, before)
    assert torch.equal(copy[:, :45], p.to(dtype)) and torch.equal(copy_t, p.t().to(dtype)) and (copy[:, 45:] == 0).all()


# at sizes either side of those at which large steps pass by the caches
@pytest.mark.parametrize("bits,n", [(32, 5003), (8, 5003), (32, (1 << 24) + 2061), (8, (1 << 25) + 2061)])
@pytest.mark.parametrize("gtype", [torch.float32, torch.bfloat16])
def test_bf16_params_step_as_f32_ones(bits, n, gtype):
    """The moments do not depend on the param's type; from the same values the new param is the f32 one rounded."""
    g = torch.Generator(device=DEV).manual_seed(2)
    p = torch.randn(n, generator=g, device=DEV).bfloat16()
    q, grad = p.float(), (1e-3 * torch.randn(n, generator=g, device=DEV)).to(gtype)
    (a, sa), (b, sb) = _table(p, grad, bits), _table(q, grad, bits)
    for t in range(2):
        q.copy_(p)
        ctr = torch.full((1,), t, dtype=torch.int64, device=DEV)
        a.step(ctr, lr=0.01, seed=3), b.step(ctr, lr=0.01, seed=3)
        assert torch.equal(p, q.bfloat16()), t
        assert len(sa) == (2 if bits == 32 else 4) and all(torch.equal(x, y) for x, y in zip(sa, sb)), t
