"""Working copies of large AdamW steps, whose params are stored past the caches and read back for the transposed ones."""
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


# past 16 M elements (f32 moments) and 32 M (8-bit ones)
@pytest.mark.parametrize("bits,rows,cols", [(32, 4099, 4111), (8, 5801, 5813)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_copies_of_a_large_param(bits, rows, cols, dtype):
    import llp_optim
    g = torch.Generator(device=DEV).manual_seed(bits)
    n = rows * cols
    p, grad = torch.randn(rows, cols, generator=g, device=DEV), torch.randn(rows, cols, generator=g, device=DEV)
    kw = {}
    if bits == 8:
        (m, ms), (v, vs) = llp_optim.AdamWTable.state8(n, DEV), llp_optim.AdamWTable.state8(n, DEV)
        kw = dict(exp_avg_scale=[ms], exp_avg_sq_scale=[vs])
    else:
        m, v = torch.zeros(n, device=DEV), torch.zeros(n, device=DEV)
    copy, wide = torch.empty(rows, cols, dtype=dtype, device=DEV), torch.full((cols, rows + 9), 7.0, dtype=dtype, device=DEV)
    tab = llp_optim.AdamWTable([p], [grad], [m], [v], copies=[copy], copies_t=[(wide[:, 4:], rows + 9)], **kw)
    ctr, before = torch.zeros(1, dtype=torch.int64, device=DEV), p.clone()
    for t in range(3):
        ctr.fill_(t)
        tab.step(ctr, lr=0.01)
        assert torch.equal(copy, p.to(dtype)) and torch.equal(wide[:, 4:4 + rows], p.t().to(dtype))
    assert (wide[:, :4] == 7).all() and (wide[:, 4 + rows:] == 7).all() and not torch.equal(before, p)
