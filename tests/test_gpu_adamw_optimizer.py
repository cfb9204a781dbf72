"""llp_optim.AdamW in an ordinary loop on the GPU."""
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


def test_zero_grad_frees_the_gradients():
    import llp_optim
    p = torch.nn.Parameter(torch.zeros(1 << 22, device=DEV))
    opt = llp_optim.AdamW([p])
    p.grad = torch.ones_like(p)
    opt.step()
    torch.cuda.synchronize()
    held = torch.cuda.memory_allocated()
    opt.zero_grad()
    assert held - torch.cuda.memory_allocated() >= 4 << 22


@pytest.mark.parametrize("bits", [32, 8])
def test_a_loop_with_fresh_gradients(bits):
    """zero_grad / backward / step, with allocations between that move the gradients: as with gradients that stay."""
    import llp_optim
    gen = torch.Generator().manual_seed(3)
    w0, b0 = torch.randn(70, 33, generator=gen), torch.randn(33, generator=gen)
    xs = [torch.randn(20, 70, generator=gen).to(DEV) for _ in range(6)]
    got = []
    for fresh in (True, False):
        w, b = torch.nn.Parameter(w0.to(DEV)), torch.nn.Parameter(b0.to(DEV))
        opt, held = llp_optim.AdamW([w, b], lr=0.01, state_bits=bits, seed=4), []
        for x in xs:
            opt.zero_grad(set_to_none=fresh)
            if fresh:
                held.append(torch.empty(70 * 33, device=DEV))       # takes the block that the gradient left
            (x @ w + b).square().mean().backward()
            opt.step()
        st = opt.state_dict()["state"]
        assert float(st[0]["step"]) == len(xs)
        got.append([w.detach(), b.detach(), *(t for s in st.values() for t in s.values())])
    assert all(torch.equal(a, b) for a, b in zip(*got))


def test_a_transposed_gradient_is_refused():
    import llp_optim
    p, g = torch.nn.Parameter(torch.zeros(6, 6, device=DEV)), torch.randn(6, 6, device=DEV)
    opt = llp_optim.AdamW([p])
    p.grad = g
    opt.step()
    before, p.grad = p.detach().clone(), g.t()
    with pytest.raises(ValueError, match="contiguous"):
        opt.step()
    assert torch.equal(p, before) and float(opt.state_dict()["state"][0]["step"]) == 1


def test_replaced_moments_are_the_ones_that_step():
    import llp_optim
    p = torch.nn.Parameter(torch.zeros(100, device=DEV))
    opt = llp_optim.AdamW([p])
    p.grad = torch.ones(100, device=DEV)
    opt.step()
    old = opt.state[p]["exp_avg_sq"]
    opt.state[p]["exp_avg_sq"] = torch.full_like(old, 0.5)
    kept = old.clone()
    opt.step()
    assert torch.equal(old, kept)
    assert (opt.state[p]["exp_avg_sq"] - (0.999 * 0.5 + 0.001)).abs().max() <= 4 * 2.0 ** -24
