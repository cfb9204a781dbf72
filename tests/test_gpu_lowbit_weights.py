"""Weights that MXFP4 evaluation takes as the f32 and bf16 evaluations do: any float type, any layout."""
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


@pytest.mark.parametrize("how", ["transposed", "double", "half"])
def test_weights_of_any_layout_and_type(how):
    import llp_eval as E
    import models
    torch.manual_seed(0)
    mlp, pred = models.MLP(2, 64, 64, 64, 0.0).to(DEV).eval(), models.LinkPredictor("mlp", 64, 64, 1, 2, 0.0).to(DEV).eval()
    x, edges = torch.randn(50, 64, device=DEV), torch.randint(0, 50, (300, 2), device=DEV)
    if how == "half":        # values that a half holds
        with torch.no_grad():
            for m in (mlp, pred):
                for p in m.parameters():
                    p.copy_(p.half())

    def answer():
        h = E.embed_mlp(mlp, x, "mxfp4")
        return h, E.EdgeScorer(pred, dtype="mxfp4")(h, edges)
    want = answer()
    for lin in (mlp.layers[0], pred.lins[0]):
        w = lin.weight.detach()
        lin.weight = torch.nn.Parameter({"transposed": lambda: w.t().contiguous().t(), "double": w.double, "half": w.half}[how]())
    assert all(torch.equal(a, b) for a, b in zip(answer(), want))
