"""Every way a training engine updates its parameters obeys clip_norm."""
import pytest
import torch

from hipdsml.data.mnist import synthetic_mnist
from hipdsml.engine.trainer import MlpTrainer
from hipdsml.models.mlp import MlpSpec
from hipdsml.parallel.dist import DistContext

SPEC = MlpSpec((784, 32, 16, 10))
DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def _ctx(dev):
    return DistContext(device=torch.device(dev, 0) if dev == "cuda" else torch.device(dev))


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("scale", [1.0, 0.25, -0.5])
@pytest.mark.parametrize("norm", [0.01, 8.0])
def test_applied_gradients_are_clipped(norm, scale, dev):
    """P -= lr * scale * g with the norm of scale * g limited; g stays as it is."""
    tr = MlpTrainer(SPEC, synthetic_mnist(64, seed=1), batch=16, lr=0.5, seed=3, clip_norm=0.1, ctx=_ctx(dev))
    g = torch.randn(tr.P.numel(), generator=torch.Generator().manual_seed(2))
    g = (g * (norm / float(g.double().norm()))).to(tr.P.device)
    before, keep = tr.P.double(), g.clone()
    tr.apply_gradients(g, scale)
    tr.synchronize()
    step = 0.5 * scale * keep.double()
    size = abs(scale) * float(keep.double().norm())
    step = step * min(1.0, 0.1 / (size + 1e-6))
    # the factor's, the product's and the update's roundings, of values below 1
    assert ((before - tr.P.double() - step).abs() <= step.abs() * 2.0 ** -22 + 2.0 ** -23).all()
    assert torch.equal(g, keep)


def test_without_a_limit_gradients_are_applied_as_they_are():
    tr = MlpTrainer(SPEC, synthetic_mnist(64, seed=1), batch=16, lr=0.5, seed=3)
    g = torch.randn(tr.P.numel(), generator=torch.Generator().manual_seed(2))
    want = tr.P - 0.5 * 0.25 * g
    tr.apply_gradients(g, 0.25)
    assert torch.allclose(tr.P, want, rtol=0, atol=2.0 ** -22)


@pytest.mark.gpu
@pytest.mark.parametrize("clip,graph_steps,said", [(0.5, 4, True), (0.5, 0, False), (0.0, 4, False)])
def test_a_clipped_engine_says_that_it_replays_no_graph(clip, graph_steps, said, caplog):
    with caplog.at_level("WARNING", logger="hipdsml.trainer"):
        tr = MlpTrainer(SPEC, synthetic_mnist(64, seed=1), batch=16, lr=0.5, seed=3, clip_norm=clip,
                        graph_steps=graph_steps, ctx=_ctx("cuda"))
    assert tr._graphs_on() is (graph_steps > 0 and not clip and not tr.persistent)
    assert any("graph_steps" in r.getMessage() for r in caplog.records) is said
