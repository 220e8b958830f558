"""Every way a training engine updates its parameters obeys clip_norm."""
import math

import pytest
import torch

from hipdsml.data.mnist import synthetic_mnist
from hipdsml.engine.trainer import MlpTrainer
from hipdsml.models.mlp import MlpLayout, MlpSpec, init_params
from hipdsml.parallel.dist import DistContext
from hipdsml.utils.checkpoint import latest_checkpoint, load_state
from hipdsml.utils.config import TrainConfig

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


@pytest.mark.parametrize("engine,model,init,dev", [
    ("fused", "784-32-10", "reference", "cpu"),
    pytest.param("fused", "784-32-10", "reference", "cuda", marks=pytest.mark.gpu),
    pytest.param("wide", "784-512-512-10", "kaiming", "cuda", marks=pytest.mark.gpu),
])
def test_a_fit_job_moves_by_lr_times_the_limit(engine, model, init, dev, tmp_path):
    from hipdsml.engine.fit import run

    P0 = init_params(MlpLayout(MlpSpec.parse(model), 64, 1), 0, init).double()
    moved = {}
    for clip in (0.01, 0.0):
        at = str(tmp_path / f"c{clip}")
        run(TrainConfig(model=model, engine=engine, samples=64, steps=1, lr=1.0, device=dev, clip_norm=clip, eval=False,
                        checkpoint=at), out=lambda *_: None)
        moved[clip] = float((load_state(latest_checkpoint(at))["params"].double() - P0).norm())
    # fp32 parameters below 1: half a step of each; the factor's and the product's roundings,
    # and eps next to the norm (1e-6 of a norm above 0.1)
    assert moved[0.0] > 0.1
    assert abs(moved[0.01] - 0.01) <= 0.01 * (1e-5 + 2.0 ** -22) + math.sqrt(P0.numel()) * 2.0 ** -25


@pytest.mark.gpu
@pytest.mark.parametrize("graph", [False, True])
def test_a_limit_that_no_gradient_reaches_moves_every_layer_as_without_one(graph):
    """Four steps of the wide engine with its gradients written out, against its fused
    form: every W and b moves, and ends where the fused form leaves it.  The two differ
    by fp32 sums in another order, which tip bf16 copies of W, H and dZ by a step at
    most: 2^-8 each of a step, on no more than four factors of it."""
    from hipdsml.engine.wide import WideMlpTrainer

    spec, ds = MlpSpec((784, 512, 512, 10)), synthetic_mnist(64 * 4, seed=5)

    def layers(tr):
        tr.synchronize()
        return [t.double().clone() for W, b in tr.layout.views(tr.P) for t in (W, b)]

    plain = WideMlpTrainer(spec, ds, batch=64, lr=0.05, seed=2, graph=False)
    at, path = layers(plain), None
    start = at
    for _ in range(4):
        plain.train_steps(1)
        now = layers(plain)
        steps = [float((a - b).norm()) for a, b in zip(now, at)]
        path = steps if path is None else [p + s for p, s in zip(path, steps)]
        at = now
    loose = WideMlpTrainer(spec, ds, batch=64, lr=0.05, seed=2, clip_norm=1e6, graph=graph)
    loose.train_steps(4)
    for i, (a, b, s, p) in enumerate(zip(at, layers(loose), start, path)):
        assert float((b - s).norm()) > 0.1 * p > 0.0, i
        assert float((a - b).norm()) <= 4 * 2.0 ** -8 * p, i


class _Alone(DistContext):
    """One replica that takes a data-parallel job's way: its collectives run, over one rank."""

    @property
    def is_distributed(self):
        return True


def _comm():
    from hipdsml.ops.native import require_native

    C = require_native()
    return C.RcclComm(C.rccl_unique_id(), 0, 1, 0, True)


@pytest.mark.gpu
@pytest.mark.parametrize("sync", ["rccl", "ring"])
@pytest.mark.parametrize("own_stream", [False, True])
def test_collectives_come_before_the_clip(sync, own_stream):
    """The RCCL and ring branches of the clipped step, over one rank: the lone replica's
    parameters, bit for bit."""
    dev = torch.device("cuda", 0)
    kw = dict(batch=16, lr=0.5, seed=3, clip_norm=0.05)
    ds = synthetic_mnist(64, seed=1)
    lone = MlpTrainer(SPEC, ds, ctx=DistContext(device=dev), **kw)
    comm = _comm()
    tr = MlpTrainer(SPEC, ds, ctx=_Alone(device=dev), sync=sync, external_comm=comm, ring_chunk_bytes=1 << 14,
                    stream=torch.cuda.Stream(dev) if own_stream else None, **kw)
    assert tr.sync_active == sync
    for t in (lone, tr):
        before = t.P.clone()
        t.train_steps(5)
        t.synchronize()
        assert not torch.equal(before, t.P)
    assert torch.equal(lone.P, tr.P)
    torch.cuda.synchronize(dev)
    comm.abort()


@pytest.mark.gpu
@pytest.mark.parametrize("sync", ["rccl", "ring"])
@pytest.mark.parametrize("graph", [False, True])
def test_the_wide_engines_buckets_are_all_reduced_before_the_clip(graph, sync, monkeypatch):
    from hipdsml.engine import wide

    dev = torch.device("cuda", 0)
    spec, ds = MlpSpec((784, 512, 512, 10)), synthetic_mnist(64 * 4, seed=5)
    kw = dict(batch=64, lr=0.5, seed=2, clip_norm=0.05, graph=graph)
    lone = wide.WideMlpTrainer(spec, ds, ctx=DistContext(device=dev), **kw)
    comm = _comm()
    monkeypatch.setattr(wide, "make_native_comm", lambda ctx: comm)
    tr = wide.WideMlpTrainer(spec, ds, ctx=_Alone(device=dev), sync=sync, **kw)
    for t in (lone, tr):
        before = t.P.clone()
        t.train_steps(8)
        t.synchronize()
        assert not torch.equal(before, t.P)
    assert torch.equal(lone.P, tr.P)
    torch.cuda.synchronize(dev)
    comm.abort()
