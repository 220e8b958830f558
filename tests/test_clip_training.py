"""Gradient clipping in the training engines (clip_norm): the averaged gradient's
global norm is limited before the update, on one replica and on several."""
import math
import os
import tempfile

import pytest
import torch
from spawn_util import spawn_group

from hipdsml.data.mnist import synthetic_mnist
from hipdsml.engine.trainer import MlpTrainer
from hipdsml.models.mlp import MlpLayout, MlpSpec, grads_ref, init_params
from hipdsml.parallel.dist import DistContext
from hipdsml.utils.config import TrainConfig, parse

SPEC = MlpSpec((784, 32, 16, 10))


def _reference(P, lay, shards, batch, steps, lr, clip, momentum=0.0):
    """fp64 SGD on the mean gradient with its norm clipped; also the norms seen."""
    P = P.double()
    V = torch.zeros_like(P)
    norms = []
    for s in range(steps):
        g = sum(grads_ref(lay, P, sh.X[s * batch:(s + 1) * batch].double(), sh.y[s * batch:(s + 1) * batch])[0]
                for sh in shards).double() / len(shards)
        n = float(g.norm())
        norms.append(n)
        g = g * min(1.0, clip / (n + 1e-6))
        V = momentum * V + g
        P = P - lr * V
    return P, norms


@pytest.mark.parametrize("momentum", [0.0, 0.9])
@pytest.mark.parametrize("clip", [0.05, 100.0])
def test_cpu_trainer_clips(clip, momentum):
    ds = synthetic_mnist(16 * 5, seed=4)
    tr = MlpTrainer(SPEC, ds, batch=16, lr=0.05, seed=3, momentum=momentum, clip_norm=clip)
    lay = MlpLayout(SPEC, 16, 5)
    want, norms = _reference(init_params(lay, 3), lay, [ds], 16, 5, 0.05, clip, momentum)
    assert min(norms) > 0.05 and max(norms) < 100.0  # one limit clips every step, the other none
    tr.train_steps(5)
    # fp32 steps of sums over at most 784 terms against fp64 ones
    assert (tr.P.double() - want).abs().max() < 1e-5


def _worker(rank, world, port, outdir):
    os.environ.update(RANK=str(rank), WORLD_SIZE=str(world), LOCAL_RANK=str(rank),
                      MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
    ctx = DistContext.from_env(device="cpu")
    ds = synthetic_mnist(16 * 4, seed=100 + rank)
    tr = MlpTrainer(SPEC, ds, batch=16, lr=0.05, ctx=ctx, seed=3, clip_norm=0.05)
    tr.train_steps(4)
    torch.save({"P": tr.P}, os.path.join(outdir, f"r{rank}.pt"))
    ctx.destroy()


def test_replicas_clip_the_mean_gradient():
    with tempfile.TemporaryDirectory() as d:
        spawn_group(_worker, 2, lambda port: (2, port, d))
        outs = [torch.load(os.path.join(d, f"r{r}.pt"), weights_only=True)["P"] for r in range(2)]
    assert torch.equal(outs[0], outs[1])
    lay = MlpLayout(SPEC, 16, 4)
    want, _ = _reference(init_params(lay, 3), lay, [synthetic_mnist(16 * 4, seed=100 + r) for r in range(2)], 16, 4,
                         0.05, 0.05)
    assert (outs[0].double() - want).abs().max() < 1e-5


def test_configuration_and_refusals():
    assert TrainConfig().clip_norm == 0.0
    assert parse(TrainConfig, ["--clip-norm", "0.5"]).clip_norm == 0.5
    ds = synthetic_mnist(64, seed=1)
    for bad in (-1.0, math.nan):
        with pytest.raises(ValueError, match="negative"):
            MlpTrainer(SPEC, ds, batch=16, clip_norm=bad)
    with pytest.raises(ValueError, match="inside the exchange"):
        MlpTrainer(SPEC, ds, batch=16, sync="pkx", clip_norm=1.0)


def test_fit_clips_on_the_cpu():
    from hipdsml.engine.fit import run

    r = run(TrainConfig(model="784-32-10", samples=64, steps=1, lr=1.0, device="cpu", clip_norm=0.01, eval=False),
            out=lambda *_: None)
    assert r["steps"] == 1


@pytest.mark.gpu
@pytest.mark.parametrize("momentum", [0.0, 0.9])
@pytest.mark.parametrize("graph_steps", [0, 4])
def test_gpu_trainer_clips_like_the_cpu(graph_steps, momentum):
    dev = DistContext(device=torch.device("cuda", 0))
    spec = MlpSpec((784, 128, 64, 10))
    ds = synthetic_mnist(64 * 4, seed=4)
    a = MlpTrainer(spec, ds, batch=64, lr=0.05, seed=3, momentum=momentum, clip_norm=0.05)
    b = MlpTrainer(spec, ds, batch=64, lr=0.05, seed=3, momentum=momentum, clip_norm=0.05, ctx=dev,
                   graph_steps=graph_steps)
    assert not b.persistent
    a.train_steps(9)
    b.train_steps(4)
    b.train_steps(5)
    b.synchronize()
    assert (a.P - b.P.cpu()).abs().max() < 2e-5


@pytest.mark.gpu
@pytest.mark.parametrize("graph", [False, True])
def test_gpu_wide_engine_clips(graph):
    """A limit no gradient reaches: the steps of the plain engine (its gradient
    written out, not fused) to a rounding; one that every gradient passes: the
    parameters move by lr times the limit."""
    from hipdsml.engine.wide import WideMlpTrainer

    spec, ds = MlpSpec((784, 512, 512, 10)), synthetic_mnist(64 * 4, seed=5)

    def run(clip, steps, lr=0.05):
        tr = WideMlpTrainer(spec, ds, batch=64, lr=lr, seed=2, clip_norm=clip, graph=graph)
        before = tr.P.double().clone()
        tr.train_steps(steps)
        tr.synchronize()
        return before, tr.P.double()

    _, plain = run(0.0, 4)
    _, loose = run(1e6, 4)
    # one step of the same gradient from each engine form differs by fp32 sums; later
    # steps by what those tip in bf16 activations (half a step, 2^-8, of lr g)
    assert (plain - loose).abs().max() < 4 * 0.05 * 2.0 ** -8 * 8
    for clip in (0.01, 0.5):
        before, after = run(clip, 1, lr=0.5)
        moved = float((after - before).norm())
        # the masters hold fp32: each moved weight is off by half a step of a value below 1
        off = math.sqrt(after.numel()) * 2.0 ** -24
        assert abs(moved - 0.5 * clip) <= 0.5 * clip * 1e-4 + off


@pytest.mark.gpu
def test_gpu_wide_refusals():
    from hipdsml.engine.wide import WideMlpTrainer

    spec, ds = MlpSpec((784, 512, 512, 10)), synthetic_mnist(64, seed=5)
    with pytest.raises(ValueError, match="negative"):
        WideMlpTrainer(spec, ds, clip_norm=-1.0)
    with pytest.raises(ValueError, match="no gradient to clip"):
        WideMlpTrainer(spec, ds, sync="xact", clip_norm=1.0)
