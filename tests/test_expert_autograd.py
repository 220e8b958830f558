"""The expert operators and clipping are explicit calls that autograd does not
record.  A tensor that requires a gradient would lose it without a word, so such
a call is refused wherever gradients are recorded, on the host as on the GPU."""
import pytest
import torch

from hipdsml.ops import experts as X
from hipdsml.ops import functional as F

BF = torch.bfloat16

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def _operands(dev):
    g = torch.Generator().manual_seed(7)
    rand = lambda *s, dt=BF: torch.randn(*s, generator=g).to(dt).to(dev)
    logits = rand(4, 3, dt=torch.float32)
    return dict(logits=logits, route=X.route_topk(logits, 2), x=rand(4, 8), w=rand(3, 6, 8),
                b=rand(3, 6, dt=torch.float32), dz=rand(8, 6), mask=rand(8, 8), dout=rand(4, 6),
                dg=rand(4, 2, dt=torch.float32), grads=[rand(5, dt=torch.float32), rand(7, dt=torch.float32)])


def _grad(t):
    return t.detach().clone().requires_grad_()


# name: the call with one operand that requires a gradient
CALLS = {
    "route logits": lambda o, q: X.route_topk(q(o["logits"]), 2),
    "route_backward dgates": lambda o, q: X.route_topk_backward(q(o["dg"]), o["logits"], o["route"]),
    "route_backward logits": lambda o, q: X.route_topk_backward(o["dg"], q(o["logits"]), o["route"], "all"),
    "route_backward gates": lambda o, q: X.route_topk_backward(
        o["dg"], o["logits"], o["route"]._replace(gates=q(o["route"].gates))),
    "linear x": lambda o, q: X.grouped_linear(q(o["x"]), o["w"], o["route"].offsets, rows=o["route"].rows),
    "linear w": lambda o, q: X.grouped_linear(o["x"], q(o["w"]), o["route"].offsets, rows=o["route"].rows),
    "linear bias": lambda o, q: X.grouped_linear(o["x"], o["w"], o["route"].offsets, q(o["b"]), rows=o["route"].rows),
    "linear out": lambda o, q: X.grouped_linear(o["x"], o["w"], o["route"].offsets, rows=o["route"].rows, out=q(o["dz"])),
    "dgrad dz": lambda o, q: X.grouped_dgrad(q(o["dz"]), o["w"], o["route"].offsets),
    "dgrad w": lambda o, q: X.grouped_dgrad(o["dz"], q(o["w"]), o["route"].offsets),
    "dgrad mask": lambda o, q: X.grouped_dgrad(o["dz"], o["w"], o["route"].offsets, mask=q(o["mask"])),
    "wgrad dz": lambda o, q: X.grouped_wgrad(q(o["dz"]), o["x"], o["route"].offsets, o["route"].rows),
    "wgrad x": lambda o, q: X.grouped_wgrad(o["dz"], q(o["x"]), o["route"].offsets, o["route"].rows),
    "wgrad dw": lambda o, q: X.grouped_wgrad(o["dz"], o["x"], o["route"].offsets, o["route"].rows,
                                             dw=q(o["w"].float())),
    "combine y": lambda o, q: X.expert_combine(q(o["dz"]), o["route"]),
    "combine gates": lambda o, q: X.expert_combine(o["dz"], o["route"]._replace(gates=q(o["route"].gates))),
    "combine_backward dout": lambda o, q: X.expert_combine_backward(q(o["dout"]), o["dz"], o["route"]),
    "combine_backward y": lambda o, q: X.expert_combine_backward(o["dout"], q(o["dz"]), o["route"]),
    "norm": lambda o, q: F.grad_norm([o["grads"][0], q(o["grads"][1])]),
    "clip a parameter": lambda o, q: F.clip_grad_norm_([o["grads"][0], q(o["grads"][1])], 0.5),
    "clip into a parameter": lambda o, q: F.clip_grad_norm_(o["grads"], 0.5, out=[q(g) for g in o["grads"]]),
}


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("call", sorted(CALLS))
def test_gradients_are_not_dropped_silently(call, dev):
    o = _operands(dev)
    with pytest.raises(RuntimeError, match="autograd does not record"):
        CALLS[call](o, _grad)


def _flat(r):
    return [r] if isinstance(r, torch.Tensor) else [t for t in r if t is not None]


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("call", sorted(CALLS))
def test_parameters_are_taken_without_recording(call, dev):
    """Under no_grad a parameter is an operand like any other."""
    want = _flat(CALLS[call](_operands(dev), lambda t: t.clone()))
    with torch.no_grad():
        got = _flat(CALLS[call](_operands(dev), _grad))
    assert len(got) == len(want)
    for a, b in zip(got, want):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dev", DEVICES)
def test_unweighted_combine_reads_no_gates(dev):
    o = _operands(dev)
    r = o["route"]._replace(gates=_grad(o["route"].gates))
    assert torch.equal(X.expert_combine(o["dz"], r, weighted=False), X.expert_combine(o["dz"], o["route"], weighted=False))


def test_native_entry_points_refuse_before_any_launch():
    from hipdsml.ops.native import load_native

    C = load_native()
    if C is None:
        pytest.skip("extension not built")
    o = _operands("cpu")
    r = o["route"]
    for fn in (lambda: C.route_topk(_grad(o["logits"]), 2),
               lambda: C.route_topk_backward(_grad(o["dg"]), o["logits"], r.gates, r.experts),
               lambda: C.grouped_linear(o["x"], _grad(o["w"]), r.offsets, rows=r.rows),
               lambda: C.grouped_dgrad(_grad(o["dz"]), o["w"], r.offsets),
               lambda: C.grouped_wgrad(o["dz"], _grad(o["x"]), r.offsets, r.rows),
               lambda: C.expert_combine(_grad(o["dz"]), r.slots, r.gates),
               lambda: C.expert_combine_backward(o["dout"], o["dz"], r.slots, _grad(r.gates), r.offsets),
               lambda: C.grad_norm([o["grads"][0], _grad(o["grads"][1])]),
               lambda: C.grad_norm(o["grads"], True, 1.0, 1e-6, [_grad(g) for g in o["grads"]])):
        with pytest.raises(RuntimeError, match="autograd does not record"):
            fn()
        with torch.no_grad(), pytest.raises(RuntimeError, match="GPU"):  # only the device is wrong
            fn()
