"""Expert-layer calls that have no right answer are refused on the host as on the
GPU (the native checks come before any launch, so host tensors reach them)."""
import pytest
import torch

from hipdsml.ops import experts as X
from hipdsml.ops.native import load_native

BF = torch.bfloat16
OFF = torch.tensor([0, 2, 4], dtype=torch.int32)


def _native():
    C = load_native()
    if C is None:
        pytest.skip("extension not built")
    return C


def _call(side, name, **kw):
    """The public call, or the native one with the same arguments."""
    if side == "host":
        return getattr(X, name)(**kw)
    if name == "expert_combine":
        r, weighted = kw.pop("route"), kw.pop("weighted", True)
        kw.update(slots=r.slots, gates=r.gates if weighted else None)
    if name == "expert_combine_backward":
        r = kw.pop("route")
        kw.update(slots=r.slots, gates=r.gates, offsets=r.offsets)
    return getattr(_native(), name)(**kw)


# 4 slots, 2 experts [4 out, 8 in], as pieces of one buffer `b` of 256 elements
def _x(b):
    return b[:32].view(4, 8)


def _dz(b):
    return b[:16].view(4, 4)


def _w(b):
    return b[64:128].view(2, 4, 8)


def _f32(b, lo, *shape):
    return b.view(torch.float32)[lo:].as_strided(shape, torch.empty(shape).stride())


OVER = {
    "linear out, x": ("grouped_linear", lambda b: dict(x=_x(b), w=_w(b), offsets=OFF, out=b[16:32].view(4, 4))),
    "linear out, weights": ("grouped_linear", lambda b: dict(x=_x(b), w=_w(b), offsets=OFF, out=b[100:116].view(4, 4))),
    "linear out, bias": ("grouped_linear", lambda b: dict(x=_x(b), w=_w(b), offsets=OFF, bias=_f32(b, 64, 2, 4),
                                                          out=b[140:156].view(4, 4))),
    "linear out, offsets": ("grouped_linear", lambda b: dict(x=_x(b), w=_w(b), offsets=b.view(torch.int32)[64:67],
                                                             out=b[128:144].view(4, 4))),
    "linear out, rows": ("grouped_linear", lambda b: dict(x=_x(b), w=_w(b), offsets=OFF, rows=b.view(torch.int32)[64:68],
                                                          out=b[134:150].view(4, 4))),
    "linear columns": ("grouped_linear", lambda b: dict(x=b[128:192].view(4, 16)[:, :8], w=_w(b), offsets=OFF,
                                                        out=b[128:192].view(4, 16)[:, 7:11])),
    "dgrad out, dz": ("grouped_dgrad", lambda b: dict(dz=_dz(b), w=_w(b), offsets=OFF, out=b[12:44].view(4, 8))),
    "dgrad out, weights": ("grouped_dgrad", lambda b: dict(dz=_dz(b), w=_w(b), offsets=OFF, out=b[96:128].view(4, 8))),
    "dgrad out, mask": ("grouped_dgrad", lambda b: dict(dz=_dz(b), w=_w(b), offsets=OFF, mask=b[128:160].view(4, 8),
                                                        out=b[128:160].view(4, 8))),
    "wgrad dw, dz": ("grouped_wgrad", lambda b: dict(dz=_dz(b), x=_w(b)[0], offsets=OFF, dw=_f32(b, 7, 2, 4, 8))),
    "wgrad dw, x": ("grouped_wgrad", lambda b: dict(dz=_dz(b), x=b[150:182].view(4, 8), offsets=OFF,
                                                    dw=_f32(b, 16, 2, 4, 8))),
    "wgrad db, dz": ("grouped_wgrad", lambda b: dict(dz=_dz(b), x=_w(b)[0], offsets=OFF, db=_f32(b, 4, 2, 4))),
    "wgrad dw, db": ("grouped_wgrad", lambda b: dict(dz=_dz(b), x=b[16:48].view(4, 8), offsets=OFF,
                                                     dw=_f32(b, 64, 2, 4, 8), db=_f32(b, 120, 2, 4))),
    "combine out, y": ("expert_combine", lambda b: dict(y=_x(b), route=_route(), out=b[8:24].view(2, 8))),
    "combine out, gates": ("expert_combine", lambda b: dict(y=_x(b), route=_route(gates=_f32(b, 64, 2, 2)),
                                                            out=b[130:146].view(2, 8))),
}


def _route(**kw):
    r = X.Route(torch.full((2, 2), 0.5), torch.tensor([[0, 1], [0, 1]], dtype=torch.int32), OFF,
                torch.tensor([0, 1, 0, 1], dtype=torch.int32), torch.tensor([[0, 2], [1, 3]], dtype=torch.int32))
    return r._replace(**kw)


@pytest.mark.parametrize("side", ["host", "native"])
@pytest.mark.parametrize("case", sorted(OVER))
def test_results_over_operands_are_refused(case, side):
    name, make = OVER[case]
    buf = torch.zeros(256, dtype=BF)
    with pytest.raises(RuntimeError, match="must not overlap an input"):
        _call(side, name, **make(buf))
    assert (buf == 0).all()


def test_results_beside_operands_are_taken():
    """Columns of one buffer, and pieces that touch: the same results as apart."""
    g = torch.Generator().manual_seed(3)
    buf = torch.randn(4, 24, generator=g).to(BF)
    w = torch.randn(2, 8, 16, generator=g).to(BF)
    want = X.grouped_linear(buf[:, :16].clone(), w, OFF)
    X.grouped_linear(buf[:, :16], w, OFF, out=buf[:, 16:])
    assert torch.equal(buf[:, 16:], want)
    flat = torch.zeros(4 * 8 + 4 * 16, dtype=BF)
    dz, out = flat[:32].view(4, 8), flat[32:].view(4, 16)
    dz.copy_(want)
    X.grouped_dgrad(dz, w, OFF, out=out)
    assert torch.equal(out, X.grouped_dgrad(want, w, OFF)) and torch.equal(dz, want)
    f = torch.zeros(2 * 8 * 16 + 2 * 8)
    dw, db = f[:256].view(2, 8, 16), f[256:].view(2, 8)
    X.grouped_wgrad(dz, out, OFF, dw=dw, db=db)
    for a, b in zip((dw, db), X.grouped_wgrad(dz, out, OFF)):
        assert torch.equal(a, b)


BAD_ARGUMENTS = {
    "combine gates type": ("expert_combine", lambda: dict(y=torch.ones(4, 8, dtype=BF), route=_route(
        gates=torch.ones(2, 2, dtype=torch.float64))), "gates must be float32"),
    "combine gates size": ("expert_combine", lambda: dict(y=torch.ones(4, 8, dtype=BF), route=_route(
        gates=torch.ones(3, 2))), "gates must hold 4"),
    "combine gates strided": ("expert_combine", lambda: dict(y=torch.ones(4, 8, dtype=BF), route=_route(
        gates=torch.ones(2, 2).t())), "gates must be contiguous"),
    "combine slots axes": ("expert_combine", lambda: dict(y=torch.ones(4, 8, dtype=BF), weighted=False, route=_route(
        slots=torch.zeros(4, dtype=torch.int32))), "slots must have 2 axes"),
    "combine choices": ("expert_combine", lambda: dict(y=torch.ones(4, 8, dtype=BF), weighted=False, route=_route(
        slots=torch.zeros(2, 17, dtype=torch.int32))), "k must be 1..16"),
    "combine no choices": ("expert_combine", lambda: dict(y=torch.ones(4, 8, dtype=BF), weighted=False, route=_route(
        slots=torch.zeros(2, 0, dtype=torch.int32))), "k must be 1..16"),
    "combine columns": ("expert_combine", lambda: dict(y=torch.ones(4, 0, dtype=BF), route=_route()), "columns"),
    "backward choices": ("expert_combine_backward", lambda: dict(
        dout=torch.ones(2, 8, dtype=BF), y=torch.ones(34, 8, dtype=BF),
        route=_route(slots=torch.zeros(2, 17, dtype=torch.int32), gates=torch.ones(2, 17))), "k must be 1..16"),
    "backward columns": ("expert_combine_backward", lambda: dict(
        dout=torch.ones(2, 0, dtype=BF), y=torch.ones(4, 0, dtype=BF), route=_route()), "columns"),
    "backward offsets": ("expert_combine_backward", lambda: dict(
        dout=torch.ones(2, 8, dtype=BF), y=torch.ones(4, 8, dtype=BF), route=_route(offsets=OFF[:1])), "experts \\+ 1"),
    "backward offsets type": ("expert_combine_backward", lambda: dict(
        dout=torch.ones(2, 8, dtype=BF), y=torch.ones(4, 8, dtype=BF), route=_route(offsets=OFF.long())), "int32"),
    "wgrad columns": ("grouped_wgrad", lambda: dict(dz=torch.ones(4, 0, dtype=BF), x=torch.ones(4, 8, dtype=BF),
                                                    offsets=OFF), "bad sizes"),
    "wgrad width": ("grouped_wgrad", lambda: dict(dz=torch.ones(4, 4, dtype=BF), x=torch.ones(4, 0, dtype=BF),
                                                  offsets=OFF), "bad sizes"),
    "linear size": ("grouped_linear", lambda: dict(
        x=torch.ones(1, 1, dtype=BF), w=torch.ones(1, 1, 1, dtype=BF).expand(1, 1 << 24, 1), offsets=OFF[:2]), "too large"),
    "linear rows": ("grouped_linear", lambda: dict(
        x=torch.ones(1, 8, dtype=BF).expand(1 << 31, 8), w=torch.ones(2, 4, 8, dtype=BF), offsets=OFF), "more than 2\\^31"),
    "dgrad rows": ("grouped_dgrad", lambda: dict(
        dz=torch.ones(1, 4, dtype=BF).expand(1 << 31, 4), w=torch.ones(2, 4, 8, dtype=BF), offsets=OFF), "more than 2\\^31"),
}


@pytest.mark.parametrize("side", ["host", "native"])
@pytest.mark.parametrize("case", sorted(BAD_ARGUMENTS))
def test_arguments_are_refused_alike(case, side):
    name, make, msg = BAD_ARGUMENTS[case]
    with pytest.raises(RuntimeError, match=msg):
        _call(side, name, **make())


@pytest.mark.parametrize("side", ["host", "native"])
def test_route_backward_takes_the_routers_types(side):
    logits = torch.randn(3, 8)
    r = X.route_topk(logits, 2)
    with pytest.raises(RuntimeError, match="float32, bfloat16 or float16"):
        if side == "host":
            X.route_topk_backward(torch.zeros(3, 2), logits.double(), r)
        else:
            _native().route_topk_backward(torch.zeros(3, 2), logits.double(), r.gates, r.experts)


@pytest.mark.parametrize("S,gathered,whole", [((1 << 29) - 1, True, True), (1 << 29, True, False),
                                              ((1 << 31) - 256, True, False), (1 << 29, False, True),
                                              ((1 << 31) - 256, False, True)])
def test_ids_of_a_weight_gradient_stay_within_32_bits(S, gathered, whole):
    """The kernel for whole 16-B words streams a group's 4-B ids behind 32-bit offsets, so
    2^29 of them or more go to the kernel for any width, which indexes in 64."""
    C = _native()
    assert C.grouped_whole_words("wgrad", S, 1 << 20, 300, 8, 8, gathered) is whole
    for op in ("linear", "dgrad"):  # they read an id a lane, in 64 bits
        assert C.grouped_whole_words(op, S, 1 << 20, 300, 8, 8, op == "linear" and gathered)
    assert not C.grouped_whole_words("wgrad", 64, 1 << 20, 2, 8, 12, gathered)
    # a gathered operand is read behind 32-bit offsets too
    for op in ("linear", "wgrad"):
        assert C.grouped_whole_words(op, 64, (1 << 28) - 32, 2, 8, 8, True)
        assert not C.grouped_whole_words(op, 64, 1 << 28, 2, 8, 8, True)


@pytest.mark.parametrize("side", ["host", "native"])
def test_weight_gradients_leave_room_for_a_step(side):
    """A group's rows are counted in steps of 64, two ahead, in 32-bit integers."""
    def call(S):
        dz, x = torch.zeros(1, 4, dtype=BF).expand(S, 4), torch.zeros(1, 8, dtype=BF).expand(S, 8)
        return _call(side, "grouped_wgrad", dz=dz, x=x, offsets=OFF)

    with pytest.raises(RuntimeError, match="more than 2\\^31 - 256 rows"):
        call((1 << 31) - 255)
    if side == "native":
        with pytest.raises(RuntimeError, match="GPU tensors"):  # only the device is wrong
            call((1 << 31) - 256)
