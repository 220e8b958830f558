"""Expert-layer operators on host tensors: the refusals of the native entry
points (their checks come before any launch), the host math against its 64-bit
form, and a layer's gradients against differences."""
import math

import pytest
import torch
from expert_util import (close, dgrad64, half_step, linear64, offsets_of, rounded_tol, route64, route_bwd64,
                         wgrad64)

from hipdsml.ops import experts as X
from hipdsml.ops import functional as F
from hipdsml.ops.native import load_native

BF = torch.bfloat16
I32 = torch.int32


def _native():
    C = load_native()
    if C is None:
        pytest.skip("extension not built")
    return C


def _w(E=2, N=4, K=8, dt=BF):
    return torch.ones(E, N, K, dtype=dt)


def _off(*v):
    return torch.tensor(v, dtype=I32)


LINEAR_BAD = {
    "type": (lambda: dict(x=torch.ones(3, 8), w=_w(dt=torch.float32), offsets=_off(0, 1, 3)), "bfloat16 or float16"),
    "mixed": (lambda: dict(x=torch.ones(3, 8, dtype=torch.float16), w=_w(), offsets=_off(0, 1, 3)), "w must have x's type"),
    "columns": (lambda: dict(x=torch.ones(3, 7, dtype=BF), w=_w(), offsets=_off(0, 1, 3)), "columns"),
    "offsets": (lambda: dict(x=torch.ones(3, 8, dtype=BF), w=_w(), offsets=_off(0, 3)), "offsets must hold 3"),
    "offsets64": (lambda: dict(x=torch.ones(3, 8, dtype=BF), w=_w(), offsets=torch.tensor([0, 1, 3])), "int32"),
    "bias": (lambda: dict(x=torch.ones(3, 8, dtype=BF), w=_w(), offsets=_off(0, 1, 3), bias=torch.ones(2, 3)), "bias must be"),
    "biastype": (lambda: dict(x=torch.ones(3, 8, dtype=BF), w=_w(), offsets=_off(0, 1, 3),
                              bias=torch.ones(2, 4, dtype=BF)), "float32"),
    "rows": (lambda: dict(x=torch.ones(3, 8, dtype=BF), w=_w(), offsets=_off(0, 1, 3), rows=torch.zeros(3)), "int32"),
    "strided": (lambda: dict(x=torch.ones(8, 3, dtype=BF).t(), w=_w(), offsets=_off(0, 1, 3)), "contiguous"),
    "axes": (lambda: dict(x=torch.ones(8, dtype=BF), w=_w(), offsets=_off(0, 1, 3)), "axes"),
    "out": (lambda: dict(x=torch.ones(3, 8, dtype=BF), w=_w(), offsets=_off(0, 1, 3), out=torch.ones(3, 5, dtype=BF)),
            "out must be"),
    "outtype": (lambda: dict(x=torch.ones(3, 8, dtype=BF), w=_w(), offsets=_off(0, 1, 3), out=torch.ones(3, 4)), "type"),
    "outrows": (lambda: dict(x=torch.ones(3, 8, dtype=BF), w=_w(), offsets=_off(0, 1, 3),
                             out=torch.ones(4, dtype=BF).expand(3, 4)), "overlap"),
    "noexperts": (lambda: dict(x=torch.ones(3, 8, dtype=BF), w=torch.ones(0, 4, 8, dtype=BF), offsets=_off(0)), "none of them 0"),
}


@pytest.mark.parametrize("side", ["host", "native"])
@pytest.mark.parametrize("case", sorted(LINEAR_BAD))
def test_linear_refusals(case, side):
    make, msg = LINEAR_BAD[case]
    fn = X.grouped_linear if side == "host" else _native().grouped_linear
    with pytest.raises(RuntimeError, match=msg):
        fn(**make())


def test_native_linear_refuses_overlap_and_host_tensors():
    C = _native()
    buf = torch.ones(64, dtype=BF)
    x = buf[:24].view(3, 8)
    with pytest.raises(RuntimeError, match="overlap an input"):
        C.grouped_linear(x, _w(), _off(0, 1, 3), out=buf[12:24].view(3, 4))
    with pytest.raises(RuntimeError, match="GPU tensors"):
        C.grouped_linear(x, _w(), _off(0, 1, 3))


GRAD_BAD = {
    "dgrad columns": ("grouped_dgrad", lambda: dict(dz=torch.ones(3, 5, dtype=BF), w=_w(), offsets=_off(0, 1, 3)), "columns"),
    "dgrad mask": ("grouped_dgrad", lambda: dict(dz=torch.ones(3, 4, dtype=BF), w=_w(), offsets=_off(0, 1, 3),
                                                 mask=torch.ones(3, 4, dtype=BF)), "mask must be"),
    "dgrad masktype": ("grouped_dgrad", lambda: dict(dz=torch.ones(3, 4, dtype=BF), w=_w(), offsets=_off(0, 1, 3),
                                                     mask=torch.ones(3, 8)), "mask must have"),
    "wgrad rows": ("grouped_wgrad", lambda: dict(dz=torch.ones(3, 4, dtype=BF), x=torch.ones(2, 8, dtype=BF),
                                                 offsets=_off(0, 1, 3)), "rows"),
    "wgrad gather": ("grouped_wgrad", lambda: dict(dz=torch.ones(3, 4, dtype=BF), x=torch.ones(2, 8, dtype=BF),
                                                   offsets=_off(0, 1, 3), rows=_off(0, 1)), "rows must hold 3"),
    "wgrad dw": ("grouped_wgrad", lambda: dict(dz=torch.ones(3, 4, dtype=BF), x=torch.ones(3, 8, dtype=BF),
                                               offsets=_off(0, 1, 3), dw=torch.ones(2, 8, 4)), "dw must be"),
    "wgrad dwtype": ("grouped_wgrad", lambda: dict(dz=torch.ones(3, 4, dtype=BF), x=torch.ones(3, 8, dtype=BF),
                                                   offsets=_off(0, 1, 3), dw=torch.ones(2, 4, 8, dtype=BF)), "float32"),
    "wgrad dwrows": ("grouped_wgrad", lambda: dict(dz=torch.ones(3, 4, dtype=BF), x=torch.ones(3, 8, dtype=BF),
                                                   offsets=_off(0, 1, 3), dw=torch.ones(4, 8).expand(2, 4, 8)), "overlap"),
    "wgrad db": ("grouped_wgrad", lambda: dict(dz=torch.ones(3, 4, dtype=BF), x=torch.ones(3, 8, dtype=BF),
                                               offsets=_off(0, 1, 3), bias=False, db=torch.ones(2, 4)), "bias=False"),
    "wgrad offsets": ("grouped_wgrad", lambda: dict(dz=torch.ones(3, 4, dtype=BF), x=torch.ones(3, 8, dtype=BF),
                                                    offsets=_off(0)), "experts \\+ 1"),
}


@pytest.mark.parametrize("side", ["host", "native"])
@pytest.mark.parametrize("case", sorted(GRAD_BAD))
def test_gradient_refusals(case, side):
    name, make, msg = GRAD_BAD[case]
    fn = getattr(X if side == "host" else _native(), name)
    with pytest.raises(RuntimeError, match=msg):
        fn(**make())


@pytest.mark.parametrize("side", ["host", "native"])
@pytest.mark.parametrize("shape,k,norm,dt,msg", [
    ((3, 513), 2, "topk", torch.float32, "1..512 experts"),
    ((3, 0), 1, "topk", torch.float32, "experts"),
    ((3, 8), 0, "topk", torch.float32, "k must be"),
    ((3, 8), 9, "topk", torch.float32, "k must be"),
    ((3, 32), 17, "topk", torch.float32, "k must be"),
    ((3, 8), 2, "rows", torch.float32, "normalize"),
    ((3, 8), 2, "topk", torch.int32, "float32, bfloat16"),
])
def test_route_refusals(shape, k, norm, dt, msg, side):
    fn = X.route_topk if side == "host" else _native().route_topk
    with pytest.raises(RuntimeError, match=msg):
        fn(torch.zeros(shape, dtype=dt), k, norm)


def test_route_backward_and_combine_refusals():
    C = _native()
    logits = torch.randn(5, 8)
    r = X.route_topk(logits, 2)
    with pytest.raises(RuntimeError, match="dgates must be float32"):
        C.route_topk_backward(torch.zeros(5, 2, dtype=BF), logits, r.gates, r.experts)
    with pytest.raises(RuntimeError, match="gates must hold"):
        C.route_topk_backward(torch.zeros(5, 3), logits, r.gates, r.experts)
    y = torch.ones(10, 8, dtype=BF)
    with pytest.raises(RuntimeError, match="bfloat16 or float16"):
        C.expert_combine(y.float(), r.slots, r.gates)
    with pytest.raises(RuntimeError, match="gates must hold"):
        C.expert_combine(y, r.slots, r.gates[:4])
    with pytest.raises(RuntimeError, match="overlap an input"):
        C.expert_combine(y, r.slots, r.gates, out=y[:5])
    with pytest.raises(RuntimeError, match="one row a slot"):
        C.expert_combine_backward(torch.ones(5, 8, dtype=BF), y[:9], r.slots, r.gates, r.offsets)
    with pytest.raises(RuntimeError, match="dout must be"):
        C.expert_combine_backward(torch.ones(4, 8, dtype=BF), y, r.slots, r.gates, r.offsets)


@pytest.mark.parametrize("side", ["host", "native"])
def test_clip_refusals(side):
    if side == "host":
        def call(g, m=1.0, out=None, eps=None):
            return F.clip_grad_norm_(g, m, *([] if eps is None else [eps]), out=out)
    else:
        C = _native()

        def call(g, m=1.0, out=None, eps=None):
            return C.grad_norm(g, True, m, 1e-6 if eps is None else eps, out)
    for args, msg in [(([],), "no gradients"), (([torch.ones(2, dtype=torch.int32)],), "float32, bfloat16"),
                      (([torch.ones(2), torch.ones(2, dtype=BF)],), "one type"),
                      (([torch.ones(4, 4).t()[:2]],), "contiguous"), (([torch.ones(2)], -1.0), "negative"),
                      (([torch.ones(2)], math.nan), "negative"),
                      (([torch.ones(2)], 1.0, None, -1e-6), "eps must not"),
                      (([torch.ones(2)], 1.0, None, math.nan), "eps must not"),
                      (([torch.ones(2)], 1.0, []), "one tensor a gradient"),
                      (([torch.ones(2)], 1.0, [torch.ones(3)]), "shapes")]:
        with pytest.raises(RuntimeError, match=msg):
            call(*args)


def test_native_clip_refuses_gradients_that_overlap():
    C = _native()
    g = torch.ones(64)
    for grads, out in [([g, g], None), ([g[:40], g[32:]], None), ([g[:32]], [g[16:48]]),
                       ([g[:16], g[16:32]], [g[32:48], g[40:56]]), ([g[:16], g[16:32]], [g[16:32], g[32:48]])]:
        with pytest.raises(RuntimeError, match="overlap"):
            C.grad_norm(grads, True, 1.0, 1e-6, out)
    with pytest.raises(RuntimeError, match="one GPU"):  # disjoint: only the device is wrong
        C.grad_norm([g[:16], g[16:32]], True, 1.0, 1e-6, [g[:16], g[32:48]])


def test_host_clip_refuses_gradients_that_overlap():
    g = torch.ones(64)
    for grads in ([g, g], [g[:40], g[32:]]):
        with pytest.raises(RuntimeError, match="overlap"):
            F.clip_grad_norm_(grads, 1.0)
    assert F.clip_grad_norm_([g[:32], g[32:]], 4.0) == 8.0 and torch.all((g - 0.5).abs() < 1e-6)


def test_columns_of_one_buffer_are_apart():
    """Operand and result as column ranges of one buffer: refused only where they meet."""
    C = _native()
    buf, w, off = torch.ones(6, 48, dtype=BF), torch.ones(1, 16, 16, dtype=BF), torch.tensor([0, 6], dtype=torch.int32)
    for x, out in [((0, 16), (16, 32)), ((16, 32), (0, 16)), ((32, 48), (8, 24))]:
        with pytest.raises(RuntimeError, match="GPU tensors"):  # only the device is wrong
            C.grouped_linear(buf[:, slice(*x)], w, off, out=buf[:, slice(*out)])
    for x, out in [((0, 16), (8, 24)), ((16, 32), (1, 17)), ((32, 48), (32, 48))]:
        with pytest.raises(RuntimeError, match="overlap an input"):
            C.grouped_linear(buf[:, slice(*x)], w, off, out=buf[:, slice(*out)])
    with pytest.raises(RuntimeError, match="overlap an input"):  # a row further on
        C.grouped_linear(buf[:5, :16], w, off[:2], out=buf[1:, 8:24])


def test_choices_without_a_slot_count_nothing_whatever_their_gate():
    y = torch.ones(2, 8, dtype=BF)
    r = X.Route(torch.tensor([[0.5, math.nan]]), torch.tensor([[0, -1]], dtype=torch.int32),
                torch.tensor([0, 1], dtype=torch.int32), torch.tensor([0, -1], dtype=torch.int32),
                torch.tensor([[0, -1]], dtype=torch.int32))
    assert torch.equal(X.expert_combine(y, r), torch.full((1, 8), 0.5, dtype=BF))
    with pytest.raises(TypeError):
        X.route_topk(torch.zeros(2, 4), 1.5)


# ---- host math --------------------------------------------------------------------
@pytest.mark.parametrize("sizes", [[3, 0, 5], [0, 0], [1]])
@pytest.mark.parametrize("dt", [BF, torch.float16])
def test_host_products(sizes, dt):
    g = torch.Generator().manual_seed(1)
    S, E, N, K = sum(sizes), len(sizes), 6, 9
    x, w = torch.randn(S, K, generator=g).to(dt), torch.randn(E, N, K, generator=g).to(dt)
    dz, b = torch.randn(S, N, generator=g).to(dt), torch.randn(E, N, generator=g)
    off = offsets_of(sizes)
    ref, mag = linear64(x, w, sizes, b, True)
    close(X.grouped_linear(x, w, off, b, True), ref, rounded_tol(ref, mag, K, dt))
    m = torch.randn(S, K, generator=g).to(dt)
    ref, mag = dgrad64(dz, w, sizes, m)
    close(X.grouped_dgrad(dz, w, off, m), ref, rounded_tol(ref, mag, N, dt))
    dw, dwm, db, dbm = wgrad64(dz, x, sizes)
    gw, gb = X.grouped_wgrad(dz, x, off)
    close(gw, dw, rounded_tol(dw, dwm, S, torch.float32))
    close(gb, db, rounded_tol(db, dbm, S, torch.float32))


@pytest.mark.parametrize("normalize", ["topk", "all"])
@pytest.mark.parametrize("T,E,k", [(1, 1, 1), (7, 5, 2), (20, 12, 4)])
def test_host_route(T, E, k, normalize):
    g = torch.Generator().manual_seed(T)
    x = torch.randn(T, E, generator=g).mul(2).round()  # many ties
    if T > 3:
        x[1] = -torch.inf
        x[2, 1:] = -torch.inf
        x[3, 0] = torch.nan
    r = X.route_topk(x, k, normalize)
    gates, *ints = route64(x, k, normalize)
    for got, want in zip(r[1:], ints):
        assert torch.equal(got, want)
    # exp and its argument's rounding, a sum of E terms, a quotient
    close(r.gates, gates, gates * (E + 12) * U32_ + 1e-30)
    dg = torch.randn(T, k, generator=g)
    ref = route_bwd64(dg, x, r.experts, normalize)
    scale = (gates * dg.double().abs()).sum(1, keepdim=True) + dg.double().abs().amax(1, keepdim=True)
    close(X.route_topk_backward(dg, x, r, normalize), ref, scale * (E + 24) * U32_)


U32_ = 2.0 ** -23


def test_host_layer_gradients_against_differences():
    """The whole layer, forward and backward, on values that bf16 holds exactly
    enough: every gradient against central differences of a 64-bit forward."""
    g = torch.Generator().manual_seed(5)
    T, E, k, D, H = 6, 4, 2, 5, 7
    dt = torch.float16
    x = torch.randn(T, D, generator=g).to(dt)
    w1, w2 = (0.5 * torch.randn(E, H, D, generator=g)).to(dt), (0.5 * torch.randn(E, D, H, generator=g)).to(dt)
    b1, b2 = 0.1 * torch.randn(E, H, generator=g), 0.1 * torch.randn(E, D, generator=g)
    logits = torch.randn(T, E, generator=g)
    up = torch.randn(T, D, generator=g).to(dt)

    def forward64(x, w1, b1, w2, b2, logits, route):
        live = route.experts.long()
        p = torch.softmax(logits.gather(1, live), 1)
        out = torch.zeros(T, D, dtype=torch.float64)
        for j in range(k):
            for t in range(T):
                e = int(live[t, j])
                h = torch.relu(w1[e] @ x[t] + b1[e])
                out[t] += p[t, j] * (w2[e] @ h + b2[e])
        return (out * up.double()).sum()

    r = X.route_topk(logits, k)
    h = X.grouped_linear(x, w1, r.offsets, b1, True, r.rows)
    y = X.grouped_linear(h, w2, r.offsets, b2)
    dy, dg = X.expert_combine_backward(up, y, r)
    dw2, db2 = X.grouped_wgrad(dy, h, r.offsets)
    dh = X.grouped_dgrad(dy, w2, r.offsets, mask=h)
    dw1, db1 = X.grouped_wgrad(dh, x, r.offsets, rows=r.rows)
    dx = X.expert_combine(X.grouped_dgrad(dh, w1, r.offsets), r, weighted=False)
    dl = X.route_topk_backward(dg, logits, r)
    args = [t.double() for t in (x, w1, b1, w2, b2, logits)]
    eps = 1e-5
    for i, got in ((0, dx), (1, dw1), (2, db1), (3, dw2), (4, db2), (5, dl)):
        flat = args[i].reshape(-1)
        num = torch.zeros_like(flat)
        for q in range(flat.numel()):
            for sgn in (1, -1):
                a = list(args)
                v = flat.clone()
                v[q] += sgn * eps
                a[i] = v.view(args[i].shape)
                num[q] += sgn * forward64(*a, r) / (2 * eps)
        # fp16 activations in between: four roundings of half a step each on paths
        # whose magnitudes sum to at most a few times the largest gradient
        scale = float(num.abs().max()) + 1.0
        assert (got.double().reshape(-1) - num).abs().max() < 16 * 4 * half_step(dt) * scale, i


def test_host_clip():
    g = torch.Generator().manual_seed(3)
    grads = [torch.randn(n, generator=g) for n in (1, 7, 300)]
    want = math.sqrt(math.fsum(float(v) ** 2 for t in grads for v in t))
    assert abs(float(F.grad_norm(grads)) - want) <= want * 2.0 ** -24 * 2
    keep = [t.clone() for t in grads]
    out = [torch.empty_like(t) for t in grads]
    n = F.clip_grad_norm_(grads, 2.0, out=out)
    assert all(torch.equal(a, b) for a, b in zip(grads, keep))
    F.clip_grad_norm_(grads, 2.0)
    c = 2.0 / (want + 1e-6)
    for a, o, t in zip(grads, out, keep):
        assert torch.equal(a, o)
        close(a, t.double() * c, t.double().abs() * c * 2.0 ** -24 * 3)
    assert abs(float(n) - want) <= want * 2.0 ** -23
    small = [t.clone() for t in grads]
    F.clip_grad_norm_(small, 1e6)
    assert all(torch.equal(a, b) for a, b in zip(small, grads))
