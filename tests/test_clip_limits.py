"""Gradient clipping at its limits: calls that have no answer are refused on the
host as on the GPU, and results at the ends of the types' ranges are right."""
import pytest
import torch

from hipdsml.ops import functional as F

# (gradients, outputs) as ranges of one buffer of 64: each writes a range twice, or
# writes over a gradient that is read as another one
OVERLAPS = {
    "twice": ([(0, 32), (0, 32)], None),
    "partly": ([(0, 40), (32, 64)], None),
    "out over its own, moved": ([(0, 32)], [(16, 48)]),
    "outs": ([(0, 16), (16, 32)], [(32, 48), (40, 56)]),
    "out over the next": ([(0, 16), (16, 32)], [(16, 32), (32, 48)]),
    "out over the one before": ([(0, 16), (16, 32)], [(32, 48), (0, 16)]),
    "out over two": ([(0, 16), (16, 32), (32, 48)], [(48, 64), (8, 24), (32, 48)]),
}
APART = {
    "in place": ([(0, 32), (32, 64)], None),
    "one in place, one not": ([(0, 16), (16, 32)], [(0, 16), (32, 48)]),
    "all moved": ([(0, 16), (16, 32)], [(48, 64), (32, 48)]),
    "none in it": ([(0, 16), (8, 8), (16, 32)], [(0, 16), (4, 4), (16, 32)]),
}


def _views(buf, spans):
    return None if spans is None else [buf[a:b] for a, b in spans]


@pytest.mark.parametrize("case", sorted(OVERLAPS))
def test_host_refuses_outputs_over_gradients(case):
    grads, out = OVERLAPS[case]
    buf = torch.arange(64, dtype=torch.float32)
    with pytest.raises(RuntimeError, match="must not overlap"):
        F.clip_grad_norm_(_views(buf, grads), 1.0, out=_views(buf, out))
    assert torch.equal(buf, torch.arange(64, dtype=torch.float32))


@pytest.mark.parametrize("case", sorted(APART))
def test_host_takes_ranges_that_lie_apart(case):
    grads, out = APART[case]
    buf = torch.arange(64, dtype=torch.float32)
    want = [buf[a:b].double() for a, b in grads]
    n = float(F.clip_grad_norm_(_views(buf, grads), 1.0, out=_views(buf, out)))
    for (a, b), g in zip(grads if out is None else out, want):
        # the roundings of the norm, the factor and the product
        assert ((buf[a:b] - g / (n + 1e-6)).abs() <= g / n * 2.0 ** -22).all()


DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16, torch.float16])
def test_zero_gradients_stay_zero_whatever_the_limit(dt, dev):
    for max_norm, eps in ((0.0, 0.0), (0.0, 1e-6), (1.0, 0.0), (float("inf"), 0.0)):
        grads = [torch.zeros(n, dtype=dt, device=dev) for n in (3, 0, 4097)]
        out = [torch.full_like(g, 7.0) for g in grads]
        assert float(F.clip_grad_norm_(grads, max_norm, eps, out=out)) == 0.0
        assert float(F.clip_grad_norm_(grads, max_norm, eps)) == 0.0
        assert all((t == 0).all() for t in grads + out)
    broken = [torch.zeros(5, dtype=dt, device=dev), torch.full((2,), float("nan"), dtype=dt, device=dev)]
    assert F.clip_grad_norm_(broken, 0.0, 0.0).isnan() and all(g.isnan().all() for g in broken)


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("max_norm", [3.0, 1e-3, 1e-30])
def test_a_factor_below_float32s_normal_range_keeps_its_bits(max_norm, dt, dev):
    """Gradients near the type's largest value: the factor is below 2^-126, the clipped
    values are not."""
    g = torch.linspace(0.5, 1.0, 4099, dtype=torch.float64)
    grads = [(s * g * 3e38).to(dt).to(dev) for s in (1.0, -0.5)]
    out = [torch.empty_like(t) for t in grads]
    n = sum(t.double().square().sum() for t in grads).sqrt()
    want = [t.double() * (max_norm / n) for t in grads]
    assert max_norm / float(n) < 2.0 ** -126
    F.clip_grad_norm_(grads, max_norm, 0.0, out=out)
    F.clip_grad_norm_(grads, max_norm, 0.0)
    for a, o, w in zip(grads, out, want):
        assert torch.equal(a, o)
        # the product's rounding and the type's
        assert ((a.double() - w).abs() <= w.abs() * (2.0 ** -23 + torch.finfo(dt).eps / 2)).all()
