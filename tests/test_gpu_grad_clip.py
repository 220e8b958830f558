"""Global gradient norm and clipping on the GPU against 64-bit sums."""
import math

import pytest
import torch
from expert_util import close, half_step

from hipdsml.ops import functional as F

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda", 0)


def _grads(sizes, dt, seed=0, scale=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return [(torch.randn(n, generator=g, device=DEV) * scale).to(dt) for n in sizes]


def _norm(grads):
    return math.sqrt(math.fsum(float(t.double().square().sum()) for t in grads))


# one element, none, piece and vector tails, more tensors than one launch holds, many pieces
SIZES = [[1], [0, 3], [5, 1, 7], [784 * 128, 128, 128 * 64, 64, 640, 10], [16384, 16385, 16383, 32768, 4],
         [i % 37 for i in range(300)], [3_000_001, 17, 20_000_000]]


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("sizes", SIZES, ids=[f"{len(s)}x{sum(s)}" for s in SIZES])
def test_norm_and_clip(sizes, dt):
    grads = _grads(sizes, dt, scale=0.5)
    want = _norm(grads)
    # fp64 sums (n terms at 2^-53 are below the last bit), one fp32 rounding
    assert abs(float(F.grad_norm(grads)) - want) <= want * 2.0 ** -23
    keep = [t.clone() for t in grads]
    for factor in (0.3, 2.0):
        m = want * factor
        out = [torch.full_like(t, 3.0) for t in grads]
        n = F.clip_grad_norm_(grads, m, out=out)
        assert abs(float(n) - want) <= want * 2.0 ** -23
        assert all(torch.equal(a, b) for a, b in zip(grads, keep))
        c = min(1.0, m / (want + 1e-6))
        for o, t in zip(out, keep):
            ref = t.double() * c
            tiny = 0.0 if dt != torch.float16 else 2.0 ** -25
            # the factor's and the product's rounding, and the type's
            close(o, ref, ref.abs() * (2.0 ** -22 + (half_step(dt) if dt != torch.float32 else 0.0)) + tiny)
        mine = [t.clone() for t in grads]
        F.clip_grad_norm_(mine, m)
        assert all(torch.equal(a, o) for a, o in zip(mine, out))


def test_unaligned_views_and_neighbours_untouched():
    buf = torch.randn(100_000, device=DEV)
    want = buf.clone()
    views = [buf[1:50_002], buf[50_003:50_006], buf[60_001:99_999]]
    n = _norm(views)
    F.clip_grad_norm_(views, n / 2)
    c = (n / 2) / (n + 1e-6)
    for a, b in ((1, 50_002), (50_003, 50_006), (60_001, 99_999)):
        close(buf[a:b], want[a:b].double() * c, want[a:b].double().abs() * 2.0 ** -22)
        want[a:b] = buf[a:b]
    assert torch.equal(buf, want)


def test_values_a_float32_square_cannot_hold():
    g = torch.full((1000,), 1e30, device=DEV)
    assert abs(float(F.grad_norm([g])) / (1e30 * math.sqrt(1000)) - 1) < 2.0 ** -22
    g = torch.full((1000,), 1e-30, device=DEV)
    assert abs(float(F.grad_norm([g])) / (1e-30 * math.sqrt(1000)) - 1) < 2.0 ** -22
    F.clip_grad_norm_([g], 1.0)
    assert (g == torch.full_like(g, 1e-30)).all()


def test_broken_gradients_show():
    a, b = torch.ones(10, device=DEV), torch.ones(10, device=DEV)
    b[3] = torch.nan
    assert math.isnan(float(F.clip_grad_norm_([a, b], 1.0))) and a.isnan().all() and b.isnan().all()
    a, b = torch.ones(10, device=DEV), torch.ones(10, device=DEV)
    b[3] = torch.inf
    assert math.isinf(float(F.clip_grad_norm_([a, b], 1.0)))
    assert (a == 0).all() and b[3].isnan() and (b[:3] == 0).all()


def test_zero_gradients_and_zero_limit():
    z = [torch.zeros(5, device=DEV), torch.zeros(0, device=DEV)]
    assert float(F.clip_grad_norm_(z, 1.0)) == 0.0 and (z[0] == 0).all()
    g = [torch.ones(4, device=DEV)]
    assert float(F.clip_grad_norm_(g, 0.0)) == 2.0 and (g[0] == 0).all()


def test_in_a_graph_and_on_another_stream():
    grads = _grads([5000, 300_000, 17], torch.float32, seed=1)
    static = [t.clone() for t in grads]
    gr = torch.cuda.CUDAGraph()
    F.clip_grad_norm_([t.clone() for t in static], 1.0)
    with torch.cuda.graph(gr):
        n = F.clip_grad_norm_(static, 1.0)
    for seed in (2, 3, 4):
        new = _grads([5000, 300_000, 17], torch.float32, seed=seed)
        for s, v in zip(static, new):
            s.copy_(v)
        gr.replay()
        m = F.clip_grad_norm_(new, 1.0)
        torch.cuda.synchronize(DEV)
        assert torch.equal(n, m) and all(torch.equal(a, b) for a, b in zip(static, new))
    want = _grads([5000, 300_000, 17], torch.float32, seed=5)
    side = torch.cuda.Stream(DEV)
    other = [t.clone() for t in want]
    F.clip_grad_norm_(want, 1.0)
    torch.cuda.synchronize(DEV)
    with torch.cuda.stream(side):
        F.clip_grad_norm_(other, 1.0)
    torch.cuda.synchronize(DEV)
    assert all(torch.equal(a, b) for a, b in zip(want, other))
