"""Expert-layer kernels against their 64-bit forms: group sizes with empty,
one-row and uneven groups, odd widths, strides, gathered rows, both types."""
import pytest
import torch
from expert_util import (close, dgrad64, half_step, linear64, offsets_of, rounded_tol, route64, route_bwd64,
                         wgrad64)

from hipdsml.ops import experts as X
from hipdsml.ops.native import require_native

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda", 0)
BF, FP = torch.bfloat16, torch.float16
U32 = 2.0 ** -23

# (group sizes, K, N): one row, empty groups, tiles that end inside, odd widths,
# widths of whole 16-B rows, groups longer than every tile
SHAPES = [
    ([1], 8, 8),
    ([0, 1, 0], 16, 24),
    ([0, 0], 64, 64),
    ([3, 0, 5, 1], 7, 13),
    ([65, 1, 130], 33, 70),
    ([64, 128, 0, 64], 64, 128),
    ([200, 17, 300], 784, 128),
    ([5, 4, 3, 2, 1, 0, 9, 8], 128, 10),
    ([257, 511, 1, 255], 264, 520),
    ([300, 700], 1000, 264),
    ([16] * 70, 72, 40),
    ([2, 1, 1, 3], 4096, 256),
    ([1, 0, 2], 200, 4096),
    ([1030, 520], 512, 768),
]

# enough tiles for every kernel: whole rounds of large tiles, their last round
# and the rows behind them in small ones, more than 64 groups, odd widths
LARGE = [
    ([3000, 500, 0, 2600], 1032, 1544),
    ([97] * 66 + [2500, 0, 1300], 520, 2312),
    ([1] * 40 + [20000], 264, 520),
    ([700, 0, 900, 333], 2056, 2056),
    ([1500, 999], 1037, 1031),
]


def _rand(g, *shape, dt=torch.float32, scale=1.0):
    return (torch.randn(*shape, generator=g, device=DEV) * scale).to(dt)


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _rows(g, S, T):
    return torch.randint(0, T, (S,), generator=g, device=DEV, dtype=torch.int32)


@pytest.mark.parametrize("dt", [BF, FP])
@pytest.mark.parametrize("sizes,K,N", SHAPES + LARGE)
@pytest.mark.parametrize("form", ["plain", "bias_relu", "gather"])
def test_linear(sizes, K, N, dt, form):
    g = _gen(len(sizes) * 1000 + K + N)
    S, E = sum(sizes), len(sizes)
    T = S if form != "gather" else max(1, S // 2)
    x, w = _rand(g, T, K, dt=dt), _rand(g, E, N, K, dt=dt, scale=K ** -0.5)
    bias = _rand(g, E, N) if form != "plain" else None
    rows = _rows(g, S, T) if form == "gather" else None
    relu = form == "bias_relu"
    got = X.grouped_linear(x, w, offsets_of(sizes).to(DEV), bias, relu, rows)
    ref, mag = linear64(x, w, sizes, bias, relu, rows)
    assert got.shape == (S, N) and got.dtype == dt
    close(got, ref, rounded_tol(ref, mag, K, dt), (sizes, K, N))


@pytest.mark.parametrize("dt", [BF, FP])
@pytest.mark.parametrize("sizes,K,N", SHAPES + LARGE)
@pytest.mark.parametrize("masked", [False, True])
def test_dgrad(sizes, K, N, dt, masked):
    g = _gen(len(sizes) * 1000 + K + N)
    S, E = sum(sizes), len(sizes)
    dz, w = _rand(g, S, N, dt=dt), _rand(g, E, N, K, dt=dt, scale=N ** -0.5)
    mask = torch.relu(_rand(g, S, K, dt=dt)) if masked else None
    got = X.grouped_dgrad(dz, w, offsets_of(sizes).to(DEV), mask)
    ref, mag = dgrad64(dz, w, sizes, mask)
    close(got, ref, rounded_tol(ref, mag, N, dt), (sizes, K, N))


@pytest.mark.parametrize("dt", [BF, FP])
@pytest.mark.parametrize("sizes,K,N", SHAPES + LARGE)
@pytest.mark.parametrize("gather", [False, True])
def test_wgrad(sizes, K, N, dt, gather):
    g = _gen(len(sizes) * 1000 + K + N)
    S = sum(sizes)
    T = max(1, S // 2) if gather else S
    dz, x = _rand(g, S, N, dt=dt), _rand(g, T, K, dt=dt)
    rows = _rows(g, S, T) if gather else None
    dw, db = X.grouped_wgrad(dz, x, offsets_of(sizes).to(DEV), rows)
    ref, mag, rb, mb = wgrad64(dz, x, sizes, rows)
    n = max(sizes)
    close(dw, ref, rounded_tol(ref, mag, n, torch.float32), (sizes, K, N))
    close(db, rb, rounded_tol(rb, mb, n, torch.float32), (sizes, K, N))
    only, none = X.grouped_wgrad(dz, x, offsets_of(sizes).to(DEV), rows, bias=False)
    assert none is None and torch.equal(only, dw)


@pytest.mark.parametrize("sizes,K,N", [([3, 0, 5, 1], 7, 13), ([40, 300, 17], 264, 136), ([1, 2], 512, 256)])
@pytest.mark.parametrize("dt", [BF, FP])
def test_strided_operands_and_slots_outside_every_group(sizes, K, N, dt):
    """Wider rows than needed, an expert axis with a gap, groups that start late
    and end early: given outputs keep their other rows, fresh ones are zero."""
    g = _gen(7)
    lead, tail, E = 3, 70, len(sizes)
    S = lead + sum(sizes) + tail
    off = offsets_of(sizes, lead).to(DEV)
    x = _rand(g, S, K + 5, dt=dt)[:, 2:2 + K]
    w = _rand(g, E, N + 1, K + 3, dt=dt, scale=K ** -0.5)[:, :N, 1:1 + K]
    dz = _rand(g, S, N + 9, dt=dt)[:, 1:1 + N]
    bias = _rand(g, E, N + 2)[:, :N]
    mask = _rand(g, S, K + 1, dt=dt)[:, :K]
    used = slice(lead, S - tail)
    ref, mag = linear64(x, w, sizes, bias, True, lead=lead)
    fresh = X.grouped_linear(x, w, off, bias, True)
    close(fresh, ref, rounded_tol(ref, mag, K, dt))
    assert (fresh[:lead] == 0).all() and (fresh[S - tail:] == 0).all()
    buf = torch.full((S, N + 4), 7.0, dtype=dt, device=DEV)
    out = buf[:, 1:1 + N]
    assert X.grouped_linear(x, w, off, bias, True, out=out).data_ptr() == out.data_ptr()
    assert torch.equal(out[used], fresh[used])
    assert (out[:lead] == 7).all() and (out[S - tail:] == 7).all() and (buf[:, 0] == 7).all() and (buf[:, 1 + N:] == 7).all()
    ref, mag = dgrad64(dz, w, sizes, mask, lead=lead)
    fresh = X.grouped_dgrad(dz, w, off, mask)
    close(fresh, ref, rounded_tol(ref, mag, N, dt))
    buf = torch.full((S, K + 8), 7.0, dtype=dt, device=DEV)
    out = X.grouped_dgrad(dz, w, off, mask, out=buf[:, 8:])
    assert torch.equal(out[used], fresh[used])
    assert (out[:lead] == 7).all() and (out[S - tail:] == 7).all() and (buf[:, :8] == 7).all()
    dw, dwm, db, dbm = wgrad64(dz, x, sizes, lead=lead)
    got, gb = X.grouped_wgrad(dz, x, off)
    close(got, dw, rounded_tol(dw, dwm, max(sizes), torch.float32))
    close(gb, db, rounded_tol(db, dbm, max(sizes), torch.float32))
    buf = torch.full((E, N + 1, K + 4), 7.0, device=DEV)
    bb = torch.full((E, N), 7.0, device=DEV)
    X.grouped_wgrad(dz, x, off, dw=buf[:, :N, 2:2 + K], db=bb)
    assert torch.equal(buf[:, :N, 2:2 + K], got) and torch.equal(bb, gb)
    assert (buf[:, N] == 7).all() and (buf[:, :, :2] == 7).all() and (buf[:, :, 2 + K:] == 7).all()


@pytest.mark.parametrize("K,N", [(24, 40), (264, 520), (25, 39), (5, 130)])
def test_infinities_and_nan_stay_in_their_rows(K, N):
    """A bad row changes no other row, a bad padding column of a strided operand
    changes nothing, and ReLU keeps a NaN."""
    g = _gen(9)
    sizes, dt = [5, 300, 2], BF
    S, off = sum(sizes), offsets_of(sizes).to(DEV)
    full = _rand(g, S, K + 8, dt=dt)
    full[:, K:] = torch.nan
    x = full[:, :K]
    wf = _rand(g, 3, N, K + 8, dt=dt)
    wf[:, :, K:] = torch.inf
    w = wf[:, :, :K]
    clean = X.grouped_linear(x, w, off, relu=True)
    assert clean.isfinite().all()
    x[7] = torch.nan
    x[100, 3] = torch.inf
    got = X.grouped_linear(x, w, off, relu=True)
    keep = torch.ones(S, dtype=torch.bool, device=DEV)
    keep[[7, 100]] = False
    assert torch.equal(got[keep], clean[keep]) and got[7].isnan().all()
    dz = _rand(g, S, N, dt=dt)
    dw0, db0 = X.grouped_wgrad(dz, full[:, :K].nan_to_num(0, 0, 0), off)
    dw, db = X.grouped_wgrad(dz, x, off)
    assert torch.equal(dw[0], dw0[0]) and torch.equal(dw[2], dw0[2]) and torch.equal(db, db0)
    assert dw[1].isnan().any()
    m = torch.full((S, K), torch.nan, dtype=dt, device=DEV)
    assert (X.grouped_dgrad(dz, w, off, m) == 0).all()  # NaN > 0 does not hold


@pytest.mark.parametrize("K,N", [(264, 136), (263, 135), (7, 130), (130, 7)])
def test_plans_out_of_range_stay_in_the_buffers(K, N):
    """Rows outside x count as zero rows; offsets are clamped to the slots."""
    g = _gen(11)
    dt = BF
    x, w = _rand(g, 50, K, dt=dt), _rand(g, 2, N, K, dt=dt)
    rows = torch.arange(100, device=DEV, dtype=torch.int32) % 50
    rows[3], rows[60], rows[99] = -1, 50, 2 ** 31 - 1
    off = torch.tensor([0, 40, 100], dtype=torch.int32, device=DEV)
    safe = rows.clone()
    bad = torch.tensor([3, 60, 99], device=DEV)
    safe[bad] = 0
    want = X.grouped_linear(x, w, off, rows=safe)
    want[bad] = 0
    assert torch.equal(X.grouped_linear(x, w, off, rows=rows), want)
    dz = _rand(g, 100, N, dt=dt)
    dz0 = dz.clone()
    dz0[bad] = 0
    assert torch.equal(X.grouped_wgrad(dz, x, off, rows)[0], X.grouped_wgrad(dz0, x, off, safe)[0])
    wide = torch.tensor([-5, 40, 10 ** 6], dtype=torch.int32, device=DEV)
    assert torch.equal(X.grouped_linear(x, w, wide, rows=safe), X.grouped_linear(x, w, off, rows=safe))
    assert X.grouped_linear(x[:0], w, off, rows=rows).abs().max() == 0
    dw, db = X.grouped_wgrad(dz, x[:0], off, rows)
    assert dw.abs().max() == 0 and torch.equal(db, X.grouped_wgrad(dz, x, off, safe)[1])


@pytest.mark.parametrize("sizes,lead,tail", [([2, 0, 3], 5, 30), ([40, 1], 9, 8), ([300, 40], 3, 9000), ([700, 2500], 300, 0),
                                             ([0, 0], 0, 700), ([0, 513], 2000, 1)])
@pytest.mark.parametrize("K,N", [(264, 520), (2056, 256)])
def test_rows_of_no_group_in_whole_words(sizes, lead, tail, K, N):
    """Aligned operands (padded row strides): the large-tile and single-token
    kernels zero the rows of no group in a fresh result and leave a given one's."""
    g, dt = _gen(13), BF
    S, off = lead + sum(sizes) + tail, offsets_of(sizes, lead).to(DEV)
    x, dz = _rand(g, S, K + 8, dt=dt)[:, 8:], _rand(g, S, N + 16, dt=dt)[:, :N]
    x[:lead], dz[:lead] = torch.nan, torch.nan
    x[S - tail:], dz[S - tail:] = torch.nan, torch.nan
    w = _rand(g, len(sizes), N, K, dt=dt, scale=K ** -0.5)
    used = slice(lead, S - tail)
    for name, call, ref, mag, red, cols in (
            ("linear", lambda out=None: X.grouped_linear(x, w, off, out=out), *linear64(x, w, sizes, None, False, lead=lead), K, N),
            ("dgrad", lambda out=None: X.grouped_dgrad(dz, w, off, out=out), *dgrad64(dz, w, sizes, None, lead=lead), N, K)):
        torch.full((S, cols), 7.0, dtype=dt, device=DEV)  # what a fresh result may find in its memory
        fresh = call()
        close(fresh[used], ref[used], rounded_tol(ref, mag, red, dt)[used])
        assert (fresh[:lead] == 0).all() and (fresh[S - tail:] == 0).all(), name
        buf = torch.full((S, cols + 8), 7.0, dtype=dt, device=DEV)
        call(buf[:, 8:])
        assert torch.equal(buf[used, 8:], fresh[used]), name
        assert (buf[:lead] == 7).all() and (buf[S - tail:] == 7).all() and (buf[:, :8] == 7).all(), name


def test_columns_of_one_buffer_as_operand_and_result():
    g, dt = _gen(14), BF
    sizes = [200, 77]
    off, w = offsets_of(sizes).to(DEV), _rand(g, 2, 128, 64, dt=dt)
    buf = _rand(g, 277, 256, dt=dt)
    want = X.grouped_linear(buf[:, 64:128].clone(), w, off)
    before = buf.clone()
    X.grouped_linear(buf[:, 64:128], w, off, out=buf[:, 128:])
    assert torch.equal(buf[:, 128:], want) and torch.equal(buf[:, :128], before[:, :128])


def test_all_tokens_to_one_of_many_experts():
    """A mean of few rows an expert, all of them in one."""
    g, dt = _gen(15), BF
    sizes = [0] * 90 + [700] + [0] * 9
    off, x, w = offsets_of(sizes).to(DEV), _rand(g, 700, 136, dt=dt), _rand(g, 100, 72, 136, dt=dt, scale=0.1)
    ref, mag = linear64(x, w, sizes, None, False)
    close(X.grouped_linear(x, w, off), ref, rounded_tol(ref, mag, 136, dt))
    dz = _rand(g, 700, 72, dt=dt)
    ref, mag = dgrad64(dz, w, sizes, None)
    close(X.grouped_dgrad(dz, w, off), ref, rounded_tol(ref, mag, 72, dt))


@pytest.mark.parametrize("sizes,K,N", [([6000], 304, 200), ([3000, 0, 2501], 264, 136), ([5001], 33, 70), ([20000], 8, 8),
                                       ([4000, 1, 130], 512, 384), ([9000, 64], 5, 3)])
@pytest.mark.parametrize("dt", [BF, FP])
@pytest.mark.parametrize("gather", [False, True])
def test_wgrad_of_few_tiles_and_many_rows(sizes, K, N, dt, gather):
    """Groups whose rows are summed in parts: the same bound, the same bits every
    time, given buffers written in place and nothing around them."""
    g = _gen(sum(sizes) + K)
    lead, tail, E = 7, 33, len(sizes)
    S = lead + sum(sizes) + tail
    off = offsets_of(sizes, lead).to(DEV)
    T = 500 if gather else S
    x, dz = _rand(g, T, K, dt=dt), _rand(g, S, N, dt=dt, scale=0.1)
    dz[:lead], dz[S - tail:] = torch.nan, torch.nan
    rows = _rows(g, S, T) if gather else None
    dw, dwm, db, dbm = wgrad64(dz, x, sizes, rows, lead=lead)
    got, gb = X.grouped_wgrad(dz, x, off, rows)
    close(got, dw, rounded_tol(dw, dwm, max(sizes), torch.float32))
    close(gb, db, rounded_tol(db, dbm, max(sizes), torch.float32))
    buf, bb = torch.full((E, N + 1, K + 4), 7.0, device=DEV), torch.full((E, N), 7.0, device=DEV)
    X.grouped_wgrad(dz, x, off, rows, dw=buf[:, :N, 4:], db=bb)
    close(buf[:, :N, 4:], dw, rounded_tol(dw, dwm, max(sizes), torch.float32))
    assert (buf[:, N] == 7).all() and (buf[:, :, :4] == 7).all() and torch.equal(bb, gb)
    again, none = X.grouped_wgrad(dz, x, off, rows, bias=False)
    assert none is None and torch.equal(again, got)


@pytest.mark.parametrize("sizes,K,N", [([5, 0, 90], 1789, 159), ([1, 3], 3001, 33), ([17] * 70, 1025, 7), ([300, 41], 643, 1001),
                                       ([0, 0], 999, 5)])
@pytest.mark.parametrize("dt", [BF, FP])
def test_odd_products_of_few_tiles_and_long_reductions(sizes, K, N, dt):
    """Reductions in parts: bias, ReLU and mask applied once to their sum, rows of no
    group cleared in a fresh result and left in a given one, the same bits every time."""
    g = _gen(K + N)
    lead, tail, E = 3, 21, len(sizes)
    S = lead + sum(sizes) + tail
    off, used = offsets_of(sizes, lead).to(DEV), slice(lead, S - tail)
    rows = _rows(g, S, 50)
    for red, cols, backward in ((K, N, False), (N, K, False), (K, N, True)):
        x = _rand(g, S if backward else 50, red, dt=dt)
        w = _rand(g, E, red, cols, dt=dt, scale=red ** -0.5) if backward else _rand(g, E, cols, red, dt=dt, scale=red ** -0.5)
        bias, mask = _rand(g, E, cols), _rand(g, S, cols, dt=dt)
        if backward:
            x[:lead], x[S - tail:] = torch.nan, torch.nan
            call = lambda out=None: X.grouped_dgrad(x, w, off, mask, out=out)
            ref, mag = dgrad64(x, w, sizes, mask, lead=lead)
        else:
            call = lambda out=None: X.grouped_linear(x, w, off, bias, True, rows, out=out)
            ref, mag = linear64(x, w, sizes, bias, True, rows, lead=lead)
        fresh = call()
        close(fresh[used], ref[used], rounded_tol(ref, mag, red, dt)[used])
        assert (fresh[:lead] == 0).all() and (fresh[S - tail:] == 0).all()
        buf = torch.full((S, cols + 3), 7.0, dtype=dt, device=DEV)
        call(buf[:, 1:1 + cols])
        assert torch.equal(buf[used, 1:1 + cols], fresh[used])
        assert (buf[:lead] == 7).all() and (buf[S - tail:] == 7).all() and (buf[:, 0] == 7).all() and (buf[:, 1 + cols:] == 7).all()


def test_wgrad_in_parts_in_two_graphs():
    """Each captured call has a workspace of its own; replayed on new values between eager calls."""
    g = _gen(21)
    off = offsets_of([3000, 2000]).to(DEV)
    dz, x = _rand(g, 5000, 72, dt=BF), _rand(g, 5000, 40, dt=BF)
    X.grouped_wgrad(dz, x, off)
    graphs, outs = [], []
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(X.grouped_wgrad(dz, x, off))
        graphs.append(gr)
    for seed in (1, 2, 3):
        dz.copy_(_rand(_gen(seed), 5000, 72, dt=BF))
        want = X.grouped_wgrad(dz, x, off)
        for gr in graphs:
            gr.replay()
        torch.cuda.synchronize(DEV)
        for o in outs:
            assert torch.equal(o[0], want[0]) and torch.equal(o[1], want[1])


def test_offsets_past_32_bits():
    """More than 2^31 output elements, and rows of x past 2^32 bytes."""
    S, K, N = 560_000, 4096, 3900
    x = torch.zeros(S, K, dtype=BF, device=DEV)
    w = torch.zeros(2, N, K, dtype=BF, device=DEV)
    w[0, :, 0], w[1, :, 0] = 1, 2
    x[:, 0] = (torch.arange(S, device=DEV) % 251).to(BF)
    off = torch.tensor([0, 100, S], dtype=torch.int32, device=DEV)
    y = X.grouped_linear(x, w, off)
    for s in (0, 99, 100, 262_143, 262_145, 550_699, S - 1):
        assert (y[s] == (s % 251) * (1 if s < 100 else 2)).all(), s
    rows = torch.arange(S - 1, -1, -1, device=DEV, dtype=torch.int32)[:1000].contiguous()
    y2 = X.grouped_linear(x, w, torch.tensor([0, 0, 1000], dtype=torch.int32, device=DEV), rows=rows)
    want = ((S - 1 - torch.arange(1000, device=DEV)) % 251).to(BF) * 2
    assert torch.equal(y2[:, 0], want) and torch.equal(y2[:, N - 1], want)


# ---- router -------------------------------------------------------------------------
ROUTES = [(1, 1, 1), (4, 8, 2), (1, 13, 3), (64, 16, 16), (255, 30, 5), (256, 64, 4), (257, 64, 4), (1000, 100, 8),
          (600, 256, 8), (300, 512, 16), (3000, 7, 2), (40, 200, 3), (70, 133, 6), (33, 301, 4), (20, 512, 2)]


def _logits(T, E, dt, seed):
    x = torch.randn(T, E, generator=_gen(seed), device=DEV).mul(3).round().div(2)  # ties
    if T > 3:
        x[1] = -torch.inf
        x[2, 1:] = -torch.inf
        x[T - 1, 0] = torch.nan
        x[T // 2] = torch.finfo(dt).min
    return x.to(dt)


@pytest.mark.parametrize("normalize", ["topk", "all"])
@pytest.mark.parametrize("dt", [torch.float32, BF, FP])
@pytest.mark.parametrize("T,E,k", ROUTES)
def test_route(T, E, k, dt, normalize):
    x = _logits(T, E, dt, T + E)
    r = X.route_topk(x, k, normalize)
    gates, *ints = route64(x, k, normalize)
    for name, got, want in zip(("experts", "offsets", "rows", "slots"), r[1:], ints):
        assert torch.equal(got.cpu(), want), name
    # exp to a step or two and its argument's rounding (< 2^4 halves a step of
    # up to 2^4), a sum of E terms, a quotient
    close(r.gates.cpu(), gates, gates * (E + 24) * U32 + 1e-37)
    dg = torch.randn(T, k, generator=_gen(T), device=DEV)
    ref = route_bwd64(dg.cpu(), x, r.experts.cpu(), normalize)
    got = X.route_topk_backward(dg, x, r, normalize)
    assert got.dtype == dt
    scale = dg.cpu().double().abs().amax(1, keepdim=True).expand(T, E)
    tiny = 0.0 if dt == torch.float32 else torch.finfo(dt).smallest_normal * torch.finfo(dt).eps
    rnd = 0.0 if dt == torch.float32 else half_step(dt)
    acc = 2 * scale * (E + 48) * U32
    close(got.cpu(), ref, rnd * (ref.abs() + acc) + acc + tiny)


def test_route_strided_logits_and_large_plan():
    g = _gen(2)
    x = torch.randn(70_000, 40, generator=g, device=DEV)[:, 3:27]
    r = X.route_topk(x, 3)
    c = X.route_topk(x.contiguous(), 3)
    assert all(torch.equal(a, b) for a, b in zip(r, c))
    ref = X.route_topk(x.cpu(), 3)
    for got, want in zip(r[1:], ref[1:]):
        assert torch.equal(got.cpu(), want)


def test_route_without_tokens():
    r = X.route_topk(torch.empty(0, 12, device=DEV), 2)
    assert (r.offsets == 0).all() and r.offsets.numel() == 13 and r.rows.numel() == 0
    assert X.route_topk_backward(torch.empty(0, 2, device=DEV), torch.empty(0, 12, device=DEV), r).shape == (0, 12)


# ---- combine --------------------------------------------------------------------------
@pytest.mark.parametrize("dt", [BF, FP])
@pytest.mark.parametrize("T,k,N", [(1, 1, 1), (3, 2, 8), (5, 4, 13), (130, 3, 70), (33, 6, 128), (64, 16, 256),
                                   (257, 2, 784), (20, 5, 4096), (9, 2, 4100),
                                   (1100, 2, 784), (1030, 5, 1001), (2000, 3, 7), (1025, 1, 519)])
def test_combine(T, k, N, dt):
    g = _gen(T + N)
    logits = torch.randn(T, max(k, 20), generator=g, device=DEV)
    if T > 2:
        logits[1] = -torch.inf  # a token without any slot
        logits[2, 1:] = -torch.inf
    r = X.route_topk(logits, k)
    y = _rand(g, T * k, N, dt=dt)
    dout = _rand(g, T, N, dt=dt)
    yd, gd = y.double(), r.gates.double()
    live = (r.slots >= 0)
    picked = torch.where(live[:, :, None], yd[r.slots.long().clamp(min=0)], torch.zeros((), device=DEV, dtype=torch.float64))
    for weighted in (True, False):
        wt = gd if weighted else live.double()
        ref = (picked * wt[:, :, None]).sum(1)
        mag = (picked.abs() * wt[:, :, None]).sum(1)
        close(X.expert_combine(y, r, weighted=weighted), ref, rounded_tol(ref, mag, k, dt))
    buf = torch.full((T, N + 3), 7.0, dtype=dt, device=DEV)
    out = X.expert_combine(y, r, out=buf[:, 1:1 + N])
    assert torch.equal(out, X.expert_combine(y, r)) and (buf[:, 0] == 7).all() and (buf[:, 1 + N:] == 7).all()
    dy, dg = X.expert_combine_backward(dout, y, r)
    dd = dout.double()
    ref = (picked * dd[:, None, :]).sum(2)
    mag = (picked.abs() * dd[:, None, :].abs()).sum(2)
    close(dg, ref, rounded_tol(ref, mag, N, torch.float32))
    want = torch.zeros(T * k, N, dtype=torch.float64, device=DEV)
    want[r.slots[live].long()] = (gd[:, :, None] * dd[:, None, :])[live]
    close(dy, want, rounded_tol(want, want.abs(), 1, dt))


# ---- together ---------------------------------------------------------------------------
def _layer(x, logits, w1, b1, w2, b2, k, up):
    r = X.route_topk(logits, k)
    h = X.grouped_linear(x, w1, r.offsets, b1, True, r.rows)
    y = X.grouped_linear(h, w2, r.offsets, b2)
    out = X.expert_combine(y, r)
    dy, dg = X.expert_combine_backward(up, y, r)
    dw2, db2 = X.grouped_wgrad(dy, h, r.offsets)
    dh = X.grouped_dgrad(dy, w2, r.offsets, mask=h)
    dw1, db1 = X.grouped_wgrad(dh, x, r.offsets, rows=r.rows)
    dx = X.expert_combine(X.grouped_dgrad(dh, w1, r.offsets), r, weighted=False)
    dl = X.route_topk_backward(dg, logits, r)
    return out, dx, dl, dw1, db1, dw2, db2


def _layer_args(T, E, D, H, seed, dt=BF):
    g = _gen(seed)
    logits = torch.randn(T, E, generator=g, device=DEV)
    if T > 8:
        logits[5] = -torch.inf
    return (_rand(g, T, D, dt=dt), logits, _rand(g, E, H, D, dt=dt, scale=D ** -0.5), _rand(g, E, H, scale=0.1),
            _rand(g, E, D, H, dt=dt, scale=H ** -0.5), _rand(g, E, D, scale=0.1), _rand(g, T, D, dt=dt))


@pytest.mark.parametrize("T,E,D,H,k", [(1, 8, 64, 128, 2), (70, 5, 33, 47, 3), (600, 8, 264, 512, 2)])
def test_layer_matches_host_math(T, E, D, H, k):
    """The chain of operators on the GPU and on the host: every step rounds to
    the same type at the same places, so they differ by fp32 sums and the
    roundings those tip over (a few half steps of the largest value)."""
    x, logits, w1, b1, w2, b2, up = _layer_args(T, E, D, H, T)
    got = _layer(x, logits, w1, b1, w2, b2, k, up)
    want = _layer(*(t.cpu() for t in (x, logits, w1, b1, w2, b2)), k, up.cpu())
    for name, a, b in zip(("out", "dx", "dlogits", "dw1", "db1", "dw2", "db2"), got, want):
        b = b.double()
        assert (a.cpu().double() - b).abs().max() <= 8 * half_step(BF) * (float(b.abs().max()) + 1e-30), name


def test_layer_in_a_graph_and_on_another_stream():
    """Captured once and replayed on new values (between eager calls), and two
    layers at once on two streams: bit for bit what the eager call gives."""
    args = _layer_args(300, 8, 264, 512, 1)
    k = 2
    static = [t.clone() for t in args]
    side = torch.cuda.Stream(DEV)
    side.wait_stream(torch.cuda.current_stream(DEV))
    with torch.cuda.stream(side):
        _layer(*static[:6], k, static[6])
    torch.cuda.current_stream(DEV).wait_stream(side)
    graphs, outs = [], []
    for _ in range(2):  # two graphs, each with its own workspaces
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(_layer(*static[:6], k, static[6]))
        graphs.append(gr)
    for seed in (2, 3, 4):
        new = _layer_args(300, 8, 264, 512, seed)
        want = _layer(*new[:6], k, new[6])
        for s, n in zip(static, new):
            s.copy_(n)
        for gr in graphs:
            gr.replay()
        torch.cuda.synchronize(DEV)
        for o in outs:
            for a, b in zip(o, want):
                assert torch.equal(a, b)
    a, b = _layer_args(300, 8, 264, 512, 5), _layer_args(300, 8, 264, 512, 6)
    want = [_layer(*t[:6], k, t[6]) for t in (a, b)]
    torch.cuda.synchronize(DEV)
    s1, s2 = torch.cuda.Stream(DEV), torch.cuda.Stream(DEV)
    with torch.cuda.stream(s1):
        r1 = _layer(*a[:6], k, a[6])
    with torch.cuda.stream(s2):
        r2 = _layer(*b[:6], k, b[6])
    torch.cuda.synchronize(DEV)
    for got, ref in ((r1, want[0]), (r2, want[1])):
        for p, q in zip(got, ref):
            assert torch.equal(p, q)


def test_the_same_call_twice_gives_the_same_bits():
    args = _layer_args(777, 8, 520, 264, 9)
    one, two = _layer(*args[:6], 4, args[6]), _layer(*args[:6], 4, args[6])
    assert all(torch.equal(p, q) for p, q in zip(one, two))


def test_native_module_has_the_kernels():
    C = require_native()
    for name in ("route_topk", "grouped_linear", "grouped_dgrad", "grouped_wgrad", "expert_combine", "grad_norm"):
        assert hasattr(C, name)
