"""Operators of an expert layer: a dense layer (product, bias, ReLU) split over
experts, each token going through the k experts its router chose.

    route = route_topk(logits, k)                        # gates, experts and the slot plan
    h = grouped_linear(x, w1, route.offsets, bias=b1, relu=True, rows=route.rows)
    y = grouped_linear(h, w2, route.offsets, bias=b2)
    out = expert_combine(y, route)

    dy, dgates = expert_combine_backward(dout, y, route)
    dw2, db2 = grouped_wgrad(dy, h, route.offsets)
    dh = grouped_dgrad(dy, w2, route.offsets, mask=h)
    dw1, db1 = grouped_wgrad(dh, x, route.offsets, rows=route.rows)
    dx = expert_combine(grouped_dgrad(dh, w1, route.offsets), route, weighted=False)
    dlogits = route_topk_backward(dgates, logits, route)

A token's choice owns a *slot*; slots are ordered by expert, then by token, and
expert e owns the slots ``offsets[e] .. offsets[e + 1] - 1``.  The plan lives on
the GPU: nothing here synchronises or copies to the host, and every call can be
captured into a graph.  The gradients are the explicit calls above: autograd does
not record a call, so where gradients are recorded an operand that requires one is
refused (parameters are taken under ``torch.no_grad()``).  Products take bfloat16 or float16 with fp32 sums; weight
and bias gradients are float32, as the trainers keep them.

A result buffer (``out``, ``dw``, ``db``) may not overlap an operand or another
result; column ranges of one buffer, and pieces that only touch, lie apart.

GPU tensors go to the HIP kernels (mandatory), host tensors to the same math in
PyTorch.  A call runs on its tensors' device, on that device's current stream.
Offsets and rows are not checked on the host (that would wait for the GPU): the
kernels clamp them to their buffers, so a wrong plan gives wrong numbers but no
access outside the operands.
"""
from __future__ import annotations

from operator import index
from typing import NamedTuple, Optional, Tuple

import torch

from .functional import check_unrecorded
from .native import require_native

MAX_EXPERTS, MAX_K = 512, 16
_HALF = (torch.bfloat16, torch.float16)


class Route(NamedTuple):
    """What the router decided for T tokens, k experts each (S = T k slots)."""
    gates: torch.Tensor    # [T, k] float32, 0 where there is no expert
    experts: torch.Tensor  # [T, k] int32, -1: none
    offsets: torch.Tensor  # [E + 1] int32: expert e owns slots offsets[e] .. offsets[e + 1] - 1
    rows: torch.Tensor     # [S] int32: the token of every slot, -1 behind offsets[E]
    slots: torch.Tensor    # [T, k] int32: the slot of every choice, -1: none


def _check(ok: bool, msg: str) -> None:
    if not ok:
        raise RuntimeError(msg)


def _rows2(t: torch.Tensor, dim: int, name: str) -> None:
    _check(t.dim() == dim, f"{name} must have {dim} axes, got {t.dim()}")
    _check(t.size(-1) <= 1 or t.stride(-1) == 1, f"{name}: the last axis must be contiguous")


def _i32(t: torch.Tensor, n: int, name: str) -> None:
    _check(t.dtype == torch.int32, f"{name} must be int32")
    _check(t.is_contiguous(), f"{name} must be contiguous")
    _check(t.numel() == n, f"{name} must hold {n} values, got {t.numel()}")


def _f32(t: torch.Tensor, n: int, name: str) -> None:
    _check(t.dtype == torch.float32, f"{name} must be float32")
    _check(t.is_contiguous(), f"{name} must be contiguous")
    _check(t.numel() == n, f"{name} must hold {n} values, got {t.numel()}")


def _out2(t: torch.Tensor, rows: int, cols: int, like: torch.Tensor, name: str = "out") -> None:
    _rows2(t, 2, name)
    _check(t.dtype == like.dtype, f"{name} must have the operands' type")
    _check(tuple(t.shape) == (rows, cols), f"{name} must be [{rows}, {cols}]")
    _check(rows <= 1 or t.stride(0) >= cols, f"{name}: rows must not overlap")


def _count(n: int, what: str) -> None:
    _check(n <= 0x7FFFFFFF, f"{what}: more than 2^31 - 1 rows")


def _weights(w: torch.Tensor) -> None:
    _rows2(w, 3, "w")
    E, N, K = w.shape
    _check(min(E, N, K) >= 1, "w must be [experts, out, in], none of them 0")
    _check(max(N, K) <= 0xFFFFFF and E <= 0xFFFF, "w is too large in one axis")


def _slots(slots: torch.Tensor, what: str) -> Tuple[int, int]:
    _check(slots.dim() == 2, f"slots must have 2 axes, got {slots.dim()}")
    T, k = slots.shape
    _check(1 <= k <= MAX_K, f"{what}: k must be 1..{MAX_K}, got {k}")
    _count(T * k, what)
    _i32(slots, T * k, "slots")
    return T, k


def _span(t: torch.Tensor) -> Tuple[int, int]:
    """The bytes from the first element to behind the last."""
    if t.numel() == 0:
        return t.data_ptr(), t.data_ptr()
    last = sum((n - 1) * s for n, s in zip(t.shape, t.stride()))
    return t.data_ptr(), t.data_ptr() + (last + 1) * t.element_size()


def _meets(a: torch.Tensor, b: torch.Tensor) -> bool:
    (alo, ahi), (blo, bhi) = _span(a), _span(b)
    if alo >= bhi or blo >= ahi:
        return False
    # column ranges of one buffer lie apart though their spans do not
    if a.dim() != 2 or b.dim() != 2:
        return True
    ea, eb = a.element_size(), b.element_size()
    ld = a.stride(0) * ea if a.shape[0] > 1 else b.stride(0) * eb
    if ld <= 0 or (b.shape[0] > 1 and b.stride(0) * eb != ld):
        return True
    at = (blo - alo) % ld  # b's first column, from a's
    return at < a.shape[1] * ea or at + b.shape[1] * eb > ld


def _apart(out: torch.Tensor, *ins: Optional[torch.Tensor], name: str = "out") -> None:
    _check(all(t is None or not _meets(out, t) for t in ins), f"{name} must not overlap an input")


def _host(*ts: Optional[torch.Tensor]) -> None:
    _check(all(t is None or not t.is_cuda for t in ts), "operands must be on one device")


# ---- router -----------------------------------------------------------------
def route_topk(logits: torch.Tensor, k: int, normalize: str = "topk") -> Route:
    """The ``k`` largest logits of every row of ``logits`` [T, E] (float32,
    bfloat16 or float16; E <= 512, k <= 16), ties to the lowest index, and the
    plan that groups them by expert.

    A logit of -inf (or NaN) is masked: its expert is never chosen.  A row with
    fewer than k others fills up with expert -1, slot -1, gate 0, so a padding
    token (all -inf) takes no slot at all.  Gates are the softmax over the
    chosen logits (``normalize="topk"``) or their part of the softmax over the
    whole row (``"all"``); they are not numbers where a chosen logit is +inf.
    """
    if logits.is_cuda:
        return Route(*require_native().route_topk(logits, index(k), normalize))
    check_unrecorded(logits)
    return _route_ref(logits, index(k), normalize)


def _check_route(T: int, E: int, k: int, normalize: str, logits: torch.Tensor) -> None:
    _check(1 <= E <= MAX_EXPERTS, f"route_topk: 1..{MAX_EXPERTS} experts, got {E}")
    _check(1 <= k <= min(E, MAX_K), f"route_topk: k must be 1..min({MAX_K}, experts), got {k}")
    _count(T * k, "route_topk")
    _check(normalize in ("topk", "all"), f"normalize must be 'topk' or 'all', got {normalize!r}")
    _check(logits.dtype in (torch.float32,) + _HALF, "logits must be float32, bfloat16 or float16")


def _route_ref(logits: torch.Tensor, k: int, normalize: str) -> Route:
    _rows2(logits, 2, "logits")
    T, E = logits.shape
    _check_route(T, E, k, normalize, logits)
    x = logits.float()
    x = torch.where(x.isnan(), torch.full_like(x, -torch.inf), x)
    val, ids = torch.sort(x, dim=1, descending=True, stable=True)
    val, ids = val[:, :k], ids[:, :k]
    live = val > -torch.inf
    m = x.amax(1, keepdim=True)
    m = torch.where(m > -torch.inf, m, torch.zeros_like(m))
    num = torch.exp(val - m)
    den = num.sum(1, keepdim=True) if normalize == "topk" else torch.exp(x - m).sum(1, keepdim=True)
    gates = torch.where(live, num / den, torch.zeros_like(num))
    flat = torch.where(live, ids, torch.full_like(ids, E)).reshape(-1)
    order = torch.argsort(flat, stable=True)
    used = int(live.sum())
    offsets = torch.zeros(E + 1, dtype=torch.int32)
    offsets[1:] = torch.bincount(flat, minlength=E + 1)[:E].cumsum(0)
    rows = torch.full((T * k,), -1, dtype=torch.int32)
    rows[:used] = (order[:used] // k).to(torch.int32)
    slots = torch.full((T * k,), -1, dtype=torch.int32)
    slots[order[:used]] = torch.arange(used, dtype=torch.int32)
    experts = torch.where(live, ids, torch.full_like(ids, -1)).to(torch.int32)
    return Route(gates, experts, offsets, rows, slots.view(T, k))


def route_topk_backward(dgates: torch.Tensor, logits: torch.Tensor, route: Route,
                        normalize: str = "topk") -> torch.Tensor:
    """The gradient of ``logits`` (its type) from the gates' ``dgates`` [T, k]
    (float32): zero at every expert that was not chosen for ``"topk"``, through
    the whole row's softmax for ``"all"``."""
    if logits.is_cuda:
        return require_native().route_topk_backward(dgates, logits, route.gates, route.experts, normalize)
    check_unrecorded(dgates, logits, route.gates)
    _host(dgates, *route)
    _rows2(logits, 2, "logits")
    T, E = logits.shape
    _check(dgates.dim() == 2, f"dgates must have 2 axes, got {dgates.dim()}")
    k = dgates.shape[1]
    _check_route(T, E, k, normalize, logits)
    for t, name in ((dgates, "dgates"), (route.gates, "gates")):
        _f32(t, T * k, name)
    _i32(route.experts, T * k, "experts")
    gates, ids = route.gates, route.experts.long()
    live = ids >= 0
    w = torch.where(live, gates * dgates, torch.zeros_like(gates))
    inner = w.sum(1, keepdim=True)
    d = torch.zeros(T, E)
    if normalize == "all":
        x = logits.float()
        x = torch.where(x.isnan(), torch.full_like(x, -torch.inf), x)
        m = x.amax(1, keepdim=True)
        ex = torch.exp(x - torch.where(m > -torch.inf, m, torch.zeros_like(m)))
        den = ex.sum(1, keepdim=True)
        d = -torch.where(den > 0, ex / den, torch.zeros_like(ex)) * inner
    else:
        w = torch.where(live, gates * (dgates - inner), torch.zeros_like(gates))
    d.scatter_add_(1, ids.clamp(min=0), w)
    return d.to(logits.dtype)


# ---- products grouped by expert -----------------------------------------------
def _groups(offsets: torch.Tensor, S: int):
    off = offsets.tolist()
    for e in range(len(off) - 1):
        a = min(max(off[e], 0), S)
        b = min(max(off[e + 1], a), S)
        yield e, a, b


def _take(x: torch.Tensor, rows: Optional[torch.Tensor]) -> torch.Tensor:
    if rows is None:
        return x.float()
    ok = (rows >= 0) & (rows < x.shape[0])
    if x.shape[0] == 0:
        return torch.zeros(rows.numel(), x.shape[1])
    return torch.where(ok[:, None], x.float()[rows.long().clamp(0, x.shape[0] - 1)], torch.zeros(()))


def grouped_linear(x: torch.Tensor, w: torch.Tensor, offsets: torch.Tensor, bias: Optional[torch.Tensor] = None,
                   relu: bool = False, rows: Optional[torch.Tensor] = None,
                   out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``y[s] = act(x[rows[s]] @ w[e].T + bias[e])`` for every slot s of group e.

    x [T, K], w [E, N, K] (the layers' [out, in] layout) and y [S, N] are
    bfloat16 or float16, bias [E, N] is float32, offsets [E + 1] and rows [S]
    are int32.  Without ``rows`` slot s reads row s.  Rows may be strided, with
    a contiguous last axis.  A slot whose row is outside x counts as a zero row.
    Slots in no group: zero in a fresh result, left as they were in ``out``.
    """
    if x.is_cuda:
        return require_native().grouped_linear(x, w, offsets, bias, relu, rows, out)
    check_unrecorded(x, w, bias, out)
    _host(w, offsets, bias, rows, out)
    _rows2(x, 2, "x")
    _weights(w)
    E, N, K = w.shape
    _check(x.dtype in _HALF, "x must be bfloat16 or float16")
    _check(w.dtype == x.dtype, "w must have x's type")
    _check(x.shape[1] == K, f"x has {x.shape[1]} columns, w takes {K}")
    _i32(offsets, E + 1, "offsets")
    if rows is not None:
        _check(rows.dim() == 1, "rows must have 1 axis")
        _i32(rows, rows.numel(), "rows")
    if bias is not None:
        _rows2(bias, 2, "bias")
        _check(bias.dtype == torch.float32, "bias must be float32")
        _check(tuple(bias.shape) == (E, N), f"bias must be [{E}, {N}]")
    S = x.shape[0] if rows is None else rows.numel()
    _count(max(S, x.shape[0]), "grouped_linear")
    if out is not None:
        _out2(out, S, N, x)
        _apart(out, x, w, offsets, bias, rows)
    y = torch.zeros(S, N, dtype=x.dtype) if out is None else out
    xs = _take(x, rows)
    for e, a, b in _groups(offsets, S):
        z = xs[a:b] @ w[e].float().t()
        if bias is not None:
            z = z + bias[e]
        y[a:b] = torch.relu(z) if relu else z
    return y


def grouped_dgrad(dz: torch.Tensor, w: torch.Tensor, offsets: torch.Tensor, mask: Optional[torch.Tensor] = None,
                  out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``dx[s] = dz[s] @ w[e]`` [S, K] for every slot s of group e, kept where
    ``mask[s] > 0`` (the activation a ReLU below produced, [S, K]).  Per slot:
    ``expert_combine(dx, route, weighted=False)`` sums a token's slots."""
    if dz.is_cuda:
        return require_native().grouped_dgrad(dz, w, offsets, mask, out)
    check_unrecorded(dz, w, mask, out)
    _host(w, offsets, mask, out)
    _rows2(dz, 2, "dz")
    _weights(w)
    E, N, K = w.shape
    _check(dz.dtype in _HALF, "dz must be bfloat16 or float16")
    _check(w.dtype == dz.dtype, "w must have dz's type")
    _check(dz.shape[1] == N, f"dz has {dz.shape[1]} columns, w gives {N}")
    _i32(offsets, E + 1, "offsets")
    S = dz.shape[0]
    _count(S, "grouped_dgrad")
    if mask is not None:
        _rows2(mask, 2, "mask")
        _check(mask.dtype == dz.dtype, "mask must have dz's type")
        _check(tuple(mask.shape) == (S, K), f"mask must be [{S}, {K}]")
    if out is not None:
        _out2(out, S, K, dz)
        _apart(out, dz, w, offsets, mask)
    dx = torch.zeros(S, K, dtype=dz.dtype) if out is None else out
    for e, a, b in _groups(offsets, S):
        z = dz[a:b].float() @ w[e].float()
        dx[a:b] = z if mask is None else torch.where(mask[a:b] > 0, z, torch.zeros(()))
    return dx


def grouped_wgrad(dz: torch.Tensor, x: torch.Tensor, offsets: torch.Tensor, rows: Optional[torch.Tensor] = None,
                  bias: bool = True, dw: Optional[torch.Tensor] = None,
                  db: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """``dw[e] = dz_e.T @ x_e`` [E, N, K] and ``db[e]`` = column sums of dz_e
    [E, N], float32, over the slots of group e (an empty group: zeros), of which
    there may be 2^31 - 256 in all.  ``dw``
    / ``db``: buffers to write (dw's rows may be strided); ``bias=False``
    leaves the bias gradient out (None)."""
    if dz.is_cuda:
        return require_native().grouped_wgrad(dz, x, offsets, rows, bias, dw, db)
    check_unrecorded(dz, x, dw, db)
    _host(x, offsets, rows, dw, db)
    _rows2(dz, 2, "dz")
    _rows2(x, 2, "x")
    _check(dz.dtype in _HALF, "dz must be bfloat16 or float16")
    _check(x.dtype == dz.dtype, "x must have dz's type")
    _check(offsets.dim() == 1 and offsets.numel() >= 2, "offsets must have 1 axis and hold experts + 1 values")
    E, (S, N), K = offsets.numel() - 1, dz.shape, x.shape[1]
    _i32(offsets, E + 1, "offsets")
    _check(min(N, K) >= 1 and max(N, K) <= 0xFFFFFF and E <= 0xFFFF, "grouped_wgrad: bad sizes")
    if rows is not None:
        _check(rows.dim() == 1, "rows must have 1 axis")
        _i32(rows, S, "rows")
    else:
        _check(x.shape[0] == S, f"x has {x.shape[0]} rows, dz {S}")
    _check(S <= 0x7FFFFFFF - 255, "grouped_wgrad: more than 2^31 - 256 rows")
    _count(x.shape[0], "grouped_wgrad")
    _check(bias or db is None, "a bias gradient buffer was given with bias=False")
    if dw is not None:
        _rows2(dw, 3, "dw")
        _check(dw.dtype == torch.float32, "dw must be float32")
        _check(tuple(dw.shape) == (E, N, K), f"dw must be [{E}, {N}, {K}]")
        _check((N <= 1 or dw.stride(1) >= K) and (E <= 1 or dw.stride(0) >= (N - 1) * dw.stride(1) + K),
               "dw: rows must not overlap")
        _apart(dw, dz, x, offsets, rows, db, name="dw")
    if db is not None:
        _f32(db, E * N, "db")
        _apart(db, dz, x, offsets, rows, name="db")
    if dw is None:
        dw = torch.empty(E, N, K)
    if db is None and bias:
        db = torch.empty(E, N)
    xs, d = _take(x, rows), dz.float()
    for e, a, b in _groups(offsets, S):
        dw[e] = d[a:b].t() @ xs[a:b]
        if bias:
            db.view(E, N)[e] = d[a:b].sum(0)
    return dw, db


# ---- combine --------------------------------------------------------------------
def expert_combine(y: torch.Tensor, route: Route, weighted: bool = True,
                   out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``out[t] = sum_j gates[t, j] * y[slots[t, j]]`` [T, N] in y's type
    (bfloat16 or float16; ``weighted=False``: every gate 1).  Choices without a
    slot contribute nothing; a token without any gets zeros."""
    gates = route.gates if weighted else None
    if y.is_cuda:
        return require_native().expert_combine(y, route.slots, gates, out)
    check_unrecorded(y, gates, out)
    _host(*route, out)
    _rows2(y, 2, "y")
    _check(y.dtype in _HALF, "y must be bfloat16 or float16")
    T, k = _slots(route.slots, "expert_combine")
    _check(1 <= y.shape[1] <= 0x3FFFFF, "expert_combine: 1..4194303 columns")
    _count(y.shape[0], "expert_combine")
    if weighted:
        _f32(gates, T * k, "gates")
    if out is not None:
        _out2(out, T, y.shape[1], y)
        _apart(out, y, route.slots, gates)
    acc = torch.zeros(T, y.shape[1])
    for j in range(k):
        v, s = _take(y, route.slots[:, j]), route.slots[:, j:j + 1]
        g = torch.where((s >= 0) & (s < y.shape[0]), gates[:, j:j + 1], torch.zeros(())) if weighted else 1.0
        acc += v * g
    if out is None:
        return acc.to(y.dtype)
    out.copy_(acc)
    return out


def expert_combine_backward(dout: torch.Tensor, y: torch.Tensor,
                            route: Route) -> Tuple[torch.Tensor, torch.Tensor]:
    """Gradients of ``expert_combine(y, route)``: ``dy[slot] = gate * dout[t]``
    in y's type (zero behind the last slot in use) and ``dgates[t, j] =
    <dout[t], y[slot]>`` in float32.  A slot belongs to one choice."""
    if y.is_cuda:
        return require_native().expert_combine_backward(dout, y, route.slots, route.gates, route.offsets)
    check_unrecorded(dout, y, route.gates)
    _host(dout, *route)
    _rows2(dout, 2, "dout")
    _rows2(y, 2, "y")
    _check(y.dtype in _HALF, "y must be bfloat16 or float16")
    _check(dout.dtype == y.dtype, "dout must have y's type")
    T, k = _slots(route.slots, "expert_combine_backward")
    S, N = y.shape
    _check(1 <= N <= 0x3FFFFF, "expert_combine_backward: 1..4194303 columns")
    _f32(route.gates, T * k, "gates")
    _check(route.offsets.dim() == 1 and route.offsets.numel() >= 2,
           "offsets must have 1 axis and hold experts + 1 values")
    _i32(route.offsets, route.offsets.numel(), "offsets")
    _check(tuple(dout.shape) == (T, N), f"dout must be [{T}, {N}]")
    _check(S == T * k, f"y must have one row a slot: {T * k}, got {S}")
    d = dout.float()
    dy = torch.zeros(S, N, dtype=y.dtype)
    dg = torch.zeros(T, k)
    for j in range(k):
        s = route.slots[:, j].long()
        t = ((s >= 0) & (s < S)).nonzero()[:, 0]
        dy[s[t]] = (d[t] * route.gates[t, j:j + 1]).to(y.dtype)
        dg[t, j] = (d[t] * y[s[t]].float()).sum(1)
    return dy, dg
