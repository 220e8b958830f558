"""Plain 64-bit forms of the expert-layer operators and the error their kernels
may make, shared by the CPU and GPU tests."""
import torch

U32 = 2.0 ** -23  # one step of an fp32 sum, truncation included


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def offsets_of(sizes, lead=0):
    off = [lead]
    for n in sizes:
        off.append(off[-1] + n)
    return torch.tensor(off, dtype=torch.int32)


def groups(sizes, lead=0):
    at = lead
    for e, n in enumerate(sizes):
        yield e, slice(at, at + n)
        at += n


def rounded_tol(ref, mag, terms, dtype):
    """|error| of a sum of `terms` products rounded once to `dtype`: half a step
    of the value, one fp32 step a term of the sum of magnitudes `mag`, and the
    smallest subnormal's half (fp16)."""
    tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2 if dtype != torch.float32 else 0.0
    acc = (terms + 2) * U32 * mag
    return half_step(dtype) * (ref.abs() + acc) + acc + tiny


def close(got, ref, tol, what=""):
    err = (got.double() - ref).abs()
    bad = ~(err <= tol)
    assert not bad.any(), (what, int(bad.sum()), float(err.max()), float((err / tol.clamp(min=1e-300)).max()))


def linear64(x, w, sizes, bias=None, relu=False, rows=None, lead=0):
    """(result, sum of magnitudes) over the slots in a group; slots outside: 0."""
    xs = x.double() if rows is None else x.double()[rows.long()]
    S, N = xs.shape[0], w.shape[1]
    y = torch.zeros(S, N, dtype=torch.float64, device=x.device)
    mag = torch.zeros_like(y)
    for e, sl in groups(sizes, lead):
        y[sl] = xs[sl] @ w[e].double().t().contiguous()
        mag[sl] = xs[sl].abs() @ w[e].double().abs().t().contiguous()
        if bias is not None:
            y[sl] += bias[e].double()
            mag[sl] += bias[e].double().abs()
    return (torch.relu(y) if relu else y), mag


def dgrad64(dz, w, sizes, mask=None, lead=0):
    S, K = dz.shape[0], w.shape[2]
    dx = torch.zeros(S, K, dtype=torch.float64, device=dz.device)
    mag = torch.zeros_like(dx)
    for e, sl in groups(sizes, lead):
        dx[sl] = dz[sl].double() @ w[e].double()
        mag[sl] = dz[sl].double().abs() @ w[e].double().abs()
    if mask is not None:
        dx = torch.where(mask > 0, dx, torch.zeros_like(dx))
    return dx, mag


def wgrad64(dz, x, sizes, rows=None, lead=0):
    xs = x.double() if rows is None else x.double()[rows.long()]
    E, N, K = len(sizes), dz.shape[1], x.shape[1]
    dw = torch.zeros(E, N, K, dtype=torch.float64, device=dz.device)
    mag, db, dbm = torch.zeros_like(dw), dw.new_zeros(E, N), dw.new_zeros(E, N)
    for e, sl in groups(sizes, lead):
        d = dz[sl].double()
        dw[e] = d.t().contiguous() @ xs[sl]
        mag[e] = d.abs().t().contiguous() @ xs[sl].abs()
        db[e], dbm[e] = d.sum(0), d.abs().sum(0)
    return dw, mag, db, dbm


def route64(logits, k, normalize):
    """Row by row, from the definition: (gates, experts, offsets, rows, slots)."""
    x = logits.double().cpu()
    T, E = x.shape
    gates = torch.zeros(T, k, dtype=torch.float64)
    experts = torch.full((T, k), -1, dtype=torch.int32)
    for t in range(T):
        row = [(-v, e) for e, v in enumerate(x[t].tolist()) if v == v and v != -float("inf")]
        pick = [e for _, e in sorted(row)[:k]]
        if not pick:
            continue
        m = max(x[t, e].item() for e in pick)
        over = pick if normalize == "topk" else [e for _, e in row]
        den = sum(torch.exp(x[t, e] - m).item() for e in over)
        for j, e in enumerate(pick):
            gates[t, j] = torch.exp(x[t, e] - m).item() / den
            experts[t, j] = e
    offsets = torch.zeros(E + 1, dtype=torch.int32)
    rows = torch.full((T * k,), -1, dtype=torch.int32)
    slots = torch.full((T, k), -1, dtype=torch.int32)
    at = 0
    for e in range(E):
        offsets[e] = at
        for t, j in (experts == e).nonzero().tolist():
            rows[at], slots[t, j] = t, at
            at += 1
    offsets[E] = at
    return gates, experts, offsets, rows, slots


def route_bwd64(dgates, logits, experts, normalize):
    x = logits.double().cpu()
    x = torch.where(x.isnan(), torch.full_like(x, -torch.inf), x)
    T, E = x.shape
    d = torch.zeros(T, E, dtype=torch.float64)
    for t in range(T):
        pick = [e for e in experts[t].tolist() if e >= 0]
        if not pick:
            continue
        sel = torch.full((E,), -torch.inf, dtype=torch.float64)
        over = pick if normalize == "topk" else range(E)
        for e in over:
            sel[e] = x[t, e]
        p = torch.softmax(sel, 0)
        up = torch.zeros(E, dtype=torch.float64)
        for j, e in enumerate(pick):
            up[e] = dgates[t, j].double()
        d[t] = p * (up - (p * up).sum())
    return d
