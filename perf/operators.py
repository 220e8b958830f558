"""What the expert-layer operators and gradient clipping are measured on.

Operators (hipdsml.ops.experts, hipdsml.ops.functional):

* route_topk / route_topk_backward: the k experts of every token, their gates and the slot plan;
* grouped_linear / grouped_dgrad / grouped_wgrad: one matrix product per expert over ragged row groups;
* expert_combine / expert_combine_backward: the gated sum of a token's expert rows;
* clip_grad_norm_: the global gradient norm over many tensors, and clipping by it.

``own = False`` computes them in plain torch, in 32 bits (sums of squares in 64), ``own = True`` calls the framework.
"""
import math
import random

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}
DEV = "cuda"


def listed():
    return [
        # Four requests' next tokens choose 2 of 8 experts: the smallest call, nothing but latency.
        dict(name="route_decode", op="route", T=4, E=8, k=2, dtype="f32", normalize="topk", drop=0.0),
        # A training batch's tokens, some of them padding (rows masked whole).
        dict(name="route_train", op="route", T=65536, E=64, k=4, dtype="bf16", normalize="topk", drop=0.03),
        # The router's gradient in training, gates normalised over all experts.
        dict(name="route_backward", op="route_bwd", T=32768, E=128, k=8, dtype="f32", normalize="all", drop=0.02),
        # Eight requests' next tokens through an expert layer: every used expert's weights are read for a few rows.
        dict(name="linear_decode", op="linear", T=8, k=2, E=8, K=4096, N=4096, dtype="bf16", skew=0.0, bias=True,
             relu=True, gather=True),
        # A prompt's rows, already grouped, over uneven experts (some empty), odd widths, no activation.
        dict(name="linear_ragged", op="linear", T=5003, k=1, E=16, K=784, N=1000, dtype="f16", skew=1.5, bias=True,
             relu=False, gather=False),
        # The largest: a training batch through the wide layer, two experts a token.
        dict(name="linear_train", op="linear", T=16384, k=2, E=8, K=4096, N=4096, dtype="bf16", skew=0.3, bias=True,
             relu=True, gather=True),
        # The activation gradient of the same kind of layer, through the ReLU below it.
        dict(name="dgrad_train", op="dgrad", T=8192, k=2, E=8, K=4096, N=4096, dtype="bf16", skew=0.3, mask=True),
        # The weight and bias gradients, rows gathered from the tokens, uneven experts.
        dict(name="wgrad_train", op="wgrad", T=8192, k=2, E=8, K=4096, N=4096, dtype="bf16", skew=0.8, gather=True),
        # Every token's expert rows back into one row.
        dict(name="combine_train", op="combine", T=16384, k=2, N=4096, dtype="bf16", weighted=True),
        # Its gradient, odd sizes and the other type.
        dict(name="combine_backward", op="combine_bwd", T=8191, k=4, N=1000, dtype="f16"),
        # The gradients of the 784-128-64-10 model, clipped: six small tensors.
        dict(name="clip_small", op="clip", sizes="mlp", count=6, total=109386, dtype="f32", over=4.0),
        # The gradients of a model of many tensors, from biases to whole expert weights.
        dict(name="clip_large", op="clip", sizes="many", count=60, total=400_000_000, dtype="f32", over=2.5),
    ]


def _logint(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["route", "route_bwd", "linear", "linear", "dgrad", "wgrad", "combine", "combine_bwd", "clip"])
    half = rng.choice(["bf16", "f16"])
    if op in ("route", "route_bwd"):
        E = _logint(rng, 2, 256)
        return dict(op=op, T=_logint(rng, 1, 65536), E=E, k=rng.randint(1, min(8, E)),
                    dtype=rng.choice(["f32", "bf16", "f16"]), normalize=rng.choice(["topk", "all"]),
                    drop=rng.choice([0.0, 0.05]))
    if op in ("linear", "dgrad", "wgrad"):
        while True:
            c = dict(op=op, T=_logint(rng, 1, 16384), k=rng.randint(1, 4), E=_logint(rng, 1, 64),
                     K=_logint(rng, 10, 4096), N=_logint(rng, 10, 4096), dtype=half, skew=rng.choice([0.0, 0.5, 1.5]))
            if rng.random() < 0.6:  # widths in whole 16-byte rows, as layers mostly have
                c["K"], c["N"] = -(-c["K"] // 8) * 8, -(-c["N"] // 8) * 8
            if c["T"] * c["k"] <= 32768 and c["E"] * c["K"] * c["N"] <= 8 * 4096 * 4096:
                break
        if op == "linear":
            c.update(bias=rng.random() < 0.7, relu=rng.random() < 0.5, gather=rng.random() < 0.5)
        elif op == "dgrad":
            c.update(mask=rng.random() < 0.5)
        else:
            c.update(gather=rng.random() < 0.5)
        if not c.get("gather", op == "dgrad"):
            c["T"], c["k"] = c["T"] * c["k"], 1
        return c
    if op in ("combine", "combine_bwd"):
        c = dict(op=op, T=_logint(rng, 1, 16384), k=rng.randint(1, 4), N=_logint(rng, 10, 4096), dtype=half)
        if op == "combine":
            c["weighted"] = rng.random() < 0.7
        return c
    return dict(op="clip", sizes="many", count=_logint(rng, 1, 60), total=_logint(rng, 1000, 200_000_000),
                dtype=rng.choice(["f32", "bf16"]), over=rng.choice([0.5, 3.0]))


# ---- what a case fixes apart from the seed ----------------------------------------------------------
def _group_sizes(c):
    """Rows of every expert: even for skew 0, the more uneven (empty ones among them) the larger it is."""
    rng = random.Random(f"{c['T']}-{c['k']}-{c['E']}-{c['K']}-{c['N']}")
    E, S = c["E"], c["T"] * c["k"]
    w = [math.exp(c["skew"] * rng.gauss(0, 1)) for _ in range(E)]
    if c["skew"] > 1 and E > 3:
        w[rng.randrange(E)] = 0.0
        w[rng.randrange(E)] = 0.0
    if sum(w) == 0.0:
        w = [1.0] * E
    tot, acc, out, prev = sum(w), 0.0, [], 0
    for e in range(E):
        acc += w[e]
        end = S if e == E - 1 else min(S, int(round(S * acc / tot)))
        out.append(end - prev)
        prev = end
    return out


def _tensor_sizes(c):
    if c["sizes"] == "mlp":
        d = (784, 128, 64, 10)
        return [n for a, b in zip(d, d[1:]) for n in (a * b, b)]
    rng = random.Random(f"{c['count']}-{c['total']}")
    w = [math.exp(2.0 * rng.gauss(0, 1)) for _ in range(c["count"])]
    return [max(1, int(c["total"] * x / sum(w))) for x in w]


def work(c):
    op, b = c["op"], BYTES[c["dtype"]]
    if op == "route":
        return {"bytes": c["T"] * (c["E"] * b + c["k"] * 16) + 4 * (c["E"] + 1), "flops": c["T"] * c["E"] * 4}
    if op == "route_bwd":
        rd = c["T"] * c["E"] * b if c["normalize"] == "all" else 0
        return {"bytes": rd + c["T"] * (c["E"] * b + c["k"] * 12), "flops": c["T"] * c["E"] * 4}
    if op in ("linear", "dgrad", "wgrad"):
        sizes = _group_sizes(c)
        S, used = sum(sizes), sum(1 for n in sizes if n)
        T = c["T"] if c.get("gather") else S
        wn = c["K"] * c["N"]
        flops = 2 * S * wn
        if op == "linear":
            by = T * c["K"] * b + used * wn * b + S * c["N"] * b + (used * c["N"] * 4 if c["bias"] else 0)
        elif op == "dgrad":
            by = S * c["N"] * b + used * wn * b + S * c["K"] * b * (2 if c["mask"] else 1)
        else:
            by = S * c["N"] * b + T * c["K"] * b + c["E"] * (wn + c["N"]) * 4
        return {"bytes": by, "flops": flops}
    if op in ("combine", "combine_bwd"):
        T, k, N = c["T"], c["k"], c["N"]
        if op == "combine":
            return {"bytes": (T * k + T) * N * b + T * k * 8, "flops": 2 * T * k * N}
        return {"bytes": (2 * T * k + T) * N * b + T * k * 12, "flops": 3 * T * k * N}
    n = sum(_tensor_sizes(c))
    # every gradient read once and its clipped value written once
    return {"bytes": 2 * n * b, "flops": 3 * n}


# ---- inputs -----------------------------------------------------------------------------------------
def _randn(g, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(*shape, generator=g, device=DEV) * scale).to(dtype)


def _logits(c, g):
    x = _randn(g, c["T"], c["E"], scale=1.5).to(DTYPES[c["dtype"]])
    if c["drop"]:  # padding: no expert may be chosen
        x[torch.rand(c["T"], generator=g, device=DEV) < c["drop"]] = -math.inf
    return x


def prepare(c, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    op, dt = c["op"], DTYPES[c["dtype"]]
    st = {"case": c}
    if own:
        from hipdsml.ops import experts, functional
        st["experts"], st["functional"] = experts, functional
    if op in ("route", "route_bwd"):
        st["logits"] = _logits(c, g)
        if op == "route_bwd":
            gates, ids, offsets, rows, slots = _plain_route(st["logits"], c["k"], c["normalize"])
            st["route"] = (gates, ids, offsets, rows, slots)
            st["dgates"] = _randn(g, c["T"], c["k"], scale=0.02)
    elif op in ("linear", "dgrad", "wgrad"):
        sizes = _group_sizes(c)
        S, E, K, N = sum(sizes), c["E"], c["K"], c["N"]
        st["sizes"] = sizes
        st["offsets"] = torch.tensor([0] + torch.tensor(sizes).cumsum(0).tolist(), dtype=torch.int32, device=DEV)
        if c.get("gather"):  # every token k times, by expert and then by token
            tok = torch.arange(S, device=DEV) // c["k"]
            tok = tok[torch.randperm(S, generator=g, device=DEV)]
            exp = torch.repeat_interleave(torch.arange(E, device=DEV), torch.tensor(sizes, device=DEV))
            st["rows"] = tok[torch.argsort(exp * c["T"] + tok)].to(torch.int32)
        if op == "linear":
            st["x"] = _randn(g, c["T"], K, dtype=dt)
            st["w"] = _randn(g, E, N, K, dtype=dt, scale=K ** -0.5)
            if c["bias"]:
                st["bias"] = _randn(g, E, N, scale=0.1)
        elif op == "dgrad":
            st["dz"] = _randn(g, S, N, dtype=dt, scale=0.1)
            st["w"] = _randn(g, E, N, K, dtype=dt, scale=K ** -0.5)
            if c["mask"]:
                st["mask"] = torch.relu(_randn(g, S, K, dtype=dt))
        else:
            st["dz"] = _randn(g, S, N, dtype=dt, scale=0.1)
            st["x"] = torch.relu(_randn(g, c["T"], K, dtype=dt))
    elif op in ("combine", "combine_bwd"):
        T, k, N = c["T"], c["k"], c["N"]
        # a plan of T k slots: choose k of max(8, 2 k) experts at random
        gates, ids, offsets, rows, slots = _plain_route(_randn(g, T, max(8, 2 * k)), k, "topk")
        st["route"] = (gates, ids, offsets, rows, slots)
        st["y"] = _randn(g, T * k, N, dtype=dt)
        if op == "combine_bwd":
            st["dout"] = _randn(g, T, N, dtype=dt, scale=0.1)
    else:
        sizes = _tensor_sizes(c)
        scale = [0.01 * (1 + 0.5 * (i % 7)) for i in range(len(sizes))]
        st["grads"] = [_randn(g, n, dtype=dt, scale=s) for n, s in zip(sizes, scale)]
        st["out"] = [torch.empty_like(t) for t in st["grads"]]
        st["max_norm"] = math.sqrt(sum(n * s * s for n, s in zip(sizes, scale))) / c["over"]
    if own and "route" in st:
        st["route"] = st["experts"].Route(*st["route"])
    return st


# ---- the plain form ---------------------------------------------------------------------------------
def _plain_route(logits, k, normalize):
    T, E = logits.shape
    x = logits.float()
    val, ids = torch.sort(x, dim=1, descending=True, stable=True)  # ties: the lowest index first
    val, ids = val[:, :k], ids[:, :k]
    live = val > -math.inf
    m = x.max(dim=1, keepdim=True).values
    m = torch.where(m > -math.inf, m, torch.zeros_like(m))
    ex = torch.exp(val - m)
    den = ex.sum(1, keepdim=True) if normalize == "topk" else torch.exp(x - m).sum(1, keepdim=True)
    gates = torch.where(live, ex / den, torch.zeros_like(ex))
    ids = torch.where(live, ids, torch.full_like(ids, -1))
    flat = torch.where(live, ids, torch.full_like(ids, E)).reshape(-1)
    order = torch.argsort(flat, stable=True)  # by expert, then by token; the masked ones last
    counts = (flat[None, :] == torch.arange(E, device=x.device)[:, None]).sum(1)
    offsets = torch.zeros(E + 1, dtype=torch.int64, device=x.device)
    offsets[1:] = counts.cumsum(0)
    slots = torch.empty_like(order)
    slots[order] = torch.arange(T * k, device=x.device)
    slots = torch.where(live.reshape(-1), slots, torch.full_like(slots, -1)).reshape(T, k)
    rows = torch.where(flat[order] < E, order // k, torch.full_like(order, -1))
    i32 = torch.int32
    return gates, ids.to(i32), offsets.to(i32), rows.to(i32), slots.to(i32)


def _plain_route_bwd(dgates, logits, gates, ids, normalize):
    T, E = logits.shape
    live = ids >= 0
    inner = (gates * dgates).sum(1, keepdim=True)
    safe = torch.where(live, ids, torch.zeros_like(ids)).long()
    if normalize == "topk":
        dl = torch.zeros(T, E, device=logits.device)
        dl.scatter_add_(1, safe, torch.where(live, gates * (dgates - inner), torch.zeros_like(gates)))
    else:
        x = logits.float()
        m = x.max(dim=1, keepdim=True).values
        m = torch.where(m > -math.inf, m, torch.zeros_like(m))
        ex = torch.exp(x - m)
        den = ex.sum(1, keepdim=True)
        p = torch.where(den > 0, ex / den, torch.zeros_like(ex))
        dl = -p * inner
        dl.scatter_add_(1, safe, torch.where(live, gates * dgates, torch.zeros_like(gates)))
    return dl.to(logits.dtype)


def _bounds(sizes):
    at = 0
    for e, n in enumerate(sizes):
        if n:
            yield e, at, at + n
        at += n


def _plain_linear(st, c):
    x = st["x"].float()
    if c["gather"]:
        x = x[st["rows"].long()]
    y = torch.empty(x.shape[0], c["N"], dtype=st["x"].dtype, device=x.device)
    for e, a, b in _bounds(st["sizes"]):
        z = x[a:b] @ st["w"][e].float().t()
        if c["bias"]:
            z = z + st["bias"][e]
        if c["relu"]:
            z = torch.relu(z)
        y[a:b] = z.to(y.dtype)
    return y


def _plain_dgrad(st, c):
    dx = torch.empty(st["dz"].shape[0], c["K"], dtype=st["dz"].dtype, device=st["dz"].device)
    for e, a, b in _bounds(st["sizes"]):
        z = st["dz"][a:b].float() @ st["w"][e].float()
        if c["mask"]:
            z = z * (st["mask"][a:b] > 0)
        dx[a:b] = z.to(dx.dtype)
    return dx


def _plain_wgrad(st, c):
    dz, x = st["dz"].float(), st["x"].float()
    if c["gather"]:
        x = x[st["rows"].long()]
    dw = torch.zeros(c["E"], c["N"], c["K"], device=dz.device)
    db = torch.zeros(c["E"], c["N"], device=dz.device)
    for e, a, b in _bounds(st["sizes"]):
        dw[e] = dz[a:b].t() @ x[a:b]
        db[e] = dz[a:b].sum(0)
    return dw, db


def _plain_combine(y, gates, slots, weighted):
    out = torch.zeros(slots.shape[0], y.shape[1], device=y.device)
    for j in range(slots.shape[1]):
        s = slots[:, j].long()
        z = y[s.clamp(min=0)].float() * (s >= 0)[:, None]
        out += z * gates[:, j:j + 1] if weighted else z
    return out.to(y.dtype)


def _plain_combine_bwd(dout, y, gates, slots):
    S = y.shape[0]
    dy = torch.zeros(S + 1, y.shape[1], dtype=y.dtype, device=y.device)  # row S takes what has no slot
    dg = torch.zeros(gates.shape, device=y.device)
    d = dout.float()
    for j in range(slots.shape[1]):
        s = slots[:, j].long()
        live = s >= 0
        dg[:, j] = (d * y[s.clamp(min=0)].float()).sum(1) * live
        dy[torch.where(live, s, torch.full_like(s, S))] = (d * gates[:, j:j + 1]).to(y.dtype)
    return dy[:S], dg


def _plain_clip(st):
    total = torch.zeros((), dtype=torch.float64, device=DEV)
    for t in st["grads"]:
        total += t.double().square().sum()
    norm = total.sqrt()
    coef = torch.clamp(st["max_norm"] / (norm + 1e-6), max=1.0).float()
    for t, o in zip(st["grads"], st["out"]):
        o.copy_(t.float() * coef)
    return norm.float(), st["out"]


def run(st):
    c = st["case"]
    op = c["op"]
    if own:
        X = st["experts"]
        if op == "route":
            return tuple(X.route_topk(st["logits"], c["k"], normalize=c["normalize"]))
        if op == "route_bwd":
            return X.route_topk_backward(st["dgates"], st["logits"], st["route"], normalize=c["normalize"])
        if op == "linear":
            return X.grouped_linear(st["x"], st["w"], st["offsets"], bias=st.get("bias"), relu=c["relu"],
                                    rows=st.get("rows"))
        if op == "dgrad":
            return X.grouped_dgrad(st["dz"], st["w"], st["offsets"], mask=st.get("mask"))
        if op == "wgrad":
            return X.grouped_wgrad(st["dz"], st["x"], st["offsets"], rows=st.get("rows"))
        if op == "combine":
            return X.expert_combine(st["y"], st["route"], weighted=c["weighted"])
        if op == "combine_bwd":
            return X.expert_combine_backward(st["dout"], st["y"], st["route"])
        norm = st["functional"].clip_grad_norm_(st["grads"], st["max_norm"], out=st["out"])
        return norm, st["out"]
    if op == "route":
        return _plain_route(st["logits"], c["k"], c["normalize"])
    if op == "route_bwd":
        gates, ids = st["route"][0], st["route"][1]
        return _plain_route_bwd(st["dgates"], st["logits"], gates, ids, c["normalize"])
    if op == "linear":
        return _plain_linear(st, c)
    if op == "dgrad":
        return _plain_dgrad(st, c)
    if op == "wgrad":
        return _plain_wgrad(st, c)
    if op == "combine":
        return _plain_combine(st["y"], st["route"][0], st["route"][4], c["weighted"])
    if op == "combine_bwd":
        return _plain_combine_bwd(st["dout"], st["y"], st["route"][0], st["route"][4])
    return _plain_clip(st)


# ---- the definition in 64 bits ----------------------------------------------------------------------
def exact(c, seed):
    global own
    was, own = own, False
    try:
        st = prepare(c, seed)
    finally:
        own = was
    op = c["op"]
    if op == "route":
        p = torch.exp(st["logits"].double())  # masked logits: exactly 0
        T, E = p.shape
        left = st["logits"].double().clone()
        k = c["k"]
        ids = torch.full((T, k), -1, dtype=torch.int64, device=DEV)
        col = torch.arange(E, device=DEV)
        for j in range(k):  # the largest that is left, the lowest index among equals
            best = left.max(1, keepdim=True).values
            at = torch.where(left == best, col, torch.full_like(col, E)).min(1).values
            ok = best[:, 0] > -math.inf
            ids[ok, j] = at[ok]
            left[torch.arange(T, device=DEV)[ok], at[ok]] = -math.inf
        live = ids >= 0
        val = torch.where(live, p.gather(1, ids.clamp(min=0)), torch.zeros(T, k, dtype=p.dtype, device=DEV))
        den = val.sum(1, keepdim=True) if c["normalize"] == "topk" else p.sum(1, keepdim=True)
        gates = torch.where(live, val / den, torch.zeros_like(val))
        slots = torch.full((T, k), -1, dtype=torch.int32, device=DEV)
        rows = torch.full((T * k,), -1, dtype=torch.int32, device=DEV)
        off = torch.zeros(E + 1, dtype=torch.int32, device=DEV)
        at = 0
        for e in range(E):
            off[e] = at
            tj = (ids == e).nonzero()
            n = tj.shape[0]
            slots[tj[:, 0], tj[:, 1]] = torch.arange(at, at + n, dtype=torch.int32, device=DEV)
            rows[at:at + n] = tj[:, 0].to(torch.int32)
            at += n
        off[E] = at
        return gates, ids.to(torch.int32), off, rows, slots
    if op == "route_bwd":
        x, ids = st["logits"].double(), st["route"][1].long()
        hot = torch.zeros_like(x, dtype=torch.bool)
        dg = torch.zeros_like(x)
        for j in range(c["k"]):
            t = (ids[:, j] >= 0).nonzero()[:, 0]
            hot[t, ids[t, j]] = True
            dg[t, ids[t, j]] = st["dgates"][t, j].double()
        p = torch.exp(x)
        if c["normalize"] == "topk":
            p = p * hot
        den = p.sum(1, keepdim=True)
        p = torch.where(den > 0, p / torch.where(den > 0, den, torch.ones_like(den)), torch.zeros_like(p))
        return p * (dg - (p * dg).sum(1, keepdim=True))
    if op in ("linear", "dgrad", "wgrad"):
        rows = st["rows"].long() if c.get("gather") else torch.arange(sum(st["sizes"]), device=DEV)
        w = st.get("w")
        parts, at = [], 0
        dw, db = [], []
        for e, n in enumerate(st["sizes"]):
            sel = slice(at, at + n)
            at += n
            if op == "linear":
                z = torch.matmul(st["x"].double()[rows[sel]], w[e].double().transpose(0, 1))
                if c["bias"]:
                    z += st["bias"][e].double()
                parts.append(z.clamp(min=0) if c["relu"] else z)
            elif op == "dgrad":
                z = torch.matmul(st["dz"][sel].double(), w[e].double())
                parts.append(torch.where(st["mask"][sel] > 0, z, torch.zeros_like(z)) if c["mask"] else z)
            else:
                d = st["dz"][sel].double()
                dw.append(torch.matmul(d.transpose(0, 1).contiguous(), st["x"].double()[rows[sel]]))
                db.append(d.sum(0))
        if op == "wgrad":
            return torch.stack(dw), torch.stack(db)
        return torch.cat(parts)
    if op == "combine":
        gates, slots = st["route"][0].double(), st["route"][4].long()
        rowsum = st["y"].double()[slots]  # every slot of these plans is used
        return (rowsum * gates[:, :, None]).sum(1) if c["weighted"] else rowsum.sum(1)
    if op == "combine_bwd":
        gates, rows, slots = st["route"][0].double(), st["route"][3].long(), st["route"][4].long()
        gate_of = torch.empty(rows.shape[0], dtype=torch.float64, device=DEV)
        gate_of[slots.reshape(-1)] = gates.reshape(-1)
        d = st["dout"].double()
        dots = (d[rows] * st["y"].double()).sum(1)
        return d[rows] * gate_of[:, None], dots[slots]
    norm = math.sqrt(math.fsum(float(t.double().pow(2).sum()) for t in st["grads"]))
    f = min(1.0, st["max_norm"] / (norm + 1e-6))
    return torch.tensor(norm, dtype=torch.float64, device=DEV), [t.double() * f for t in st["grads"]]
