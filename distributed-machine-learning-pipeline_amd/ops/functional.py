"""Tensor-level ops: GPU tensors go to the hand-written HIP kernels (mandatory),
host tensors use the equivalent PyTorch reference math (for CPU-only tests and
the simulated device runtime).
"""
from __future__ import annotations

from typing import List, Optional, Sequence

import torch

from .native import require_native

SUM, PROD, MIN, MAX = 0, 1, 2, 3
OP_NAMES = {"sum": SUM, "prod": PROD, "min": MIN, "max": MAX}


def _op_id(op) -> int:
    if isinstance(op, str):
        return OP_NAMES[op.lower()]
    return int(op)


def reduce_ref(a: torch.Tensor, b: torch.Tensor, op) -> torch.Tensor:
    """Reference elementwise reduction. u8 wraps like the reference's byte
    arithmetic (gpu_coordinator_server.go:542)."""
    op = _op_id(op)
    if a.dtype in (torch.bfloat16, torch.float16):
        af, bf = a.float(), b.float()
        out = _reduce_f(af, bf, op)
        return out.to(a.dtype)
    if a.dtype == torch.uint8:
        ai, bi = a.to(torch.int32), b.to(torch.int32)
        out = _reduce_f(ai, bi, op)
        return (out & 0xFF).to(torch.uint8)
    return _reduce_f(a, b, op)


def _reduce_f(a, b, op):
    if op == SUM:
        return a + b
    if op == PROD:
        return a * b
    if op == MIN:
        return torch.minimum(a, b)
    if op == MAX:
        return torch.maximum(a, b)
    raise ValueError(f"bad reduce op {op}")


def reduce_into(dst: torch.Tensor, a: torch.Tensor, b: torch.Tensor, op="sum") -> torch.Tensor:
    if dst.is_cuda:
        require_native().reduce_into(dst, a, b, _op_id(op))
    else:
        dst.copy_(reduce_ref(a, b, op))
    return dst


def reduce_(dst: torch.Tensor, src: torch.Tensor, op="sum") -> torch.Tensor:
    return reduce_into(dst, dst, src, op)


def sgd_update_(P: torch.Tensor, G: torch.Tensor, scale: float) -> torch.Tensor:
    if P.is_cuda:
        require_native().sgd_update_(P, G, float(scale))
    else:
        P.sub_(G, alpha=float(scale))
    return P


def sgd_momentum_(P, G, V, lr, momentum, weight_decay=0.0, gscale=1.0):
    if P.is_cuda:
        require_native().sgd_momentum_(P, G, V, float(lr), float(momentum), float(weight_decay),
                                       float(gscale))
    else:
        g = G * gscale + weight_decay * P
        V.mul_(momentum).add_(g)
        P.sub_(V, alpha=lr)
    return P


def u8_to_f32(src: torch.Tensor, scale: float = 1.0 / 255.0) -> torch.Tensor:
    """idx pixel bytes -> f32 * scale (client.go:307-310)."""
    dst = torch.empty(src.shape, dtype=torch.float32, device=src.device)
    if src.is_cuda:
        require_native().u8_to_f32(dst, src.contiguous(), float(scale))
    else:
        dst.copy_(src.float() * scale)
    return dst


def scale_(x: torch.Tensor, alpha: float) -> torch.Tensor:
    if x.is_cuda:
        require_native().scale_(x, float(alpha))
    else:
        x.mul_(alpha)
    return x


def check_unrecorded(*ts: Optional[torch.Tensor]) -> None:
    """Refuse operands that require a gradient where gradients are recorded: the
    kernels are not, and the gradient would be lost without a word."""
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in ts):
        raise RuntimeError("an operand requires a gradient, and autograd does not record this call: make it under "
                           "torch.no_grad(), with the explicit gradient calls, or detach the operand")


def _norm_ref(grads: Sequence[torch.Tensor]) -> torch.Tensor:
    return sum(g.double().square().sum() for g in grads).sqrt()


def _check_grads(grads: Sequence[torch.Tensor], out: Optional[Sequence[torch.Tensor]]) -> None:
    check_unrecorded(*grads, *(out or []))
    if not grads:
        raise RuntimeError("no gradients given")
    if grads[0].dtype not in (torch.float32, torch.bfloat16, torch.float16):
        raise RuntimeError("gradients must be float32, bfloat16 or float16")
    if any(g.dtype != grads[0].dtype for g in grads):
        raise RuntimeError("gradients must have one type")
    if any(not g.is_contiguous() for g in grads):
        raise RuntimeError("gradients must be contiguous")
    if out is not None:
        if len(out) != len(grads):
            raise RuntimeError("out must hold one tensor a gradient")
        if any(o.dtype != g.dtype for o, g in zip(out, grads)):
            raise RuntimeError("out must have the gradients' type")
        if any(not o.is_contiguous() or o.shape != g.shape for o, g in zip(out, grads)):
            raise RuntimeError("out must be contiguous and of the gradients' shapes")
    if any(t.is_cuda for t in list(grads) + list(out or [])):
        raise RuntimeError("gradients must be on one device")


def _check_written_once(grads: Sequence[torch.Tensor], out: Sequence[torch.Tensor]) -> None:
    """What is written must be written once, and not read as another gradient."""
    spans = []
    for g, o in zip(grads, out):
        size = g.numel() * g.element_size()
        if size:
            spans.append((o.data_ptr(), size, True))
            if o.data_ptr() != g.data_ptr():
                spans.append((g.data_ptr(), size, False))
    end_w = end_r = 0
    for lo, size, write in sorted(spans):
        if lo < end_w or (write and lo < end_r):
            raise RuntimeError("clipped gradients must not overlap")
        if write:
            end_w = max(end_w, lo + size)
        else:
            end_r = max(end_r, lo + size)


def grad_norm(grads: Sequence[torch.Tensor]) -> torch.Tensor:
    """``sqrt(sum g^2)`` over every element of every gradient (float32, bfloat16
    or float16, one type, contiguous), as a 0-dim float32 tensor on their device:
    nothing is copied to the host.  Squares are summed in float64.  Autograd does
    not record it: tensors that require a gradient are refused where gradients are
    recorded."""
    grads = list(grads)
    if grads and grads[0].is_cuda:
        return require_native().grad_norm(grads)
    _check_grads(grads, None)
    return _norm_ref(grads).float()


def clip_grad_norm_(grads: Sequence[torch.Tensor], max_norm: float, eps: float = 1e-6,
                    out: Optional[List[torch.Tensor]] = None) -> torch.Tensor:
    """Scale the gradients (tensors as ``grad_norm`` takes them, not the parameters)
    by ``min(1, max_norm / (norm + eps))`` and return their norm before that.  In
    place, or into the tensors of ``out`` (the gradients then stay as they are), of
    which none may lie over another one or over a gradient, its own in full
    excepted.  A norm that is not a number makes every gradient so too; an infinite
    one makes them 0 (not a number where they are infinite)."""
    grads = list(grads)
    if grads and grads[0].is_cuda:
        return require_native().grad_norm(grads, True, float(max_norm), float(eps), out)
    for value, name in ((max_norm, "max_norm"), (eps, "eps")):
        if not value >= 0:
            raise RuntimeError(f"{name} must not be negative, got {value}")
    _check_grads(grads, out)
    _check_written_once(grads, grads if out is None else out)
    norm = _norm_ref(grads)
    coef = torch.clamp(max_norm / (norm + eps), max=1.0)
    coef = torch.where(norm + eps == 0, torch.ones_like(coef), coef)  # nothing but zeros: not 0 / 0
    # below 2^-126 float32 drops bits of the factor: a product in float64 there
    fine = 0.0 < float(coef) < 2.0 ** -126
    for g, o in zip(grads, grads if out is None else out):
        o.copy_((g.double() * coef).float() if fine else g.float() * coef.float())
    return norm.float()
