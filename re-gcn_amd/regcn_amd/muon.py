"""The Muon optimiser on HIP: momentum whose two-dimensional updates are orthogonalised.

`orthogonalize` runs the Newton-Schulz iteration

    X = G / (|G|_F + eps);   A = X X^T,  X = a X + (b A + c A A) X,   `steps` times,

on a matrix's shorter side, for any number of matrices of any shapes in one set of launches
(regcn_orthogonalize): the products of operands split into fp16 halves run on the matrix cores.  With the
default coefficients the singular values end near 1 (0.7 to 1.2), the singular vectors stay.  Coefficients and the
step's scale are those published with the optimiser (K. Jordan and others, "Muon: An optimizer for hidden layers in neural
networks", 2024).
"""
import functools

import torch

from . import _lib

COEFFS = (3.4445, -4.7750, 2.0315)
_LIMIT, _LIMIT_B = 2.0, 16.0
SPLIT_STEPS = 8  # most steps of operands in halves


@functools.lru_cache(maxsize=64)
def _check_coeffs(a, b, c, steps):
    """The operands are held in halves of fp16: the iteration of a singular value from [0, 1] has to stay
    small.  A grid of 2049 starts, finer than the polynomial turns."""
    s = torch.linspace(0, 1, 2049, dtype=torch.float64)
    for _ in range(steps):
        poly = b * s ** 2 + c * s ** 4
        s = a * s + s * poly
        if not bool((s.abs() <= _LIMIT).all() and (poly.abs() <= _LIMIT_B).all()):  # NaN and infinities too
            raise ValueError("coefficients %r leave |s| <= %g or |b s^2 + c s^4| <= %g within %d steps"
                             % ((a, b, c), _LIMIT, _LIMIT_B, steps))


def _plan(g):
    """(contiguous tensor, whether the result is its transpose) of a matrix: a transposed view is taken as
    the matrix it views (the iteration commutes with transposition)."""
    if g.dim() != 2:
        raise ValueError("a matrix has two dimensions (got %s)" % (tuple(g.shape),))
    if g.dtype not in _lib.DTYPES:
        raise TypeError("matrices are float32, bfloat16 or float16 (got %s)" % g.dtype)
    if not g.is_cuda:
        raise ValueError("matrices must live on a HIP device (got %s); the HIP path has no CPU fallback" % g.device)
    g = g.detach()
    if g.is_contiguous():
        return g, False
    t = g.t()
    return (t, True) if t.is_contiguous() else (g.contiguous(), False)


def orthogonalize(g, steps=5, coeffs=COEFFS, eps=1e-7, full_fp32=False):
    """Newton-Schulz orthogonalisation of a matrix (m x n), of a stack of them (... x m x n), or of a list
    or tuple of matrices of any shapes and types on one device; the same structure is returned, each result
    in its matrix's type.  An all-zero matrix stays zero (with an eps of 0 it becomes NaN), a matrix without elements is returned as it is;
    infinities and NaN make their matrix's result NaN.  No gradient flows through the iteration.

    Matrices of more than 64 rows and columns are iterated on operands of 22 bits (two fp16 halves) that keep nothing
    below 2^-37 of the matrix's norm: the error is that of fp32 in the norm of the whole, but rows 1e-4, 1e-5, 1e-6 of the
    others are off by 4e-6, 4e-5, 4e-4 of themselves.  `full_fp32` keeps fp32 operands, on the fp32 matrix
    instructions (1.2 to 2.8 times the time: 8 steps of 200 x 200 214 us for 164, of 4096 x 4096 16.9 ms for 6.0); more than 8
    steps always do, since small rows have grown to the others' size by then."""
    steps = int(steps)
    if not 1 <= steps <= 1000:
        raise ValueError("1 to 1000 steps (got %d)" % steps)
    a, b, c = (float(v) for v in coeffs)
    _check_coeffs(a, b, c, steps)
    eps = float(eps)
    if not 0.0 <= eps < float("inf"):
        raise ValueError("eps must be a number >= 0 (got %r)" % eps)
    if isinstance(g, torch.Tensor):
        if g.dim() == 2:
            return _run([g], steps, a, b, c, eps, full_fp32)[0]
        if g.dim() < 2:
            raise ValueError("a matrix has two dimensions (got %s)" % (tuple(g.shape),))
        m, n = g.shape[-2:]
        if g.numel() == 0:
            return g.detach().clone()
        out = _run(list(g.detach().reshape(-1, m, n).unbind(0)), steps, a, b, c, eps, full_fp32)
        return torch.stack(out).reshape(g.shape)
    if not isinstance(g, (list, tuple)) or not all(isinstance(x, torch.Tensor) for x in g):
        raise TypeError("orthogonalize takes a tensor or a list of matrices (got %s)" % type(g).__name__)
    out = _run(g, steps, a, b, c, eps, full_fp32)
    return out if isinstance(g, list) else tuple(out)


def _run(mats, steps, a, b, c, eps, full_fp32):
    plans = [_plan(g) for g in mats]
    if not plans:
        return []
    device = plans[0][0].device
    if any(p.device != device for p, _ in plans):
        raise ValueError("the matrices must live on one device")
    outs = [torch.empty_like(p) for p, _ in plans]
    live = [k for k, (p, _) in enumerate(plans) if p.numel()]
    if live:
        desc = (_lib.Matrix * len(live))()
        flags = _lib.FULL_FP32 if full_fp32 or steps > SPLIT_STEPS else 0
        for d, k in zip(desc, live):
            p = plans[k][0]
            d.x, d.out, d.rows, d.cols, d.dtype = p.data_ptr(), outs[k].data_ptr(), p.shape[0], p.shape[1], \
                _lib.DTYPES[p.dtype] | flags
        size = _lib.lib().regcn_orthogonalize_workspace_bytes(desc, len(live))
        ws = torch.empty(size, device=device, dtype=torch.uint8)
        _lib.launch("regcn_orthogonalize", device, desc, len(live), steps, a, b, c, eps, ws.data_ptr(), size)
    return [o.t() if t else o for o, (_, t) in zip(outs, plans)]


class Muon(torch.optim.Optimizer):
    """Momentum with orthogonalised updates for two-dimensional parameters:

        buf = momentum * buf + grad
        d = grad + momentum * buf          (nesterov; otherwise buf)
        p = (1 - lr * weight_decay) * p - lr * sqrt(max(1, rows / cols)) * orthogonalize(d)

    One call of `orthogonalize` serves all the parameters of a group (per device; `full_fp32` as there).  The momentum and the step
    are fp32 whatever the parameter's type: a 16-bit parameter is rounded once, at the end.  Parameters without a
    gradient are left alone; sparse gradients are refused.  The step holds no host synchronisation, so a
    training step with it can be captured in a HIP graph (training.GraphedSteps) once each parameter has taken a step: a
    momentum buffer made within a capture would be cleared by every replay, and is refused.  A capture keeps the
    settings (lr and the others) that it was made with."""

    def __init__(self, params, lr=0.02, momentum=0.95, nesterov=True, weight_decay=0.0, steps=5, coeffs=COEFFS,
                 eps=1e-7, full_fp32=False):
        if not lr >= 0.0:
            raise ValueError("lr must be >= 0 (got %r)" % (lr,))
        if not 0.0 <= momentum < 1.0:
            raise ValueError("momentum must be in [0, 1) (got %r)" % (momentum,))
        if not weight_decay >= 0.0:
            raise ValueError("weight_decay must be >= 0 (got %r)" % (weight_decay,))
        if not 1 <= int(steps) <= 1000:
            raise ValueError("1 to 1000 steps (got %r)" % (steps,))
        _check_coeffs(*(float(v) for v in coeffs), int(steps))
        super().__init__(params, dict(lr=lr, momentum=momentum, nesterov=nesterov, weight_decay=weight_decay,
                                      steps=steps, coeffs=tuple(coeffs), eps=eps, full_fp32=bool(full_fp32)))

    def add_param_group(self, param_group):
        super().add_param_group(param_group)
        for p in self.param_groups[-1]["params"]:
            if p.dim() != 2 or p.dtype not in _lib.DTYPES:
                self.param_groups.pop()
                raise ValueError("Muon takes two-dimensional fp32, bf16 or fp16 parameters (got %s %s)"
                                 % (tuple(p.shape), p.dtype))

    def load_state_dict(self, state_dict):
        super().load_state_dict(state_dict)
        # the base class casts a state to its parameter's type; the momentum stays fp32
        keys = [k for g in state_dict["param_groups"] for k in g["params"]]
        for k, p in zip(keys, (p for g in self.param_groups for p in g["params"])):
            if "momentum_buffer" in state_dict["state"].get(k, {}):
                self.state[p]["momentum_buffer"] = state_dict["state"][k]["momentum_buffer"].to(
                    device=p.device, dtype=torch.float32, copy=True)

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            by_device = {}
            for p in group["params"]:
                if p.grad is not None:
                    if p.grad.is_sparse:
                        raise RuntimeError("Muon does not take sparse gradients")
                    by_device.setdefault(p.device, []).append(p)
            for ps in by_device.values():
                self._update(ps, group)
        return loss

    def _update(self, ps, group):
        grads, bufs = [p.grad for p in ps], []
        for p in ps:
            st = self.state[p]
            if "momentum_buffer" not in st:
                if p.is_cuda and torch.cuda.is_current_stream_capturing():
                    raise RuntimeError("a parameter's first Muon step cannot be captured: run one before the capture")
                st["momentum_buffer"] = torch.zeros_like(p, dtype=torch.float32)
            bufs.append(st["momentum_buffer"])
        mu, lr = group["momentum"], group["lr"]
        torch._foreach_mul_(bufs, mu)
        torch._foreach_add_(bufs, grads)
        d = bufs
        if group["nesterov"]:
            d = torch._foreach_mul(bufs, mu)
            torch._foreach_add_(d, grads)
        o = orthogonalize(d, group["steps"], group["coeffs"], group["eps"], group.get("full_fp32", False))
        torch._foreach_mul_(o, [max(1.0, p.shape[0] / p.shape[1]) ** 0.5 if p.numel() else 1.0 for p in ps])
        w = [p if p.dtype == torch.float32 else p.float() for p in ps]
        if group["weight_decay"]:
            torch._foreach_mul_(w, 1.0 - lr * group["weight_decay"])
        torch._foreach_add_(w, o, alpha=-lr)
        for p, x in zip(ps, w):
            if x is not p:
                p.copy_(x)


TABLES = ("dynamic_emb", "emb_rel")  # rows looked up by id: not matrices of a product


def split_parameters(model):
    """(parameters for Muon, the others) of a model: its matrices of at least two rows and columns, but not
    the entity and relation tables."""
    mats, rest = [], []
    for name, p in model.named_parameters():
        if not p.requires_grad:
            continue
        table = name.rsplit(".", 1)[-1] in TABLES
        (mats if p.dim() == 2 and min(p.shape) > 1 and not table else rest).append(p)
    return mats, rest
