"""Optimiser steps on matrices: orthogonalisation of updates by Newton-Schulz products (gmc_orthogonalise) and the Muon
update around it (gmc_muon_update), for Net.matrix_parameters() and any other parameters that are matrices. In a data-parallel
run the step follows gmc.sharding.all_reduce_gradients: every rank then computes the same update."""
import math
import typing

import torch
from torch import Tensor

from gmc import _native

COEFFICIENTS = (3.4445, -4.7750, 2.0315)
MAX_SIDE, MAX_SHORT_SIDE = 32768, 16384


def _coefficients(coefficients):
    if len(coefficients) != 3:
        raise _native.GmcError("coefficients are three numbers (a, b, c)")
    return [float(v) for v in coefficients]


def _check_sides(rows: int, cols: int) -> None:
    if max(rows, cols) > MAX_SIDE or min(rows, cols) > MAX_SHORT_SIDE:
        raise _native.GmcError(f"matrices may be up to {MAX_SIDE} x {MAX_SHORT_SIDE}, got {rows} x {cols}")


def _workspace(packed: bytes, n: int, device: torch.device):
    """Device scratch for one call, aligned to 1024 bytes: (tensor that holds it, address, bytes)."""
    size = _native.lib.gmc_orthogonalise_workspace_bytes(packed, n)
    if size == 0:
        return None, None, 0
    hold = torch.empty(size + 1024, dtype=torch.uint8, device=device)
    return hold, (hold.data_ptr() + 1023) // 1024 * 1024, size


def orthogonalise(updates: typing.Union[Tensor, typing.Sequence[Tensor]], steps: int = 5,
                  coefficients: typing.Sequence[float] = COEFFICIENTS, epsilon: float = 1e-7):
    """The Newton-Schulz iterate of each matrix of `updates` ([..., rows, cols], or a list of such tensors of one type and
    device; float32, bfloat16 or float16, CUDA): X = U / (|U| + epsilon), then `steps` times X <- a X + (b A + c A A) X with
    A = X X^T. Its singular values are near 1 whatever those of U were. Returns new tensors of the same shapes and type, with
    the error of a 32-bit evaluation for float32 and of the rounding for 16-bit types; not differentiable. A zero matrix gives
    zero, one with NaN or infinity gives NaN. Matrices may be up to 32768 x 16384."""
    single = isinstance(updates, Tensor)
    tensors = [updates] if single else list(updates)
    a, b, c = _coefficients(coefficients)
    outs, entries, held = [], [], []
    for t in tensors:
        code = _native.dtype_code(t, "updates")
        if t.dim() < 2:
            raise _native.GmcError(f"updates must be matrices [..., rows, cols], got {tuple(t.shape)}")
        if t.dtype != tensors[0].dtype or t.device != tensors[0].device:
            raise _native.GmcError("updates of one call must have one type and device")
        rows, cols = t.shape[-2:]
        _check_sides(rows, cols)
        t = t.detach()
        if t.dim() > 2 and not t.is_contiguous() or t.stride(-1) != 1 and cols > 1 or rows > 1 and t.stride(-2) < cols:
            t = t.contiguous()
            held.append(t)
        out = torch.empty(t.shape, dtype=t.dtype, device=t.device)
        outs.append(out)
        if t.numel() == 0:
            continue
        stride = max(t.stride(-2), cols) if t.dim() == 2 else cols
        size = t.element_size()
        source, target = t.data_ptr(), out.data_ptr()
        for i in range(t.numel() // (rows * cols)):
            step = i * rows * cols * size
            entries.append(_native.matrix_struct.pack(source + step, 0, target + step, rows, cols, stride, cols, 0.0))
    if entries:
        packed = b"".join(entries)
        with torch.cuda.device_of(tensors[0]):
            hold, address, size = _workspace(packed, len(entries), tensors[0].device)
            _native.check(_native.lib.gmc_orthogonalise(packed, len(entries), code, int(steps), a, b, c, float(epsilon), address,
                                                        size, _native.stream_of(tensors[0])), "orthogonalisation")
    return outs[0] if single else outs


def muon_update(params: typing.Sequence[Tensor], grads: typing.Sequence[Tensor], momenta: typing.Sequence[Tensor], lr: float,
                momentum: float = 0.95, weight_decay: float = 0.0, nesterov: bool = True, steps: int = 5,
                coefficients: typing.Sequence[float] = COEFFICIENTS, epsilon: float = 1e-7) -> None:
    """One Muon step on every parameter, in place, in a fixed number of kernels for up to 48 matrices:

        m <- momentum m + (1 - momentum) g;   u = (1 - momentum) g + momentum m  (nesterov)  or  m
        p <- (1 - lr weight_decay) p - lr sqrt(max(1, rows / cols)) orthogonalise(u)

    Parameters and gradients share one type (float32, bfloat16 or float16); momenta are float32, shaped like the parameters.
    A parameter with more than two axes counts as the matrix [shape[0], everything else]. Parameters and momenta must be
    contiguous and may not appear twice; no gradient may share their memory."""
    if not len(params) == len(grads) == len(momenta):
        raise _native.GmcError("params, grads and momenta must have one entry per parameter")
    if not params:
        return
    if not (math.isfinite(lr) and math.isfinite(weight_decay)):
        raise _native.GmcError("lr and weight_decay must be finite")
    a, b, c = _coefficients(coefficients)
    first = params[0]
    code = _native.dtype_code(first, "params")
    entries, held, seen, read = [], [], set(), set()
    for p, g, m in zip(params, grads, momenta):
        if p.dtype != first.dtype or g.dtype != first.dtype or p.device != first.device or g.device != first.device:
            raise _native.GmcError("parameters and gradients of one call must have one type and device")
        if p.dim() < 2 or p.numel() == 0 or not p.is_contiguous():
            raise _native.GmcError(f"parameters must be contiguous, not empty and have two or more axes, got {tuple(p.shape)}")
        if g.shape != p.shape or g.layout != torch.strided:
            raise _native.GmcError(f"a gradient must be dense and shaped like its parameter, got {tuple(g.shape)}")
        if m.shape != p.shape or m.dtype != torch.float32 or m.device != p.device or not m.is_contiguous():
            raise _native.GmcError("momenta must be contiguous float32, shaped like their parameters and on their device")
        if p.data_ptr() in seen or m.data_ptr() in seen or p.data_ptr() == m.data_ptr():
            raise _native.GmcError("a parameter or momentum appears twice")
        seen.update((p.data_ptr(), m.data_ptr()))
        if not g.is_contiguous():
            g = g.contiguous()
            held.append(g)
        read.add(g.data_ptr())
        rows = p.shape[0]
        cols = p.numel() // rows
        _check_sides(rows, cols)
        entries.append(_native.matrix_struct.pack(g.data_ptr(), m.data_ptr(), p.data_ptr(), rows, cols, cols, cols,
                                                  lr * math.sqrt(max(1.0, rows / cols))))
    if read & seen:
        raise _native.GmcError("a gradient must not share its memory with a parameter or momentum")
    packed = b"".join(entries)
    with torch.cuda.device_of(first):
        hold, address, size = _workspace(packed, len(entries), first.device)
        _native.check(_native.lib.gmc_muon_update(packed, len(entries), code, int(steps), a, b, c, float(epsilon), float(momentum),
                                                  int(nesterov), 1.0 - lr * weight_decay, address, size, _native.stream_of(first)),
                      "Muon update")
    # written behind autograd's back: whoever keeps something by a tensor's version has to see the change
    torch.autograd.graph.increment_version([*params, *momenta])


class Muon(torch.optim.Optimizer):
    """Muon for parameters with two or more axes (muon_update per type and device). The momentum is kept in float32."""

    def __init__(self, params, lr: float = 0.02, momentum: float = 0.95, weight_decay: float = 0.0, nesterov: bool = True,
                 steps: int = 5, coefficients: typing.Sequence[float] = COEFFICIENTS, epsilon: float = 1e-7):
        super().__init__(params, dict(lr=lr, momentum=momentum, weight_decay=weight_decay, nesterov=nesterov, steps=steps,
                                      coefficients=tuple(_coefficients(coefficients)), epsilon=epsilon))

    def add_param_group(self, param_group):
        super().add_param_group(param_group)
        for p in self.param_groups[-1]["params"]:
            if p.dim() < 2:
                self.param_groups.pop()
                raise _native.GmcError(f"Muon takes parameters with two or more axes, got {tuple(p.shape)}")

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            parts: typing.Dict[tuple, tuple] = {}
            for p in group["params"]:
                if p.grad is None:
                    continue
                state = self.state[p]
                if "momentum_buffer" not in state:
                    state["momentum_buffer"] = torch.zeros(p.shape, dtype=torch.float32, device=p.device)
                part = parts.setdefault((p.dtype, p.device), ([], [], []))
                for to, t in zip(part, (p, p.grad, state["momentum_buffer"])):
                    to.append(t)
            for part in parts.values():
                muon_update(*part, **{k: group[k] for k in ("lr", "momentum", "weight_decay", "nesterov", "steps", "coefficients",
                                                            "epsilon")})
        return loss

    def load_state_dict(self, state_dict):
        super().load_state_dict(state_dict)
        # the base class converts states to the parameter's type; the momentum stays in 32 bits
        for group, saved in zip(self.param_groups, state_dict["param_groups"]):
            for p, key in zip(group["params"], saved["params"]):
                buffer = state_dict["state"].get(key, {}).get("momentum_buffer")
                if buffer is not None:
                    self.state[p]["momentum_buffer"] = buffer.detach().to(device=p.device, dtype=torch.float32, copy=True).contiguous()
