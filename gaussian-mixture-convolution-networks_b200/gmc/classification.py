"""What a classifier answers and is trained on: log-probabilities of given classes with the entropy of the distribution and
its likeliest classes, in one pass over the logits, differentiable (gmc_log_probabilities_forward / _backward)."""
import typing

import torch
from torch import Tensor
from torch.autograd import forward_ad

from gmc import _native

MAX_TOP = 32
MIN_TEMPERATURE, MAX_TEMPERATURE = 1e-6, 1e6


class LogProbabilities(typing.NamedTuple):
    """Per row of logits; None for what was not asked for. All fp32, top_indices int64."""
    target: typing.Optional[Tensor]          # log-probability of the row's target class; 0 where it is ignored
    entropy: Tensor                          # in nats
    top: typing.Optional[Tensor]             # [..., n_top] log-probabilities of the likeliest classes, descending
    top_indices: typing.Optional[Tensor]     # [..., n_top] these classes; equal logits by the lower class


def _forward(logits: Tensor, code: int, targets: typing.Optional[Tensor], n_top: int, temperature: float, ignore_index: int,
             keep_stats: bool):
    n, c = logits.shape
    device, f32 = logits.device, torch.float32
    target = torch.empty(n, dtype=f32, device=device) if targets is not None else None
    entropy = torch.empty(n, dtype=f32, device=device)
    stats = torch.empty((n, 2), dtype=f32, device=device) if keep_stats else None
    top = torch.empty((n, n_top), dtype=f32, device=device) if n_top else None
    top_indices = torch.empty((n, n_top), dtype=torch.int64, device=device) if n_top else None
    with torch.cuda.device_of(logits):
        _native.check(_native.lib.gmc_log_probabilities_forward(
            logits.data_ptr(), code, _address(targets), n, c, logits.stride(0), temperature, ignore_index, n_top,
            _address(target), entropy.data_ptr(), _address(stats), _address(top), _address(top_indices),
            _native.stream_of(logits)), "log-probabilities")
    return target, entropy, top, top_indices, stats


def _address(t: typing.Optional[Tensor]) -> typing.Optional[int]:
    return None if t is None else t.data_ptr()


class _LogProbabilities(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, code, targets, n_top, temperature, ignore_index):
        ctx.set_materialize_grads(False)
        target, entropy, top, top_indices, stats = _forward(logits, code, targets, n_top, temperature, ignore_index, True)
        ctx.save_for_backward(logits, targets, entropy, top_indices, stats)
        ctx.config = (code, n_top, temperature, ignore_index)
        if top_indices is not None:
            ctx.mark_non_differentiable(top_indices)
        return target, entropy, top, top_indices

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_target, grad_entropy, grad_top, _):
        if grad_target is None and grad_entropy is None and grad_top is None:
            return None, None, None, None, None, None
        logits, targets, entropy, top_indices, stats = ctx.saved_tensors
        code, n_top, temperature, ignore_index = ctx.config
        grads = [None if g is None else g.contiguous() for g in (grad_target, grad_entropy, grad_top)]
        n, c = logits.shape
        grad_logits = torch.empty((n, c), dtype=logits.dtype, device=logits.device)
        with torch.cuda.device_of(logits):
            _native.check(_native.lib.gmc_log_probabilities_backward(
                logits.data_ptr(), code, _address(targets), _address(top_indices), stats.data_ptr(), entropy.data_ptr(),
                _address(grads[0]), _address(grads[1]), _address(grads[2]), grad_logits.data_ptr(), n, c, logits.stride(0),
                temperature, ignore_index, n_top, _native.stream_of(logits)), "gradient of log-probabilities")
        return grad_logits, None, None, None, None, None


def log_probabilities(logits: Tensor, targets: typing.Optional[Tensor] = None, n_top: int = 0, temperature: float = 1.0,
                      ignore_index: int = -100) -> LogProbabilities:
    """Log-probabilities of softmax(logits / temperature) for logits [..., n_classes] (float32, bfloat16 or float16, CUDA).

    `targets` (int64, logits.shape[:-1]) names one class per row; a row whose target is `ignore_index` gets 0 and no gradient
    from it, a target out of range gives NaN and the device check word's bit 8 (_native.sync_and_check raises). `n_top` (at
    most 32) asks for the likeliest classes. Masked classes hold -inf; a row with nothing else has log-probabilities -inf,
    entropy 0 and gradient 0. NaN and +inf in a row make its values and gradient NaN.

    target, entropy and top are differentiable once with respect to the logits, in reverse mode. Logits whose classes are not adjacent in
    memory are copied; rows may be any distance apart."""
    if not isinstance(logits, Tensor) or logits.dim() < 1 or logits.shape[-1] < 1:
        raise _native.GmcError("logits must be a tensor [..., n_classes] with at least one class")
    if forward_ad.unpack_dual(logits).tangent is not None:
        raise _native.GmcError("log_probabilities has no forward-mode derivative")
    code = _native.dtype_code(logits, "logits")
    c = logits.shape[-1]
    if not 0 <= n_top <= min(MAX_TOP, c):
        raise _native.GmcError(f"n_top must be between 0 and min({MAX_TOP}, n_classes = {c}), got {n_top}")
    if not MIN_TEMPERATURE <= temperature <= MAX_TEMPERATURE:
        raise _native.GmcError(f"temperature must be between {MIN_TEMPERATURE} and {MAX_TEMPERATURE}, got {temperature}")
    lead = logits.shape[:-1]
    if targets is not None:
        if targets.device != logits.device or targets.dtype != torch.int64 or targets.shape != lead:
            raise _native.GmcError(f"targets must be int64 {tuple(lead)} on {logits.device}, "
                                   f"got {targets.dtype} {tuple(targets.shape)} on {targets.device}")
        targets = targets.contiguous() if targets.dim() == 1 else targets.reshape(-1).contiguous()
    rows = logits if logits.dim() == 2 else logits.reshape(-1, c)
    if rows.stride(1) != 1 and c > 1:
        rows = rows.contiguous()
    n_top, temperature, ignore_index = int(n_top), float(temperature), int(ignore_index)
    if logits.requires_grad and torch.is_grad_enabled():
        target, entropy, top, top_indices = _LogProbabilities.apply(rows, code, targets, n_top, temperature, ignore_index)
    else:
        target, entropy, top, top_indices, _ = _forward(rows, code, targets, n_top, temperature, ignore_index, False)
    if logits.dim() != 2:
        target = None if target is None else target.view(lead)
        entropy = entropy.view(lead)
        if n_top:
            top, top_indices = top.view(*lead, n_top), top_indices.view(*lead, n_top)
    return LogProbabilities(target, entropy, top, top_indices)
