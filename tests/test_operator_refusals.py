"""CPU: what the training-step operators refuse before any GPU work is issued."""
import ctypes

import pytest
import torch

NULL = ctypes.c_void_p(0)
ONE = ctypes.c_void_p(16)          # never dereferenced: argument checks come first


def test_log_probabilities_argument_checks():
    from gmc import _native
    f = _native.lib.gmc_log_probabilities_forward

    def forward(logits=ONE, dtype=0, targets=ONE, n=2, c=8, stride=8, t=1.0, top=0, target=ONE, entropy=ONE, tops=NULL, idx=NULL):
        return f(logits, dtype, targets, n, c, stride, t, -100, top, target, entropy, NULL, tops, idx, NULL)

    assert forward(c=0) == 1 and forward(n=-1) == 1 and forward(stride=-8) == 1 and forward(c=(1 << 30) + 1) == 1
    assert forward(n=(1 << 27) + 1) == 1
    assert forward(dtype=3) == 4 and forward(dtype=-1) == 4
    assert forward(t=0.0) == 4 and forward(t=-1.0) == 4 and forward(t=float("nan")) == 4 and forward(t=float("inf")) == 4
    assert forward(top=9) == 4 and forward(top=33, c=100) == 4 and forward(top=-1) == 4
    assert forward(logits=NULL) == 3 and forward(entropy=NULL) == 3
    assert forward(targets=NULL) == 3 and forward(target=NULL) == 3           # both or neither
    assert forward(top=3) == 3
    assert forward(n=0, logits=NULL) == 0
    b = _native.lib.gmc_log_probabilities_backward

    def backward(logits=ONE, dtype=0, targets=ONE, idx=NULL, stats=ONE, gt=NULL, gk=NULL, out=ONE, n=2, c=8, top=0):
        return b(logits, dtype, targets, idx, stats, ONE, gt, NULL, gk, out, n, c, 8, 1.0, -100, top, NULL)

    assert backward(c=0) == 1 and backward(dtype=7) == 4 and backward(top=9) == 4
    assert backward(logits=NULL) == 3 and backward(stats=NULL) == 3 and backward(out=NULL) == 3
    assert backward(targets=NULL, gt=ONE) == 3
    assert backward(gk=ONE, idx=ONE, top=0) == 3 and backward(gk=ONE, top=2) == 3
    assert backward(n=0, logits=NULL) == 0


def test_log_probabilities_refuses_what_it_cannot_do():
    from gmc._native import GmcError
    from gmc.classification import log_probabilities
    with pytest.raises(GmcError, match="no CPU implementation"):
        log_probabilities(torch.zeros(2, 3))
    with pytest.raises(GmcError, match="at least one class"):
        log_probabilities(torch.zeros(2, 0))
    with pytest.raises(GmcError, match="at least one class"):
        log_probabilities([1.0, 2.0])
