"""GPU: log-probabilities of given classes, entropy, top alternatives and their gradient against a 64-bit restatement.

Error bounds, u = 2^-24 (half a step of fp32), C classes, x = z - max, y = x / T:
  * a term e^y carries the roundings of x, k = log2(e) / T (two) and x k, an exponent error of at most 4 u |y|, and the
    approximate exponential's 4 u; weighted by e / s the mean of |y| is at most log2 C (+ the entropy's own scale);
  * a thread adds at most C / 256 terms one after the other (long rows; 32 for short ones), 5 + 3 + 3 merges follow, each
    with a rescaling: C / 256 + 48 roundings in all;
so log s is off by at most u (4 log2 C + C / 256 + 52) =: u S, log p = y - log s by u (S + 4 |y|), and the entropy, whose
second sum has the factor |y| on each term, by u (1 + log2 C) 2 S. A gradient p (a + b (log p + H)) inherits the relative
error of p, u (S + 4 |y| + 4), on every one of its terms, and half a step of its own type."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def _scale(c):
    return 4 * math.log2(max(c, 2)) + c / 256 + 52


def _reference(z, targets, n_top, temperature, ignore_index, grads=None):
    """64 bits on the CPU, from the formulas; rows with nothing but -inf as documented."""
    z = z.detach().cpu().double()
    n, c = z.shape
    empty = (z == -math.inf).all(dim=1)
    safe = torch.where(empty.unsqueeze(1), torch.zeros_like(z), z)
    y = (safe - safe.max(dim=1, keepdim=True).values) / temperature
    log_s = y.exp().sum(dim=1, keepdim=True).log()
    log_p = y - log_s
    p = log_p.exp()
    entropy = -torch.where(p > 0, p * log_p, torch.zeros_like(p)).sum(dim=1)
    log_p[empty], p[empty], entropy[empty] = -math.inf, 0.0, 0.0
    t = targets.cpu()
    kept = t != ignore_index
    at = torch.where(kept, t, 0)
    target = torch.where(kept, log_p.gather(1, at.unsqueeze(1)).squeeze(1), 0.0)
    top_indices = torch.sort(z, dim=1, descending=True, stable=True).indices[:, :n_top]
    out = {"target": target, "entropy": entropy, "top": log_p.gather(1, top_indices), "top_indices": top_indices, "y": y}
    if grads is not None:
        g_t, g_h, g_k = (g.cpu().double() for g in grads)
        own = torch.zeros_like(z)
        g_t = torch.where(kept, g_t, 0.0)
        own.scatter_add_(1, at.unsqueeze(1), g_t.unsqueeze(1))
        own.scatter_add_(1, top_indices, g_k)
        total = (g_t + g_k.sum(dim=1)).unsqueeze(1)
        h = torch.where(p > 0, g_h.unsqueeze(1) * (log_p + entropy.unsqueeze(1)), 0.0)
        grad = (own - p * total - p * h) / temperature
        grad[empty] = 0.0
        each = ((g_t.abs() + g_k.abs().sum(dim=1)).unsqueeze(1)
                + g_h.abs().unsqueeze(1) * (log_p.clamp_min(-200).abs() + y.clamp_min(-200).abs() + entropy.unsqueeze(1)
                                            + log_s.abs())) / temperature
        # p below 2^-126 is flushed to 0: off by at most 2^-126 times what it is multiplied with
        out["grad"] = grad
        out["grad_tolerance"] = (U * (_scale(c) + 4 * y.clamp_min(-200).abs() + 8) * (own.abs() / temperature + p * each)
                                 + 2.0 ** -126 * each)
    return out


def _close(got, ref, tolerance, what):
    got = got.detach().cpu().double()
    ref = torch.where(ref.abs() > torch.finfo(torch.float32).max, ref.sign() * math.inf, ref)     # beyond the output's range
    assert torch.equal(torch.isfinite(got), torch.isfinite(ref)), what
    assert torch.equal(got[~torch.isfinite(ref)], ref[~torch.isfinite(ref)]), what
    off = (torch.where(torch.isfinite(ref), got - ref, 0.0).abs() - tolerance).max() if got.numel() else torch.tensor(-1.0)
    assert off <= 0, f"{what}: {off.item():.3e} beyond the bound"


def _check(logits, targets, n_top, temperature=1.0, ignore_index=-100, seed=0):
    """Forward without and with gradient, and the gradient, of logits [n, c] (any strides)."""
    from gmc.classification import log_probabilities
    n, c = logits.shape
    g = torch.Generator(device="cuda").manual_seed(seed)
    grads = [torch.randn(n, device="cuda", generator=g), torch.randn(n, device="cuda", generator=g),
             torch.randn(n, n_top, device="cuda", generator=g)]
    ref = _reference(logits, targets, n_top, temperature, ignore_index, grads)
    leaf = logits.detach().requires_grad_(True)
    results = [log_probabilities(logits.detach(), targets, n_top, temperature, ignore_index),
               log_probabilities(leaf, targets, n_top, temperature, ignore_index)]
    at = torch.where(targets == ignore_index, 0, targets).cpu().unsqueeze(1)
    y_t = ref["y"].gather(1, at).squeeze(1).clamp_min(-1e30).abs()
    s = _scale(c)
    for r in results:
        _close(r.target, ref["target"], U * (s + 4 * y_t), "target")
        _close(r.entropy, ref["entropy"], U * 2 * s * (1 + math.log2(max(c, 2))), "entropy")
        if n_top:
            assert torch.equal(r.top_indices.cpu(), ref["top_indices"])
            y_k = ref["y"].gather(1, ref["top_indices"]).clamp_min(-1e30).abs()
            _close(r.top, ref["top"], U * (s + 4 * y_k), "top")
        else:
            assert r.top is None and r.top_indices is None
    values = [results[1].target, results[1].entropy] + ([results[1].top] if n_top else [])
    (got,) = torch.autograd.grad(values, leaf, grads[:len(values)])
    assert got.dtype == logits.dtype and got.shape == logits.shape
    half = torch.finfo(logits.dtype).eps / 2
    _close(got, ref["grad"], ref["grad_tolerance"] + half * ref["grad"].abs() + torch.finfo(logits.dtype).tiny, "gradient")
    return results[1], got


def _logits(n, c, dtype, seed, spread=3.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    z = spread * torch.randn(n, c, device="cuda", generator=g)
    t = torch.randint(0, c, (n,), device="cuda", generator=g)
    if n > 2:
        t[n // 2] = -100
    return z.to(dtype), t


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,c,n_top", [(1, 1, 1), (1, 10, 5), (5, 32, 32), (3, 33, 0), (9, 40, 3), (4, 127, 20), (2, 1000, 32),
                                       (3, 1024, 8), (3, 1025, 8), (7, 2049, 1), (2, 5000, 32), (300, 4099, 4), (1, 50257, 20),
                                       (3, 131072, 32), (700, 1031, 0)])
def test_forward_and_gradient(dtype, n, c, n_top):
    z, t = _logits(n, c, dtype, 100 + n + c)
    _check(z, t, n_top)


@pytest.mark.parametrize("n,c,n_top,spread", [(5, 40, 3, 3.0), (3, 1024, 8, 3.0), (4, 4099, 4, 3.0), (2, 50257, 20, 3.0), (2, 131072, 32, 3.0),
                                              (3, 1500, 2, 0.1), (2, 70001, 0, 6.0)])
def test_small_gradients_of_fp16_logits(n, c, n_top, spread):
    """Most elements of a long row's gradient are subnormal fp16 numbers: their own rounding is half a step, 2^-25, whatever their
    size, beside half a step of the value above the smallest normal number."""
    from gmc.classification import log_probabilities
    z, t = _logits(n, c, torch.float16, 300 + c, spread)
    z.requires_grad_(True)
    g = torch.Generator(device="cuda").manual_seed(c)
    grads = [torch.randn(n, device="cuda", generator=g), torch.randn(n, device="cuda", generator=g),
             torch.randn(n, n_top, device="cuda", generator=g)]
    ref = _reference(z, t, n_top, 1.0, -100, grads)
    r = log_probabilities(z, t, n_top)
    values = [r.target, r.entropy] + ([r.top] if n_top else [])
    (got,) = torch.autograd.grad(values, z, grads[:len(values)])
    info = torch.finfo(torch.float16)
    own = torch.where(ref["grad"].abs() < info.smallest_normal, torch.full_like(ref["grad"], 2.0 ** -25), info.eps / 2 * ref["grad"].abs())
    # a value within the evaluation's error of the border between two steps may go either way: the rounding is of the computed value
    _close(got, ref["grad"], ref["grad_tolerance"] * (1 + info.eps) + own, "gradient")
    assert (got != 0).sum() >= (ref["grad"].abs() > 2.0 ** -24).sum()


@pytest.mark.parametrize("temperature", [1e-6, 0.05, 0.7, 3.0, 1e6])
@pytest.mark.parametrize("c", [17, 3001])
def test_temperatures(temperature, c):
    z, t = _logits(4, c, torch.float32, 7)
    _check(z, t, 4, temperature)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("c", [29, 900, 1500, 40001])
def test_masks(dtype, c):
    """Masked classes, by -inf and by the lowest value; rows with one class left and with none."""
    z, t = _logits(9, c, dtype, 21)
    z[0, c // 2:] = -math.inf
    z[1, : c // 2] = torch.finfo(dtype).min
    z[2] = -math.inf
    z[3] = -math.inf
    z[3, c - 1] = 1.5
    z[4] = torch.finfo(dtype).min                # all at the lowest value: a uniform distribution
    z[5, ::2] = -math.inf
    z[6] = torch.finfo(dtype).max
    z[7, 0] = torch.finfo(dtype).max
    z[7, 1:] = torch.finfo(dtype).min
    t[0], t[3], t[5] = 0, c - 1, 2                # t[3]: the one class that is left, t[5]: a masked target
    t[7] = 0
    _check(z, t, min(c, 16))


@pytest.mark.parametrize("others", [-3e38, -1e36, -2e35, -1e34, 0.0])
def test_logits_at_both_ends_of_the_range(others):
    """Two classes share a maximum of 3e38: probabilities 1/2 and 0 exactly (differences of 1e35 and more), so the entropy and the
    target's log-probability are ln 2 to the three roundings of a logarithm and its products."""
    from gmc.classification import log_probabilities
    z = torch.full((3, 5000), others, device="cuda")
    z[:, [7, 4001]] = 3e38
    z = z.bfloat16().requires_grad_(True)
    t = torch.full((3,), 4001, device="cuda")
    r = log_probabilities(z, t, n_top=2)
    ln2 = 0.6931471805599453
    for v in (r.entropy, -r.target, -r.top[:, 0], -r.top[:, 1]):
        assert (v.double() - ln2).abs().max() <= 4 * 2.0 ** -24
    assert (r.top_indices == torch.tensor([7, 4001], device="cuda")).all()
    (g,) = torch.autograd.grad(r.target.sum(), z)
    want = torch.zeros_like(g)
    want[:, 7], want[:, 4001] = -0.5, 0.5
    assert (g.double() - want.double()).abs().max() <= 2.0 ** -9


@pytest.mark.parametrize("temperature", [1.0, 2.0, 1e6])
@pytest.mark.parametrize("c", [6, 1024, 3001, 70000])
def test_logits_further_apart_than_the_range(c, temperature):
    """z - max is -6e38, beyond fp32, and log p, its quotient by T, need not be. The bound is u (S + 4 |y|) with the whole |y|, up to
    6.4e32 here: 1 / T, the two products by it and their difference are rounded once each."""
    from gmc.classification import log_probabilities
    g = torch.Generator(device="cuda").manual_seed(c)
    z = torch.randn(5, c, device="cuda", generator=g)
    z[:, 0] = 3e38
    z[1, 1:], z[2, 3], z[3, 1:], z[4, c - 1] = -3e38, -3e38, -math.inf, -3.4e38
    z[3, 4] = -3e38
    t, n_top = torch.tensor([1, c - 1, 3, 4, c - 1], device="cuda"), min(c, 5)
    z.requires_grad_(True)
    r = log_probabilities(z, t, n_top, temperature)
    (grad,) = torch.autograd.grad(r.target.sum() + r.entropy.sum(), z)
    ref = _reference(z, t, n_top, temperature, -100, [torch.ones(5), torch.ones(5), torch.zeros(5, n_top)])
    y_t, y_k = ref["y"].gather(1, t.cpu().unsqueeze(1)).squeeze(1).abs(), ref["y"].gather(1, ref["top_indices"]).abs()
    _close(r.target, ref["target"], U * (_scale(c) + 4 * y_t), "target")
    _close(r.top, ref["top"], U * (_scale(c) + 4 * y_k), "top")
    _close(r.entropy, ref["entropy"], U * 2 * _scale(c) * (1 + math.log2(c)), "entropy")
    _close(grad, ref["grad"], ref["grad_tolerance"] + U * ref["grad"].abs() + 2.0 ** -149, "gradient")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("temperature,scale", [(1e-6, 1e8), (1e-3, 1e14), (1.0, 1e30), (1e6, 1e30)])
@pytest.mark.parametrize("c", [20, 1024, 3001])
def test_large_incoming_gradients_of_the_entropy(c, temperature, scale, dtype):
    """A class of probability 0 gets no gradient, masked or not, however large the incoming one (a loss scale over a small
    temperature): here one class has all of the probability and its own gradient -p g (log p + H) / T is 0 as well."""
    from gmc.classification import log_probabilities
    z = torch.full((3, c), -math.inf, device="cuda", dtype=dtype)
    z[0, 1], z[1, 2], z[2, c - 1] = 1.0, 0.0, 60000.0
    if temperature <= 1.0:
        z[1, 5:] = -4000.0
        z[2, :4] = -30000.0
    z.requires_grad_(True)
    r = log_probabilities(z, temperature=temperature)
    (grad,) = torch.autograd.grad(r.entropy, z, torch.full_like(r.entropy, scale))
    assert (r.entropy == 0).all() and (grad == 0).all()


@pytest.mark.parametrize("c", [20, 1024, 1025, 70000])
def test_nan_and_infinity_make_the_row_nan(c):
    from gmc.classification import log_probabilities
    z, t = _logits(6, c, torch.float32, 5)
    z[1, c - 1] = math.nan
    z[2, 0] = math.inf
    z[3] = math.nan
    t[1:4] = 3
    leaf = z.clone().requires_grad_(True)
    r = log_probabilities(leaf, t, n_top=5)
    (r.target.sum() + r.entropy.sum() + r.top.sum()).backward()
    for i in (1, 2, 3):
        assert r.entropy[i].isnan() and r.target[i].isnan() and r.top[i].isnan().all() and leaf.grad[i].isnan().all()
    assert ((r.top_indices >= 0) & (r.top_indices < c)).all() and r.top_indices[3].tolist() == list(range(5))
    assert r.top_indices[2, 0] == 0
    order = torch.sort(torch.where(z[1].isnan(), -math.inf, z[1]), descending=True, stable=True).indices[:5]
    assert torch.equal(r.top_indices[1], order)
    rest = [0, 4, 5]
    assert torch.isfinite(leaf.grad[rest]).all() and torch.isfinite(r.entropy[rest]).all()


@pytest.mark.parametrize("c", [31, 32, 512, 1024, 1025, 4096, 30011])
def test_ties_go_to_the_lowest_class(c):
    """Equal rows, few distinct values, both zeros, and a row that rises and one that falls."""
    n_top = min(c, 32)
    z = torch.zeros(6, c, device="cuda")
    z[1] = torch.randint(0, 3, (c,), device="cuda", generator=torch.Generator(device="cuda").manual_seed(3)).float()
    z[2, ::2] = -0.0
    z[3] = torch.arange(c, device="cuda") * 0.01
    z[4] = -torch.arange(c, device="cuda") * 0.01
    z[5, -3:] = 1.0
    r, _ = _check(z, torch.zeros(6, dtype=torch.int64, device="cuda"), n_top)
    assert r.top_indices[0].tolist() == list(range(n_top)) and r.top_indices[2].tolist() == list(range(n_top))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("c", [100, 1030, 9001])
def test_strides_and_alignment(dtype, c):
    n = 5
    g = torch.Generator(device="cuda").manual_seed(9)
    t = torch.randint(0, c, (n,), device="cuda", generator=g)
    wide = torch.randn(n, 2 * c + 13, device="cuda", generator=g).to(dtype)
    for first in (0, 1, 3, 7, 8):
        _check(wide[:, first:first + c], t, 6)                                  # rows apart, each start aligned differently
    _check(torch.randn(c, n, device="cuda", generator=g).to(dtype).t(), t, 6)   # classes not adjacent
    _check(torch.randn(1, c, device="cuda", generator=g).to(dtype).expand(n, c), t, 6)   # one row for all
    _check(wide[::2, :c], t[::2].contiguous(), 6)


@pytest.mark.parametrize("n,c", [(36000, 65537), (2500000, 900)])
def test_offsets_beyond_32_bits(n, c):
    """More than 2^31 logits in both kernels: the first rows, those around the 2^31st element and the last ones, and their gradients."""
    from gmc.classification import log_probabilities
    some = torch.cat([torch.arange(3), 2 ** 31 // c + torch.arange(-2, 3), n - 1 - torch.arange(3)]).cuda()
    rows, t_some = _logits(len(some), c, torch.bfloat16, 3)
    z = torch.zeros(n, c, device="cuda", dtype=torch.bfloat16)
    z[some] = rows
    t = torch.zeros(n, dtype=torch.int64, device="cuda")
    t[some] = t_some
    z.requires_grad_(True)
    r = log_probabilities(z, t, n_top=2)
    one = torch.ones(n, device="cuda")
    (grad,) = torch.autograd.grad([r.target, r.entropy], z, [one, one])
    ref = _reference(rows, t_some, 2, 1.0, -100, [torch.ones(len(some)), torch.ones(len(some)), torch.zeros(len(some), 2)])
    y = ref["y"].gather(1, torch.where(t_some == -100, 0, t_some).cpu().unsqueeze(1)).squeeze(1).abs()
    _close(r.target[some], ref["target"], U * (_scale(c) + 4 * y), "target")
    _close(r.entropy[some], ref["entropy"], U * 2 * _scale(c) * (1 + math.log2(c)), "entropy")
    assert torch.equal(r.top_indices[some].cpu(), ref["top_indices"])
    _close(grad[some], ref["grad"], ref["grad_tolerance"] + 2.0 ** -8 * ref["grad"].abs() + torch.finfo(torch.float32).smallest_normal, "gradient")
    # all other rows are uniform: the target's gradient is 1 - 1 / c, the others' -1 / c, the entropy's 0
    others = torch.ones(n, dtype=torch.bool, device="cuda")
    others[some] = False
    u = U * (_scale(c) + 16)
    assert ((r.entropy - math.log(c)).abs()[others] <= 2 * u * (1 + math.log2(c))).all()
    assert ((grad[:, 0].float() - (1 - 1 / c)).abs()[others] <= 2.0 ** -8).all()
    assert ((grad[:, c - 1].float() * c + 1).abs()[others] <= 2.0 ** -8 + 64 * u).all()


def test_the_gradient_of_a_broadcast_row_is_summed():
    from gmc.classification import log_probabilities
    row = torch.randn(1, 2000, device="cuda", requires_grad=True)
    t = torch.randint(0, 2000, (8,), device="cuda")
    log_probabilities(row.expand(8, 2000), t).target.sum().backward()
    ref = row.detach().double().requires_grad_(True)
    torch.log_softmax(ref.expand(8, 2000), 1).gather(1, t.unsqueeze(1)).sum().backward()
    assert (row.grad.double() - ref.grad).abs().max() <= 8 * U * (_scale(2000) + 60)


def test_leading_dimensions_targets_and_empty_batches():
    from gmc.classification import log_probabilities
    z, t = _logits(6, 50, torch.float32, 1)
    flat = log_probabilities(z, t, n_top=3)
    shaped = log_probabilities(z.view(2, 3, 50), t.view(2, 3), n_top=3)
    assert shaped.target.shape == (2, 3) and shaped.top.shape == (2, 3, 3)
    for a, b in zip(flat, shaped):
        assert torch.equal(a, b.reshape(a.shape))
    one = log_probabilities(z[1], t[1], n_top=3)
    assert one.target.shape == () and torch.equal(one.target, flat.target[1]) and torch.equal(one.top, flat.top[1])
    free = log_probabilities(z, n_top=3)
    assert free.target is None and torch.equal(free.top, flat.top)
    none = log_probabilities(z[:0].requires_grad_(True), t[:0], n_top=3)
    assert none.target.shape == (0,) and none.top.shape == (0, 3)
    none.target.sum().backward()


def test_ignored_rows_and_partial_gradients():
    from gmc.classification import log_probabilities
    z, t = _logits(5, 3000, torch.float32, 2)
    t[:] = torch.tensor([0, 7, 0, 2999, 0])
    _check(z, t, 2, ignore_index=0)
    leaf = z.clone().requires_grad_(True)
    r = log_probabilities(leaf, t, n_top=2, ignore_index=0)
    assert (r.target[[0, 2, 4]] == 0).all()
    (only_target,) = torch.autograd.grad(r.target.sum(), leaf, retain_graph=True)
    assert (only_target[[0, 2, 4]] == 0).all() and (only_target[1] != 0).any()
    (only_entropy,) = torch.autograd.grad(r.entropy.sum(), leaf, retain_graph=True)
    (only_top,) = torch.autograd.grad(r.top.sum(), leaf, retain_graph=True)
    (together,) = torch.autograd.grad(r.target.sum() + r.entropy.sum() + r.top.sum(), leaf)
    # each gradient is at most 2 (1 + log2 C) per value; three of them and their sum are rounded once each
    assert (only_target + only_entropy + only_top - together).abs().max() <= 8 * U * 2 * (1 + math.log2(3000))


@pytest.mark.parametrize("c", [60, 6000])
def test_a_target_out_of_range_is_reported(c):
    from gmc import _native
    from gmc.classification import log_probabilities
    z, t = _logits(4, c, torch.float32, 3)
    t[:] = torch.tensor([1, c, -1, c - 1])
    leaf = z.clone().requires_grad_(True)
    r = log_probabilities(leaf, t)
    r.target.sum().backward()
    assert r.target.isnan().tolist() == [False, True, True, False]
    assert leaf.grad.isnan().any(dim=1).tolist() == [False, True, True, False] and leaf.grad[1].isnan().all()
    assert torch.isfinite(r.entropy).all()
    assert _native.device_check_word() == 8
    log_probabilities(z, t.clamp(0, c - 1))
    assert _native.device_check_word() == 0


def test_reports_of_several_kernels_are_read_and_cleared_together():
    from gmc import _native
    from gmc.classification import log_probabilities
    u = torch.randn(200, 300, device="cuda")
    packed = _native.matrix_struct.pack(u.data_ptr(), 0, u.data_ptr(), 200, 300, 300, 300, 0.0)
    size = _native.lib.gmc_orthogonalise_workspace_bytes(packed, 1)
    hold = torch.empty(size + 1024, dtype=torch.uint8, device="cuda")
    stream = _native.stream_of(u)
    assert _native.lib.gmc_sync_and_check(stream) == 0
    _native.check(_native.lib.gmc_debug_orthogonalise_lost_wait(packed, 1, 0, 5, 3.4445, -4.775, 2.0315, 1e-7,
                                                                (hold.data_ptr() + 1023) // 1024 * 1024, size, 0, stream), "")
    log_probabilities(torch.zeros(1, 4, device="cuda"), torch.tensor([4], device="cuda"))
    assert _native.device_check_word() == 1 | 8
    assert _native.device_check_word() == 0
    log_probabilities(torch.zeros(1, 4, device="cuda"), torch.tensor([-1], device="cuda"))
    assert _native.lib.gmc_sync_and_check(stream) == 7 and _native.lib.gmc_sync_and_check(stream) == 0


@pytest.mark.parametrize("c", [12, 2500])
def test_gradient_against_differences(c):
    """Central differences of the forward values along random directions: cut-off error h^2 / 6 |f'''| with |f'''| <= 12 |v|^3
    for log p and 40 (1 + log C) |v|^3 for the entropy in units of the largest |v|, rounding error 2 u S (1 + log2 C) / h.
    Where the step swaps an alternative i for another j, the slope of their sum has a kink of |v_i - v_j| <= 2 for each."""
    from gmc.classification import log_probabilities
    z, t = _logits(3, c, torch.float32, 31, spread=1.0)
    leaf = z.clone().requires_grad_(True)
    f = lambda q: (lambda r: r.target.double() + r.entropy.double() + r.top.double().sum(dim=1))(log_probabilities(q, t, n_top=2))  # noqa: E731
    (grad,) = torch.autograd.grad(f(leaf).sum(), leaf)
    for seed in range(4):
        v = torch.randn(3, c, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed)).sign()
        h = 2.0 ** -6
        up, down = z + h * v, z - h * v
        slope = (f(up) - f(down)) / (2 * h)
        along = (grad.double() * v.double()).sum(dim=1)
        bound = h * h / 6 * (3 * 12 + 40 * (1 + math.log(c))) + 4 * U * _scale(c) * (1 + math.log2(c)) / h
        a, b = (log_probabilities(q, n_top=2).top_indices.sort(dim=1).values for q in (up, down))
        assert ((slope - along).abs() <= bound + 2.0 * (a != b).sum(dim=1)).all()


def test_another_stream_and_two_calls_at_once():
    from gmc.classification import log_probabilities
    z, t = _logits(64, 20001, torch.bfloat16, 4)
    want = log_probabilities(z, t, n_top=8)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for s in streams:
        with torch.cuda.stream(s):
            got.append(log_probabilities(z, t, n_top=8))
    torch.cuda.synchronize()
    for r in got:
        for a, b in zip(want, r):
            assert torch.equal(a, b)


@pytest.mark.parametrize("n,c", [(4, 100), (3, 20001)])
def test_captured_and_replayed_with_its_gradient(n, c):
    from gmc.classification import log_probabilities
    inputs = [_logits(n, c, torch.float32, s) for s in (1, 2)]
    static_z, static_t = inputs[0][0].clone().requires_grad_(True), inputs[0][1].clone()

    def step():
        r = log_probabilities(static_z, static_t, n_top=4)
        (g,) = torch.autograd.grad(r.target.sum() + 0.5 * r.entropy.sum() + r.top.sum(), static_z)
        return [r.target, r.entropy, r.top, r.top_indices, g]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for z, t in inputs:
        with torch.no_grad():
            static_z.copy_(z)
            static_t.copy_(t)
        graph.replay()
        got = [o.clone() for o in out]
        for a, b in zip(got, step()):
            assert torch.equal(a, b)


def test_repeated_runs_are_identical():
    from gmc.classification import log_probabilities
    z, t = _logits(16, 77777, torch.bfloat16, 8)
    leaf = z.clone().requires_grad_(True)
    runs = []
    for _ in range(3):
        r = log_probabilities(leaf, t, n_top=16)
        runs.append([*r, *torch.autograd.grad(r.target.sum() + r.entropy.sum() + r.top.sum(), leaf)])
    for other in runs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(runs[0], other))


def test_network_answers_and_loss():
    """Net.log_probabilities against the network's own forward: the same distribution, loss and parameter gradients."""
    import gmc.model as model
    import synthetic_inputs as synthetic
    cfg = model.Config(n_dims=2)
    cfg.layers = [model.Layer(4, 1, 24, 12), model.Layer(10, 1, 16, 8)]
    cfg.mlp = [24, 10]
    torch.manual_seed(11)
    net = model.Net(config=cfg).cuda().train()
    x = synthetic.fit_target_2d(6, 1, 20, 5)
    x[..., 0] = x[..., 0].abs() + 0.1
    x, t = x.cuda(), torch.arange(6, device="cuda") % 10
    losses, state = [], {k: v.clone() for k, v in net.state_dict().items()}
    for which in range(2):
        net.load_state_dict(state)         # a training pass moves the running averages that the network divides by
        net.zero_grad()
        torch.manual_seed(2)
        if which:
            r = net.log_probabilities(x, t, n_top=5)
            loss = -r.target.mean()
            assert r.top_indices.shape == (6, 5) and (r.entropy > 0).all()
        else:
            loss = torch.nn.functional.nll_loss(net(x), t)
        loss.backward()
        losses.append((loss.detach(), [p.grad.clone() for p in net.mlp.parameters()]))
    assert (losses[0][0] - losses[1][0]).abs() <= 2 * U * (_scale(10) + 40)
    for a, b in zip(losses[0][1], losses[1][1]):
        # two fp32 computations of the same gradient through a batch norm over six rows
        assert (a - b).abs().max() <= 2.0 ** -10 * a.abs().max() + 2.0 ** -20
