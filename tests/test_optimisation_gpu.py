"""GPU: orthogonalisation by Newton-Schulz products and the Muon update against 64-bit restatements.

Error bound. The operands carry 22 bits where a 32-bit evaluation carries 24, and the polynomial amplifies either by the same
factors: the error (2-norm over the matrix) may be 2^2 times that of the plain 32-bit evaluation of the same formula on the
same input. The plain one can be exact by luck (equal elements round alike), so there is a floor, from the last step alone:
its terms a s, b s^3, c s^5 of a singular value s <= 1.21 add up to 4.2 + 8.5 + 5.3 = 18 in absolute value, each passes through
four roundings (norm of X, A, A A, B X), 72 x 2^-24, and the result is at least 0.68: 106 x 2^-24 of it, below 2^-17. Last, half a step of the
output's type on every value."""
import copy
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

COEFFICIENTS = (3.4445, -4.7750, 2.0315)
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def _plain(u, steps, coefficients, epsilon):
    a, b, c = coefficients
    tall = u.shape[-2] > u.shape[-1]
    x = u.mT if tall else u
    x = x / (x.square().sum(dim=(-1, -2), keepdim=True).sqrt() + epsilon)
    for _ in range(steps):
        g = x @ x.mT
        x = a * x + (b * g + c * (g @ g)) @ x
    return x.mT if tall else x


def _check(got, u, steps=5, coefficients=COEFFICIENTS, epsilon=1e-7):
    ref = _plain(u.double(), steps, coefficients, epsilon)
    plain = _plain(u.float(), steps, coefficients, epsilon).double()
    assert got.shape == u.shape and got.dtype == u.dtype
    norm = lambda t: torch.linalg.matrix_norm(t)  # noqa: E731
    half = torch.finfo(u.dtype).eps / 2 if u.dtype != torch.float32 else 0.0
    bound = 4 * norm(plain - ref) + (2.0 ** -17 + half) * norm(ref) + torch.finfo(u.dtype).tiny * math.sqrt(u.shape[-1] * u.shape[-2])
    off = norm(got.double() - ref)
    assert (off <= bound).all(), f"{(off / norm(ref)).max().item():.3e} against {(bound / norm(ref)).min().item():.3e}"


def _update(*shape, seed=0, dtype=torch.float32):
    """A few strong directions over noise, as gradients have them."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    *lead, m, n = shape
    rank = max(1, min(m, n, 12) // 2)
    strong = (torch.randn(*lead, m, rank, device="cuda", generator=g) * torch.exp(-0.5 * torch.arange(rank, device="cuda"))) \
        @ torch.randn(*lead, rank, n, device="cuda", generator=g)
    return (1e-3 * (strong + 0.3 * torch.randn(*shape, device="cuda", generator=g))).to(dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,n", [(1, 1), (1, 7), (9, 1), (5, 5), (16, 40), (64, 64), (64, 160), (65, 63), (127, 129), (128, 128),
                                 (129, 127), (130, 600), (257, 64), (64, 2000), (3000, 17), (300, 1000), (1000, 300), (513, 769),
                                 (1025, 1031)])
def test_orthogonalise(m, n, dtype):
    from gmc.optimisation import orthogonalise
    u = _update(m, n, seed=m * 7 + n, dtype=dtype)
    before = u.clone()
    _check(orthogonalise(u), u)
    assert torch.equal(u, before)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("m,n", [(8, 9000), (16, 513), (17, 300), (64, 4096), (64, 4097), (65, 1536), (128, 1536), (128, 1537), (2000, 100),
                                 (16, 32768), (32768, 3), (129, 5000), (256, 6000), (6000, 250), (1500, 4100)])
def test_where_one_kernel_ends_and_the_next_begins(m, n, dtype):
    """Both sides of the shapes that decide between fp32 tiles, one cluster, and the whole GPU; columns shared out; long axes."""
    from gmc.optimisation import orthogonalise
    u = _update(m, n, seed=m + n, dtype=dtype)
    _check(orthogonalise(u), u)


def test_a_long_inner_axis():
    """The sums of X X^T over 20000 columns, all of one sign on the diagonal."""
    from gmc.optimisation import orthogonalise
    u = _update(200, 20000, seed=5)
    _check(orthogonalise(u), u)


@pytest.mark.parametrize("m,n", [(1, 1), (16, 40), (64, 160), (64, 2000), (128, 1536), (129, 127), (200, 20000), (1025, 1031), (32768, 3),
                                 (300, 9000), (6000, 250)])
def test_fp16_results_down_to_the_smallest_numbers(m, n):
    """The file's bound with fp16's own absolute error: half a step where values are subnormal, 2^-25."""
    from gmc.optimisation import orthogonalise
    u = _update(m, n, seed=m + n, dtype=torch.float16)
    got = orthogonalise(u)
    ref, plain = _plain(u.double(), 5, COEFFICIENTS, 1e-7), _plain(u.float(), 5, COEFFICIENTS, 1e-7).double()
    norm = torch.linalg.matrix_norm
    bound = 4 * norm(plain - ref) + (2.0 ** -17 + torch.finfo(torch.float16).eps / 2) * norm(ref) \
        + torch.finfo(torch.float16).smallest_normal * 2.0 ** -11 * math.sqrt(m * n)
    assert norm(got.double() - ref) <= bound, f"{(norm(got.double() - ref) / norm(ref)).item():.3e} against {(bound / norm(ref)).item():.3e}"


@pytest.mark.parametrize("m,n", [(20, 3000), (100, 1000), (256, 6000), (1500, 4100), (4100, 1500), (2048, 2048)])
def test_updates_of_one_sign(m, n):
    """Updates behind a rectifier have one sign: the tensor core's sums then lose bits in one direction everywhere."""
    from gmc.optimisation import orthogonalise
    g = torch.Generator(device="cuda").manual_seed(m * n)
    for u in (0.1 + torch.rand(m, n, device="cuda", generator=g), torch.rand(m, n, device="cuda", generator=g).square(),
              -torch.rand(m, n, device="cuda", generator=g).relu() * (torch.rand(m, 1, device="cuda", generator=g) < 0.3)):
        _check(orthogonalise(u), u)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("signs", ["random", "one"])
@pytest.mark.parametrize("m,n", [(200, 20000), (1500, 4100), (2048, 2048), (2000, 30000), (4095, 6001)])
def test_16_bit_results_of_long_axes_before_their_rounding(m, n, signs, dtype):
    """The rounding's own error is known (that of the rounded 64-bit result); what the evaluation adds to it is independent of
    where a value lies between two 16-bit numbers, so that the squares add up, and may be what the bound above allows an
    fp32 result: four times the plain evaluation's error and 2^-17."""
    from gmc.optimisation import orthogonalise
    g = torch.Generator(device="cuda").manual_seed(m + n)
    u = torch.randn(m, n, device="cuda", generator=g) if signs == "random" else 0.1 + torch.rand(m, n, device="cuda", generator=g)
    u = u.to(dtype)
    got = orthogonalise(u).double()
    ref = _plain(u.double(), 5, COEFFICIENTS, 1e-7)
    norm = torch.linalg.matrix_norm
    bound = 4 * norm(_plain(u.float(), 5, COEFFICIENTS, 1e-7).double() - ref) + 2.0 ** -17 * norm(ref)
    added = (got - ref).square().sum() - (ref.to(dtype).double() - ref).square().sum()
    assert added.clamp_min(0).sqrt() <= bound, f"{(added.clamp_min(0).sqrt() / norm(ref)).item():.3e} against {(bound / norm(ref)).item():.3e}"


@pytest.mark.parametrize("m,n", [(20, 50), (200, 333)])
def test_inputs_at_the_edges(m, n):
    """Rank one, nearly rank one, one element, equal elements, very small and very large values, orthogonal rows."""
    from gmc.optimisation import orthogonalise
    g = torch.Generator(device="cuda").manual_seed(1)
    left, right = torch.randn(m, 1, device="cuda", generator=g), torch.randn(1, n, device="cuda", generator=g)
    one = torch.zeros(m, n, device="cuda")
    one[m // 2, n // 3] = -2.5
    inputs = [left @ right, left @ right + 1e-4 * torch.randn(m, n, device="cuda", generator=g), one,
              torch.full((m, n), 3.0, device="cuda"), torch.linalg.qr(torch.randn(n, m, device="cuda", generator=g))[0].mT.contiguous()]
    for u in inputs:
        _check(orthogonalise(u), u)
    for scale in (1e-22, 1e22):                                  # squares beyond fp32: the norm is a 64-bit sum
        u = scale * inputs[1]
        got, want = orthogonalise(u, epsilon=1e-30), orthogonalise(inputs[1], epsilon=1e-30)
        # the input is rounded by the scaling (2^-24 a value), and its error grows at most 4^5 times
        assert torch.linalg.matrix_norm(got - want) <= 4 ** 5 * 2.0 ** -23 * torch.linalg.matrix_norm(want)
    assert (orthogonalise(torch.zeros(m, n, device="cuda")) == 0).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("m,n", [(2, 3), (12, 30), (8, 32768), (16, 20000), (20000, 16), (20, 50), (100, 3000), (200, 333), (333, 200), (300, 5000)])
def test_norms_beyond_the_range_of_fp32(m, n, dtype):
    """Finite updates whose norm is not a finite fp32 number, the same by a power of two as an ordinary one: the same result, to
    the same bound."""
    from gmc.optimisation import orthogonalise
    u = _update(m, n, seed=n, dtype=dtype)
    u = u * 2.0 ** -math.frexp(u.abs().max().item())[1]           # the largest element in [0.5, 1)
    huge = u * 2.0 ** 127 * 2                                     # in [2^127, 2^128)
    assert torch.isfinite(huge).all() and torch.linalg.matrix_norm(huge.double()) > torch.finfo(torch.float32).max * (m > 10)
    _check(orthogonalise(huge, epsilon=1e-30), u, epsilon=1e-30)


@pytest.mark.parametrize("m,n", [(12, 30), (140, 260)])
def test_nan_and_infinity_stay_in_their_matrix(m, n):
    from gmc.optimisation import orthogonalise
    u = _update(4, m, n)
    clean = orthogonalise(u)            # the same call but for the values
    u[1, m - 1, n - 1] = math.nan
    u[2, 0, 0] = math.inf
    got = orthogonalise(u)
    assert got[1].isnan().all() and got[2].isnan().all()
    assert torch.equal(got[[0, 3]], clean[[0, 3]])


@pytest.mark.parametrize("steps,coefficients", [(1, COEFFICIENTS), (8, COEFFICIENTS), (6, (1.875, -1.25, 0.375)), (7, (1.5, -0.5, 0.0))])
@pytest.mark.parametrize("m,n", [(24, 70), (150, 200)])
def test_steps_and_coefficients(m, n, steps, coefficients):
    from gmc.optimisation import orthogonalise
    u = _update(m, n, seed=3)
    _check(orthogonalise(u, steps=steps, coefficients=coefficients), u, steps, coefficients)


@pytest.mark.parametrize("c", [0.0, 1e-20, -1e-20, 1e-9])
@pytest.mark.parametrize("m,n", [(24, 70), (150, 200)])
def test_iterates_above_one_with_a_last_coefficient_near_zero(m, n, c):
    """Two equal singular values, 1 / sqrt 2 of the norm, go to sqrt 2 and stay there (up to their sign) under x (3 - 2 x^2): the
    range of X and A that the operands' scale has to hold."""
    from gmc.optimisation import orthogonalise
    u = torch.zeros(m, n, device="cuda")
    u[m // 3, 5] = u[m - 1, n - 2] = 1.0
    # the slope at sqrt 2 is 3 - 6 x^2 = -9: an error there grows to 9^4 of itself in four more steps; c adds c x^5 = 5.7 c a step
    want = torch.zeros_like(u, dtype=torch.float64)
    want[m // 3, 5] = want[m - 1, n - 2] = 2 ** 0.5                # +, then -, +, -, + after five steps
    assert (orthogonalise(u, coefficients=(3.0, -2.0, c)).double() - want).abs().max() <= 2 * 9 ** 4 * (4 * 2.0 ** -22 + 5.7 * abs(c))


@pytest.mark.parametrize("m,n", [(48, 100), (400, 256)])
def test_singular_values_end_near_one(m, n):
    from gmc.optimisation import orthogonalise
    u = torch.randn(m, n, device="cuda", generator=torch.Generator(device="cuda").manual_seed(2))
    s = torch.linalg.svdvals(orthogonalise(u).double())
    # the smallest singular value of these inputs is above 0.01 of the norm: five steps bring it into the band
    assert s.max() < 1.21 and s.min() > 0.3


def test_batches_lists_and_strides():
    from gmc.optimisation import orthogonalise
    # how many CTAs share a matrix's sums depends on what else is in the call: every result is held to the bound by itself
    u = _update(3, 2, 70, 90)
    _check(orthogonalise(u), u)
    for shape in ((101, 10, 12), (50, 130, 70), (50, 150, 200), (2, 1, 300, 200)):
        many = _update(*shape)
        _check(orthogonalise(many), many)
    shapes = [(30, 40), (300, 140), (1, 9), (130, 700), (64, 64), (64, 3000), (700, 90), (1000, 1000), (260, 3000)]
    mixed = [_update(m, n, seed=i) for i, (m, n) in enumerate(shapes)]
    for o, t in zip(orthogonalise(mixed), mixed):
        _check(o, t)
    for size in (40, 200):
        wide = _update(size, 3 * size + 5)
        for view in (wide[:, 3:3 + size], wide[::2, 1:size], wide[:, :size].t(), wide[:1].expand(size, -1)):
            assert torch.equal(orthogonalise(view), orthogonalise(view.contiguous()))
    assert orthogonalise(torch.zeros(0, 4, 5, device="cuda")).shape == (0, 4, 5)
    assert orthogonalise(torch.zeros(4, 0, device="cuda")).shape == (4, 0) and orthogonalise([]) == []


def _muon_reference(p, g, m, lr, momentum, weight_decay, nesterov):
    p, g, m = p.double(), g.double(), m.double()
    m = momentum * m + (1 - momentum) * g
    u = (1 - momentum) * g + momentum * m if nesterov else m
    rows, cols = p.shape[0], p[0].numel()
    x = _plain(u.view(rows, cols), 5, COEFFICIENTS, 1e-7).view(p.shape)
    return (1 - lr * weight_decay) * p - lr * math.sqrt(max(1.0, rows / cols)) * x, m


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("nesterov", [True, False])
@pytest.mark.parametrize("shapes", [[(8, 1, 5, 1), (16, 8, 5, 1), (64, 32, 5, 1), (40, 64)], [(300, 129), (129, 400), (20, 7)], [(640, 2)]])
def test_muon_update(shapes, nesterov, dtype):
    from gmc.optimisation import muon_update
    gen = torch.Generator(device="cuda").manual_seed(4)
    params = [torch.randn(s, device="cuda", generator=gen).to(dtype) for s in shapes]
    grads = [_update(s[0], math.prod(s[1:]), seed=i, dtype=dtype).view(s) for i, s in enumerate(shapes)]
    momenta = [_update(s[0], math.prod(s[1:]), seed=50 + i).view(s) for i, s in enumerate(shapes)]
    lr, momentum, weight_decay = 0.05, 0.9, 0.1
    want = [_muon_reference(p, g, m, lr, momentum, weight_decay, nesterov) for p, g, m in zip(params, grads, momenta)]
    before, versions = [p.clone() for p in params], [p._version for p in params]
    muon_update(params, grads, momenta, lr, momentum, weight_decay, nesterov)
    for p, m, (wp, wm), old, version in zip(params, momenta, want, before, versions):
        assert p._version > version
        # momentum: three roundings of fp32
        assert ((m.double() - wm).abs() <= 3 * 2.0 ** -24 * (wm.abs() + 0.01)).all()
        # parameter: its own rounding, and an update of lr sqrt(..) times an orthogonal matrix whose relative error is below
        # 4^5 times the three roundings of the momentum (the polynomial's largest slope is below 4) and 2^-12 for the products
        half = torch.finfo(dtype).eps / 2
        step = torch.linalg.vector_norm(wp - old.double())
        assert torch.linalg.vector_norm(p.double() - wp) <= (2 * half + 3 * 2.0 ** -24) * torch.linalg.vector_norm(wp) \
            + (4 ** 5 * 3 * 2.0 ** -24 + 2.0 ** -12) * step


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("momentum", [0.0, 0.9, 0.95, 0.999, 0.9999])
@pytest.mark.parametrize("shapes", [[(16, 40)], [(64, 160)], [(300, 129), (9, 700)]])
def test_the_weights_of_the_running_average(shapes, momentum, dtype):
    """Each of b m and (1 - b) g carries the roundings of its factor, of the product and of the sum: three half steps of fp32.
    Nothing is kept of the momenta, and then much, so that either term is seen."""
    from gmc.optimisation import muon_update
    for share in (0.0, 1.0):
        params = [torch.zeros(s, device="cuda", dtype=dtype) for s in shapes]
        grads = [_update(*s, seed=i, dtype=dtype) for i, s in enumerate(shapes)]
        momenta = [share * _update(*s, seed=50 + i) for i, s in enumerate(shapes)]
        old = [m.clone() for m in momenta]
        muon_update(params, grads, momenta, 0.1, momentum)
        for m, o, g in zip(momenta, old, grads):
            kept, new = momentum * o.double(), (1 - momentum) * g.double()
            assert ((m.double() - (kept + new)).abs() <= 3 * 2.0 ** -24 * (kept.abs() + new.abs()) + 2.0 ** -149).all()


def test_muon_update_of_many_matrices_and_strided_gradients():
    """More matrices than one launch takes, of all kinds, with gradients that are transposed or broadcast views."""
    from gmc.optimisation import muon_update
    gen = torch.Generator(device="cuda").manual_seed(8)
    shapes = [(5 + i, 7 + 3 * i) for i in range(60)] + [(130 + i, 140 + i) for i in range(50)]
    params = [torch.randn(s, device="cuda", generator=gen) for s in shapes]
    grads = [_update(s[1], s[0], seed=i).t() if i % 2 else torch.randn(1, s[1], device="cuda", generator=gen).expand(s) for i, s in enumerate(shapes)]
    momenta = [torch.zeros(s, device="cuda") for s in shapes]
    want = [_muon_reference(p, g, m, 0.1, 0.9, 0.0, True) for p, g, m in zip(params, grads, momenta)]
    before = [p.clone() for p in params]
    muon_update(params, grads, momenta, 0.1, 0.9)
    for p, (wp, _), old in zip(params, want, before):
        step = torch.linalg.vector_norm(wp - old.double())
        assert torch.linalg.vector_norm(p.double() - wp) <= 2.0 ** -23 * torch.linalg.vector_norm(wp) + (4 ** 5 * 3 * 2.0 ** -24 + 2.0 ** -12) * step


def test_the_same_tensor_twice_is_refused():
    from gmc._native import GmcError
    from gmc.optimisation import muon_update, orthogonalise
    p, g, m = (torch.zeros(3, 4, device="cuda") for _ in range(3))
    with pytest.raises(GmcError, match="appears twice"):
        muon_update([p, p], [g, g], [m, m.clone()], 0.1)
    with pytest.raises(GmcError, match="share its memory"):
        muon_update([p], [m], [m], 0.1)
    with pytest.raises(GmcError, match="contiguous"):
        muon_update([p.t()], [g.t()], [m.t()], 0.1)
    with pytest.raises(GmcError, match="float32"):
        muon_update([p], [g], [m.bfloat16()], 0.1)
    with pytest.raises(GmcError, match="one type"):
        muon_update([p], [g.bfloat16()], [m], 0.1)
    with pytest.raises(GmcError, match="one type"):
        orthogonalise([p, g.bfloat16()])
    with pytest.raises(GmcError, match="matrices"):
        orthogonalise(torch.zeros(5, device="cuda"))
    with pytest.raises(GmcError, match="up to 32768"):
        orthogonalise(torch.zeros(1, 1, device="cuda").expand(40000, 3))
    with pytest.raises(GmcError, match="unsupported parameter"):
        orthogonalise(p, coefficients=(9.0, 0.0, 0.0))
    with pytest.raises(GmcError, match="unsupported parameter"):
        orthogonalise(p, steps=0)


def test_memory_shared_between_arguments_is_refused():
    """It would be read while it is written. Nothing is changed by the refused call; one gradient for two parameters is fine."""
    from gmc._native import GmcError
    from gmc.optimisation import muon_update
    p, q, m, k = (torch.randn(30, 40, device="cuda") for _ in range(4))
    g = _update(30, 40)
    before = [t.clone() for t in (p, q, m, k)]
    for grads in ([q, g], [g, p], [k, g], [g, m], [p, g], [g, k]):
        with pytest.raises(GmcError, match="share its memory"):
            muon_update([p, q], grads, [m, k], 0.1)
    for params, momenta in (([p, q], [m, q]), ([p, q], [q, k]), ([p], [p])):
        with pytest.raises(GmcError, match="appears twice"):
            muon_update(params, [g] * len(params), momenta, 0.1)
    assert all(torch.equal(a, b) for a, b in zip(before, (p, q, m, k)))
    muon_update([p, q], [g, g], [m, k], 0.1)
    assert not torch.equal(q, before[1])


def test_optimiser_steps_and_state():
    """Three steps of the class on an fp32 and a bf16 parameter against the restatement; the state survives a save and load in
    32 bits; parameters without a gradient are left alone."""
    from gmc.optimisation import Muon
    gen = torch.Generator(device="cuda").manual_seed(6)
    params = [torch.nn.Parameter(torch.randn(48, 96, device="cuda", generator=gen)),
              torch.nn.Parameter(torch.randn(130, 200, device="cuda", generator=gen).bfloat16()),
              torch.nn.Parameter(torch.randn(10, 10, device="cuda", generator=gen))]
    opt = Muon(params, lr=0.03, momentum=0.8, weight_decay=0.05)
    idle = params[2].detach().clone()
    mom = [torch.zeros_like(p, dtype=torch.float32) for p in params[:2]]
    for step in range(3):
        for i, p in enumerate(params[:2]):
            p.grad = _update(*p.shape, seed=10 * step + i, dtype=p.dtype)
        want = [_muon_reference(p.detach(), p.grad, m, 0.03, 0.8, 0.05, True) for p, m in zip(params, mom)]
        if step == 2:
            other = Muon(params, lr=1.0)
            other.load_state_dict(copy.deepcopy(opt.state_dict()))
            opt = other
            for p, m in zip(params, mom):
                assert opt.state[p]["momentum_buffer"].dtype == torch.float32 and torch.equal(opt.state[p]["momentum_buffer"], m)
        opt.step()
        mom = [opt.state[p]["momentum_buffer"].clone() for p in params[:2]]
        for p, m, (wp, wm) in zip(params, mom, want):
            assert torch.linalg.vector_norm(m.double() - wm) <= 2.0 ** -22 * torch.linalg.vector_norm(wm)
            half = torch.finfo(p.dtype).eps / 2
            assert torch.linalg.vector_norm(p.detach().double() - wp) <= (2 * half + 2.0 ** -16) * torch.linalg.vector_norm(wp)
    assert torch.equal(params[2], idle) and params[2] not in opt.state


@pytest.mark.parametrize("dtype", [0, 1, 2])
@pytest.mark.parametrize("m,n", [(1, 5), (5, 9), (9, 5), (16, 2000), (64, 160), (160, 64), (100, 1000), (130, 9), (200, 333), (333, 200),
                                 (700, 1031)])
@pytest.mark.parametrize("gap,first", [(0, 0), (3, 1), (8, 8)])
def test_strided_results_in_place_of_the_update_and_beside_it(m, n, dtype, gap, first):
    """The C entry with rows apart: what lies between them, before and behind stays as it was, with the result in the update's own
    place and elsewhere."""
    from gmc import _native
    u = _update(m, n, seed=m * n, dtype=DTYPES[dtype])
    stride = n + gap
    for in_place in (True, False):
        source = torch.full((first + (m + 1) * stride,), 7.0, device="cuda", dtype=u.dtype)
        source[first:first + m * stride].view(m, stride)[:, :n] = u
        target = source if in_place else torch.full_like(source, 9.0)
        before, place = target.clone(), first * u.element_size()
        packed = _native.matrix_struct.pack(source.data_ptr() + place, 0, target.data_ptr() + place, m, n, stride, stride, 0.0)
        size = _native.lib.gmc_orthogonalise_workspace_bytes(packed, 1)
        hold = torch.empty(size + 1024, dtype=torch.uint8, device="cuda")
        _native.check(_native.lib.gmc_orthogonalise(packed, 1, dtype, 5, *COEFFICIENTS, 1e-7, (hold.data_ptr() + 1023) // 1024 * 1024, size,
                                                    _native.stream_of(u)), "")
        _check(target[first:first + m * stride].view(m, stride)[:, :n], u)
        for t in (target, before):
            t[first:first + m * stride].view(m, stride)[:, :n] = 0.0
        assert torch.equal(target, before)


def test_captured_and_replayed_on_another_stream():
    from gmc.optimisation import muon_update, orthogonalise
    shapes = [(20, 45), (200, 150)]
    params = [torch.randn(s, device="cuda") for s in shapes]
    grads = [_update(*s, seed=1) for s in shapes]
    momenta = [torch.zeros(s, device="cuda") for s in shapes]
    start = [t.clone() for t in params + momenta]
    eager = []
    for _ in range(2):
        muon_update(params, grads, momenta, 0.02)
        eager.append([t.clone() for t in params + momenta])
    graphs, outs = [], []
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        muon_update(params, grads, momenta, 0.02)
        orthogonalise(grads)
    torch.cuda.current_stream().wait_stream(side)
    for _ in range(2):                                              # two graphs, each with its own workspace
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            muon_update(params, grads, momenta, 0.02)
            outs.append(orthogonalise(grads))
        graphs.append(graph)
    for t, s in zip(params + momenta, start):
        t.copy_(s)
    want = orthogonalise(grads)
    for i, graph in enumerate(graphs):
        graph.replay()
        for t, e in zip(params + momenta, eager[i]):
            assert torch.equal(t, e)
        for a, b in zip(outs[i], want):
            assert torch.equal(a, b)


def test_two_calls_at_once():
    from gmc.optimisation import orthogonalise
    u = [_update(300, 500, seed=i) for i in range(2)]
    want = [orthogonalise(v) for v in u]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in u], []
    for s, v in zip(streams, u):
        with torch.cuda.stream(s):
            got.append(orthogonalise(v))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", [(200, 20000), (300, 6000), (6, 400, 1500), (513, 769)])
def test_repeated_calls_are_identical(shape, dtype):
    """Sums of X X^T that several CTAs share are read back by others in every step: the same bits call after call, with other
    values in the workspace in between."""
    from gmc.optimisation import orthogonalise
    u, other = _update(*shape, seed=1, dtype=dtype), _update(*shape, seed=2, dtype=dtype)
    want = orthogonalise(u)
    for _ in range(10):
        orthogonalise(other)
        assert torch.equal(orthogonalise(u), want)


@pytest.mark.parametrize("dtype", [0, 1])
@pytest.mark.parametrize("m,n", [(200, 20000), (300, 700), (1500, 4100)])
def test_a_wait_that_runs_out_gives_nan_and_an_error(m, n, dtype):
    """One warp's first wait counts as run out, early and late in the grid, in tiles of either width and with shared sums: the
    other warps, which have seen what it has not, still meet it at every barrier, and the launch ends by itself."""
    from gmc import _native
    from gmc.optimisation import orthogonalise
    u = _update(m, n, seed=1, dtype=DTYPES[dtype])
    out = torch.zeros_like(u)
    packed = _native.matrix_struct.pack(u.data_ptr(), 0, out.data_ptr(), m, n, n, n, 0.0)
    size = _native.lib.gmc_orthogonalise_workspace_bytes(packed, 1)
    hold = torch.empty(size + 1024, dtype=torch.uint8, device="cuda")
    address = (hold.data_ptr() + 1023) // 1024 * 1024
    assert _native.device_check_word() == 0
    for lost in (0, 5, 8 + 2, 8 * 3 + 7):
        assert _native.lib.gmc_debug_orthogonalise_lost_wait(packed, 1, dtype, 5, *COEFFICIENTS, 1e-7, address, size, lost,
                                                             _native.stream_of(u)) == 0
        assert _native.device_check_word() == 1
        assert out.isnan().all()
    _check(orthogonalise(u), u)
    assert _native.device_check_word() == 0


def test_clusters_of_several_calls_at_once():
    """Small clusters from several streams, more of them than fit side by side: none may wait for what another one holds."""
    from gmc.optimisation import orthogonalise
    gen = torch.Generator(device="cuda").manual_seed(9)
    u = [torch.randn(30, m, n, device="cuda", generator=gen) for m, n in ((64, 500), (40, 600), (100, 700), (12, 900))]
    want = [orthogonalise(v) for v in u]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in u]
    for _ in range(5):
        got = []
        for s, v in zip(streams, u):
            with torch.cuda.stream(s):
                got.append(orthogonalise(v))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_a_training_step_of_the_network():
    """Loss, gradient and both optimisers together: log_probabilities -> backward -> Muon on the matrices, Adam on the rest.
    The matrices move by the restatement's update of the gradients that the backward pass left."""
    import gmc.model as model
    import synthetic_inputs as synthetic
    from gmc.optimisation import Muon
    cfg = model.Config(n_dims=2)
    cfg.layers = [model.Layer(4, 1, 24, 12), model.Layer(10, 1, 16, 8)]
    cfg.mlp = [24, 10]
    torch.manual_seed(11)
    net = model.Net(config=cfg).cuda().train()
    x = synthetic.fit_target_2d(6, 1, 20, 5)
    x[..., 0] = x[..., 0].abs() + 0.1
    x, t = x.cuda(), torch.arange(6, device="cuda") % 10
    matrices = net.matrix_parameters()
    assert len(matrices) == 4
    chosen = {id(p) for p in matrices}
    optimisers = [Muon(matrices, lr=0.01, momentum=0.9), torch.optim.Adam([p for p in net.parameters() if id(p) not in chosen], lr=1e-3)]
    for _ in range(2):
        for o in optimisers:
            o.zero_grad()
        r = net.log_probabilities(x, t)
        (-r.target.mean() - 0.01 * r.entropy.mean()).backward()
        before = [(p.detach().clone(), p.grad.clone(), optimisers[0].state[p].get("momentum_buffer", torch.zeros_like(p)).clone())
                  for p in matrices]
        for o in optimisers:
            o.step()
        for p, (old, g, m) in zip(matrices, before):
            assert torch.isfinite(p).all() and (g != 0).any()
            want, _ = _muon_reference(old, g, m, 0.01, 0.9, 0.0, True)
            bound = 2.0 ** -23 * torch.linalg.vector_norm(want) + (4 ** 5 * 3 * 2.0 ** -24 + 2.0 ** -12) * torch.linalg.vector_norm(want - old)
            assert torch.linalg.vector_norm(p.detach().double() - want) <= bound
    net.eval()
    with torch.no_grad():
        kernels = net.gmcs[0].kernels()
        before = kernels.clone()
        matrices[0].grad = torch.ones_like(matrices[0])
        optimisers[0].step()
        assert not torch.equal(net.gmcs[0].kernels(), before)          # the cached kernel mixture sees the update
