"""CPU: what the training-step operators refuse before any GPU work is issued."""
import ctypes
import os
import subprocess
import sys

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


def test_log_probabilities_refuses_forward_mode_derivatives():
    """A dual tensor does not require a gradient; its tangent must not be dropped in silence."""
    from torch.autograd import forward_ad

    from gmc._native import GmcError
    from gmc.classification import log_probabilities
    z = torch.zeros(2, 3)
    with forward_ad.dual_level():
        with pytest.raises(GmcError, match="forward-mode"):
            log_probabilities(forward_ad.make_dual(z, torch.ones(2, 3)))
        with pytest.raises(GmcError, match="no CPU implementation"):
            log_probabilities(z)
    with pytest.raises(GmcError, match="forward-mode"):
        with forward_ad.dual_level():
            log_probabilities(forward_ad.make_dual(torch.nn.Parameter(z), torch.ones(2, 3)) * 2)


def test_orthogonalise_argument_checks():
    from gmc import _native
    address = 1024

    def run(rows=130, cols=140, us=140, os_=140, update=16, out=16, momentum=16, dtype=0, steps=5, abc=(3.4445, -4.775, 2.0315), eps=1e-7,
            n=1, work=address, size=1 << 30, muon=False, beta=0.9):
        m = _native.matrix_struct.pack(update, momentum, out, rows, cols, us, os_, 0.1)
        if muon:
            return _native.lib.gmc_muon_update(m, n, dtype, steps, *abc, eps, beta, 1, 1.0, work, size, NULL)
        return _native.lib.gmc_orthogonalise(m, n, dtype, steps, *abc, eps, work, size, NULL)

    assert run(rows=16385, cols=16385, us=16385, os_=16385) == 1
    assert run(rows=0) == 1 and run(cols=0) == 1 and run(rows=32769) == 1 and run(us=139) == 1 and run(os_=139) == 1 and run(n=-1) == 1
    assert run(dtype=3) == 4 and run(steps=0) == 4 and run(steps=33) == 4 and run(eps=0.0) == 4 and run(eps=float("nan")) == 4
    assert run(abc=(10.0, 0.0, 0.0)) == 4 and run(abc=(float("nan"), 0.0, 0.0)) == 4 and run(abc=(1.0, -4.0, 0.0)) == 4
    assert run(update=0) == 3 and run(out=0) == 3 and run(work=0) == 3 and run(work=address + 16) == 4
    assert run(size=64) == 10 and run(n=0, update=0) == 0
    assert run(muon=True, momentum=0) == 3 and run(muon=True, beta=1.0) == 4 and run(muon=True, beta=-0.1) == 4
    m = _native.matrix_struct.pack(16, 0, 16, 300, 500, 500, 500, 0.0)
    assert _native.lib.gmc_orthogonalise_workspace_bytes(m, 1) > 0
    assert _native.lib.gmc_orthogonalise_workspace_bytes(_native.matrix_struct.pack(16, 0, 16, 30, 50, 50, 50, 0.0), 1) == 0
    assert _native.lib.gmc_orthogonalise_workspace_bytes(_native.matrix_struct.pack(16, 0, 16, 0, 5, 5, 5, 0.0), 1) == 0


@pytest.mark.parametrize("c", [1e-20, -1e-20, 1e-30, 1e-16, 1e-8, 0.0])
def test_coefficients_are_bounded_however_small_the_last_one_is(c):
    """x (a + b x^2) with a = 3.4, b = -2.4 reaches 1.557 at x^2 = a / -3b and leaves the range from there; with a = 3, b = -2 it
    stays below 1.415 for ever. A c this small changes neither. (A workspace that is too small is found after the coefficients.)"""
    from gmc import _native
    m = _native.matrix_struct.pack(16, 0, 16, 130, 140, 140, 140, 0.0)

    def run(a, b):
        return _native.lib.gmc_orthogonalise(m, 1, 0, 5, a, b, c, 1e-7, 1024, 64, NULL)

    assert run(3.4, -2.4) == 4 and run(3.0, -2.0) == 10


def test_optimisation_refuses_what_it_cannot_do():
    from gmc._native import GmcError
    from gmc.optimisation import Muon, muon_update, orthogonalise
    t = torch.zeros(3, 4)
    with pytest.raises(GmcError, match="no CPU implementation"):
        orthogonalise(t)
    with pytest.raises(GmcError, match="three numbers"):
        orthogonalise(t, coefficients=(1.0, 2.0))
    with pytest.raises(GmcError, match="one entry per parameter"):
        muon_update([t], [t], [], 0.1)
    with pytest.raises(GmcError, match="finite"):
        muon_update([t], [t], [t], float("nan"))
    with pytest.raises(GmcError, match="no CPU implementation"):
        muon_update([t], [t], [t], 0.1)
    with pytest.raises(GmcError, match="two or more axes"):
        Muon([torch.nn.Parameter(torch.zeros(5))])
    muon_update([], [], [], 0.1)


def test_muon_refuses_parameters_with_one_axis_in_later_groups():
    from gmc._native import GmcError
    from gmc.optimisation import Muon
    opt = Muon([torch.nn.Parameter(torch.zeros(5, 3))])
    with pytest.raises(GmcError, match="two or more axes"):
        opt.add_param_group({"params": [torch.nn.Parameter(torch.zeros(4, 3)), torch.nn.Parameter(torch.zeros(5))]})
    assert len(opt.param_groups) == 1
    opt.add_param_group({"params": torch.nn.Parameter(torch.zeros(4, 3)), "lr": 0.5})
    assert [g["lr"] for g in opt.param_groups] == [0.02, 0.5]


def test_muon_loads_states_without_a_momentum():
    """A parameter whose state was only looked at has an empty one; it is saved and loaded like any other."""
    from gmc.optimisation import Muon
    params = [torch.nn.Parameter(torch.zeros(5, 3)), torch.nn.Parameter(torch.zeros(3, 4, dtype=torch.bfloat16))]
    opt, other = Muon(params), Muon(params)
    assert opt.state[params[0]] == {}
    opt.state[params[1]]["momentum_buffer"] = torch.full((3, 4), 1 / 3)
    other.load_state_dict(opt.state_dict())
    assert "momentum_buffer" not in other.state[params[0]]
    assert torch.equal(other.state[params[1]]["momentum_buffer"], torch.full((3, 4), 1 / 3))


FAKE_RUNTIME = """
int launches;
int cudaGetDevice(int* device) { *device = 0; return 0; }
int cudaDeviceGetAttribute(int* value, int attribute, int device) { *value = 148; return 0; }
int cudaFuncSetAttribute(const void* f, int attribute, int value) { return 0; }
int cudaOccupancyMaxActiveClusters(int* n, const void* f, const void* config) { *n = PAIRS; return 0; }
int cudaLaunchKernelExC(const void* config, const void* f, void** arguments) { ++launches; return 0; }
int cudaLaunchKernel() { ++launches; return 0; }
int cudaGetLastError(void) { return 0; }
"""
CALL = """
import ctypes, struct, sys
fake, lib = ctypes.CDLL(sys.argv[1]), ctypes.CDLL(sys.argv[2])
pack = lambda rows, cols: struct.pack("@PPPqqqqf4x", 16, 16, 16, rows, cols, cols, cols, 0.1)
lib.gmc_muon_update.argtypes = ([ctypes.c_char_p] + [ctypes.c_int] * 3 + [ctypes.c_float] * 4 + [ctypes.BETA]
                                + [ctypes.c_int, ctypes.c_float, ctypes.c_void_p, ctypes.c_size_t, ctypes.c_void_p])
status = lib.gmc_muon_update(pack(64, 160) + pack(300, 500), 2, 0, 5, 3.4445, -4.775, 2.0315, 1e-7, 0.9, 1, 1.0, 1024, 1 << 30, None)
print(status, ctypes.c_int.in_dll(fake, "launches").value)
"""


@pytest.mark.parametrize("pairs,expected", [(47, "4 0"), (48, "0 5"), (74, "0 5")])
def test_a_device_that_cannot_hold_the_call_is_refused_before_anything_is_launched(tmp_path, pairs, expected):
    """A fake of the runtime counts launches: the cooperative kernel that the larger matrix needs wants 48 pairs of CTAs. Where they
    are missing, the smaller matrix's parameters must not have moved."""
    from gmc import _native
    source, fake = tmp_path / "fake.c", tmp_path / "fake.so"
    source.write_text(FAKE_RUNTIME.replace("PAIRS", str(pairs)))
    subprocess.run(["gcc", "-shared", "-fPIC", "-w", "-o", fake, source], check=True)
    beta = {4: "c_float", 8: "c_double"}[ctypes.sizeof(_native.lib.gmc_muon_update.argtypes[8])]
    out = subprocess.run([sys.executable, "-c", CALL.replace("BETA", beta), str(fake), _native.lib._name], capture_output=True, text=True,
                         env=dict(os.environ, LD_PRELOAD=str(fake), LD_LIBRARY_PATH=os.pathsep.join(
                             filter(None, [os.path.dirname(_runtime_path()), os.environ.get("LD_LIBRARY_PATH")]))))
    assert out.stdout.strip() == expected, out.stdout + out.stderr


def _runtime_path():
    """The CUDA runtime that this process has loaded with the library."""
    with open("/proc/self/maps") as maps:
        return next(line.split()[-1] for line in maps if "libcudart.so" in line)
