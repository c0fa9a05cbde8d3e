"""On which device the 8-bit expert operators do their work, and which one is
current afterwards: the host code of rows.cu and fp8.cu on a CUDA runtime of two
devices that is a fake on the host (fake_cudart.cpp).  No GPU."""
import ctypes as C
import os
import subprocess
from types import SimpleNamespace

import numpy as np
import pytest

import qauntrunner_b200 as Q
from qauntrunner_b200 import build as B

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
A = 1 << 20   # stands for an aligned device address: nothing here reads it
OURS = [n for n in Q._SIGS if n.startswith("qrm_fp8_") or n == "qrm_last_error" or
        n.startswith(("qrm_sort", "qrm_gather", "qrm_combine", "qrm_quantize", "qrm_swiglu"))]


@pytest.fixture(scope="module")
def built(tmp_path_factory):
    B.build(quiet=True)
    cuda = os.path.join(os.path.dirname(os.path.dirname(os.path.realpath(B.nvcc()))), "include")
    so = tmp_path_factory.mktemp("fake") / "libfake.so"
    # (-Bsymbolic: a process with torch in it has another CUDA runtime's functions of the same names)
    subprocess.run(["g++", "-O1", "-std=c++17", "-shared", "-fPIC", "-Wl,-Bsymbolic", "-I", cuda,
                    os.path.join(ROOT, "tests", "fake_cudart.cpp"), os.path.join(B.BUILD, "rows.o"),
                    os.path.join(B.BUILD, "fp8.o"), "-o", str(so)], check=True)
    lib = C.CDLL(str(so))
    lib.fake_events.restype = C.c_char_p
    lib.fake_place.argtypes = [C.c_void_p, C.c_int]
    for n in OURS:
        getattr(lib, n).restype, getattr(lib, n).argtypes = Q._SIGS[n]
    return lib


@pytest.fixture
def fake(built, monkeypatch):
    monkeypatch.setattr(Q, "_lib", built)
    built.fake_reset(0)
    return built


def events(fake):
    return fake.fake_events().decode().split("\n")[:-1]


def host_matrix(device=None):
    return Q.Fp8Matrix(200, 300, np.zeros((2, 200, 300), np.uint8), np.ones((2, 2, 3), np.float32), groups=2,
                       device=device)


@pytest.mark.parametrize("caller,device", [(0, 1), (1, 0), (0, 0), (1, 1)])
def test_a_matrix_leaves_the_current_device(fake, caller, device):
    fake.fake_reset(caller)
    m = host_matrix(device)
    assert fake.fake_current() == caller
    assert set(e.split()[1] for e in events(fake)) == {str(device)}
    for f, pitch in ((m.product, {"ld_x": 304}), (m.product_t, {"ld_y": 208})):
        fake.fake_reset(caller)
        f(Q.QuantFormat.F32, A, A, 8, A, offsets=A, **pitch)
        assert events(fake) == [f"launch {device}"] and fake.fake_current() == caller
    fake.fake_reset(caller)
    m.sync()
    assert events(fake)[0] == f"synchronise {device}" and fake.fake_current() == caller
    fake.fake_reset(caller)
    m.close()
    assert events(fake) == [f"synchronise {device}", f"free {device}"] and fake.fake_current() == caller
    Q.quantize_fp8(Q.QuantFormat.F32, A, 8, 256, A, A)
    assert events(fake)[-1] == f"launch {caller}"


def test_a_collected_matrix_leaves_the_current_device(fake):
    m = host_matrix(1)
    del m
    assert fake.fake_current() == 0 and events(fake)[-1] == "free 1"


def test_refusals_leave_the_current_device(fake):
    fake.fake_fail_malloc()
    with pytest.raises(Q.QrmError) as e:
        host_matrix(1)
    assert e.value.code == Q.E_NOMEM and fake.fake_current() == 0
    fake.fake_reset(1)
    with pytest.raises(Q.QrmError) as e:
        host_matrix(2)
    assert e.value.code == Q.E_INVALID and fake.fake_current() == 1


class OnDevice:
    """What Fp8Matrix takes of a tensor on a device."""
    is_cuda, nbytes = True, 0

    def __init__(self, fake, array, index, dtype):
        self._a, self.nbytes, self.dtype = array, array.nbytes, dtype
        self.device = SimpleNamespace(index=index)
        fake.fake_place(array.ctypes.data, index)

    def contiguous(self):
        return self

    def element_size(self):
        return self._a.itemsize

    def data_ptr(self):
        return self._a.ctypes.data


@pytest.mark.parametrize("caller", [0, 1])
@pytest.mark.parametrize("codes_on,scales_on,device,kept", [
    (1, 1, None, 1), (0, 0, None, 0), (1, 1, 0, 0), (0, 0, 1, 1), (1, 0, None, 1), (0, 1, 0, 0)])
def test_a_matrix_is_kept_where_its_codes_are(fake, codes_on, scales_on, device, kept, caller):
    fake.fake_reset(caller)
    codes = OnDevice(fake, np.zeros((2, 200, 300), np.uint8), codes_on, "torch.uint8")
    scales = OnDevice(fake, np.ones((2, 2, 3), np.float32), scales_on, "torch.float32")
    m = Q.Fp8Matrix(200, 300, codes, scales, groups=2, device=device)
    log = events(fake)
    assert f"allocate {kept}" in log and fake.fake_current() == caller
    before = log[:log.index(f"copy {kept}")]   # every device that may still write the sources was waited for
    assert {f"synchronise {d}" for d in (kept, codes_on, scales_on)} <= set(before)
    m.close()


def test_host_arrays_go_to_the_first_device_or_the_one_named(fake):
    for device, kept in ((None, 0), (0, 0), (1, 1)):
        fake.fake_reset(1)
        m = host_matrix(device)
        assert f"allocate {kept}" in events(fake)
        m.close()
