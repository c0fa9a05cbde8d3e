"""What the norm and the 4-bit operators refuse before any device is touched,
their plain forms on small known answers, and on which device a 4-bit matrix
does its work (the host code of fp4.cu on a CUDA runtime that is a fake on the
host).  No GPU."""
import ctypes as C
import os
import subprocess

import numpy as np
import pytest

import qauntrunner_b200 as Q
from qauntrunner_b200 import build as B
from tests import fp4_plain as P

torch = pytest.importorskip("torch")
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
A = 1 << 20   # stands for an aligned device address: nothing here reads it


def refused(f, *a, **k):
    with pytest.raises(Q.QrmError) as e:
        f(*a, **k)
    assert str(e.value)
    return e.value.code


def test_norm_arguments():
    n = (4, 256, A, 1e-5)   # rows, d, w, eps
    assert refused(Q.rms_norm, 3, A, *n, A) == Q.E_FORMAT
    assert refused(Q.rms_norm, 0, A, -1, 256, A, 1e-5, A) == Q.E_INVALID
    assert refused(Q.rms_norm, 0, A, 4, 0, A, 1e-5, A) == Q.E_INVALID
    assert refused(Q.rms_norm, 0, A, 4, (1 << 24) + 1, A, 1e-5, A) == Q.E_INVALID
    for eps in (-1e-5, float("nan"), float("inf")):
        assert refused(Q.rms_norm, 0, A, 4, 256, A, eps, A) == Q.E_INVALID
        assert refused(Q.rms_norm_grad, 0, A, A, 4, 256, A, eps, A) == Q.E_INVALID
    assert refused(Q.rms_norm, 0, None, *n, A) == Q.E_INVALID
    assert refused(Q.rms_norm, 0, A, *n, None) == Q.E_INVALID
    assert refused(Q.rms_norm, 0, A + 2, *n, A) == Q.E_INVALID
    assert refused(Q.rms_norm, 1, A, *n, A, add=A + 1) == Q.E_INVALID
    assert refused(Q.rms_norm, 1, A, *n, A, ld_x=255) == Q.E_INVALID
    assert refused(Q.rms_norm, 1, A, *n, A, sum=A, ld_sum=255) == Q.E_INVALID
    assert refused(Q.rms_norm, 1, A, 4, 256, A + 2, 1e-5, A) == Q.E_INVALID
    assert refused(Q.rms_norm_fp8, 2, A, *n, None, A) == Q.E_INVALID
    assert refused(Q.rms_norm_fp8, 2, A, *n, A, A + 1) == Q.E_INVALID
    assert refused(Q.rms_norm_fp8, 2, A, *n, A, A, ld_scales=1) == Q.E_INVALID
    assert refused(Q.rms_norm_fp4, 2, A, *n, A, A, ld_codes=127) == Q.E_INVALID
    assert refused(Q.rms_norm_fp4, 2, A, *n, A, A, ld_scales=7) == Q.E_INVALID
    assert refused(Q.rms_norm_fp4, 2, A, *n, A, A, y=A + 1) == Q.E_INVALID
    assert refused(Q.rms_norm_grad, 0, None, A, *n, A) == Q.E_INVALID
    assert refused(Q.rms_norm_grad, 0, A, A, *n, None) == Q.E_INVALID
    assert refused(Q.rms_norm_grad, 0, A, A, *n, A, dw=A) == Q.E_INVALID        # no workspace
    assert refused(Q.rms_norm_grad, 0, A, A, *n, A, dw=A + 1, work=A) == Q.E_INVALID
    assert refused(Q.rms_norm_grad, 0, A, A, *n, A, ld_dy=255) == Q.E_INVALID


def test_norm_workspace():
    assert Q.rms_norm_grad_work(1, 7168) == 0 and Q.rms_norm_grad_work(0, 7168) == 0 and Q.rms_norm_grad_work(5, 0) == 0
    assert Q.rms_norm_grad_work(2, 7168) == 2 * 7168 and Q.rms_norm_grad_work(1 << 20, 7168) == 148 * 7168
    assert Q.rms_norm_grad_work(1 << 20, 1024) % 1024 == 0 and Q.rms_norm_grad_work(1 << 20, 1024) >= 148 * 1024


def test_rows_arguments():
    assert refused(Q.quantize_fp4, 4, A, 8, 256, A, A) == Q.E_FORMAT
    assert refused(Q.quantize_fp4, 0, A, -1, 256, A, A) == Q.E_INVALID
    assert refused(Q.quantize_fp4, 0, A, 8, 33, A, A, ld_codes=31) == Q.E_INVALID
    assert refused(Q.quantize_fp4, 0, A, 8, 33, A, A, ld_scales=1) == Q.E_INVALID
    assert refused(Q.quantize_fp4, 0, A, 8, 33, A, A, n_rows=A + 1) == Q.E_INVALID
    assert refused(Q.quantize_fp4, 1, A + 1, 8, 33, A, A) == Q.E_INVALID
    assert refused(Q.gather_rows_fp4, 0, A, A, 1 << 30, 8, 256, A, A, 8) == Q.E_INVALID
    assert refused(Q.gather_rows_fp4, 0, A, None, 4, 2, 256, A, A, 8) == Q.E_INVALID
    assert refused(Q.gather_rows_fp4, 0, A, A, 4, 2, 256, None, A, 8) == Q.E_INVALID
    assert refused(Q.gather_rows_fp4, 0, A, A, 4, 2, 256, A, A, -1) == Q.E_INVALID


def test_matrix_arguments():
    c, s = np.zeros((2, 200, 160), np.uint8), np.zeros((2, 200, 10), np.uint8)
    assert refused(Q.Fp4Matrix, 200, 300, c, s) == Q.E_SIZE
    assert refused(Q.Fp4Matrix, 200, 300, c, s[:, :1], groups=2) == Q.E_SIZE
    assert refused(Q.Fp4Matrix, 200, 0, c, s, groups=2) == Q.E_INVALID
    assert refused(Q.Fp4Matrix, (1 << 22) + 1, 32, c, s) == Q.E_INVALID
    assert refused(Q.Fp4Matrix, 1, 1, np.zeros(1025 * 16, np.uint8), np.zeros(1025, np.uint8), groups=1025) == Q.E_CAPACITY
    with pytest.raises(ValueError):
        Q.Fp4Matrix(200, 300, c.astype(np.int16), s, groups=2)
    with pytest.raises(ValueError):
        Q.Fp4Matrix(200, 300, c, s.astype(np.float32), groups=2)
    h = C.c_void_p()
    L = Q.lib()
    assert L.qrm_fp4_create(0, 1, 8, 32, None, 128, None, 8, C.byref(h)) == Q.E_INVALID and not h
    assert L.qrm_fp4_product(None, A, 0, A, 0, None, 1, 0, A, 0, None) == Q.E_INVALID
    assert L.qrm_fp4_swiglu(None, A, 0, A, 0, None, 1, 0.0, 0, A, 0, None) == Q.E_INVALID
    assert L.qrm_fp4_swiglu_fp4(None, A, 0, A, 0, None, 1, 0.0, A, 0, A, 0, None) == Q.E_INVALID
    assert L.qrm_fp4_sync(None) == Q.E_INVALID
    L.qrm_fp4_destroy(None)


@pytest.mark.skipif(torch.cuda.is_available(), reason="checks the no-device error path")
def test_without_a_device_the_error_is_clean():
    c, s = np.zeros((2, 200, 160), np.uint8), np.zeros((2, 200, 10), np.uint8)
    assert refused(Q.Fp4Matrix, 200, 300, c, s, groups=2) == Q.E_CUDA
    assert refused(Q.rms_norm, 0, A, 4, 256, A, 1e-5, A) == Q.E_CUDA
    assert refused(Q.quantize_fp4, 0, A, 8, 256, A, A) == Q.E_CUDA


def test_plain_forms():
    x = torch.zeros(1, 34)
    x[0, 0], x[0, 1], x[0, 2], x[0, 3], x[0, 33] = 6.0, -5.0, 0.25, 7.9, 3.0
    codes, scales = P.quantize(x)
    assert scales.tolist() == [[127, 126]] and codes.shape == (1, 32)
    # 5 and 0.25 are ties (to 4 and 0); 7.9 is cut off at 6; 3 is 6 halves
    v = P.values(codes, scales, 34)
    assert v[0, :4].tolist() == [6.0, -4.0, 0.0, 6.0] and v[0, 33] == 3.0
    assert int(codes[0, 0]) == 7 | (14 << 4) and int(codes[0, 16]) == 7 << 4


# ------------------------------------------------------------ devices

@pytest.fixture(scope="module")
def built(tmp_path_factory):
    B.build(quiet=True)
    cuda = os.path.join(os.path.dirname(os.path.dirname(os.path.realpath(B.nvcc()))), "include")
    so = tmp_path_factory.mktemp("fake4") / "libfake4.so"
    subprocess.run(["g++", "-O1", "-std=c++17", "-shared", "-fPIC", "-Wl,-Bsymbolic", "-I", cuda,
                    os.path.join(ROOT, "tests", "fake_cudart.cpp"), os.path.join(B.BUILD, "norm.o"),
                    os.path.join(B.BUILD, "fp4.o"), "-o", str(so)], check=True)
    lib = C.CDLL(str(so))
    lib.fake_events.restype = C.c_char_p
    for n in Q._SIGS:
        if n.startswith(("qrm_fp4_", "qrm_rms_")) or n == "qrm_last_error":
            getattr(lib, n).restype, getattr(lib, n).argtypes = Q._SIGS[n]
    return lib


@pytest.fixture
def fake(built, monkeypatch):
    monkeypatch.setattr(Q, "_lib", built)
    built.fake_reset(0)
    return built


def events(fake):
    return fake.fake_events().decode().split("\n")[:-1]


def host_matrix(device=None, rows=200, groups=2):
    return Q.Fp4Matrix(rows, 300, np.zeros((groups, rows, 160), np.uint8), np.zeros((groups, rows, 10), np.uint8), groups=groups,
                       device=device)


@pytest.mark.parametrize("caller,device", [(0, 1), (1, 0), (0, 0), (1, 1)])
def test_a_matrix_leaves_the_current_device(fake, caller, device):
    fake.fake_reset(caller)
    m = host_matrix(device)
    assert fake.fake_current() == caller and set(e.split()[1] for e in events(fake)) == {str(device)}
    for call in (lambda: m.product(0, A, A, 8, A, offsets=A), lambda: m.swiglu(0, A, A, 8, A, offsets=A),
                 lambda: m.swiglu_fp4(A, A, 8, A, A, offsets=A)):
        fake.fake_reset(caller)
        call()
        assert events(fake) == [f"launch {device}"] and fake.fake_current() == caller
    fake.fake_reset(caller)
    m.sync()
    assert events(fake)[0] == f"synchronise {device}" and fake.fake_current() == caller
    fake.fake_reset(caller)
    m.close()
    assert events(fake) == [f"synchronise {device}", f"free {device}"] and fake.fake_current() == caller
    Q.rms_norm(0, A, 4, 256, A, 1e-5, A)
    assert events(fake)[-1] == f"launch {caller}"


def test_a_failed_creation_keeps_nothing(fake):
    fake.fake_fail_malloc()
    with pytest.raises(Q.QrmError) as e:
        host_matrix(1)
    assert e.value.code == Q.E_NOMEM and fake.fake_current() == 0
    assert "allocate 1" not in events(fake)


def test_product_arguments(fake):
    m, odd = host_matrix(), host_matrix(rows=201)
    ok = dict(offsets=A)
    assert refused(m.product, 3, A, A, 8, A, **ok) == Q.E_FORMAT
    assert refused(m.product, 0, A, A, -1, A, **ok) == Q.E_INVALID
    assert refused(m.product, 0, A, A, 1 << 31, A, **ok) == Q.E_INVALID
    assert refused(m.product, 0, A, A, (1 << 31) - 1, A, **ok) == Q.E_INVALID   # (tiles' ends would pass 32 bits)
    assert refused(m.swiglu, 0, A, A, (1 << 31) - 500, A, **ok) == Q.E_INVALID
    assert refused(m.product, 0, A, A, 8, A) == Q.E_INVALID                    # two matrices need offsets
    assert refused(m.product, 0, A + 8, A, 8, A, **ok) == Q.E_INVALID
    assert refused(m.product, 0, A, A, 8, A, ld_x=168, **ok) == Q.E_INVALID
    assert refused(m.product, 0, A, A, 8, A, ld_x=144, **ok) == Q.E_INVALID
    assert refused(m.product, 0, A, A, 8, A, ld_scales=9, **ok) == Q.E_INVALID
    assert refused(m.product, 0, A, A, 8, A + 2, **ok) == Q.E_INVALID
    assert refused(m.product, 0, A, A, 8, A, ld_y=199, **ok) == Q.E_INVALID
    assert refused(m.product, 0, A, A, 8, A, offsets=A + 1) == Q.E_INVALID
    assert refused(m.product, 0, A, None, 8, A, **ok) == Q.E_INVALID
    assert refused(odd.swiglu, 0, A, A, 8, A, **ok) == Q.E_INVALID
    for limit in (-1.0, float("nan")):
        assert refused(m.swiglu, 0, A, A, 8, A, limit=limit, **ok) == Q.E_INVALID
    assert refused(m.swiglu, 0, A, A, 8, A, ld_h=99, **ok) == Q.E_INVALID
    assert refused(m.swiglu_fp4, A, A, 8, A + 8, A, **ok) == Q.E_INVALID
    assert refused(m.swiglu_fp4, A, A, 8, A, None, **ok) == Q.E_INVALID
    assert refused(m.swiglu_fp4, A, A, 8, A, A, ld_codes=56, **ok) == Q.E_INVALID
    assert refused(m.swiglu_fp4, A, A, 8, A, A, ld_scales=3, **ok) == Q.E_INVALID
    n = len(events(fake))
    m.product(0, None, None, 0, None)   # no rows: nothing to do, nothing refused
    assert len(events(fake)) == n
    m.close()
    odd.close()
