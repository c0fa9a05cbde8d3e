"""What the 8-bit expert operators refuse before any device is touched, and
their plain forms checked on small known answers (no GPU)."""
import ctypes as C

import numpy as np
import pytest

import qauntrunner_b200 as Q
from tests import fp8_plain as F

torch = pytest.importorskip("torch")
A = 1 << 20   # stands for an aligned device address: nothing here reads it


def refused(f, *a, **k):
    with pytest.raises(Q.QrmError) as e:
        f(*a, **k)
    assert str(e.value)
    return e.value.code


def test_arguments_are_checked_before_the_device():
    assert refused(Q.sort_tokens, A, 8, 2, 1025, A, A, A) == Q.E_CAPACITY
    assert refused(Q.sort_tokens, A, 8, 2, 4, A, A + 2, A) == Q.E_INVALID
    assert refused(Q.sort_tokens, A, 1 << 30, 8, 4, A, A, A) == Q.E_INVALID
    assert refused(Q.gather_rows, 3, A, A, 4, 2, 256, A, 8) == Q.E_FORMAT
    assert refused(Q.gather_rows, 0, A, A, 4, 2, 0, A, 8) == Q.E_INVALID
    assert refused(Q.gather_rows, 0, A, A, 4, 2, 256, A, 8, ld_x=255) == Q.E_INVALID
    assert refused(Q.gather_rows_fp8, 2, A, A, 4, 2, 256, A, None, 8) == Q.E_INVALID
    assert refused(Q.combine_rows, 1, A + 1, 8, A, A, 4, 2, 256, A) == Q.E_INVALID
    assert refused(Q.combine_rows_grad, 0, A, A, 8, A, A + 1, 4, 2, 256, A, A) == Q.E_INVALID
    assert refused(Q.combine_rows_grad_fp8, 0, A, A, 8, A, A, 4, 2, 256, A, A, ld_scales=1) == Q.E_INVALID
    assert refused(Q.quantize_fp8, 0, A, -1, 256, A, A) == Q.E_INVALID
    assert refused(Q.swiglu_fp8, 0, A, 8, 256, A, A, limit=float("nan")) == Q.E_INVALID
    assert refused(Q.swiglu_fp8_grad, 0, A, A, 8, 200, A, A) == Q.E_INVALID
    assert Q.lib().qrm_fp8_product(None, A, 0, A, 0, None, 1, 0, A, 0, None) == Q.E_INVALID
    assert Q.lib().qrm_fp8_sync(None) == Q.E_INVALID
    Q.lib().qrm_fp8_destroy(None)


def test_matrix_sizes_are_checked_before_the_device():
    c, s = np.zeros((2, 200, 300), np.uint8), np.ones((2, 2, 3), np.float32)
    assert refused(Q.Fp8Matrix, 200, 300, c, s) == Q.E_SIZE
    assert refused(Q.Fp8Matrix, 200, 300, c, s[:, :1], groups=2) == Q.E_SIZE
    assert refused(Q.Fp8Matrix, 200, 0, c, s, groups=2) == Q.E_INVALID
    assert refused(Q.Fp8Matrix, 1, 1, np.zeros(1025, np.uint8), np.ones(1025, np.float32), groups=1025) == Q.E_CAPACITY
    h = C.c_void_p()
    assert Q.lib().qrm_fp8_create(0, 1, 8, 8, None, 64, None, 4, C.byref(h)) == Q.E_INVALID and not h


@pytest.mark.skipif(torch.cuda.is_available(), reason="checks the no-device error path")
def test_without_a_device_the_error_is_clean():
    c, s = np.zeros((2, 200, 300), np.uint8), np.ones((2, 2, 3), np.float32)
    assert refused(Q.Fp8Matrix, 200, 300, c, s, groups=2) == Q.E_CUDA
    assert refused(Q.sort_tokens, A, 8, 2, 4, A, A, A) == Q.E_CUDA
    assert refused(Q.quantize_fp8, 0, A, 8, 256, A, A) == Q.E_CUDA


def test_plain_forms():
    idx = torch.tensor([[2, 0], [1, 2], [5, 0]], dtype=torch.int32)
    perm, pos, off = F.order(idx, 0, 3)
    assert perm == [1, 5, 2, 0, 3, -1] and pos == [3, 0, 2, 4, -1, 1] and off == [0, 2, 3, 5]
    x = torch.zeros(1, 130)
    x[0, 0], x[0, 1], x[0, 129] = 448.0, 17.0, -2.0
    c, s = F.quantize(x)
    assert s.tolist() == [[1.0, np.float32(2.0) / np.float32(448.0)]]
    v = F.values(c, s)
    assert v[0, 0] == 448.0 and v[0, 1] == 16.0 and abs(float(v[0, 129]) + 2.0) < 1e-6   # 17: a tie, to the even code
