"""The 8-bit product's kernel for large groups (QRM_FP8_PAIR=1), by itself: it
takes outputs whose rows start on 16 bytes, writes rows that start on 32 bytes
with other stores, and the last values of a row one by one.  Every case here has
such rows, which is asserted, so none falls to the other kernel.  Tolerances as
in test_gpu_fp8.py (check_product: rows outside the groups and the gaps between
rows stay as they were)."""
import pytest

from tests import fp8_plain as F
from tests.test_gpu_fp8 import BF16, F16, F32, check_product, gen, matrices

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def gap(outputs, type, start):
    """Values between rows of `outputs`, so that they start on multiples of `start` bytes and of no larger power of two
    below 64."""
    size = torch.finfo(F.DTYPE[type]).bits // 8
    extra = next(e for e in range(64) if (outputs + e) * size % (2 * start) == start)
    assert (outputs + extra) * size % 16 == 0
    return extra


@pytest.mark.parametrize("start", [16, 32])
@pytest.mark.parametrize("type", [F32, F16, BF16])
@pytest.mark.parametrize("back", [False, True])
@pytest.mark.parametrize("outputs", [1, 7, 120, 127, 130, 200, 255, 257, 513, 1001, 1032])
def test_ends_of_rows(monkeypatch, outputs, back, type, start):
    monkeypatch.setenv("QRM_FP8_PAIR", "1")
    counts = [1, 0, 130, 5]
    codes, scales = matrices(gen(outputs), len(counts), *((144, outputs) if back else (outputs, 144)))
    check_product(codes, scales, counts, type, back, outputs + type, lead=3, extra=gap(outputs, type, start))


@pytest.mark.parametrize("start", [16, 32])
@pytest.mark.parametrize("type", [F32, F16, BF16])
@pytest.mark.parametrize("back", [False, True])
@pytest.mark.parametrize("counts,lead", [([300], 0), ([256, 128, 0, 127], 1), ([0, 0, 513, 1, 257], 130), ([129, 255], 7)])
def test_groups(monkeypatch, counts, lead, back, type, start):
    monkeypatch.setenv("QRM_FP8_PAIR", "1")
    n, k = 392, 272
    codes, scales = matrices(gen(len(counts)), len(counts), n, k)
    check_product(codes, scales, counts, type, back, sum(counts) + type, lead=lead, extra=gap(k if back else n, type, start))
