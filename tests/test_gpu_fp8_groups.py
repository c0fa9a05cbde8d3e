"""Groups of the 8-bit product whose offsets make no sense: which rows they leave
untouched, in both kernels and directions.  Tolerances as in test_gpu_fp8.py
(check_product)."""
import pytest

import qauntrunner_b200 as Q
from tests import fp8_plain as F
from tests.test_gpu_fp8 import F32, U, gen, matrices

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def rows_of(off, T):
    """Each group's rows: none where the offsets do not ascend within [0, T], or start below one before."""
    return [(a, b) if 0 <= a <= b <= T and a >= max(off[:g + 1]) else (0, 0)
            for g, (a, b) in enumerate(zip(off, off[1:]))]


def test_the_plain_rule():
    assert rows_of([0, 10, 5, 20, 64], 64) == [(0, 10), (0, 0), (0, 0), (20, 64)]
    assert rows_of([0, 70, 5, 20, 64], 64) == [(0, 0)] * 4
    assert rows_of([-1, 10, 20, 20, 64], 64) == [(0, 0), (10, 20), (20, 20), (20, 64)]


@pytest.mark.parametrize("pair", ["0", "1"])
@pytest.mark.parametrize("back", [False, True])
@pytest.mark.parametrize("off", [[0, 10, 5, 20, 64], [0, 300, 0, 300, 0, 300], [40, 30, 20, 310], [-1, 10, 200, 300],
                                 [0, 100, 301, 200, 300], [0, 1] * 20 + [300], [0] * 33 + [7, 5, 6, 290, 300]])
def test_no_row_is_in_two_groups(monkeypatch, off, back, pair):
    monkeypatch.setenv("QRM_FP8_PAIR", pair)
    groups, T, N, K = len(off) - 1, 300, 144, 272
    kin, kout = (N, K) if back else (K, N)
    g = gen(groups)
    codes, scales = matrices(g, groups, N, K)
    x, xs = F.quantize(torch.randn(T, kin, generator=g))
    m = Q.Fp8Matrix(N, K, codes, scales, groups=groups)
    out = torch.full((T, kout), 5.0).cuda()
    (m.product_t if back else m.product)(F32, x.cuda(), xs.cuda(), T, out, torch.tensor(off, dtype=torch.int32).cuda())
    with pytest.raises(Q.QrmError) as e:
        m.sync()
    assert e.value.code == Q.E_INVALID
    got, xv = out.cpu().double(), F.values(x, xs)
    tol = 128 * 2.0 ** -23 + (F.blocks(kin) + 3) * U
    free = torch.ones(T, dtype=torch.bool)
    for i, (a, b) in enumerate(rows_of(off, T)):
        free[a:b] = False
        w = F.values(codes[i], scales[i], 128)
        w = w if back else w.T
        want, size = xv[a:b] @ w, xv[a:b].abs() @ w.abs()
        assert bool(((got[a:b] - want).abs() <= (tol + 2 * F.ROUND[F32]) * size).all()), i
    assert bool((got[free] == 5.0).all())
    m.close()
