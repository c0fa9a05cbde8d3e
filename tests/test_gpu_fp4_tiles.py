"""The 4-bit products where a pair of SMs takes several tiles, one after the
other: both accumulators, the rings and the scales' buffers carried from tile to
tile.  Tolerances are those of test_gpu_fp4.py: sums are exact, SwiGLU is within
16 u."""
import pytest

import qauntrunner_b200 as Q
from tests import fp4_plain as P
from tests import fp8_plain as F
from tests.test_gpu_fp4 import TYPES, U, form, gen, rows4  # noqa: F401 (form: a fixture)

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def gated_slack(want, f, gated, type):
    """As in test_gated."""
    slack = 16 * U * gated.abs() + 4 * 2.0 ** -149 * (want[:, :f] * want[:, f:]).abs()
    return slack + F.ROUND[type] * (gated.abs() + slack) + F.HALF_STEP[type]


def run(sizes, n, k, spread, limit):
    """The product in all types, the gated one in all types and in 4-bit rows."""
    T, groups, f = sum(sizes), len(sizes), n // 2
    g = gen(T + groups + n + k)
    w, x = P.random_rows(g, groups * n, k, spread), P.random_rows(g, T, k, spread)
    edges = torch.tensor([0] + sizes).cumsum(0)
    want = torch.empty(T, n, dtype=torch.float64)
    for i in range(groups):
        a, b = int(edges[i]), int(edges[i + 1])
        wi, xi = P.values(w[0][i * n:(i + 1) * n], w[1][i * n:(i + 1) * n], k), P.values(x[0][a:b], x[1][a:b], k)
        want[a:b] = xi @ wi.T
        # magnitudes of a sum's terms, multiples of 2^-2 2^-2 spread: f32 holds their sums
        assert a == b or float(xi.abs().sum(1).max()) * float(wi.abs().max()) < 2.0 ** (22 - 2 * spread)
    off = edges.int().cuda() if groups > 1 else None
    m = Q.Fp4Matrix(n, k, w[0].cuda(), w[1].cuda(), groups=groups)
    codes, scales = x[0].cuda(), x[1].cuda()
    for type in TYPES:
        y = torch.full((T + 1, n), 5.0, dtype=F.DTYPE[type]).cuda()
        m.product(type, codes, scales, T, y, offsets=off)
        m.sync()
        assert torch.equal(y[:T].cpu(), want.float().to(F.DTYPE[type])) and bool((y[T] == 5).all())
    # (gates of up to some tens: exact smaller sums)
    scales, want = (scales.int() - 4).to(torch.uint8), want / 16
    gated = P.gate(want, limit)
    for type in TYPES:
        h = torch.full((T + 1, f), 5.0, dtype=F.DTYPE[type]).cuda()
        m.swiglu(type, codes, scales, T, h, offsets=off, limit=limit)
        m.sync()
        got = h.cpu()
        top = float(torch.finfo(F.DTYPE[type]).max)
        fits = gated.abs() < top * (1 - 2.0 ** -10)
        assert bool(((got[:T].double() - gated).abs() <= gated_slack(want, f, gated, type))[fits].all())
        assert bool((got[T] == 5).all())
        if type == 0:
            h32 = got[:T]
    c4, s4 = rows4(T + 1, f)
    m.swiglu_fp4(codes, scales, T, c4, s4, offsets=off, limit=limit)
    m.sync()
    qc, qs = P.quantize(h32)
    assert torch.equal(c4[:T].cpu(), qc) and torch.equal(s4[:T].cpu(), qs)
    assert bool((c4[T] == 0x77).all()) and bool((s4[T] == 0x77).all())
    m.close()


@pytest.mark.parametrize("rows,n,k,limit", [(2100, 9000, 300, 0.0), (1300, 14336, 32, 7.0), (2560, 5632, 1100, 7.0)])
def test_one_matrix(rows, n, k, limit, form):  # noqa: F811
    """Some 220 to 340 tiles, of two, one and five stages each."""
    run([rows], n, k, 1 if k > 1000 else 2, limit)


@pytest.mark.parametrize("groups,n,k", [(75, 1000, 1800), (30, 2600, 2304)])
def test_groups_with_a_few_rows_behind_a_tile(groups, n, k, form):  # noqa: F811
    """Some 300 tiles, most of them with a tail of 1 to 64 rows, of 8 and 9 stages."""
    run([257 + 7 * i % 64 if i % 10 else 256 * (i % 3) for i in range(groups)], n, k, 1, 7.0)
