"""The 4-bit expert operators on the GPU against plain forms in 64 bits.

Tolerances (u = 2^-24):
* codes and scales of given values are exact, bit for bit;
* a product of two codes and two scales is exact, and so are sums as long as f32
  holds them: with scales of 2^-2 to 2^2 every term is a multiple of 2^-6, so
  sums below 2^18 are.  There the products in f32 are equal bit for bit, and in
  16 bits after their one rounding;
* where sums do not fit, each addition loses at most 2^-23 of the sum of the
  magnitudes, and there are K of them;
* SwiGLU: exp within 2 ulp, the other operations round once: 16 u of the value.
  Below a gate of -87 sigma is a denormal, a multiple of 2^-149: exp's 2 ulp, its
  correction and the product are 4 such steps, which |gate up| multiplies.
"""
import pytest

import qauntrunner_b200 as Q
from tests import fp4_plain as P
from tests import fp8_plain as F

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
U = F.U
TYPES = (0, 1, 2)


def gen(seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return g


def rows4(rows, cols, extra=0, fill=0x77):
    """Room for 4-bit rows, filled with something."""
    return (torch.full((rows, 16 * P.blocks(cols) + 16 * extra), fill, dtype=torch.uint8).cuda(),
            torch.full((rows, P.blocks(cols) + extra), fill, dtype=torch.uint8).cuda())


# ------------------------------------------------------------ rows into 4 bits

@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 31), (2, 32), (3, 33), (5, 70), (2, 1000), (7, 1091), (3, 7168), (2, 9000)])
@pytest.mark.parametrize("type", TYPES)
def test_quantize(rows, cols, type):
    g = gen(rows + 3 * cols)
    x = (torch.randn(rows, cols, generator=g) * torch.exp(3 * torch.randn(rows, cols, generator=g))).to(F.DTYPE[type])
    x[torch.rand(rows, cols, generator=g) < 0.1] = 0
    want = P.quantize(x)
    codes, scales = rows4(rows + 1, cols)
    Q.quantize_fp4(type, x.cuda(), rows, cols, codes, scales)
    assert torch.equal(codes[:rows].cpu(), want[0]) and torch.equal(scales[:rows].cpu(), want[1])
    assert bool((codes[rows] == 0x77).all()) and bool((scales[rows] == 0x77).all())
    # pitches, a start off any boundary, fewer rows by a number on the device
    ld = cols + 1
    big = torch.zeros(rows * ld + 1, dtype=F.DTYPE[type]).cuda()
    view = big[1:].view(rows, ld)
    view[:, :cols] = x.cuda()
    ld_c, ld_s = 16 * P.blocks(cols) + 3, P.blocks(cols) + 5
    cb, sb = (torch.full((rows * n + 1,), 0x77, dtype=torch.uint8).cuda() for n in (ld_c, ld_s))
    c, s = cb[1:].view(rows, ld_c), sb[1:].view(rows, ld_s)
    held = torch.tensor([rows - 1], dtype=torch.int32).cuda()
    Q.quantize_fp4(type, view, rows, cols, c, s, n_rows=held, ld_x=ld, ld_codes=ld_c, ld_scales=ld_s)
    assert torch.equal(c[:-1, :-3].cpu(), want[0][:-1]) and torch.equal(s[:-1, :-5].cpu(), want[1][:-1])
    assert bool((c[:, -3:] == 0x77).all()) and bool((s[:, -5:] == 0x77).all()) and bool((c[-1] == 0x77).all())


def test_quantize_every_middle_and_edge():
    """Ties, the largest and smallest exponents, denormals, zeros of both signs."""
    base = torch.tensor([0.0, 0.25, 0.5, 0.75, 1.0, 1.25, 1.5, 1.75, 2.0, 2.5, 3.0, 3.5, 4.0, 5.0, 6.0, 7.0, 7.9])
    near = torch.cat([base, torch.nextafter(base, torch.tensor(9.0)), torch.nextafter(base, torch.tensor(-9.0))])
    rows = []
    for e in (0, 1, -3, 60, -60, 125, -126, -140):
        for at in (0, 20):
            r = near[at:at + 30].clone()
            r = torch.cat([r, torch.tensor([4.0, -4.0])])
            rows.append(torch.ldexp(r.double(), torch.tensor(e)).float() * torch.where(torch.arange(32) % 2 == 1, -1.0, 1.0))
    rows.append(torch.zeros(32))
    rows.append(-torch.zeros(32))
    x = torch.stack(rows)
    x = torch.where(torch.isfinite(x), x, torch.tensor(3.4028234663852886e38))
    codes, scales = rows4(len(x), 32)
    Q.quantize_fp4(0, x.cuda(), len(x), 32, codes, scales)
    want = P.quantize(x)
    assert torch.equal(scales.cpu(), want[1]) and torch.equal(codes.cpu(), want[0])


def test_quantize_not_finite():
    x = torch.ones(2, 96)
    x[0, 40], x[1, 95] = float("nan"), float("-inf")
    codes, scales = rows4(2, 96)
    Q.quantize_fp4(0, x.cuda(), 2, 96, codes, scales)
    assert scales.tolist() == [[125, 255, 125], [125, 125, 255]]
    assert torch.equal(P.values(codes.cpu(), scales.cpu(), 96).isnan(), P.values(*P.quantize(x), 96).isnan())


@pytest.mark.parametrize("T,k,d,n_rows", [(1, 1, 32, 1), (1, 8, 7168, 8), (5, 2, 100, 10), (37, 6, 1000, 200), (9, 3, 33, 20)])
@pytest.mark.parametrize("type", TYPES)
def test_gather(T, k, d, n_rows, type):
    g = gen(T * k + d)
    x = torch.randn(T, d, generator=g).to(F.DTYPE[type])
    pos = torch.randperm(max(T * k, n_rows), generator=g)[:T * k].int()
    pos[torch.rand(T * k, generator=g) < 0.2] = -1
    codes, scales = rows4(n_rows, d)
    Q.gather_rows_fp4(type, x.cuda(), pos.cuda(), T, k, d, codes, scales, n_rows)
    c, s = (t.cpu() for t in rows4(n_rows, d))
    qc, qs = P.quantize(x)
    for a, r in enumerate(pos.tolist()):
        if 0 <= r < n_rows:
            c[r], s[r] = qc[a // k], qs[a // k]
    assert torch.equal(codes.cpu(), c) and torch.equal(scales.cpu(), s)


# ------------------------------------------------------------ products

class Case:
    """groups matrices, rows in 4 bits spread over them, and what comes out."""

    def __init__(self, rows, groups, n, k, spread=2, seed=0, even=False):
        g = gen(seed + rows * 3 + groups * 5 + n * 7 + k)
        self.rows, self.groups, self.n, self.k = rows, groups, n, k
        self.w = P.random_rows(g, groups * n, k, spread)
        self.x = P.random_rows(g, rows, k, spread)
        cut = torch.sort(torch.randint(0, rows + 1, (groups + 1,), generator=g)).values
        cut[0], cut[-1] = (0, rows) if groups == 1 or even else (cut[0], cut[-1])
        self.offsets = cut.int()
        w = P.values(*self.w, k).reshape(groups, n, k)
        x = P.values(*self.x, k)
        self.want, self.size = torch.full((rows, n), float("nan"), dtype=torch.float64), torch.zeros(rows, n, dtype=torch.float64)
        for i in range(groups):
            a, b = int(cut[i]), int(cut[i + 1])
            self.want[a:b] = x[a:b] @ w[i].T
            self.size[a:b] = x[a:b].abs() @ w[i].abs().T
        self.inside = ~self.want.isnan().any(1)

    def matrix(self):
        return Q.Fp4Matrix(self.n, self.k, self.w[0].cuda(), self.w[1].cuda(), groups=self.groups)


@pytest.fixture(params=["0", "1", None], ids=["split", "pair", "chosen"])
def form(request, monkeypatch):
    if request.param is None:
        monkeypatch.delenv("QRM_FP4_PAIR", raising=False)
    else:
        monkeypatch.setenv("QRM_FP4_PAIR", request.param)
    return request.param


SIZES = [(1, 1, 1, 1), (1, 1, 128, 32), (2, 1, 16, 256), (1, 1, 300, 2048), (3, 1, 257, 96), (17, 1, 130, 70), (16, 4, 128, 512),
         (64, 2, 384, 500), (65, 1, 256, 320), (200, 3, 304, 1000), (129, 7, 72, 1056), (257, 1, 520, 288), (530, 5, 640, 768),
         (5, 40, 40, 64), (300, 33, 136, 4096), (385, 1, 264, 544), (800, 3, 130, 300), (1500, 2, 72, 800)]


def check(got, want, inside, type, untouched):
    got = got.cpu()
    assert torch.equal(got[inside], want[inside].to(F.DTYPE[type])), \
        float((got[inside].double() - want[inside]).abs().max())
    assert bool((got[~inside] == untouched).all())


@pytest.mark.parametrize("rows,groups,n,k", SIZES)
def test_product_is_exact(rows, groups, n, k, form):
    c = Case(rows, groups, n, k)
    assert float(c.size.max()) < 2 ** 18
    m = c.matrix()
    for type in TYPES:
        y = torch.full((rows + 1, n), 5.0, dtype=F.DTYPE[type]).cuda()
        m.product(type, c.x[0].cuda(), c.x[1].cuda(), rows, y, offsets=c.offsets.cuda() if groups > 1 else None)
        m.sync()
        # (64 bits to 16 by way of f32, as the kernel does)
        check(y[:rows], c.want.float(), c.inside, type, 5.0)
        assert bool((y[rows] == 5).all())
    m.close()


@pytest.mark.parametrize("rows,groups,n,k", [(1, 1, 256, 7168), (16, 3, 200, 4000), (300, 2, 520, 2048)])
def test_product_of_wide_scales(rows, groups, n, k, form):
    """Scales over 2^-20 to 2^20: sums that f32 does not hold."""
    c = Case(rows, groups, n, k, spread=20)
    m = c.matrix()
    y = torch.full((rows, n), 5.0).cuda()
    m.product(0, c.x[0].cuda(), c.x[1].cuda(), rows, y, offsets=c.offsets.cuda())
    m.sync()
    off = (y.cpu().double() - c.want).abs()[c.inside]
    assert bool((off <= k * 2.0 ** -23 * c.size[c.inside]).all()), float((off / c.size[c.inside]).max())
    m.close()


GATED = [(1, 1, 1, 32), (1, 1, 16, 256), (1, 1, 128, 2048), (3, 1, 33, 96), (17, 1, 100, 70), (16, 4, 128, 512), (64, 2, 200, 500),
         (200, 3, 152, 1000), (257, 1, 384, 288), (530, 5, 320, 768), (5, 40, 40, 64), (700, 2, 80, 544)]


@pytest.mark.parametrize("rows,groups,f,k", GATED)
@pytest.mark.parametrize("limit", [0.0, 7.0])
def test_gated(rows, groups, f, k, limit, form):
    c = Case(rows, groups, 2 * f, k, spread=2)
    # sums of some hundreds; a quarter of the rows far smaller, where the gate's curve is
    c.x[1][::4] -= 8
    c.want[::4] *= 2.0 ** -8
    m = c.matrix()
    h64, parts = P.gate(c.want, limit), (c.want[:, :f] * c.want[:, f:]).abs()
    off = c.offsets.cuda() if groups > 1 else None
    for type in TYPES:
        h = torch.full((rows + 1, f), 5.0, dtype=F.DTYPE[type]).cuda()
        m.swiglu(type, c.x[0].cuda(), c.x[1].cuda(), rows, h, offsets=off, limit=limit)
        m.sync()
        got = h.cpu()
        assert bool((got[:rows][~c.inside] == 5).all()) and bool((got[rows] == 5).all())
        want, got = h64[c.inside], got[:rows][c.inside].double()
        slack = 16 * U * want.abs() + 4 * 2.0 ** -149 * parts[c.inside]
        slack = slack + F.ROUND[type] * (want.abs() + slack) + F.HALF_STEP[type]
        top = float(torch.finfo(F.DTYPE[type]).max)
        fits = want.abs() < top * (1 - 2.0 ** -10)
        assert bool(((got - want).abs() <= slack)[fits].all())
        if type == 0:
            h32 = h[:rows].cpu()
    # the same in 4-bit rows: the codes of the f32 values
    codes, scales = rows4(rows + 1, f)
    m.swiglu_fp4(c.x[0].cuda(), c.x[1].cuda(), rows, codes, scales, offsets=off, limit=limit)
    m.sync()
    qc, qs = P.quantize(h32)
    i = c.inside
    assert torch.equal(scales[:rows].cpu()[i], qs[i]) and torch.equal(codes[:rows].cpu()[i], qc[i])
    assert bool((codes[:rows].cpu()[~i] == 0x77).all()) and bool((scales[:rows].cpu()[~i] == 0x77).all())
    assert bool((codes[rows] == 0x77).all()) and bool((scales[rows] == 0x77).all())
    m.close()


@pytest.mark.parametrize("rows", [5, 200])
@pytest.mark.parametrize("type", TYPES)
def test_pitches_and_alignment(rows, type, form):
    """Rows of everything further apart than dense, outputs and scales that start off any boundary."""
    n, k = 136, 200
    c = Case(rows, 1, n, k)
    m = c.matrix()
    xc, xs = rows4(rows, k, extra=2)
    xc[:, :16 * P.blocks(k)] = c.x[0].cuda()
    for ld_s, at in ((P.blocks(k) + 2, 0), (P.blocks(k) + 2, 1), (16, 0), (16, 8)):
        buf = torch.full((rows * ld_s + 64,), 255, dtype=torch.uint8).cuda()
        xs = buf[at:at + rows * ld_s].view(rows, ld_s)
        xs[:, :P.blocks(k)] = c.x[1].cuda()
        for ld_y, first in ((n, 0), (n + 1, 0), (n + 8, 0), (n + 8, 1), (n + 24, 8)):
            y = torch.full((rows * ld_y + 64,), 5.0, dtype=F.DTYPE[type]).cuda()
            view = y[first:first + rows * ld_y].view(rows, ld_y)
            m.product(type, xc, xs, rows, view, ld_x=xc.shape[1], ld_scales=ld_s, ld_y=ld_y)
            check(view[:, :n], c.want.float(), c.inside, type, 5.0)
            assert bool((view[:, n:] == 5).all()) and bool((y[:first] == 5).all()) and bool((y[first + rows * ld_y:] == 5).all())
    m.sync()
    m.close()


def test_tails_hold_anything(form):
    """Bytes past the last column of the rows and of the matrix count nothing:
    codes there are cleared in the matrix, scales of x are not read."""
    rows, n, k = 70, 96, 70
    c = Case(rows, 1, n, k)
    dirty_w, dirty_x = c.w[0].clone(), c.x[0].clone()
    for t in (dirty_w, dirty_x):
        t[:, k // 2:] = 0x7F
    m = Q.Fp4Matrix(n, k, dirty_w.cuda(), c.w[1].cuda())
    xs = torch.full((rows, 16), 255, dtype=torch.uint8).cuda()
    xs[:, :P.blocks(k)] = c.x[1].cuda()
    y = torch.empty(rows, n).cuda()
    m.product(0, dirty_x.cuda(), xs, rows, y, ld_scales=16)
    check(y, c.want.float(), c.inside, 0, 0)
    m.close()


def test_not_a_number_stays_in_its_row_and_output(form):
    rows, n, k = 150, 200, 512
    c = Case(rows, 1, n, k)
    c.x[1][3, 5] = 255
    c.w[1][17, 2] = 255
    m = c.matrix()
    y = torch.empty(rows, n).cuda()
    m.product(0, c.x[0].cuda(), c.x[1].cuda(), rows, y)
    y = y.cpu()
    assert bool(y[3].isnan().all()) and bool(y[:, 17].isnan().all())
    keep = torch.ones(rows, n, dtype=torch.bool)
    keep[3], keep[:, 17] = False, False
    assert torch.equal(y[keep], c.want.float()[keep])
    m.close()


@pytest.mark.parametrize("offsets,bad", [([0, 3, 3, 10], []), ([2, 5, 4, 10], [1, 2]), ([0, -1, 4, 10], [0, 1]),
                                         ([0, 4, 10, 11], [2]), ([5, 8, 2, 6], [1, 2]), ([10, 10, 10, 10], [])])
def test_offsets_that_make_no_sense(offsets, bad, form):
    """Such a group counts as empty, and sync says so; the others come out."""
    c = Case(10, 3, 64, 256)
    w, x = P.values(*c.w, 256).reshape(3, 64, 256), P.values(*c.x, 256)
    want = torch.full((10, 64), 5.0, dtype=torch.float64)
    for g in range(3):
        if g not in bad:
            a, b = offsets[g], offsets[g + 1]
            want[a:b] = x[a:b] @ w[g].T
    m = c.matrix()
    y = torch.full((10, 64), 5.0).cuda()
    m.product(0, c.x[0].cuda(), c.x[1].cuda(), 10, y, offsets=torch.tensor(offsets, dtype=torch.int32).cuda())
    if bad:
        with pytest.raises(Q.QrmError) as e:
            m.sync()
        assert e.value.code == Q.E_INVALID
    m.sync()
    assert torch.equal(y.cpu(), want.float())
    m.close()


@pytest.mark.parametrize("offsets,bad", [([3, 9], False), ([4, 4], False), ([0, 11], True), ([6, 2], True), ([-1, 5], True)])
def test_one_group_of_some_rows(offsets, bad, form):
    """One matrix, whose weights are asked for before the offsets are known."""
    c = Case(10, 1, 96, 2100)
    m = c.matrix()
    y = torch.full((10, 96), 5.0).cuda()
    m.product(0, c.x[0].cuda(), c.x[1].cuda(), 10, y, offsets=torch.tensor(offsets, dtype=torch.int32).cuda())
    want = torch.full((10, 96), 5.0)
    if bad:
        with pytest.raises(Q.QrmError) as e:
            m.sync()
        assert e.value.code == Q.E_INVALID
    else:
        m.sync()
        a, b = offsets
        want[a:b] = c.want.float()[a:b]
    assert torch.equal(y.cpu(), want)
    m.close()


@pytest.mark.parametrize("offsets", [[5, 140], [0, 150], [149, 150], [70, 70], [0, 64], [16, 81]])
def test_one_group_of_many_rows(offsets, form):
    """Several tiles of rows and of outputs, some of them empty; the product and the gated one."""
    c = Case(150, 1, 700, 1300)
    assert float(c.size.max()) < 2 ** 18
    m = c.matrix()
    off = torch.tensor(offsets, dtype=torch.int32).cuda()
    y = torch.full((150, 700), 5.0).cuda()
    m.product(0, c.x[0].cuda(), c.x[1].cuda(), 150, y, offsets=off)
    h, every = torch.full((150, 350), 5.0).cuda(), torch.empty(150, 350).cuda()
    m.swiglu(0, c.x[0].cuda(), c.x[1].cuda(), 150, h, offsets=off)
    m.swiglu(0, c.x[0].cuda(), c.x[1].cuda(), 150, every)
    m.sync()
    inside = torch.zeros(150, dtype=torch.bool)
    inside[offsets[0]:offsets[1]] = True
    check(y, c.want.float(), inside, 0, 5.0)
    h, every = h.cpu(), every.cpu()
    want = P.gate(c.want, 0.0)
    slack = 16 * U * want.abs() + 4 * 2.0 ** -149 * (c.want[:, :350] * c.want[:, 350:]).abs()
    slack = slack + F.ROUND[0] * (want.abs() + slack) + F.HALF_STEP[0]   # (as in test_gated)
    assert bool(((every.double() - want).abs() <= slack).all())
    assert torch.equal(h[inside], every[inside]) and bool((h[~inside] == 5).all())
    m.close()


@pytest.mark.parametrize("first,second", [(0, 1), (3, 37), (31, 32), (38, 39)])
@pytest.mark.parametrize("type", TYPES)
def test_two_groups_of_forty(first, second, type, form):
    """Room for 120 rows, 50 of them held, the rest and the other groups without any."""
    c = Case(120, 40, 300, 520)
    w, x = P.values(*c.w, 520).reshape(40, 300, 520), P.values(*c.x, 520)
    offsets = torch.zeros(41, dtype=torch.int32)
    offsets[first + 1:] = 33
    offsets[second + 1:] = 50
    want = torch.full((120, 300), 5.0, dtype=torch.float64)
    want[:33], want[33:50] = x[:33] @ w[first].T, x[33:50] @ w[second].T
    assert float((x[:50].abs() @ w[[first, second]].abs().reshape(600, 520).T).max()) < 2 ** 18
    m = c.matrix()
    y = torch.full((120, 300), 5.0, dtype=F.DTYPE[type]).cuda()
    m.product(type, c.x[0].cuda(), c.x[1].cuda(), 120, y, offsets=offsets.cuda())
    m.sync()
    assert torch.equal(y.cpu(), want.float().to(F.DTYPE[type]))   # (sums are exact in f32: see test_product_is_exact)
    m.close()


# groups of whole tiles of 256 rows and a few more, of tiles without more, of one row, of none
TAILS = [[257, 288, 256, 320], [321, 0, 576, 1, 577], [300, 300], [64, 1000, 319]]


@pytest.mark.parametrize("sizes", TAILS, ids=str)
@pytest.mark.parametrize("odd", [0, 1], ids=["aligned", "odd"])
@pytest.mark.parametrize("n,k", [(300, 1900), (256, 2304), (130, 4100)])
def test_few_rows_behind_a_tile(sizes, odd, n, k, form):
    """Products and gated ones; odd: rows of scales and outputs that start anywhere."""
    T, f = sum(sizes), n // 2
    c = Case(T, len(sizes), n, k, spread=1)
    offsets = torch.tensor([0] + sizes).cumsum(0)
    w, x = P.values(*c.w, k).reshape(len(sizes), n, k), P.values(*c.x, k)
    want = torch.cat([x[offsets[i]:offsets[i + 1]] @ w[i].T for i in range(len(sizes))])
    assert max(float((x[offsets[i]:offsets[i + 1]].abs() @ w[i].abs().T).max()) for i in range(len(sizes)) if sizes[i]) < 2 ** 18
    off, m = offsets.int().cuda(), c.matrix()
    codes, scales = c.x[0].cuda(), torch.zeros(T, c.x[1].shape[1] + odd, dtype=torch.uint8).cuda()
    scales[:, :c.x[1].shape[1]] = c.x[1].cuda()
    ld = scales.shape[1]
    for type in TYPES:
        y = torch.full((T + 1, n + odd), 5.0, dtype=F.DTYPE[type]).cuda()
        m.product(type, codes, scales, T, y, offsets=off, ld_scales=ld, ld_y=n + odd)
        m.sync()
        assert torch.equal(y[:T, :n].cpu(), want.float().to(F.DTYPE[type]))
        assert bool((y[T] == 5).all()) and bool((y[:, n:] == 5).all())
    # (gates of up to some tens, so that a rounding of the product is within the test's slack)
    scales = (scales.int() - 4).to(torch.uint8)
    want = want / 16
    h = torch.full((T + 1, f + odd), 5.0).cuda()
    m.swiglu(0, codes, scales, T, h, offsets=off, limit=7.0, ld_scales=ld, ld_h=f + odd)
    c4, s4 = rows4(T + 1, f)
    m.swiglu_fp4(codes, scales, T, c4, s4, offsets=off, limit=7.0, ld_xs=ld)
    m.sync()
    h, gated = h.cpu(), P.gate(want, 7.0)
    slack = 16 * U * gated.abs() + 4 * 2.0 ** -149 * (want[:, :f] * want[:, f:2 * f]).abs()
    slack = slack + F.ROUND[0] * (gated.abs() + slack) + F.HALF_STEP[0]   # (as in test_gated)
    assert bool(((h[:T, :f].double() - gated).abs() <= slack).all())
    assert bool((h[T] == 5).all()) and bool((h[:, f:] == 5).all())
    qc, qs = P.quantize(h[:T, :f].contiguous())
    assert torch.equal(c4[:T].cpu(), qc) and torch.equal(s4[:T].cpu(), qs)
    assert bool((c4[T] == 0x77).all()) and bool((s4[T] == 0x77).all())
    m.close()


@pytest.mark.parametrize("groups", [100, 300])
def test_many_groups_with_a_few_rows_behind_a_tile(groups, form):
    """(300: a table of groups that leaves less shared memory for the products' stages)"""
    sizes = [257 + i % 70 if i % 2 else i % 100 for i in range(groups)]
    T, n, k = sum(sizes), 48, 1800
    c = Case(T, groups, n, k, spread=1)
    w, x = P.values(*c.w, k).reshape(groups, n, k), P.values(*c.x, k)
    offsets = torch.tensor([0] + sizes).cumsum(0)
    want = torch.cat([x[offsets[i]:offsets[i + 1]] @ w[i].T for i in range(groups)])
    assert T > 128 * groups and float((x.abs() @ w.abs().amax(0).T).max()) < 2 ** 18
    m = c.matrix()
    y = torch.empty(T, n).cuda()
    m.product(0, c.x[0].cuda(), c.x[1].cuda(), T, y, offsets=offsets.int().cuda())
    m.sync()
    assert torch.equal(y.cpu(), want.float())
    m.close()


def test_many_groups():
    """1024 matrices, most without rows."""
    c = Case(40, 1024, 32, 64)
    m = c.matrix()
    y = torch.full((40, 32), 5.0).cuda()
    m.product(0, c.x[0].cuda(), c.x[1].cuda(), 40, y, offsets=c.offsets.cuda())
    m.sync()
    check(y, c.want.float(), c.inside, 0, 5.0)
    m.close()


def test_host_arrays_give_the_same_matrix():
    c = Case(9, 2, 100, 90, even=True)
    outs = []
    for w in ((c.w[0].cuda(), c.w[1].cuda()), (c.w[0], c.w[1]), (c.w[0].numpy(), c.w[1].numpy())):
        m = Q.Fp4Matrix(100, 90, *w, groups=2)
        y = torch.empty(9, 100).cuda()
        m.product(0, c.x[0].cuda(), c.x[1].cuda(), 9, y, offsets=c.offsets.cuda())
        m.sync()
        outs.append(y.cpu())
        m.close()
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])


def test_calls_on_two_streams_and_captured(form):
    """Calls of one matrix at the same time, on two streams and in two graphs."""
    cases = [Case(rows, 3, 512, 2048, spread=1, seed=s, even=True) for s, rows in enumerate((40, 300, 1000))]
    cases[2].offsets = torch.tensor([0, 300, 620, 1000], dtype=torch.int32)   # (with a few rows behind a tile)
    m = cases[0].matrix()
    for c in cases[1:]:   # the same matrix
        x, w = P.values(*c.x, c.k), P.values(*cases[0].w, c.k).reshape(3, 512, c.k)
        for i in range(3):
            a, b = int(c.offsets[i]), int(c.offsets[i + 1])
            c.want[a:b] = x[a:b] @ w[i].T
            assert a == b or float((x[a:b].abs() @ w[i].abs().T).max()) < 2 ** 18
    ins = [(c.x[0].cuda(), c.x[1].cuda(), c.offsets.cuda()) for c in cases]
    outs = [torch.zeros(c.rows, c.n).cuda() for c in cases]
    streams, graphs = [torch.cuda.Stream() for _ in cases], [torch.cuda.CUDAGraph() for _ in cases]
    torch.cuda.synchronize()

    def call(i, stream):
        m.product(0, ins[i][0], ins[i][1], cases[i].rows, outs[i], offsets=ins[i][2], stream=stream)

    for _ in range(20):
        for i, s in enumerate(streams):
            call(i, s.cuda_stream)
    m.sync()
    for c, y in zip(cases, outs):
        check(y, c.want.float(), c.inside, 0, 0.0)
        y.zero_()
    for i, gr in enumerate(graphs):
        with torch.cuda.graph(gr):
            call(i, torch.cuda.current_stream().cuda_stream)
    for _ in range(5):
        for s, gr in zip(streams, graphs):
            with torch.cuda.stream(s):
                gr.replay()
    m.sync()
    for c, y in zip(cases, outs):
        check(y, c.want.float(), c.inside, 0, 0.0)
    m.close()
