"""The norm and its gradient where a CTA has many rows: its ring of rows goes
round several times, rows' ways out by shared memory are used again, the weight's
gradient is summed over all of them.  Tolerances are those of test_gpu_norm.py."""
import pytest

import qauntrunner_b200 as Q
from tests import fp4_plain as P
from tests import fp8_plain as F
from tests.test_gpu_norm import TYPES, U, gen, near, randn, within

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

# at least five rows for each of the 148 SMs' CTAs, and more rows than slots
SHAPES = [(5000, 1024), (12000, 64), (2000, 7168), (2000, 7001), (1500, 2819), (700, 8200), (1000, 12000)]


def case(rows, d, type, add=True):
    g = gen(rows + 5 * d + type)
    x, r, w = randn(g, rows, d, type=type, scale=2.0), randn(g, rows, d, type=type), 1.0 + 0.3 * torch.randn(d, generator=g)
    return x, r, w, (x.float() + r.float()).to(F.DTYPE[type]) if add else x


@pytest.mark.parametrize("rows,d", SHAPES)
@pytest.mark.parametrize("type", TYPES)
@pytest.mark.parametrize("add", [False, True])
def test_norm_in_place(rows, d, type, add):
    """The sum over the residual (or over x), then y over what was added to it, and everything in one place."""
    x, r, w, s = case(rows, d, type, add)
    want = P.norm(s, w, 1e-5)
    y, total = x.cuda(), r.cuda()
    if add:
        Q.rms_norm(type, y, rows, d, w.cuda(), 1e-5, y, add=total, sum=total)
        assert torch.equal(total.cpu(), s)
    else:
        Q.rms_norm(type, y, rows, d, w.cuda(), 1e-5, y)
    near(y.cpu(), want, within(d) * want.abs(), type)
    if add:
        y = x.cuda()
        Q.rms_norm(type, y, rows, d, w.cuda(), 1e-5, total, add=r.cuda(), sum=y)   # the sum over x, y elsewhere
        assert torch.equal(y.cpu(), s)
        near(total.cpu(), want, within(d) * want.abs(), type)
        Q.rms_norm(type, y, rows, d, w.cuda(), 1e-5, y)
        assert torch.equal(y, total)


@pytest.mark.parametrize("rows,d", SHAPES)
@pytest.mark.parametrize("type", TYPES)
@pytest.mark.parametrize("odd", [0, 1], ids=["aligned", "odd"])
def test_norm_into_8_and_4_bits(rows, d, type, odd):
    """Codes are those of the y that comes with them (f32), or of the plain norm's up to a step; odd: no row of the
    outputs starts on 16 bytes but by chance."""
    x, r, w, s = case(rows, d, type)
    want = P.norm(s, w, 1e-6)
    off = within(d) * want.abs()
    for bits in (8, 4):
        cols = d if bits == 8 else 16 * P.blocks(d)
        ld, ld_c = d + odd, cols + odd
        codes = torch.full((rows, ld_c), 0x77, dtype=torch.uint8).cuda()
        scales = torch.zeros(rows, F.blocks(d)).cuda() if bits == 8 else torch.zeros(rows, P.blocks(d), dtype=torch.uint8).cuda()
        y, total = (torch.full((rows, ld), 9.0, dtype=F.DTYPE[type]).cuda() for _ in range(2))
        f = Q.rms_norm_fp8 if bits == 8 else Q.rms_norm_fp4
        f(type, x.cuda(), rows, d, w.cuda(), 1e-6, codes, scales, add=r.cuda(), sum=total, y=y, ld_sum=ld, ld_y=ld, ld_codes=ld_c)
        assert torch.equal(total[:, :d].cpu(), s)
        assert bool((total[:, d:] == 9).all()) and bool((y[:, d:] == 9).all()) and bool((codes[:, cols:] == 0x77).all())
        y, c, z = y[:, :d].contiguous().cpu(), codes[:, :cols].contiguous().cpu(), scales.cpu()
        near(y, want, off, type)
        if type == 0:
            qc, qs = (F if bits == 8 else P).quantize(y)
            assert torch.equal(c, qc) and torch.equal(z, qs)
        elif bits == 8:
            v = F.values(c, z)
            assert bool(((v - want).abs() <= F.code_bound(want, z) * (1 + 2.0 ** -9) + 2 * off).all())
        else:   # (as in test_gpu_norm.py)
            v, size = P.values(c, z, d), torch.pow(2.0, z.double() - 127).repeat_interleave(32, 1)[:, :d]
            a = want.abs() / size
            step = torch.where(a < 2, 0.25, torch.where(a < 4, 0.5, 1.0)) * size
            step = torch.where(a > 6, (a - 6) * size, step)
            assert bool((a < 8 * (1 + 2.0 ** -12)).all()) and bool(((v - want).abs() <= step * (1 + 2.0 ** -9) + 2 * off).all())


@pytest.mark.parametrize("rows,d", SHAPES)
@pytest.mark.parametrize("type", TYPES)
@pytest.mark.parametrize("add", [False, True])
def test_gradient_over_each_of_its_inputs(rows, d, type, add):
    s, r, w, _ = case(rows, d, type, False)
    g = gen(rows + d)
    dy = randn(g, rows, d, type=type)
    want, want_w, size, size_w = P.norm_grad(dy, s, w, 1e-5, r if add else None)
    n = Q.rms_norm_grad_work(rows, d)
    dx, dw, work = torch.empty(rows, d, dtype=F.DTYPE[type]).cuda(), torch.empty(d).cuda(), torch.full((n + 1,), float("nan")).cuda()
    Q.rms_norm_grad(type, dy.cuda(), s.cuda(), rows, d, w.cuda(), 1e-5, dx, dw=dw, work=work, add=r.cuda() if add else None)
    assert bool(torch.isnan(work[n]))
    near(dx.cpu(), want, (3 * within(d) + 10 * U) * size, type)
    assert bool(((dw.cpu().double() - want_w).abs() <= (within(d) + (rows + 4) * U) * size_w + 1e-300).all())
    for over in ("dy", "x", "add")[:3 if add else 2]:
        a = {"dy": dy.cuda(), "x": s.cuda(), "add": r.cuda() if add else None}
        dw2 = torch.empty(d).cuda()
        Q.rms_norm_grad(type, a["dy"], a["x"], rows, d, w.cuda(), 1e-5, a[over], dw=dw2, work=work, add=a["add"])
        assert torch.equal(a[over], dx) and torch.equal(dw2, dw), over


@pytest.mark.parametrize("type", [0, 2])
def test_rows_that_start_anywhere(type):
    """Inputs and dx an odd number of values apart, off 16 bytes."""
    rows, d, ld = 2000, 1030, 1033
    x, r, w, s = case(rows, d, type)
    t = F.DTYPE[type]

    def apart(v):
        big = torch.full((rows * ld + 1,), 5.0, dtype=t).cuda()
        view = big[1:].view(rows, ld)
        if v is not None:
            view[:, :d] = v.cuda()
        return view

    xs, rs, ys, dx = apart(x), apart(r), apart(None), apart(None)
    Q.rms_norm(type, xs, rows, d, w.cuda(), 1e-5, ys, add=rs, sum=rs, ld_x=ld, ld_add=ld, ld_sum=ld, ld_y=ld)
    want = P.norm(s, w, 1e-5)
    assert torch.equal(rs[:, :d].cpu(), s) and bool((rs[:, d:] == 5).all()) and bool((ys[:, d:] == 5).all())
    near(ys[:, :d].cpu(), want, within(d) * want.abs(), type)
    want, want_w, size, size_w = P.norm_grad(x, s, w, 1e-5, None)
    dw, work = torch.empty(d).cuda(), torch.empty(Q.rms_norm_grad_work(rows, d)).cuda()
    Q.rms_norm_grad(type, xs, rs, rows, d, w.cuda(), 1e-5, dx, dw=dw, work=work, ld_dy=ld, ld_x=ld, ld_dx=ld)
    near(dx[:, :d].cpu(), want, (3 * within(d) + 10 * U) * size, type)
    assert bool((dx[:, d:] == 5).all())
    assert bool(((dw.cpu().double() - want_w).abs() <= (within(d) + (rows + 4) * U) * size_w + 1e-300).all())
