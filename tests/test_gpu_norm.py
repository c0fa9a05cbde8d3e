"""The root-mean-square norm and its gradient on the GPU against 64 bits.

Tolerances (u = 2^-24): a thread's squares are summed one after the other, d /
512 of them at most or 32, ten more additions join the threads'; all are
positive, so the mean is within (max(32, d / 512) + 13) u and its root within
half of that; the root's own roundings, the reciprocal and two products are 5 u.
y is then rounded once to its type.  The gradient's second sum has the same
additions over its parts' magnitudes, and some 8 roundings more.
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


def randn(g, *shape, type=0, scale=1.0):
    return (scale * torch.randn(*shape, generator=g)).to(F.DTYPE[type])


def within(d):
    return ((max(32, d / 512) + 13) / 2 + 5) * U


def near(got, want, bound, type):
    """got (of `type`) is want up to bound and one rounding."""
    slack = bound + F.ROUND[type] * (want.abs() + bound) + F.HALF_STEP[type]
    off = (got.double() - want).abs()
    assert bool((off <= slack).all()), float((off / slack).max())


SHAPES = [(1, 1), (1, 7), (2, 8), (3, 33), (5, 130), (4, 1024), (3, 2049), (2, 2816), (400, 300), (3, 2820), (3, 7168), (2, 8193), (2, 12288), (2, 16385),
          (300, 64)]


@pytest.mark.parametrize("rows,d", SHAPES)
@pytest.mark.parametrize("type", TYPES)
@pytest.mark.parametrize("add", [False, True])
def test_norm(rows, d, type, add):
    g = gen(rows * 7 + d)
    x, r, w = randn(g, rows, d, type=type, scale=2.0), randn(g, rows, d, type=type), 1.0 + 0.3 * torch.randn(d, generator=g)
    s = (x.float() + r.float()).to(F.DTYPE[type]) if add else x
    y, total = (torch.full((rows + 1, d), 9.0, dtype=F.DTYPE[type]).cuda() for _ in range(2))
    Q.rms_norm(type, x.cuda(), rows, d, w.cuda(), 1e-5, y, add=r.cuda() if add else None, sum=total)
    want = P.norm(s, w, 1e-5)
    assert torch.equal(total[:rows].cpu(), s) and bool((total[rows] == 9).all()) and bool((y[rows] == 9).all())
    near(y[:rows].cpu(), want, within(d) * want.abs(), type)


@pytest.mark.parametrize("rows,d", SHAPES)
@pytest.mark.parametrize("type", TYPES)
def test_norm_into_8_and_4_bits(rows, d, type):
    """With f32 activations y is what the codes are made of, so they are equal
    bit for bit to those of the y that comes with them; else their values are
    within half a step of it."""
    g = gen(rows * 11 + d)
    x, r, w = randn(g, rows, d, type=type, scale=2.0), randn(g, rows, d, type=type), 1.0 + 0.3 * torch.randn(d, generator=g)
    s = (x.float() + r.float()).to(F.DTYPE[type])
    want = P.norm(s, w, 1e-6)
    off = within(d) * want.abs()
    for bits in (8, 4):
        cols = d if bits == 8 else 16 * P.blocks(d)
        codes = torch.full((rows + 1, cols), 0x77, dtype=torch.uint8).cuda()
        scales = torch.full((rows + 1, F.blocks(d)), 3.0).cuda() if bits == 8 else \
            torch.full((rows + 1, P.blocks(d)), 3, dtype=torch.uint8).cuda()
        y, total = torch.empty(rows, d, dtype=F.DTYPE[type]).cuda(), torch.empty(rows, d, dtype=F.DTYPE[type]).cuda()
        f = Q.rms_norm_fp8 if bits == 8 else Q.rms_norm_fp4
        f(type, x.cuda(), rows, d, w.cuda(), 1e-6, codes, scales, add=r.cuda(), sum=total, y=y)
        assert torch.equal(total.cpu(), s)
        near(y.cpu(), want, off, type)
        c, z = codes[:rows].cpu(), scales[:rows].cpu()
        assert bool((codes[rows] == 0x77).all()) and bool((scales[rows] == 3).all())
        if type == 0:
            qc, qs = (F if bits == 8 else P).quantize(y.cpu())
            assert torch.equal(c, qc) and torch.equal(z, qs)
        elif bits == 8:
            v = F.values(c, z)
            assert bool(((v - want).abs() <= F.code_bound(want, z) * (1 + 2.0 ** -9) + 2 * off).all())
        else:
            # a block's largest magnitude lands in [4, 8) scales, or may be either side of a power of two
            v, size = P.values(c, z, d), torch.pow(2.0, z.double() - 127).repeat_interleave(32, 1)[:, :d]
            a = want.abs() / size
            step = torch.where(a < 2, 0.25, torch.where(a < 4, 0.5, 1.0)) * size
            step = torch.where(a > 6, (a - 6) * size, step)
            assert bool((a < 8 * (1 + 2.0 ** -12)).all()) and bool(((v - want).abs() <= step * (1 + 2.0 ** -9) + 2 * off).all())
        # without the extra outputs, the same codes
        codes2, scales2 = torch.zeros_like(codes), torch.zeros_like(scales)
        f(type, total, rows, d, w.cuda(), 1e-6, codes2, scales2)
        assert torch.equal(codes2[:rows].cpu(), c) and torch.equal(scales2[:rows].cpu(), z)


@pytest.mark.parametrize("type", TYPES)
@pytest.mark.parametrize("d", [40, 5000, 20000])
def test_norm_in_place_strided_and_unaligned(type, d):
    g = gen(d + type)
    rows, t = 5, F.DTYPE[type]
    x, r, w = randn(g, rows, d, type=type), randn(g, rows, d, type=type), torch.rand(d, generator=g) + 0.5
    s = (x.float() + r.float()).to(t)
    want = P.norm(s, w, 1e-5)
    ld = d + 3
    big = torch.full((rows * ld + 1,), 5.0, dtype=t).cuda()
    xs = big[1:].view(rows, ld)
    xs[:, :d] = x.cuda()
    total = r.cuda().clone()
    Q.rms_norm(type, xs, rows, d, w.cuda(), 1e-5, xs, add=total, sum=total, ld_x=ld, ld_y=ld)   # y over x, sum over add
    assert torch.equal(total.cpu(), s) and bool((xs[:, d:] == 5).all()) and float(big[0]) == 5
    near(xs[:, :d].cpu(), want, within(d) * want.abs(), type)
    Q.rms_norm(type, total, rows, d, w.cuda(), 1e-5, total)   # all in one place
    near(total.cpu(), want, within(d) * want.abs(), type)


def test_norm_of_zeros_large_and_not_finite():
    d = 300
    x = torch.zeros(5, d)
    x[1, 3] = float("inf")
    x[2, 4] = float("nan")
    x[3] = 1e15
    y = torch.empty(5, d).cuda()
    Q.rms_norm(0, x.cuda(), 5, d, None, 1e-5, y)
    y = y.cpu()
    assert bool((y[0] == 0).all()) and bool((y[4] == 0).all()) and bool(torch.isnan(y[2]).all())
    assert bool(torch.isnan(y[1, 3])) and bool((y[1, :3] == 0).all()) and bool(((y[3] - 1).abs() < 1e-5).all())
    codes, scales = torch.empty(5, 16 * P.blocks(d), dtype=torch.uint8).cuda(), torch.empty(5, P.blocks(d), dtype=torch.uint8).cuda()
    Q.rms_norm_fp4(0, x.cuda(), 5, d, None, 1e-5, codes, scales)
    assert scales[1].tolist() == [255] + [0] * 9 and scales[2].tolist() == [255] * 10 and scales[0].tolist() == [0] * 10
    assert bool((codes[0] == 0).all())


@pytest.mark.parametrize("rows,d", [(1, 1), (1, 7168), (2, 9), (3, 2816), (700, 300), (5, 2820), (7, 33), (700, 64), (149, 7168), (600, 1030), (5, 8200), (301, 8300)])
@pytest.mark.parametrize("type", TYPES)
@pytest.mark.parametrize("add", [False, True])
def test_gradient(rows, d, type, add):
    g = gen(rows * 3 + d)
    s, dy, r = randn(g, rows, d, type=type, scale=2.0), randn(g, rows, d, type=type), randn(g, rows, d, type=type)
    w = 1.0 + 0.3 * torch.randn(d, generator=g)
    dx, dw = torch.full((rows + 1, d), 9.0, dtype=F.DTYPE[type]).cuda(), torch.full((d + 1,), 9.0).cuda()
    n = Q.rms_norm_grad_work(rows, d)
    work = torch.full((n + 1,), float("nan")).cuda()
    args = dict(work=work, add=r.cuda() if add else None)
    Q.rms_norm_grad(type, dy.cuda(), s.cuda(), rows, d, w.cuda(), 1e-5, dx, dw=dw, **args)
    want, want_w, size, size_w = P.norm_grad(dy, s, w, 1e-5, r if add else None)
    assert bool((dx[rows] == 9).all()) and float(dw[d]) == 9 and bool(torch.isnan(work[n]))
    near(dx[:rows].cpu(), want, (3 * within(d) + 10 * U) * size, type)
    # a column's rows one after the other in a CTA, its parts in 16 runs: at most rows additions
    assert bool(((dw[:d].cpu().double() - want_w).abs() <= (within(d) + (rows + 4) * U) * size_w + 1e-300).all())
    again, dw2 = torch.empty_like(dx), torch.empty_like(dw)
    Q.rms_norm_grad(type, dy.cuda(), s.cuda(), rows, d, w.cuda(), 1e-5, again, dw=dw2, **args)
    assert torch.equal(again[:rows], dx[:rows]) and torch.equal(dw2[:d], dw[:d])
    Q.rms_norm_grad(type, dy.cuda(), s.cuda(), rows, d, w.cuda(), 1e-5, again, add=args["add"])   # dx alone
    assert torch.equal(again[:rows], dx[:rows])
    there = dy.cuda()
    Q.rms_norm_grad(type, there, s.cuda(), rows, d, w.cuda(), 1e-5, there, dw=dw2, **args)   # dx over dy
    assert torch.equal(there, dx[:rows]) and torch.equal(dw2[:d], dw[:d])


def test_gradient_against_differences():
    """Central differences of the 64-bit forward along random directions."""
    g = gen(3)
    rows, d, eps, h = 4, 96, 1e-5, 1e-6
    s, dy, w = randn(g, rows, d), randn(g, rows, d), 1.0 + 0.3 * torch.randn(d, generator=g)
    dx, dw, work = torch.empty(rows, d).cuda(), torch.empty(d).cuda(), torch.empty(Q.rms_norm_grad_work(rows, d)).cuda()
    Q.rms_norm_grad(0, dy.cuda(), s.cuda(), rows, d, w.cuda(), eps, dx, dw=dw, work=work)

    def loss(s, w):
        return float((P.norm(s, w, eps) * dy.double()).sum())

    for _ in range(3):
        a, b = torch.randn(rows, d, generator=g).double(), torch.randn(d, generator=g).double()
        by_s = (loss(s.double() + h * a, w.double()) - loss(s.double() - h * a, w.double())) / (2 * h)
        by_w = (loss(s.double(), w.double() + h * b) - loss(s.double(), w.double() - h * b)) / (2 * h)
        # the differences' own error: h^2 and 2^-53 / h, both below 1e-8 here
        assert abs(by_s - float((dx.cpu().double() * a).sum())) < 1e-4
        assert abs(by_w - float((dw.cpu().double() * b).sum())) < 1e-4


def test_no_rows():
    dw = torch.full((5,), 3.0).cuda()
    Q.rms_norm(0, None, 0, 5, None, 1e-5, None)
    Q.rms_norm_grad(0, None, None, 0, 5, None, 1e-5, None, dw=dw)
    assert dw.tolist() == [0.0] * 5


def test_norm_captured_and_on_another_stream():
    g = gen(5)
    rows, d = 33, 1024
    x, r, w = randn(g, rows, d, type=2).cuda(), randn(g, rows, d, type=2).cuda(), (torch.rand(d, generator=g) + 0.5).cuda()
    y, total, dx = torch.empty_like(x), torch.empty_like(x), torch.empty_like(x)
    dw, work = torch.empty(d).cuda(), torch.empty(Q.rms_norm_grad_work(rows, d)).cuda()
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()

    def call(stream):
        Q.rms_norm(2, x, rows, d, w, 1e-5, y, add=r, sum=total, stream=stream)
        Q.rms_norm_grad(2, y, total, rows, d, w, 1e-5, dx, dw=dw, work=work, add=r, stream=stream)

    with torch.cuda.stream(side):
        call(side.cuda_stream)
    side.synchronize()
    first = [t.clone() for t in (y, total, dx, dw)]
    with torch.cuda.graph(graph):
        call(torch.cuda.current_stream().cuda_stream)
    for k in range(2):
        x.copy_(randn(g, rows, d, type=2))
        graph.replay()
        torch.cuda.synchronize()
        now = [t.clone() for t in (y, total, dx, dw)]
        call(None)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(now, (y, total, dx, dw)))
        assert not torch.equal(now[0], first[0])
