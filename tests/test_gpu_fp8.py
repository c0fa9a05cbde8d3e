"""The 8-bit expert operators on the GPU against plain forms in 64 bits.

Tolerances, from the formats and the operations' order (u = 2^-24):
* order and codes of given values are exact: each step is exact or one IEEE
  operation, so the codes and scales are equal bit for bit;
* a sum of n products in f32 is within (n + 1) u times the sum of their
  magnitudes, plus one rounding to the result's type (2^-p of the value, or
  half the distance of the type's denormals);
* a product's inner sums over a block of 128 may truncate (2^-23 for each
  addition), its outer sum over the blocks rounds (u each), and the two scales
  are multiplied before (2 u);
* SwiGLU: exp is within 2 ulp, the other operations round once: 16 u of the
  value (of the parts of the sum, for the gate's gradient), then half the
  distance between neighbouring codes.
"""
import numpy as np
import pytest

import qauntrunner_b200 as Q
from tests import fp8_plain as F

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
F32, F16, BF16 = 0, 1, 2
TYPES = (F32, F16, BF16)
U = F.U


def gen(seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return g


def cuda(a):
    return a.cuda()


def randn(g, *shape, type=F32):
    return torch.randn(*shape, generator=g).to(F.DTYPE[type])


def pitched(a, extra, fill=float("nan")):
    """a's rows `extra` values apart from dense, the gap filled; (view, pitch)."""
    rows, cols = a.shape
    big = torch.full((rows, cols + extra), fill, dtype=torch.float32).to(a.dtype) if a.dtype != torch.uint8 else \
        torch.full((rows, cols + extra), 0x7F, dtype=torch.uint8)
    big[:, :cols] = a
    return big.cuda(), cols + extra


# ------------------------------------------------------------ order

@pytest.mark.parametrize("T,k,experts,first", [
    (0, 8, 256, 0), (1, 1, 1, 0), (1, 8, 256, 0), (3, 2, 8, 0), (37, 6, 64, 16), (511, 8, 256, 0), (513, 8, 1024, 5),
    (600, 8, 7, 0), (4096, 8, 256, 32), (4099, 7, 160, 0)])
def test_sort_tokens(T, k, experts, first):
    g = gen(T * 31 + k)
    idx = torch.randint(first - 2, first + experts + 2, (T, k), generator=g, dtype=torch.int32)
    n = T * k
    perm, pos = (torch.full((n + 1,), 77, dtype=torch.int32).cuda() for _ in range(2))
    off = torch.full((experts + 2,), 77, dtype=torch.int32).cuda()
    Q.sort_tokens(idx.cuda(), T, k, experts, perm, pos, off, first=first)
    torch.cuda.synchronize()
    want = F.order(idx, first, experts)
    assert perm.tolist() == want[0] + [77]
    assert pos.tolist() == want[1] + [77]
    assert off.tolist() == want[2] + [77]


def test_sort_tokens_none_held_and_all_one_expert():
    T, k = 700, 8
    for idx, experts in ((torch.full((T, k), -1, dtype=torch.int32), 16), (torch.full((T, k), 3, dtype=torch.int32), 16)):
        perm, pos = (torch.empty(T * k, dtype=torch.int32).cuda() for _ in range(2))
        off = torch.empty(experts + 1, dtype=torch.int32).cuda()
        Q.sort_tokens(idx.cuda(), T, k, experts, perm, pos, off)
        want = F.order(idx, 0, experts)
        assert (perm.tolist(), pos.tolist(), off.tolist()) == want


# ------------------------------------------------------------ rows out and back

def routed(g, T, k, n_rows, held=0.8):
    """Distinct rows for a share of the T k assignments, -1 for the others."""
    pos = torch.randperm(n_rows, generator=g)[: T * k]
    pos = torch.where(torch.rand(T * k, generator=g) < held, pos, torch.full_like(pos, -1))
    return pos.int()


SHAPES = [(1, 1, 1), (1, 8, 7168), (3, 2, 7), (5, 6, 130), (9, 8, 1536), (33, 3, 1001), (130, 2, 384)]


@pytest.mark.parametrize("T,k,d", SHAPES)
@pytest.mark.parametrize("type", TYPES)
@pytest.mark.parametrize("extra", [0, 3, 16])
def test_gather_rows(T, k, d, type, extra):
    g = gen(T + d + extra)
    x, n = randn(g, T, d, type=type), T * k + 2
    pos = routed(g, T, k, n)
    xd, ld = pitched(x, extra)
    rows = torch.full((n, d + extra), 5.0, dtype=x.dtype).cuda()
    Q.gather_rows(type, xd, pos.cuda(), T, k, d, rows, n, ld_x=ld, ld_rows=d + extra)
    codes = torch.full((n, d + extra), 9, dtype=torch.uint8).cuda()
    scales = torch.full((n, F.blocks(d) + extra), 5.0).cuda()
    Q.gather_rows_fp8(type, xd, pos.cuda(), T, k, d, codes, scales, n, ld_x=ld, ld_codes=d + extra,
                      ld_scales=F.blocks(d) + extra)
    want = torch.full((n, d + extra), 5.0, dtype=x.dtype)
    c1, s1 = F.quantize(x)
    want_c, want_s = torch.full((n, d + extra), 9, dtype=torch.uint8), torch.full((n, F.blocks(d) + extra), 5.0)
    for a, p in enumerate(pos.tolist()):
        if p >= 0:
            want[p, :d], want_c[p, :d], want_s[p, :F.blocks(d)] = x[a // k], c1[a // k], s1[a // k]
    assert torch.equal(rows.cpu(), want)
    assert torch.equal(codes.cpu(), want_c)
    assert torch.equal(scales.cpu(), want_s)


def test_gather_rows_passes_over_rows_outside():
    g = gen(3)
    x = randn(g, 2, 64)
    pos = torch.tensor([0, 9, -5, 2], dtype=torch.int32)
    rows = torch.zeros(4, 64).cuda()   # two of its rows are n_rows
    Q.gather_rows(F32, x.cuda(), pos.cuda(), 2, 2, 64, rows, 2)
    assert torch.equal(rows.cpu()[0], x[0]) and float(rows[1:].abs().max()) == 0.0


@pytest.mark.parametrize("T,k,d", SHAPES)
@pytest.mark.parametrize("type", TYPES)
@pytest.mark.parametrize("extra,with_w,with_add", [(0, True, True), (3, True, False), (16, False, True), (0, False, False)])
def test_combine_rows(T, k, d, type, extra, with_w, with_add):
    g = gen(T + 2 * d + extra)
    n = T * k + 1
    rows, add = randn(g, n, d, type=type), randn(g, T, d, type=type)
    w = torch.randn(T, k, generator=g)
    pos = routed(g, T, k, n)
    if T > 2:
        pos[:k] = -1   # a token without any row
    rd, ld = pitched(rows, extra)
    ad, _ = pitched(add, extra)
    out = torch.full((T, d + extra), 5.0, dtype=rows.dtype).cuda()
    Q.combine_rows(type, rd, n, pos.cuda(), w.cuda() if with_w else None, T, k, d, out, add=ad if with_add else None,
                   ld_rows=ld, ld_add=ld, ld_out=d + extra)
    want, size = F.combine(rows, pos.reshape(T, k), w if with_w else None, add if with_add else None)
    got = out.cpu().double()
    assert bool((got[:, d:] == 5.0).all())
    assert bool(((got[:, :d] - want).abs() <= (k + 1) * U * size + F.ROUND[type] * (want.abs() + (k + 1) * U * size)
                 + F.HALF_STEP[type]).all())
    # in place on the residual stream
    if with_add and not extra:
        Q.combine_rows(type, rd, n, pos.cuda(), w.cuda() if with_w else None, T, k, d, ad, add=ad)
        assert torch.equal(ad, out)


@pytest.mark.parametrize("T,k,d", SHAPES + [(2, 17, 256), (2, 8, 9000)])
@pytest.mark.parametrize("type", TYPES)
@pytest.mark.parametrize("extra", [0, 3])
def test_combine_rows_grad(T, k, d, type, extra):
    g = gen(T + 3 * d + extra)
    n = T * k + 1
    rows, dout, w = randn(g, n, d, type=type), randn(g, T, d, type=type), torch.randn(T, k, generator=g)
    pos = routed(g, T, k, n)
    if T > 2:
        pos[:k] = -1
    rd, ld = pitched(rows, extra)
    gd, _ = pitched(dout, extra)
    drows = torch.full((n, d + extra), 5.0, dtype=rows.dtype).cuda()
    codes, scales = torch.full((n, d + extra), 9, dtype=torch.uint8).cuda(), torch.full((n, F.blocks(d)), 5.0).cuda()
    dw, dw8 = (torch.full((T, k), 7.0).cuda() for _ in range(2))
    Q.combine_rows_grad(type, gd, rd, n, pos.cuda(), w.cuda(), T, k, d, drows, dw, ld_dout=ld, ld_rows=ld, ld_drows=d + extra)
    Q.combine_rows_grad_fp8(type, gd, rd, n, pos.cuda(), w.cuda(), T, k, d, codes, scales, dw8, ld_dout=ld, ld_rows=ld,
                            ld_codes=d + extra)
    want = torch.full((n, d + extra), 5.0, dtype=rows.dtype)
    want_c, want_s = torch.full((n, d + extra), 9, dtype=torch.uint8), torch.full((n, F.blocks(d)), 5.0)
    want_dw, size = torch.zeros(T, k, dtype=torch.float64), torch.zeros(T, k, dtype=torch.float64)
    for a, p in enumerate(pos.tolist()):
        if p < 0:
            continue
        t, j = a // k, a % k
        v = w[t, j] * dout[t].float()   # one f32 rounding
        want[p, :d] = v.to(rows.dtype)
        c, s = F.quantize(v[None])
        want_c[p, :d], want_s[p] = c[0], s[0]
        want_dw[t, j] = (dout[t].double() * rows[p].double()).sum()
        size[t, j] = (dout[t].double() * rows[p].double()).abs().sum()
    assert torch.equal(drows.cpu(), want)
    assert torch.equal(codes.cpu(), want_c)
    assert torch.equal(scales.cpu(), want_s)
    for got in (dw, dw8):
        assert bool(((got.cpu().double() - want_dw).abs() <= (d + 1) * U * size).all())
    if T > 2:
        assert bool((dw[0] == 0).all())


def test_combine_grad_is_the_derivative():
    """Differences of combine_rows along a direction of (rows, w) against the gradient's."""
    g = gen(11)
    T, k, d = 6, 4, 200
    n = T * k
    rows, w, dout = randn(g, n, d), torch.randn(T, k, generator=g), randn(g, T, d)
    vr, vw = randn(g, n, d), torch.randn(T, k, generator=g)
    pos = routed(g, T, k, n).cuda()

    def loss(h):   # <dout, combine> at (rows + h vr, w + h vw)
        out = torch.empty(T, d).cuda()
        Q.combine_rows(F32, (rows + h * vr).cuda(), n, pos, (w + h * vw).cuda(), T, k, d, out)
        return float((out.cpu().double() * dout.double()).sum())

    drows, dw = torch.zeros(n, d).cuda(), torch.empty(T, k).cuda()
    Q.combine_rows_grad(F32, dout.cuda(), rows.cuda(), n, pos, w.cuda(), T, k, d, drows, dw)
    along = float((drows.cpu().double() * vr.double()).sum() + (dw.cpu().double() * vw.double()).sum())
    # the loss is bilinear, so the symmetric difference has no truncation error; f32 rounding of
    # some T d k terms of size ~1 each: 1e-5 of their root-sum-square, over h = 0.5
    assert abs((loss(0.5) - loss(-0.5)) - along) <= 1e-5 * (T * d * k) ** 0.5 * 8
    # without weights combine_rows is the gradient of gather_rows: <gather(x), r> = <x, combine(r)>
    x, out, r = randn(g, T, d), torch.empty(T, d).cuda(), torch.zeros(n, d).cuda()
    Q.gather_rows(F32, x.cuda(), pos, T, k, d, r, n)
    Q.combine_rows(F32, rows.cuda(), n, pos, None, T, k, d, out)
    a = float((r.cpu().double() * rows.double()).sum())
    b = float((x.double() * out.cpu().double()).sum())
    assert abs(a - b) <= 1e-5 * (T * d * k) ** 0.5 * 8


def test_combine_grad_without_dw_does_not_read_rows():
    g = gen(5)
    dout, w, pos = randn(g, 3, 64), torch.randn(3, 2, generator=g), routed(g, 3, 2, 6, held=1.1)
    drows = torch.zeros(6, 64).cuda()
    Q.combine_rows_grad(F32, dout.cuda(), None, 6, pos.cuda(), w.cuda(), 3, 2, 64, drows)
    for a, p in enumerate(pos.tolist()):
        assert torch.equal(drows[p].cpu(), w.reshape(-1)[a] * dout[a // 2])


# ------------------------------------------------------------ 8 bits

@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 128), (3, 129), (17, 1000), (5, 7168)])
@pytest.mark.parametrize("type", TYPES)
def test_quantize_rows(rows, cols, type):
    g = gen(rows + cols)
    x = randn(g, rows, cols, type=type) * torch.exp2(torch.randint(-12, 12, (rows, 1), generator=g).float()).to(F.DTYPE[type])
    codes, scales = torch.zeros(rows, cols, dtype=torch.uint8).cuda(), torch.zeros(rows, F.blocks(cols)).cuda()
    Q.quantize_fp8(type, x.cuda(), rows, cols, codes, scales)
    c, s = F.quantize(x)
    assert torch.equal(codes.cpu(), c) and torch.equal(scales.cpu(), s)
    err = (F.values(codes.cpu(), scales.cpu()) - x.double()).abs()
    assert bool((err <= F.code_bound(x.double(), s) * (1 + 4 * U) + 4 * U * x.double().abs()).all())
    # only the first rows
    codes2 = torch.full((rows, cols), 9, dtype=torch.uint8).cuda()
    n = torch.tensor([rows - 1], dtype=torch.int32).cuda()
    Q.quantize_fp8(type, x.cuda(), rows, cols, codes2, scales, n_rows=n)
    c[rows - 1:] = 9
    assert torch.equal(codes2.cpu(), c)


def test_quantize_special_blocks():
    x = torch.zeros(1, 128 * 6)
    x[0, 128:256] = 1e-42          # denormals
    x[0, 256 + 5] = float("nan")
    x[0, 256 + 6] = 1.0
    x[0, 384 + 7] = float("inf")
    x[0, 512:640] = torch.finfo(torch.float32).max
    x[0, 640:768] = -torch.finfo(torch.float32).max
    codes, scales = torch.zeros(1, 768, dtype=torch.uint8).cuda(), torch.zeros(1, 6).cuda()
    Q.quantize_fp8(F32, x.cuda(), 1, 768, codes, scales)
    v, s = F.values(codes.cpu(), scales.cpu())[0], scales.cpu()[0]
    assert s[0] == F.MIN_SCALE and s[1] == F.MIN_SCALE and bool((v[:128] == 0).all())
    assert bool((v[128:256] - 1e-42).abs().max() <= F.MIN_SCALE * 2.0 ** -10)
    assert bool(v[256:384].isnan().all()) and bool(v[384:512].isnan().all())
    big = float(torch.finfo(torch.float32).max)
    assert bool(((v[512:640] - big).abs() <= 4 * U * big).all()) and bool(((v[640:] + big).abs() <= 4 * U * big).all())


@pytest.mark.parametrize("groups,rows,cols", [(1, 1, 1), (2, 128, 256), (3, 130, 72), (1, 500, 1000)])
@pytest.mark.parametrize("type", TYPES)
def test_quantize_weights(groups, rows, cols, type):
    w = randn(gen(rows), groups, rows, cols, type=type)
    codes = torch.zeros(groups, rows, cols, dtype=torch.uint8).cuda()
    scales = torch.zeros(groups, F.blocks(rows), F.blocks(cols)).cuda()
    Q.quantize_fp8_weights(type, w.cuda(), rows, cols, codes, scales, groups=groups)
    for i in range(groups):
        c, s = F.quantize(w[i], 128)
        assert torch.equal(codes[i].cpu(), c) and torch.equal(scales[i].cpu(), s)


@pytest.mark.parametrize("rows,f", [(1, 1), (1, 128), (3, 200), (7, 1536), (64, 2816), (2, 11008)])
@pytest.mark.parametrize("type", TYPES)
@pytest.mark.parametrize("limit", [0.0, 1.5])
def test_swiglu(rows, f, type, limit):
    gu = 3 * randn(gen(f), rows, 2 * f, type=type)
    gu[0, 0] = -90.0   # exp(90) is large, the sigmoid tiny
    codes, scales = torch.zeros(rows, f, dtype=torch.uint8).cuda(), torch.zeros(rows, F.blocks(f)).cuda()
    Q.swiglu_fp8(type, gu.cuda(), rows, f, codes, scales, limit=limit)
    h = F.swiglu(gu[:, :f], gu[:, f:], limit)
    s = scales.cpu()
    pad = torch.nn.functional.pad(h.abs(), (0, -f % 128)).reshape(rows, -1, 128).amax(2)
    assert bool(((s.double() - (pad / 448).clamp_min(F.MIN_SCALE)).abs() <= 17 * U * (pad / 448) + 1e-45).all())
    err = (F.values(codes.cpu(), s) - h).abs()
    assert bool((err <= F.code_bound(h, s) * (1 + 32 * U) + 32 * U * h.abs()).all())


@pytest.mark.parametrize("rows,f", [(1, 128), (5, 256), (64, 2816), (2, 2048)])
@pytest.mark.parametrize("type", TYPES)
@pytest.mark.parametrize("limit", [0.0, 1.5])
def test_swiglu_grad(rows, f, type, limit):
    g = gen(f + rows)
    gu, dh = 3 * randn(g, rows, 2 * f, type=type), randn(g, rows, f, type=type)
    if limit:
        gu[0, 0], gu[0, f], gu[0, f + 1] = limit, limit, -limit   # on the edge nothing is cut off
    codes, scales = torch.zeros(rows, 2 * f, dtype=torch.uint8).cuda(), torch.zeros(rows, 2 * f // 128).cuda()
    Q.swiglu_fp8_grad(type, gu.cuda(), dh.cuda(), rows, f, codes, scales, limit=limit)
    dg, du, parts = F.swiglu_grad(gu[:, :f], gu[:, f:], dh, limit)
    want, size = torch.cat([dg, du], 1), torch.cat([torch.where(dg == 0, 0.0, parts), du.abs()], 1)
    err = (F.values(codes.cpu(), scales.cpu()) - want).abs()
    assert bool((err <= F.code_bound(want.abs() + 32 * U * size, scales.cpu()) * (1 + 32 * U) + 32 * U * size).all())
    # the formula against differences of SwiGLU in 64 bits, away from the cut-offs
    e = 1e-5
    gate, up = gu[:, :f].double(), gu[:, f:].double()
    flat = (gate - limit).abs().gt(1e-3) & (up.abs() - limit).abs().gt(1e-3) if limit else torch.ones_like(gate, dtype=torch.bool)
    ng = (F.swiglu(gate + e, up, limit) - F.swiglu(gate - e, up, limit)) / (2 * e) * dh.double()
    nu = (F.swiglu(gate, up + e, limit) - F.swiglu(gate, up - e, limit)) / (2 * e) * dh.double()
    scale = 1 + dh.double().abs() * (1 + up.abs()) * (1 + gate.abs())
    assert bool(((ng - dg).abs()[flat] <= 1e-8 * scale[flat]).all())
    assert bool(((nu - du).abs()[flat] <= 1e-8 * scale[flat]).all())


# ------------------------------------------------------------ products

def matrices(g, groups, rows, cols):
    q = [F.quantize(0.02 * torch.randn(rows, cols, generator=g), 128) for _ in range(groups)]
    codes, scales = torch.stack([c for c, _ in q]), torch.stack([s for _, s in q])
    # uneven block scales, so that a wrong block shows
    scales *= torch.exp2(torch.randint(-3, 4, scales.shape, generator=g).float())
    return codes, scales


def check_product(codes, scales, counts, type, back, seed, lead=0, extra=0, stream=None, m=None):
    """One product through `m` against 64 bits; rows outside the groups (`lead`
    before, three after) must stay untouched."""
    g = gen(seed)
    groups, N, K = codes.shape
    kin, kout = (N, K) if back else (K, N)
    off = torch.tensor([lead] + (lead + np.cumsum(counts)).tolist(), dtype=torch.int32)
    T = int(off[-1]) + 3
    x, xs = F.quantize(torch.randn(T, kin, generator=g))
    xs = xs * torch.exp2(torch.randint(-3, 4, xs.shape, generator=g).float())
    gap = -kin % 16 + 16 * extra
    xd, ld = pitched(x, gap)
    own = m or Q.Fp8Matrix(N, K, codes, scales, groups=groups)
    out = torch.full((T, kout + extra), 5.0, dtype=F.DTYPE[type]).cuda()
    torch.cuda.synchronize()
    f = own.product_t if back else own.product
    f(type, xd, xs.cuda(), T, out, off.cuda(), ld, 0, kout + extra, stream)
    own.sync()
    got = out.cpu().double()
    xv = F.values(x, xs)
    tol = 128 * 2.0 ** -23 + (F.blocks(kin) + 3) * U
    touched = torch.zeros(T, dtype=torch.bool)
    for i in range(groups):
        a, b = int(off[i]), int(off[i + 1])
        touched[a:b] = True
        if a == b:
            continue
        w = F.values(codes[i], scales[i], 128)
        w = w if back else w.T
        want, size = xv[a:b] @ w, xv[a:b].abs() @ w.abs()
        err = (got[a:b, :kout] - want).abs()
        assert bool((err <= tol * size + F.ROUND[type] * (want.abs() + tol * size)
                     + F.HALF_STEP[type]).all()), (i, float((err / size).max()))
    assert bool((got[~touched] == 5.0).all()) and bool((got[:, kout:] == 5.0).all())
    if m is None:
        own.close()
    return out


@pytest.mark.parametrize("back", [False, True])
@pytest.mark.parametrize("N,K", [(1, 16), (128, 128), (130, 272), (384, 1024), (1000, 144), (77, 640), (2049, 130)])
@pytest.mark.parametrize("T", [1, 5, 16, 17, 100, 128, 129, 300])
def test_product_dense(N, K, T, back):
    codes, scales = matrices(gen(N + K), 1, N, K)
    check_product(codes, scales, [T], F32, back, T + N)


@pytest.mark.parametrize("back", [False, True])
@pytest.mark.parametrize("type", TYPES)
@pytest.mark.parametrize("counts,lead", [([0, 3, 0, 0, 130, 1, 16], 0), ([1] * 40, 5), ([0, 0, 0], 2), ([257, 0, 64], 0),
                                         ([20, 200, 2, 129, 128, 127], 1), ([900, 700], 0)])
def test_product_grouped(counts, lead, type, back):
    codes, scales = matrices(gen(len(counts)), len(counts), 200, 336)
    check_product(codes, scales, counts, type, back, 3, lead=lead, extra=1)


@pytest.mark.parametrize("back", [False, True])
def test_product_long_and_many_rows(back):
    codes, scales = matrices(gen(1), 1, 1536, 2816)
    for T in (1, 40, 700, 2000):
        check_product(codes, scales, [T], BF16, back, T)


@pytest.mark.parametrize("back", [False, True])
def test_product_keeps_rows_apart(back):
    """NaN in one row, one group or past the matrix's end reaches no other row."""
    g = gen(8)
    N, K = 200, 336
    kin, kout = (N, K) if back else (K, N)
    codes, scales = matrices(g, 3, N, K)
    codes[1], scales[1] = 0x7F, float("nan")   # the middle matrix is NaN
    x, xs = F.quantize(torch.randn(60, kin, generator=g))
    xd, ld = pitched(x, -kin % 16 + 16)        # NaN codes in the gap
    off = torch.tensor([0, 20, 40, 60], dtype=torch.int32)
    bad = 7
    xd[bad, :kin] = 0x7F
    m = Q.Fp8Matrix(N, K, codes, scales, groups=3)
    out = torch.zeros(60, kout).cuda()
    if back:
        m.product_t(F32, xd, xs.cuda(), 60, out, off.cuda(), ld_y=ld)
    else:
        m.product(F32, xd, xs.cuda(), 60, out, off.cuda(), ld_x=ld)
    m.sync()
    nan = out.isnan().cpu()
    assert bool(nan[bad].all()) and bool(nan[20:40].all())
    rest = torch.ones(60, dtype=torch.bool)
    rest[bad] = False
    rest[20:40] = False
    assert not bool(nan[rest].any())
    m.close()


def test_product_twice_is_the_same_and_offsets_are_checked():
    codes, scales = matrices(gen(4), 4, 256, 512)
    m = Q.Fp8Matrix(256, 512, codes.cuda(), scales.cuda(), groups=4)
    a = check_product(codes, scales, [3, 0, 50, 140], F32, False, 6, m=m)
    b = check_product(codes, scales, [3, 0, 50, 140], F32, False, 6, m=m)
    assert torch.equal(a, b)
    x, xs = F.quantize(torch.randn(64, 512, generator=gen(2)))
    out = torch.full((64, 256), 5.0).cuda()
    for off in ([0, 10, 5, 20, 64], [0, 10, 20, 30, 65], [-1, 10, 20, 30, 40], [0, 2000000000, 20, 30, 40]):
        m.product(F32, x.cuda(), xs.cuda(), 64, out, torch.tensor(off, dtype=torch.int32).cuda())
        with pytest.raises(Q.QrmError) as e:
            m.sync()
        assert e.value.code == Q.E_INVALID
    m.sync()   # the report is given once
    check_product(codes, scales, [3, 0, 50, 140], F32, False, 6, m=m)
    m.close()


def test_product_on_another_stream_and_in_a_graph():
    codes, scales = matrices(gen(9), 1, 512, 1024)
    m = Q.Fp8Matrix(512, 1024, codes, scales)
    side = torch.cuda.Stream()
    check_product(codes, scales, [33], F32, False, 1, stream=side.cuda_stream, m=m)
    g = gen(12)
    x = torch.randn(5, 1024, generator=g).cuda()
    c, s = torch.zeros(5, 1024, dtype=torch.uint8).cuda(), torch.zeros(5, 8).cuda()
    out = torch.zeros(5, 512).cuda()

    def step(stream):
        Q.quantize_fp8(F32, x, 5, 1024, c, s, stream=stream)
        m.product(F32, c, s, 5, out, stream=stream)

    step(torch.cuda.current_stream().cuda_stream)
    m.sync()
    want = out.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(torch.cuda.current_stream().cuda_stream)
    for _ in range(3):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
    x.mul_(2.0)   # a power of two: the codes stay, the scales double
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, 2.0 * want)
    m.close()


def test_rows_past_32_bits():
    """A row whose offset passes 2^32 elements, out, back and through a product."""
    d, n = 7168, 620_000   # 4.4e9 codes
    g = gen(2)
    x = randn(g, 2, d)
    pos = torch.tensor([n - 1, 5], dtype=torch.int32).cuda()
    codes, scales = torch.empty(n, d, dtype=torch.uint8, device="cuda"), torch.empty(n, 56, device="cuda")
    Q.gather_rows_fp8(F32, x.cuda(), pos, 2, 1, d, codes, scales, n)
    c, s = F.quantize(x)
    assert torch.equal(codes[n - 1].cpu(), c[0]) and torch.equal(codes[5].cpu(), c[1])
    assert torch.equal(scales[n - 1].cpu(), s[0])
    wc, ws = matrices(g, 1, 128, d)
    m = Q.Fp8Matrix(128, d, wc, ws)
    out = torch.zeros(n, 128, device="cuda")
    off = torch.tensor([n - 1, n], dtype=torch.int32).cuda()
    m.product(F32, codes, scales, n, out, off)
    m.sync()
    want = F.values(c[:1], s[:1]) @ F.values(wc[0], ws[0], 128).T
    assert bool(((out[n - 1].cpu().double() - want[0]).abs() <= 1e-5 * want.abs().max()).all())
    assert float(out[: n - 1].abs().max()) == 0.0
    m.close()


# ------------------------------------------------------------ refusals

def code_of(f, *a, **k):
    with pytest.raises(Q.QrmError) as e:
        f(*a, **k)
    return e.value.code


def test_refusals():
    i = torch.zeros(64, dtype=torch.int32).cuda()
    x = torch.zeros(64, 256).cuda()
    c, s = torch.zeros(64, 512, dtype=torch.uint8).cuda(), torch.zeros(64, 4).cuda()
    assert code_of(Q.sort_tokens, i, 8, 0, 4, i, i, i) == Q.E_INVALID
    assert code_of(Q.sort_tokens, i, -1, 2, 4, i, i, i) == Q.E_INVALID
    assert code_of(Q.sort_tokens, i, 2 ** 31, 2, 4, i, i, i) == Q.E_INVALID
    assert code_of(Q.sort_tokens, i, 8, 2, 0, i, i, i) == Q.E_INVALID
    assert code_of(Q.sort_tokens, i, 8, 2, 1025, i, i, i) == Q.E_CAPACITY
    assert code_of(Q.sort_tokens, i, 8, 2, 4, i, i, None) == Q.E_INVALID
    assert code_of(Q.sort_tokens, i, 8, 2, 4, i.data_ptr() + 2, i, i) == Q.E_INVALID
    assert code_of(Q.gather_rows, 6, x, i, 4, 2, 256, x, 64) == Q.E_FORMAT
    assert code_of(Q.gather_rows, F32, None, i, 4, 2, 256, x, 64) == Q.E_INVALID
    assert code_of(Q.gather_rows, F32, x, i, 4, 2, 256, x, 64, ld_x=255) == Q.E_INVALID
    assert code_of(Q.gather_rows, F32, x.data_ptr() + 1, i, 4, 2, 256, x, 64) == Q.E_INVALID
    assert code_of(Q.gather_rows_fp8, F32, x, i, 4, 2, 256, c, s, 64, ld_scales=1) == Q.E_INVALID
    assert code_of(Q.combine_rows, F32, x, -1, i, None, 4, 2, 256, x) == Q.E_INVALID
    assert code_of(Q.combine_rows, F32, x, 64, None, None, 4, 2, 256, x) == Q.E_INVALID
    assert code_of(Q.combine_rows_grad, F32, x, None, 64, i, None, 4, 2, 256, x, s) == Q.E_INVALID
    assert code_of(Q.quantize_fp8, F32, x, 64, 0, c, s) == Q.E_INVALID
    assert code_of(Q.quantize_fp8_weights, F32, x, 64, 256, c, s, groups=0) == Q.E_INVALID
    assert code_of(Q.swiglu_fp8, F32, x, 64, 128, c, s, limit=-1.0) == Q.E_INVALID
    assert code_of(Q.swiglu_fp8, F32, x, 64, 128, c, s, limit=float("nan")) == Q.E_INVALID
    assert code_of(Q.swiglu_fp8_grad, F32, x, x, 64, 100, c, s) == Q.E_INVALID
    # nothing to do is no error
    Q.gather_rows(F32, None, None, 0, 2, 256, None, 0)
    Q.combine_rows(F32, None, 0, None, None, 0, 2, 256, None)
    Q.quantize_fp8(F32, None, 0, 256, None, None)
    Q.swiglu_fp8(F32, None, 0, 128, None, None)


def test_matrix_refusals():
    c, s = np.zeros((2, 200, 300), np.uint8), np.ones((2, 2, 3), np.float32)
    assert code_of(Q.Fp8Matrix, 200, 300, c, s, groups=1) == Q.E_SIZE
    assert code_of(Q.Fp8Matrix, 200, 300, c, s[:, :1], groups=2) == Q.E_SIZE
    assert code_of(Q.Fp8Matrix, 0, 300, c, s, groups=2) == Q.E_INVALID
    assert code_of(Q.Fp8Matrix, 200, 300, c, s, groups=2, device=99) == Q.E_INVALID
    assert code_of(Q.Fp8Matrix, 1, 1, np.zeros(1025, np.uint8), np.ones(1025, np.float32), groups=1025) == Q.E_CAPACITY
    with pytest.raises(ValueError):
        Q.Fp8Matrix(200, 300, torch.zeros(2, 200, 300, dtype=torch.uint8).cuda(), torch.ones(2, 2, 3), groups=2)
    m = Q.Fp8Matrix(200, 300, c, s, groups=2)
    x, xs = torch.zeros(8, 304, dtype=torch.uint8).cuda(), torch.zeros(8, 3).cuda()
    y, off = torch.zeros(8, 200).cuda(), torch.tensor([0, 4, 8], dtype=torch.int32).cuda()
    assert code_of(m.product, 6, x, xs, 8, y, off, ld_x=304) == Q.E_FORMAT
    assert code_of(m.product, F32, x, xs, 8, y, None, ld_x=304) == Q.E_INVALID
    assert code_of(m.product, F32, x, xs, 8, y, off) == Q.E_INVALID               # rows of 300 bytes
    assert code_of(m.product, F32, x.data_ptr() + 8, xs, 4, y, off, ld_x=304) == Q.E_INVALID
    assert code_of(m.product, F32, x, xs, 8, y, off, ld_x=288) == Q.E_INVALID
    assert code_of(m.product, F32, x, xs, 8, y, off, ld_x=304, ld_scales=2) == Q.E_INVALID
    assert code_of(m.product, F32, x, xs, 8, y, off, ld_x=304, ld_y=199) == Q.E_INVALID
    assert code_of(m.product, F32, x, None, 8, y, off, ld_x=304) == Q.E_INVALID
    assert code_of(m.product, F32, x, xs, -1, y, off, ld_x=304) == Q.E_INVALID
    m.product(F32, None, None, 0, None)
    m.product(F32, x, xs, 8, y, off, ld_x=304)
    m.sync()
    assert float(y.abs().max()) == 0.0
    m.close()
