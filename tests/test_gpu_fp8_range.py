"""The 8-bit expert operators at the ends of their types' ranges, on the GPU
against the plain forms in 64 bits.

Tolerances as in test_gpu_fp8.py: 32 u of the value (u = 2^-24; 16 u of each of
two factors), then half the distance between neighbouring codes.  The gate's
gradient is a sum, 1 + g (1 - sigma), whose parts cancel nowhere here: sigma is
0 or 1 to the last bit at the gates that are large, and the others are ordinary.
"""
import pytest

import qauntrunner_b200 as Q
from tests import fp8_plain as F
from tests.test_gpu_fp8 import BF16, F16, F32, U, gen, randn

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


# ------------------------------------------------------------ SwiGLU's gate

def large_gates(type):
    """Gates at and below the type's largest magnitude, and around 2^128 / log2(e)
    = 2.3587e38, where g log2(e) passes the f32 range."""
    top = float(torch.finfo(F.DTYPE[type]).max)
    return [v for v in (top, 0.99 * top, 2.4e38, 2.36e38, 2.358e38, 2.3e38, 1e30, 60000.0, 129.0, 128.0, 105.0, 89.0)
            if v <= top]


def extremes(type, f, sign):
    """gu, dh of four rows: ordinary values, and among the first block of 128
    some large gates of one sign.  Where the gate passes, up and dh are small
    enough for the f32 range, and half of the columns are masked by 0."""
    g = gen(f + type)
    gu, dh = randn(g, 4, 2 * f, type=type), randn(g, 4, f, type=type)
    for i, v in enumerate(large_gates(type)):
        for row in range(4):
            c = 7 * i + row
            gu[row, c] = sign * v
            if sign > 0:
                small = 0.0 if row % 2 else 1.0 / max(v, 1.0)
                gu[row, f + c] = small if type != F16 else 2.0 ** -10
                dh[row, c] = dh[row, c] * (2.0 ** -10 if v < 1e30 else 2.0 ** -40)
    return gu, dh


def close(codes, scales, want, size):
    assert not bool(scales.isnan().any()) and not bool((codes & 0x7F == 0x7F).any())
    err = (F.values(codes, scales) - want).abs()
    return bool((err <= F.code_bound(want.abs() + 32 * U * size, scales) * (1 + 32 * U) + 32 * U * size).all())


@pytest.mark.parametrize("type", [F32, F16, BF16])
@pytest.mark.parametrize("limit", [0.0, 7.0])
@pytest.mark.parametrize("sign", [-1.0, 1.0])
def test_swiglu_of_large_gates(type, limit, sign):
    f = 256
    gu, _ = extremes(type, f, sign)
    codes, scales = torch.zeros(4, f, dtype=torch.uint8).cuda(), torch.zeros(4, 2).cuda()
    Q.swiglu_fp8(type, gu.cuda(), 4, f, codes, scales, limit=limit)
    h = F.swiglu(gu[:, :f], gu[:, f:], limit)
    assert close(codes.cpu(), scales.cpu(), h, h.abs())


@pytest.mark.parametrize("type", [F32, F16, BF16])
@pytest.mark.parametrize("limit", [0.0, 7.0])
@pytest.mark.parametrize("sign", [-1.0, 1.0])
def test_swiglu_grad_of_large_gates(type, limit, sign):
    f = 256
    gu, dh = extremes(type, f, sign)
    codes, scales = torch.zeros(4, 2 * f, dtype=torch.uint8).cuda(), torch.zeros(4, 4).cuda()
    Q.swiglu_fp8_grad(type, gu.cuda(), dh.cuda(), 4, f, codes, scales, limit=limit)
    dg, du, parts = F.swiglu_grad(gu[:, :f], gu[:, f:], dh, limit)
    ordinary = gu[:, :f].double().abs() < 80
    size = torch.where(ordinary & (dg != 0), parts, dg.abs())
    assert close(codes.cpu(), scales.cpu(), torch.cat([dg, du], 1), torch.cat([size, du.abs()], 1))


def test_a_masked_gate_leaves_its_block_as_it_is():
    """The type's lowest value as a gate, as a mask would put it: h is 0 there and
    the other columns' codes are what they are without it."""
    for type in (F32, BF16):
        gu = randn(gen(3), 2, 512, type=type)
        gu[1] = gu[0]
        gu[1, 5:256:9] = torch.finfo(F.DTYPE[type]).min
        gu[0, 5:256:9] = 0.0
        codes, scales = torch.zeros(2, 256, dtype=torch.uint8).cuda(), torch.zeros(2, 2).cuda()
        Q.swiglu_fp8(type, gu.cuda(), 2, 256, codes, scales)
        v = F.values(codes.cpu(), scales.cpu())
        assert torch.equal(v[0], v[1]) and bool((v[1, 5:256:9] == 0).all())


# ------------------------------------------------------------ as many rows as a count holds

MANY = 2 ** 31 - 1


def test_combine_of_the_most_tokens():
    """One column, one slot: the walk's last steps, where a signed row number would turn negative (13 GB)."""
    pos = torch.full((MANY,), -1, dtype=torch.int32, device="cuda")
    pos[0], pos[MANY - 5000], pos[-1] = 1, 2, 0
    rows = torch.tensor([3.0, -2.0, 0.5], dtype=torch.float16, device="cuda")
    out = torch.full((MANY,), 5.0, dtype=torch.float16, device="cuda")
    Q.combine_rows(F16, rows, 3, pos, None, MANY, 1, 1, out)
    torch.cuda.synchronize()
    assert (float(out[0]), float(out[MANY - 5000]), float(out[-1])) == (-2.0, 0.5, 3.0)
    assert int(out.count_nonzero()) == 3


def test_swiglu_of_the_most_rows():
    """One column: 20 GB."""
    gu = torch.zeros(MANY, 2, dtype=torch.float16, device="cuda")
    gu[0], gu[-1] = 1.0, -1.0
    codes = torch.full((MANY,), 9, dtype=torch.uint8, device="cuda")
    scales = torch.full((MANY,), 5.0, device="cuda")
    Q.swiglu_fp8(F16, gu, MANY, 1, codes, scales)
    torch.cuda.synchronize()
    h = F.swiglu(gu[:, :1][[0, -1]].cpu(), gu[:, 1:][[0, -1]].cpu(), 0.0)[:, 0]
    got = torch.tensor([float(scales[0]), float(scales[-1])], dtype=torch.float64) * 448
    assert bool(((got - h.abs()).abs() <= 32 * U * h.abs()).all())
    assert int((codes & 0x7F == 0x7E).count_nonzero()) == 2 and int(codes.count_nonzero()) == 2   # 448, and 0
    assert float(scales[1:-1].max()) == F.MIN_SCALE


# ------------------------------------------------------------ blocks of tiny values

def tiny_blocks(g, type):
    """Blocks whose largest magnitude is 2^-149 to 2^-85.  In three rows of four that is 7 times an odd number up to 15,
    so the scale (a 448th) is that odd number and some power of two, and the others are the scale times 5 bits, which is
    a tie between codes; in the fourth row any values.  (Where a value does not fit the type it is no tie any more.)"""
    e = torch.arange(-149, -84).repeat_interleave(64)[:, None].float()
    n = e.shape[0]
    odd = 2 * torch.randint(0, 8, (n, 1), generator=g).float() + 1
    ties = odd * (2 * torch.randint(8, 16, (n, 128), generator=g).float() + 1)
    ties = torch.where(torch.rand(n, 128, generator=g) < 0.5, ties, -ties) * torch.exp2(torch.randint(-19, -3, (n, 128), generator=g).float())
    any_ = 7 * odd * (2 * torch.rand(n, 128, generator=g) - 1)
    x = torch.where(torch.arange(n)[:, None] % 4 > 0, ties, any_)
    x[:, 0:1] = 7 * odd
    return torch.ldexp(x, e - 5).to(F.DTYPE[type])


@pytest.mark.parametrize("type", [F32, BF16])
def test_quotients_of_tiny_blocks(type):
    """Codes and scales bit for bit, against IEEE division (bf16's few bits make more ties)."""
    x = tiny_blocks(gen(3 + type), type)
    n = x.shape[0]
    codes, scales = torch.zeros(n, 128, dtype=torch.uint8).cuda(), torch.zeros(n, 1).cuda()
    Q.quantize_fp8(type, x.cuda(), n, 128, codes, scales)
    v = x.float()
    s = (v.abs().amax(1, keepdim=True) / 448.0).clamp_min(F.MIN_SCALE)
    want = (v / s).to(torch.float8_e4m3fn).view(torch.uint8)
    assert torch.equal(scales.cpu(), s) and torch.equal(codes.cpu(), want)
    # the other operators that write 8-bit rows of given values
    rows, rs = torch.zeros_like(codes), torch.zeros_like(scales)
    pos = torch.arange(n, dtype=torch.int32).cuda()
    Q.gather_rows_fp8(type, x.cuda(), pos, n, 1, 128, rows, rs, n)
    assert torch.equal(rows.cpu(), want) and torch.equal(rs.cpu(), s)
    rows, rs, w = torch.zeros_like(codes), torch.zeros_like(scales), torch.full((n, 1), -1.0).cuda()
    Q.combine_rows_grad_fp8(type, x.cuda(), None, n, pos, w, n, 1, 128, rows, rs)
    assert torch.equal(rows.cpu(), want ^ 0x80) and torch.equal(rs.cpu(), s)


def test_quotients_of_tiny_weights():
    x = tiny_blocks(gen(9), F32)[:4096].reshape(32, 128, 128)   # a block of 128 x 128 for each exponent or two
    codes, scales = torch.zeros(32, 128, 128, dtype=torch.uint8).cuda(), torch.zeros(32, 1, 1).cuda()
    Q.quantize_fp8_weights(F32, x.cuda(), 128, 128, codes, scales, groups=32)
    s = (x.abs().amax((1, 2), keepdim=True) / 448.0).clamp_min(F.MIN_SCALE)
    assert torch.equal(scales.cpu(), s)
    assert torch.equal(codes.cpu(), (x / s).to(torch.float8_e4m3fn).view(torch.uint8))
