"""The 8-bit operators together (examples/fp8_experts.py), both product kernels
at the same sizes, and the quotient that stands for a division.

The layer is compared with the same steps in plain operations: sums in 64 bits,
8-bit and bf16 roundings in the same places.  The two can differ only where a
sum that is a few f32 roundings off falls on the other side of a rounding
boundary; one such bf16 value is 2^-8 off, one such code 2^-3, and they are rare
(a boundary within 1e-5 of the value: 1 in 200 values and 1 in 6000 codes), so
0.01 of the norm, bf16's own bound, holds for every output.
"""
import importlib.util
import os

import pytest

import qauntrunner_b200 as Q
from tests import fp8_plain as F
from tests.test_gpu_fp8 import check_product, gen, matrices

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def example():
    spec = importlib.util.spec_from_file_location("fp8_experts", os.path.join(ROOT, "examples", "fp8_experts.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def bf16(v):
    return v.float().bfloat16().double()


def q8(v):
    return F.values(*F.quantize(v))


@pytest.mark.parametrize("T,k,E,d,f,limit", [(1, 8, 16, 256, 128, 0.0), (37, 2, 4, 384, 256, 1.0), (300, 3, 3, 512, 128, 0.0)])
def test_layer_forward_and_backward(T, k, E, d, f, limit):
    g = gen(T)
    w13, w2 = torch.randn(E, 2 * f, d, generator=g) * d ** -0.5, torch.randn(E, d, f, generator=g) * f ** -0.5
    idx = torch.stack([torch.randperm(E + 1, generator=g)[:k] if k <= E else torch.randint(0, E + 1, (k,), generator=g)
                       for _ in range(T)]).int()
    idx = torch.where(idx == E, -1, idx)   # some slots have no expert
    if T > 1:
        idx[T // 2] = -1                   # nor has one token in any slot
    w = torch.rand(T, k, generator=g)
    x, dout = torch.randn(T, d, generator=g).bfloat16(), torch.randn(T, d, generator=g).bfloat16()
    layer = example().Fp8Experts(w13.cuda(), w2.cuda(), limit=limit)
    out, kept = layer.forward(x.cuda(), idx.cuda(), w.cuda())
    dx, dw = layer.backward(dout.cuda(), kept)
    layer.sync()
    layer.close()

    want_out, want_dx, want_dw = x.double(), dout.double(), torch.zeros(T, k, dtype=torch.float64)
    for e in range(E):
        a, b = F.values(*F.quantize(w13[e], 128), 128), F.values(*F.quantize(w2[e], 128), 128)
        t, j = (idx == e).nonzero(as_tuple=True)
        if not t.numel():
            continue
        gu = bf16(q8(x[t]) @ a.T)
        y = bf16(q8(F.swiglu(gu[:, :f], gu[:, f:], limit)) @ b.T)
        want_out = want_out.index_add(0, t, w[t, j, None].double() * y)
        want_dw[t, j] = (dout[t].double() * y).sum(1)
        dh = bf16(q8(w[t, j, None] * dout[t].float()) @ b)
        dg, du, _ = F.swiglu_grad(gu[:, :f], gu[:, f:], dh, limit)
        want_dx = want_dx.index_add(0, t, bf16(torch.cat([q8(dg), q8(du)], 1) @ a))
    for name, got, ref in (("out", out, want_out), ("dx", dx, want_dx), ("dw", dw, want_dw)):
        off = float((got.cpu().double() - ref).norm() / ref.norm())
        assert off <= 0.01, (name, off)
    if T > 1:
        assert torch.equal(out[T // 2].cpu(), x[T // 2]) and torch.equal(dx[T // 2].cpu(), dout[T // 2])
        assert float(dw[T // 2].abs().max()) == 0.0


@pytest.mark.parametrize("pair", ["0", "1"])
@pytest.mark.parametrize("back", [False, True])
@pytest.mark.parametrize("counts,N,K", [([1], 640, 1040), ([0, 3, 127, 128, 129], 384, 272), ([256, 0, 257, 1], 513, 640),
                                        ([31, 32, 33, 383, 385], 130, 144), ([700], 1536, 256)])
def test_both_kernels(monkeypatch, counts, N, K, back, pair):
    monkeypatch.setenv("QRM_FP8_PAIR", pair)
    codes, scales = matrices(gen(N + K), len(counts), N, K)
    for type, lead, extra in ((0, 0, 0), (2, 3, 1), (1, 0, 16)):
        check_product(codes, scales, counts, type, back, len(counts) + type, lead=lead, extra=extra)


@pytest.mark.parametrize("pair", ["0", "1"])
def test_many_groups(monkeypatch, pair):
    monkeypatch.setenv("QRM_FP8_PAIR", pair)
    codes, scales = matrices(gen(5), 40, 64, 48)
    codes, scales = codes.repeat(25, 1, 1)[:1000], scales.repeat(25, 1, 1)[:1000]
    counts = [(7 * i) % 5 for i in range(1000)]
    check_product(codes, scales, counts, 0, False, 3)


def test_quotients_are_rounded_like_divisions():
    """Scales and codes over many magnitudes of a block's largest value, against
    IEEE division, bit for bit (ties of 8-bit codes among them: few-bit values)."""
    g = gen(77)
    n = 4096
    top = torch.exp2(torch.randint(-100, 100, (n, 1), generator=g).float()) * (1 + torch.rand(n, 1, generator=g))
    x = top * (torch.randint(-256, 257, (n, 128), generator=g).float() / 256)
    x[:, 0:1] = top
    x[::2] = x[::2].bfloat16().float()
    codes, scales = torch.zeros(n, 128, dtype=torch.uint8).cuda(), torch.zeros(n, 1).cuda()
    Q.quantize_fp8(0, x.cuda(), n, 128, codes, scales)
    s = x.abs().amax(1, keepdim=True) / 448.0
    assert torch.equal(scales.cpu(), s)
    assert torch.equal(codes.cpu(), (x / s).to(torch.float8_e4m3fn).view(torch.uint8))
