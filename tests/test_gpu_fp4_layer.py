"""The norm and the 4-bit operators together, as the examples use them
(examples/fp4_experts.py), and the norm with its gradient around the 8-bit
experts (examples/fp8_experts.py).

The layers are compared with the same steps in plain operations: sums in 64
bits, 4-bit, 8-bit and bf16 roundings in the same places.  The two differ only
where a value that is a few f32 roundings off falls on the other side of a
rounding boundary.  Such a bf16 value is 2^-8 off, such an 8-bit code 2^-3, such a
4-bit code a half at most, and they are rare: f32 sums are within 1e-5 of the
value, boundaries of 4-bit codes lie a quarter of the value apart or more, so
fewer than 1e-4 of the codes change, which is sqrt(1e-4) / 2 = 0.005 of the norm.
With bf16's own 2^-8 that is below 0.01, for every output.
"""
import importlib.util
import os

import pytest

import qauntrunner_b200 as Q
from tests import fp4_plain as P
from tests import fp8_plain as F

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def example(name):
    spec = importlib.util.spec_from_file_location(name, os.path.join(ROOT, "examples", name + ".py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def gen(seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return g


def bf16(v):
    return v.float().bfloat16().double()


def q4(v):
    return P.values(*P.quantize(v), v.shape[1])


def close(got, want):
    assert float((got.cpu().double() - want).norm() / want.norm()) < 0.01


def routing(g, T, k, E):
    idx = torch.stack([torch.randperm(E + 1, generator=g)[:k] for _ in range(T)]).int()
    idx = torch.where(idx == E, -1, idx)   # some slots have no expert
    if T > 1:
        idx[T // 2] = -1                   # nor has one token in any slot
    return idx, torch.rand(T, k, generator=g)


@pytest.mark.parametrize("T,k,E,d,f,limit", [(1, 8, 16, 256, 128, 0.0), (37, 2, 4, 384, 160, 1.0), (300, 3, 3, 512, 96, 0.0)])
def test_experts(T, k, E, d, f, limit):
    g = gen(T)
    w13, w2 = torch.randn(E, 2 * f, d, generator=g) * d ** -0.5, torch.randn(E, d, f, generator=g) * f ** -0.5
    norm_w = 1 + 0.2 * torch.randn(d, generator=g)
    idx, w = routing(g, T, k, E)
    x, r = torch.randn(T, d, generator=g).bfloat16(), torch.randn(T, d, generator=g).bfloat16()
    layer = example("fp4_experts").Fp4Experts(w13.cuda(), w2.cuda(), norm_w.cuda(), limit=limit)
    routed = idx.cuda(), w.cuda()
    out = layer.forward(x.cuda(), r.cuda(), lambda y: routed)
    layer.sync()

    s = bf16(x.float() + r.float())
    y4 = q4(bf16(P.norm(s, norm_w, 1e-5)))
    want = s.clone()
    for e in range(E):
        t, j = (idx == e).nonzero(as_tuple=True)
        h = q4(P.gate(y4[t] @ q4(w13[e]).T, limit).float()) if len(t) else torch.zeros(0, f, dtype=torch.float64)
        want.index_add_(0, t, w.double()[t, j, None] * bf16(h @ q4(w2[e]).T))
    close(out, want)
    # captured, replayed on other inputs: the bits of a call
    xs, rs = x.cuda(), r.cuda()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = layer.forward(xs, rs, lambda y: routed)
    xs.copy_(torch.randn(T, d, generator=g))
    graph.replay()
    again = layer.forward(xs, rs, lambda y: routed)
    torch.cuda.synchronize()
    assert torch.equal(captured, again) and not torch.equal(captured, out)
    layer.close()


@pytest.mark.parametrize("T,d,f", [(1, 256, 544), (65, 544, 200), (400, 320, 768)])
def test_dense(T, d, f):
    g = gen(T)
    w13, w2 = torch.randn(2 * f, d, generator=g) * d ** -0.5, torch.randn(d, f, generator=g) * f ** -0.5
    norm_w = 1 + 0.2 * torch.randn(d, generator=g)
    x, r = torch.randn(T, d, generator=g).bfloat16(), torch.randn(T, d, generator=g).bfloat16()
    ffn = example("fp4_experts").DenseFfn(w13.cuda(), w2.cuda(), norm_w.cuda())
    total, out = ffn.forward(x.cuda(), r.cuda())
    s = bf16(x.float() + r.float())
    h = q4(P.gate(q4(P.norm(s, norm_w, 1e-5).float()) @ q4(w13).T, 0.0).float())
    assert torch.equal(total.cpu().double(), s)
    close(out, h @ q4(w2).T)
    ffn.close()


@pytest.mark.parametrize("T,k,E,d,f", [(1, 4, 8, 256, 128), (65, 2, 4, 384, 128)])
def test_norm_around_the_8_bit_experts_and_its_gradients(T, k, E, d, f):
    g = gen(T + 1)
    w13, w2 = torch.randn(E, 2 * f, d, generator=g) * d ** -0.5, torch.randn(E, d, f, generator=g) * f ** -0.5
    norm_w = 1 + 0.2 * torch.randn(d, generator=g)
    idx, w = routing(g, T, k, E)
    x, r, dout = (torch.randn(T, d, generator=g).bfloat16() for _ in range(3))
    m = example("fp8_experts")
    experts = m.Fp8Experts(w13.cuda(), w2.cuda())
    layer = m.PreNormExperts(experts, norm_w.cuda())
    out, kept = layer.forward(x.cuda(), r.cuda(), idx.cuda(), w.cuda())
    dx, dnorm, dw = layer.backward(dout.cuda(), kept)
    experts.sync()
    # the experts alone on the same normed rows give the gradient that enters the norm's
    s = (x.float() + r.float()).to(torch.bfloat16)
    assert torch.equal(kept[0].cpu(), s)
    y = torch.empty(T, d, dtype=torch.bfloat16).cuda()
    Q.rms_norm(2, s.cuda(), T, d, norm_w.cuda(), 1e-5, y)
    alone, inner = experts.forward(y, idx.cuda(), w.cuda(), add=s.cuda())
    dy, dw_alone = experts.backward(dout.cuda(), inner, through=False)
    assert torch.equal(alone, out) and torch.equal(dw_alone, dw)
    want, want_w, size, size_w = P.norm_grad(dy.cpu(), s, norm_w, 1e-5, dout)
    close(dx, want)
    assert bool(((dnorm.cpu().double() - want_w).abs() <= (T + 100) * F.U * size_w + 1e-300).all())
    experts.close()
