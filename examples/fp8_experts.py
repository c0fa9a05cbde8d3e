"""An MoE layer's experts in 8-bit floating point, forward and backward.

    python examples/fp8_experts.py [--tokens 512] [--experts 32] [--top-k 8] [--d 1024] [--ffn 512]

The weights (gate and up as one matrix of each expert, and down) are quantised
once, with a scale for each 128 x 128 block, and kept in HBM.  A forward sorts
the tokens by expert, writes their rows in 8 bits, runs both grouped products
with SwiGLU between them and brings the rows back to the tokens, weighted, on
top of the residual stream.  The backward gives the gradients of the tokens and
of the routing weights; the quantised experts themselves stay as they are.
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import qauntrunner_b200 as Q  # noqa: E402

BF16 = Q.QuantFormat.BF16


def rows8(rows, cols, device="cuda"):
    """Room for 8-bit rows: codes and scales."""
    return (torch.zeros(rows, cols, dtype=torch.uint8, device=device),
            torch.zeros(rows, -(-cols // 128), device=device))


class Fp8Experts:
    """w_gate_up [experts, 2 ffn, d] and w_down [experts, d, ffn]: tensors on the
    device, f32, f16 or bf16.  Activations are bf16."""

    def __init__(self, w_gate_up, w_down, limit=0.0):
        self.experts, two_f, self.d = w_gate_up.shape
        self.ffn, self.limit = two_f // 2, limit
        self.gate_up, self.down = self._matrix(w_gate_up), self._matrix(w_down)

    @staticmethod
    def _matrix(w):
        groups, rows, cols = w.shape
        type = {torch.float32: Q.QuantFormat.F32, torch.float16: Q.QuantFormat.F16, torch.bfloat16: BF16}[w.dtype]
        codes = torch.empty(groups, rows, cols, dtype=torch.uint8, device=w.device)
        scales = torch.empty(groups, -(-rows // 128), -(-cols // 128), device=w.device)
        Q.quantize_fp8_weights(type, w.contiguous(), rows, cols, codes, scales, groups=groups,
                               stream=torch.cuda.current_stream().cuda_stream)
        return Q.Fp8Matrix(rows, cols, codes, scales, groups=groups, device=w.device.index or 0)

    def forward(self, x, topk_idx, topk_w):
        """x [T, d] bf16, topk_idx [T, k] int32 (-1: none), topk_w [T, k] f32 ->
        (x + the experts' weighted outputs, what the backward needs)."""
        stream = torch.cuda.current_stream().cuda_stream
        T, k = topk_idx.shape
        n = T * k
        new = dict(device=x.device)
        perm, pos = torch.empty(n, dtype=torch.int32, **new), torch.empty(n, dtype=torch.int32, **new)
        offsets = torch.empty(self.experts + 1, dtype=torch.int32, **new)
        held = offsets[self.experts:]   # how many rows there are, on the device
        x8, h8 = rows8(n, self.d), rows8(n, self.ffn)
        gu = torch.empty(n, 2 * self.ffn, dtype=torch.bfloat16, **new)
        y = torch.empty(n, self.d, dtype=torch.bfloat16, **new)
        out = torch.empty_like(x)
        Q.sort_tokens(topk_idx, T, k, self.experts, perm, pos, offsets, stream=stream)
        Q.gather_rows_fp8(BF16, x, pos, T, k, self.d, *x8, n, stream=stream)
        self.gate_up.product(BF16, *x8, n, gu, offsets, stream=stream)
        Q.swiglu_fp8(BF16, gu, n, self.ffn, *h8, limit=self.limit, n_rows=held, stream=stream)
        self.down.product(BF16, *h8, n, y, offsets, stream=stream)
        Q.combine_rows(BF16, y, n, pos, topk_w, T, k, self.d, out, add=x, stream=stream)
        return out, (pos, offsets, gu, y, topk_w)

    def backward(self, dout, kept):
        """dout [T, d] bf16 -> (dx, dw)."""
        stream = torch.cuda.current_stream().cuda_stream
        pos, offsets, gu, y, w = kept
        T, k = w.shape
        n = T * k
        new = dict(device=dout.device)
        held = offsets[self.experts:]
        dy8, dgu8 = rows8(n, self.d), rows8(n, 2 * self.ffn)
        dh = torch.empty(n, self.ffn, dtype=torch.bfloat16, **new)
        dxr = torch.empty(n, self.d, dtype=torch.bfloat16, **new)
        dx, dw = torch.empty_like(dout), torch.empty(T, k, **new)
        Q.combine_rows_grad_fp8(BF16, dout, y, n, pos, w, T, k, self.d, *dy8, dw, stream=stream)
        self.down.product_t(BF16, *dy8, n, dh, offsets, stream=stream)
        Q.swiglu_fp8_grad(BF16, gu, dh, n, self.ffn, *dgu8, limit=self.limit, n_rows=held, stream=stream)
        self.gate_up.product_t(BF16, *dgu8, n, dxr, offsets, stream=stream)
        # the gradient of the gather, on top of the residual stream's own
        Q.combine_rows(BF16, dxr, n, pos, None, T, k, self.d, dx, add=dout, stream=stream)
        return dx, dw

    def sync(self):
        """Waits and raises what the products met."""
        self.gate_up.sync()
        self.down.sync()

    def close(self):
        self.gate_up.close()
        self.down.close()


def plain(x, idx, w, w_gate_up, w_down, limit=0.0):
    """The layer in plain f32 torch operations, for autograd."""
    out = x
    f = w_down.shape[2]
    for e in range(w_down.shape[0]):
        t, j = (idx == e).nonzero(as_tuple=True)
        if t.numel():
            gu = x[t] @ w_gate_up[e].T
            g, u = gu[:, :f], gu[:, f:]
            if limit:
                g, u = g.clamp(max=limit), u.clamp(-limit, limit)
            out = out.index_add(0, t, w[t, j, None] * ((g * torch.sigmoid(g) * u) @ w_down[e].T))
    return out


def main():
    ap = argparse.ArgumentParser()
    for name, value in (("tokens", 512), ("experts", 32), ("top-k", 8), ("d", 1024), ("ffn", 512)):
        ap.add_argument("--" + name, type=int, default=value)
    a = ap.parse_args()
    g = torch.Generator(device="cuda")
    g.manual_seed(1)

    def randn(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    w13, w2 = randn(a.experts, 2 * a.ffn, a.d) * a.d ** -0.5, randn(a.experts, a.d, a.ffn) * a.ffn ** -0.5
    layer = Fp8Experts(w13, w2)
    top = (randn(a.tokens, a.experts) + randn(a.experts)).topk(a.top_k, 1)
    idx, w = top.indices.int(), torch.softmax(top.values, 1).contiguous()
    x, dout = randn(a.tokens, a.d).bfloat16(), randn(a.tokens, a.d).bfloat16()

    out, kept = layer.forward(x, idx, w)
    dx, dw = layer.backward(dout, kept)
    layer.sync()
    xf, wf = x.float().requires_grad_(), w.clone().requires_grad_()
    want = plain(xf, idx, wf, w13, w2)
    want.backward(dout.float())
    for name, got, ref in (("out", out, want), ("dx", dx, xf.grad), ("dw", dw, wf.grad)):
        ref = ref.detach()
        print(f"{name}: {float((got.float() - ref).norm() / ref.norm()):.2%} from f32 weights and activations")

    start, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    for what, call in (("forward", lambda: layer.forward(x, idx, w)), ("backward", lambda: layer.backward(dout, kept))):
        for _ in range(3):
            call()
        start.record()
        for _ in range(20):
            call()
        end.record()
        torch.cuda.synchronize()
        print(f"{what}: {start.elapsed_time(end) / 20 * 1e3:.1f} us for {a.tokens} tokens")
    layer.close()


if __name__ == "__main__":
    main()
