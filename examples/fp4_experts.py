"""An MoE layer's experts in 4-bit microscaled floating point, as a server runs
them: the residual's addition and the norm, tokens sorted by expert into 4-bit
rows, gate and up with SwiGLU in one product, down, and back to the tokens.

    python examples/fp4_experts.py [--tokens 512] [--experts 32] [--top-k 8] [--d 1024] [--ffn 512]

The weights (gate and up as one matrix of each expert, and down) are quantised
once, with a scale for each 32 columns, and kept in HBM.  DenseFfn is the same
without experts: a dense layer, or the expert that all tokens share.
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import qauntrunner_b200 as Q  # noqa: E402

BF16 = Q.QuantFormat.BF16
TYPES = {torch.float32: Q.QuantFormat.F32, torch.float16: Q.QuantFormat.F16, torch.bfloat16: BF16}


def rows4(rows, cols, device="cuda"):
    """Room for 4-bit rows: codes and scales."""
    blocks = -(-cols // 32)
    return (torch.empty(rows, 16 * blocks, dtype=torch.uint8, device=device),
            torch.empty(rows, blocks, dtype=torch.uint8, device=device))


def matrix(w):
    """w [groups, rows, cols] on the device as a 4-bit matrix."""
    groups, rows, cols = w.shape
    codes, scales = rows4(groups * rows, cols, w.device)
    Q.quantize_fp4(TYPES[w.dtype], w.contiguous(), groups * rows, cols, codes, scales,
                   stream=torch.cuda.current_stream().cuda_stream)
    return Q.Fp4Matrix(rows, cols, codes, scales, groups=groups)


class Fp4Experts:
    """w_gate_up [experts, 2 ffn, d], w_down [experts, d, ffn], norm_w [d] f32:
    tensors on the device.  Activations are bf16."""

    def __init__(self, w_gate_up, w_down, norm_w, eps=1e-5, limit=0.0):
        self.experts, two_f, self.d = w_gate_up.shape
        self.ffn, self.limit, self.w, self.eps = two_f // 2, limit, norm_w, eps
        self.gate_up, self.down = matrix(w_gate_up), matrix(w_down)

    def forward(self, x, residual, route):
        """s = x + residual -> s + the weighted outputs of the experts for norm(s).
        route(y) gives topk_idx [T, k] int32 (-1: none) and topk_w [T, k] f32."""
        stream = torch.cuda.current_stream().cuda_stream
        T = x.shape[0]
        total, y = torch.empty_like(x), torch.empty_like(x)
        Q.rms_norm(BF16, x, T, self.d, self.w, self.eps, y, add=residual, sum=total, stream=stream)
        topk_idx, topk_w = route(y)
        k = topk_idx.shape[1]
        n = T * k
        perm, pos = (torch.empty(n, dtype=torch.int32, device=x.device) for _ in range(2))
        offsets = torch.empty(self.experts + 1, dtype=torch.int32, device=x.device)
        x4, h4 = rows4(n, self.d, x.device), rows4(n, self.ffn, x.device)
        rows, out = torch.empty(n, self.d, dtype=x.dtype, device=x.device), torch.empty_like(x)
        Q.sort_tokens(topk_idx, T, k, self.experts, perm, pos, offsets, stream=stream)
        Q.gather_rows_fp4(BF16, y, pos, T, k, self.d, *x4, n, stream=stream)
        self.gate_up.swiglu_fp4(*x4, n, *h4, offsets=offsets, limit=self.limit, stream=stream)
        self.down.product(BF16, *h4, n, rows, offsets=offsets, stream=stream)
        Q.combine_rows(BF16, rows, n, pos, topk_w, T, k, self.d, out, add=total, stream=stream)
        return out

    def sync(self):
        """Waits and raises what the products met."""
        self.gate_up.sync()
        self.down.sync()

    def close(self):
        self.gate_up.close()
        self.down.close()


class DenseFfn:
    """w_gate_up [2 ffn, d], w_down [d, ffn], norm_w [d] f32."""

    def __init__(self, w_gate_up, w_down, norm_w, eps=1e-5, limit=0.0):
        self.ffn, self.d = w_gate_up.shape[0] // 2, w_gate_up.shape[1]
        self.limit, self.w, self.eps = limit, norm_w, eps
        self.gate_up, self.down = matrix(w_gate_up[None]), matrix(w_down[None])

    def forward(self, x, residual):
        """s = x + residual -> (s, the block's output for norm(s)); the next norm adds them."""
        stream = torch.cuda.current_stream().cuda_stream
        T = x.shape[0]
        total, out = torch.empty_like(x), torch.empty_like(x)
        x4, h4 = rows4(T, self.d, x.device), rows4(T, self.ffn, x.device)
        Q.rms_norm_fp4(BF16, x, T, self.d, self.w, self.eps, *x4, add=residual, sum=total, stream=stream)
        self.gate_up.swiglu_fp4(*x4, T, *h4, limit=self.limit, stream=stream)
        self.down.product(BF16, *h4, T, out, stream=stream)
        return total, out

    def close(self):
        self.gate_up.close()
        self.down.close()


def plain(x, residual, route, w_gate_up, w_down, norm_w, eps=1e-5):
    """The layer in plain f32 torch operations."""
    s = x + residual
    y = s * torch.rsqrt(s.square().mean(1, keepdim=True) + eps) * norm_w
    idx, w = route(y)
    out, f = s, w_down.shape[2]
    for e in range(w_down.shape[0]):
        t, j = (idx == e).nonzero(as_tuple=True)
        if t.numel():
            gu = y[t] @ w_gate_up[e].T
            out = out.index_add(0, t, w[t, j, None] * ((torch.nn.functional.silu(gu[:, :f]) * gu[:, f:]) @ w_down[e].T))
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
    norm_w = 1 + 0.1 * randn(a.d)
    layer = Fp4Experts(w13, w2, norm_w)
    top = (randn(a.tokens, a.experts) + randn(a.experts)).topk(a.top_k, 1)
    routed = top.indices.int(), torch.softmax(top.values, 1).contiguous()
    x, r = randn(a.tokens, a.d).bfloat16(), randn(a.tokens, a.d).bfloat16()
    out = layer.forward(x, r, lambda y: routed)
    layer.sync()
    want = plain(x.float(), r.float(), lambda y: routed, w13, w2, norm_w)
    print(f"{float((out.float() - want).norm() / want.norm()):.2%} from f32 weights and activations")
    start, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    for _ in range(3):
        layer.forward(x, r, lambda y: routed)
    start.record()
    for _ in range(20):
        layer.forward(x, r, lambda y: routed)
    end.record()
    torch.cuda.synchronize()
    print(f"{start.elapsed_time(end) / 20 * 1e3:.1f} us for {a.tokens} tokens")
    layer.close()


if __name__ == "__main__":
    main()
