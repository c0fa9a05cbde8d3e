"""Plain forms of the 8-bit expert operators for the tests, in 64 bits (sums)
and in exact integers (orders, codes), on the CPU."""
import torch

U = 2.0 ** -24                                  # unit roundoff of f32
ROUND = {0: 2.0 ** -24, 1: 2.0 ** -11, 2: 2.0 ** -8}   # of the activation types F32, F16, BF16
HALF_STEP = {0: 2.0 ** -150, 1: 2.0 ** -25, 2: 2.0 ** -134}   # half the distance of their denormals
DTYPE = {0: torch.float32, 1: torch.float16, 2: torch.bfloat16}
MIN_SCALE = 2.0 ** -126


def order(idx, first, experts):
    """(perm, pos, offsets) by Python's stable sort."""
    a = [(int(e) - first, i) for i, e in enumerate(idx.reshape(-1).tolist())]
    held = sorted((e, i) for e, i in a if 0 <= e < experts)
    perm = [i for _, i in held] + [-1] * (len(a) - len(held))
    pos = [-1] * len(a)
    for p, (_, i) in enumerate(held):
        pos[i] = p
    offsets = [sum(1 for e, _ in held if e < x) for x in range(experts + 1)]
    return perm, pos, offsets


def blocks(n):
    return -(-n // 128)


def quantize(v, across=1):
    """(codes as uint8, scales f32) of v [rows, cols] f32: the operations the
    kernels are defined by, which are exact or rounded once each."""
    v = v.float()
    rows, cols = v.shape
    codes = torch.zeros(rows, cols, dtype=torch.uint8)
    scales = torch.zeros(-(-rows // across), blocks(cols))
    for i in range(scales.shape[0]):
        for j in range(scales.shape[1]):
            b = v[i * across:(i + 1) * across, j * 128:(j + 1) * 128]
            s = (b.abs().max() / 448.0).clamp_min(MIN_SCALE)
            scales[i, j] = s
            codes[i * across:(i + 1) * across, j * 128:(j + 1) * 128] = (b / s).to(torch.float8_e4m3fn).view(torch.uint8)
    return codes, scales


def values(codes, scales, across=1):
    """What codes and scales stand for, in 64 bits."""
    rows, cols = codes.shape
    s = scales.double().repeat_interleave(across, 0)[:rows].repeat_interleave(128, 1)[:, :cols]
    return codes.view(torch.float8_e4m3fn).float().double() * s


def code_bound(v, scales):
    """Half the distance of neighbouring codes around v (64 bits)."""
    s = scales.double().repeat_interleave(128, 1)[:, :v.shape[1]]
    return torch.maximum(v.abs() * 2.0 ** -4, s * 2.0 ** -10)


def swiglu(gate, up, limit):
    g, u = gate.double(), up.double()
    if limit:
        g, u = g.clamp(max=limit), u.clamp(-limit, limit)
    return g * torch.sigmoid(g) * u


def swiglu_grad(gate, up, dh, limit):
    """(dg, du, how large the parts of dg's sum are)."""
    gate, up, dh = gate.double(), up.double(), dh.double()
    g = gate.clamp(max=limit) if limit else gate
    u = up.clamp(-limit, limit) if limit else up
    s = torch.sigmoid(g)
    dg = dh * u * s * (1.0 + g * (1.0 - s))
    du = dh * g * s
    if limit:
        dg = torch.where(gate > limit, 0.0, dg)
        du = torch.where(up.abs() > limit, 0.0, du)
    return dg, du, dh.abs() * u.abs() * s * (1.0 + g.abs())


def combine(rows, pos, w, add):
    """(out, sum of the magnitudes) in 64 bits; pos, w [T, k]."""
    T, k = pos.shape
    out = torch.zeros(T, rows.shape[1], dtype=torch.float64) if add is None else add.double().clone()
    size = out.abs()
    for t in range(T):
        for j in range(k):
            p = int(pos[t, j])
            if 0 <= p < rows.shape[0]:
                v = rows[p].double() * (1.0 if w is None else float(w[t, j]))
                out[t] += v
                size[t] += v.abs()
    return out, size
