"""Plain forms of the 4-bit operators and of the norm for the tests, in 64 bits
and exact steps, on the CPU."""
import torch

E2M1 = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)


def blocks(n):
    return -(-n // 32)


def quantize(v):
    """(codes, scales), bytes, of the rows v [rows, cols], by comparison with the
    middles between neighbouring numbers (64 bits, so every step is exact)."""
    v = v.double()
    rows, cols = v.shape
    nb = blocks(cols)
    p = torch.zeros(rows, 32 * nb, dtype=torch.float64)
    p[:, :cols] = v
    b = p.reshape(rows, nb, 32)
    top = b.abs().amax(2)
    exp = (torch.frexp(top).exponent - 3).clamp_min(-127)
    exp = torch.where(top == 0, -127, exp)
    bad = ~torch.isfinite(b).all(2)
    scales = torch.where(bad, 255, exp + 127).to(torch.uint8)
    a = (b.abs() / torch.pow(2.0, exp.double())[..., None])
    middle = (E2M1[1:] + E2M1[:-1]) / 2
    index = torch.zeros(b.shape, dtype=torch.int64)
    for i in range(7):   # a tie goes to the even code
        index += (a >= middle[i]) if i % 2 else (a > middle[i])
    code = index | (torch.signbit(b).long() << 3)
    code[bad] = 0
    code = code.reshape(rows, -1).to(torch.uint8)
    return code[:, 0::2] | (code[:, 1::2] << 4), scales


def values(codes, scales, cols):
    """What codes and scales stand for, in 64 bits (NaN where the scale is 255)."""
    code = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).long()
    v = E2M1[code & 7] * torch.where(code > 7, -1.0, 1.0)
    s = torch.pow(2.0, scales.double() - 127.0)
    s = torch.where(scales == 255, float("nan"), s)
    return (v * s.repeat_interleave(32, -1))[..., :cols]


def random_rows(g, rows, cols, spread=3):
    """Random codes (of all sixteen) and scales around 1, `spread` powers of two
    either way; what lies past the last column is 0."""
    nb = blocks(cols)
    code = torch.randint(0, 16, (rows, 32 * nb), generator=g, dtype=torch.uint8)
    code[:, cols:] = 0
    scales = torch.randint(127 - spread, 128 + spread, (rows, nb), generator=g, dtype=torch.uint8)
    return code[:, 0::2] | (code[:, 1::2] << 4), scales


def gate(y, limit):
    """h of gate's and up's sums side by side, in 64 bits."""
    f = y.shape[1] // 2
    g, u = y[:, :f].double(), y[:, f:].double()
    if limit:
        g, u = g.clamp(max=limit), u.clamp(-limit, limit)
    return g * torch.sigmoid(g) * u


def norm(s, w, eps):
    """y of the stored sums s, in 64 bits."""
    s = s.double()
    y = s / torch.sqrt((s * s).mean(1, keepdim=True) + eps)
    return y if w is None else y * w.double()


def norm_grad(dy, s, w, eps, add):
    """(dx, dw, how large the parts of dx's and of dw's sums are)."""
    dy, s = dy.double(), s.double()
    inv = 1.0 / torch.sqrt((s * s).mean(1, keepdim=True) + eps)
    n = s * inv
    g = dy if w is None else dy * w.double()
    along = (g * n).mean(1, keepdim=True)
    dx = inv * (g - n * along)
    size = inv * (g.abs() + n.abs() * (g * n).abs().mean(1, keepdim=True))
    if add is not None:
        dx = dx + add.double()
        size = size + add.double().abs()
    return dx, (dy * n).sum(0), size, (dy * n).abs().sum(0)
