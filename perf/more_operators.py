"""Measured cases of the operators around experts in 4-bit microscaled floating
point: root-mean-square norm of the residual stream (the residual's addition in
front of it, its output in the activations' type or in 8-bit rows) and its
gradient; the 4-bit product, dense or grouped by expert; the gated product
(gate, up and SwiGLU in one); and the two runs that a layer makes of them:
routed experts from tokens to expert rows, and a dense feed-forward block from
the residual stream to its output.

`run` computes a case in plain torch operations (32 bits, rounded once at the
end), or, with `own` set, through this package's entry points.  Sizes are those
of the package's MoE configurations (d_model 1024 to 7168, 1536 to 14336
columns in an expert, 8 to 256 experts, top-2 to top-8) and odd ones between.

4-bit rows: e2m1 codes, two to a byte (the even column in the low four bits),
one e8m0 scale for each 32 columns, 2^(floor(log2 max|v|) - 2); codes are
rounded to nearest even and saturate at 6.
"""
import torch

own = False

E4M3_MAX = 448.0
MIN_SCALE = 2.0 ** -126
BLOCK8 = 128   # columns of an 8-bit row with one scale
BLOCK4 = 32    # columns of a 4-bit row with one scale
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}


def listed():
    return [
        # one token's decode step: the residual comes in, 8-bit rows for the 8-bit products go out
        {"name": "norm_token", "kind": "norm", "rows": 1, "d": 7168, "type": "f32", "add": True, "fp8": True},
        # the same for a prefill batch
        {"name": "norm_prefill", "kind": "norm", "rows": 4096, "d": 7168, "type": "bf16", "add": True, "fp8": True},
        # fine-tuning on a small, odd batch: gradients of the rows and of the weight
        {"name": "norm_grad_odd", "kind": "norm_grad", "rows": 1021, "d": 2816, "type": "f32", "add": False},
        # fine-tuning, prefill size, on top of the gradient that the residual stream brings
        {"name": "norm_grad_prefill", "kind": "norm_grad", "rows": 4096, "d": 7168, "type": "bf16", "add": True},
        # one token through one matrix, its row quantised on the way
        {"name": "product_token", "kind": "product", "rows": 1, "groups": 1, "N": 4096, "K": 7168, "type": "f32",
         "quantize": True, "skew": 0.0},
        # prefill through one large dense matrix
        {"name": "product_dense", "kind": "product", "rows": 4096, "groups": 1, "N": 28672, "K": 4096, "type": "bf16",
         "quantize": True, "skew": 0.0},
        # prefill through the down matrices of a rank's 32 experts, uneven groups, rows already in 4 bits
        {"name": "product_experts", "kind": "product", "rows": 8192, "groups": 32, "N": 7168, "K": 2048,
         "type": "bf16", "quantize": False, "skew": 0.3},
        # one token through a shared expert's gate and up
        {"name": "gated_token", "kind": "gated", "rows": 1, "groups": 1, "f": 2048, "K": 7168, "type": "f32",
         "limit": 0.0, "skew": 0.0},
        # a batch through the gate and up of 20 experts, an odd number of rows, clamped
        {"name": "gated_batch", "kind": "gated", "rows": 2559, "groups": 20, "f": 1536, "K": 6144, "type": "f16",
         "limit": 7.0, "skew": 0.3},
        # decode of 16 tokens on a rank that holds 32 of 256 experts: most slots belong to other ranks
        {"name": "experts_decode", "kind": "experts", "T": 16, "k": 8, "E": 256, "local": 32, "d": 7168, "f": 2048,
         "type": "bf16", "limit": 0.0},
        # prefill through all of 32 experts
        {"name": "experts_prefill", "kind": "experts", "T": 1024, "k": 8, "E": 32, "local": 32, "d": 7168, "f": 2048,
         "type": "bf16", "limit": 0.0},
        # a dense layer's feed-forward block: residual, norm, gate and up, down
        {"name": "block_dense", "kind": "block", "rows": 2048, "d": 4096, "f": 14336, "type": "bf16", "limit": 0.0},
    ]


def _log(rng, lo, hi, step=1):
    """A size spread over the logarithm of [lo, hi], a multiple of step."""
    v = lo * (hi / lo) ** rng.random()
    return int(min(hi, max(lo, round(v / step) * step)))


def draw(rng):
    kind = rng.choice(["norm", "norm", "norm_grad", "norm_grad", "product", "product", "product", "gated", "gated",
                       "experts", "block"])
    type_ = rng.choice(["f32", "f16", "bf16", "bf16"])
    if kind in ("norm", "norm_grad"):
        c = {"kind": kind, "rows": _log(rng, 1, 4096), "d": _log(rng, 1024, 7168, rng.choice([1, 8, 128])),
             "type": type_, "add": rng.random() < 0.6}
        if kind == "norm":
            c["fp8"] = rng.random() < 0.6
        return c
    limit = rng.choice([0.0, 7.0])
    if kind in ("product", "gated"):
        wide = rng.random() < 0.5
        n, k = _log(rng, 1024, 14336, 1 if rng.random() < 0.3 else 32), _log(rng, 1024, 7168, 32 if wide else 1)
        if kind == "gated":
            n //= 2
        groups = rng.choice([1, 1, 8, 20, 32])
        weights = n * k * (2 if kind == "gated" else 1)
        groups = max(1, min(groups, int(4.7e8 / weights)))   # no more weights than the largest listed case
        rows = max(1, min(_log(rng, 1, 8192), int(4.0e11 / weights)))
        c = {"kind": kind, "rows": rows, "groups": groups, "K": k, "type": type_, "skew": rng.choice([0.0, 0.3])}
        if kind == "product":
            return {**c, "N": n, "quantize": rng.random() < 0.5}
        return {**c, "f": n, "limit": limit}
    type_ = rng.choice(["f16", "bf16"])
    if kind == "block":
        d, f = _log(rng, 1024, 7168, 32), _log(rng, 1024, 14336, 32)
        rows = max(1, min(_log(rng, 1, 4096), int(3.0e11 / (3 * d * f))))
        return {"kind": kind, "rows": rows, "d": d, "f": f, "type": type_, "limit": limit}
    k = rng.choice([2, 6, 8])
    e = rng.choice([32, 64, 160, 256])
    d, f = _log(rng, 1024, 7168, 32), _log(rng, 1024, 2816, 32)
    local = max(1, min(e // rng.choice([1, 2, 4, 8]), int(1.4e9 / (3 * d * f)), 32))
    return {"kind": kind, "T": _log(rng, 16, 8192 // k), "k": k, "E": e, "local": local, "d": d, "f": f, "type": type_,
            "limit": limit}


# ------------------------------------------------------------ inputs


def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _e2m1(v):
    """The 4-bit number nearest to v (ties to even), |v| cut off at 6."""
    a = v.abs()
    step = torch.where(a < 2.0, 0.5, torch.where(a < 4.0, 1.0, 2.0))
    return (torch.round(v / step) * step).clamp(-6.0, 6.0)


def _blocks4(v):
    """v [..., cols] in blocks of 32 columns: (numbers that the codes stand for
    [..., blocks, 32], exponents of the scales [..., blocks]), in 32 bits."""
    b = torch.nn.functional.pad(v.float(), (0, -v.shape[-1] % BLOCK4)).unflatten(-1, (-1, BLOCK4))
    top = b.abs().amax(-1)
    exp = torch.where(top > 0, torch.frexp(top).exponent - 3, -127).clamp_min(-127)
    return _e2m1(torch.ldexp(b, -exp[..., None])), exp


def _pack(v):
    """v [..., cols] as packed codes [..., 16 blocks] and scales [..., blocks], bytes both."""
    q, exp = _blocks4(v)
    a = q.abs()
    index = torch.where(a < 2.0, 2.0 * a, torch.where(a < 4.0, a + 2.0, 0.5 * a + 4.0)).to(torch.uint8)
    code = index | (torch.signbit(q).to(torch.uint8) << 3)
    return (code[..., 0::2] | (code[..., 1::2] << 4)).flatten(-2), (exp + 127).to(torch.uint8)


def _unpack(codes, scales, cols):
    """The 32-bit values of `cols` columns of packed codes and scales."""
    code = torch.stack([codes & 15, codes >> 4], -1).flatten(-2)
    a = (code & 7).float()
    v = torch.where(a < 4.0, 0.5 * a, torch.where(a < 6.0, a - 2.0, 2.0 * a - 8.0)) * torch.where(code > 7, -1.0, 1.0)
    v = torch.ldexp(v.unflatten(-1, (-1, BLOCK4)), scales[..., None].int() - 127)
    return v.flatten(-2)[..., :cols]


def _rounded4(v):
    """v after a way through 4-bit rows, in 32 bits."""
    q, exp = _blocks4(v)
    return torch.ldexp(q, exp[..., None]).flatten(-2)[..., :v.shape[-1]]


def _weights(s, name, groups, rows, cols, g):
    """Packed random matrices, and with `own` the package's handle of them."""
    codes = torch.empty(groups, rows, 16 * -(-cols // BLOCK4), dtype=torch.uint8, device="cuda")
    scales = torch.empty(groups, rows, -(-cols // BLOCK4), dtype=torch.uint8, device="cuda")
    for i in range(groups):
        codes[i], scales[i] = _pack(0.02 * torch.randn(rows, cols, generator=g, device="cuda"))
    if own:
        s[name] = s["q"].Fp4Matrix(rows, cols, codes, scales, groups=groups)
    else:
        s[name] = (codes, scales)


def _rows4(rows, cols):
    """Room for 4-bit rows."""
    return (torch.zeros(rows, 16 * -(-cols // BLOCK4), dtype=torch.uint8, device="cuda"),
            torch.zeros(rows, -(-cols // BLOCK4), dtype=torch.uint8, device="cuda"))


def _share(s, rows, groups, skew, g):
    """How the rows are spread over the groups."""
    share = torch.softmax(skew * torch.randn(groups, generator=g, device="cuda"), 0)
    _members(s, torch.multinomial(share, rows, True, generator=g).sort().values, groups)


def _members(s, member, groups):
    """The groups' offsets, and what the plain form goes by: the groups that
    have rows and each row's place in its group."""
    counts = torch.bincount(member, minlength=groups)
    s["offsets"] = torch.zeros(groups + 1, dtype=torch.int32, device="cuda")
    s["offsets"][1:] = counts.cumsum(0)
    s["used"] = counts.nonzero()[:, 0]
    s["member"] = torch.searchsorted(s["used"], member)
    s["place"] = torch.arange(member.numel(), device="cuda") - s["offsets"][member].long()
    s["most"] = int(counts.max())


def prepare(case, seed):
    g = _generator(seed)
    dev = {"device": "cuda"}
    s = {"case": dict(case), "type": TYPES[case["type"]]}
    if own:
        s["q"] = _package()
        s["t"] = {"f32": s["q"].QuantFormat.F32, "f16": s["q"].QuantFormat.F16, "bf16": s["q"].QuantFormat.BF16}[
            case["type"]]
    kind = case["kind"]

    def rows_of(rows, cols, scale=1.0):
        return (scale * torch.randn(rows, cols, generator=g, **dev)).to(s["type"])

    def empty(rows, cols):
        return torch.empty(rows, cols, dtype=s["type"], **dev)

    if kind in ("norm", "norm_grad", "block"):
        rows, d = case["rows"], case["d"]
        s["eps"] = 1e-5
        s["w"] = 1.0 + 0.2 * torch.randn(d, generator=g, **dev)
        s["x"] = rows_of(rows, d, 2.0)
        if kind == "block" or case["add"]:
            s["add"] = rows_of(rows, d)
            s["sum"] = empty(rows, d)
    if kind == "norm":
        if case["fp8"]:
            s["out"] = torch.empty(rows, d, dtype=torch.float8_e4m3fn, **dev)
            s["scales"] = torch.empty(rows, -(-d // BLOCK8), **dev)
        else:
            s["out"] = empty(rows, d)
    elif kind == "norm_grad":
        s["dy"] = rows_of(rows, d)
        s["out"] = empty(rows, d)
        s["dw"] = torch.empty(d, **dev)
        if own:
            s["work"] = torch.empty(s["q"].rms_norm_grad_work(rows, d), **dev)
    elif kind == "block":
        _weights(s, "gate_up", 1, 2 * case["f"], d, g)
        _weights(s, "down", 1, d, case["f"], g)
        s["x4"], s["h4"] = _rows4(rows, d), _rows4(rows, case["f"])
        s["out"] = empty(rows, d)
    elif kind in ("product", "gated"):
        rows, k = case["rows"], case["K"]
        n = case["N"] if kind == "product" else 2 * case["f"]
        _weights(s, "matrix", case["groups"], n, k, g)
        _share(s, rows, case["groups"], case["skew"], g)
        s["x"] = rows_of(rows, k)
        s["x4"] = _rows4(rows, k)
        if not case.get("quantize"):
            s["x4"] = _pack(s["x"])
        s["out"] = empty(rows, case["N"] if kind == "product" else case["f"])
    else:
        t, k, e, local, d, f = (case[n] for n in ("T", "k", "E", "local", "d", "f"))
        # top-k experts with an uneven load; another rank's have no position here
        logits = torch.randn(t, e, generator=g, **dev) + torch.randn(e, generator=g, **dev)
        a = logits.topk(k, 1).indices.reshape(-1)
        key = torch.where(a < local, a, torch.full_like(a, local))
        perm = torch.sort(key, stable=True).indices
        held = key < local
        pos = torch.empty_like(perm)
        pos[perm] = torch.arange(t * k, device="cuda")
        s["pos"] = torch.where(held, pos, -1).int()
        _members(s, key[perm][:int(held.sum())], local)
        s["token"] = (perm // k)[:s["member"].numel()]
        _weights(s, "gate_up", local, 2 * f, d, g)
        _weights(s, "down", local, d, f, g)
        s["x"] = rows_of(t, d)
        s["x4"], s["h4"] = _rows4(t * k, d), _rows4(t * k, f)
        s["out"] = torch.zeros(t * k, d, dtype=s["type"], **dev)
    return s


def _package():
    import qauntrunner_b200
    return qauntrunner_b200


# ------------------------------------------------------------ the operators


def run(s):
    return _run_own(s) if own else _run_plain(s)


def _run_own(s):
    q, c, t = s["q"], s["case"], s["t"]
    stream = torch.cuda.current_stream().cuda_stream
    kind = c["kind"]
    if kind == "norm":
        add, total = s.get("add"), s.get("sum")
        out = {} if total is None else {"sum": total}
        if c["fp8"]:
            q.rms_norm_fp8(t, s["x"], c["rows"], c["d"], s["w"], s["eps"], s["out"], s["scales"], add=add, sum=total,
                           stream=stream)
            return {**out, "codes": s["out"], "scales": s["scales"]}
        q.rms_norm(t, s["x"], c["rows"], c["d"], s["w"], s["eps"], s["out"], add=add, sum=total, stream=stream)
        return {**out, "y": s["out"]}
    if kind == "norm_grad":
        q.rms_norm_grad(t, s["dy"], s["x"], c["rows"], c["d"], s["w"], s["eps"], s["out"], dw=s["dw"], work=s["work"],
                        add=s.get("add"), stream=stream)
        return {"dx": s["out"], "dw": s["dw"]}
    if kind == "block":
        rows = c["rows"]
        q.rms_norm_fp4(t, s["x"], rows, c["d"], s["w"], s["eps"], *s["x4"], add=s["add"], sum=s["sum"], stream=stream)
        s["gate_up"].swiglu_fp4(*s["x4"], rows, *s["h4"], limit=c["limit"], stream=stream)
        s["down"].product(t, *s["h4"], rows, s["out"], stream=stream)
        return {"sum": s["sum"], "y": s["out"]}
    if kind == "experts":
        n = c["T"] * c["k"]
        q.gather_rows_fp4(t, s["x"], s["pos"], c["T"], c["k"], c["d"], *s["x4"], n, stream=stream)
        s["gate_up"].swiglu_fp4(*s["x4"], n, *s["h4"], offsets=s["offsets"], limit=c["limit"], stream=stream)
        s["down"].product(t, *s["h4"], n, s["out"], offsets=s["offsets"], stream=stream)
        return s["out"]
    if kind == "gated":
        s["matrix"].swiglu(t, *s["x4"], c["rows"], s["out"], offsets=s["offsets"], limit=c["limit"], stream=stream)
        return s["out"]
    if c["quantize"]:
        q.quantize_fp4(t, s["x"], c["rows"], c["K"], *s["x4"], stream=stream)
    s["matrix"].product(t, *s["x4"], c["rows"], s["out"], offsets=s["offsets"], stream=stream)
    return s["out"]


def _norm(s):
    """(the sum in its type, its norm in 32 bits)."""
    total = s["x"]
    if "add" in s:
        total = (total.float() + s["add"].float()).to(s["type"])
    v = total.float()
    return total, v * torch.rsqrt(v.square().mean(1, keepdim=True) + s["eps"]) * s["w"]


def _grouped(s, x, matrix):
    """x [rows, K] times each row's own matrix, in 32 bits."""
    codes, scales = matrix
    if codes.shape[0] == 1:
        return x @ _unpack(codes[0], scales[0], x.shape[1]).T
    w = _unpack(codes[s["used"]], scales[s["used"]], x.shape[1])
    padded = torch.zeros(w.shape[0], s["most"], x.shape[1], device="cuda")
    padded[s["member"], s["place"]] = x
    return torch.bmm(padded, w.transpose(1, 2))[s["member"], s["place"]]


def _swiglu(gu, limit):
    gate, up = gu.chunk(2, 1)
    lim = limit or float("inf")
    gate, up = gate.clamp(max=lim), up.clamp(-lim, lim)
    return gate / (1.0 + torch.exp(-gate)) * up


def _run_plain(s):
    c, kind = s["case"], s["case"]["kind"]
    if kind == "norm":
        total, y = _norm(s)
        out = {"sum": total} if c["add"] else {}
        if not c["fp8"]:
            return {**out, "y": y.to(s["type"])}
        b = torch.nn.functional.pad(y, (0, -c["d"] % BLOCK8)).unflatten(1, (-1, BLOCK8))
        scales = (b.abs().amax(-1) / torch.full((), E4M3_MAX, device="cuda")).clamp_min(MIN_SCALE)
        codes = (b / scales[..., None]).flatten(1)[:, :c["d"]].to(torch.float8_e4m3fn)
        return {**out, "codes": codes, "scales": scales}
    if kind == "norm_grad":
        x, dy = s["x"].float(), s["dy"].float()
        inv = torch.rsqrt(x.square().mean(1, keepdim=True) + s["eps"])
        n, g = x * inv, dy * s["w"]
        dx = inv * (g - n * (g * n).mean(1, keepdim=True))
        return {"dx": (dx + s["add"].float() if c["add"] else dx).to(s["type"]), "dw": (dy * n).sum(0)}
    if kind == "block":
        total, y = _norm(s)
        h = _swiglu(_grouped(s, _rounded4(y), s["gate_up"]), c["limit"])
        return {"sum": total, "y": _grouped(s, _rounded4(h), s["down"]).to(s["type"])}
    if kind == "experts":
        x = _rounded4(s["x"])[s["token"]]
        h = _swiglu(_grouped(s, x, s["gate_up"]), c["limit"])
        out = torch.zeros_like(s["out"])
        out[:x.shape[0]] = _grouped(s, _rounded4(h), s["down"]).to(s["type"])
        return out
    if kind == "gated":
        return _swiglu(_grouped(s, _unpack(*s["x4"], c["K"]), s["matrix"]), c["limit"]).to(s["type"])
    x = _rounded4(s["x"]) if c["quantize"] else _unpack(*s["x4"], c["K"])
    return _grouped(s, x, s["matrix"]).to(s["type"])


# ------------------------------------------------------------ what a pass cannot do without


def work(case):
    kind, b = case["kind"], SIZE[case["type"]]

    def row4(cols):
        return 17 * -(-cols // BLOCK4)

    def matrices(groups, rows, n, k):
        """Bytes of the matrices that have a row, on average."""
        return groups * (1.0 - (1.0 - 1.0 / groups) ** rows) * n * row4(k)

    if kind in ("norm", "norm_grad"):
        rows, d = case["rows"], case["d"]
        if kind == "norm":
            out = d + 4 * -(-d // BLOCK8) if case["fp8"] else d * b
            return {"bytes": 4 * d + rows * (d * b * (3 if case["add"] else 1) + out), "flops": 5 * rows * d}
        return {"bytes": 8 * d + rows * d * b * (4 if case["add"] else 3), "flops": 12 * rows * d}
    if kind == "block":
        rows, d, f = case["rows"], case["d"], case["f"]
        return {"bytes": 4 * d + rows * d * b * 4 + 2 * f * row4(d) + d * row4(f), "flops": 6.0 * rows * d * f}
    if kind == "experts":
        t, k, d, f = case["T"], case["k"], case["d"], case["f"]
        rows = t * k * case["local"] / case["E"]
        return {"bytes": 4 * t * k + t * d * b + rows * d * b + matrices(case["local"], rows, 2 * f, d) +
                matrices(case["local"], rows, d, f), "flops": 6.0 * rows * d * f}
    rows, k = case["rows"], case["K"]
    n = case["N"] if kind == "product" else 2 * case["f"]
    taken = k * b if case.get("quantize") else row4(k)
    return {"bytes": matrices(case["groups"], rows, n, k) + rows * (taken + (n if kind == "product" else case["f"]) * b),
            "flops": 2.0 * rows * n * k}


# ------------------------------------------------------------ the definitions in 64 bits

_E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _values64(codes, scales, cols):
    """What packed codes and scales stand for."""
    v = torch.empty(*codes.shape[:-1], 2 * codes.shape[-1], dtype=torch.float64, device=codes.device)
    for half in (0, 1):
        code = (codes >> (4 * half)) & 15
        part = torch.zeros(codes.shape, dtype=torch.float64, device=codes.device)
        for i, number in enumerate(_E2M1):
            part[code == i] = number
            part[code == i + 8] = -number
        v[..., half::2] = part
    size = torch.pow(2.0, scales.to(torch.float64) - 127.0)
    return (v * size.repeat_interleave(BLOCK4, -1))[..., :cols]


def _through64(v):
    """v [rows, cols] after a way through 4-bit rows: the nearest number of each
    block's eight magnitudes, the one with the even code where two are as near."""
    out = torch.empty_like(v)
    table = torch.tensor(_E2M1, dtype=torch.float64, device=v.device)
    middle = (table[1:] + table[:-1]) / 2
    odd = torch.arange(7, device=v.device) % 2 == 1   # a tie above an odd code goes up
    for j in range(0, v.shape[1], BLOCK4):
        part = v[:, j:j + BLOCK4]
        top = part.abs().max(1, keepdim=True).values
        size = torch.pow(2.0, torch.clamp(torch.floor(torch.log2(top.clamp_min(1e-300))) - 2.0, min=-127.0))
        a = part.abs() / size
        index = torch.zeros(part.shape, dtype=torch.long, device=v.device)
        for i in range(7):
            index += (a >= middle[i]) if odd[i] else (a > middle[i])
        out[:, j:j + BLOCK4] = torch.sign(part) * table[index] * size
    return out


def _e4m3(v):
    """The e4m3 number nearest to v (ties to even), in 64 bits."""
    _, e = torch.frexp(v)
    step = torch.ldexp(torch.ones_like(v), (e - 1).clamp_min(-6) - 3)
    return (torch.round(v / step) * step).clamp(-E4M3_MAX, E4M3_MAX)


def _each(s, x, matrix):
    """Every group's rows of x times its matrix."""
    codes, scales = matrix
    edges = s["offsets"].tolist() if "offsets" in s else [0, x.shape[0]]
    parts = []
    for i in range(codes.shape[0]):
        a, b = edges[i], edges[i + 1]
        if a < b:
            parts.append(torch.matmul(x[a:b], _values64(codes[i], scales[i], x.shape[1]).T))
    return torch.cat(parts) if parts else torch.zeros(0, codes.shape[1], dtype=torch.float64, device="cuda")


def _gate64(gu, limit):
    f = gu.shape[1] // 2
    g, u = gu[:, :f], gu[:, f:]
    if limit:
        g, u = torch.minimum(g, torch.full_like(g, limit)), u.clamp(-limit, limit)
    return g * torch.sigmoid(g) * u


def exact(case, seed):
    if work(case)["flops"] > 2e12:
        return None
    s = prepare(case, seed)
    kind, f64 = case["kind"], torch.float64
    if kind in ("norm", "block"):
        x = s["x"].to(f64)
        whole = x + s["add"].to(f64) if "add" in s else x
        v = whole.to(s["type"]).to(f64)   # the norm is that of the sum as it is stored
        y = s["w"].to(f64) * v / torch.sqrt(torch.einsum("rd,rd->r", v, v) / case["d"] + s["eps"])[:, None]
        out = {"sum": whole} if "add" in s else {}
        if kind == "block":
            h = _gate64(_each(s, _through64(y), s["gate_up"]), case["limit"])
            return {**out, "y": _each(s, _through64(h), s["down"])}
        if not case["fp8"]:
            return {**out, "y": y}
        codes, scales = torch.empty_like(y), torch.empty(s["scales"].shape, dtype=f64, device="cuda")
        for j in range(scales.shape[1]):
            part = y[:, j * BLOCK8:(j + 1) * BLOCK8]
            scales[:, j] = torch.clamp(part.abs().max(1).values / E4M3_MAX, min=MIN_SCALE)
            codes[:, j * BLOCK8:(j + 1) * BLOCK8] = _e4m3(part / scales[:, j:j + 1])
        return {**out, "codes": codes, "scales": scales}
    if kind == "norm_grad":
        x, dy, w = s["x"].to(f64), s["dy"].to(f64), s["w"].to(f64)
        size = torch.einsum("rd,rd->r", x, x) / case["d"] + s["eps"]
        along = torch.einsum("rd,rd,d->r", dy, x, w) / case["d"]
        dx = dy * w / torch.sqrt(size)[:, None] - x * (along * size ** -1.5)[:, None]
        if case["add"]:
            dx = dx + s["add"].to(f64)
        return {"dx": dx, "dw": torch.einsum("rd,rd,r->d", dy, x, size ** -0.5)}
    if kind == "experts":
        x = _through64(s["x"].to(f64))[s["token"]]
        out = torch.zeros(s["out"].shape, dtype=f64, device="cuda")
        h = _gate64(_each(s, x, s["gate_up"]), case["limit"])
        out[:x.shape[0]] = _each(s, _through64(h), s["down"])
        return out
    x = _through64(s["x"].to(f64)) if case.get("quantize") else _values64(*s["x4"], case["K"])
    y = _each(s, x, s["matrix"])
    return _gate64(y, case["limit"]) if kind == "gated" else y
