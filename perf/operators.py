"""Measured cases of the FP8 expert operators: tokens sorted by expert and
back (with their gradients), the 8-bit floating-point product with a scale for
each block of 128 (dense, grouped by expert, and transposed for the input
gradient), and SwiGLU into 8-bit rows with its gradient.

`run` computes a case in plain torch operations (32 bits, rounded once at the
end), or, with `own` set, through this package's entry points.  Sizes are those
of the package's MoE configurations (d_model 1024 to 7168, experts of 1536 to
14336 columns, 8 to 256 experts, top-2 to top-8) and odd ones between them.

Conventions of the outputs: 8-bit codes come back as torch.float8_e4m3fn with
their f32 scales beside them; a row or an assignment that does not exist has
position -1 and leaves its output rows as they were (zero here).
"""
import torch

own = False

E4M3_MAX = 448.0
MIN_SCALE = 2.0 ** -126
BLOCK = 128
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}


def listed():
    return [
        # one token enters the experts: the decode step of the 256-expert layer
        {"name": "order_decode", "kind": "order", "T": 1, "k": 8, "E": 256, "local": 256, "d": 7168, "type": "f32",
         "fp8": True},
        # a prefill batch of the same layer, bf16 activations
        {"name": "order_prefill", "kind": "order", "T": 4096, "k": 8, "E": 256, "local": 256, "d": 7168,
         "type": "bf16", "fp8": True},
        # one of eight expert-parallel ranks: most assignments belong to the others; rows stay f16
        {"name": "order_share", "kind": "order", "T": 1021, "k": 8, "E": 160, "local": 20, "d": 6144, "type": "f16",
         "fp8": False},
        # expert rows back to their tokens on top of the residual stream
        {"name": "combine_residual", "kind": "combine", "T": 2048, "k": 6, "E": 64, "local": 64, "d": 4096,
         "type": "bf16", "add": True},
        # fine-tuning: gradient of the combine, its rows in 8 bits for the transposed product
        {"name": "combine_grad", "kind": "combine_grad", "T": 4096, "k": 8, "E": 256, "local": 256, "d": 7168,
         "type": "bf16", "fp8": True},
        # one token through one matrix (a shared expert's gate and up)
        {"name": "product_token", "kind": "product", "rows": 1, "groups": 1, "N": 4096, "K": 7168, "type": "f32",
         "back": False, "skew": 0.0},
        # decode of 16 tokens on a rank that holds 32 experts
        {"name": "product_decode", "kind": "product", "rows": 16, "groups": 32, "N": 4096, "K": 7168, "type": "bf16",
         "back": False, "skew": 0.0},
        # prefill through one large dense matrix
        {"name": "product_dense", "kind": "product", "rows": 4096, "groups": 1, "N": 28672, "K": 4096, "type": "bf16",
         "back": False, "skew": 0.0},
        # prefill through a rank's 32 experts, uneven groups
        {"name": "product_experts", "kind": "product", "rows": 8192, "groups": 32, "N": 4096, "K": 7168,
         "type": "bf16", "back": False, "skew": 0.3},
        # fine-tuning: input gradient through 20 experts, an odd number of rows
        {"name": "product_back", "kind": "product", "rows": 2559, "groups": 20, "N": 2816,
         "K": 6144, "type": "bf16", "back": True, "skew": 0.3},
        # a small batch of a small layer, f32 all along
        {"name": "swiglu_small", "kind": "swiglu", "rows": 64, "f": 2816, "type": "f32", "limit": 0.0},
        # fine-tuning: gradient of the clamped SwiGLU over a prefill batch's rows
        {"name": "swiglu_grad", "kind": "swiglu_grad", "rows": 16384, "f": 2048, "type": "bf16", "limit": 7.0},
    ]


def _log(rng, lo, hi, step=1):
    """A size spread over the logarithm of [lo, hi], a multiple of step."""
    v = lo * (hi / lo) ** rng.random()
    return int(min(hi, max(lo, round(v / step) * step)))


def draw(rng):
    kind = rng.choice(["order", "combine", "combine_grad", "product", "product", "product", "swiglu", "swiglu_grad"])
    type_ = rng.choice(["f32", "f16", "bf16", "bf16"])
    if kind in ("order", "combine", "combine_grad"):
        k = rng.choice([2, 6, 8])
        e = rng.choice([8, 64, 160, 256]) if k > 2 else 8
        c = {"kind": kind, "T": _log(rng, 1, 4096), "k": k, "E": e, "local": e if rng.random() < 0.7 else e // 4,
             "d": _log(rng, 1024, 7168, rng.choice([1, 8, 128])), "type": type_}
        if kind == "combine":
            c["add"] = rng.random() < 0.5
        else:
            c["fp8"] = rng.random() < 0.6
        return c
    if kind == "product":
        back = rng.random() < 0.35
        # rows of 8-bit codes start on 16 bytes; the kept dimension may be any
        n, k = _log(rng, 1024, 14336, 16 if back else 1), _log(rng, 1024, 7168, 1 if back else 16)
        groups = rng.choice([1, 1, 8, 20, 32])
        groups = max(1, min(groups, int(9.4e8 / (n * k))))   # no more weights than the largest listed case
        rows = _log(rng, 1, 8192)
        rows = max(1, min(rows, int(4.8e11 / n / k)))
        return {"kind": kind, "rows": rows, "groups": groups, "N": n, "K": k, "type": type_,
                "back": back, "skew": rng.choice([0.0, 0.3])}
    return {"kind": kind, "rows": _log(rng, 1, 16384), "f": _log(rng, 1024, 2816, 128), "type": type_,
            "limit": rng.choice([0.0, 7.0])}


# ------------------------------------------------------------ inputs


def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _blocks(v, across=1):
    """v [..., rows, cols] in 8 bits: e4m3 codes and f32 scales, one scale for
    `across` x 128 values: scale = max|v| / 448, code = v / scale."""
    rows, cols = v.shape[-2:]
    pr, pc = -rows % across, -cols % BLOCK
    p = torch.nn.functional.pad(v, (0, pc, 0, pr))
    b = p.reshape(*v.shape[:-2], (rows + pr) // across, across, (cols + pc) // BLOCK, BLOCK)
    scale = (b.abs().amax((-3, -1)) / E4M3_MAX).clamp_min(MIN_SCALE)
    codes = (b / scale[..., :, None, :, None]).reshape(p.shape)[..., :rows, :cols]
    return codes.to(torch.float8_e4m3fn), scale


def _values(codes, scales, across=1):
    """The 32-bit values that codes and scales stand for."""
    rows, cols = codes.shape[-2:]
    s = scales.repeat_interleave(across, -2)[..., :rows, :].repeat_interleave(BLOCK, -1)[..., :cols]
    return codes.float() * s


def _routing(case, g):
    """Top-k experts of T tokens with an uneven load, -1 where another rank
    holds the expert, and combine weights that sum to 2.5."""
    t, k, e = case["T"], case["k"], case["E"]
    logits = torch.randn(t, e, generator=g, device="cuda") + torch.randn(e, generator=g, device="cuda")
    top = logits.topk(k, 1)
    idx = torch.where(top.indices < case["local"], top.indices, torch.full_like(top.indices, -1)).int()
    w = torch.sigmoid(top.values)
    return idx, (2.5 * w / w.sum(1, keepdim=True)).contiguous()


def _order(idx, experts):
    """perm (assignments in expert order, -1 past the last), pos (its inverse,
    -1 for an assignment without an expert) and the experts' offsets."""
    a = idx.reshape(-1).long()
    key = torch.where(a < 0, torch.full_like(a, experts), a)
    perm = torch.sort(key, stable=True).indices
    counts = (a[None, :] == torch.arange(experts, device=a.device)[:, None]).sum(1)
    offsets = torch.zeros(experts + 1, dtype=torch.int64, device=a.device)
    offsets[1:] = counts.cumsum(0)
    at = torch.arange(a.numel(), device=a.device)
    pos = torch.empty_like(perm)
    pos[perm] = at
    held = at < offsets[-1]
    return torch.where(held, perm, -1).int(), torch.where(a >= 0, pos, -1).int(), offsets.int()


def prepare(case, seed):
    g = _generator(seed)
    dev = {"device": "cuda"}
    s = {"case": dict(case), "type": TYPES[case["type"]]}
    kind = case["kind"]
    if kind in ("order", "combine", "combine_grad"):
        t, k, d = case["T"], case["k"], case["d"]
        n = t * k
        s["idx"], s["w"] = _routing(case, g)
        if kind == "order":
            s["x"] = torch.randn(t, d, generator=g, **dev).to(s["type"])
            s["perm"] = torch.empty(n, dtype=torch.int32, **dev)
            s["pos"] = torch.empty(n, dtype=torch.int32, **dev)
            s["offsets"] = torch.empty(case["local"] + 1, dtype=torch.int32, **dev)
        else:
            s["perm"], s["pos"], s["offsets"] = _order(s["idx"], case["local"])
            s["rows"] = torch.randn(n, d, generator=g, **dev).to(s["type"])
            s["x"] = torch.randn(t, d, generator=g, **dev).to(s["type"])
        if kind == "combine":
            s["out"] = torch.empty(t, d, dtype=s["type"], **dev)
        else:
            s["dw"] = torch.empty(t, k, **dev)
            _out_rows(s, n, d, case["fp8"])
    elif kind == "product":
        _prepare_product(s, case, g)
    else:
        rows, f = case["rows"], case["f"]
        s["gu"] = (2.0 * torch.randn(rows, 2 * f, generator=g, **dev)).to(s["type"])
        if kind == "swiglu_grad":
            s["dh"] = torch.randn(rows, f, generator=g, **dev).to(s["type"])
        _out_rows(s, rows, f if kind == "swiglu" else 2 * f, True)
    if own:
        s["q"] = _package()
        s["t"] = {"f32": s["q"].QuantFormat.F32, "f16": s["q"].QuantFormat.F16, "bf16": s["q"].QuantFormat.BF16}[
            case["type"]]
        if kind == "product":
            s["m"] = s["q"].Fp8Matrix(case["N"], case["K"], s["codes"], s["scales"], groups=case["groups"])
    return s


def _package():
    import qauntrunner_b200
    return qauntrunner_b200


def _out_rows(s, rows, cols, fp8):
    if fp8:
        s["out"] = torch.zeros(rows, cols, dtype=torch.float8_e4m3fn, device="cuda")
        s["out_scales"] = torch.zeros(rows, -(-cols // BLOCK), device="cuda")
    else:
        s["out"] = torch.zeros(rows, cols, dtype=s["type"], device="cuda")


def _prepare_product(s, case, g):
    rows, groups, n, k = case["rows"], case["groups"], case["N"], case["K"]
    s["codes"] = torch.empty(groups, n, k, dtype=torch.float8_e4m3fn, device="cuda")
    s["scales"] = torch.empty(groups, -(-n // BLOCK), -(-k // BLOCK), device="cuda")
    for i in range(groups):
        s["codes"][i], s["scales"][i] = _blocks(0.02 * torch.randn(n, k, generator=g, device="cuda"), BLOCK)
    s["x"], s["x_scales"] = _blocks(torch.randn(rows, n if case["back"] else k, generator=g, device="cuda"))
    share = torch.softmax(case["skew"] * torch.randn(groups, generator=g, device="cuda"), 0)
    member = torch.multinomial(share, rows, True, generator=g).sort().values
    counts = torch.bincount(member, minlength=groups)
    s["offsets"] = torch.zeros(groups + 1, dtype=torch.int32, device="cuda")
    s["offsets"][1:] = counts.cumsum(0)
    # what the plain form goes by: the groups that have rows, each row's place in its group
    s["used"] = counts.nonzero()[:, 0]
    s["member"] = torch.searchsorted(s["used"], member)
    s["place"] = torch.arange(rows, device="cuda") - s["offsets"][member].long()
    s["most"] = int(counts.max())
    s["out"] = torch.empty(rows, k if case["back"] else n, dtype=s["type"], device="cuda")


# ------------------------------------------------------------ the operators


def run(s):
    return _run_own(s) if own else _run_plain(s)


def _run_own(s):
    q, c, t = s["q"], s["case"], s["t"]
    stream = torch.cuda.current_stream().cuda_stream
    kind = c["kind"]
    if kind == "order":
        n = c["T"] * c["k"]
        q.sort_tokens(s["idx"], c["T"], c["k"], c["local"], s["perm"], s["pos"], s["offsets"], stream=stream)
        out = {"perm": s["perm"], "pos": s["pos"], "offsets": s["offsets"]}
        if c["fp8"]:
            q.gather_rows_fp8(t, s["x"], s["pos"], c["T"], c["k"], c["d"], s["out"], s["out_scales"], n, stream=stream)
            return {**out, "codes": s["out"], "scales": s["out_scales"]}
        q.gather_rows(t, s["x"], s["pos"], c["T"], c["k"], c["d"], s["out"], n, stream=stream)
        return {**out, "rows": s["out"]}
    if kind == "combine":
        q.combine_rows(t, s["rows"], c["T"] * c["k"], s["pos"], s["w"], c["T"], c["k"], c["d"], s["out"],
                       add=s["x"] if c["add"] else None, stream=stream)
        return s["out"]
    if kind == "combine_grad":
        n = c["T"] * c["k"]
        if c["fp8"]:
            q.combine_rows_grad_fp8(t, s["x"], s["rows"], n, s["pos"], s["w"], c["T"], c["k"], c["d"], s["out"],
                                    s["out_scales"], s["dw"], stream=stream)
            return {"codes": s["out"], "scales": s["out_scales"], "dw": s["dw"]}
        q.combine_rows_grad(t, s["x"], s["rows"], n, s["pos"], s["w"], c["T"], c["k"], c["d"], s["out"], s["dw"],
                            stream=stream)
        return {"rows": s["out"], "dw": s["dw"]}
    if kind == "product":
        f = s["m"].product_t if c["back"] else s["m"].product
        f(t, s["x"], s["x_scales"], c["rows"], s["out"], offsets=s["offsets"], stream=stream)
        return s["out"]
    if kind == "swiglu":
        q.swiglu_fp8(t, s["gu"], c["rows"], c["f"], s["out"], s["out_scales"], limit=c["limit"], stream=stream)
    else:
        q.swiglu_fp8_grad(t, s["gu"], s["dh"], c["rows"], c["f"], s["out"], s["out_scales"], limit=c["limit"],
                          stream=stream)
    return {"codes": s["out"], "scales": s["out_scales"]}


def _rows_out(s, values, pos):
    """values [n, cols], one for each assignment, to their rows: in 8 bits or
    rounded to the case's type; rows without an assignment are zero."""
    n = pos.numel()
    to = torch.where(pos < 0, n, pos.long())   # an assignment without a row goes past the last
    if s["case"]["fp8"]:
        codes, scales = _blocks(values)
        c = torch.zeros(n + 1, values.shape[1], dtype=torch.uint8, device="cuda")
        c[to] = codes.view(torch.uint8)
        b = torch.zeros(n + 1, scales.shape[1], device="cuda")
        b[to] = scales
        return {"codes": c[:n].view(torch.float8_e4m3fn), "scales": b[:n]}
    r = torch.zeros(n + 1, values.shape[1], dtype=s["type"], device="cuda")
    r[to] = values.to(s["type"])
    return {"rows": r[:n]}


def _run_plain(s):
    c, kind = s["case"], s["case"]["kind"]
    if kind == "order":
        perm, pos, offsets = _order(s["idx"], c["local"])
        x = s["x"].float()
        out = {"perm": perm, "pos": pos, "offsets": offsets}
        source = perm.long().clamp_min(0) // c["k"]
        held = (perm >= 0)[:, None]
        if c["fp8"]:   # the rows in 8 bits first, then copied
            codes, scales = _blocks(x)
            rows = torch.where(held, codes.view(torch.uint8)[source], 0).view(torch.float8_e4m3fn)
            return {**out, "codes": rows, "scales": torch.where(held, scales[source], 0.0)}
        return {**out, "rows": torch.where(held, s["x"][source], 0.0)}
    if kind in ("combine", "combine_grad"):
        pos = s["pos"].long()
        held = (pos >= 0).reshape(c["T"], c["k"])
        picked = s["rows"][pos.clamp_min(0)].float().reshape(c["T"], c["k"], c["d"])
        if kind == "combine":
            y = torch.where(held[..., None], picked * s["w"][..., None], 0.0).sum(1)
            return (y + s["x"].float() if c["add"] else y).to(s["type"])
        dout = s["x"].float()
        dw = torch.where(held, (picked * dout[:, None, :]).sum(-1), 0.0)
        grads = (s["w"][..., None] * dout[:, None, :]).reshape(-1, c["d"])
        return {**_rows_out(s, grads, s["pos"]), "dw": dw}
    if kind == "product":
        w = _values(s["codes"][s["used"]], s["scales"][s["used"]], BLOCK)
        x = _values(s["x"], s["x_scales"])
        if c["groups"] == 1:
            return (x @ (w[0] if c["back"] else w[0].T)).to(s["type"])
        padded = torch.zeros(w.shape[0], s["most"], x.shape[1], device="cuda")
        padded[s["member"], s["place"]] = x
        y = torch.bmm(padded, w if c["back"] else w.transpose(1, 2))
        return y[s["member"], s["place"]].to(s["type"])
    gate, up = s["gu"][:, :c["f"]].float(), s["gu"][:, c["f"]:].float()
    lim = c["limit"] or float("inf")
    g, u = gate.clamp(max=lim), up.clamp(-lim, lim)
    sig = 1.0 / (1.0 + torch.exp(-g))
    if kind == "swiglu":
        codes, scales = _blocks(g * sig * u)
        return {"codes": codes, "scales": scales}
    dh = s["dh"].float()
    dg = torch.where(gate <= lim, dh * u * (sig * (1.0 + g * (1.0 - sig))), 0.0)
    du = torch.where(up.abs() <= lim, dh * (g * sig), 0.0)
    codes, scales = _blocks(torch.cat([dg, du], 1))
    return {"codes": codes, "scales": scales}


# ------------------------------------------------------------ what a pass cannot do without


def work(case):
    kind, b = case["kind"], SIZE[case["type"]]
    if kind in ("order", "combine", "combine_grad"):
        t, k, d = case["T"], case["k"], case["d"]
        n = t * k
        held = n * case["local"] // case["E"]
        row8 = d + 4 * -(-d // BLOCK)
        if kind == "order":
            row = row8 if case["fp8"] else d * b
            return {"bytes": 12 * n + 4 * (case["local"] + 1) + t * d * b + held * row, "flops": 3 * t * d if case["fp8"] else 0}
        if kind == "combine":
            return {"bytes": 8 * n + held * d * b + t * d * b * (2 if case["add"] else 1), "flops": 2 * held * d}
        return {"bytes": 12 * n + t * d * b + held * d * b + held * (row8 if case["fp8"] else d * b),
                "flops": 3 * held * d}
    if kind == "product":
        rows, groups, n, k = case["rows"], case["groups"], case["N"], case["K"]
        used = groups * (1.0 - (1.0 - 1.0 / groups) ** rows)   # groups with a row, on average
        scales = 4 * -(-n // BLOCK) * -(-k // BLOCK)
        contracted, kept = (n, k) if case["back"] else (k, n)
        return {"bytes": used * (n * k + scales) + rows * (contracted + 4 * -(-contracted // BLOCK) + kept * b),
                "flops": 2.0 * rows * n * k}
    rows, f = case["rows"], case["f"]
    if kind == "swiglu":
        return {"bytes": rows * (2 * f * b + f + 4 * -(-f // BLOCK)), "flops": 12 * rows * f}
    return {"bytes": rows * (3 * f * b + 2 * f + 4 * -(-2 * f // BLOCK)), "flops": 25 * rows * f}


# ------------------------------------------------------------ the definitions in 64 bits


def _e4m3(v):
    """The e4m3 number nearest to v (ties to even), in 64 bits."""
    _, e = torch.frexp(v)
    step = torch.ldexp(torch.ones_like(v), (e - 1).clamp_min(-6) - 3)
    return (torch.round(v / step) * step).clamp(-E4M3_MAX, E4M3_MAX)


def _codes64(v):
    """(codes, scales) of the rows of v, block by block."""
    n, cols = v.shape
    nb = -(-cols // BLOCK)
    codes, scales = torch.zeros_like(v), torch.zeros(n, nb, dtype=torch.float64, device=v.device)
    for j in range(nb):
        part = v[:, j * BLOCK:(j + 1) * BLOCK]
        top = part.abs().max(1).values
        scales[:, j] = torch.clamp(top / E4M3_MAX, min=MIN_SCALE)
        codes[:, j * BLOCK:(j + 1) * BLOCK] = _e4m3(part / scales[:, j:j + 1])
    return codes, scales


def exact(case, seed):
    s = prepare(case, seed)
    kind, f64 = case["kind"], torch.float64
    if kind in ("order", "combine", "combine_grad"):
        t, k, d = case["T"], case["k"], case["d"]
        x = s["x"].to(f64)
        token = torch.arange(t * k, device="cuda") // k
        if kind == "order":
            a = s["idx"].reshape(-1)
            # assignments with an expert, by (expert, assignment)
            rank = (a.to(f64) * (t * k) + torch.arange(t * k, device="cuda"))[a >= 0]
            order = torch.nonzero(a >= 0)[:, 0][torch.argsort(rank)]
            whole = {"perm": None, "pos": None, "offsets": None}
            if not case["fp8"]:
                rows = torch.zeros(t * k, d, dtype=f64, device="cuda")
                rows[:order.numel()] = x[token[order]]
                return {**whole, "rows": rows}
            c1, s1 = _codes64(x)
            codes = torch.zeros(t * k, d, dtype=f64, device="cuda")
            scales = torch.zeros(t * k, s1.shape[1], dtype=f64, device="cuda")
            codes[:order.numel()] = c1[token[order]]
            scales[:order.numel()] = s1[token[order]]
            return {**whole, "codes": codes, "scales": scales}
        pos = s["pos"].long().reshape(t, k)
        w = s["w"].to(f64)
        if kind == "combine":
            y = x.clone() if case["add"] else torch.zeros_like(x)
            for j in range(k):
                here = torch.nonzero(pos[:, j] >= 0)[:, 0]
                y[here] += w[here, j, None] * s["rows"][pos[here, j]].to(f64)
            return y
        dw = torch.zeros(t, k, dtype=f64, device="cuda")
        shape = (t * k, d)
        out = torch.zeros(shape, dtype=f64, device="cuda")
        scales = torch.zeros(t * k, -(-d // BLOCK), dtype=f64, device="cuda")
        for j in range(k):
            here = torch.nonzero(pos[:, j] >= 0)[:, 0]
            dw[here, j] = torch.einsum("td,td->t", x[here], s["rows"][pos[here, j]].to(f64))
            v = w[here, j, None] * x[here]
            if case["fp8"]:
                out[pos[here, j]], scales[pos[here, j]] = _codes64(v)
            else:
                out[pos[here, j]] = v
        return {"codes": out, "scales": scales, "dw": dw} if case["fp8"] else {"rows": out, "dw": dw}
    if kind == "product":
        if 2.0 * case["rows"] * case["N"] * case["K"] > 2e12:
            return None
        edges = s["offsets"].tolist()
        y = torch.zeros(s["out"].shape, dtype=f64, device="cuda")
        for i in range(case["groups"]):
            a, b = edges[i], edges[i + 1]
            if a == b:
                continue
            w = s["codes"][i].to(f64)
            for r in range(0, case["N"], BLOCK):
                at = s["scales"][i, r // BLOCK].to(f64).repeat_interleave(BLOCK)[:case["K"]]
                w[r:r + BLOCK] *= at
            x = s["x"][a:b].to(f64)
            x *= s["x_scales"][a:b].to(f64).repeat_interleave(BLOCK, 1)[:, :x.shape[1]]
            y[a:b] = torch.matmul(x, w if case["back"] else w.T)
        return y
    f = case["f"]
    gate, up = s["gu"][:, :f].to(f64), s["gu"][:, f:].to(f64)
    lim = case["limit"]
    g = torch.minimum(gate, torch.full_like(gate, lim)) if lim else gate
    u = torch.maximum(torch.minimum(up, torch.full_like(up, lim)), torch.full_like(up, -lim)) if lim else up
    silu = g * torch.sigmoid(g)
    if kind == "swiglu":
        codes, scales = _codes64(silu * u)
        return {"codes": codes, "scales": scales}
    dh = s["dh"].to(f64)
    slope = torch.sigmoid(g) + silu * torch.sigmoid(-g)
    dg, du = dh * u * slope, dh * silu
    if lim:
        dg[gate > lim] = 0
        du[(up > lim) | (up < -lim)] = 0
    cg, sg = _codes64(dg)
    cu, su = _codes64(du)
    return {"codes": torch.cat([cg, cu], 1), "scales": torch.cat([sg, su], 1)}
