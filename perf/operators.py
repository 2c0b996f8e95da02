"""The block-scaled fp8 products, the block quantiser and the Newton-Schulz orthogonalisation: the
cases they are measured on, their plain forms and their definition in 64 bits.

Layouts are the library's: operands [batch][2][rows][k] (planar) or [batch][rows][k][2]
(interleaved), C[b] = A[b] x B[b]^T.
"""
import math

import torch

own = False

BLOCK = 128
FMAX = {"e4m3": 448.0, "e5m2": 57344.0}
FP8 = {"e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}
FLOAT = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
WIDTH = {"f16": 2, "bf16": 2, "f32": 4}
TINY = 2.0 ** -126  # smallest scale: its reciprocal is finite in 32 bits
QUINTIC = (3.4445, -4.7750, 2.0315)  # steep at zero, ends near 1
CONVERGENT = (1.875, -1.25, 0.375)  # Newton-Schulz of fifth order, converges to 1


def _ceil(a, b):
    return -(-a // b)


def _quantize(name, batch, rows, k, tin, tout, axis, order, block_rows):
    return {"name": name, "op": "quantize", "batch": batch, "rows": rows, "k": k, "tin": tin,
            "tout": tout, "axis": axis, "order": order, "block_rows": block_rows}


def _gemm(name, batch, m, n, k, ta, tb, tout, axis, order, ga, gb):
    return {"name": name, "op": "gemm", "batch": batch, "m": m, "n": n, "k": k, "ta": ta,
            "tb": tb, "tout": tout, "axis": axis, "order": order, "ga": ga, "gb": gb}


def _orth(name, batch, m, n, tin, tout, axis, steps, converge):
    return {"name": name, "op": "orth", "batch": batch, "m": m, "n": n, "tin": tin, "tout": tout,
            "axis": axis, "steps": steps, "converge": converge}


def listed():
    return [
        # one small block of weights before a product: latency
        _quantize("quantize_small", 1, 1024, 1024, "f16", "e4m3", "planar", "row", 1),
        # voltage samples as they arrive: interleaved float32, one scale per row and block
        _quantize("quantize_samples", 4, 4096, 16384, "f32", "e4m3", "interleaved", "row", 1),
        # weights contracted over their other axis (transposed operand), odd sizes, square blocks
        _quantize("quantize_other_axis", 3, 5003, 4001, "bf16", "e5m2", "planar", "col", 128),
        # one sample against many beams: memory bound, one row
        _gemm("gemm_one_row", 1, 1, 8192, 8192, "e4m3", "e4m3", "f32", "planar", "row", 1, 128),
        # a few rows, odd
        _gemm("gemm_few_rows", 2, 13, 4096, 16384, "e4m3", "e4m3", "f16", "planar", "row", 1, 1),
        # a single product that does not fill the device
        _gemm("gemm_1024", 1, 1024, 1024, 1024, "e4m3", "e4m3", "f32", "planar", "row", 1, 128),
        # many short products
        _gemm("gemm_short_k", 512, 256, 2048, 512, "e4m3", "e4m3", "bf16", "planar", "row", 1, 128),
        # ragged everywhere, gradients in e5m2, interleaved column-major result
        _gemm("gemm_ragged_mixed", 3, 1000, 2501, 1990, "e5m2", "e4m3", "f32", "interleaved",
              "col", 1, 1),
        # the library's large fp8 product, four items of its batch
        _gemm("gemm_large", 4, 4096, 4096, 16384, "e4m3", "e4m3", "f32", "planar", "row", 1, 128),
        # many small bases of a subspace iteration
        _orth("orth_small_bases", 64, 33, 70, "f32", "bf16", "interleaved", 5, False),
        # one square set of weights
        _orth("orth_square", 1, 1024, 1024, "bf16", "bf16", "planar", 5, False),
        # several tall sets, to convergence
        _orth("orth_tall", 8, 4096, 1024, "f16", "f16", "planar", 8, True),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    op = rng.choice(["quantize", "quantize", "gemm", "gemm", "gemm", "orth", "orth"])
    if op == "quantize":
        while True:
            batch, rows, k = rng.randint(1, 16), _log(rng, 1, 16384), _log(rng, 1, 16384)
            if 1 << 10 <= batch * rows * k <= 4 * 4096 * 16384 // 2:
                break
        return _quantize("", batch, rows, k, rng.choice(list(FLOAT)), rng.choice(list(FP8)),
                         rng.choice(["planar", "interleaved"]), rng.choice(["row", "col"]),
                         rng.choice([1, 128]))
    if op == "gemm":
        while True:
            batch, m, n, k = (_log(rng, 1, 512), _log(rng, 1, 8192), _log(rng, 1, 8192),
                              _log(rng, 1, 16384))
            if batch * m * n * k <= 4096 * 4096 * 16384 and batch * (m + n) * k <= 1 << 28 \
                    and batch * m * n <= 1 << 28 and n * k >= 1 << 12:
                break
        return _gemm("", batch, m, n, k, rng.choice(list(FP8)), rng.choice(list(FP8)),
                     rng.choice(list(FLOAT)), rng.choice(["planar", "interleaved"]),
                     rng.choice(["row", "col"]), rng.choice([1, 128]), rng.choice([1, 128]))
    while True:
        batch, m, n = _log(rng, 1, 256), _log(rng, 1, 4096), _log(rng, 1, 4096)
        short, long = min(m, n), max(m, n)
        if short <= 1024 and batch * short * short * long <= 8 * 1024 * 1024 * 2048 \
                and batch * m * n <= 1 << 24 and m * n > 1:
            break
    return _orth("", batch, m, n, rng.choice(list(FLOAT)), rng.choice(["f16", "bf16"]),
                 rng.choice(["planar", "interleaved"]), rng.randint(3, 8), rng.random() < 0.5)


# ---------------------------------------------------------------------------- inputs


def _normal(shape, gen):
    return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32)


def _signal(batch, rows, k, gen):
    """Planar complex samples [batch][2][rows][k] whose level differs by row (gains) and by block
    (bands, bursts); one row in 64 is silent (a dead input)."""
    x = _normal((batch, 2, rows, k), gen)
    gain = torch.rand((batch, 1, rows, 1), generator=gen, device="cuda") * 8 - 4
    gain = torch.exp(gain)
    gain[torch.rand(gain.shape, generator=gen, device="cuda") < 1 / 64] = 0
    level = torch.rand((batch, 1, 1, _ceil(k, BLOCK)), generator=gen, device="cuda") * 4 - 2
    x *= gain
    x *= torch.exp(level).repeat_interleave(BLOCK, 3)[..., :k]
    return x


def _block_scales(x, block_rows, fmax):
    """[batch][ceil(k/128)][ceil(rows/block_rows)] scales of planar x, and the per-element
    reciprocals [batch][rows][k]."""
    batch, _, rows, k = x.shape
    big = torch.where(torch.isfinite(x), x, torch.zeros_like(x)).abs().amax(dim=1)
    kb, rb = _ceil(k, BLOCK), _ceil(rows, block_rows)
    pad = big.new_zeros((batch, rb * block_rows, kb * BLOCK))
    pad[:, :rows, :k] = big
    amax = pad.view(batch, rb, block_rows, kb, BLOCK).amax(dim=(2, 4))
    scale = (amax / fmax).clamp_min(TINY)
    inv = (1.0 / scale).repeat_interleave(block_rows, 1).repeat_interleave(BLOCK, 2)
    return scale.transpose(1, 2).contiguous(), inv[:, :rows, :k]


def _to_fp8(x, inv, name, pitch):
    """x * inv rounded to fp8, rows padded with zeros to `pitch`.  NaN stays, infinities stay in
    e5m2 and become NaN in e4m3, which has none."""
    q = x * inv[:, None]
    q = torch.where(torch.isfinite(q), q.clamp(-FMAX[name], FMAX[name]), q).to(FP8[name])
    out = torch.zeros(q.shape[:3] + (pitch,), dtype=torch.uint8, device=q.device)
    out[..., : q.shape[3]] = q.view(torch.uint8)
    return out.view(FP8[name])


def _pitch(k):
    return _ceil(k, 16) * 16


def _lay_out(x, axis, order):
    """Planar [batch][2][rows][k] -> the order in which the caller holds it."""
    if order == "col":
        x = x.transpose(2, 3)
    return (x.permute(0, 2, 3, 1) if axis == "interleaved" else x).contiguous()


def _planar(x, axis, order):
    if axis == "interleaved":
        x = x.permute(0, 3, 1, 2)
    return x.transpose(2, 3) if order == "col" else x


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    s = {"case": case}
    op, batch = case["op"], case["batch"]
    if op == "quantize":
        x = _signal(batch, case["rows"], case["k"], gen)
        s["x"] = _lay_out(x.to(FLOAT[case["tin"]]), case["axis"], case["order"])
    elif op == "gemm":
        for side, rows, kind, g in (("a", case["m"], case["ta"], case["ga"]),
                                    ("b", case["n"], case["tb"], case["gb"])):
            # levels as a front end sets them: products stay inside float16's range
            x = _signal(batch, rows, case["k"], gen) * 2.0 ** -6
            scale, inv = _block_scales(x, g, FMAX[kind])
            s[side], s[side + "_scale"] = _to_fp8(x, inv, kind, _pitch(case["k"])), scale
            del x, inv
    else:
        x = _normal((batch, 2, case["m"], case["n"]), gen)
        x *= torch.exp(_normal((batch, 1, 1, 1), gen))
        # what is orthogonalised has a few strong directions
        u, v = _normal((batch, 2, case["m"], 1), gen), _normal((batch, 1, 1, case["n"]), gen)
        s["x"] = _lay_out((x + u * v).to(FLOAT[case["tin"]]), case["axis"], "row")
    if own:
        _own_prepare(s)
    return s


# ---------------------------------------------------------------------------- the framework's calls


def _codes(capi):
    return {"e4m3": capi.FLOAT8E4M3, "e5m2": capi.FLOAT8E5M2, "f16": capi.FLOAT16,
            "bf16": capi.BFLOAT16, "f32": capi.FLOAT32, "planar": capi.PLANAR,
            "interleaved": capi.INTERLEAVED, "row": capi.ROW_MAJOR, "col": capi.COL_MAJOR}


def _c_shape(case):
    m, n = (case["m"], case["n"]) if case["order"] == "row" else (case["n"], case["m"])
    return (case["batch"], m, n, 2) if case["axis"] == "interleaved" else (case["batch"], 2, m, n)


def _own_prepare(s):
    from ccglib_b200 import capi

    case, code = s["case"], _codes(capi)
    s["capi"], s["code"] = capi, code
    if case["op"] == "quantize":
        batch, rows, k = case["batch"], case["rows"], case["k"]
        s["q"] = torch.empty((batch, 2, rows, _pitch(k)), dtype=FP8[case["tout"]], device="cuda")
        s["scale"] = torch.empty((batch, _ceil(k, BLOCK), _ceil(rows, case["block_rows"])),
                                 dtype=torch.float32, device="cuda")
    elif case["op"] == "gemm":
        s["c"] = torch.empty(_c_shape(case), dtype=FLOAT[case["tout"]], device="cuda")
        s["plan"] = capi.ScaledGemmPlan(
            case["batch"], case["m"], case["n"], case["k"], code[case["ta"]], code[case["tb"]],
            code[case["tout"]], a_block_rows=case["ga"], b_block_rows=case["gb"],
            c_complex_axis=code[case["axis"]], c_mem_order=code[case["order"]])
    else:
        s["y"] = torch.empty((case["batch"], 2, case["m"], case["n"]), dtype=FLOAT[case["tout"]],
                             device="cuda")
        s["plan"] = capi.OrthogonalizePlan(
            case["batch"], case["m"], case["n"], code[case["tin"]], code[case["tout"]],
            steps=case["steps"], coefficients=CONVERGENT if case["converge"] else QUINTIC,
            input_complex_axis=code[case["axis"]])


def _own_run(s):
    case = s["case"]
    stream = torch.cuda.current_stream().cuda_stream
    if case["op"] == "quantize":
        code = s["code"]
        s["capi"].quantize(case["batch"], case["rows"], case["k"], code[case["tin"]],
                           code[case["tout"]], s["x"].data_ptr(), s["q"].data_ptr(),
                           s["scale"].data_ptr(), stream, input_complex_axis=code[case["axis"]],
                           input_mem_order=code[case["order"]], block_rows=case["block_rows"])
        return {"q": s["q"], "scale": s["scale"]}
    if case["op"] == "gemm":
        s["plan"].run(s["a"].data_ptr(), s["a_scale"].data_ptr(), s["b"].data_ptr(),
                      s["b_scale"].data_ptr(), s["c"].data_ptr(), stream)
        return {"c": s["c"]}
    s["plan"].run(s["x"].data_ptr(), s["y"].data_ptr(), stream)
    return {"y": s["y"]}


# ---------------------------------------------------------------------------- plain forms


def _dequantize(q, scale, block_rows, k, dtype):
    """Complex values [batch][rows][k] of fp8 planes and block scales."""
    rows = q.shape[2]
    v = q[..., :k].to(dtype)
    full = scale.to(dtype).transpose(1, 2).repeat_interleave(block_rows, 1)[:, :rows]
    full = full.repeat_interleave(BLOCK, 2)[..., :k]
    return torch.complex(v[:, 0] * full, v[:, 1] * full)


def _lay_out_c(c, case):
    """Complex [batch][m][n] -> the requested layout of C, real and imaginary parts apart."""
    if case["order"] == "col":
        c = c.transpose(1, 2)
    c = torch.view_as_real(c.contiguous())
    return c if case["axis"] == "interleaved" else c.permute(0, 3, 1, 2)


def _newton_schulz(x, case, norm):
    a, b, c = CONVERGENT if case["converge"] else QUINTIC
    wide = case["m"] <= case["n"]
    x = x / norm
    for _ in range(case["steps"]):
        xh = x.mH
        s = x @ xh if wide else xh @ x
        p = b * s + c * (s @ s)
        x = a * x + (p @ x if wide else x @ p)
    return x


def run(state):
    if own:
        return _own_run(state)
    case = state["case"]
    if case["op"] == "quantize":
        x = _planar(state["x"].float(), case["axis"], case["order"])
        scale, inv = _block_scales(x, case["block_rows"], FMAX[case["tout"]])
        return {"q": _to_fp8(x, inv, case["tout"], _pitch(case["k"])), "scale": scale}
    if case["op"] == "gemm":
        a = _dequantize(state["a"], state["a_scale"], case["ga"], case["k"], torch.float32)
        b = _dequantize(state["b"], state["b_scale"], case["gb"], case["k"], torch.float32)
        c = a @ b.transpose(1, 2)
        return {"c": _lay_out_c(c, case).to(FLOAT[case["tout"]]).contiguous()}
    x = _planar(state["x"].float(), case["axis"], "row")
    norm = x.double().square().sum(dim=(1, 2, 3)).sqrt().float().clamp_min(TINY)[:, None, None]
    y = _newton_schulz(torch.complex(x[:, 0].contiguous(), x[:, 1].contiguous()), case, norm)
    return {"y": torch.stack((y.real, y.imag), 1).to(FLOAT[case["tout"]])}


# ---------------------------------------------------------------------------- what a pass costs


def work(case):
    batch = case["batch"]
    if case["op"] == "quantize":
        n = 2 * batch * case["rows"] * case["k"]
        blocks = batch * _ceil(case["k"], BLOCK) * _ceil(case["rows"], case["block_rows"])
        # per real value: |x|, maximum, product, rounding
        return {"bytes": n * WIDTH[case["tin"]] + n + 4 * blocks, "flops": 4 * n}
    if case["op"] == "gemm":
        m, n, k = case["m"], case["n"], case["k"]
        blocks = _ceil(k, BLOCK) * (_ceil(m, case["ga"]) + _ceil(n, case["gb"]))
        return {"bytes": batch * (2 * (m + n) * k + 4 * blocks + 2 * m * n * WIDTH[case["tout"]]),
                "flops": 8 * batch * m * n * k}
    short, long = min(case["m"], case["n"]), max(case["m"], case["n"])
    # S and S^2 are Hermitian: half of each is enough
    step = 4 * short * short * long + 4 * short ** 3 + 8 * short * short * long
    return {"bytes": 2 * batch * short * long * (WIDTH[case["tin"]] + WIDTH[case["tout"]]),
            "flops": batch * case["steps"] * step}


# ---------------------------------------------------------------------------- 64 bits


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "quantize":
        x = s["x"].double()
        if case["axis"] == "interleaved":
            x = torch.stack((x[..., 0], x[..., 1]), 1)
        if case["order"] == "col":
            x = x.transpose(2, 3)
        batch, _, rows, k = x.shape
        g, top = case["block_rows"], FMAX[case["tout"]]
        scale = x.new_empty((batch, _ceil(k, BLOCK), _ceil(rows, g)))
        q = x.new_zeros((batch, 2, rows, _pitch(k)))
        mag = torch.maximum(x[:, 0].abs(), x[:, 1].abs())
        for i in range(_ceil(k, BLOCK)):
            lo, hi = i * BLOCK, min(k, (i + 1) * BLOCK)
            col = mag[:, :, lo:hi].amax(dim=2)
            if g > 1:
                col = torch.stack([part.amax(dim=1) for part in col.split(g, dim=1)], 1)
            scale[:, i] = torch.clamp(col / top, min=TINY)
            per_row = scale[:, i].repeat_interleave(g, 1)[:, :rows]
            q[..., lo:hi] = _round_fp8(x[..., lo:hi] / per_row[:, None, :, None], case["tout"])
        return {"q": q, "scale": scale}
    if case["op"] == "gemm":
        k = case["k"]
        c_re, c_im = 0.0, 0.0
        for lo in range(0, k, 16 * BLOCK):
            hi = min(k, lo + 16 * BLOCK)
            planes = []
            for side, g in (("a", case["ga"]), ("b", case["gb"])):
                v = s[side][..., lo:hi].double()
                f = s[side + "_scale"][:, lo // BLOCK: _ceil(hi, BLOCK)].double()
                f = f.repeat_interleave(BLOCK, 1)[:, : hi - lo].repeat_interleave(g, 2)
                planes.append(v * f[:, :, : v.shape[2]].transpose(1, 2)[:, None])
            a, b = planes[0], planes[1].transpose(2, 3)
            c_re = c_re + a[:, 0] @ b[:, 0] - a[:, 1] @ b[:, 1]
            c_im = c_im + a[:, 0] @ b[:, 1] + a[:, 1] @ b[:, 0]
        if case["order"] == "col":
            c_re, c_im = c_re.transpose(1, 2), c_im.transpose(1, 2)
        return {"c": torch.stack((c_re, c_im), 3 if case["axis"] == "interleaved" else 1)}
    x = s["x"].double()
    if case["axis"] == "interleaved":
        x = x.permute(0, 3, 1, 2)
    x = torch.complex(x[:, 0].contiguous(), x[:, 1].contiguous())
    # on the singular values: the iteration keeps the singular vectors and maps every value
    norm = torch.linalg.vector_norm(x, dim=(1, 2), keepdim=True)
    x = x / norm
    wide = case["m"] <= case["n"]
    gram = x @ x.mH if wide else x.mH @ x
    lam, u = torch.linalg.eigh(gram)
    a, b, c = CONVERGENT if case["converge"] else QUINTIC
    lam = lam.clamp_min(0)
    gain = torch.ones_like(lam)
    for _ in range(case["steps"]):
        t = lam * gain * gain
        gain = gain * (a + b * t + c * t * t)
    w = (u * gain[:, None].to(u.dtype)) @ u.mH
    y = w @ x if wide else x @ w
    return {"y": torch.stack((y.real, y.imag), 1)}


def _round_fp8(v, name):
    """Nearest fp8 value, ties to even, of 64-bit v with |v| at most a hair over the largest."""
    bits, low, top = (3, -6, 448.0) if name == "e4m3" else (2, -14, 57344.0)
    _, e = torch.frexp(v)
    step = torch.exp2((e - 1).clamp(min=low).double() - bits)
    return (torch.round(v / step) * step).clamp(-top, top)
