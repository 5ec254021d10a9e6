"""The narrow-format operators of a training step, as a user calls them and in plain form.

Three kinds of operator: the root-mean-square norm that leaves its output quantised (8 bits with a scale per row, or 4 bits in
microscaled blocks of 32), the microscaled 4-bit format itself (quantisation, product, the linear layer made of both and its
gradients), and the AdamW step over all fields of a packed object at once with moments in 8 bits or in 32.

``own`` false: elementary torch operations in 32 bits.  ``own`` true: the calls of ``dataflow_b200.ops``.
"""
import math

import torch

own = False

BF, F32, F64, F8, U8 = torch.bfloat16, torch.float32, torch.float64, torch.float8_e4m3fn, torch.uint8
DEV = "cuda"
BLOCK = 32            # elements that share a scale in the 4-bit format
STATE_BLOCK = 128     # elements that share a scale in 8-bit optimizer moments
EPS = 1e-5

# the weight fields of one decoder layer of the 8-billion-parameter configuration (hidden 4096, MLP 14336, 32 / 8 heads of 128)
LAYER = "4096,4096x6144,4096x4096,4096,4096x28672,14336x4096"
# a small block with a bias in every projection: vectors of a few thousand numbers between small matrices
SMALL = "256,256,256x768,768,256x256,256,256,256,256x1024,1024,1024x256,256"
# widths that no tile divides
RAGGED = "1000003,129,4095x1001,1,127,2047x513,128,33"


def listed():
    return [
        # the optimizer task of one large layer with 8-bit moments: what decides the end of a step
        {"name": "adamw_8bit_layer", "op": "adamw", "bits": 8, "weights": "bf16", "grad": "bf16", "sizes": LAYER},
        # a small block's twelve fields: one launch, latency
        {"name": "adamw_8bit_small", "op": "adamw", "bits": 8, "weights": "bf16", "grad": "bf16", "sizes": SMALL},
        # fp32 master, fp32 moments, fp32 gradients, widths that nothing divides
        {"name": "adamw_32bit_ragged", "op": "adamw", "bits": 32, "weights": "master", "grad": "fp32", "sizes": RAGGED},
        # the mixed policy's optimizer task at a quarter of the large layer
        {"name": "adamw_32bit_master", "op": "adamw", "bits": 32, "weights": "master", "grad": "bf16", "sizes": "4096x6144,4096x4096,4096,4096"},
        # the norm in front of a block's projections over one round of 4 x 4096 tokens, residual added on the way
        {"name": "norm_fp8_round", "op": "norm", "fmt": "fp8", "rows": 16384, "cols": 4096, "residual": True},
        # the same for a handful of tokens
        {"name": "norm_fp8_tokens", "op": "norm", "fmt": "fp8", "rows": 5, "cols": 4096, "residual": True},
        # an under-full round of a 2048-wide model, straight into 4-bit blocks
        {"name": "norm_mxfp4_ragged", "op": "norm", "fmt": "mxfp4", "rows": 8191, "cols": 2048, "residual": False},
        # activations to 4 bits and back to the values (what fake quantisation does)
        {"name": "quant_mxfp4_rows", "op": "quant", "rows": 8192, "cols": 4096, "transpose": False},
        # a weight stored (in, out), quantised along `in`
        {"name": "quant_mxfp4_weight", "op": "quant", "rows": 4096, "cols": 14336, "transpose": True},
        # the product alone, at the size of the up and gate projections of one round of 2 x 4096 tokens
        {"name": "product_large", "op": "product", "m": 8192, "n": 28672, "k": 4096, "out": "bf16", "add": False},
        # the product for a few tokens, added to the residual
        {"name": "product_tokens", "op": "product", "m": 17, "n": 4096, "k": 4096, "out": "bf16", "add": True},
        # one linear layer of a training step, forward and both gradients, ragged rows
        {"name": "linear_train", "op": "linear", "m": 4095, "n": 6144, "k": 4096},
    ]


def _log(rng, lo, hi, step=1):
    """A size between lo and hi, spread over its logarithm, a multiple of ``step``."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi))) / step)) * step))


def draw(rng):
    op = rng.choice(["adamw", "adamw", "norm", "norm", "quant", "product", "product", "linear"])
    if op == "adamw":
        left, sizes = _log(rng, 2000, 100_000_000), []
        for _ in range(rng.randint(1, 40)):
            n = _log(rng, 1, max(2, left))
            sizes.append("%dx%d" % (max(1, n // 513), 513) if n > 4000 and rng.random() < 0.5 else str(n))
            left -= n
            if left < 2:
                break
        bits = rng.choice([8, 32])
        return {"op": op, "bits": bits, "weights": rng.choice(["bf16", "fp32", "master"]), "grad": rng.choice(["bf16", "fp32"]),
                "sizes": ",".join(sizes)}
    if op == "norm":
        fmt = rng.choice(["fp8", "mxfp4"])
        return {"op": op, "fmt": fmt, "rows": _log(rng, 1, 12000), "cols": _log(rng, 64, 5376, 16 if fmt == "fp8" else 32),
                "residual": rng.random() < 0.5}
    if op == "quant":
        t = rng.random() < 0.5
        a, b = _log(rng, 32, 4096, 32), _log(rng, 1, 14336)
        return {"op": op, "rows": a if t else b, "cols": b if t else a, "transpose": t}
    m, k = _log(rng, 1, 8192), _log(rng, 32, 8192, 32)
    n = _log(rng, 8, max(8, min(14336, int(9e11 / (2.0 * m * k)))), rng.choice([1, 8, 8]))
    if op == "product":
        return {"op": op, "m": m, "n": n, "k": k, "out": rng.choice(["bf16", "bf16", "fp32"]), "add": rng.random() < 0.4}
    return {"op": op, "m": max(1, m // 2), "n": n, "k": k}


# ------------------------------------------------------------------ the 4-bit format, written out
def _e8m0(e):
    """2 ** (e - 127) of the scale bytes e; 255 is NaN."""
    e = e.to(torch.int32)
    bits = torch.where(e == 0, torch.full_like(e, 0x00400000), e << 23)
    return torch.where(e == 255, torch.full_like(bits, 0x7FC00000), bits).view(F32)


def _e2m1_round(a):
    """Nearest of 0 0.5 1 1.5 2 3 4 6 to |a| (ties to the even code), with a's sign."""
    b = a.abs()
    step = torch.where(b < 2, 0.5, torch.where(b < 4, 1.0, 2.0)).to(a.dtype)
    return torch.copysign((torch.round(b / step) * step).clamp(max=6.0), a)


def _mx_blocks(y):
    """Scale bytes (rows, K / 32) and rounded elements (rows, K / 32, 32) of y (rows, K) in 32 bits."""
    b = y.reshape(y.shape[0], -1, BLOCK)
    amax = b.abs().amax(-1)
    e = (amax.view(torch.int32) >> 23) & 255
    s = torch.where(e == 255, e, (e - 2).clamp(min=0))
    inv = ((254 - s.clamp(max=253)) << 23).view(F32)
    return s, _e2m1_round(b * inv.unsqueeze(-1))


def _mx_values(y):
    """y (rows, K) rounded to the 4-bit format, as the values it stands for."""
    s, q = _mx_blocks(y)
    return (q * _e8m0(s).unsqueeze(-1)).reshape(y.shape)


def _mx_pack(y):
    """(codes (rows, K / 2) uint8, low nibble first; scale bytes (ceil(rows / 128), 2 ceil(K / 256), 512) uint8): the operand
    form of the product.  The scale of row r, block b is byte (r % 32) * 16 + (r % 128 // 32) * 4 + b % 4 of tile
    (r // 128, b // 4); bytes past the rows and blocks are zero."""
    s, q = _mx_blocks(y)
    mag = q.abs()
    code = torch.where(mag < 2, mag * 2, torch.where(mag < 4, mag + 2, mag / 2 + 4)).to(U8)
    code = (code | (torch.signbit(q).to(U8) << 3)).reshape(y.shape[0], -1, 2)
    rows, blocks = s.shape
    R, C = -(-rows // 128), 2 * -(-blocks // 8)
    pad = torch.zeros(R * 128, C * 4, dtype=U8, device=y.device)
    pad[:rows, :blocks] = s.to(U8)
    tiles = pad.view(R, 4, 32, C, 4).permute(0, 3, 2, 1, 4).reshape(R, C, 512).contiguous()
    return (code[..., 0] | (code[..., 1] << 4)).contiguous(), tiles


def _mx_unpack(q, tiles, dtype=F32):
    rows, K = q.shape[0], q.shape[1] * 2
    code = torch.stack([q & 15, q >> 4], -1).reshape(rows, K // BLOCK, BLOCK)
    mag = (code & 7).to(dtype)
    mag = torch.where(mag < 4, mag / 2, torch.where(mag < 6, mag - 2, (mag - 4) * 2))
    val = torch.where(code >= 8, -mag, mag)
    R, C, _ = tiles.shape
    s = tiles.view(R, C, 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(R * 128, C * 4)[:rows, :K // BLOCK]
    return (val * _e8m0(s).to(dtype).unsqueeze(-1)).reshape(rows, K)


# ------------------------------------------------------------------ inputs
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed))


def _shapes(text):
    return [tuple(int(v) for v in s.split("x")) for s in text.split(",")]


def _activations(g, rows, cols):
    """A residual stream: rows of different size, a few columns that stand out."""
    x = torch.randn(rows, cols, device=DEV, generator=g)
    x *= torch.exp(0.5 * torch.randn(rows, 1, device=DEV, generator=g))
    return (x * (1 + 8 * (torch.rand(cols, device=DEV, generator=g) > 0.995))).to(BF)


_K = None


def _kernels():
    global _K
    if _K is None:
        from dataflow_b200.ops import resolve_kernels
        _K = resolve_kernels().lowbit
    return _K


def prepare(case, seed):
    g, op = _gen(seed), case["op"]
    if op == "adamw":
        shapes = _shapes(case["sizes"])
        numel = [math.prod(s) for s in shapes]
        starts, at = [], 0
        for n in numel:                                   # fields at multiples of 128 elements, as in a packed object
            starts.append(at)
            at += -(-n // STATE_BLOCK) * STATE_BLOCK
        live = torch.zeros(at // STATE_BLOCK, STATE_BLOCK, device=DEV)
        st = {"op": op, "bits": case["bits"], "N": at, "step": 7, "lr": 3e-4}
        for a, n in zip(starts, numel):
            live.view(-1)[a:a + n] = 1
        live = live.view(-1)

        def normal(scale):
            return torch.randn(at, device=DEV, generator=g) * scale * live

        # gradients whose size changes from block to block, moments that fit them
        size = torch.exp(2.0 * torch.randn(at // STATE_BLOCK, 1, device=DEV, generator=g)).expand(-1, STATE_BLOCK).reshape(-1) * 1e-3
        grad, m, r = normal(1.0) * size, normal(0.3) * size, normal(1.0).abs() * size * live
        w = normal(0.02)
        if case["weights"] == "fp32":
            st["w"] = w
        else:
            st["w"] = w.to(BF)
            if case["weights"] == "master":
                st["master"] = w
        st["g"] = grad.to(BF if case["grad"] == "bf16" else F32)
        if case["bits"] == 8:
            for name, t in (("m", m), ("v", r)):
                b = t.view(-1, STATE_BLOCK)
                s = (b.abs().amax(-1) / 448).clamp(min=2.0 ** -120)
                st[name], st[name + "_scale"] = (b / s[:, None]).clamp(-448, 448).to(F8).view(-1), s
        else:
            st["m"], st["v"] = m, r * r
        # the element index inside its own field, and the weight decay (matrices only), per block of 128
        first = torch.zeros(at // STATE_BLOCK, dtype=torch.int64, device=DEV)
        wd = torch.zeros(at // STATE_BLOCK, device=DEV)
        for a, n, s in zip(starts, numel, shapes):
            lo, hi = a // STATE_BLOCK, -(-(a + n) // STATE_BLOCK)
            first[lo:hi] = a
            wd[lo:hi] = 0.1 if len(s) > 1 else 0.0
        st["first"], st["wd"] = first, wd
        st["wds"] = [0.1 if len(s) > 1 else 0.0 for s in shapes]
        st["fields"] = {}
        for name in ("w", "g", "m", "v", "master"):
            if name in st:
                st["fields"][name] = [st[name][a:a + n] for a, n in zip(starts, numel)]
        for name in ("m_scale", "v_scale"):
            if name in st:
                st["fields"][name] = [st[name][a // STATE_BLOCK:-(-(a + n) // STATE_BLOCK)] for a, n in zip(starts, numel)]
        return st
    if op == "norm":
        rows, cols = case["rows"], case["cols"]
        return {"op": op, "fmt": case["fmt"], "x": _activations(g, rows, cols),
                "residual": _activations(g, rows, cols) if case["residual"] else None,
                "w": (1 + 0.2 * torch.randn(cols, device=DEV, generator=g)).to(BF)}
    if op == "quant":
        x = _activations(g, case["rows"], case["cols"])
        return {"op": op, "x": x * 0.02 if case["transpose"] else x, "transpose": case["transpose"]}
    m, n, k = case["m"], case["n"], case["k"]
    if op == "product":
        xq, xs = _mx_pack(_activations(g, m, k).float())
        wq, ws = _mx_pack(torch.randn(n, k, device=DEV, generator=g) * k ** -0.5)
        add = torch.randn(m, n, device=DEV, generator=g).to(BF if case["out"] == "bf16" else F32) if case["add"] else None
        return {"op": op, "xq": xq, "xs": xs, "wq": wq, "ws": ws, "add": add, "dtype": BF if case["out"] == "bf16" else F32}
    return {"op": op, "x": _activations(g, m, k), "w": (torch.randn(k, n, device=DEV, generator=g) * k ** -0.5).to(BF),
            "dy": (torch.randn(m, n, device=DEV, generator=g) * 0.1).to(BF)}


# ------------------------------------------------------------------ one pass
B1, B2, ADAM_EPS = 0.9, 0.95, 1e-8


def run(st):
    return {"adamw": _run_adamw, "norm": _run_norm, "quant": _run_quant, "product": _run_product, "linear": _run_linear}[st["op"]](st)


def _hash32(x):
    """A 32-bit mix of integers in [0, 2^32), held in 64 bits."""
    x = x ^ (x >> 16)
    x = (x * 0x7FEB352D) & 0xFFFFFFFF
    x = x ^ (x >> 15)
    x = (x * 0x846CA68B) & 0xFFFFFFFF
    return x ^ (x >> 16)


def _dither(st):
    """Two 16-bit random numbers per element from its index in its own field and the step."""
    idx = (torch.arange(st["N"], device=DEV).view(-1, STATE_BLOCK) - st["first"][:, None]).view(-1)
    h = _hash32((idx * 0x9E3779B9 + st["step"] * 0x85EBCA6B) & 0xFFFFFFFF)
    return h & 0xFFFF, h >> 16


def _e4m3_dithered(y, rnd, floor):
    """e4m3 of y (|y| <= 448): up or down to a neighbour with the odds of the distance; a nonzero |y| is at least ``floor``."""
    a = y.abs()
    base = torch.where(a < 2.0 ** -6, 2.0 ** -6, 0.0)
    bits = ((a + base).view(torch.int32) + (rnd << 4).to(torch.int32)) & -0x100000
    q = (bits.view(F32) - base).clamp(max=448.0)
    if floor:
        q = torch.where(a > 0, q.clamp(min=floor), q)
    return torch.copysign(q, y).to(F8)


def _run_adamw(st):
    if own:
        f = st["fields"]
        _kernels().adamw_multi_step(f["w"], f["g"], f["m"], f["v"], st["lr"], B1, B2, ADAM_EPS, st["wds"], st["step"],
                                    masters=f.get("master"), m_scales=f.get("m_scale"), v_scales=f.get("v_scale"))
        return {k: st[k] for k in ("w", "m", "v", "master", "m_scale", "v_scale") if k in st}
    bc1, bc2 = 1 - B1 ** st["step"], 1 - B2 ** st["step"]
    g = st["g"].float()
    each = lambda s: s[:, None].expand(-1, STATE_BLOCK).reshape(-1)
    if st["bits"] == 8:
        m = st["m"].float() * each(st["m_scale"])
        r = st["v"].float() * each(st["v_scale"])
        m = m * B1 + g * (1 - B1)
        r = torch.sqrt((r * r) * B2 + (g * g) * (1 - B2))
        lo, hi = _dither(st)
        for name, t, rnd, floor in (("m", m, lo, 0.0), ("v", r, hi, 2.0 ** -9)):
            s = (t.view(-1, STATE_BLOCK).abs().amax(-1) / 448).clamp(min=2.0 ** -120)
            st[name + "_scale"].copy_(s)
            st[name].copy_(_e4m3_dithered(t * each(1 / s), rnd, floor))
    else:
        m = st["m"] * B1 + g * (1 - B1)
        v = st["v"] * B2 + (g * g) * (1 - B2)
        st["m"].copy_(m)
        st["v"].copy_(v)
        r = torch.sqrt(v)
    w = st["master"] if "master" in st else st["w"].float()
    w = w - st["lr"] * ((m / bc1) / (r / math.sqrt(bc2) + ADAM_EPS) + each(st["wd"]) * w)
    if "master" in st:
        st["master"].copy_(w)
    st["w"].copy_(w)
    return {k: st[k] for k in ("w", "m", "v", "master", "m_scale", "v_scale") if k in st}


def _run_norm(st):
    x, w, res = st["x"], st["w"], st["residual"]
    if own:
        K = _kernels()
        if st["fmt"] == "fp8":
            q, s, h, rstd = K.rmsnorm_fp8(x, w, EPS, residual=res)
            return {"q": q, "scale": s, "h": h, "rstd": rstd}
        q, s, h, rstd = K.rmsnorm_mxfp4(x, w, EPS, residual=res)
        return {"values": K.dequant_mxfp4(q, s), "h": h, "rstd": rstd}
    h = x if res is None else (x.float() + res.float()).to(BF)
    hf = h.float()
    rstd = torch.rsqrt((hf * hf).mean(-1) + EPS)
    y = hf * rstd[:, None] * w.float()
    if st["fmt"] == "fp8":
        amax = y.abs().amax(-1)
        s = torch.where(amax > 0, (amax / 448).clamp(min=2.0 ** -120), 1.0)
        return {"q": (y * (1 / s)[:, None]).clamp(-448, 448).to(F8), "scale": s, "h": h, "rstd": rstd}
    return {"values": _mx_values(y).to(BF), "h": h, "rstd": rstd}


def _run_quant(st):
    if own:
        K = _kernels()
        return K.dequant_mxfp4(*K.quant_mxfp4(st["x"], transpose=st["transpose"]))
    x = st["x"].t() if st["transpose"] else st["x"]
    return _mx_values(x.float().contiguous()).to(BF)


def _run_product(st):
    if own:
        return _kernels().linear_mxfp4(st["xq"], st["xs"], st["wq"], st["ws"], add=st["add"], out_dtype=st["dtype"])
    y = _mx_unpack(st["xq"], st["xs"]) @ _mx_unpack(st["wq"], st["ws"]).t()
    if st["add"] is not None:
        y = y + st["add"].float()
    return y.to(st["dtype"])


def _run_linear(st):
    x, w, dy = st["x"], st["w"], st["dy"]
    if own:
        from dataflow_b200.models import _forms
        x, w = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
        y = _forms.linear(x, w, "mxfp4")
        dx, dw = torch.autograd.grad(y, [x, w], dy)
        return {"y": y.detach(), "dx": dx, "dw": dw}
    xf, wf, df = x.float(), w.float(), dy.float()
    y = _mx_values(xf) @ _mx_values(wf.t().contiguous()).t()
    # the backward passes the rounding straight through: exact operands
    return {"y": y.to(BF), "dx": (df @ wf.t()).to(BF), "dw": (xf.t() @ df).to(BF)}


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    op = case["op"]
    if op == "adamw":
        n = sum(math.prod(s) for s in _shapes(case["sizes"]))
        wb = {"bf16": 4, "fp32": 8, "master": 8 + 2}[case["weights"]]
        sb = 4 * (1 + 4 / STATE_BLOCK) if case["bits"] == 8 else 16
        return {"bytes": n * (wb + sb + (2 if case["grad"] == "bf16" else 4)), "flops": 18.0 * n}
    if op == "norm":
        n = case["rows"] * case["cols"]
        out = n * 1.0 if case["fmt"] == "fp8" else n * 2.0          # codes, or the values in 16 bits
        return {"bytes": n * (2 + (4 if case["residual"] else 0)) + out + 8 * case["rows"] + 2 * case["cols"], "flops": 6.0 * n}
    if op == "quant":
        n = case["rows"] * case["cols"]
        return {"bytes": 4.0 * n, "flops": 4.0 * n}
    m, n, k = case["m"], case["n"], case["k"]
    if op == "product":
        ob = 2 if case["out"] == "bf16" else 4
        return {"bytes": (m + n) * k * (0.5 + 1 / BLOCK) + m * n * ob * (2 if case["add"] else 1), "flops": 2.0 * m * n * k}
    return {"bytes": 2.0 * (2 * m * k + 2 * k * n + 2 * m * n), "flops": 6.0 * m * n * k}


# ------------------------------------------------------------------ the definition in 64 bits
def _exact_e4m3(y):
    """Nearest e4m3 of y in 64 bits, ties to the even code."""
    a = y.abs().clamp(max=448.0)
    _, e = torch.frexp(a)
    step = torch.ldexp(torch.ones_like(a), ((e - 1).clamp(min=-6) - 3))
    return torch.copysign(torch.round(a / step) * step, y)


def _exact_mx(y):
    b = y.reshape(y.shape[0], -1, BLOCK)
    _, e = torch.frexp(b.abs().amax(-1))
    e = torch.where(b.abs().amax(-1) > 0, (e - 1 - 2).clamp(min=-127), torch.full_like(e, -127))
    X = torch.ldexp(torch.ones_like(e, dtype=F64), e).unsqueeze(-1)
    return (_e2m1_round(b / X) * X).reshape(y.shape)


def exact(case, seed):
    st, op = prepare(case, seed), case["op"]
    if op == "adamw":
        each = lambda s: s.double()[:, None].expand(-1, STATE_BLOCK).reshape(-1)
        g, out = st["g"].double(), {}
        bc1, bc2 = 1 - B1 ** st["step"], 1 - B2 ** st["step"]
        if case["bits"] == 8:
            m = B1 * st["m"].double() * each(st["m_scale"]) + (1 - B1) * g
            r = torch.sqrt(B2 * (st["v"].double() * each(st["v_scale"])).square() + (1 - B2) * g * g)
            for name, t, rnd, floor in (("m", m, _dither(st)[0], 0.0), ("v", r, _dither(st)[1], 2.0 ** -9)):
                s = (t.view(-1, STATE_BLOCK).abs().amax(-1) / 448).clamp(min=2.0 ** -120)
                a = (t / each(s)).abs()
                _, e = torch.frexp(a)
                grid = torch.ldexp(torch.ones_like(a), (e - 1).clamp(min=-6) - 3)
                q = (torch.floor(a / grid + rnd.double() / 65536) * grid).clamp(max=448.0)
                q = torch.where(a > 0, q.clamp(min=floor), q)
                out[name], out[name + "_scale"] = torch.copysign(q, t), s
                del a, e, grid, q
        else:
            m = B1 * st["m"].double() + (1 - B1) * g
            v = B2 * st["v"].double() + (1 - B2) * g * g
            out["m"], out["v"], r = m, v, torch.sqrt(v)
        w = (st["master"] if "master" in st else st["w"]).double()
        w = w - st["lr"] * ((m / bc1) / (r / math.sqrt(bc2) + ADAM_EPS) + each(st["wd"]) * w)
        out["w"] = w
        if "master" in st:
            out["master"] = w
        return out
    if op == "norm":
        h = st["x"].double()
        if st["residual"] is not None:
            h = (st["x"].double() + st["residual"].double()).to(BF).double()     # the stream itself is kept in 16 bits
        rstd = 1 / torch.sqrt(h.square().mean(-1) + EPS)
        y = h * rstd[:, None] * st["w"].double()
        if case["fmt"] == "mxfp4":
            return {"values": _exact_mx(y), "h": h, "rstd": rstd}
        amax = y.abs().amax(-1)
        s = torch.where(amax > 0, (amax / 448).clamp(min=2.0 ** -120), 1.0)
        return {"q": _exact_e4m3(y / s[:, None]), "scale": s, "h": h, "rstd": rstd}
    if op == "quant":
        x = st["x"].double()
        return _exact_mx((x.t() if case["transpose"] else x).contiguous())
    if op == "product":
        y = _mx_unpack(st["xq"], st["xs"], F64) @ _mx_unpack(st["wq"], st["ws"], F64).t()
        return y if st["add"] is None else y + st["add"].double()
    x, w, dy = st["x"].double(), st["w"].double(), st["dy"].double()
    return {"y": _exact_mx(x) @ _exact_mx(w.t().contiguous()).t(), "dx": dy @ w.t(), "dw": x.t() @ dy}
