"""Plain-torch lane of the narrow-format operators (``K.lowbit``): the oracle of their tests and the path on machines without
a GPU.  The mathematics is in 32 bits and rounds once into the narrow format.

**8 bits with a scale per row** (``rmsnorm_fp8``): codes e4m3, x ~= q * scale[row]; the form ``linear_fp8`` takes.

**Microscaled 4 bits** (``mxfp4``): blocks of 32 elements along the contraction share a power-of-two scale X (one e8m0 byte,
255 = NaN) and hold e2m1 codes (0 0.5 1 1.5 2 3 4 6 and their negatives).  X = 2^max(floor(log2 amax) - 2, -127); an element is
x / X rounded to nearest even, saturating at 6 (amax / X lies in [4, 8)).  A block that holds an infinity or a NaN gets X = NaN.
Codes are packed two to a byte, the even element in the low nibble.  Scales are stored in tiles of 128 rows x 4 blocks, the
form the tensor core's scale memory wants: ``scale`` is (ceil(rows / 128), 2 ceil(K / 256), 512) uint8 and the byte of row r,
block b is ``scale[r // 128, b // 4, (r % 32) * 16 + (r % 128 // 32) * 4 + b % 4]``; bytes past the rows and blocks are zero.

**8-bit optimizer moments** (``adamw_multi_step``): the first moment and the ROOT of the second are e4m3 codes with an fp32
scale per 128 consecutive elements (amax / 448).  They round stochastically: a moment that moves by less than half a step per
update (one minus beta is smaller than the format's step) would otherwise never move, and the second moment would only ever
grow.  The random bits are a hash of (element index, seed), so a step is reproducible.  A positive root never rounds to zero,
so no update divides by epsilon alone where the gradient was merely small beside its neighbours.
"""
from __future__ import annotations

import math

import torch

from .eager import linear_fp8, split_master_cut, split_master_join          # noqa: F401
from .registry import register

MX_BLOCK = 32
STATE_BLOCK = 128
E4M3_MAX = 448.0
MIN_SCALE = 2.0 ** -120          # floor of an fp32 scale: its reciprocal stays finite


def _reg(op):
    return register(op, "eager", op_set="lowbit")


def _need(ok, msg):
    if not ok:
        raise ValueError(msg)


# ------------------------------------------------------------------ the 4-bit format
def mxfp4_scale_shape(rows: int, K: int) -> tuple[int, int, int]:
    return (-(-rows // 128), 2 * -(-K // 256), 512)


def mxfp4_scale_tiles(s):
    """Scale bytes (rows, K / 32) in row order -> the tiled form the operators take."""
    rows, blocks = s.shape
    R, C, _ = mxfp4_scale_shape(rows, blocks * MX_BLOCK)
    pad = torch.zeros(R * 128, C * 4, dtype=torch.uint8, device=s.device)
    pad[:rows, :blocks] = s
    return pad.view(R, 4, 32, C, 4).permute(0, 3, 2, 1, 4).reshape(R, C, 512).contiguous()


def mxfp4_scale_rows(scale, rows: int, K: int):
    """The inverse: the tiled scale bytes -> (rows, K / 32) in row order."""
    R, C, _ = scale.shape
    return scale.view(R, C, 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(R * 128, C * 4)[:rows, :K // MX_BLOCK]


def _e8m0(s):
    e = s.to(torch.int32)
    bits = torch.where(e == 0, torch.full_like(e, 0x00400000), e << 23)
    return torch.where(e == 255, torch.full_like(e, 0x7FC00000), bits).view(torch.float32)


def _mx_encode(y):
    """y (rows, K) fp32 -> (codes (rows, K / 2), tiled scales)."""
    rows, K = y.shape
    b = y.reshape(rows, K // MX_BLOCK, MX_BLOCK)
    amax = torch.where(b == b, b.abs(), torch.full_like(b, math.inf)).amax(-1) if K else b.new_zeros(rows, 0)
    e = (amax.view(torch.int32) >> 23) & 255
    s = torch.where(e == 255, e, (e - 2).clamp(min=0))
    a = b * ((254 - s.clamp(max=253)) << 23).view(torch.float32).unsqueeze(-1)          # x / X, exact: X is a power of two
    mag = a.abs()
    step = torch.where(mag < 2, 0.5, torch.where(mag < 4, 1.0, 2.0))
    mag = torch.nan_to_num((torch.round(mag / step) * step).clamp(max=6.0), nan=6.0)
    code = torch.where(mag < 2, mag * 2, torch.where(mag < 4, mag + 2, mag / 2 + 4)).to(torch.uint8)
    code = (code | (torch.signbit(a).to(torch.uint8) << 3)).reshape(rows, K // 2, 2)
    return (code[..., 0] | (code[..., 1] << 4)).contiguous(), mxfp4_scale_tiles(s.to(torch.uint8))


@_reg("quant_mxfp4")
def quant_mxfp4(x, transpose: bool = False):
    """x (rows, K) bf16 or fp32 -> (q (rows, K / 2) uint8, scale tiles); ``transpose``: x is stored (K, rows), the way weights
    are ((in, out) with the contraction first).  K is a multiple of 32; rows of x may be strided."""
    _need(x.dim() == 2, "quant_mxfp4: x is a matrix")
    _need(x.dtype in (torch.bfloat16, torch.float32), "quant_mxfp4: x is bf16 or fp32")
    _need(x.stride(1) == 1 or x.shape[1] <= 1, "quant_mxfp4: the last axis of x must be contiguous (transpose=True takes a weight as it is stored)")
    K = x.shape[0] if transpose else x.shape[1]
    _need(K > 0 and K % MX_BLOCK == 0, "quant_mxfp4: the contraction length must be a positive multiple of 32")
    return _mx_encode((x.t() if transpose else x).float().contiguous())


@_reg("dequant_mxfp4")
def dequant_mxfp4(q, scale, dtype=torch.bfloat16):
    """The values (rows, K) that codes and scales stand for, exact in bf16 and in fp32."""
    _check_mx("dequant_mxfp4", q, scale)
    _need(dtype in (torch.bfloat16, torch.float32), "dequant_mxfp4: values are bf16 or fp32")
    rows, K = q.shape[0], q.shape[1] * 2
    code = torch.stack([q & 15, q >> 4], -1).reshape(rows, K // MX_BLOCK, MX_BLOCK)
    mag = (code & 7).float()
    mag = torch.where(mag < 4, mag / 2, torch.where(mag < 6, mag - 2, (mag - 4) * 2))
    val = torch.where(code >= 8, -mag, mag)
    return (val * _e8m0(mxfp4_scale_rows(scale, rows, K)).unsqueeze(-1)).reshape(rows, K).to(dtype)


def _check_mx(op, q, scale, what=""):
    _need(q.dim() == 2 and q.dtype == torch.uint8 and q.is_contiguous(), f"{op}: {what}codes are a contiguous (rows, K / 2) uint8 matrix")
    _need(q.shape[1] > 0 and q.shape[1] % 16 == 0, f"{op}: {what}codes cover a positive multiple of 32 elements per row")
    _need(scale.dtype == torch.uint8 and scale.is_contiguous() and tuple(scale.shape) == mxfp4_scale_shape(q.shape[0], 2 * q.shape[1]),
          f"{op}: {what}scales are a contiguous uint8 tensor of shape (ceil(rows / 128), 2 ceil(K / 256), 512)")


@_reg("linear_mxfp4")
def linear_mxfp4(xq, x_scale, wq, w_scale, out=None, add=None, bias=None, out_dtype=torch.bfloat16):
    """y (M, N) = x (M, K) @ w (N, K)^T (+ bias) (+ add) of two operands in the 4-bit format, fp32 accumulation, one rounding."""
    _check_mx("linear_mxfp4", xq, x_scale, "x ")
    _check_mx("linear_mxfp4", wq, w_scale, "w ")
    _need(xq.shape[1] == wq.shape[1], "linear_mxfp4: both operands have the same K")
    M, N = xq.shape[0], wq.shape[0]
    dt = out.dtype if out is not None else out_dtype
    _need(dt in (torch.bfloat16, torch.float32), "linear_mxfp4: the result is bf16 or fp32")
    _need(out is None or (tuple(out.shape) == (M, N) and out.stride(1) == 1), "linear_mxfp4: out is (M, N) with contiguous rows")
    _need(add is None or (tuple(add.shape) == (M, N) and add.dtype == dt and add.stride(1) == 1), "linear_mxfp4: add is like the result")
    _need(bias is None or (tuple(bias.shape) == (N,) and bias.dtype == torch.bfloat16), "linear_mxfp4: bias is (N,) bf16")
    y = dequant_mxfp4(xq, x_scale, torch.float32) @ dequant_mxfp4(wq, w_scale, torch.float32).t()
    if bias is not None:
        y = y + bias.float()
    if add is not None:
        y = y + add.float()
    if out is not None:
        out.copy_(y)
        return out
    return y.to(dt)


@_reg("linear_fwd_mxfp4")
def linear_fwd_mxfp4(x, w, out=None, add=None, bias=None):
    """``linear_fwd_bf16`` with both operands rounded to the 4-bit format along the contraction first: x (M, K), w (K, N)
    stored (in, out)."""
    xq, xs = quant_mxfp4(x)
    wq, ws = quant_mxfp4(w, transpose=True)
    return linear_mxfp4(xq, xs, wq, ws, out=out, add=add, bias=bias, out_dtype=out.dtype if out is not None else x.dtype)


# ------------------------------------------------------------------ the norm with a narrow output
def _norm(op, x, w, eps, residual, rstd, h_out, mult):
    cols = x.shape[-1] if x.dim() else 0
    _need(x.dim() >= 1 and cols > 0 and cols % mult == 0, f"{op}: the width must be a positive multiple of {mult}")
    _need(tuple(w.shape) == (cols,), f"{op}: w has one entry per column")
    _need(residual is None or residual.shape == x.shape, f"{op}: residual is like x")
    _need(h_out is None or (residual is not None and h_out.shape == x.shape and h_out.dtype == x.dtype),
          f"{op}: h_out is like x and comes with a residual")
    _need(rstd is None or rstd.numel() == x.numel() // cols, f"{op}: rstd has one entry per row")
    h = x if residual is None else (x.float() + residual.float()).to(x.dtype)
    if h_out is not None:
        h = h_out.copy_(h)
    hf = h.float().reshape(-1, cols)
    rstd = torch.rsqrt(hf.pow(2).mean(-1) + eps) if rstd is None else rstd.reshape(-1).float()
    return hf * rstd[:, None] * w.float(), h, rstd


@_reg("rmsnorm_fp8")
def rmsnorm_fp8(x, w, eps: float = 1e-5, residual=None, rstd=None, h_out=None):
    """h = x (+ residual, rounded to x's type); y = h * rstd * w, left as e4m3 codes with one fp32 scale per row.
    Returns (q like x, scale (rows,), h, rstd (rows,)).  ``rstd``: statistics saved by an earlier call, applied instead of
    computed (the same codes again).  The gradient, straight through the rounding, is ``rmsnorm_bwd(dy, h, w, rstd, dx_add=dh)``."""
    y, h, rstd = _norm("rmsnorm_fp8", x, w, eps, residual, rstd, h_out, 8)
    amax = torch.where(y == y, y.abs(), torch.zeros_like(y)).amax(-1)
    s = torch.where(amax > 0, (amax * (1 / E4M3_MAX)).clamp(min=MIN_SCALE), torch.ones_like(amax))
    q = (y * (1 / s)[:, None]).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)
    return q.view(x.shape), s, h, rstd


@_reg("rmsnorm_mxfp4")
def rmsnorm_mxfp4(x, w, eps: float = 1e-5, residual=None, rstd=None, h_out=None):
    """``rmsnorm_fp8`` with its output in the 4-bit format instead: (q (rows, cols / 2) uint8, scale tiles, h, rstd)."""
    y, h, rstd = _norm("rmsnorm_mxfp4", x, w, eps, residual, rstd, h_out, MX_BLOCK)
    q, s = _mx_encode(y)
    return q, s, h, rstd


# ------------------------------------------------------------------ AdamW over many tensors
def _mix32(x):
    """32-bit integer mixer (two xor-shift-multiply rounds; shifts and factors from C. Wellons, "Prospecting for Hash Functions", 2018),
    on int64 tensors that hold values below 2^32."""
    x = x ^ (x >> 16)
    x = (x * 0x7FEB352D) & 0xFFFFFFFF
    x = x ^ (x >> 15)
    x = (x * 0x846CA68B) & 0xFFFFFFFF
    return x ^ (x >> 16)


def state_dither(n: int, seed: int, device=None):
    """The two 16-bit random numbers (first moment, root of the second) of every element of a tensor of ``n``."""
    idx = torch.arange(n, dtype=torch.int64, device=device)
    h = _mix32(((idx & 0xFFFFFFFF) * 0x9E3779B9 + (idx >> 32) * 0xC2B2AE35 + (int(seed) & 0xFFFFFFFF) * 0x85EBCA6B) & 0xFFFFFFFF)
    return h & 0xFFFF, h >> 16


def dither_e4m3(y, rnd, floor: float = 0.0):
    """e4m3 of y (|y| <= 448) rounded up or down with the odds of the distance; ``rnd``: 16 random bits per element."""
    a = y.abs()
    base = torch.where(a < 2.0 ** -6, 2.0 ** -6, 0.0)            # brings subnormal codes onto one binade's grid
    bits = ((a + base).view(torch.int32) + (rnd << 4).to(torch.int32)) & -0x100000
    q = torch.where(a == a, (bits.view(torch.float32) - base).clamp(max=E4M3_MAX), a)          # a NaN's bits would carry over
    if floor:
        q = torch.where(a > 0, q.clamp(min=floor), q)
    return torch.copysign(q, y).to(torch.float8_e4m3fn)


def _state_load(q, scale):
    n = q.numel()
    return q.float() * scale.repeat_interleave(STATE_BLOCK)[:n]


def _state_store(t, q, scale, rnd, floor):
    n = t.numel()
    pad = torch.nn.functional.pad(torch.where(t == t, t.abs(), torch.zeros_like(t)), (0, -n % STATE_BLOCK))
    scale.copy_((pad.view(-1, STATE_BLOCK).amax(-1) * (1 / E4M3_MAX)).clamp(min=MIN_SCALE))
    q.copy_(dither_e4m3(t * (1 / scale).repeat_interleave(STATE_BLOCK)[:n], rnd, floor))


@_reg("adamw_multi_step")
def adamw_multi_step(ws, gs, ms, vs, lr, beta1=0.9, beta2=0.95, eps=1e-8, wds=0.0, step=1, masters=None, los=None,
                     m_scales=None, v_scales=None, gscale=1.0, seed=None):
    """One decoupled-weight-decay Adam update of every tensor of the lists, in place; returns ``ws``.

    ws bf16 (alone, or the working copy of an fp32 ``masters``, or the high half of a split master whose int16 low halves are
    ``los``) or fp32; gs bf16 or fp32; moments fp32, or 8 bits (``float8_e4m3fn``, with ``m_scales`` / ``v_scales`` fp32 of
    ceil(n / 128) entries; ``vs`` then holds the root of the second moment).  One choice of types per call.  ``wds``: weight
    decay, a number or one per tensor.  ``seed`` of the 8-bit rounding, a number or one per tensor, defaults to ``step``: element
    i of every tensor then rounds with the same random bits.  The result of a tensor does not depend on the others in the list."""
    n = len(ws)
    lists = [("gs", gs), ("ms", ms), ("vs", vs), ("masters", masters), ("los", los), ("m_scales", m_scales), ("v_scales", v_scales)]
    for name, l in lists:
        _need(l is None or len(l) == n, f"adamw_multi_step: {name} has one entry per tensor")
    wds = [float(wds)] * n if isinstance(wds, (int, float)) else [float(x) for x in wds]
    _need(len(wds) == n, "adamw_multi_step: wds has one entry per tensor")
    _need(masters is None or los is None, "adamw_multi_step: masters and los exclude each other")
    _need(int(step) >= 1, "adamw_multi_step: step counts from 1")
    bits8 = bool(n) and ms[0].dtype == torch.float8_e4m3fn
    _need(not bits8 or (m_scales is not None and v_scales is not None), "adamw_multi_step: 8-bit moments come with m_scales and v_scales")
    _need(bits8 or (m_scales is None and v_scales is None) or not n, "adamw_multi_step: scales belong to 8-bit moments")
    spans = sorted((t.data_ptr(), t.data_ptr() + t.numel() * t.element_size(), written)
                   for l, written in ((ws, True), (gs, False), (ms, True), (vs, True), (masters, True), (los, True), (m_scales, True), (v_scales, True))
                   if l is not None for t in l if t.numel())
    end_written = end_any = 0               # how far the spans so far reach
    for start, end, written in spans:
        _need(start >= end_written and (not written or start >= end_any),
              "adamw_multi_step: a tensor that is written appears twice or overlaps another")
        end_written, end_any = max(end_written, end if written else 0), max(end_any, end)
    bc1, bc2 = 1 - beta1 ** int(step), 1 - beta2 ** int(step)
    seeds = list(seed) if isinstance(seed, (list, tuple)) else [int(step) if seed is None else int(seed)] * n
    _need(len(seeds) == n, "adamw_multi_step: seed has one entry per tensor")
    for i in range(n):
        w, g, m, v = ws[i], gs[i], ms[i], vs[i]
        k = w.numel()
        st = torch.float8_e4m3fn if bits8 else torch.float32
        _need(m.dtype == st and v.dtype == st, "adamw_multi_step: moments are all fp32 or all float8_e4m3fn")
        _need(w.dtype == ws[0].dtype and w.dtype in (torch.bfloat16, torch.float32), "adamw_multi_step: weights are all bf16 or all fp32")
        _need(g.dtype == gs[0].dtype and g.dtype in (torch.bfloat16, torch.float32), "adamw_multi_step: gradients are all bf16 or all fp32")
        _need((masters is None and los is None) or w.dtype == torch.bfloat16, "adamw_multi_step: masters and los go with bf16 weights")
        _need(masters is None or masters[i].dtype == torch.float32, "adamw_multi_step: masters are fp32")
        _need(los is None or los[i].dtype == torch.int16, "adamw_multi_step: los are int16")
        same = [g, m, v] + ([masters[i]] if masters is not None else []) + ([los[i]] if los is not None else [])
        _need(all(t.numel() == k for t in same), "adamw_multi_step: every operand of a tensor has its element count")
        _need(all(t.is_contiguous() for t in [w] + same), "adamw_multi_step: operands are contiguous")
        if bits8:
            nb = -(-k // STATE_BLOCK)
            _need(all(s.dtype == torch.float32 and s.numel() == nb and s.is_contiguous() for s in (m_scales[i], v_scales[i])),
                  "adamw_multi_step: scales are fp32, one per 128 elements")
        if not k:
            continue
        w, m, v = w.view(-1), m.view(-1), v.view(-1)
        gf = g.reshape(-1).float() * gscale
        if bits8:
            r = _state_load(v, v_scales[i].view(-1))
            m1 = _state_load(m, m_scales[i].view(-1)) * beta1 + gf * (1 - beta1)
            # correctly rounded everywhere: torch's own 32-bit root on the CPU is a last place off now and then
            r1 = torch.sqrt(((r * r) * beta2 + (gf * gf) * (1 - beta2)).double()).float()
            lo16, hi16 = state_dither(k, seeds[i], w.device)
            _state_store(m1, m, m_scales[i].view(-1), lo16, 0.0)
            _state_store(r1, v, v_scales[i].view(-1), hi16, 2.0 ** -9)
        else:
            m1 = m * beta1 + gf * (1 - beta1)
            v1 = v * beta2 + (gf * gf) * (1 - beta2)
            m.copy_(m1)
            v.copy_(v1)
            r1 = torch.sqrt(v1)
        wf = masters[i].view(-1) if masters is not None else split_master_join(w, los[i].view(-1)) if los is not None else w.float()
        wf = wf - lr * ((m1 * (1 / bc1)) / (r1 * (1 / math.sqrt(bc2)) + eps) + wds[i] * wf)
        if los is not None:
            hi, low = split_master_cut(wf)
            w.copy_(hi)
            los[i].view(-1).copy_(low)
        else:
            if masters is not None:
                masters[i].view(-1).copy_(wf)
            w.copy_(wf)
    return ws
