"""Native lane of the narrow-format operators, ``K.lowbit.<op>``: hand-written sm_100a kernels (``csrc/adamw_multi.cu``,
``norm_quant.cu``, ``mxfp4.cu``, ``gemm_mxfp4.cu``).  Formats, shapes and semantics: ``lowbit_eager``, whose functions these
replace one for one.  Arguments are checked in the extension; a refusal raises ``ValueError``.  Each call works on the device of
its operands, on that device's current stream, and can be captured into a graph."""
from __future__ import annotations

import torch

from . import lowbit_eager as E
from . import native
from .cuda import LAUNCHES, P, _native
from .registry import register


def _reg(op, launches=1):
    def deco(f):
        def counted(*a, **k):
            LAUNCHES.total += launches
            return f(*a, **k)
        counted.__name__, counted.__doc__ = f.__name__, getattr(E, op).__doc__
        register(op, "sm100", counted, priority=P, requires=_native, native=True, op_set="lowbit")
        return f
    return deco


@_reg("quant_mxfp4")
def quant_mxfp4(x, transpose: bool = False):
    return native().quant_mxfp4(x, transpose)


@_reg("dequant_mxfp4")
def dequant_mxfp4(q, scale, dtype=torch.bfloat16):
    return native().dequant_mxfp4(q, scale, dtype)


@_reg("linear_mxfp4")
def linear_mxfp4(xq, x_scale, wq, w_scale, out=None, add=None, bias=None, out_dtype=torch.bfloat16):
    return native().linear_mxfp4(xq, x_scale, wq, w_scale, out, add, bias, out_dtype)


@_reg("linear_fwd_mxfp4", launches=3)
def linear_fwd_mxfp4(x, w, out=None, add=None, bias=None):
    xq, xs = native().quant_mxfp4(x, False)
    wq, ws = native().quant_mxfp4(w, True)
    return native().linear_mxfp4(xq, xs, wq, ws, out, add, bias, x.dtype)


@_reg("rmsnorm_fp8")
def rmsnorm_fp8(x, w, eps: float = 1e-5, residual=None, rstd=None, h_out=None):
    return native().rmsnorm_fp8(x, w, eps, residual, rstd, h_out)


@_reg("rmsnorm_mxfp4")
def rmsnorm_mxfp4(x, w, eps: float = 1e-5, residual=None, rstd=None, h_out=None):
    return native().rmsnorm_mxfp4(x, w, eps, residual, rstd, h_out)


@_reg("adamw_multi_step")
def adamw_multi_step(ws, gs, ms, vs, lr, beta1=0.9, beta2=0.95, eps=1e-8, wds=0.0, step=1, masters=None, los=None,
                     m_scales=None, v_scales=None, gscale=1.0, seed=None):
    wds = [float(wds)] * len(ws) if isinstance(wds, (int, float)) else wds
    each = isinstance(seed, (list, tuple))
    native().adamw_multi(ws, gs, ms, vs, lr, beta1, beta2, eps, wds, step, masters, los, m_scales, v_scales, gscale,
                         0 if each else (step if seed is None else seed) & 0xFFFFFFFF, [s & 0xFFFFFFFF for s in seed] if each else None)
    return ws
