"""Narrow-format operators (``K.lowbit``): the quantising RMS norm, the microscaled 4-bit format and its product, AdamW over many
tensors with 8-bit or 32-bit moments.  Every numerics test runs on the plain-torch lane (CPU) and, on a device, on the kernels,
against the definition in 64 bits.

Tolerances count roundings: u = 2^-24 for one fp32 rounding, half a step of the output type for the last one."""
import math

import pytest
import torch

from dataflow_b200.ops import lowbit_eager as E
from dataflow_b200.ops import native, native_available, registered_ops, resolve_kernels

BF, F32, F64, F8, U8 = torch.bfloat16, torch.float32, torch.float64, torch.float8_e4m3fn, torch.uint8
U = 2.0 ** -24
LANES = [pytest.param("cpu", id="eager"), pytest.param("cuda", id="sm100", marks=pytest.mark.gpu)]
OPS = ["adamw_multi_step", "dequant_mxfp4", "linear_fwd_mxfp4", "linear_mxfp4", "quant_mxfp4", "rmsnorm_fp8", "rmsnorm_mxfp4"]


def lane(dev):
    K = resolve_kernels(kernel_set="eager" if dev == "cpu" else None).lowbit
    assert dev == "cpu" or K.native_ops() == OPS
    return K


def rnd(dev, *shape, seed=0, scale=1.0, dtype=BF):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype).to(dev)


def half_step(t):
    return torch.finfo(t).eps / 2


# ------------------------------------------------------------------ the definitions in 64 bits
def e2m1(a):
    """Nearest of 0 0.5 1 1.5 2 3 4 6 (ties to the even code), written as a search over the eight values."""
    grid = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=F64, device=a.device)
    d = (a.abs().unsqueeze(-1) - grid).abs()
    even = torch.arange(8, device=a.device) % 2
    best = torch.argmin(d + 1e-9 * even, -1)          # at a tie the even code is nearer by nothing but this
    return torch.copysign(grid[best], a)


def mx_ref(y):
    """Values of y (rows, K) fp64 in the 4-bit format, and the block scales."""
    b = y.double().reshape(y.shape[0], -1, 32)
    amax = b.abs().amax(-1)
    e = torch.where(amax > 0, torch.frexp(amax)[1] - 3, -127).clamp(min=-127)         # exact, unlike a logarithm's floor
    X = torch.ldexp(torch.ones_like(amax), e).unsqueeze(-1)
    return (e2m1(b / X) * X).reshape(y.shape), X.squeeze(-1)


def pow2(byte):
    return torch.ldexp(torch.ones(byte.shape, dtype=F64, device=byte.device), byte.to(torch.int32) - 127)


def unpack(K, q, s, dtype=F32):
    return K.dequant_mxfp4(q, s, dtype)


# ------------------------------------------------------------------ the table
def test_the_set_is_complete_and_every_op_has_the_plain_lane():
    resolve_kernels(kernel_set="eager")
    table = registered_ops("lowbit")
    assert sorted(table) == OPS
    for op, impls in table.items():
        names = {k.name: k for k in impls}
        assert set(names) == {"eager", "sm100"} and names["sm100"].native and names["sm100"].requires is not None and not names["eager"].native
    K = resolve_kernels(kernel_set="eager")
    assert K.lowbit.ops() == OPS and K.lowbit.native_ops() == [] and not set(OPS) & set(K.ops())
    with pytest.raises(AttributeError):
        K.lowbit.no_such_op


# ------------------------------------------------------------------ quantisation
@pytest.mark.parametrize("dev", LANES)
@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("transpose", [False, True], ids=["rows", "cols"])
@pytest.mark.parametrize("rows,K", [(1, 32), (1, 4096), (129, 32), (33, 96), (200, 288), (7, 2080), (300, 512), (65, 1056)])
def test_quant_is_the_format(dev, dtype, transpose, rows, K):
    """Powers of two scale exactly and the rounding is defined: codes and scales agree to the bit."""
    k = lane(dev)
    x = rnd(dev, rows, K, seed=rows + K, dtype=F32) * torch.exp(3 * rnd(dev, rows, 1, seed=1, dtype=F32))
    x = x.to(dtype)
    xin = x.t().contiguous() if transpose else x
    q, s = k.quant_mxfp4(xin, transpose=transpose)
    assert q.shape == (rows, K // 2) and tuple(s.shape) == E.mxfp4_scale_shape(rows, K)
    want, X = mx_ref(x)
    for dt in (BF, F32):
        got = k.dequant_mxfp4(q, s, dt)
        assert got.dtype == dt and torch.equal(got.double(), want)
    sr = E.mxfp4_scale_rows(s, rows, K)
    assert torch.equal(pow2(sr), X)
    assert torch.equal(E.mxfp4_scale_tiles(sr), s)            # every byte past the rows and blocks is zero


@pytest.mark.parametrize("dev", LANES)
def test_quant_edges(dev):
    """Ties go to the even code, values past 6 saturate, zero blocks stay zero, the smallest and the largest numbers, negative
    zero, and an infinity or a NaN makes its block (and only it) NaN."""
    k = lane(dev)
    x = torch.zeros(8, 64, dtype=F32)
    x[0, :16] = torch.tensor([4, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5, -5, -0.25, 6.9, 7.9, -7.9, -0.0, 0.26, 2.51])   # X = 1
    x[1, 0], x[1, 40] = float("inf"), 1.0
    x[2, 5], x[2, 41] = float("nan"), 1.0
    x[3, 0] = 2.0 ** -126
    x[4, 0], x[4, 1] = 3.0e38, -1.5e38
    x[5, 0] = 1e-44                                             # subnormal: below the smallest scale's half step
    x[6] = 1.0
    q, s = k.quant_mxfp4(x.to(dev))
    y = k.dequant_mxfp4(q, s, F32).cpu()
    assert y[0, :16].tolist() == [4, 0, 1, 1, 2, 2, 4, 4, -4, -0.0, 6, 6, -6, -0.0, 0.5, 3]
    assert torch.signbit(y[0, 13]) and torch.signbit(y[0, 9])
    for r, c in ((1, 0), (2, 0)):
        assert torch.isnan(y[r, :32]).all() and y[r, 32:].isfinite().all()
    assert y[1, 40] == 1 and y[2, 41] == 1
    assert y[3, 0] == 2.0 ** -126 and y[4, 0] == 1.5 * 2.0 ** 127
    assert torch.equal(y[3:5].double(), mx_ref(x[3:5])[0]) and y[5].abs().max() == 0 and torch.equal(y[6], x[6]) and y[7].abs().max() == 0
    sr = E.mxfp4_scale_rows(s.cpu(), 8, 64)
    assert sr[1, 0] == 255 and sr[2, 0] == 255 and sr[7, 0] == 0 and sr[5, 0] == 0


@pytest.mark.parametrize("dev", LANES)
def test_quant_takes_strided_and_offset_rows(dev):
    k = lane(dev)
    big = rnd(dev, 50, 200, seed=3)
    for view in (big[:, 3:99], big[:, 8:104], big[::2, :96], big[5:6, 1:65]):
        q, s = k.quant_mxfp4(view)
        q2, s2 = k.quant_mxfp4(view.contiguous())
        assert torch.equal(q, q2) and torch.equal(s, s2)
    for view in (big[:32, 3:100], big[:32, 8:9], big[18:, :77]):
        q, s = k.quant_mxfp4(view, transpose=True)
        q2, s2 = k.quant_mxfp4(view.t().contiguous())
        assert torch.equal(q, q2) and torch.equal(s, s2)


@pytest.mark.gpu
def test_more_rows_than_a_grid_axis_holds():
    """Both walks go out in slices there; rows behind the first slice are what a call on them alone gives."""
    k = lane("cuda")
    rows = 2_200_013
    x = torch.randn(rows, 32, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)).to(BF)
    q, s = k.quant_mxfp4(x)
    y = k.dequant_mxfp4(q, s)
    for a, b in ((0, 300), (2_096_896, 2_097_280), (rows - 141, rows)):
        q1, s1 = k.quant_mxfp4(x[a:b])
        assert torch.equal(q[a:b], q1) and torch.equal(y[a:b], k.dequant_mxfp4(q1, s1))


@pytest.mark.parametrize("dev", LANES)
def test_no_rows(dev):
    k = lane(dev)
    q, s = k.quant_mxfp4(torch.empty(0, 64, dtype=BF, device=dev))
    wq, ws = k.quant_mxfp4(rnd(dev, 24, 64))
    assert k.dequant_mxfp4(q, s).shape == (0, 64)
    assert k.linear_mxfp4(q, s, wq, ws).shape == (0, 24) and k.linear_mxfp4(wq, ws, q, s).shape == (24, 0)
    for fn in (k.rmsnorm_fp8, k.rmsnorm_mxfp4):
        out = fn(torch.empty(0, 64, dtype=BF, device=dev), rnd(dev, 64), residual=torch.empty(0, 64, dtype=BF, device=dev))
        assert out[2].shape == (0, 64) and out[3].numel() == 0
    assert k.adamw_multi_step([], [], [], [], 1e-3) == []
    z = lambda dt: [torch.empty(0, dtype=dt, device=dev)]
    k.adamw_multi_step(z(BF), z(BF), z(F32), z(F32), 1e-3)


# ------------------------------------------------------------------ the product
def product_bound(A, B, K, out):
    """fp32 accumulation of K exact products, each addition off by at most 2^-23 of the running magnitude (an adder that cuts
    instead of rounding), then one rounding to the output type."""
    return (K + 2) * 2.0 ** -23 * (A.abs() @ B.abs().t()) + half_step(out) * (A @ B.t()).abs() + 1e-30


@pytest.mark.parametrize("dev", LANES)
@pytest.mark.parametrize("out", [BF, F32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("M,N,K", [(1, 1, 32), (1, 8, 64), (3, 7, 96), (128, 128, 256), (129, 257, 288), (17, 520, 1056), (300, 40, 544),
                                   (257, 264, 2048), (130, 72, 32), (640, 513, 160), (65, 300, 4128), (2309, 4104, 544), (2100, 4099, 64)])
def test_product(dev, out, M, N, K):
    k = lane(dev)
    x = rnd(dev, M, K, seed=M, dtype=F32) * torch.exp(rnd(dev, M, 1, seed=2, dtype=F32))
    w = rnd(dev, N, K, seed=N + 1, scale=K ** -0.5, dtype=F32)
    a, b = k.quant_mxfp4(x), k.quant_mxfp4(w)
    A, B = unpack(k, *a).double(), unpack(k, *b).double()
    y = k.linear_mxfp4(*a, *b, out_dtype=out)
    assert y.dtype == out and y.shape == (M, N)
    bound = product_bound(A, B, K, out)
    assert ((y.double() - A @ B.t()).abs() <= bound).all()
    if dev == "cuda":
        assert native().gemm_mxfp4_last_error() == 0            # no bounded wait ran out
    add, bias = rnd(dev, M, N, seed=5, dtype=out), rnd(dev, N, seed=6)
    z = k.linear_mxfp4(*a, *b, add=add, bias=bias, out_dtype=out)
    want = A @ B.t() + add.double() + bias.double()
    extra = 2 * U * (add.double().abs() + bias.double().abs() + (A @ B.t()).abs()) + half_step(out) * want.abs()
    assert ((z.double() - want).abs() <= bound + extra).all()


@pytest.mark.parametrize("dev", LANES)
@pytest.mark.parametrize("M,N,K", [(1, 18944, 96), (17, 18945, 288), (64, 20001, 32), (65, 19001, 64), (5, 37889, 544)])
def test_product_few_tokens_of_a_wide_matrix(dev, M, N, K):
    """Either side of one wave of 128-row tiles, where the choice between the two product kernels turns."""
    k = lane(dev)
    a, b = k.quant_mxfp4(rnd(dev, M, K, seed=M)), k.quant_mxfp4(rnd(dev, N, K, seed=N, scale=K ** -0.5))
    A, B = unpack(k, *a).double(), unpack(k, *b).double()
    for out in (BF, F32):
        y = k.linear_mxfp4(*a, *b, out_dtype=out)
        assert ((y.double() - A @ B.t()).abs() <= product_bound(A, B, K, out)).all()
    if dev == "cuda":
        assert native().gemm_mxfp4_last_error() == 0


@pytest.mark.parametrize("dev", LANES)
def test_product_reads_every_scale_where_it_belongs(dev):
    """One row and one block at a time carries a scale of its own; exact in fp32."""
    k = lane(dev)
    M, N, K = 260, 300, 640
    x, w = torch.zeros(M, K), torch.zeros(N, K)
    for r in range(M):
        x[r, (37 * r) % K] = 2.0 ** ((r % 41) - 20)
    for n in range(N):
        w[n, (13 * n) % K] = 2.0 ** ((n % 29) - 14)
        w[n, (37 * n) % K] = -1.5 * 2.0 ** (n % 7)
    a, b = k.quant_mxfp4(x.to(dev)), k.quant_mxfp4(w.to(dev))
    want = unpack(k, *a).cpu().double() @ unpack(k, *b).cpu().double().t()
    assert torch.equal(k.linear_mxfp4(*a, *b, out_dtype=F32).cpu().double(), want)


@pytest.mark.parametrize("dev", LANES)
def test_product_out_add_and_strides(dev):
    k = lane(dev)
    M, N, K = 150, 96, 64
    a, b = k.quant_mxfp4(rnd(dev, M, K)), k.quant_mxfp4(rnd(dev, N, K, seed=1))
    bias = rnd(dev, N, seed=9)
    for dt in (BF, F32):
        base = k.linear_mxfp4(*a, *b, out_dtype=dt)
        add = rnd(dev, M, N, seed=4, dtype=dt)
        want = k.linear_mxfp4(*a, *b, add=add, bias=bias, out_dtype=dt)
        for off in (0, 8, 5):                                   # column ranges of a wider buffer, aligned and not
            buf = torch.full((M, 3 * N), 7.0, dtype=dt, device=dev)
            out = buf[:, off:off + N]
            assert k.linear_mxfp4(*a, *b, out=out) is out and torch.equal(out, base)
            rest = torch.cat([buf[:, :off], buf[:, off + N:]], 1)
            assert (rest == 7).all()                            # neighbours untouched
            side = torch.zeros(M, 3 * N, dtype=dt, device=dev)
            side[:, off:off + N] = add
            assert torch.equal(k.linear_mxfp4(*a, *b, add=side[:, off:off + N], bias=bias, out_dtype=dt), want)
        acc = add.clone()
        assert torch.equal(k.linear_mxfp4(*a, *b, out=acc, add=acc, bias=bias), want)              # accumulate in place
        wide = torch.cat([torch.zeros_like(add), add], 1)
        out, src = wide[:, :N], wide[:, N:]
        assert torch.equal(k.linear_mxfp4(*a, *b, out=out, add=src, bias=bias), want) and torch.equal(src, add)


@pytest.mark.parametrize("dev", LANES)
def test_product_propagates_nan_of_its_own_rows_only(dev):
    k = lane(dev)
    x, w = rnd(dev, 140, 320), rnd(dev, 136, 320, seed=2)
    x[5, 300] = float("nan")
    w[130, 0] = float("inf")
    y = k.linear_mxfp4(*k.quant_mxfp4(x), *k.quant_mxfp4(w))
    bad = torch.isnan(y)
    want = torch.zeros_like(bad)
    want[5], want[:, 130] = True, True
    assert torch.equal(bad, want)


@pytest.mark.parametrize("dev", LANES)
@pytest.mark.parametrize("M,K,N", [(1, 32, 8), (100, 256, 72), (129, 320, 40), (64, 96, 33)])
def test_linear_fwd(dev, M, K, N):
    k = lane(dev)
    x, w, add = rnd(dev, M, K), rnd(dev, K, N, seed=1, scale=0.1), rnd(dev, M, N, seed=2)
    A, B = mx_ref(x)[0], mx_ref(w.t())[0]
    y = k.linear_fwd_mxfp4(x, w, add=add)
    want = A @ B.t() + add.double()
    bound = product_bound(A, B, K, BF) + 2 * U * add.double().abs() + half_step(BF) * want.abs()
    assert y.dtype == BF and ((y.double() - want).abs() <= bound).all()
    out = torch.empty(M, N, dtype=F32, device=dev)
    assert k.linear_fwd_mxfp4(x, w, out=out) is out and ((out.double() - A @ B.t()).abs() <= product_bound(A, B, K, F32)).all()


# ------------------------------------------------------------------ the norm
@pytest.mark.parametrize("dev", LANES)
@pytest.mark.parametrize("res", [False, True], ids=["plain", "residual"])
@pytest.mark.parametrize("rows,cols", [(1, 32), (1, 4096), (5, 1024), (130, 96), (33, 2080), (3, 8192), (2, 16416), (1, 40032), (300, 352)])
def test_norm(dev, res, rows, cols):
    """Statistics: a sum of `cols` squares in fp32 is off by at most cols u, its root by half of that; y takes three more
    roundings.  Codes: half a step of the code's binade beyond y's own error."""
    k = lane(dev)
    x = rnd(dev, rows, cols, seed=rows + cols, dtype=F32) * torch.exp(rnd(dev, rows, 1, seed=3, dtype=F32))
    x = x.to(BF)
    r = rnd(dev, rows, cols, seed=7) if res else None
    w = (1 + 0.2 * rnd(dev, cols, seed=8, dtype=F32)).to(BF)
    eps = 1e-5
    h64 = (x.float() + r.float()).to(BF).double() if res else x.double()
    rstd64 = 1 / torch.sqrt(h64.square().mean(-1) + eps)
    y64 = h64 * rstd64[:, None] * w.double()
    tol = (cols / 2 + 8) * U
    q, s, h, rstd = k.rmsnorm_fp8(x, w, eps, residual=r)
    assert q.dtype == F8 and q.shape == x.shape and s.shape == (rows,) and rstd.shape == (rows,)
    assert torch.equal(h.double(), h64) and (res or h is x or h.data_ptr() == x.data_ptr())
    assert ((rstd.double() - rstd64).abs() <= tol * rstd64).all()
    assert ((s.double() - y64.abs().amax(-1) / 448).abs() <= (tol + 4 * U) * s.double()).all()
    a = (y64 / s.double()[:, None]).abs()
    step = torch.ldexp(torch.ones_like(a), torch.frexp((a * (1 + 2 * tol)).clamp(min=2.0 ** -6))[1] - 4)
    assert ((q.double().abs() - a).abs() <= step / 2 + a * (tol + 4 * U)).all() and q.double().abs().max() == 448
    # the 4-bit output: the same y, the same h and statistics
    q4, s4, h4, rstd4 = k.rmsnorm_mxfp4(x, w, eps, residual=r)
    assert torch.equal(h4, h) and torch.equal(rstd4, rstd)
    v = unpack(k, q4, s4).double()
    X = pow2(E.mxfp4_scale_rows(s4, rows, cols)).repeat_interleave(32, 1)
    amax = y64.abs().reshape(rows, -1, 32).amax(-1).repeat_interleave(32, 1)
    # amax / X is in [4, 8) but for y's own error
    assert (amax / X >= 4 * (1 - tol)).all() and (amax / X <= 8 * (1 + tol)).all()
    b = (y64 / X).abs().clamp(max=6)
    step = torch.where(b * (1 + tol) < 2, 0.5, torch.where(b * (1 + tol) < 4, 1.0, 2.0))
    assert ((v / X).abs() - b).abs().le(step / 2 + b * tol + 1e-30).all()
    # given statistics: the same codes again
    q2, s2, _, rstd2 = k.rmsnorm_fp8(h, w, eps, rstd=rstd)
    assert torch.equal(q2.view(U8), q.view(U8)) and torch.equal(s2, s) and torch.equal(rstd2, rstd)
    q3, s3, _, _ = k.rmsnorm_mxfp4(h, w, eps, rstd=rstd)
    assert torch.equal(q3, q4) and torch.equal(s3, s4)


@pytest.mark.parametrize("dev", LANES)
def test_norm_layouts_and_edges(dev):
    k = lane(dev)
    w = (1 + 0.1 * rnd(dev, 64, seed=1, dtype=F32)).to(BF)
    wide = rnd(dev, 20, 200, seed=2)
    x, r = wide[:, 8:72], wide[:, 80:144]
    want = k.rmsnorm_fp8(x.contiguous(), w, residual=r.contiguous())
    got = k.rmsnorm_fp8(x, w, residual=r)
    for a, b in zip(want, got):
        assert torch.equal(a.view(U8), b.contiguous().view(U8))
    # rows that start on 32 bytes, on 16 only, and widths that are not 16s: the same numbers
    for cols, off in ((320, 8), (320, 16), (2080, 8), (4128, 8), (8224, 8), (16416, 8), (328, 0), (1032, 8), (2056, 0)):
        big = rnd(dev, 3, cols + 64, seed=cols)
        gain = (1 + 0.1 * rnd(dev, cols + 8, seed=3, dtype=F32)).to(BF)
        xv, rv, gv = big[:, off:off + cols], big[:, 48:48 + cols], gain[:cols]
        for fn in (k.rmsnorm_fp8, k.rmsnorm_mxfp4) if cols % 32 == 0 else (k.rmsnorm_fp8,):
            for g_, w_ in zip(fn(xv, gv, residual=rv), fn(xv.contiguous(), gv.clone(), residual=rv.contiguous())):
                if g_.dtype == F32:               # the threads of a row differ between the forms, and with them the sum's order
                    assert ((g_ - w_).abs() <= (cols + 8) * U * w_.abs()).all()
                elif g_.dtype == BF:
                    assert torch.equal(g_, w_)
                else:
                    assert (g_.contiguous().view(U8) != w_.view(U8)).double().mean() < 1e-2
    # the sum may replace the residual stream in place, as a view of a wider buffer
    buf = wide.clone()
    q, s, h, rstd = k.rmsnorm_fp8(x, w, residual=buf[:, 80:144], h_out=buf[:, 80:144])
    assert torch.equal(h, want[2]) and torch.equal(buf[:, 80:144], want[2]) and torch.equal(buf[:, 144:], wide[:, 144:])
    assert torch.equal(buf[:, :80], wide[:, :80]) and torch.equal(q.view(U8), want[0].view(U8))
    # leading axes
    x3 = rnd(dev, 2, 5, 64, seed=4)
    q, s, h, rstd = k.rmsnorm_fp8(x3, w)
    assert q.shape == x3.shape and s.shape == (10,) and rstd.shape == (10,)
    q, s, h, rstd = k.rmsnorm_mxfp4(x3, w)
    assert q.shape == (10, 32)
    # a row of zeros: codes zero, scale 1 (8 bits) or the smallest (4 bits); NaN and infinities stay in their row
    x = rnd(dev, 4, 64, seed=5)
    x[1], x[2, 3] = 0, float("nan")
    q, s, _, _ = k.rmsnorm_fp8(x, w)
    assert s[1] == 1 and (q[1].float() == 0).all() and torch.isnan(q[2].float()).all() and q[3].float().isfinite().all()
    v = unpack(k, *k.rmsnorm_mxfp4(x, w)[:2])
    assert (v[1] == 0).all() and torch.isnan(v[2]).all() and v[0].isfinite().all() and v[3].isfinite().all()
    # sums of subnormal numbers are sums, and zeros keep their sign's rules
    a = torch.tensor([1e-39, -1e-39, 3e-39, -0.0, 0.0, -0.0, 2e-38, 1.0] * 8).to(BF).to(dev).view(1, 64)
    b = torch.tensor([1e-39, 5e-40, -3e-39, -0.0, -0.0, 0.0, -1.9e-38, 2.0 ** -9] * 8).to(BF).to(dev).view(1, 64)
    h = k.rmsnorm_fp8(a, w, residual=b)[2]
    assert torch.equal(h.view(torch.int16), (a.float().cpu() + b.float().cpu()).to(BF).to(dev).view(torch.int16))
    # a gain so small that 448 steps of it leave the normal numbers
    tiny = torch.full((64,), 2.0 ** -126, dtype=BF, device=dev)
    q, s, _, _ = k.rmsnorm_fp8(x[:1], tiny)
    assert s[0] == 2.0 ** -120 and q.float().isfinite().all()


# ------------------------------------------------------------------ AdamW
FORMS = ["bf16", "fp32", "master", "split"]


def opt_state(dev, sizes, form, gdt, bits, seed=0, offset=0):
    """Tensors of the given sizes; ``offset`` shifts every start off its alignment."""
    g = torch.Generator().manual_seed(seed)

    def make(n, dt, scale=1.0, positive=False):
        t = torch.randn(n + offset, generator=g) * scale
        t = t.abs() if positive else t
        return t.to(dt).to(dev)[offset:]
    st = {"ws": [], "gs": [], "ms": [], "vs": []}
    for n in sizes:
        w = make(n, F32, 0.05)
        if form == "fp32":
            st["ws"].append(w)
        elif form == "split":
            hi, lo = E.split_master_cut(w.cpu())
            pad = lambda t: torch.cat([torch.zeros(offset, dtype=t.dtype), t]).to(dev)[offset:]
            st["ws"].append(pad(hi))
            st.setdefault("los", []).append(pad(lo))
        else:
            st["ws"].append(make(0, BF) if not n else torch.cat([torch.zeros(offset, dtype=BF, device=dev), w.to(BF)])[offset:])
            if form == "master":
                st.setdefault("masters", []).append(w)
        st["gs"].append(make(n, gdt, 1e-2))
        m, r = make(n, F32, 5e-3), make(n, F32, 1e-2, positive=True)
        if bits == 8:
            for name, t in (("m", m), ("v", r)):
                nb = -(-n // 128)
                pad = torch.nn.functional.pad(t.abs(), (0, -n % 128)).view(-1, 128)
                s = (pad.amax(-1) / 448).clamp(min=2.0 ** -120) if n else torch.empty(0, device=dev)
                q = (t / s.repeat_interleave(128)[:n]).clamp(-448, 448).to(F8)
                st[name + "s"].append(torch.cat([torch.zeros(offset, device=dev).to(F8).view(U8), q.view(U8)]).view(F8)[offset:])
                st.setdefault(name + "_scales", []).append(s)
        else:
            st["ms"].append(m)
            st["vs"].append(r * r)
    return st


def clone(st):
    return {k: [t.clone() for t in v] for k, v in st.items()}


def adam_ref(st, i, lr, b1, b2, eps, wd, step, gscale=1.0):
    """(m', r' or v', w') in 64 bits."""
    g = st["gs"][i].double() * gscale
    n = g.numel()
    if "m_scales" in st:
        up = lambda s: s.double().repeat_interleave(128)[:n]
        m, v = st["ms"][i].double() * up(st["m_scales"][i]), (st["vs"][i].double() * up(st["v_scales"][i])).square()
    else:
        m, v = st["ms"][i].double(), st["vs"][i].double()
    m, v = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
    w = st["masters"][i].double() if "masters" in st else E.split_master_join(st["ws"][i], st["los"][i]).double() if "los" in st else st["ws"][i].double()
    upd = lr * ((m / (1 - b1 ** step)) / (torch.sqrt(v / (1 - b2 ** step)) + eps) + wd * w)
    return m, v, w, w - upd


def dither_ref(y, rnd16):
    """Codes of y = t / scale by the definition: the grid point below y / step + random part."""
    a = y.abs()
    step = torch.ldexp(torch.ones_like(a), torch.frexp(a.clamp(min=2.0 ** -6))[1] - 4)
    pos = a / step + rnd16.double() / 65536
    return torch.floor(pos) * step, (pos - torch.round(pos)).abs(), step


@pytest.mark.parametrize("dev", LANES)
@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("gdt", [BF, F32], ids=["gbf16", "gfp32"])
@pytest.mark.parametrize("offset", [0, 1, 8, 16], ids=["aligned", "odd", "by8", "by16"])
def test_adamw(dev, bits, form, gdt, offset):
    k = lane(dev)
    sizes = [1, 127, 128, 129, 0, 4096, 4097, 10000, 33]
    wds = [0.1 * (i % 2) for i in range(len(sizes))]
    st = opt_state(dev, sizes, form, gdt, bits, seed=bits, offset=offset)
    old = clone(st)
    lr, b1, b2, eps, step, gs = 1e-2, 0.9, 0.95, 1e-8, 3, 0.5
    ws = k.adamw_multi_step(st["ws"], st["gs"], st["ms"], st["vs"], lr, b1, b2, eps, wds, step, gscale=gs,
                            **{n: st[n] for n in ("masters", "los", "m_scales", "v_scales") if n in st})
    assert ws is st["ws"]
    for i, n in enumerate(sizes):
        if not n:
            continue
        m, v, w0, w1 = adam_ref(old, i, lr, b1, b2, eps, wds[i], step, gs)
        if bits == 32:
            # four roundings each, relative to the terms' magnitudes
            mb = 4 * U * (b1 * old["ms"][i].double().abs() + (1 - b1) * gs * old["gs"][i].double().abs())
            assert ((st["ms"][i].double() - m).abs() <= mb).all() and ((st["vs"][i].double() - v).abs() <= 6 * U * v).all()
        else:
            lo16, hi16 = E.state_dither(n, step, dev)
            for name, t, rnd16, floor in (("m", m, lo16, 0.0), ("v", torch.sqrt(v), hi16, 2.0 ** -9)):
                amax = torch.nn.functional.pad(t.abs(), (0, -n % 128)).view(-1, 128).amax(-1)
                s = st[name + "_scales"][i]
                assert ((s.double() - amax / 448).abs() <= 16 * U * s.double() + 2.0 ** -120).all()
                y = t / s.double().repeat_interleave(128)[:n]
                want, dist, grid = dither_ref(y, rnd16)
                want = torch.where(y.abs() > 0, want.clamp(min=floor, max=448), want)
                got = st[name + "s"][i].double().abs()
                # y carries at most 16 roundings (cancellation in m: relative to its terms); in units of the grid y is at most 16
                terms = (b1 * old["ms"][i].double().abs() * old["m_scales"][i].double().repeat_interleave(128)[:n] + gs * old["gs"][i].double().abs()) if name == "m" else t.abs()
                err = 16 * U * terms / s.double().repeat_interleave(128)[:n] / grid
                sure = dist > err
                # an element may sit within err of a border by chance; a block's largest does whenever its random part is near 0 or 1
                assert int((~sure).sum()) <= 2 + n // 100 and torch.equal(got[sure], want[sure])
                assert ((got - want).abs() <= grid * (1 + 1e-6)).all()
                assert (got[t.abs() > 0] >= floor).all()
        upd_err = lr * 64 * U * ((m.abs() + gs * old["gs"][i].double().abs()) / (1 - b1 ** step)) / (torch.sqrt(v / (1 - b2 ** step)) + eps) + 8 * U * w0.abs()
        got = st["ws"][i].double()
        if form == "master":
            assert ((st["masters"][i].double() - w1).abs() <= upd_err).all()
        if form == "split":
            full = E.split_master_join(st["ws"][i], st["los"][i])
            assert ((full.double() - w1).abs() <= upd_err).all()
            hi, lo = E.split_master_cut(full)
            assert torch.equal(hi.view(torch.int16), st["ws"][i].view(torch.int16)) and torch.equal(lo, st["los"][i])
        if form == "fp32":
            assert ((got - w1).abs() <= upd_err).all()
        else:
            assert ((got - w1).abs() <= upd_err + half_step(BF) * w1.abs() * (1 + 1e-6) + 1e-40).all()
        assert torch.equal(st["gs"][i], old["gs"][i])


@pytest.mark.parametrize("dev", LANES)
def test_adamw_result_of_a_tensor_does_not_depend_on_the_list(dev):
    k = lane(dev)
    sizes = [300 + 17 * i for i in range(600)]                  # more than one launch's table
    st = opt_state(dev, sizes, "bf16", BF, 8, seed=4)
    one = clone(st)
    args = (1e-3, 0.9, 0.95, 1e-8, 0.1, 5)
    k.adamw_multi_step(st["ws"], st["gs"], st["ms"], st["vs"], *args, m_scales=st["m_scales"], v_scales=st["v_scales"])
    for i in (0, 1, 255, 256, 257, 511, 512, 599):
        k.adamw_multi_step(*[[one[n][i]] for n in ("ws", "gs", "ms", "vs")], *args, m_scales=[one["m_scales"][i]], v_scales=[one["v_scales"][i]])
        for n in st:
            assert torch.equal(st[n][i].view(U8), one[n][i].view(U8)), (i, n)


@pytest.mark.parametrize("dev", LANES)
def test_adamw_8bit_moments_fall_and_follow(dev):
    """A second moment under a gradient that shrank a hundredfold follows it down, at the rate the mathematics gives: rounding
    to nearest would hold it where it is.  500 steps at beta2 = 0.99: v falls by 0.99^500 = 0.0066 towards 1e-4 of its start."""
    k = lane(dev)
    n = 4096
    g = torch.Generator().manual_seed(1)
    grad = (torch.randn(n, generator=g) * 1e-4).to(dev)
    w = torch.zeros(n, device=dev)
    m, v = torch.zeros(n, device=dev).to(F8), torch.full((n,), 448.0, device=dev).to(F8)
    ms, vs = torch.full((32,), 2.0 ** -120, device=dev), torch.full((32,), 1e-2 / 448, device=dev)
    # every 128th element keeps the large gradient, so that the block's scale does not fall for the others
    grad[::128] = 1e-2
    for step in range(1, 501):
        k.adamw_multi_step([w], [grad], [m], [v], 0.0, 0.9, 0.99, 1e-8, 0.0, step, m_scales=[ms], v_scales=[vs])
    got = (v.float() * vs.repeat_interleave(128)).square()
    want = 1e-4 * 0.99 ** 500 + (1 - 0.99 ** 500) * grad.square()
    rest = torch.ones(n, dtype=torch.bool, device=dev)
    rest[::128] = False
    assert abs(float(got[rest].mean() / want[rest].mean()) - 1) < 0.25          # 4000 elements, each within one code of its value
    assert abs(float(got[~rest].mean() / want[~rest].mean()) - 1) < 0.25


@pytest.mark.parametrize("dev", LANES)
def test_adamw_nan_and_zero_gradients(dev):
    k = lane(dev)
    st = opt_state(dev, [300], "master", F32, 8, seed=9)
    st["gs"][0][5] = float("nan")
    st["gs"][0][130:] = 0
    for n in ("ms", "vs"):
        st[n][0][130:] = torch.zeros(170, device=dev).to(F8)
    k.adamw_multi_step(st["ws"], st["gs"], st["ms"], st["vs"], 1e-3, step=1, masters=st["masters"], m_scales=st["m_scales"], v_scales=st["v_scales"])
    w = st["masters"][0]
    assert torch.isnan(w[5]) and torch.isnan(st["ms"][0][5].float()) and w[:5].isfinite().all() and w[6:].isfinite().all()
    assert (st["ms"][0][130:].float() == 0).all() and (st["vs"][0][130:].float() == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("form", FORMS)
def test_adamw_kernel_and_plain_lane_agree_to_the_bit_in_8_bit_state(form):
    """The arithmetic in front of the rounding is the same sequence of rounded fp32 operations in both lanes."""
    sizes = [70000, 129, 4096]
    st = opt_state("cuda", sizes, form, BF, 8, seed=11)
    ref = clone(st)
    for s, K in ((st, lane("cuda")), (ref, resolve_kernels(kernel_set="eager").lowbit)):
        for step in (1, 2, 3):
            K.adamw_multi_step(s["ws"], s["gs"], s["ms"], s["vs"], 1e-3, wds=0.1, step=step,
                               **{n: s[n] for n in ("masters", "los", "m_scales", "v_scales") if n in s})
    for n in ("ms", "vs", "m_scales", "v_scales"):
        for a, b in zip(st[n], ref[n]):
            assert torch.equal(a.view(U8), b.view(U8)), n


# ------------------------------------------------------------------ refusals: the plain lane, and the extension on host tensors
def refusals():
    x, w = torch.zeros(4, 64, dtype=BF), torch.zeros(64, dtype=BF)
    q, s = E.quant_mxfp4(x)
    buf = torch.zeros(8, 64, dtype=BF)
    yield "no matrix", lambda K: K.quant_mxfp4(torch.zeros(64, dtype=BF))
    yield "half", lambda K: K.quant_mxfp4(x.half())
    yield "K not 32s", lambda K: K.quant_mxfp4(torch.zeros(4, 48, dtype=BF))
    yield "K not 32s, transposed", lambda K: K.quant_mxfp4(torch.zeros(48, 4, dtype=BF), transpose=True)
    yield "K zero", lambda K: K.quant_mxfp4(torch.zeros(4, 0, dtype=BF))
    yield "columns strided", lambda K: K.quant_mxfp4(torch.zeros(64, 64, dtype=BF).t())
    yield "codes dtype", lambda K: K.dequant_mxfp4(q.to(torch.int32), s)
    yield "scales shape", lambda K: K.dequant_mxfp4(q, s[:, :1].contiguous())
    yield "values dtype", lambda K: K.dequant_mxfp4(q, s, torch.float16)
    yield "different K", lambda K: K.linear_mxfp4(q, s, *E.quant_mxfp4(torch.zeros(4, 96, dtype=BF)))
    yield "result dtype", lambda K: K.linear_mxfp4(q, s, q, s, out_dtype=torch.float16)
    yield "out shape", lambda K: K.linear_mxfp4(q, s, q, s, out=torch.zeros(4, 5, dtype=BF))
    yield "out columns strided", lambda K: K.linear_mxfp4(q, s, q, s, out=torch.zeros(4, 4, dtype=BF).t())
    yield "add dtype", lambda K: K.linear_mxfp4(q, s, q, s, add=torch.zeros(4, 4))
    yield "bias shape", lambda K: K.linear_mxfp4(q, s, q, s, bias=torch.zeros(5, dtype=BF))
    yield "scales of the other operand", lambda K: K.linear_mxfp4(q, s, *[E.quant_mxfp4(torch.zeros(200, 64, dtype=BF))[0], s])
    yield "width not 8s", lambda K: K.rmsnorm_fp8(torch.zeros(4, 20, dtype=BF), torch.zeros(20, dtype=BF))
    yield "width not 32s", lambda K: K.rmsnorm_mxfp4(torch.zeros(4, 48, dtype=BF), torch.zeros(48, dtype=BF))
    yield "gain length", lambda K: K.rmsnorm_fp8(x, torch.zeros(32, dtype=BF))
    yield "residual shape", lambda K: K.rmsnorm_fp8(x, w, residual=torch.zeros(3, 64, dtype=BF))
    yield "h_out alone", lambda K: K.rmsnorm_fp8(x, w, h_out=torch.zeros_like(x))
    yield "rstd length", lambda K: K.rmsnorm_fp8(x, w, rstd=torch.zeros(3))
    f, i16, c = lambda n=128: [torch.zeros(n)], [torch.zeros(128, dtype=torch.int16)], [torch.zeros(128).to(F8)]
    b = [torch.zeros(128, dtype=BF)]
    yield "list lengths", lambda K: K.adamw_multi_step(b, b + b, f(), f(), 1e-3)
    yield "decay list", lambda K: K.adamw_multi_step(b, f(), f(), f(), 1e-3, wds=[0.1, 0.1])
    yield "element counts", lambda K: K.adamw_multi_step(b, f(), f(64), f(), 1e-3)
    yield "step zero", lambda K: K.adamw_multi_step(b, f(), f(), f(), 1e-3, step=0)
    yield "bf16 moments", lambda K: K.adamw_multi_step(f(), f(), [b[0].clone()], [b[0].clone()], 1e-3)
    yield "mixed moments", lambda K: K.adamw_multi_step(b, f(), c, f(), 1e-3, m_scales=f(1), v_scales=f(1))
    yield "8 bits without scales", lambda K: K.adamw_multi_step(b, f(), c, [c[0].clone()], 1e-3)
    yield "scale count", lambda K: K.adamw_multi_step(b, f(), c, [c[0].clone()], 1e-3, m_scales=f(2), v_scales=f(1))
    yield "scales without 8 bits", lambda K: K.adamw_multi_step(b, f(), f(), f(), 1e-3, m_scales=f(1), v_scales=f(1))
    yield "master and split", lambda K: K.adamw_multi_step(b, f(), f(), f(), 1e-3, masters=f(), los=i16)
    yield "master of fp32 weights", lambda K: K.adamw_multi_step(f(), f(), f(), f(), 1e-3, masters=f())
    yield "los dtype", lambda K: K.adamw_multi_step(b, f(), f(), f(), 1e-3, los=f())
    yield "strided weight", lambda K: K.adamw_multi_step([torch.zeros(256, dtype=BF)[::2]], f(), f(), f(), 1e-3)
    t = torch.zeros(128)
    yield "the same tensor twice", lambda K: K.adamw_multi_step([t, t], f() + f(), f() + f(), f() + f(), 1e-3)
    yield "moment over moment", lambda K: K.adamw_multi_step(b, f(), [t], [t], 1e-3)
    yield "gradient over weight", lambda K: K.adamw_multi_step([t], [t], f(), f(), 1e-3)


REFUSALS = dict(refusals())


@pytest.mark.parametrize("name", REFUSALS)
def test_refusals_plain_lane(name):
    with pytest.raises(ValueError):
        REFUSALS[name](resolve_kernels(kernel_set="eager").lowbit)


@pytest.mark.parametrize("name", REFUSALS)
def test_refusals_of_the_extension_come_before_the_device(name):
    """Host tensors: the argument itself is refused, with its own message, not the place it lives in."""
    if not native_available():
        pytest.skip("extension not built")
    from dataflow_b200.ops import lowbit
    with pytest.raises(ValueError) as e:
        REFUSALS[name](lowbit)
    assert "must be CUDA tensors" not in str(e.value)


def test_extension_refuses_host_tensors_and_overlaps():
    if not native_available():
        pytest.skip("extension not built")
    from dataflow_b200.ops import lowbit as K
    x, w = torch.zeros(4, 64, dtype=BF), torch.zeros(64, dtype=BF)
    q, s = E.quant_mxfp4(x)
    f = lambda: [torch.zeros(128)]
    for call in (lambda: K.quant_mxfp4(x), lambda: K.dequant_mxfp4(q, s), lambda: K.linear_mxfp4(q, s, q, s), lambda: K.rmsnorm_fp8(x, w),
                 lambda: K.rmsnorm_mxfp4(x, w), lambda: K.adamw_multi_step(f(), f(), f(), f(), 1e-3)):
        with pytest.raises(ValueError, match="must be CUDA tensors"):
            call()
    buf = torch.zeros(16, 64, dtype=BF)
    with pytest.raises(ValueError, match="overlap"):
        K.rmsnorm_fp8(buf[:8], w, residual=buf[8:], h_out=buf[4:12])
    flat = torch.zeros(64, dtype=BF)
    with pytest.raises(ValueError, match="overlap"):
        K.linear_mxfp4(q, s, q, s, out=flat[:16].view(4, 4), add=flat[4:20].view(4, 4))
    with pytest.raises(ValueError, match="overlaps an operand"):
        K.linear_mxfp4(q, s, q, s, out=q.view(-1)[:32].view(BF).view(4, 4))
    big = torch.zeros(256)
    with pytest.raises(ValueError, match="twice or overlaps"):
        K.adamw_multi_step([big[:128]], f(), [big[100:228]], f(), 1e-3)
    with pytest.raises(ValueError, match="16-byte aligned"):
        K.rmsnorm_fp8(torch.zeros(300, dtype=BF)[1:257].view(4, 64), w)


# ------------------------------------------------------------------ through the framework's own paths
@pytest.mark.parametrize("dev", LANES)
@pytest.mark.parametrize("n,k,m", [(48, 64, 32), (33, 96, 40), (5, 32, 7)])
def test_linear_form_and_its_gradients(dev, n, k, m):
    """Forward on the rounded operands; the backward is that of the plain product (straight through), checked against the
    formula and, for the rounded operands held fixed, against differences of the forward."""
    from dataflow_b200.models import _forms as F
    dt = BF if dev == "cuda" else F32
    x = rnd(dev, n, k, seed=1, dtype=dt).requires_grad_(True)
    w = rnd(dev, k, m, seed=2, scale=0.1, dtype=dt).requires_grad_(True)
    y = F.linear(x, w, "mxfp4")
    A, B = mx_ref(x.detach())[0], mx_ref(w.detach().t())[0]
    assert y.dtype == dt and ((y.detach().double() - A @ B.t()).abs() <= product_bound(A, B, k, dt)).all()
    dy = rnd(dev, n, m, seed=3, dtype=dt)
    dx, dw = torch.autograd.grad(y, [x, w], dy)
    wx, ww = dy.double() @ w.detach().double().t(), x.detach().double().t() @ dy.double()
    ax, aw = dy.double().abs() @ w.detach().double().abs().t(), x.detach().double().abs().t() @ dy.double().abs()
    assert ((dx.double() - wx).abs() <= (m + 2) * 2.0 ** -23 * ax + half_step(dt) * wx.abs() + 1e-30).all()
    assert ((dw.double() - ww).abs() <= (n + 2) * 2.0 ** -23 * aw + half_step(dt) * ww.abs() + 1e-30).all()
    # differences: <dy, f(x + t v) - f(x - t v)> / 2t of the product the gradient belongs to (linear: exact for any t)
    v = rnd(dev, n, k, seed=4, dtype=F64)
    f = lambda xx: (dy.double() * (xx @ w.detach().double())).sum()
    diff = (f(x.detach().double() + v) - f(x.detach().double() - v)) / 2
    assert abs(float(diff - (dx.double() * v).sum())) <= float((half_step(dt) * wx.abs() * v.abs() + (m + 2) * 2.0 ** -23 * ax * v.abs()).sum()) + 1e-9 * float(diff.abs())
    # only what is asked for
    y = F.linear(x.detach(), w, "mxfp4")
    assert torch.equal(torch.autograd.grad(y, w, dy)[0], dw)
    # a contraction the format does not take falls back to the plain product
    assert F.linear(x.detach()[:, :20], w.detach()[:20], "mxfp4").shape == (n, m)


@pytest.mark.parametrize("dev", LANES)
def test_a_training_step_in_narrow_formats(dev):
    """The operators in the order a step uses them: norm with the residual -> 4-bit product -> loss gradient -> norm backward,
    and AdamW with 8-bit moments on gain and weight; against the same step in 64 bits on the same rounded operands."""
    Kall = resolve_kernels(kernel_set="eager" if dev == "cpu" else None)
    K = Kall.lowbit
    n, d, m = 96, 128, 64
    x, res, gain, w = rnd(dev, n, d, seed=1), rnd(dev, n, d, seed=2), (1 + 0.1 * rnd(dev, d, seed=3, dtype=F32)).to(BF), rnd(dev, d, m, seed=4, scale=0.1)
    dy = rnd(dev, n, m, seed=5, scale=0.1)
    q, s, h, rstd = K.rmsnorm_mxfp4(x, gain, 1e-5, residual=res)
    wq, ws = K.quant_mxfp4(w, transpose=True)
    y = K.linear_mxfp4(q, s, wq, ws)
    A, B = unpack(K, q, s).double(), unpack(K, wq, ws).double()
    assert ((y.double() - A @ B.t()).abs() <= product_bound(A, B, d, BF)).all()
    hn = Kall.rmsnorm_apply(h, gain, rstd)
    dw = torch.zeros_like(w)
    Kall.linear_wgrad_bf16(hn, dy, dw)
    dhn = Kall.linear_dgrad_bf16(dy, w)
    dgain = torch.zeros_like(gain)
    dx = Kall.rmsnorm_bwd(dhn, h, gain, rstd, dw=dgain)
    h64 = h.double().requires_grad_(True)
    g64, w64 = gain.double().requires_grad_(True), w.double().requires_grad_(True)
    y64 = (h64 / torch.sqrt(h64.square().mean(-1, keepdim=True) + 1e-5) * g64) @ w64
    grads = torch.autograd.grad(y64, [h64, g64, w64], dy.double())
    for got, want in zip((dx, dgain, dw), grads):
        # three bf16 roundings on the way (normalised rows or dhn, the product, the result), as a root mean square
        assert float((got.double() - want).norm() / want.norm()) < 3 * half_step(BF)
    opt = opt_state(dev, [gain.numel(), w.numel()], "bf16", BF, 8, seed=1)
    old = clone({"ws": [gain, w.view(-1)], "gs": [dgain, dw.view(-1)], **{n: opt[n] for n in ("ms", "vs", "m_scales", "v_scales")}})
    K.adamw_multi_step([gain, w], [dgain, dw], opt["ms"], opt["vs"], 1e-3, wds=[0.0, 0.1], step=1, m_scales=opt["m_scales"], v_scales=opt["v_scales"])
    assert not torch.equal(w.view(-1), old["ws"][1])
    for i, (t, wd) in enumerate(((gain, 0.0), (w.view(-1), 0.1))):
        # a gain near 1 moves by less than half a bf16 step here: the bound, not a change, is what the definition asks for
        _, _, w0, w1 = adam_ref(old, i, 1e-3, 0.9, 0.95, 1e-8, wd, 1)
        assert ((t.double() - w1).abs() <= half_step(BF) * w1.abs() * (1 + 1e-6) + 64 * U * ((w1 - w0).abs() + w0.abs())).all()


def _trainer_losses(dev, steps=3, hyper=None, lower=None, budget=None, family="llama3", **over):
    import dataclasses
    from dataflow_b200.models.families import resolve_family
    from dataflow_b200.run.driver import Trainer, synthetic_rounds
    cfg = dataclasses.replace(resolve_family(family).presets["tiny"](), **over)
    tr = Trainer(family, cfg, budget_gib=budget, device=None if dev == "cpu" else 0, hyper={"lr": 3e-3, **(hyper or {})}, seed=3,
                 **({"lower_kwargs": lower} if lower else {}))
    out = [tr.step(synthetic_rounds(cfg, tr.rounds, tr.T, 64, 11, s)) for s in range(steps)]
    tr.close()
    return out


@pytest.mark.parametrize("dev", LANES)
@pytest.mark.parametrize("family", ["llama3", "qwen3", "olmoe"])
def test_llama_like_blocks_in_4_bits(dev, family):
    """Dense blocks, blocks with q / k norms, and a mixture-of-experts MLP behind 4-bit attention projections."""
    base, got = _trainer_losses(dev, family=family), _trainer_losses(dev, family=family, hyper={"linear_precision": "mxfp4"})
    assert base != got and all(math.isfinite(v) for v in got)
    for level in (1, 2):                                        # recomputed context comes from the same codes
        again = _trainer_losses(dev, family=family, hyper={"linear_precision": "mxfp4"}, lower={"recompute_levels": {0: level, 1: level}})
        assert again == got


def test_reference_form_family_in_4_bits():
    """The twin runs the same forms, so both quantise; the engine and the twin stay together."""
    from dataflow_b200.testing.family_gate import run_pair
    base = run_pair("dsv32", steps=3)["engine"]
    low = run_pair("dsv32", steps=3, overrides={"linear_precision": "mxfp4"})
    assert low["engine"] != base and low["max_loss_rel"] < 1e-3


@pytest.mark.parametrize("dev", LANES)
@pytest.mark.parametrize("policy", ["bf16_8bit", "bf16_split_master_8bit"])
def test_8bit_policies_run_and_shrink_the_state(dev, policy):
    import dataclasses
    from dataflow_b200.blocks.layouts import DTypePolicy
    from dataflow_b200.models.families import resolve_family
    fam = resolve_family("llama3")
    cfg = fam.presets["tiny"]()
    dims = fam.derive_dims(cfg)
    size = lambda p: fam.family_layouts(dims, DTypePolicy.named(p), "adamw").head_o.size_bytes
    wide = {"bf16_8bit": "bf16", "bf16_split_master_8bit": "bf16_split_master"}[policy]
    per = {"bf16_8bit": (2.0625, 4), "bf16_split_master_8bit": (4.0625, 6)}[policy]
    assert abs(size(policy) / size(wide) - per[0] / per[1]) < 0.01
    got = _trainer_losses(dev, dtype_policy=policy)
    ref = _trainer_losses(dev, dtype_policy=wide)
    assert got[0] == ref[0] and all(math.isfinite(v) for v in got)          # the same weights until the first update
    assert got == _trainer_losses(dev, dtype_policy=policy)                 # and reproducible


def test_refusals_of_the_policies():
    from dataflow_b200.blocks.layouts import DTypePolicy, Field, opt_state_layout
    f = [Field("w", (4, 4))]
    pol = DTypePolicy.named("bf16_8bit")
    names = opt_state_layout(f, pol).names()
    assert names == ["w.s0", "w.s0_scale", "w.s1", "w.s1_scale"]
    with pytest.raises(ValueError):
        opt_state_layout(f, pol, rule_of=lambda f: "muon")
    import dataclasses
    from dataflow_b200.models.families import resolve_family
    from dataflow_b200.parallel.zero import zero_lower_kwargs
    from dataflow_b200.run.driver import Trainer
    cfg = dataclasses.replace(resolve_family("llama3").presets["tiny"](), dtype_policy="bf16_8bit")
    with pytest.raises(ValueError, match="8-bit optimizer state"):
        Trainer("llama3", cfg, budget_gib=None, device=None, lower_kwargs=zero_lower_kwargs("fsdp", 0, 2), init=False)
    from dataflow_b200.run.recipe import Recipe
    assert Recipe(linear_precision="mxfp4").hyper()["linear_precision"] == "mxfp4"


# ------------------------------------------------------------------ streams, graphs, poisoned memory
@pytest.mark.gpu
def test_every_output_byte_is_written():
    K = lane("cuda")
    x, w = rnd("cuda", 133, 352), (1 + rnd("cuda", 352, seed=1, scale=0.1, dtype=F32)).to(BF)
    wt = rnd("cuda", 352, 77, seed=2)

    def calls():
        yield K.quant_mxfp4(x)
        yield K.quant_mxfp4(wt, transpose=True)
        yield (K.dequant_mxfp4(*K.quant_mxfp4(x)),)
        yield K.rmsnorm_fp8(x, w, residual=x)
        yield K.rmsnorm_mxfp4(x, w, residual=x)
        yield (K.linear_fwd_mxfp4(x, wt),)
        yield K.quant_mxfp4(x[:1, :32].contiguous())
        yield (K.linear_fwd_mxfp4(x[:1], wt[:, :1].contiguous()),)
    runs = []
    for byte in (0x5A, 0xC3):
        junk = [torch.full((n << 20,), byte, dtype=U8, device="cuda") for n in (512, 1, 1, 1, 1, 1, 1, 1, 1)]
        torch.cuda.synchronize()
        del junk
        runs.append([[t.contiguous().view(-1).view(U8).clone() for t in out] for out in calls()])
    for a, b in zip(*runs):
        for s, t in zip(a, b):
            assert torch.equal(s, t)


@pytest.mark.gpu
def test_another_stream_and_a_captured_graph():
    K = lane("cuda")
    x, w, wt = rnd("cuda", 200, 256), rnd("cuda", 256, seed=1), rnd("cuda", 256, 136, seed=2)
    want_n, want_y = K.rmsnorm_fp8(x, w), K.linear_fwd_mxfp4(x, wt)
    st = opt_state("cuda", [1000, 129], "bf16", BF, 8, seed=3)
    ref = clone(st)

    def adam(s):
        K.adamw_multi_step(s["ws"], s["gs"], s["ms"], s["vs"], 1e-3, step=2, m_scales=s["m_scales"], v_scales=s["v_scales"])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = K.rmsnorm_fp8(x, w)
        y = K.linear_fwd_mxfp4(x, wt)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got[0].view(U8), want_n[0].view(U8)) and torch.equal(y, want_y)
    graphs = []
    for _ in range(2):                                          # two graphs of the same work, replayed on two streams at once
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = (K.rmsnorm_fp8(x, w)[0], K.linear_fwd_mxfp4(x, wt), K.dequant_mxfp4(*K.rmsnorm_mxfp4(x, w)[:2]))
        graphs.append((g, out))
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(5):
        for stream, (g, _) in zip((a, b), graphs):
            with torch.cuda.stream(stream):
                g.replay()
    torch.cuda.synchronize()
    for _, out in graphs:
        assert torch.equal(out[0].view(U8), want_n[0].view(U8)) and torch.equal(out[1], want_y)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        adam(st)
    for _ in range(3):
        g.replay()
        adam(ref)
    torch.cuda.synchronize()
    for n in st:
        for s, t in zip(st[n], ref[n]):
            assert torch.equal(s.view(U8), t.view(U8))


@pytest.mark.gpu
def test_offsets_past_32_bits():
    """Matrices and a tensor of more than 2^31 elements: their last rows are what a call on those rows alone gives."""
    K = lane("cuda")
    g = torch.Generator(device="cuda").manual_seed(5)
    rows, cols = 262_200, 8224                                   # 2.16e9 elements
    x = torch.empty(rows, cols, dtype=BF, device="cuda")
    for i in range(0, rows, 65536):
        x[i:i + 65536] = torch.randn(min(65536, rows - i), cols, device="cuda", generator=g).to(BF)
    w = (1 + 0.1 * rnd("cuda", cols, seed=1, dtype=F32)).to(BF)
    tail = slice(rows - 77, rows)
    q, s, h, r = K.rmsnorm_fp8(x, w, residual=x)
    q1, s1, h1, r1 = K.rmsnorm_fp8(x[tail], w, residual=x[tail])
    assert torch.equal(q[tail].view(U8), q1.view(U8)) and torch.equal(s[tail], s1) and torch.equal(h[tail], h1) and torch.equal(r[tail], r1)
    del q, h
    for fn in (K.quant_mxfp4, lambda t: K.rmsnorm_mxfp4(t, w)[:2]):
        q, s = fn(x)
        q1, s1 = fn(x[tail])
        assert torch.equal(q[tail], q1) and torch.equal(K.dequant_mxfp4(q, s)[tail], K.dequant_mxfp4(q1, s1))
    del q, s
    xt = x.view(-1)[:8224 * 262_144].view(8224, 262_144)         # stored (K, rows)
    q, s = K.quant_mxfp4(xt, transpose=True)
    q1, s1 = K.quant_mxfp4(xt[:, -60:].contiguous(), transpose=True)
    assert torch.equal(q[-60:], q1)
    del q, s, xt, x
    a, b = K.quant_mxfp4(rnd("cuda", 46_400, 32)), K.quant_mxfp4(rnd("cuda", 46_400, 32, seed=1))
    y = K.linear_mxfp4(*a, *b)                                   # 2.15e9 results
    a1 = K.quant_mxfp4(K.dequant_mxfp4(*a)[-50:])
    assert torch.equal(y[-50:], K.linear_mxfp4(*a1, *b))
    del y
    n, k = 2 ** 31 + 1024 + 37, 1024 + 37
    for bits in (8, 32):
        ws, gs = torch.zeros(n, dtype=BF, device="cuda"), torch.zeros(n, dtype=BF, device="cuda")
        ws[-k:], gs[-k:] = rnd("cuda", k, seed=2), rnd("cuda", k, seed=3)
        mk = lambda c: torch.zeros(c, dtype=U8, device="cuda").view(F8) if bits == 8 else torch.zeros(c, device="cuda")
        sc = lambda c: [torch.zeros(-(-c // 128), device="cuda")] if bits == 8 else None
        one = [t[-k:].clone() for t in (ws, gs)]
        m, v, ms, vs, m1, v1, ms1, vs1 = mk(n), mk(n), sc(n), sc(n), mk(k), mk(k), sc(k), sc(k)
        K.adamw_multi_step([ws], [gs], [m], [v], 1e-2, m_scales=ms, v_scales=vs)
        K.adamw_multi_step([one[0]], [one[1]], [m1], [v1], 1e-2, m_scales=ms1, v_scales=vs1)
        assert torch.equal(ws[-k:], one[0])
        if bits == 8:                                            # the random bits go by the index, the scales do not
            assert torch.equal(ms[0][-9:], ms1[0]) and torch.equal(vs[0][-9:], vs1[0])
            up = lambda q, s: q[-k:].float() * s[0][-9:].repeat_interleave(128)[:k]
            assert ((up(m, ms) - up(m1, ms1)).abs() <= 0.125 * up(m1, ms1).abs() + ms1[0].max() * 2 ** -9).all()
        else:
            assert torch.equal(m[-k:], m1) and torch.equal(v[-k:], v1)
        del ws, gs, m, v
