"""Narrow-format operators (``K.lowbit``) where their ranges end: squares below and above the normal numbers, rows whose statistic is
not a number, lists and matrices long enough that a block walks on.  Runs on the plain-torch lane (CPU) and, on a device, on the kernels."""
import math

import pytest
import torch

from dataflow_b200.ops import lowbit_eager as E
from dataflow_b200.ops import resolve_kernels

BF, F32, F64, F8, U8 = torch.bfloat16, torch.float32, torch.float64, torch.float8_e4m3fn, torch.uint8
LANES = [pytest.param("cpu", id="eager"), pytest.param("cuda", id="sm100", marks=pytest.mark.gpu)]


def lane(dev):
    return resolve_kernels(kernel_set="eager" if dev == "cpu" else None).lowbit


def plain():
    return resolve_kernels(kernel_set="eager").lowbit


def same_bytes(a, b):
    return torch.equal(a.contiguous().view(U8), b.contiguous().view(U8))


# ------------------------------------------------------------------ AdamW: the root of the second moment
def lone_gradients(n, seed):
    """One gradient per block of 128, over the whole range of fp32, so that a block's scale tells its root."""
    g = torch.Generator().manual_seed(seed)
    e = torch.randint(-78, 64, (n,), generator=g)
    v = torch.ldexp(1 + torch.rand(n, generator=g), e) * torch.where(torch.rand(n, generator=g) < 0.5, -1.0, 1.0)
    ends = torch.tensor([0.0, -0.0, 1e-20, -3e-21, 1e-22, 4e-23, 1e-30, 1e-44, 1.9e19, 3e19, -1e20, 1e30, -1e38, 2.0 ** -63, 2.0 ** -45,
                         2.0 ** -44, float("inf"), float("nan")])
    v[:len(ends)] = ends
    return v


@pytest.mark.parametrize("dev", LANES)
def test_adamw_8bit_root_over_the_whole_range(dev):
    """The scale of a block with one gradient is the root of its square, both rounded as the definition says (a root in 64 bits,
    rounded once to 32, is the correctly rounded one), from the smallest subnormal square up to squares that overflow."""
    k, n = lane(dev), 1 << (13 if dev == "cpu" else 19)
    lone = lone_gradients(n, 3)
    x = (lone * lone) * torch.tensor(1 - 0.95, dtype=F32)
    r = torch.sqrt(x.double()).float()
    want = torch.where(r == r, r * torch.tensor(1 / 448, dtype=F32), torch.zeros(())).clamp(min=2.0 ** -120)
    grad = torch.zeros(n, 128)
    grad[:, 77] = lone
    grad = grad.view(-1).to(dev)
    w0 = torch.ones(n * 128, device=dev)
    w, m, v = w0.clone(), torch.zeros(n * 128, device=dev).to(F8), torch.zeros(n * 128, device=dev).to(F8)
    ms, vs = torch.zeros(n, device=dev), torch.zeros(n, device=dev)
    k.adamw_multi_step([w], [grad], [m], [v], 1e-3, 0.9, 0.95, 1e-8, 0.0, 1, m_scales=[ms], v_scales=[vs])
    bad = vs.cpu().view(torch.int32) != want.view(torch.int32)
    assert not bad.any(), [(float(lone[i]), float(vs[i]), float(want[i])) for i in torch.nonzero(bad).view(-1)[:5].tolist()]
    got = v.view(n, 128)[:, 77].float().cpu() * vs.cpu()
    fine = r.isfinite()
    # a block's largest code is 448 or, rounded down, 416
    assert ((got - r).abs()[fine] <= r[fine] / 14 * (1 + 1e-6) + 2.0 ** -126).all() and torch.isnan(got[~fine]).all()
    # a square that overflows is an infinite root: the weight stays; only an infinite gradient or a NaN takes it along
    w = w.view(n, 128)[:, 77].cpu()
    assert torch.equal(torch.isnan(w), ~lone.isfinite()) and (w[r == math.inf][lone[r == math.inf].isfinite()] == 1).all()


@pytest.mark.gpu
def test_adamw_lanes_agree_to_the_bit_over_the_whole_range():
    """Whole blocks of tiny, ordinary and huge gradients, and states that these left behind, over three steps."""
    g = torch.Generator().manual_seed(8)
    n = 4096 * 128
    size = torch.pow(10.0, torch.rand(n // 128, 1, generator=g, dtype=F64) * 44 - 24.5)
    runs = []
    grads = [(torch.randn(n // 128, 128, generator=g) * size).float().view(-1).cuda() for _ in range(2)] + [torch.zeros(n, device="cuda")]
    for K in (lane("cuda"), plain()):
        w, m, v = torch.ones(n, device="cuda"), torch.zeros(n, device="cuda").to(F8), torch.zeros(n, device="cuda").to(F8)
        ms, vs = torch.zeros(n // 128, device="cuda"), torch.zeros(n // 128, device="cuda")
        steps = []
        for i, grad in enumerate(grads):
            K.adamw_multi_step([w], [grad], [m], [v], 1e-3, step=i + 1, m_scales=[ms], v_scales=[vs])
            steps.append([t.clone() for t in (m.float(), v.float(), ms, vs, w.isfinite().float())])
        runs.append(steps)
    for a, b in zip(*runs):
        for i, (s, t) in enumerate(zip(a, b)):
            assert torch.equal(torch.isnan(s), torch.isnan(t)), i
            assert torch.equal(torch.nan_to_num(s, nan=-1.0), torch.nan_to_num(t, nan=-1.0)), i


# ------------------------------------------------------------------ the norm: rows whose statistic is not a number
@pytest.mark.parametrize("dev", LANES)
@pytest.mark.parametrize("cols", [32, 96, 352, 608, 1056, 2080, 4128, 8224, 16416])
@pytest.mark.parametrize("off", [0, 8], ids=["on32", "on16"])
def test_norm_scale_bytes_past_the_blocks_are_zero_in_every_row(dev, cols, off):
    """A NaN, an infinity and statistics that are neither: the row's own blocks may be NaN, the bytes behind them are zero, and the
    other rows are those of a call without these."""
    k, g = lane(dev), torch.Generator().manual_seed(cols)
    buf = torch.randn(6, cols + 32, generator=g).to(BF).to(dev)
    w = torch.randn(cols, generator=g).to(BF).to(dev)
    clean = k.rmsnorm_mxfp4(buf[:, off:off + cols], w)
    bad = buf.clone()
    bad[1, off + cols - 1], bad[4, off] = float("nan"), float("inf")
    for res in (None, torch.zeros_like(buf)[:, off:off + cols]):
        q, s, _, rstd = k.rmsnorm_mxfp4(bad[:, off:off + cols], w, residual=res)
        assert torch.isnan(rstd[1]) and rstd[4] == 0
        rows = E.mxfp4_scale_rows(s, 6, cols)
        assert torch.equal(E.mxfp4_scale_tiles(rows), s)
        assert (rows[1] == 255).all()
        for r in (0, 2, 3, 5):
            assert torch.equal(q[r], clean[0][r]) and torch.equal(rows[r], E.mxfp4_scale_rows(clean[1], 6, cols)[r])
    for value in (float("nan"), float("inf"), -float("inf")):
        given = clean[3].clone()
        given[3] = value
        s = k.rmsnorm_mxfp4(buf[:, off:off + cols], w, rstd=given)[1]
        assert torch.equal(E.mxfp4_scale_tiles(E.mxfp4_scale_rows(s, 6, cols)), s)


# ------------------------------------------------------------------ the linear form: what the forward takes, the backward takes
@pytest.mark.parametrize("dev", LANES)
@pytest.mark.parametrize("m", [32, 7], ids=["m32", "m7"])
def test_linear_form_of_views_that_start_anywhere(dev, m):
    """Contiguous views one element into their storage, and a gradient that is one: the same numbers as of copies on their own."""
    from dataflow_b200.models import _forms as F
    n, k = 48, 64
    dt = BF if dev == "cuda" else F32
    g = torch.Generator().manual_seed(4)
    flat = [torch.randn(a * b + 1, generator=g).to(dt).to(dev) for a, b in ((n, k), (k, m), (n, m))]
    off = [t[1:].view(a, b) for t, (a, b) in zip(flat, ((n, k), (k, m), (n, m)))]
    on = [t.clone() for t in off]
    assert all(t.is_contiguous() and t.data_ptr() % 16 for t in off)
    outs = []
    for x, w, dy in (on, off):
        x, w = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
        y = F.linear(x, w, "mxfp4")
        outs.append((y.detach(), *torch.autograd.grad(y, [x, w], dy)))
    for a, b in zip(*outs):
        assert torch.equal(a, b)


def test_linear_form_refuses_operands_of_two_types():
    """The plain product does, and the backward would."""
    from dataflow_b200.models import _forms as F
    for a, b in ((BF, F32), (F32, BF)):
        with pytest.raises(ValueError, match="one type"):
            F.linear(torch.zeros(3, 64, dtype=a), torch.zeros(64, 8, dtype=b), "mxfp4")


# ------------------------------------------------------------------ AdamW: random bits of several tensors
def eight_bit(dev, sizes, seed):
    g = torch.Generator().manual_seed(seed)
    mk = lambda n, s: torch.randn(n, generator=g).mul(s).to(dev)
    zero = lambda n: torch.zeros(n, device=dev)
    return {"ws": [mk(n, 0.05) for n in sizes], "gs": [mk(n, 1e-2) for n in sizes], "ms": [mk(n, 9).to(F8) for n in sizes],
            "vs": [mk(n, 9).abs().to(F8) for n in sizes], "m_scales": [zero(-(-n // 128)) + 1e-4 for n in sizes],
            "v_scales": [zero(-(-n // 128)) + 1e-4 for n in sizes]}


def adam8(k, st, **kw):
    k.adamw_multi_step(st["ws"], st["gs"], st["ms"], st["vs"], 1e-3, wds=0.1, step=3, m_scales=st["m_scales"], v_scales=st["v_scales"], **kw)


@pytest.mark.parametrize("dev", LANES)
def test_adamw_takes_a_seed_per_tensor(dev):
    """A list of seeds is one call per tensor with its own; a number is the same for all, and the step where there is none."""
    k, sizes, seeds = lane(dev), [300 + 40 * i for i in range(30)], [(7 * i * i + 1) * 0x12345 for i in range(30)]
    runs = {}
    for name, kw in (("list", {"seed": seeds}), ("number", {"seed": 3}), ("same", {"seed": [3] * 30}), ("none", {})):
        adam8(k, runs.setdefault(name, eight_bit(dev, sizes, 1)), **kw)
    one = eight_bit(dev, sizes, 1)
    for i, s in enumerate(seeds):
        adam8(k, {n: [t[i]] for n, t in one.items()}, seed=s)
    for n in one:
        for i in range(30):
            assert same_bytes(runs["list"][n][i], one[n][i]) and same_bytes(runs["number"][n][i], runs["same"][n][i])
            assert same_bytes(runs["number"][n][i], runs["none"][n][i])
    assert not same_bytes(runs["list"]["ms"][5], runs["none"]["ms"][5])
    for bad in (seeds[:-1], seeds + [1], []):
        with pytest.raises(ValueError, match="seed"):
            adam8(k, one, seed=bad)


def test_every_field_of_every_layer_rounds_with_random_bits_of_its_own():
    """The same bits for element i of all layers would add their rounding errors up instead of averaging them."""
    import dataclasses
    from dataflow_b200.models.families import resolve_family
    from dataflow_b200.run.driver import Trainer, synthetic_rounds
    cfg = dataclasses.replace(resolve_family("llama3").presets["tiny"](), dtype_policy="bf16_8bit")

    def seeds_of_two_steps():
        K, calls = resolve_kernels(kernel_set="eager"), []
        step = K.lowbit.adamw_multi_step

        def recorded(ws, *a, seed=None, **kw):
            calls.extend(seed if isinstance(seed, list) else [seed] * len(ws))
            return step(ws, *a, seed=seed, **kw)
        K.lowbit.adamw_multi_step = recorded
        tr = Trainer("llama3", cfg, budget_gib=None, device=None, hyper={"lr": 1e-3}, seed=0, kernels=K)
        for s in range(2):
            tr.step(synthetic_rounds(cfg, tr.rounds, tr.T, 64, 1, s))
        tr.close()
        return calls
    calls = seeds_of_two_steps()
    assert None not in calls and len(set(calls)) == len(calls) == 2 * (5 * cfg.n_layers + 1 + 2 + cfg.n_layers)
    assert calls == seeds_of_two_steps()


# ------------------------------------------------------------------ AdamW: overlaps that are not neighbours
def overlapping_lists():
    f = lambda n=128: torch.zeros(n)
    big = torch.zeros(1024)
    yield "a weight inside a long gradient, a short one between", ([f(512), f(), big[300:428]], [big[:512], big[100:228], f()], 3)
    yield "a moment inside a long gradient, a short one between", ([f(512), f(), f()], [big[:512], big[100:228], f()], big[300:428])
    yield "weights and gradients are one list", (None, None, 1)


@pytest.mark.parametrize("name,args", list(overlapping_lists()), ids=[n for n, _ in overlapping_lists()])
@pytest.mark.parametrize("where", ["plain lane", "extension"])
def test_adamw_refuses_a_written_tensor_inside_a_longer_one(name, args, where):
    from dataflow_b200.ops import lowbit, native_available
    if where == "extension" and not native_available():
        pytest.skip("extension not built")
    K = plain() if where == "plain lane" else lowbit
    ws, gs, last = args
    if ws is None:
        ws = gs = [torch.zeros(128)]
        ms, vs = [torch.zeros(128)], [torch.zeros(128)]
    else:
        ms, vs = [torch.zeros(t.numel()) for t in ws], [torch.zeros(t.numel()) for t in ws]
        if torch.is_tensor(last):
            vs[-1] = last
    with pytest.raises(ValueError, match="twice or overlaps"):
        K.adamw_multi_step(ws, gs, ms, vs, 1e-3)


def test_adamw_gradients_may_share_memory():
    """They are only read."""
    big, f = torch.ones(512), lambda n: torch.zeros(n)
    ws = plain().adamw_multi_step([f(512), f(128), f(128)], [big, big[100:228], big[100:228]], [f(512), f(128), f(128)], [f(512), f(128), f(128)], 1e-3)
    assert all((w < 0).all() for w in ws)


# ------------------------------------------------------------------ blocks that walk on
def poison():
    """Freed memory that is neither zero nor what an earlier call left."""
    junk = [torch.full((n << 20,), 0xA5, dtype=U8, device="cuda") for n in (256, 64, 64, 8, 2, 1, 1, 1)]
    torch.cuda.synchronize()
    del junk


def sm_count():
    return torch.cuda.get_device_properties(0).multi_processor_count


@pytest.mark.gpu
@pytest.mark.parametrize("off", [0, 8], ids=["on32", "on16"])
@pytest.mark.parametrize("cols", [96, 256, 512, 1024, 2048, 4096, 8192, 16384])
@pytest.mark.parametrize("fmt", ["fp8", "mxfp4"])
def test_norm_rows_behind_the_first_of_a_block(fmt, cols, off):
    """A block holds the next row's loads while it works on one and comes back for more rows when the matrix has more than the grid:
    every row, its codes, scales (raw tiles, padding included), stream and statistic are those of slices that no block walks over."""
    k = lane("cuda")
    fn = k.rmsnorm_fp8 if fmt == "fp8" else k.rmsnorm_mxfp4
    # threads of a row: one warp up to 1024 columns, else 128, 256 or 512 (twice as many in the 16-byte form); 1024 an SM at once
    threads = 32 if cols <= 1024 else {2048: 128, 4096: 128, 8192: 256, 16384: 512}[cols]
    rows = 2 * sm_count() * (1024 // threads) + sm_count() * (512 // threads) + 77
    g = torch.Generator(device="cuda").manual_seed(cols + off)
    big = torch.randn(rows, cols + 16, device="cuda", generator=g).to(BF)
    res = torch.randn(rows, cols + 16, device="cuda", generator=g).to(BF)
    w = (1 + 0.1 * torch.randn(cols, device="cuda", generator=g)).to(BF)
    x, r = big[:, off:off + cols], res[:, off:off + cols]
    for residual in (None, r):
        poison()
        got = fn(x, w, residual=residual)
        given = fn(x, w, residual=residual, rstd=got[3])
        for a in range(0, rows, 256):
            b = min(a + 256, rows)
            want = fn(x[a:b], w, residual=None if residual is None else residual[a:b])
            for full, part in ((got, want), (given, want)):
                assert same_bytes(full[0][a:b], part[0]) and same_bytes(full[2][a:b], part[2]) and torch.equal(full[3][a:b], part[3])
                if fmt == "fp8":
                    assert torch.equal(full[1][a:b], part[1])
                else:
                    assert torch.equal(full[1][a // 128:a // 128 + part[1].shape[0]], part[1])
    # the sum in place of the residual, rows already on their way included
    out = res.clone()
    q, s, h, rstd = fn(x, w, residual=out[:, off:off + cols], h_out=out[:, off:off + cols])
    assert same_bytes(q, got[0]) and torch.equal(s, got[1]) and same_bytes(h, got[2]) and torch.equal(rstd, got[3])
    assert torch.equal(out[:, :off], res[:, :off]) and torch.equal(out[:, off + cols:], res[:, off + cols:])


def adam_lists(form, gdt, sizes, seed, starts):
    """Lists with 8-bit moments; ``starts``: bytes by which weights, gradients and masters, and states, miss a multiple of 512."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    wide, state = starts

    def at(t, miss):
        off = miss // t.element_size()
        buf = torch.empty(off + t.numel(), dtype=t.dtype, device="cuda")
        buf[off:] = t
        assert (buf[off:].data_ptr() - miss) % 512 == 0
        return buf[off:]
    rnd = lambda n, s: torch.randn(n, device="cuda", generator=g) * s
    st = {n: [] for n in ("ws", "gs", "ms", "vs", "m_scales", "v_scales")}
    for n in sizes:
        full = rnd(n, 0.05)
        if form == "fp32":
            st["ws"].append(at(full, wide))
        elif form == "split":
            hi, lo = E.split_master_cut(full)
            st["ws"].append(at(hi, wide))
            st.setdefault("los", []).append(at(lo, wide))
        else:
            st["ws"].append(at(full.to(BF), wide))
            if form == "master":
                st.setdefault("masters", []).append(at(full, wide))
        st["gs"].append(at(rnd(n, 1e-2).to(gdt), wide))
        st["ms"].append(at(rnd(n, 60).to(F8), state))
        st["vs"].append(at(rnd(n, 60).abs().to(F8), state))
        for name in ("m_scales", "v_scales"):
            st[name].append(1e-5 * (1 + torch.rand(-(-n // 128), device="cuda", generator=g)))
    return st


def adam_step(k, st, only=None):
    pick = (lambda l: l) if only is None else (lambda l: [l[only]])
    k.adamw_multi_step(*[pick(st[n]) for n in ("ws", "gs", "ms", "vs")], 1e-3, wds=0.1, step=3,
                       **{n: pick(st[n]) for n in ("masters", "los", "m_scales", "v_scales") if n in st})


# more elements than blocks of one group take: ragged ends, an end inside a block's 8192, one inside a group of 512, whole blocks
def long_sizes():
    least = 2 * sm_count() * 16 * 8192
    return [least // 2 + 3, least // 2 + 8192 * 5 + 517, 8192 * 64, 300, 8192 * 3 + 128, 129, 1]


@pytest.mark.gpu
@pytest.mark.parametrize("gdt", [BF, F32], ids=["gbf16", "gfp32"])
@pytest.mark.parametrize("form", ["bf16", "fp32", "master", "split"])
@pytest.mark.parametrize("starts", [(0, 0), (16, 16), (0, 16), (16, 0), (2, 1), (32, 48)], ids=["aligned", "on16", "states16", "weights16", "odd", "by32"])
def test_adamw_long_lists(form, gdt, starts):
    """Lists of more than 2 x SMs x 16 x 8192 elements, where a block takes 8192 at a time with the next group on its way: every
    element of every tensor as in a call on that tensor alone, which takes one group a block, from 512-byte starts."""
    if starts[0] % 4 and (form in ("fp32", "master") or gdt == F32):
        starts = (4, starts[1])
    k, sizes = lane("cuda"), long_sizes()
    st, one = adam_lists(form, gdt, sizes, 5, starts), adam_lists(form, gdt, sizes, 5, (0, 0))
    assert sum(sizes) >= 2 * sm_count() * 16 * 8192 > max(sizes)
    adam_step(k, st)
    for i in range(len(sizes)):
        adam_step(k, one, only=i)
        for n in st:
            assert same_bytes(st[n][i], one[n][i]), (n, i)


@pytest.mark.gpu
@pytest.mark.parametrize("starts", [(0, 0), (16, 16)], ids=["on32", "on16"])
def test_adamw_long_lists_against_the_plain_lane(starts):
    """The state to the bit, and the weights by the definition in 64 bits on the plain lane's unrounded arithmetic: lr times a
    quotient that is off by at most 8 roundings and the approximate reciprocal (2^-23), and 4 roundings of the weight."""
    sizes = long_sizes()
    st, ref = adam_lists("master", BF, sizes, 6, starts), adam_lists("master", BF, sizes, 6, (0, 0))
    old = [t.clone() for t in ref["masters"]]
    adam_step(lane("cuda"), st)
    adam_step(plain(), ref)
    for i in range(len(sizes)):
        for n in ("ms", "vs", "m_scales", "v_scales"):
            assert same_bytes(st[n][i], ref[n][i]), (n, i)
        moved = (ref["masters"][i].double() - old[i].double()).abs()
        err = (st["masters"][i].double() - ref["masters"][i].double()).abs()
        assert (err <= 16 * 2.0 ** -24 * moved + 8 * 2.0 ** -24 * old[i].double().abs()).all()
        assert torch.equal(st["ws"][i], st["masters"][i].to(BF))


@pytest.mark.gpu
@pytest.mark.parametrize("form", ["bf16", "fp32", "master", "split"])
@pytest.mark.parametrize("starts", [(16, 16), (0, 16), (16, 0), (48, 32)], ids=["on16", "states16", "weights16", "by16"])
def test_adamw_short_lists_that_start_on_16_bytes(form, starts):
    """Weights on 16 but not 32 bytes with states on 16: the kernel's 16-byte form, which a common offset of elements never meets."""
    k, sizes = lane("cuda"), [512 * 7, 4096, 512 + 77, 128]
    st, one = adam_lists(form, BF, sizes, 7, starts), adam_lists(form, BF, sizes, 7, (0, 0))
    adam_step(k, st)
    adam_step(k, one)
    for n in st:
        for a, b in zip(st[n], one[n]):
            assert same_bytes(a, b), n


# ------------------------------------------------------------------ the norm's 8-bit operand in the 8-bit product
@pytest.mark.parametrize("dev", LANES)
@pytest.mark.parametrize("M,K,N", [(1, 32, 16), (130, 208, 72), (300, 1040, 264)])
def test_norm_to_fp8_feeds_the_fp8_product(dev, M, K, N):
    """Codes and scales go into ``linear_fp8`` as they are: against 64 bits on the same codes, K products of 8-bit codes summed in 32
    bits (each addition off by at most 2^-23 of the running magnitude), two scalings, one rounding to bf16."""
    ks = resolve_kernels(kernel_set="eager" if dev == "cpu" else None)
    g = torch.Generator().manual_seed(M + N)
    x, res = torch.randn(M, K, generator=g).to(BF).to(dev), torch.randn(M, K, generator=g).to(BF).to(dev)
    gain, w = (1 + 0.1 * torch.randn(K, generator=g)).to(BF).to(dev), (torch.randn(N, K, generator=g) * K ** -0.5).to(BF).to(dev)
    q, s, h, rstd = ks.lowbit.rmsnorm_fp8(x, gain, residual=res)
    wq, sw = ks.quant_fp8_rowwise(w)
    y = ks.linear_fp8(q, s, wq, sw)
    A, B = q.double() * s.double()[:, None], wq.double() * sw.double()[:, None]
    want = A @ B.t()
    bound = ((K + 2) * 2.0 ** -23 + 3 * 2.0 ** -24) * (A.abs() @ B.abs().t()) + torch.finfo(BF).eps / 2 * want.abs()
    assert y.dtype == BF and ((y.double() - want).abs() <= bound).all()
    # and what the codes stand for is the norm of the sum, off by half a code (2^-4 of the value, or of the smallest normal code)
    h64 = (x.float() + res.float()).to(BF).double()
    y64 = h64 / torch.sqrt(h64.square().mean(-1, keepdim=True) + 1e-5) * gain.double()
    assert torch.equal(h.double(), h64)
    assert ((A - y64).abs() <= (2.0 ** -4 + (K + 16) * 2.0 ** -24) * y64.abs() + s.double()[:, None] * 2.0 ** -10).all()
