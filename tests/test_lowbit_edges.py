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
