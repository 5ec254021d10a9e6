"""``linear_precision`` of a run's recipe reaches the blocks that compute it, or the run is refused: llama-like blocks read it from
the hyper-parameters, families in reference form from their configuration, and no family ignores it."""
import dataclasses
import subprocess
import sys
from pathlib import Path

import pytest

from dataflow_b200.models.families import resolve_family
from dataflow_b200.run.driver import Trainer, synthetic_rounds
from dataflow_b200.run.recipe import Recipe

ROOT = Path(__file__).resolve().parent.parent
READS = ["llama3", "qwen3", "olmoe", "qwen3moe", "dsv3", "dsv32", "glm52"]
DOES_NOT = ["gpt2", "qwen35", "qwen35moe", "tp_mlp"]


def losses(family, hyper=None, steps=2, **over):
    cfg = dataclasses.replace(resolve_family(family).presets["tiny"](), **over)
    tr = Trainer(family, cfg, budget_gib=None, device=None, hyper={"lr": 3e-3, **(hyper or {})}, seed=3, recompute=False)
    try:
        return [tr.step(synthetic_rounds(cfg, tr.rounds, tr.T, 64, 11, s)) for s in range(steps)]
    finally:
        tr.close()


@pytest.mark.parametrize("family", ["dsv3", "dsv32", "glm52"])
def test_the_recipe_reaches_a_configuration_field(family):
    said_nothing = Recipe().hyper() | {"schedule": None}
    for p in ("fp8", "mxfp4"):
        got = losses(family, hyper=Recipe(linear_precision=p).hyper() | {"schedule": None})
        assert got == losses(family, hyper=said_nothing, linear_precision=p) and got != losses(family, hyper=said_nothing)
    base = losses(family)
    # and back: a recipe that says bf16 wins over a configuration that says otherwise, one that says nothing does not
    assert losses(family, hyper={"linear_precision": "bf16"}, linear_precision="fp8") == base
    assert losses(family, linear_precision="fp8") != base


@pytest.mark.parametrize("family", READS)
def test_families_that_read_it(family):
    cfg = resolve_family(family).presets["tiny"]()
    for p in (None, "bf16", "fp8", "mxfp4"):
        tr = Trainer(family, cfg, budget_gib=None, device=None, hyper={"linear_precision": p} if p else None, recompute=False, init=False)
        assert tr.linear_precision == (p or "bf16")
        tr.close()


@pytest.mark.parametrize("family", DOES_NOT)
def test_families_that_do_not_refuse(family):
    cfg = resolve_family(family).presets["tiny"]()
    for p in ("fp8", "mxfp4"):
        with pytest.raises(ValueError, match="linear_precision"):
            Trainer(family, cfg, budget_gib=None, device=None, hyper={"linear_precision": p}, recompute=False, init=False)
    if family != "tp_mlp":
        Trainer(family, cfg, budget_gib=None, device=None, hyper={"linear_precision": "bf16"}, recompute=False, init=False).close()


@pytest.mark.parametrize("family", READS + DOES_NOT)
def test_unknown_values_are_refused(family):
    cfg = resolve_family(family).presets["tiny"]()
    for p in ("fp4", "MXFP4", "", 8):
        with pytest.raises(ValueError, match="linear_precision"):
            Trainer(family, cfg, budget_gib=None, device=None, hyper={"linear_precision": p}, recompute=False, init=False)


def test_through_a_run_spec():
    from dataflow_b200.run.conductor import RunSpec, run
    spec = RunSpec(preset="dsv32:tiny", steps=2, device=None, data="synthetic:vocab=64,mean_len=48,seed=0", recompute=False)
    by_recipe = run(dataclasses.replace(spec, recipe={"linear_precision": "mxfp4"})).losses
    by_config = run(dataclasses.replace(spec, overrides={"linear_precision": "mxfp4"})).losses
    assert by_recipe == by_config and by_recipe != run(spec).losses


def test_through_the_service_spec():
    from types import SimpleNamespace
    from dataflow_b200.register import build_model_family_resolver, canonical_spec
    for family, ok in (("dsv32", True), ("llama3", True), ("gpt2", False)):
        spec = canonical_spec(family, resolve_family(family).presets["tiny"](), Recipe(linear_precision="mxfp4").hyper())
        if ok:
            build_model_family_resolver(spec, SimpleNamespace(device=None))
        else:
            with pytest.raises(ValueError, match="linear_precision"):
                build_model_family_resolver(spec, SimpleNamespace(device=None))


def test_the_twin_runs_the_same_forms():
    from dataflow_b200.testing.family_gate import run_pair
    hyper = {"lr": 2e-3, "weight_decay": 0.1}
    base = run_pair("dsv32", steps=2, hyper=hyper)["engine"]
    low = run_pair("dsv32", steps=2, hyper={**hyper, "linear_precision": "mxfp4"})
    assert low["engine"] != base and low["max_loss_rel"] < 1e-3


def test_the_command_line_refuses_in_one_line():
    r = subprocess.run([sys.executable, "tools/train/train.py", "train", "--preset", "gpt2:tiny", "--device", "cpu", "--steps", "1",
                        "--linear-precision", "mxfp4"], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert r.returncode == 2 and "linear_precision" in r.stderr and "Traceback" not in r.stderr, r.stderr


def test_an_unknown_precision_is_refused_where_it_is_written():
    """In the configuration and in the form itself: a value that no branch knows used to run as the plain product."""
    import torch
    from dataflow_b200.models import _forms as F
    for family in ("dsv3", "dsv32", "glm52"):
        cfg = resolve_family(family).presets["tiny"]()
        for p in ("fp4", "mxfp8", "", None):
            with pytest.raises(ValueError, match="linear_precision"):
                dataclasses.replace(cfg, linear_precision=p)
    x, w = torch.zeros(3, 64), torch.zeros(64, 5)
    for p in ("fp4", "", None):
        with pytest.raises(ValueError, match="linear_precision"):
            F.linear(x, w, p)
        with pytest.raises(ValueError, match="linear_precision"):
            F.swiglu_mlp(x, torch.zeros(64, 64), torch.zeros(32, 5), p)


def test_measured_costs_of_one_precision_are_not_used_for_another():
    """The cost cache's key: the precision is a hyper-parameter of the llama-like families, not a field of their configuration."""
    from dataflow_b200.run.profiling import profile_key
    keys = {}
    for family in ("llama3", "dsv32"):
        cfg = resolve_family(family).presets["tiny"]()
        for p in (None, "bf16", "fp8", "mxfp4"):
            tr = Trainer(family, cfg, budget_gib=None, device=None, hyper={"linear_precision": p} if p else None, recompute=False, init=False)
            keys[family, p] = profile_key(tr, tr.cfg)
            tr.close()
        assert keys[family, None] == keys[family, "bf16"] and len({keys[family, p] for p in ("bf16", "fp8", "mxfp4")}) == 3
