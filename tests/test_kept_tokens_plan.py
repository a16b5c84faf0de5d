"""Plans count the sums of weights that a bounded cache keeps beside its pages."""
import dataclasses
import json

import pytest
import torch

from eredu_b200.models import config as C
from eredu_b200.runtime import plan as P
from eredu_b200.runtime.kv_cache import PAGE, PagedKVCache
from test_kv8_plan import checkpoint  # noqa: F401  (a fixture)


@pytest.mark.parametrize("heads, dim, layers", [(8, 128, 32), (2, 64, 3), (1, 80, 2)])
def test_estimates_are_the_bytes_of_the_cache(heads, dim, layers):
    cfg = dataclasses.replace(C.llama3_8b(), num_hidden_layers=layers, num_key_value_heads=heads, head_dim=dim)
    kv = PagedKVCache(layers, heads, dim, 10, torch.bfloat16, "cpu", weighed=True)
    assert P.estimate_runtime_state(cfg, weighed=True).kv_bytes_per_token * 10 * PAGE == kv.bytes()
    assert P.estimate_runtime_state(cfg, weighed=False) == P.estimate_runtime_state(cfg)


def test_plan_and_load_counts_sums(checkpoint, monkeypatch):  # noqa: F811
    from eredu_b200.api import LoadedModel, ModelLoadOptions

    seen = []
    plan = P.AutomaticPlanner.plan
    monkeypatch.setattr(P.AutomaticPlanner, "plan", lambda self, cfg, prof, **more: seen.append(prof) or plan(self, cfg, prof, **more))
    for keep in (None, 32):
        lm = LoadedModel.plan_and_load(str(checkpoint), ModelLoadOptions(device="cpu", max_seq_len=64, kv_keep=keep))
        assert (lm.engine.keep is not None) == (keep is not None)
    cfg = lm.config
    assert seen[1].kv_bytes_per_token - seen[0].kv_bytes_per_token == 4 * cfg.num_key_value_heads * cfg.num_hidden_layers


def test_command_line_counts_sums(checkpoint, tmp_path, capsys):  # noqa: F811
    from eredu_b200.cli.main import main

    cache = tmp_path / "plans.json"
    for more in ([], ["--kv-keep", "32"]):
        assert main(["-m", str(checkpoint), "hi", "--raw", "--device", "cpu", "--auto", "plan", "--auto-cache", str(cache), *more]) == 0
    assert len(json.loads(cache.read_text())) == 2
    capsys.readouterr()
