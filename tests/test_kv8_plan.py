"""Plans count the bytes of a cache held in 8 bits, and trials of a plan run with it."""
import dataclasses
import json
import subprocess

import pytest
import torch

from eredu_b200.models import config as C
from eredu_b200.runtime import plan as P
from eredu_b200.runtime.kv_cache import PAGE, PagedKVCache


@pytest.mark.parametrize("heads, dim, layers", [(8, 128, 32), (2, 64, 3), (1, 80, 2)])
def test_estimates_are_the_bytes_of_the_cache(heads, dim, layers):
    cfg = dataclasses.replace(C.llama3_8b(), num_hidden_layers=layers, num_key_value_heads=heads, head_dim=dim)
    kv = PagedKVCache(layers, heads, dim, 10, torch.bfloat16, "cpu", kv_bits=8)
    prof = P.estimate_runtime_state(cfg, kv_bits=8)
    # whole bytes a token and layer
    assert 0 <= prof.kv_bytes_per_token - kv.bytes() / (10 * PAGE) <= layers
    assert P.kv_bytes_for(prof, 10 * PAGE, 3) == 3 * 10 * PAGE * prof.kv_bytes_per_token
    assert P.estimate_runtime_state(cfg, kv_bits=16) == P.estimate_runtime_state(cfg)


def test_states_are_counted_in_their_own_type():
    from test_lfm2 import lfm2_cfg
    from test_qwen_next import next_cfg

    for cfg in (lfm2_cfg(), next_cfg()):
        a, b = P.estimate_runtime_state(cfg, kv_bits=8), P.estimate_runtime_state(cfg)
        assert a.state_bytes_per_sequence == b.state_bytes_per_sequence > 0
        assert 0.5 * b.kv_bytes_per_token < a.kv_bytes_per_token < 0.6 * b.kv_bytes_per_token


def test_contexts_that_fit_in_8_bits_are_admitted_and_planned():
    cfg = C.llama3_8b()
    bf16, kv8 = (P.estimate_runtime_state(cfg, kv_bits=bits) for bits in (16, 8))
    room = bf16.weight_bytes + bf16.workspace_bytes + int(0.75 * P.kv_bytes_for(bf16, 8192, 64))
    assert not P.apply_admission_policy(bf16, room, 8192, 64).admitted and P.apply_admission_policy(kv8, room, 8192, 64).admitted
    planner = P.AutomaticPlanner(P.HardwareProfile(device_count=1))
    planner.hw.device_memory_bytes = int(room / planner.fraction)
    modes = [planner.plan(cfg, prof, context=8192, batch=64, allow_quantization=False).residency["mode"] for prof in (bf16, kv8)]
    assert modes == ["layerwise_host", "fully_resident"]


@pytest.fixture
def checkpoint(tmp_path):
    from eredu_b200.formats import checkpoint as ck
    from eredu_b200.models.llama import random_state
    from test_cli import make_bundle

    b = make_bundle(tmp_path)
    cfg = dataclasses.replace(C.tiny_llama(), vocab_size=b.vocab_size(), eos_token_id=-1)
    ck.save_safetensors_checkpoint(tmp_path, cfg, random_state(cfg, seed=0, std=0.05), torch.float32)
    return tmp_path


def test_plan_and_load_counts_8_bits(checkpoint, monkeypatch):
    from eredu_b200.api import LoadedModel, ModelLoadOptions

    seen = []
    plan = P.AutomaticPlanner.plan
    monkeypatch.setattr(P.AutomaticPlanner, "plan", lambda self, cfg, prof, **kw: seen.append(prof.kv_bytes_per_token) or plan(self, cfg, prof, **kw))
    for bits in (None, 8):
        lm = LoadedModel.plan_and_load(str(checkpoint), ModelLoadOptions(device="cpu", max_seq_len=64, kv_bits=bits))
        assert lm.engine.kv.kv_bits == bits
    cfg = C.tiny_llama()
    per_layer = 2 * cfg.num_key_value_heads
    assert seen == [per_layer * cfg.head_dim * 2 * cfg.num_hidden_layers, -(-per_layer * (16 * cfg.head_dim + 4) // 16) * cfg.num_hidden_layers]


def test_plans_of_either_cache_are_kept_apart(checkpoint, capsys):
    from eredu_b200.cli.main import main

    cache = checkpoint / "auto.json"
    for bits in ("16", "8", "16"):
        assert main(["-m", str(checkpoint), "hi", "--device", "cpu", "-n", "2", "--auto-cache", str(cache), "--kv-bits", bits]) == 0
    assert len(json.loads(cache.read_text())) == 2


@pytest.mark.parametrize("bits", ["8", "16"])
def test_trials_run_with_the_cache_that_was_asked_for(checkpoint, capsys, monkeypatch, bits):
    from eredu_b200.cli.main import build_parser, main

    asked = []

    def run(cmd, **how):
        asked.append(build_parser().parse_args(cmd[3:]).kv_bits)
        return subprocess.CompletedProcess(cmd, 1, b"", b"not run")

    monkeypatch.setattr(subprocess, "run", run)
    try:
        main(["-m", str(checkpoint), "--device", "cpu", "--auto", "benchmark", "--auto-benchmark-tokens", "2", "--kv-bits", bits, "hello"])
    except (SystemExit, RuntimeError):
        pass                                # (no candidate is left)
    assert asked and set(asked) == {int(bits)}
