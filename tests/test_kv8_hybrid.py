"""Models with recurrent states beside 8-bit pages: what is not a page of keys or values keeps the model's type."""
import pytest
import torch

from eredu_b200.models import config as C
from eredu_b200.models.llama import build_from_tensors, random_state
from eredu_b200.models.moe import make_moe_factory
from eredu_b200.ops import SamplingParams
from eredu_b200.runtime.engine import Engine
from eredu_b200.runtime.kv_cache import PagedKVCache

GREEDY = SamplingParams(temperature=0.0)
DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def built(family, device):
    """A small model of the family (heads of 64, which the GPU's kernels take). Where there are experts every token takes all of them: a choice that
    falls to the other side would move logits by more than the cache does."""
    if family == "lfm2":
        from test_lfm2 import lfm2_cfg

        cfg = lfm2_cfg(hidden_size=256, num_attention_heads=4, num_key_value_heads=2, vocab_size=512)
        sd = random_state(cfg, seed=8, std=0.05)
    elif family == "qwen_next":
        from test_qwen_next import next_cfg, state_for

        cfg = next_cfg(hidden_size=256, head_dim=64, linear_key_head_dim=64, linear_value_head_dim=64, vocab_size=512, num_experts_per_tok=8,
                       moe_intermediate_size=64, shared_expert_intermediate_size=64)
        sd = {k: v * (0.6 if v.dim() == 2 else 1.0) for k, v in state_for(cfg, seed=4).items()}
    else:
        from test_nemotron_h import nh_cfg, state_for

        cfg = nh_cfg(hybrid_override_pattern="M-M*-M*", hidden_size=256, head_dim=64, mamba_num_heads=8, mamba_head_dim=64, ssm_state_size=64, vocab_size=512)
        sd = {k: v * (0.6 if v.dim() == 2 else 1.0) for k, v in state_for(cfg, seed=3).items()}
    more = {"moe_factory": make_moe_factory()} if family == "qwen_next" else {}
    return build_from_tensors(cfg, sd.__getitem__, sd.__contains__, device, torch.float32 if device == "cpu" else torch.bfloat16, **more)


def prompt(n, seed=0):
    return torch.randint(0, 512, (n,), generator=torch.Generator().manual_seed(seed)).tolist()


def fed(model, bits, tokens, more):
    eng = Engine(model, max_batch=2, max_seq_len=128, kv_bits=bits)
    seq = eng.new_sequence(tokens, GREEDY, max_new_tokens=16)
    out = [eng.feed_logits(seq, tokens)] + [eng.feed_logits(seq, [t]) for t in more]
    return torch.stack(out).float().cpu(), eng, seq


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("family", ["lfm2", "qwen_next", "nemotron_h"])
@pytest.mark.parametrize("n", [1, 16, 41])
def test_logits_are_near_those_of_the_plain_cache(device, family, n):
    """A cached value is off by a per cent or two of a typical one; a state that is cut to whole numbers moves logits by as much as they are large. A tenth lies between."""
    model = built(family, device)
    want = fed(model, None, prompt(n), prompt(5, seed=7))[0]
    got, eng, _ = fed(model, 8, prompt(n), prompt(5, seed=7))
    kv = eng.kv
    for t in (kv.conv_state, kv.la_conv_state):
        assert t is None or t.dtype == model.dtype
    assert kv.conv_state is not None or kv.la_conv_state is not None
    assert kv.k.dtype == torch.int8
    assert ((got - want).norm(dim=1) <= 0.1 * want.norm(dim=1)).all()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("family", ["lfm2", "qwen_next", "nemotron_h"])
def test_forked_and_moved_states(device, family):
    """A fork and a sequence whose pages move go on as the sequence itself does; states are copied as they are."""
    model = built(family, device)
    more = prompt(4, seed=9)
    want = fed(model, 8, prompt(37), more)[0][1:]
    _, eng, seq = fed(model, 8, prompt(37), [])
    stranger = eng.new_sequence(prompt(20, seed=2), GREEDY, max_new_tokens=4)
    other = eng.fork(seq)
    assert not set(other.pages) & set(seq.pages)
    eng.release(stranger)
    assert eng.compact([seq, other]) > 0
    got = [torch.stack([eng.feed_logits(s, [t]).float().cpu() for t in more]) for s in (other, seq)]
    assert torch.equal(got[0], want) and torch.equal(got[1], want)
    assert len(eng.generate([prompt(9), prompt(22)], GREEDY, max_new_tokens=6, samples=1)[0]) == 6


@pytest.mark.gpu
@pytest.mark.parametrize("family", ["lfm2", "qwen_next", "nemotron_h"])
def test_captured_steps_are_the_eager_ones(family):
    model = built(family, "cuda")
    prompts = [prompt(n, seed=n) for n in (7, 40)]
    out = [Engine(model, max_batch=2, max_seq_len=128, kv_bits=8, use_cuda_graph=graph).generate(prompts, GREEDY, max_new_tokens=6) for graph in (True, False)]
    assert out[0] == out[1] and [len(o) for o in out[0]] == [6, 6]


def test_states_of_a_cache_keep_the_type_that_was_asked_for():
    for kind in (torch.float32, torch.bfloat16):
        kv = PagedKVCache(3, 1, 64, 5, kind, "cpu", attention_layers=[1], conv_layers=[0], conv_channels=8, conv_hist=2, kv_bits=8)
        kv.enable_linear_attention_state([2], slots=3, conv_hist=3, conv_channels=8, heads=1, dk=4, dv=4)
        assert kv.k.dtype == kv.v.dtype == torch.int8 and kv.conv_state.dtype == kv.la_conv_state.dtype == kind
        half = kv.bytes()
        kv = PagedKVCache(3, 1, 64, 5, kind, "cpu", attention_layers=[1], conv_layers=[0], conv_channels=8, conv_hist=2)
        kv.enable_linear_attention_state([2], slots=3, conv_hist=3, conv_channels=8, heads=1, dk=4, dv=4)
        assert kv.conv_state.dtype == kv.la_conv_state.dtype == kind and half < kv.bytes()
