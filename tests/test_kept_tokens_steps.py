"""Caches of bounded size under a scheduler: rows that are held back, steps that fail, calls that are refused."""
import dataclasses

import pytest
import torch

from eredu_b200.models import config as C
from eredu_b200.models.llama import build_from_tensors, random_state
from eredu_b200.ops import SamplingParams
from eredu_b200.runtime.engine import Engine
from eredu_b200.runtime.kv_cache import KeptTokens
from eredu_b200.runtime.server import Server

GREEDY = SamplingParams(temperature=0.0)
DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def build(device="cpu"):
    cfg = dataclasses.replace(C.tiny_llama(), num_hidden_layers=2, vocab_size=512)
    sd = random_state(cfg, seed=0, std=0.08)
    return build_from_tensors(cfg, sd.__getitem__, sd.__contains__, device, torch.float32 if device == "cpu" else torch.bfloat16)


def prompt(n, seed=0):
    return torch.randint(0, 512, (n,), generator=torch.Generator().manual_seed(seed)).tolist()


def joined(eng, *prompts, new=40):
    eng.open_decode()
    seqs = []
    for p in prompts:
        s = eng.new_sequence(p, GREEDY, max_new_tokens=new)
        s.output.append(int(eng.prefill([s])[0]))
        eng.join(s, s.output[-1])
        seqs.append(s)
    return seqs


def step(eng, stepping):
    st = eng._decode_state
    eng.set_step_mask(stepping)
    st["stepped"] = stepping
    eng.commit(eng.decode_step().tolist())


def sums(eng, seq):
    """Of every cached token of a sequence, all layers and heads."""
    at = torch.tensor(seq.pages, device=eng.device)
    return eng.kv.weights[0][0][:, at].transpose(1, 2).flatten(2)[..., :seq.cached].cpu()


@pytest.mark.parametrize("device", DEVICES)
def test_a_row_that_is_held_back_gives_no_weight(device):
    """Its tokens keep their sums, bit by bit, and what it says afterwards is what it says without a pause."""
    model = build(device)
    rule = KeptTokens(keep=32, recent=8, slack=6)
    outs = []
    for pauses in ((), (0, 1, 5, 6, 7, 20)):
        eng = Engine(model, max_batch=2, max_seq_len=256, kv_keep=rule)
        held, other = joined(eng, prompt(30), prompt(45, 1), new=60)
        for i in range(45):
            if i in pauses:
                eng._shrink_decoding(eng._decode_state)      # (a row at its bound is cut down ahead of any step)
                before = sums(eng, held)
                step(eng, [False, True])
                assert torch.equal(sums(eng, held), before)
            step(eng, [True, True])
        outs.append(held.output)
    assert len(outs[0]) == 46 and outs[0] == outs[1]


@pytest.mark.parametrize("device", DEVICES)
def test_a_free_slot_and_a_finished_row_give_no_weight(device):
    """Pages that nobody decodes into - page 0, which free slots point at, and those of a row that has ended - keep their sums."""
    eng = Engine(build(device), max_batch=3, max_seq_len=128, kv_keep=64)
    a, b = joined(eng, prompt(20), prompt(20, 1))
    b.finished = True
    nobody, ended = eng.kv.weights[0][0][:, 0].clone(), sums(eng, b)
    for _ in range(3):
        step(eng, [True, True, True])
    assert torch.equal(eng.kv.weights[0][0][:, 0], nobody) and torch.equal(sums(eng, b), ended) and len(a.output) == 4


@pytest.mark.parametrize("budget, chunk", [(17, 16), (64, 48), (4, 16)])
@pytest.mark.parametrize("seed", [0, 10, 20])
def test_a_budget_that_holds_rows_back_changes_no_answer(budget, chunk, seed):
    model = build()
    rule = KeptTokens(keep=32, recent=4, slack=5)
    prompts = [prompt(n, seed + i) for i, n in enumerate((70, 9, 45, 33))]
    alone = [Engine(model, max_batch=1, max_seq_len=256, kv_keep=rule).generate([p], GREEDY, max_new_tokens=60)[0] for p in prompts]
    server = Server(Engine(model, max_batch=4, max_seq_len=256, kv_keep=rule), prefill_chunk=chunk, max_step_tokens=budget)
    ids = [server.submit(p, GREEDY, 60) for p in prompts]
    server.run_until_idle(max_steps=2000)
    assert [server.result(i).tokens for i in ids] == alone


def failing(eng, monkeypatch, at):
    """The ``at``-th forward pass from now on raises."""
    forward, count = eng.model.forward, [0]

    def once(*a, **k):
        count[0] += 1
        if count[0] == at:
            raise RuntimeError("a step that fails")
        return forward(*a, **k)

    monkeypatch.setattr(eng.model, "forward", once)


@pytest.mark.parametrize("device", DEVICES)
def test_a_step_that_fails_is_not_one_to_commit(device, monkeypatch):
    eng = Engine(build(device), max_batch=1, max_seq_len=128, kv_keep=64, use_cuda_graph=False)
    joined(eng, prompt(10))
    failing(eng, monkeypatch, 2)
    step(eng, [True])
    with pytest.raises(RuntimeError, match="fails"):
        eng.decode_step()
    step(eng, [True])
    eng.decode_step()
    with pytest.raises(RuntimeError, match="committed"):
        eng.decode_step()


def test_a_server_goes_on_after_a_step_that_fails(monkeypatch):
    model = build()
    alone = Engine(model, max_batch=1, max_seq_len=128, kv_keep=64).generate([prompt(12, 1)], GREEDY, max_new_tokens=10)[0]
    server = Server(Engine(model, max_batch=2, max_seq_len=128, kv_keep=64))
    failing(server.engine, monkeypatch, 3)
    first = server.submit(prompt(10), GREEDY, 10)
    server.run_until_idle(max_steps=100)
    second = server.submit(prompt(12, 1), GREEDY, 10)
    server.run_until_idle(max_steps=100)
    assert server.result(first).failed and not server.result(second).failed and server.result(second).tokens == alone


def test_a_continuation_that_is_refused_changes_nothing():
    """No token is given up for a call that then raises."""
    eng = Engine(build(), max_batch=1, max_seq_len=256, kv_keep=KeptTokens(keep=32, recent=8, slack=16))
    seq = eng.new_sequence(prompt(40), GREEDY, max_new_tokens=100)
    eng.feed_logits(seq, prompt(40))
    before, pages = sums(eng, seq), list(seq.pages)
    with pytest.raises(ValueError):
        eng.feed_logits(seq, prompt(60, 2))
    assert seq.cached == seq.kv_len == 40 and seq.evicted == 0 and seq.pages == pages and torch.equal(sums(eng, seq), before)
    eng.feed_logits(seq, prompt(12, 3))                      # 32 + 12 find room
    assert seq.kv_len == 52 and seq.cached == 44


def test_single_tokens_of_many_sequences_stay_within_the_bound():
    """``forward_tokens`` of sequences with a reservation: the same logits as one by one, and no more pages than the bound has."""
    rule = KeptTokens(keep=32, recent=8, slack=8)
    logits, pages = [], []
    for together in (False, True):
        eng = Engine(build(), max_batch=2, max_seq_len=256, kv_keep=rule)
        seqs = [eng.new_sequence(prompt(n, n), GREEDY, max_new_tokens=100) for n in (50, 36)]
        for s in seqs:
            eng.feed_logits(s, s.prompt)
        rows = []
        for t in range(30):
            if together:
                rows.append(eng.forward_tokens([(s, [t + i], [0]) for i, s in enumerate(seqs)]))
            else:
                rows.append(torch.stack([eng.feed_logits(s, [t + i]) for i, s in enumerate(seqs)]))
        assert [s.kv_len for s in seqs] == [80, 66] and all(s.cached <= rule.limit for s in seqs)
        logits.append(torch.stack(rows))
        pages.append([len(s.pages) for s in seqs])
    assert pages == [[3, 3], [3, 3]]
    assert torch.allclose(*logits, rtol=1e-4, atol=1e-4)
