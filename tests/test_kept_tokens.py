"""The engine with caches of bounded size: tokens that attention gives the least weight are given up."""
import dataclasses

import pytest
import torch

from eredu_b200 import ops
from eredu_b200.models import config as C
from eredu_b200.models.llama import build_from_tensors, random_state
from eredu_b200.ops import SamplingParams
from eredu_b200.runtime.engine import Engine
from eredu_b200.runtime.kv_cache import PAGE, KeptTokens
from eredu_b200.runtime.server import Server
from eredu_b200.runtime.speculative import SpeculativeDecoder

GREEDY = SamplingParams(temperature=0.0)
DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def build(device="cpu", **change):
    cfg = dataclasses.replace(C.tiny_llama(), num_hidden_layers=2, vocab_size=512, **change)
    sd = random_state(cfg, seed=0, std=0.08)
    return build_from_tensors(cfg, sd.__getitem__, sd.__contains__, device, torch.float32 if device == "cpu" else torch.bfloat16)


def prompt(n, seed=0):
    return torch.randint(0, 512, (n,), generator=torch.Generator().manual_seed(seed)).tolist()


def record(monkeypatch):
    """(lengths, keep) of every eviction."""
    calls, evict = [], ops.evict_tokens

    def spy(k, v, w, table, lens, keep, **more):
        calls.append((lens.tolist(), keep))
        return evict(k, v, w, table, lens, keep, **more)

    monkeypatch.setattr(ops, "evict_tokens", spy)
    return calls


@pytest.mark.parametrize("device", DEVICES)
def test_what_is_never_reached_changes_nothing(device):
    """A bound above the whole conversation: the same tokens as without one."""
    model = build(device)
    prompts = [prompt(40), prompt(7, 1)]
    plain = Engine(model, max_batch=2, max_seq_len=128).generate(prompts, GREEDY, max_new_tokens=20)
    if device == "cpu":
        assert Engine(model, max_batch=2, max_seq_len=128, kv_keep=100).generate(prompts, GREEDY, max_new_tokens=20) == plain
    else:
        # (two kernels round differently: the logits of the same steps are near one another)
        logits = []
        for keep in (None, 100):
            eng = Engine(model, max_batch=2, max_seq_len=128, kv_keep=keep)
            seq = eng.new_sequence(prompts[0], GREEDY, max_new_tokens=20)
            logits.append(torch.stack([eng.feed_logits(seq, prompts[0])] + [eng.feed_logits(seq, [t]) for t in plain[0]]).float())
        assert ((logits[0] - logits[1]).norm(dim=1) <= 0.02 * logits[0].norm(dim=1)).all()


@pytest.mark.parametrize("device", DEVICES)
def test_sequences_are_cut_down_behind_the_prompt_and_while_decoding(device, monkeypatch):
    model = build(device)
    calls = record(monkeypatch)
    eng = Engine(model, max_batch=3, max_seq_len=256, kv_keep=KeptTokens(keep=40, recent=10, first=2, slack=6))
    free = eng.kv.allocator.free_pages()
    out = eng.generate([prompt(100), prompt(30, 1), prompt(45, 2)], GREEDY, max_new_tokens=30)
    assert [len(o) for o in out] == [30, 30, 30] and eng.kv.allocator.free_pages() == free
    # behind the prompt the long one alone; then each as soon as one more token would be the 47th: from 40 every seventh step, from 45 and 30 first the 2nd and the 17th
    assert calls[0] == ([100], 40)
    steps = [lens for lens, _ in calls[1:]]
    assert all(set(lens) == {46} for lens in steps)
    grown = [40, 30, 45]
    expect = []
    for _ in range(29):
        full = [i for i in range(3) if grown[i] == 46]
        if full:
            expect.append([46] * len(full))
        grown = [40 if i in full else grown[i] for i in range(3)]
        grown = [n + 1 for n in grown]
    assert steps == expect


def kept_logits(eng, seq, tokens):
    return torch.stack([eng.feed_logits(seq, [t]) for t in tokens]).float().cpu()


@pytest.mark.parametrize("device", DEVICES)
def test_tokens_that_are_left_are_seen_as_they_were(device):
    """An engine that gave tokens up, against attention over the whole context from which those tokens are hidden: keys keep their rotation, positions go on."""
    model = build(device)
    rule = KeptTokens(keep=24, recent=8, first=2, slack=100)
    eng, whole = (Engine(model, max_batch=1, max_seq_len=192, kv_keep=k) for k in (rule, KeptTokens(keep=180)))
    text, more = prompt(90), prompt(6, 3)
    seqs = [e.new_sequence(text, GREEDY, max_new_tokens=60) for e in (eng, whole)]
    for e, s in zip((eng, whole), seqs):
        e.feed_logits(s, text)
    # the bound is put to use here, on pages whose weights both engines have
    for (w,), (other,) in zip(eng.kv.weights, whole.kv.weights):
        a, b = (x[:, torch.tensor(s.pages[:6], device=x.device)].transpose(1, 2).flatten(2)[..., :90] for x, s in ((w, seqs[0]), (other, seqs[1])))
        assert torch.equal(a, b)
    stays = []
    k_all = whole.kv.pools[0][0][:, torch.tensor(seqs[1].pages, device=eng.device)].transpose(1, 2).flatten(2, 3)
    eng.keep = dataclasses.replace(rule, slack=1)
    eng._shrink([seqs[0]])
    assert seqs[0].cached == 24 and seqs[0].kv_len == 90 and len(seqs[0].pages) == 2
    k_left = eng.kv.pools[0][0][:, torch.tensor(seqs[0].pages, device=eng.device)].transpose(1, 2).flatten(2, 3)[:, :, :24]
    for layer in range(2):
        stays.append([])
        for h in range(k_left.shape[1]):
            at = [int((k_all[layer, h, :90] == row).all(1).nonzero()[0]) for row in k_left[layer, h]]
            assert at == sorted(at) and at[:2] == [0, 1] and at[-8:] == list(range(82, 90))
            stays[-1].append(at)
    # the whole context with everything else hidden: keys far from all queries, values of zero (each layer and head its own)
    hidden = whole.kv.pools[0]
    for layer in range(2):
        for h, at in enumerate(stays[layer]):
            gone = torch.tensor([t for t in range(90) if t not in at], device=eng.device)
            page = torch.tensor(seqs[1].pages, device=eng.device)[gone // PAGE]
            hidden[1][layer][page, h, gone % PAGE] = 0
    # (values of zero still take their share of the sum: compare attention itself, layer 0, where queries are the same)
    q = torch.randn((1, model.n_q_local, model.cfg.head_dim), generator=torch.Generator().manual_seed(5)).to(hidden[0].dtype).to(eng.device)
    got = ops.attention_decode(q, eng.kv.pools[0][0][0], eng.kv.pools[0][1][0], eng._block_table([seqs[0]]), eng._t([24], torch.int32), 1, 0.3,
                               weights=eng.kv.weights[0][0][0].clone())
    k, v = (x[0, torch.tensor(seqs[1].pages, device=eng.device)].transpose(0, 1).flatten(1, 2).double() for x in hidden)
    group = model.n_q_local // model.n_kv_local
    want = torch.stack([torch.softmax(q[0, i].double() @ k[i // group][stays[0][i // group]].t() * 0.3, 0) @ v[i // group][stays[0][i // group]]
                        for i in range(model.n_q_local)])
    assert (got[0].double() - want).abs().max() <= 2.0 ** -6 * want.abs().max()
    eng.keep = rule
    assert torch.isfinite(kept_logits(eng, seqs[0], more)).all() and seqs[0].kv_len == 96 and seqs[0].cached == 30


@pytest.mark.parametrize("device", DEVICES)
def test_slots_join_and_leave(device):
    """Continuous batching gives the tokens that a batch of its own gives: places and positions are the sequence's."""
    model = build(device)
    rule = KeptTokens(keep=32, recent=16, slack=5)
    alone = []
    for i, n in enumerate((70, 9)):
        eng = Engine(model, max_batch=1, max_seq_len=256, kv_keep=rule)
        alone.append(eng.generate([prompt(n, i)], GREEDY, max_new_tokens=40)[0])
    eng = Engine(model, max_batch=2, max_seq_len=256, kv_keep=rule)
    eng.open_decode()
    seqs = []
    for step in range(60):
        if step in (0, 6):
            s = eng.new_sequence(prompt((70, 9)[len(seqs)], len(seqs)), GREEDY, max_new_tokens=40)
            s.output.append(int(eng.prefill([s])[0]))
            eng.join(s, s.output[-1])
            seqs.append(s)
        eng.set_step_mask([s is not None for s in eng._decode_state["seqs"]])
        for s, fin in zip(list(eng._decode_state["seqs"]), eng.commit(eng.decode_step().tolist())):
            if fin:
                eng.leave(s)
        if len(seqs) == 2 and all(s.finished for s in seqs):
            break
    if device == "cpu":
        assert [s.output for s in seqs] == alone
    else:      # (batches of other sizes take other kernels: the first tokens, which nothing near a tie has touched)
        assert [s.output[:3] for s in seqs] == [o[:3] for o in alone] and all(len(s.output) == 40 for s in seqs)


def test_continuations_of_a_prompt_have_pages_of_their_own():
    """A fork shares no page with what an eviction changes in place."""
    model = build()
    rule = KeptTokens(keep=32, recent=8, slack=4)
    eng = Engine(model, max_batch=3, max_seq_len=256, kv_keep=rule)
    out = eng.generate([prompt(100)], GREEDY, max_new_tokens=24, samples=3)
    assert out[0] == out[1] == out[2] and len(out[0]) == 24


def test_a_server_gives_what_a_batch_gives():
    """Prompts in portions between other requests' steps, each with its own evictions."""
    model = build()
    rule = KeptTokens(keep=32, recent=12, slack=6)
    prompts = [prompt(n, i) for i, n in enumerate((70, 9, 45))]
    alone = [Engine(model, max_batch=1, max_seq_len=256, kv_keep=rule).generate([p], GREEDY, max_new_tokens=30)[0] for p in prompts]
    server = Server(Engine(model, max_batch=2, max_seq_len=256, kv_keep=rule), prefill_chunk=16, max_step_tokens=40)
    ids = [server.submit(p, GREEDY, 30) for p in prompts]
    server.run_until_idle(max_steps=400)
    assert [server.result(i).tokens for i in ids] == alone


def test_command_line(tmp_path, capsys):
    from eredu_b200.cli.main import build_parser, main, validate_args
    from eredu_b200.formats import checkpoint
    from test_text_streaming import make_bundle

    for bad in (["--kv-keep", "0"], ["--kv-keep", "64", "--kv-bits", "8"]):
        with pytest.raises(SystemExit):
            validate_args(build_parser().parse_args(["-m", "x", "hi", *bad]))
    bundle = make_bundle(tmp_path)
    cfg = dataclasses.replace(C.tiny_llama(), vocab_size=bundle.vocab_size(), eos_token_id=bundle.eos_ids[0])
    checkpoint.save_safetensors_checkpoint(tmp_path, cfg, random_state(cfg, seed=0, std=0.05), torch.float32)
    assert main(["-m", str(tmp_path), "hello", "--device", "cpu", "-n", "40", "--kv-keep", "6"]) == 0
    assert capsys.readouterr().out


def test_bounds_are_checked():
    for wrong in (dict(keep=0), dict(keep=8, recent=6, first=4), dict(keep=8, slack=0), dict(keep=8, recent=-1), dict(keep=20, observed=-1)):
        with pytest.raises(ValueError):
            KeptTokens(**wrong)
    assert KeptTokens(1).first == 1 and KeptTokens(6).first == 3 and KeptTokens(64).recent == 32 and KeptTokens(64).limit == 80 and KeptTokens(1024).slack == 64


def test_what_does_not_go_with_a_bound_is_refused():
    model = build()
    for other in (dict(kv_bits=8), dict(prefix_cache=True)):
        with pytest.raises(NotImplementedError):
            Engine(model, max_seq_len=64, kv_keep=32, **other)
    with pytest.raises(NotImplementedError):
        Engine(build(sliding_window=24, model_type="mistral"), max_seq_len=64, kv_keep=32)
    eng = Engine(model, max_batch=1, max_seq_len=256, kv_keep=32)
    with pytest.raises(NotImplementedError):
        eng.open_sequence()
    with pytest.raises(NotImplementedError):
        SpeculativeDecoder(eng, Engine(model, max_batch=1, max_seq_len=256))
    from eredu_b200.runtime.kv_residency import KVHostTier

    with pytest.raises(NotImplementedError):
        KVHostTier(eng)
    seq = eng.new_sequence(prompt(20), GREEDY, max_new_tokens=100)
    eng.feed_logits(seq, prompt(20))
    with pytest.raises(ValueError):
        eng.feed_logits(seq, prompt(60, 2))


def test_steps_are_committed_one_by_one():
    eng = Engine(build(), max_batch=1, max_seq_len=128, kv_keep=64)
    s = eng.new_sequence(prompt(10), GREEDY, max_new_tokens=8)
    eng.start_decode([s], eng.prefill([s]))
    eng.decode_step()
    with pytest.raises(RuntimeError):
        eng.decode_step()
    eng.commit([1])
    eng.decode_step()


def test_pools_that_move_and_grow_keep_the_weights():
    model = build()
    eng = Engine(model, max_batch=2, max_seq_len=128, kv_keep=64)
    a, b = (eng.new_sequence(prompt(40, i), GREEDY, max_new_tokens=8) for i in range(2))
    for s in (a, b):
        eng.feed_logits(s, s.prompt)
    held = [w[:, b.pages].clone() for w, in eng.kv.weights]
    eng.release(a)
    eng.resize_cache(40, [b])
    assert all(torch.equal(w[:, b.pages], h) for (w,), h in zip(eng.kv.weights, held)) and eng.kv.weights[0][0].shape[1] == 40
    assert eng.kv.bytes() > sum(k.numel() + v.numel() for k, v in eng.kv.pools) * 4
