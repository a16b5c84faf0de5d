"""The engine over 8-bit pages, and sequences that are forked, moved and continued several times over pages of any kind."""
import dataclasses

import pytest
import torch
import torch.utils._python_dispatch

from eredu_b200 import ops
from eredu_b200.models import config as C
from eredu_b200.models.llama import build_from_tensors, random_state
from eredu_b200.ops import SamplingParams
from eredu_b200.runtime.engine import Engine
from eredu_b200.runtime.kv_cache import PAGE, PageAllocator, PagedKVCache

GREEDY = SamplingParams(temperature=0.0)
DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def build(device="cpu", seed=0, **change):
    cfg = dataclasses.replace(C.tiny_llama(), num_hidden_layers=2, vocab_size=512, **change)
    sd = random_state(cfg, seed=seed, std=0.08)
    return build_from_tensors(cfg, sd.__getitem__, sd.__contains__, device, torch.float32 if device == "cpu" else torch.bfloat16)


def prompt(n, seed=0):
    return torch.randint(0, 512, (n,), generator=torch.Generator().manual_seed(seed)).tolist()


def pages_of(eng, seq, li=0):
    """Codes and scales of the sequence's cached tokens."""
    at = torch.tensor(seq.pages, device=eng.device)
    k, v = eng.kv.layer(li)
    return [t[at] for t in (k.codes, k.scales, v.codes, v.scales)]


# ------------------------------------------------------------------------------------------ 8-bit pages
@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("change", [dict(), dict(qk_norm=True, model_type="qwen3"), dict(sliding_window=24, model_type="mistral"), dict(partial_rotary_factor=0.5)])
def test_logits_are_near_those_of_the_plain_cache(device, change):
    """A cached value is off by half a scale at most, 0.3 % to 0.5 % of the block's largest in the mean: a per cent or two of a typical one. What a wrong
    page, scale or position gives is off by the size of the logits themselves; a tenth of it lies between."""
    model = build(device, **change)
    for n in (1, 15, 16, 40, 131):
        got = []
        for bits in (None, 8):
            eng = Engine(model, max_batch=2, max_seq_len=192, kv_bits=bits)
            seq = eng.new_sequence(prompt(n), GREEDY, max_new_tokens=8)
            first = eng.feed_logits(seq, seq.prompt)
            got.append(torch.stack([first] + [eng.feed_logits(seq, [t]) for t in prompt(5, seed=7)]).float().cpu())
        assert torch.isfinite(got[1]).all()
        assert ((got[1] - got[0]).norm(dim=1) <= 0.1 * got[0].norm(dim=1)).all()


@pytest.mark.parametrize("device", DEVICES)
def test_portions_of_whole_pages_leave_what_one_prompt_leaves(device):
    model = build(device)
    held = []
    for limits in ((70,), (32, 16, 22)):
        eng = Engine(model, max_batch=1, max_seq_len=128, kv_bits=8)
        seq = eng.new_sequence(prompt(70), GREEDY, max_new_tokens=8)
        for n in limits:
            eng.prefill([seq], limits=[n])
        held.append(pages_of(eng, seq))
    # the first layer's rows come from the tokens alone
    for a, b in zip(*held):
        assert torch.equal(a[:5], b[:5]) if device == "cpu" else (a[:5].float() - b[:5].float()).abs().max() <= 1


@pytest.mark.parametrize("device", DEVICES)
def test_generation_over_8_bits(device):
    model = build(device)
    eng = Engine(model, max_batch=3, max_seq_len=96, kv_bits=8)
    prompts = [prompt(n, seed=n) for n in (5, 17, 33)]
    out = eng.generate(prompts, GREEDY, max_new_tokens=20)
    assert [len(o) for o in out] == [20] * 3
    assert eng.kv.bytes() < 0.6 * Engine(model, max_batch=3, max_seq_len=96).kv.bytes()
    if device == "cpu":
        assert [Engine(model, max_batch=1, max_seq_len=96, kv_bits=8).generate([p], GREEDY, max_new_tokens=20)[0] for p in prompts] == out
    else:
        assert Engine(model, max_batch=3, max_seq_len=96, kv_bits=8, use_cuda_graph=False).generate(prompts, GREEDY, max_new_tokens=20) == out


@pytest.mark.parametrize("device", DEVICES)
def test_prefix_reuse_over_8_bits(device):
    model = build(device)
    eng = Engine(model, max_batch=2, max_seq_len=128, kv_bits=8, prefix_cache=True)
    p = prompt(50)
    a = eng.generate([p], GREEDY, max_new_tokens=8)
    b = eng.generate([p], GREEDY, max_new_tokens=8)
    assert a == b and eng.prefix_stats["hit_tokens"] == 48


@pytest.mark.parametrize("device", DEVICES)
def test_drafts_are_verified_over_8_bits(device):
    """Every token kept is the target's own choice at its place, so a draft of the same weights is kept nearly always, and rows that were not are written again."""
    from eredu_b200.runtime.speculative import SpeculativeDecoder

    model = build(device)
    target, draft = (Engine(model, max_batch=1, max_seq_len=128, kv_bits=8) for _ in "td")
    out = SpeculativeDecoder(target, draft, k=3).generate([prompt(21)], GREEDY, max_new_tokens=24)[0]
    assert len(out) == 24
    other = SpeculativeDecoder(Engine(model, max_batch=1, max_seq_len=128, kv_bits=8), Engine(build(device, seed=9), max_batch=1, max_seq_len=128, kv_bits=8), k=3)
    assert len(other.generate([prompt(21)], GREEDY, max_new_tokens=24)[0]) == 24


@pytest.mark.parametrize("device", DEVICES)
def test_passes_of_a_speculative_round_state_their_portions(device, monkeypatch):
    """Ragged passes, of which every round has one, and the logits of a prompt: of the memory that a table of 32768 tokens would take they need what is there."""
    from eredu_b200.api import LoadedModel
    from eredu_b200.runtime.speculative import SpeculativeDecoder

    model = build(device)
    stated = []
    plain = ops.attention_prefill

    def attention_prefill(*args, portions=None, **more):
        lens, cu = args[4].tolist(), args[5].tolist()
        stated.append(portions is not None and [tuple(p) for p in portions] == [(n - (b - a), b - a) for n, a, b in zip(lens, cu, cu[1:])])
        return plain(*args, portions=portions, **more)

    monkeypatch.setattr(ops, "attention_prefill", attention_prefill)
    target, draft = (Engine(model, max_batch=2, max_seq_len=32768, num_pages=200, kv_bits=8) for _ in "td")
    dec = SpeculativeDecoder(target, draft, k=3)
    dec.generate([prompt(21), prompt(40, seed=1)], GREEDY, max_new_tokens=4)
    if device == "cuda":
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        before = torch.cuda.memory_allocated()
    assert [len(o) for o in dec.generate([prompt(21), prompt(40, seed=1)], GREEDY, max_new_tokens=12)] == [12, 12]
    lm = LoadedModel.__new__(LoadedModel)
    lm.engine, lm.model = target, model
    assert torch.isfinite(lm.prefill_logits(prompt(33))).all()
    assert stated and all(stated)
    if device == "cuda":
        # (2 sequences x 2048 pages x 8 KB would be 33 MB)
        assert torch.cuda.max_memory_allocated() - before <= 8 << 20


@pytest.mark.gpu
def test_a_long_sequence_beside_short_ones_takes_the_memory_of_one():
    """A pass over sequences of unequal lengths: keys and values in bf16 of what they see, 8 KB a page here, not as many times the longest as there are sequences."""
    model = build("cuda", num_attention_heads=4, num_key_value_heads=2, head_dim=64)
    eng = Engine(model, max_batch=16, max_seq_len=8192, num_pages=700, kv_bits=8)
    seqs = [eng.new_sequence(prompt(n, seed=n), GREEDY, max_new_tokens=8) for n in (8000, *range(20, 35))]
    eng.prefill(seqs[:1], limits=[7990])
    eng.prefill(seqs, limits=[2] + [len(s.prompt) - 3 for s in seqs[1:]])      # (so that nothing is set up for the first time below)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    eng.prefill(seqs)
    peak = torch.cuda.max_memory_allocated() - before
    seen = sum(-(-len(s.prompt) // PAGE) for s in seqs)
    assert 16 * 500 * 8192 > 60e6 and peak <= 2 * seen * 8192 + (8 << 20)


def test_what_does_not_take_8_bit_pages_says_so(tmp_path):
    from eredu_b200.runtime.kv_residency import KVHostTier
    from eredu_b200.runtime.prompt_cache import load_prompt_cache, save_prompt_cache

    eng = Engine(build(), max_batch=1, max_seq_len=64, kv_bits=8)
    seq = eng.new_sequence(prompt(20), GREEDY, max_new_tokens=4)
    eng.prefill([seq])
    for call in (lambda: save_prompt_cache(eng, seq, tmp_path, "f"), lambda: load_prompt_cache(eng, tmp_path, prompt(20), "f"),
                 lambda: KVHostTier(eng),
                 lambda: Engine(build(), max_seq_len=64, kv_bits=8, prefix_cache=True, kv_host_tier_bytes=1 << 20)):
        with pytest.raises(NotImplementedError, match="8-bit pages"):
            call()
    with pytest.raises(ValueError, match="kv_bits"):
        PagedKVCache(1, 1, 64, 4, torch.float32, "cpu", kv_bits=4)
    with pytest.raises(NotImplementedError, match="one width"):
        PagedKVCache(1, 1, 64, 4, torch.float32, "cpu", kv_bits=8, value_dim=32)
    model = build()
    model.cfg = dataclasses.replace(model.cfg, kv_lora_rank=32)
    if model.cfg.is_mla:
        with pytest.raises(NotImplementedError, match="does not take 8-bit pages"):
            Engine(model, max_seq_len=64, kv_bits=8)


@pytest.mark.gpu
def test_head_sizes_without_kernels_are_refused():
    with pytest.raises(NotImplementedError, match="head sizes"):
        Engine(build("cuda", head_dim=32), max_seq_len=64, kv_bits=8)


# ------------------------------------------------------------------------------------------ forks
@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("bits", [None, 8])
@pytest.mark.parametrize("n", [1, 16, 37])
def test_a_forked_sequence_goes_its_own_way(device, bits, n):
    model = build(device)
    eng = Engine(model, max_batch=2, max_seq_len=128, kv_bits=bits)
    seq = eng.new_sequence(prompt(n), GREEDY, max_new_tokens=40)
    eng.feed_logits(seq, seq.prompt)
    free = eng.kv.allocator.free_pages()
    other = eng.fork(seq)
    shared = n // PAGE
    assert other.pages[:shared] == seq.pages[:shared] and not set(other.pages[shared:]) & set(seq.pages) and len(other.pages) == len(seq.pages)
    assert eng.kv.allocator.free_pages() == free - (len(seq.pages) - shared)
    mine, theirs = prompt(20, seed=3), prompt(20, seed=4)
    got = [(eng.feed_logits(seq, [a]).clone(), eng.feed_logits(other, [b]).clone()) for a, b in zip(mine, theirs)]
    for tokens, column in ((mine, 0), (theirs, 1)):
        solo = Engine(model, max_batch=2, max_seq_len=128, kv_bits=bits)
        s = solo.new_sequence(prompt(n), GREEDY, max_new_tokens=40)
        solo.feed_logits(s, s.prompt)
        for i, t in enumerate(tokens):
            assert torch.equal(solo.feed_logits(s, [t]), got[i][column])
    for s in (seq, other):
        eng.release(s)
    assert eng.kv.allocator.free_pages() == eng.kv.num_pages - 1


@pytest.mark.parametrize("device", DEVICES)
def test_several_continuations_of_a_prompt(device):
    model = build(device)
    prompts = [prompt(n, seed=n) for n in (1, 16, 21)]
    plain = Engine(model, max_batch=6, max_seq_len=64).generate([p for p in prompts for _ in range(2)], GREEDY, max_new_tokens=12)
    eng = Engine(model, max_batch=6, max_seq_len=64)
    out = eng.generate(prompts, GREEDY, max_new_tokens=12, samples=2)
    assert [len(o) for o in out] == [12] * 6 and eng.kv.allocator.free_pages() == eng.kv.num_pages - 1
    assert out[0::2] == out[1::2]
    if device == "cpu":
        assert out == plain
    hot = SamplingParams(temperature=1.0, seed=3)
    drawn = eng.generate(prompts[2:], hot, max_new_tokens=12, samples=4)
    assert len({tuple(o) for o in drawn}) > 1
    hist = eng.generate(prompts[2:], dataclasses.replace(hot, repeat_penalty=1.2), max_new_tokens=6, samples=2, eos_ids=(5,))
    assert all(1 <= len(o) <= 6 for o in hist)


def test_forks_and_continuations_that_are_refused():
    eng = Engine(build(), max_batch=2, max_seq_len=64)
    with pytest.raises(ValueError, match="continuations"):
        eng.generate([prompt(4)], GREEDY, samples=0)
    seq = eng.new_sequence(prompt(20), GREEDY, max_new_tokens=4)
    eng.prefill([seq])
    pages, seq.pages = seq.pages, []                 # as a parked sequence has none
    with pytest.raises(RuntimeError, match="parked"):
        eng.fork(seq)
    seq.pages = pages
    small = Engine(build(), max_batch=1, max_seq_len=64, num_pages=4)
    s = small.new_sequence(prompt(20), GREEDY, max_new_tokens=4)
    small.prefill([s])
    free = small.kv.allocator.free_pages()
    big = small.fork(s)                              # one page more
    with pytest.raises(RuntimeError, match="exhausted"):
        small.fork(s)
    assert small.kv.allocator.free_pages() == free - 1 and small.kv.allocator.refcount(s.pages[0]) == 2
    small.release(big)


def test_hybrid_models_fork_their_states():
    from test_lfm2 import lfm2_cfg           # a model with convolution states, found by a sequence's first page

    cfg = lfm2_cfg()
    sd = random_state(cfg, seed=1, std=0.08)
    model = build_from_tensors(cfg, sd.__getitem__, sd.__contains__, "cpu", torch.float32)
    eng = Engine(model, max_batch=2, max_seq_len=64)
    seq = eng.new_sequence(list(range(1, 20)), GREEDY, max_new_tokens=20)
    eng.feed_logits(seq, seq.prompt)
    other = eng.fork(seq)
    assert not set(other.pages) & set(seq.pages)
    a = [eng.feed_logits(seq, [t]).clone() for t in (3, 4, 5)]
    b = [eng.feed_logits(other, [t]).clone() for t in (3, 4, 5)]
    assert all(torch.equal(x, y) for x, y in zip(a, b))


# ------------------------------------------------------------------------------------------ moved pages
@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("bits", [None, 8])
def test_compaction_under_a_decode_state(device, bits):
    """Sequences leave, the others' pages move to the front between two steps of a batch (captured, on a GPU), and the tokens are those of an engine that
    has never moved any."""
    model = build(device)
    prompts = [prompt(n, seed=n) for n in (40, 17, 33, 64)]

    def run(move):
        eng = Engine(model, max_batch=4, max_seq_len=128, kv_bits=bits, prefix_cache=True)
        seqs = [eng.new_sequence(p, GREEDY, max_new_tokens=30) for p in prompts]
        eng.prefill(seqs)
        for s in (seqs[0], seqs[2]):
            eng.release(s)
        left = [seqs[1], seqs[3]]
        eng.start_decode(left, torch.tensor([7, 8], dtype=torch.int32))
        for i in range(12):
            if move and i in (3, 8):
                if i == 8:          # a stranger comes and goes in between
                    eng.release(eng.new_sequence(prompt(20, seed=99), GREEDY, max_new_tokens=4))
                before = [list(s.pages) for s in left]
                moved = eng.compact(left)
                assert moved > 0 if i == 3 else moved >= 0
                assert i != 3 or before != [s.pages for s in left]
                live = len(eng.kv.allocator.held()) + eng.kv.allocator.cached_pages()
                assert max(p for s in left for p in s.pages) <= live
            eng.commit(eng.decode_step().tolist())
        out = [list(s.output) for s in left]
        # a published prefix is found where it has moved to
        again = eng.new_sequence(prompts[0], GREEDY, max_new_tokens=4)
        assert again.cached_tokens == 32
        logits = eng.feed_logits(again, again.prompt[32:])
        return out, logits.clone()

    (a, x), (b, y) = run(False), run(True)
    assert a == b and torch.equal(x, y)


@pytest.mark.parametrize("bits", [None, 8])
def test_the_pool_changes_its_size(bits):
    model = build()
    eng = Engine(model, max_batch=4, max_seq_len=64, kv_bits=bits)
    seqs = [eng.new_sequence(prompt(20, seed=i), GREEDY, max_new_tokens=20) for i in range(4)]
    for s in seqs:
        eng.feed_logits(s, s.prompt)
    eng.release(seqs[0])
    eng.release(seqs[2])
    twin = Engine(model, max_batch=4, max_seq_len=64, kv_bits=bits)
    t = twin.new_sequence(seqs[3].prompt, GREEDY, max_new_tokens=20)
    twin.feed_logits(t, t.prompt)
    with pytest.raises(ValueError, match="held by none"):
        eng.resize_cache(8, [seqs[1]])
    size = eng.kv.bytes()
    eng.resize_cache(8, [seqs[1], seqs[3]])
    assert eng.kv.num_pages == 8 and eng.kv.bytes() < size and sorted(seqs[1].pages + seqs[3].pages) == [1, 2, 3, 4, 5, 6]
    assert torch.equal(eng.feed_logits(seqs[3], [5]), twin.feed_logits(t, [5]))
    with pytest.raises(Exception, match="contents|pages"):
        eng.resize_cache(4, [seqs[1], seqs[3]])
    eng.resize_cache(40, [seqs[1], seqs[3]])
    assert torch.equal(eng.feed_logits(seqs[3], [6]), twin.feed_logits(t, [6])) and eng.kv.allocator.free_pages() == 33
    eng.start_decode([seqs[1]], torch.tensor([1], dtype=torch.int32))
    with pytest.raises(RuntimeError, match="decode state"):
        eng.resize_cache(50, [seqs[1], seqs[3]])


class Failing(torch.utils._python_dispatch.TorchDispatchMode):
    """The n-th new tensor of the pool's shapes cannot be had."""

    def __init__(self, n, pages):
        super().__init__()
        self.left, self.pages, self.seen = n, pages, []

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        name = func.overloadpacket.__name__
        out = func(*args, **(kwargs or {}))
        if (name.startswith("new_") or name in ("empty", "zeros", "full", "clone")) and torch.is_tensor(out) and self.pages in out.shape:
            self.left -= 1
            self.seen.append(name)
            if self.left < 0:
                raise torch.OutOfMemoryError("no memory left")
        return out


@pytest.mark.parametrize("bits", [None, 8])
@pytest.mark.parametrize("pages", [9, 41])
@pytest.mark.parametrize("hybrid", [False, True])
def test_a_pool_that_cannot_change_its_size_goes_on(bits, pages, hybrid):
    """Whichever of the new tensors cannot be had: every tensor has the pages that the allocator gives, contents are what they were, and the next attempt succeeds."""
    if hybrid:
        from test_lfm2 import lfm2_cfg

        cfg = lfm2_cfg(vocab_size=512)
        sd = random_state(cfg, seed=1, std=0.08)
        model = build_from_tensors(cfg, sd.__getitem__, sd.__contains__, "cpu", torch.float32)
    else:
        model = build()
    twin = Engine(model, max_batch=4, max_seq_len=64, kv_bits=bits)
    t = twin.new_sequence(prompt(20), GREEDY, max_new_tokens=20)
    twin.feed_logits(t, t.prompt)
    want = [twin.feed_logits(t, [x]).clone() for x in (5, 6)]
    want.append(twin.feed_logits(twin.new_sequence(prompt(20), GREEDY, max_new_tokens=20), prompt(20) + [5]).clone())
    for n in range(20):
        eng = Engine(model, max_batch=4, max_seq_len=64, kv_bits=bits)
        gone = eng.new_sequence(prompt(30), GREEDY, max_new_tokens=20)
        seq = eng.new_sequence(prompt(20), GREEDY, max_new_tokens=20)
        eng.feed_logits(seq, seq.prompt)
        eng.release(gone)
        try:
            with Failing(n, pages):
                eng.resize_cache(pages, [seq])
            failed = False
        except torch.OutOfMemoryError:
            failed = True
        kv = eng.kv

        def consistent():
            assert all(x.shape[1] == kv.num_pages for x in kv.page_tensors() + ([] if kv.conv_state is None else [kv.conv_state]))
            assert kv.k is kv.pools[0][0] and kv.v is kv.pools[0][1]
            assert len(kv.allocator.held()) + kv.allocator.free_pages() == kv.num_pages - 1
            taken = kv.allocator.alloc(kv.allocator.free_pages())
            assert max(taken) < kv.num_pages
            kv.allocator.release(taken)

        consistent()
        assert kv.num_pages in ((pages,) if not failed else (17, min(17, pages)))
        assert torch.equal(eng.feed_logits(seq, [5]), want[0])
        eng.resize_cache(pages, [seq])
        consistent()
        assert kv.num_pages == pages and torch.equal(eng.feed_logits(seq, [6]), want[1])
        last = eng.new_sequence(prompt(20), GREEDY, max_new_tokens=20)
        assert torch.equal(eng.feed_logits(last, last.prompt + [5]), want[2])
        if not failed:
            break
    assert not failed and n == (2 if bits is None else 4) + hybrid


def test_new_pages_of_a_pool_are_those_of_a_new_pool():
    """And no more than one tensor of the pool is there twice at a time."""
    import weakref

    kv = PagedKVCache(2, 3, 64, 6, torch.float32, "cpu", kv_bits=8)
    old = [weakref.ref(t) for t in kv.pools[0]]
    alive = []

    class Watched(Failing):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            before = len(self.seen)
            out = super().__torch_dispatch__(func, types, args, kwargs)
            if len(self.seen) > before:
                alive.append(sum(ref() is not None for ref in old))
            return out

    with Watched(99, 11):
        kv.resize(11)
    assert alive[:2] == [2, 1] and alive[-1] == 0
    assert kv.scales[0][0].shape == (2, 11, 3) and all((s == 2.0 ** -100).all() for s in kv.scales[0])
    assert not kv.k.any() and not kv.v.any()


def test_scales_of_new_pages_are_those_of_a_new_pool():
    """A block that nobody has opened has the smallest scale there is."""
    kv = PagedKVCache(2, 3, 64, 6, torch.float32, "cpu", kv_bits=8)
    kv.scales[0][0][:, 2] = 0.5
    kv.resize(11)
    assert (kv.scales[0][0][:, 2] == 0.5).all() and (kv.scales[0][0][:, 3:] == 2.0 ** -100).all() and (kv.scales[0][1] == 2.0 ** -100).all()


def allocators(n):
    from eredu_b200.lib import _eredu_host

    return [PageAllocator(n), _eredu_host.BlockManager(n)]


@pytest.mark.parametrize("which", [0, 1])
def test_allocators_rename_pages(which):
    al = allocators(20)[which]
    a, b, c = al.alloc(5), al.alloc(4), al.alloc(3)
    al.release(a)
    assert al.held() == sorted(b + c)
    moves = dict(al.compact())
    assert len(moves) == 5 and not set(moves) & set(moves.values())
    b, c = ([moves.get(p, p) for p in x] for x in (b, c))
    assert sorted(b + c) == list(range(1, 8)) == al.held()
    assert al.alloc(1) == [8]
    al.resize(12)
    assert al.free_pages() == 3 and len(al.alloc(3)) == 3
    with pytest.raises(Exception):
        al.alloc(1)
    al.release(b)
    with pytest.raises(Exception):
        al.resize(5)
    assert al.compact() and al.held() == list(range(1, 8))


def test_published_pages_move_with_their_names():
    al = allocators(16)[1]
    first, second = al.alloc(4), al.alloc(3)
    tokens = list(range(48))
    al.seal_prefix(second, tokens)
    al.release(first)
    al.release(second)                       # published, held by nobody
    moves = dict(al.compact())
    assert al.match_prefix(tokens) == [moves.get(p, p) for p in second] and al.cached_pages() == 0
    assert all(al.refcount(moves.get(p, p)) == 1 for p in second)


def test_page_0_is_not_copied():
    kv = PagedKVCache(2, 1, 8, 6, torch.float32, "cpu")
    for src, dst in (([0], [1]), ([1], [0])):
        with pytest.raises(IndexError):
            kv.copy_pages(src, dst)
