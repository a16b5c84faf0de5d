"""Calls of attention with weights that are rare: other devices' limits, odd windows, scales and lengths, and what must not be touched."""
import pytest
import torch

from eredu_b200 import ops
from eredu_b200.ops import eviction
from test_eviction import arguments, attended, cache, compare, layout

PAGE = eviction.PAGE


def packed(monkeypatch, cluster, sms=148):
    """Arguments of the decode kernel as the host packs them, on a device whose largest cluster is ``cluster``; nothing is launched."""
    calls = []

    class Lib:
        @staticmethod
        def eredu_weighed_decode(block, size):
            names = ("q", "k", "v", "out", "table", "lens", "sinks", "weights", "scores", "part_o", "part_ml", "status", "stream", "batch", "q_per_seq", "pitch",
                     "max_tokens", "room", "pages", "n_q", "n_kv", "D", "splits", "window", "scale")
            calls.append(dict(zip(names, eviction._DECODE.unpack(block))))
            return 0

    monkeypatch.setattr(eviction, "lib", Lib)
    monkeypatch.setattr(eviction, "_device", lambda device: (sms, cluster))
    monkeypatch.setattr(eviction, "_kernels_take", lambda *a: True)
    monkeypatch.setattr(eviction, "status_word", lambda device: torch.zeros(1, dtype=torch.int32))
    monkeypatch.setattr(eviction, "stream_ptr", lambda device: 0)
    return calls


# ------------------------------------------------------------------------------------------ clusters
@pytest.mark.parametrize("cluster", [8, 16])
def test_splits_are_a_cluster_that_the_device_has_room_for_or_leave_parts(monkeypatch, cluster):
    """More splits than the device's largest cluster leave their parts in memory, whatever their number."""
    calls = packed(monkeypatch, cluster)
    seen = set()
    for heads in range(1, 41):
        for pages in (64, 1024, 4096):
            k = torch.empty((1, heads, PAGE, 64), dtype=torch.bfloat16)
            table = torch.zeros((1, pages), dtype=torch.int32)
            q = torch.empty((1, heads, 64), dtype=torch.bfloat16)
            ops.attention_decode(q, k, k, table, torch.tensor([pages * PAGE], dtype=torch.int32), 1, 0.1, weights=torch.empty((1, heads, PAGE)))
            call = calls.pop()
            joined = call["splits"] > cluster
            assert (call["part_o"] != 0) == (call["part_ml"] != 0) == joined and (call["scores"] != 0 or not joined)
            seen.add(call["splits"])
    assert any(s > cluster for s in seen) and any(1 < s <= cluster for s in seen)


@pytest.mark.gpu
@pytest.mark.parametrize("heads, lens, new", [((14, 14, 64), [16500], 1), ((24, 12, 128), [16400], 3), ((16, 8, 128), [700, 40], 1)])
def test_step_on_a_device_without_large_clusters(monkeypatch, heads, lens, new):
    monkeypatch.setattr(eviction, "_device", lambda device: (148, 8))
    n_q, n_kv, dim = heads
    num, table = layout(lens, "cuda", wider=2)
    k, v, w = cache(num, n_kv, dim, "cuda")
    q = torch.randn((len(lens) * new, n_q, dim), generator=torch.Generator().manual_seed(1)).bfloat16().cuda()
    before, scale = w.clone(), dim ** -0.5
    out = ops.attention_decode(q, k, v, table, torch.tensor(lens, dtype=torch.int32, device="cuda"), new, scale, weights=w, max_kv_len=max(lens))
    expect = attended(q, k, v, table, lens, [new] * len(lens), scale)
    compare(out, w, before, expect, dim, new * n_q // n_kv, True)
    ops.native.check_status(torch.device("cuda", 0))


@pytest.mark.gpu
def test_asking_for_clusters_leaves_the_kernels_as_they_are():
    """The question may come behind launches (two threads' first calls): those with scores in shared memory, which take the most of it, go on."""
    num, table = layout([500], "cuda")
    k, v, w = cache(num, 1, 128, "cuda")
    q = torch.randn((1, 16, 128), generator=torch.Generator().manual_seed(2)).bfloat16().cuda()
    lens = torch.tensor([500], dtype=torch.int32, device="cuda")
    outs = []
    for _ in range(2):
        own = w.clone()
        outs.append((ops.attention_decode(q, k, v, table, lens, 1, 0.1, weights=own, max_kv_len=500), own))
        assert ops.native.lib().eredu_weighed_clusters() in (0, 1)
    assert all(torch.equal(a, b) for a, b in zip(*outs))


# ------------------------------------------------------------------------------------------ windows
WIDE = [2 ** 31 - 1, 2 ** 31 - 200, 2 ** 31, 2 ** 40]


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("window", WIDE)
@pytest.mark.parametrize("new", [1, 40])
def test_a_window_wider_than_any_sequence_hides_nothing(device, window, new):
    """Some configurations write "none" so. Steps, steps of so many rows that they go to the prompt's kernels, and prompts: bit by bit what no window gives."""
    lens = [300, 50]
    num, table = layout(lens, device)
    k, v, w = cache(num, 2, 64, device)
    q = torch.randn((2 * new, 8, 64), generator=torch.Generator().manual_seed(3)).bfloat16().to(device)
    at = torch.tensor(lens, dtype=torch.int32, device=device)
    cu = torch.tensor([0, new, 2 * new], dtype=torch.int32, device=device)
    for call in (lambda w, window: ops.attention_decode(q, k, v, table, at, new, 0.125, window=window, weights=w, max_kv_len=300),
                 lambda w, window: ops.attention_prefill(q, k, v, table, at, cu, new, 0.125, window=window, weights=w, max_kv_len=300),
                 lambda w, window: ops.attention_prefill(q, k, v, table, at, cu, new, 0.125, window=window, weights=w, observed=3)):
        got = []
        for hide in (0, window):
            own = w.clone()
            got.append((call(own, hide), own))
        assert all(torch.equal(a, b) for a, b in zip(*got))


def test_windows_that_the_kernels_are_given_are_narrower_than_the_table(monkeypatch):
    """Sums of a position and a window then stay within 32 bits."""
    calls = packed(monkeypatch, 16)
    prompts = []
    monkeypatch.setattr(eviction.lib, "eredu_weighed_prefill", staticmethod(lambda block, size: prompts.append(eviction._PROMPT.unpack(block)) or 0), raising=False)
    q, k, v, w, table, lens = arguments()
    for window in (0, 5, 31, 32, 33, *WIDE):
        ops.attention_decode(q, k, v, table, lens, 1, 0.1, window=window, weights=w)
        ops.attention_prefill(q, k, v, table, lens, torch.tensor([0, 1, 2], dtype=torch.int32), 1, 0.1, window=window, weights=w)
        want = window if window < 32 else 0
        assert calls.pop()["window"] == want and prompts.pop()[12 + 9] == want


# ------------------------------------------------------------------------------------------ scales
@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("scale", [-0.125, 0.0, -0.0])
@pytest.mark.parametrize("new", [3, 40])
def test_scales_of_zero_and_below(device, scale, new):
    """What the decode form takes is taken with any number of rows, and by the prompt form."""
    lens, dim = [200, 41], 64
    num, table = layout(lens, device)
    k, v, w = cache(num, 2, dim, device)
    q = torch.randn((2 * new, 8, dim), generator=torch.Generator().manual_seed(4)).bfloat16().to(device)
    at = torch.tensor(lens, dtype=torch.int32, device=device)
    cu = torch.tensor([0, new, 2 * new], dtype=torch.int32, device=device)
    expect = attended(q, k, v, table, lens, [new, new], scale)
    for call in (lambda w: ops.attention_decode(q, k, v, table, at, new, scale, weights=w), lambda w: ops.attention_prefill(q, k, v, table, at, cu, new, scale, weights=w)):
        own = w.clone()
        compare(call(own), own, w, expect, dim, new * 4, device == "cuda")


def test_a_scale_that_is_no_number_is_refused(monkeypatch):
    packed(monkeypatch, 16)
    q, k, v, w, table, lens = arguments()
    with pytest.raises(ValueError):
        ops.attention_prefill(q, k, v, table, lens, torch.tensor([0, 1, 2], dtype=torch.int32), 1, float("nan"), weights=w)


# ------------------------------------------------------------------------------------------ rows that see nothing
@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_tables_without_pages_give_zeros(monkeypatch, device):
    """Steps and prompts over no pages at all: no row sees a token."""
    k, v, w = cache(3, 2, 64, device)
    if device == "cpu":
        packed(monkeypatch, 16)                              # the checks and the allocation in front of the kernels
        real = torch.empty_like
        monkeypatch.setattr(torch, "empty_like", lambda t: real(t).fill_(float("nan")))
    before = w.clone()
    q = torch.ones((2, 4, 64), dtype=torch.bfloat16, device=device)
    table, lens, cu = (torch.zeros(s, dtype=torch.int32, device=device) for s in ((2, 0), (2,), (3,)))
    cu[1:] = torch.tensor([1, 2])
    for out in (None, torch.full_like(q, 3)):
        for got in (ops.attention_decode(q, k, v, table, lens, 1, 0.1, weights=w, out=out), ops.attention_prefill(q, k, v, table, lens, cu, 1, 0.1, weights=w, out=out)):
            assert bool((got == 0).all()) and torch.equal(w, before)


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("lens, new", [([0, 5, 310], 300), ([0], 600), ([45, 256, 0], 300), ([44, 700], 300), ([1, 128], 129)])
@pytest.mark.parametrize("sinks", [False, True])
def test_sequences_shorter_than_their_rows(device, lens, new, sinks):
    """Many rows a head, the first of which stand in front of a sequence's first token: they see nothing and give zeros, the others are as ever."""
    num, table = layout(lens, device, wider=1)
    k, v, w = cache(num, 2, 64, device)
    q = torch.randn((len(lens) * new, 4, 64), generator=torch.Generator().manual_seed(5)).bfloat16().to(device)
    sink = torch.randn(4, generator=torch.Generator().manual_seed(6)).to(device) if sinks else None
    expect = attended(q, k, v, table, lens, [new] * len(lens), 0.125, sinks=sink)
    for known in (0, max(lens)):
        own = w.clone()
        out = ops.attention_decode(q, k, v, table, torch.tensor(lens, dtype=torch.int32, device=device), new, 0.125, sinks=sink, weights=own, max_kv_len=known)
        compare(out, own, w, expect, 64, new * 2, device == "cuda")
    if device == "cuda":
        ops.native.check_status(torch.device("cuda", 0))


# ------------------------------------------------------------------------------------------ what must not be touched
CALLS = {
    "step": lambda q, k, v, w, table, lens, cu: ops.attention_decode(q, k, v, table, lens, 1, 0.1, weights=w),
    "prompt": lambda q, k, v, w, table, lens, cu: ops.attention_prefill(q, k, v, table, lens, cu, 1, 0.1, weights=w),
    "evict": lambda q, k, v, w, table, lens, cu: ops.evict_tokens(k[None], v[None], w[None], table, lens, 8),
}


@pytest.mark.gpu
@pytest.mark.parametrize("what", CALLS)
@pytest.mark.parametrize("fault", ["length", "page behind the pool", "page before it"])
def test_what_the_table_does_not_name_stays_as_it_is(what, fault):
    """A length beyond the table's row, or a page that is none, is reported; pages that the sequences do not have are what they were, bit by bit."""
    q, k, v, w, table, lens = arguments("cuda", 128)
    table = table.clone()
    if fault == "length":
        lens = lens + torch.tensor([100, 0], dtype=torch.int32, device="cuda")
    else:
        table[0, 1] = 1 << 20 if "behind" in fault else -3
    mine = [int(p) for p in table.flatten().tolist() if 0 < p < k.shape[0]]
    others = [p for p in range(k.shape[0]) if p not in mine]
    assert others
    before = [x[others].clone() for x in (k, v, w)]
    CALLS[what](q, k, v, w, table, lens, torch.tensor([0, 1, 2], dtype=torch.int32, device="cuda"))
    with pytest.raises(RuntimeError, match="bad argument"):
        ops.native.check_status(torch.device("cuda", 0))
    assert all(torch.equal(x[others], old) for x, old in zip((k, v, w), before))


@pytest.mark.gpu
@pytest.mark.parametrize("what", ["step", "prompt"])
@pytest.mark.parametrize("beyond", [1, 100, 1 << 24])
def test_lengths_beyond_the_table_are_taken_as_what_it_holds(what, beyond):
    """Attention and weights go by the same length."""
    q, k, v, w, table, lens = arguments("cuda", 128)
    q = torch.randn(q.shape, generator=torch.Generator().manual_seed(7)).bfloat16().cuda()
    cu = torch.tensor([0, 1, 2], dtype=torch.int32, device="cuda")
    most = table.shape[1] * PAGE
    got = []
    for length in (most, most + beyond):
        own, at = w.clone(), lens.clone()
        at[0] = length
        got.append((CALLS[what](q, k, v, own, table, at, cu), own))
        if length > most:
            with pytest.raises(RuntimeError, match="bad argument"):
                ops.native.check_status(torch.device("cuda", 0))
        ops.native.check_status(torch.device("cuda", 0))
    assert all(torch.equal(a, b) for a, b in zip(*got))


@pytest.mark.parametrize("what", CALLS)
@pytest.mark.parametrize("fault", ["length", "page behind the pool", "page before it"])
def test_tensor_operations_refuse_what_the_table_does_not_name(what, fault):
    """The plain forms - on the CPU, and for heads that have no kernel - look at lengths and pages first: on a GPU an index out of range would end the process."""
    q, k, v, w, table, lens = arguments(dim=80)
    cu = torch.tensor([0, 1, 2], dtype=torch.int32)
    table[1, 1] = 99                                         # (nobody's: the second sequence has one page)
    CALLS[what](q, k, v, w.clone(), table, torch.tensor([20, 5], dtype=torch.int32), cu)
    if fault == "length":
        lens = lens + torch.tensor([100, 0], dtype=torch.int32)
    else:
        table[0, 1] = 1 << 20 if "behind" in fault else -3
    before = [x.clone() for x in (k, v, w)]
    with pytest.raises(ValueError):
        CALLS[what](q, k, v, w, table, lens, cu)
    assert all(torch.equal(x, old) for x, old in zip((k, v, w), before))


# ------------------------------------------------------------------------------------------ layers that lie apart
@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("apart", ["kvw", "k", "w"])
def test_layers_may_lie_apart(device, apart):
    """A part of the pages of every layer, as a pool has them that could not change its size."""
    num, table = layout([100, 20], device, seed=3)
    pools = dict(zip("kvw", cache(num, 2, 64, device, 4, layers=(3,))))
    lens = torch.tensor([100, 20], dtype=torch.int32, device=device)
    want = {x: t.clone() for x, t in pools.items()}
    ops.evict_tokens(want["k"], want["v"], want["w"], table, lens, 32, recent=4, first=1)
    for x in apart:
        room = pools[x].new_full((3, num + 5, *pools[x].shape[2:]), 7)
        room[:, :num] = pools[x]
        pools[x] = room[:, :num]
    left = ops.evict_tokens(pools["k"], pools["v"], pools["w"], table, lens, 32, recent=4, first=1)
    assert left.tolist() == [32, 20] and all(torch.equal(pools[x], want[x]) for x in "kvw")
    assert all(bool((pools[x]._base[:, num:] == 7).all()) for x in apart)


@pytest.mark.parametrize("pages", [9, 41])
def test_a_bounded_cache_goes_on_in_a_pool_that_could_not_change_its_size(pages):
    from eredu_b200.runtime.engine import Engine
    from test_kept_tokens_steps import GREEDY, build, prompt
    from test_kv8_engine import Failing

    model = build()
    outs = []
    for n in (None, 0, 1, 2):
        eng = Engine(model, max_batch=2, max_seq_len=128, kv_keep=eviction_rule())
        seq = eng.new_sequence(prompt(40), GREEDY, max_new_tokens=60)
        eng.feed_logits(seq, seq.prompt)
        if n is not None:
            with pytest.raises(torch.OutOfMemoryError), Failing(n, pages):
                eng.resize_cache(pages, [seq])
        outs.append(torch.stack([eng.feed_logits(seq, [5 + t]) for t in range(30)]))
        assert seq.cached < 40
    assert all(torch.equal(o, outs[0]) for o in outs[1:])


def eviction_rule():
    from eredu_b200.runtime.kv_cache import KeptTokens

    return KeptTokens(keep=24, recent=6, slack=8)
