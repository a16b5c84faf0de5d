"""Caches that give up tokens: attention that adds up the weight every cached token gets, and eviction by it, against the definition in 64 bits."""
import math
import re
from pathlib import Path

import pytest
import torch

from eredu_b200 import ops
from eredu_b200.ops import eviction
from eredu_b200.ops.kv8 import Pages8

PAGE = 16
DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


# ------------------------------------------------------------------------------------------ the definition
def attended(q, k, v, table, seq_lens, q_lens, scale, window=0, sinks=None, observed=0):
    """In 64 bits: (output, sum of p |v|, {(page, head, offset): (weight given, is the token new)}, largest sum of |q k| scale)."""
    q, k, v = q.double().cpu(), k.double().cpu(), v.double().cpu()
    out, size, given, most = torch.zeros((*q.shape[:2], v.shape[3]), dtype=torch.float64), torch.zeros((*q.shape[:2], v.shape[3]), dtype=torch.float64), {}, 0.0
    group, start = q.shape[1] // k.shape[1], 0
    for b, (n, m) in enumerate(zip(seq_lens, q_lens)):
        at = table[b, :-(-n // PAGE)].long().cpu() if n > 0 else torch.zeros(0, dtype=torch.long)
        for h in range(k.shape[1]):
            kk, vv = (t[at, h].reshape(-1, t.shape[3])[:max(n, 0)] for t in (k, v))
            total = torch.zeros(max(n, 0), dtype=torch.float64)
            for i in range(m):
                pos = n - m + i
                low = max(0, pos - window + 1) if window else 0
                if pos < 0:
                    continue
                rows = q[start + i, h * group:(h + 1) * group]
                s = rows @ kk[low:pos + 1].t() * scale
                most = max(most, float((rows.abs() @ kk[low:pos + 1].abs().t()).max()) * abs(scale))
                if sinks is not None:
                    s = torch.cat((s, sinks[h * group:(h + 1) * group].double().cpu()[:, None]), 1)
                p = torch.softmax(s, 1)[:, :pos + 1 - low]
                out[start + i, h * group:(h + 1) * group] = p @ vv[low:pos + 1]
                size[start + i, h * group:(h + 1) * group] = p @ vv[low:pos + 1].abs()
                if not observed or i >= m - observed:
                    total[low:pos + 1] += p.sum(0)
            for t in range(max(n, 0)):
                if m:
                    given[(int(at[t // PAGE]), h, t % PAGE)] = (float(total[t]), t >= n - m)
        start += m
    return out, size, given, most


def evicted(k, v, w, table, seq_lens, keep, recent, first):
    """Copies of the pools behind an eviction, token by token."""
    k, v, w = (t.cpu().clone() for t in (k, v, w))
    table = table.cpu()
    for b, n in enumerate(seq_lens):
        if n <= keep:
            continue
        cell = [(int(table[b, t // PAGE]), t % PAGE) for t in range(n)]
        for layer in range(k.shape[0]):
            for h in range(k.shape[2]):
                between = range(first, n - recent)
                value = [float(w[layer, p, h, o]) for p, o in cell]
                rank = sorted(between, key=lambda t: (math.isnan(value[t]), -value[t] if not math.isnan(value[t]) else 0.0, t))
                stays = sorted([*range(first), *rank[:keep - first - recent], *range(n - recent, n)])
                for x in (k, v, w):
                    rows = [x[layer, cell[t][0], h, cell[t][1]].clone() for t in stays]
                    for (p, o), row in zip(cell, rows):
                        x[layer, p, h, o] = row
    return k, v, w


def layout(seq_lens, device, seed=0, wider=0):
    """(pages in all, block table with pages in any order, a pitch wider than its rows)."""
    g = torch.Generator().manual_seed(seed)
    count = [-(-max(n, 0) // PAGE) for n in seq_lens]
    place = 1 + torch.randperm(sum(count) + 2, generator=g)
    wide = max(max(count), 1) + wider
    table = torch.zeros((len(seq_lens), wide + 3), dtype=torch.int32)
    at = 0
    for i, c in enumerate(count):
        table[i, :c] = place[at:at + c].to(torch.int32)
        at += c
    return sum(count) + 3, table.to(device)[:, :wide]


def cache(num, heads, dim, device, seed=0, dtype=torch.bfloat16, layers=()):
    g = torch.Generator().manual_seed(seed)
    k, v = ((torch.randn((*layers, num, heads, PAGE, dim), generator=g)).to(dtype).to(device) for _ in "kv")
    w = torch.exp(torch.randn((*layers, num, heads, PAGE), generator=g)).to(device)
    return k, v, w


def compare(out, w, before, expect, dim, terms, on_gpu, prior=1):
    """Output: rounded to bf16 (2^-8), probabilities rounded to bf16 in front of the values by the kernels, and what the scores are off by. A score is a sum of dim
    products (2^-24 of the sum of their magnitudes for each addition; twice that on the tensor cores, which may cut where others round); a weight is off by twice that, relatively, by
    some roundings of its own (64) and by those of the sum of ``terms`` of them; ``prior`` sums of earlier calls are rounded once more each."""
    ref, size, given, most = expect
    score = (dim + 16) * 2.0 ** -23 * most + 2.0 ** -20
    p_round = 2.0 ** -8 if on_gpu else 0.0
    tol = 2.0 ** -8 * ref.abs() + (p_round + 2 * score) * size * (1 + 2.0 ** -8) + 1e-30
    assert bool(((out.double().cpu() - ref).abs() <= tol).all()), ((out.double().cpu() - ref).abs() / tol).max()
    w, before = w.double().cpu(), before.double().cpu()
    untouched = torch.ones(w.shape, dtype=torch.bool)
    for at, (value, new) in given.items():
        untouched[at] = False
        want = value if new else float(before[at]) + value
        bound = (2 * score + (terms + 64) * 2.0 ** -24) * value + prior * 2.0 ** -24 * want + 1e-37
        assert abs(float(w[at]) - want) <= bound, (at, float(w[at]), want, bound)
    assert torch.equal(w[untouched].nan_to_num(7), before[untouched].nan_to_num(7))


def spoil(k, v, w, table, seq_lens):
    """What lies behind the last token of a sequence, and pages that nobody has, are no numbers."""
    mine = torch.zeros(w.shape[0], w.shape[2], dtype=torch.bool)
    for b, n in enumerate(seq_lens):
        for t in range(max(n, 0)):
            mine[int(table[b, t // PAGE]), t % PAGE] = True
    for x in (k, v, w):
        rows = x.transpose(1, 2)
        rows[~mine.to(x.device)] = float("nan")


# ------------------------------------------------------------------------------------------ steps
STEPS = [
    # heads, lengths, new tokens, window, sinks
    ((32, 8, 64), [1], 1, 0, False),
    ((8, 2, 128), [16, 17, 1], 1, 0, False),
    ((16, 2, 128), [300, 33, 128, 5], 1, 0, True),
    ((4, 4, 64), [200, 2], 1, 70, False),
    ((8, 8, 128), [95, 40], 5, 0, True),
    ((8, 2, 64), [130, 4, 64], 4, 33, True),
    ((6, 2, 128), [77, 9], 3, 0, False),
    ((14, 2, 64), [50, 129], 2, 16, False),
    ((16, 1, 128), [222], 1, 1, False),
    ((8, 1, 128), [140, 35], 5, 0, True),
    ((12, 2, 64), [300, 17, 65], 7, 40, False),
    ((16, 2, 64), [200, 31, 8], 8, 50, False),
    ((8, 2, 128), [600], 8, 0, False),
    ((16, 1, 128), [100, 6], 5, 0, True),
    ((33, 1, 64), [70], 1, 0, False),
    ((8, 2, 128), [0, 30, 1], 1, 0, False),
    ((16, 2, 64), [3, 0, 20], 5, 8, True),
]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("heads, lens, new, window, sinks", STEPS)
def test_step(device, heads, lens, new, window, sinks):
    n_q, n_kv, dim = heads
    num, table = layout(lens, device, wider=2)
    k, v, w = cache(num, n_kv, dim, device)
    spoil(k, v, w, table, lens)
    g = torch.Generator().manual_seed(1)
    q = torch.randn((len(lens) * new, n_q, dim), generator=g).bfloat16().to(device)
    sink = torch.randn(n_q, generator=g).to(device) if sinks else None
    before, scale = w.clone(), dim ** -0.5
    out = ops.attention_decode(q, k, v, table, torch.tensor(lens, dtype=torch.int32, device=device), new, scale, window=window, sinks=sink, weights=w,
                               max_kv_len=max(lens))
    expect = attended(q, k, v, table, lens, [new] * len(lens), scale, window, sink)
    compare(out, w, before, expect, dim, new * n_q // n_kv, device == "cuda")
    if device == "cuda":
        ops.native.check_status(torch.device("cuda", 0))


@pytest.mark.gpu
@pytest.mark.parametrize("splits", [1, 2, 3, 5, 8, 12, 16, 17, 64])
@pytest.mark.parametrize("heads, lens, new, window", [((8, 2, 128), [1000, 17, 3], 1, 0), ((8, 1, 64), [777, 300], 2, 400),
                                                      ((8, 2, 64), [700, 90], 5, 0), ((16, 2, 128), [600, 33], 7, 300)])
def test_step_in_any_number_of_splits(monkeypatch, splits, heads, lens, new, window):
    monkeypatch.setattr(eviction, "weighed_splits", lambda *a: splits)
    test_step("cuda", heads, lens, new, window, True)


@pytest.mark.gpu
def test_steps_add_up_and_are_the_same_each_time():
    """Weights of a thousand tokens over twenty steps: what rows give sums up to the rows; two runs agree bit by bit."""
    runs = []
    for _ in range(2):
        num, table = layout([1000], "cuda")
        k, v, w = cache(num, 8, 128, "cuda")
        w.zero_()
        g = torch.Generator().manual_seed(3)
        for _ in range(20):
            q = torch.randn((1, 32, 128), generator=g).bfloat16().cuda()
            ops.attention_decode(q, k, v, table, torch.tensor([999], dtype=torch.int32, device="cuda"), 1, 128 ** -0.5, weights=w)
        runs.append(w.clone())
    assert torch.equal(*runs)
    # the new token's place is set anew by every step: what the other tokens got is 20 steps' weights but for that
    heads = runs[0].sum((0, 2))
    assert bool((heads <= 20 * 4 * (1 + 2.0 ** -10)).all()) and bool((heads > 19 * 4 * 0.9).all())


# ------------------------------------------------------------------------------------------ prompts
PROMPTS = [
    # heads, (cached, new) of every sequence, window, sinks, observed
    ((8, 2, 128), [(0, 1)], 0, False, 0),
    ((8, 2, 128), [(0, 130), (37, 5), (0, 17)], 0, True, 0),
    ((4, 4, 64), [(100, 33), (5, 200)], 0, False, 0),
    ((8, 1, 128), [(0, 257), (300, 3)], 90, True, 0),
    ((6, 2, 64), [(0, 300)], 0, False, 7),
    ((8, 2, 128), [(260, 45), (0, 2), (511, 1)], 0, False, 16),
    ((14, 2, 128), [(3, 70), (0, 0), (129, 140)], 33, False, 50),
    ((16, 1, 64), [(40, 9)], 0, True, 1),
    ((3, 3, 128), [(0, 129), (256, 256)], 256, False, 0),
]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("known", [False, True])
@pytest.mark.parametrize("heads, spans, window, sinks, observed", PROMPTS)
def test_prompt(device, known, heads, spans, window, sinks, observed):
    n_q, n_kv, dim = heads
    lens, new = [a + n for a, n in spans], [n for _, n in spans]
    num, table = layout(lens, device, seed=4, wider=1)
    k, v, w = cache(num, n_kv, dim, device, seed=5)
    spoil(k, v, w, table, lens)
    g = torch.Generator().manual_seed(6)
    q = torch.randn((sum(new), n_q, dim), generator=g).bfloat16().to(device)
    sink = torch.randn(n_q, generator=g).to(device) if sinks else None
    cu_q = torch.tensor([sum(new[:i]) for i in range(len(new) + 1)], dtype=torch.int32, device=device)
    before, scale = w.clone(), dim ** -0.5
    out = ops.attention_prefill(q, k, v, table, torch.tensor(lens, dtype=torch.int32, device=device), cu_q, max(new), scale, window=window, sinks=sink,
                                weights=w, observed=observed, max_kv_len=max(lens) if known else 0)
    expect = attended(q, k, v, table, lens, new, scale, window, sink, observed)
    compare(out, w, before, expect, dim, max(new) * n_q // n_kv, device == "cuda")
    if device == "cuda":
        ops.native.check_status(torch.device("cuda", 0))


@pytest.mark.gpu
def test_long_prompt():
    """Several blocks of keys and many tiles of rows, against 64 bits on the GPU."""
    n_q, n_kv, dim, n = 16, 4, 128, 1500
    num, table = layout([n], "cuda", seed=7)
    k, v, w = cache(num, n_kv, dim, "cuda", seed=8)
    q = torch.randn((n, n_q, dim), generator=torch.Generator().manual_seed(9)).bfloat16().cuda()
    ops.attention_prefill(q, k, v, table, torch.tensor([n], dtype=torch.int32, device="cuda"), torch.tensor([0, n], dtype=torch.int32, device="cuda"), n, dim ** -0.5,
                          weights=w, max_kv_len=n)
    at = table[0].long()
    kk = k[at].transpose(0, 1).reshape(n_kv, -1, dim)[:, :n].double()
    s = torch.einsum("qhgd,hkd->hgqk", q.double().view(n, n_kv, -1, dim), kk) * dim ** -0.5
    s = s.masked_fill(torch.ones(n, n, dtype=torch.bool, device="cuda").triu(1), float("-inf"))
    want = torch.softmax(s, -1).sum((1, 2))
    got = w[at].transpose(0, 1).reshape(n_kv, -1)[:, :n].double()
    most = float((q.double().abs().amax() * kk.abs().sum(-1).amax()) * dim ** -0.5)
    assert bool(((got - want).abs() <= (2 * (dim + 16) * 2.0 ** -23 * most + (4 * n + 64) * 2.0 ** -24) * want).all())


# ------------------------------------------------------------------------------------------ eviction
EVICTIONS = [
    # layers, heads, widths, lengths, keep, recent, first
    (1, 1, (64, 64), [2], 1, 0, 0),
    (2, 3, (128, 128), [40, 17, 100, 16], 17, 5, 2),
    (3, 2, (64, 128), [200, 31], 32, 32, 0),
    (1, 2, (8, 8), [65, 300], 64, 0, 64),
    (2, 1, (80, 80), [129, 0, 128, 130], 128, 10, 4),
    (1, 4, (128, 128), [2500], 700, 100, 4),
]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("layers, heads, widths, lens, keep, recent, first", EVICTIONS)
def test_evict(device, dtype, layers, heads, widths, lens, keep, recent, first):
    num, table = layout(lens, device, seed=10, wider=1)
    k, _, w = cache(num, heads, widths[0], device, 11, dtype, (layers,))
    v = cache(num, heads, widths[1], device, 12, dtype, (layers,))[1]
    # equal weights, both zeros, infinities and what is no number
    g = torch.Generator().manual_seed(13)
    special = torch.tensor([0.0, -0.0, 1.0, 1.0, float("inf"), float("-inf"), float("nan"), -2.0, 1e-42])
    pick = torch.randint(0, 24, w.shape, generator=g)
    w.copy_(torch.where(pick < len(special), special[pick.clamp_max(len(special) - 1)], w.cpu()).to(device))
    expect = evicted(k, v, w, table, lens, keep, recent, first)
    left = ops.evict_tokens(k, v, w, table, torch.tensor(lens, dtype=torch.int32, device=device), keep, recent=recent, first=first)
    assert left.dtype == torch.int32 and left.tolist() == [min(n, keep) for n in lens]
    for got, want in zip((k, v, w), expect):
        kind = torch.int16 if got.dtype == torch.bfloat16 else torch.int32
        assert torch.equal(got.cpu().view(kind), want.view(kind))
    if device == "cuda":
        ops.native.check_status(torch.device("cuda", 0))


@pytest.mark.gpu
@pytest.mark.parametrize("n, keep", [(60001, 4000), (49153, 49152), (50000, 33)])
def test_evict_long_sequences(n, keep):
    """More weights than shared memory holds; many of them equal."""
    num, table = layout([n], "cuda", seed=14)
    k, v, w = cache(num, 2, 8, "cuda", 15, layers=(1,))
    w.copy_((w * 20).round() / 20)
    at = table[0].long()
    flat = [x[0, at].transpose(0, 1).flatten(1, 2)[:, :n].clone() for x in (k, v, w)]
    stays = torch.sort(flat[2], dim=1, descending=True, stable=True)[1][:, :keep].sort(1)[0]
    ops.evict_tokens(k, v, w, table, torch.tensor([n], dtype=torch.int32, device="cuda"), keep)
    for x, old in zip((k, v, w), flat):
        now = x[0, at].transpose(0, 1).flatten(1, 2)
        for h in range(2):
            assert torch.equal(now[h, :keep], old[h][stays[h]]) and torch.equal(now[h, keep:n], old[h, keep:])


def test_layers_in_portions(monkeypatch):
    """A call whose lists would take too much memory goes layer by layer."""
    calls = []
    monkeypatch.setattr(eviction, "LIST_BYTES", 1)
    monkeypatch.setattr(eviction, "evict_tokens_ref", lambda *a: calls.append(a) or a[4].clamp_max(a[5]))
    num, table = layout([40], "cpu")
    k, v, w = cache(num, 1, 16, "cpu", layers=(3,))
    assert ops.evict_tokens(k, v, w, table, torch.tensor([40], dtype=torch.int32), 20).tolist() == [20] and len(calls) == 1


@pytest.mark.gpu
def test_layers_in_portions_on_the_gpu(monkeypatch):
    monkeypatch.setattr(eviction, "LIST_BYTES", 4 * 4 * 3 * 17 * 2)
    test_evict("cuda", torch.bfloat16, 3, 3, (128, 128), [40, 17, 100, 16], 17, 5, 2)


# ------------------------------------------------------------------------------------------ all of them together
@pytest.mark.parametrize("device", DEVICES)
def test_a_cache_of_bounded_size(device):
    """A prompt, its eviction, steps and another eviction, beside a sequence that stays short; every call is checked on what it was given."""
    n_q, n_kv, dim, keep, layers = 8, 2, 64, 48, 2
    g = torch.Generator().manual_seed(20)
    lens = [100, 20]
    num, table = layout([128, 64], device, seed=21)
    k, v, w = cache(num, n_kv, dim, device, 22, layers=(layers,))
    scale = dim ** -0.5
    as_int = lambda x: torch.tensor(x, dtype=torch.int32, device=device)     # noqa: E731
    for layer in range(layers):
        q = torch.randn((sum(lens), n_q, dim), generator=g).bfloat16().to(device)
        before = w[layer].clone()
        out = ops.attention_prefill(q, k[layer], v[layer], table, as_int(lens), as_int([0, 100, 120]), 100, scale, weights=w[layer])
        compare(out, w[layer], before, attended(q, k[layer], v[layer], table, lens, lens, scale), dim, 400, device == "cuda")
    for _ in range(2):
        expect = evicted(k, v, w, table, lens, keep, 8, 2)
        left = ops.evict_tokens(k, v, w, table, as_int(lens), keep, recent=8, first=2)
        lens = [min(n, keep) for n in lens]
        assert left.tolist() == lens and all(torch.equal(a.cpu(), b) for a, b in zip((k, v, w), expect))
        for _ in range(6):
            lens = [n + 1 for n in lens]
            for layer in range(layers):
                q = torch.randn((2, n_q, dim), generator=g).bfloat16().to(device)
                before = w[layer].clone()
                out = ops.attention_decode(q, k[layer], v[layer], table, as_int(lens), 1, scale, weights=w[layer])
                compare(out, w[layer], before, attended(q, k[layer], v[layer], table, lens, [1, 1], scale), dim, 4, device == "cuda")


# ------------------------------------------------------------------------------------------ what is refused, and calls of odd kinds
def arguments(device="cpu", dim=64):
    num, table = layout([20, 5], device)
    k, v, w = cache(num, 2, dim, device)
    q = torch.zeros((2, 4, dim), dtype=torch.bfloat16, device=device)
    return q, k, v, w, table, torch.tensor([20, 5], dtype=torch.int32, device=device)


def test_formats_and_header_agree():
    """The argument blocks as Python packs them and as the header has them: as many pointers, whole and real numbers, in whole multiples of eight bytes."""
    header = (Path(ops.__file__).resolve().parent.parent / "csrc/common/weights_args.h").read_text()
    for name, block in (("EvictArgs", eviction._EVICT), ("WeighedDecodeArgs", eviction._DECODE), ("WeighedPrefillArgs", eviction._PROMPT)):
        body = re.sub(r"//.*", "", header.partition(f"struct {name} {{")[2].partition("};")[0])
        kinds = ""
        for line in body.split(";"):
            names = line.count(",") + 1
            kinds += "" if not line.strip() else ("Q" if "*" in line or "cudaStream_t" in line else "f" if "float" in line else "i") * names
        assert kinds == "".join(c * int(n or 1) for n, c in re.findall(r"(\d*)([Qif])", block.format)) and block.size % 8 == 0


def test_refusals_of_attention():
    q, k, v, w, table, lens = arguments()
    step = lambda **o: ops.attention_decode(o.get("q", q), o.get("k", k), o.get("v", v), o.get("table", table), o.get("lens", lens), 1, 0.1, sinks=o.get("sinks"),  # noqa: E731
                                            weights=o.get("w", w), chunk=o.get("chunk", 0), out=o.get("out"))
    step()
    for wrong in (dict(w=w.double()), dict(w=w[:, :1]), dict(w=w.transpose(1, 2).contiguous().transpose(1, 2)), dict(table=table.long()), dict(table=table[:1]),
                  dict(lens=lens.long()), dict(q=q[:1]), dict(q=q[:, :3]), dict(v=v[:-1]), dict(sinks=torch.zeros(3)), dict(out=q.float())):
        with pytest.raises(ValueError):
            step(**wrong)
    with pytest.raises(NotImplementedError):
        step(chunk=16)
    with pytest.raises(NotImplementedError):
        step(k=Pages8.empty(5, 2, 64, "cpu"), v=Pages8.empty(5, 2, 64, "cpu"))
    cu = torch.tensor([0, 1, 2], dtype=torch.int32)
    ops.attention_prefill(q, k, v, table, lens, cu, 1, 0.1, weights=w)
    for more in (dict(observed=-1), ):
        with pytest.raises(ValueError):
            ops.attention_prefill(q, k, v, table, lens, cu, 1, 0.1, weights=w, **more)
    with pytest.raises(ValueError):
        ops.attention_prefill(q, k, v, table, lens, cu[:2], 1, 0.1, weights=w)


def test_refusals_of_evictions():
    _, k, v, w, table, lens = arguments()
    k, v, w = k[None], v[None], w[None]
    evict = lambda keep=8, k=k, v=v, w=w, table=table, lens=lens, **o: ops.evict_tokens(k, v, w, table, lens, keep, **o)     # noqa: E731
    for wrong in (dict(keep=0), dict(recent=5, first=4), dict(recent=-1), dict(first=-1), dict(w=w[0]), dict(w=w.double()), dict(k=k[0]), dict(v=v[:, 1:]),
                  dict(v=v.float()), dict(table=table.long()), dict(table=table[:1]), dict(lens=lens.long()), dict(k=k.transpose(1, 2).contiguous().transpose(1, 2))):
        with pytest.raises(ValueError):
            evict(**wrong)
    with pytest.raises(NotImplementedError):
        evict(k=k.to(torch.int8), v=v.to(torch.int8))


@pytest.mark.gpu
def test_refusals_of_the_kernels():
    q, k, v, w, table, lens = arguments("cuda")
    with pytest.raises(ValueError):
        ops.attention_decode(q.float(), k.float(), v.float(), table, lens, 1, 0.1, weights=w)
    with pytest.raises(ValueError):
        ops.attention_decode(q, k, v, table, lens.cpu(), 1, 0.1, weights=w)
    with pytest.raises(NotImplementedError):
        ops.evict_tokens(k[None, ..., :4].contiguous(), v[None, ..., :4].contiguous(), w[None], table, lens, 8)


@pytest.mark.gpu
def test_lengths_and_pages_that_the_table_does_not_have_are_reported():
    """Reported, and nothing outside of the pages is read or written."""
    dev = torch.device("cuda", 0)
    for what in ("length", "page"):
        q, k, v, w, table, lens = arguments("cuda")
        if what == "length":
            lens = lens + 100
        else:
            table = table.clone()
            table[0, 0] = 1 << 20
        cu = torch.tensor([0, 1, 2], dtype=torch.int32, device="cuda")
        for call in (lambda: ops.attention_decode(q, k, v, table, lens, 1, 0.1, weights=w),
                     lambda: ops.evict_tokens(k[None], v[None], w[None], table, lens, 8)):
            call()
            with pytest.raises(RuntimeError, match="bad argument"):
                ops.native.check_status(dev)
        del cu


def test_calls_for_another_device_are_made_there(monkeypatch):
    """A launch takes the stream of the current device: tensors of another one make it the current one first."""
    current, made = [0], []

    class On:
        device = torch.device("cuda", 1)

        @staticmethod
        def get_device():
            return 1

    class Device:
        def __init__(self, device):
            self.index = device.index

        def __enter__(self):
            current.append(self.index)

        def __exit__(self, *_):
            current.pop()

    monkeypatch.setattr(eviction, "_current", lambda: current[-1])
    monkeypatch.setattr(torch.cuda, "device", Device)
    monkeypatch.setattr(eviction, "_kernels_take", lambda *a: made.append(current[-1]) or 1 / 0)
    for call in (lambda: eviction.weighed_decode(On, On, On, None, torch.zeros(1), 1, 1.0, 0, None, None, None, 0, 0),
                 lambda: eviction.weighed_prefill(On, On, On, None, torch.zeros(1), None, 1, 1.0, 0, None, None, None, 0, 0, 0)):
        with pytest.raises(ZeroDivisionError):
            call()
    assert made == [1, 1] and current == [0]


@pytest.mark.parametrize("device", DEVICES)
def test_keys_that_are_infinite(device):
    """A key that is minus infinity in the direction of every query gets no weight, and no other token notices (three rows: one of a kernel's four is empty)."""
    k, v, w = cache(4, 1, 64, device, 30)
    k[:] = k.abs()
    k[2, 0, 5] = float("-inf")
    q = torch.rand((1, 3, 64), generator=torch.Generator().manual_seed(31)).bfloat16().to(device) + 0.1
    table, lens, before = torch.tensor([[2, 3]], dtype=torch.int32, device=device), torch.tensor([20], dtype=torch.int32, device=device), w.clone()
    out = ops.attention_decode(q, k, v, table, lens, 1, 0.125, weights=w)
    at = ops.attention_prefill(q, k, v, table, lens, torch.tensor([0, 1], dtype=torch.int32, device=device), 1, 0.125, weights=before.clone())
    assert torch.isfinite(out).all() and torch.isfinite(at).all() and torch.isfinite(w[2:]).all() and w[2, 0, 5] == before[2, 0, 5]
    given = torch.cat((w[2, 0] - before[2, 0], w[3, 0, :3] - before[3, 0, :3], w[3, 0, 3:4]))
    assert abs(float(given.double().sum()) - 3) <= 3 * 2.0 ** -12


@pytest.mark.gpu
def test_two_calls_at_once():
    """Calls on two streams have nothing in common but their inputs."""
    cases = []
    for seed in (40, 41):
        num, table = layout([1500, 700], "cuda", seed)
        k, v, w = cache(num, 2, 128, "cuda", seed)
        q = torch.randn((2, 8, 128), generator=torch.Generator().manual_seed(seed)).bfloat16().cuda()
        cases.append((q, k, v, table, torch.tensor([1500, 700], dtype=torch.int32, device="cuda"), w))
    alone = []
    for q, k, v, table, lens, w in cases:
        own = w.clone()
        alone.append((ops.attention_decode(q, k, v, table, lens, 1, 0.1, weights=own), own))
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    got = []
    for _ in range(5):
        got = []
        for stream, (q, k, v, table, lens, w) in zip(streams, cases):
            with torch.cuda.stream(stream):
                own = w.clone()
                got.append((ops.attention_decode(q, k, v, table, lens, 1, 0.1, weights=own), own))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for pair, other in zip(got, alone) for a, b in zip(pair, other))


@pytest.mark.gpu
def test_a_longest_length_that_is_none_is_reported():
    q, k, v, w, table, lens = arguments("cuda", 128)
    num, table = layout([600], "cuda")
    k, v, w = cache(num, 2, 128, "cuda")
    cu = torch.tensor([0, 1], dtype=torch.int32, device="cuda")
    lens = torch.tensor([600], dtype=torch.int32, device="cuda")
    ops.attention_prefill(q[:1], k, v, table, lens, cu, 1, 0.1, weights=w, max_kv_len=100)
    with pytest.raises(RuntimeError, match="bad argument"):
        ops.native.check_status(torch.device("cuda", 0))


@pytest.mark.gpu
def test_other_head_sizes_take_tensor_operations():
    test_step("cuda", (4, 2, 80), [33, 7], 1, 0, False)


@pytest.mark.gpu
def test_replayed_calls_and_other_streams():
    """A step, a prompt's portion and an eviction captured into a graph on a stream of its own."""
    q, k, v, w, table, lens = arguments("cuda")
    cu = torch.tensor([0, 1, 2], dtype=torch.int32, device="cuda")
    saved = [x.clone() for x in (k, v, w)]

    def body():
        a = ops.attention_decode(q, k, v, table, lens, 1, 0.1, weights=w)
        b = ops.attention_prefill(q, k, v, table, lens, cu, 1, 0.1, weights=w)
        return a, b, ops.evict_tokens(k[None], v[None], w[None], table, lens, 8, recent=2)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        eager = [x.clone() for x in (*body(), k, v, w)]
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        outs = body()
    for _ in range(2):
        for x, old in zip((k, v, w), saved):
            x.copy_(old)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip((*outs, k, v, w), eager))
