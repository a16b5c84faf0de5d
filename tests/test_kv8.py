"""Keys and values held in 8 bits: pages written, read, attended to and moved, against the definition in 64 bits."""
import math
import re
from pathlib import Path

import pytest
import torch

from eredu_b200 import ops
from eredu_b200.ops import kv8
from eredu_b200.ops.kv8 import FLOOR, PAGE, Pages8

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


# ------------------------------------------------------------------------------------------ the definition
def rounded(rows, codes, scales, page, first):
    """Rows [n, heads, dim] (64 bits) behind the first ``first`` of a page, into copies that are 64 bits wide."""
    need = torch.exp2(torch.ceil(torch.log2(rows.abs().amax((0, 2)) / 127))).clamp_min(FLOOR)
    need = torch.where(torch.isfinite(rows).all(2).all(0), need, torch.full_like(need, math.nan))
    if first:
        before = scales[page].clone()
        need = torch.where(torch.isnan(before) | torch.isnan(need), torch.full_like(need, math.nan), torch.maximum(before, need))
        codes[page, :, :first] = torch.round(codes[page, :, :first] * (before / need)[:, None, None])
    scales[page] = need
    codes[page, :, first:first + len(rows)] = torch.round(rows / need[:, None]).transpose(0, 1)


def stored(x, slots, pages):
    """What ``pages`` hold behind a write of rows ``x``: (codes, scales) in 64 bits."""
    codes, scales = pages.codes.double().cpu(), pages.scales.double().cpu()
    at, i, x = slots.tolist(), 0, x.double().cpu()
    while i < len(at):
        n = 1
        if at[i] >= 0:
            while i + n < len(at) and (at[i] + n) % PAGE and at[i + n] == at[i] + n:
                n += 1
            rounded(x[i:i + n], codes, scales, at[i] // PAGE, at[i] % PAGE)
        i += n
    return codes, scales


def attended(q, k, v, table, seq_lens, q_lens, scale, window=0, chunk=0, sinks=None):
    """(output, sum of p |v|) in 64 bits; zeros where a row sees nothing. k, v: [pages, heads, 16, dim] values."""
    q, k, v = q.double().cpu(), k.double().cpu(), v.double().cpu()
    out, size = torch.zeros_like(q), torch.zeros_like(q)
    group, start = q.shape[1] // k.shape[1], 0
    for b, (n, m) in enumerate(zip(seq_lens, q_lens)):
        at = table[b, :-(-n // PAGE)].long().cpu()
        for i in range(m):
            pos = n - m + i
            low = max(0, pos - window + 1) if window else pos - pos % chunk if chunk and pos > 0 else 0
            if pos < 0:
                continue
            for h in range(k.shape[1]):
                kk, vv = (t[at, h].reshape(-1, t.shape[3])[low:pos + 1] for t in (k, v))
                s = q[start + i, h * group:(h + 1) * group] @ kk.t() * scale
                if sinks is not None:
                    s = torch.cat((s, sinks[h * group:(h + 1) * group].double().cpu()[:, None]), 1)
                p = torch.softmax(s, 1)[:, :pos + 1 - low]
                out[start + i, h * group:(h + 1) * group] = p @ vv
                size[start + i, h * group:(h + 1) * group] = p @ vv.abs()
        start += m
    return out, size


def filled(num, heads, dim, device, seed=0, spread=1.0):
    """Random pages: codes all over the range, scales within a few powers of two of one another."""
    g = torch.Generator().manual_seed(seed)
    codes = (torch.randn((num, heads, PAGE, dim), generator=g) * 40).round().clamp(-127, 127).to(torch.int8)
    scales = torch.exp2(torch.randint(-1, 2, (num, heads), generator=g).float() * spread - 6)
    return Pages8(codes.to(device), scales.to(device))


def layout(seq_lens, device, seed=0, more=0, wider=0):
    """(pages in all, block table [B, widest + wider] with pages in any order)."""
    g = torch.Generator().manual_seed(seed)
    count = [-(-n // PAGE) for n in seq_lens]
    place = 1 + torch.randperm(sum(count) + more, generator=g)
    table = torch.zeros((len(seq_lens), max(max(count), 1) + wider), dtype=torch.int32)
    for b, n in enumerate(count):
        table[b, :n] = place[sum(count[:b]):sum(count[:b]) + n].to(torch.int32)
    return sum(count) + more + 1, table.to(device)


def ints(values, device, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device=device)


# ------------------------------------------------------------------------------------------ writing
def test_scales_are_the_smallest_powers_of_two():
    x = torch.tensor([0.0, 127.0, 127.0 * 2 ** -3, 127.5, 1.0, 1e-40, 2.0 ** 127, 64.0, 63.5])
    want = [FLOOR, 1.0, 2.0 ** -3, 2.0, 2.0 ** -6, FLOOR, 2.0 ** 121, 1.0, 0.5]
    assert kv8.needed_scale(x).tolist() == want
    assert kv8.needed_scale(torch.tensor([math.inf, math.nan])).isnan().all()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("heads, dim", [(1, 64), (8, 128), (3, 128), (2, 64)])
@pytest.mark.parametrize("start, new", [((0,), (1,)), ((0, 0), (16, 33)), ((5, 31, 16), (1, 1, 1)), ((3, 47, 0), (40, 20, 300)), ((15, 1), (2, 700))])
def test_rows_are_stored_as_defined(device, heads, dim, start, new):
    """Values of any kind, exactly: quotients by powers of two are."""
    total = [a + n for a, n in zip(start, new)]
    num, table = layout(total, device, more=3)
    g = torch.Generator().manual_seed(dim + sum(new))
    rows = sum(new)
    k, v = ((torch.randn((rows, heads, dim), generator=g) * torch.exp2(torch.randint(-6, 7, (rows, heads, 1), generator=g).float())).bfloat16().to(device)
            for _ in "kv")
    k[0] = 0                                                     # a row of nothing
    v[-1, 0, 0] = 127.0 * 64                                     # a largest value that just fits
    at = torch.cat([torch.arange(a, a + n) for a, n in zip(start, new)])
    seq = torch.repeat_interleave(torch.arange(len(new)), torch.tensor(new))
    slots = (table.cpu()[seq, at // PAGE].long() * PAGE + at % PAGE)
    slots[rows // 2] = -1                                        # not stored: the rows behind it begin a run of their own
    if rows > 1:
        slots[rows // 2:rows // 2 + (PAGE - int(at[rows // 2]) % PAGE)] = -1
    pages = [filled(num, heads, dim, device, seed=i) for i in range(2)]
    want = [stored(x, slots, p) for x, p in zip((k, v), pages)]
    ops.store_kv(k, v, slots.to(device), *pages)
    for p, (codes, scales) in zip(pages, want):
        assert torch.equal(p.scales.double().cpu(), scales) and torch.equal(p.codes.double().cpu(), codes)


@pytest.mark.parametrize("device", DEVICES)
def test_rows_of_any_pitch_are_stored(device):
    heads, dim = 2, 64
    both = torch.randn(20, 2 * heads * dim + 12, device=device).bfloat16()
    k, v = (both[:, i * heads * dim + 4:(i + 1) * heads * dim + 4].view(20, heads, dim) for i in range(2))
    slots = torch.arange(16, 36, device=device)
    pages = [Pages8.empty(4, heads, dim, device) for _ in "kv"]
    want = [stored(x, slots, p) for x, p in zip((k, v), pages)]
    ops.store_kv(k, v, slots, *pages)
    for p, (codes, scales) in zip(pages, want):
        assert torch.equal(p.codes.double().cpu(), codes) and torch.equal(p.scales.double().cpu(), scales)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_what_is_no_number_marks_its_block(device, bad):
    heads, dim = 2, 64
    k = torch.ones((3, heads, dim), dtype=torch.bfloat16, device=device)
    k[1, 1, 7] = bad
    pages = [Pages8.empty(3, heads, dim, device) for _ in "kv"]
    slots = torch.tensor([16, 17, 33], device=device)
    ops.store_kv(k, torch.ones_like(k), slots, *pages)
    s = pages[0].scales.cpu()
    assert s[1, 1].isnan() and s[1, 0] == 2.0 ** -6 and (s[2] == 2.0 ** -6).all() and not pages[1].scales.isnan().any()
    # it stays so for the rows behind, and ends when the block is opened again
    ops.store_kv(torch.ones_like(k[:1]), torch.ones_like(k[:1]), torch.tensor([18], device=device), *pages)
    assert pages[0].scales[1, 1].isnan()
    ops.store_kv(torch.ones_like(k[:1]), torch.ones_like(k[:1]), torch.tensor([16], device=device), *pages)
    assert pages[0].scales[1].tolist() == [2.0 ** -6] * 2


@pytest.mark.parametrize("device", DEVICES)
def test_raised_scales_keep_values_within_one_step(device):
    """Sixteen rows, each twice as large as the last: every block's scale is raised up to fifteen times."""
    heads, dim = 2, 128
    g = torch.Generator().manual_seed(1)
    x = ((torch.rand((16, heads, dim), generator=g) * 2 - 1) * torch.exp2(torch.arange(16.0))[:, None, None]).bfloat16().to(device)
    pages = [Pages8.empty(2, heads, dim, device) for _ in "kv"]
    for i in range(16):
        ops.store_kv(x[i:i + 1], x[i:i + 1], torch.tensor([16 + i], device=device), *pages)
    off = (pages[0].values()[1].transpose(0, 1) - x.float()).abs()
    assert (off <= pages[0].scales[1][None, :, None]).all()
    # the last row has been rounded once
    assert (off[15] <= pages[0].scales[1][:, None] / 2).all()


ROPE = [dict(), dict(rot=32), dict(interleaved=True), dict(rot=16, interleaved=True), dict(norm=True), dict(norm=True, norm_w_off=1.0, attn_factor=1.3)]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("n_q, n_kv, dim", [(4, 4, 64), (12, 2, 128), (32, 8, 128), (5, 1, 64)])
@pytest.mark.parametrize("how", range(len(ROPE)))
@pytest.mark.parametrize("start, new", [((0, 70000, 9), (1, 1, 1)), ((30, 0), (290, 50))])
def test_rope_kv_writes_8_bits(device, n_q, n_kv, dim, how, start, new):
    how = dict(ROPE[how])
    norm = how.pop("norm", False)
    rot = how.get("rot", dim)
    rows = sum(new)
    g = torch.Generator().manual_seed(n_q + dim)
    qkv = torch.randn((rows, (n_q + 2 * n_kv) * dim + 8), generator=g).bfloat16().to(device)[:, :(n_q + 2 * n_kv) * dim]
    weights = [(1 + 0.1 * torch.randn(dim, generator=g)).to(device) if norm else None for _ in "qk"]
    inv_freq = torch.tensor([10000.0 ** (-2 * i / rot) for i in range(rot // 2)]).to(device)
    num, table = layout([n + a % PAGE for a, n in zip(start, new)], device)
    positions = torch.cat([torch.arange(a, a + n) for a, n in zip(start, new)])
    slots = torch.cat([table.cpu()[b, (at := torch.arange(a % PAGE, a % PAGE + n)) // PAGE].long() * PAGE + at % PAGE for b, (a, n) in enumerate(zip(start, new))])
    pages = [filled(num, n_kv, dim, device, seed=i) for i in range(2)]
    # in 64 bits
    x = qkv.double().cpu().view(rows, n_q + 2 * n_kv, dim)
    q, k, v = x.split((n_q, n_kv, n_kv), 1)
    ang = positions.double()[:, None] * inv_freq.double().cpu()
    factor = how.get("attn_factor", 1.0)
    cos, sin = ang.cos()[:, None] * factor, ang.sin()[:, None] * factor

    def turned(t, w):
        if w is not None:
            t = t * torch.rsqrt(t.square().mean(-1, keepdim=True) + 1e-6) * (w.double().cpu() + how.get("norm_w_off", 0.0))
        y = t.clone()
        a, b = (slice(0, rot, 2), slice(1, rot, 2)) if how.get("interleaved") else (slice(0, rot // 2), slice(rot // 2, rot))
        y[..., a], y[..., b] = t[..., a] * cos - t[..., b] * sin, t[..., b] * cos + t[..., a] * sin
        return y

    q, k = turned(q, weights[0]), turned(k, weights[1])
    want_k, want_v = stored(k, slots, pages[0]), stored(v, slots, pages[1])
    before = pages[0].codes.cpu().clone()
    got = ops.rope_kv(qkv, positions.to(torch.int32).to(device), slots.to(device), inv_freq, *pages, n_q, n_kv, dim, q_norm_w=weights[0],
                      k_norm_w=weights[1], norm_eps=1e-6, **how)
    # 32-bit arithmetic in front of one rounding to bf16: sums of a norm, an angle's sine and cosine, two products (the CPU's angles are single products)
    fine = 2.0 ** -18 if device == "cuda" else 2.0 ** -18 + 70000 * 2.0 ** -24
    assert got.shape == (rows, n_q, dim)
    assert ((got.double().cpu() - q).abs() <= 2.0 ** -8 * q.abs() + fine * q.abs().amax(-1, keepdim=True)).all()
    # values are rows as they are: exact
    assert torch.equal(pages[1].codes.double().cpu(), want_v[0]) and torch.equal(pages[1].scales.double().cpu(), want_v[1])
    # keys: a code may fall to the other side only where the quotient lies next to a border
    assert torch.equal(pages[0].scales.double().cpu(), want_k[1])
    off = (pages[0].codes.double().cpu() - want_k[0]).abs()
    assert off.max() <= 1 and (off > 0).float().mean() <= 200 * fine
    written = torch.zeros(before.shape[0], PAGE, dtype=torch.bool)
    written[slots // PAGE, slots % PAGE] = True
    tops = torch.zeros(before.shape[0], dtype=torch.long).scatter_reduce(0, slots // PAGE, slots % PAGE, "amax", include_self=True)
    behind = (torch.arange(PAGE) > tops[:, None]) | ~written.any(1)[:, None]
    assert torch.equal(pages[0].codes.cpu().transpose(1, 2)[behind], before.transpose(1, 2)[behind])     # left as they were


# ------------------------------------------------------------------------------------------ reading
@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("heads, dim", [(1, 64), (8, 128), (3, 64)])
def test_page_values(device, heads, dim):
    k, v = (filled(9, heads, dim, device, seed=i, spread=30.0) for i in range(2))
    pages = ints([3, 8, 3, 0], device)
    for got, t in zip(ops.page_values(k, v, pages), (k, v)):
        assert got.dtype == torch.bfloat16 and torch.equal(got.double(), t.codes[pages.long()].double() * t.scales[pages.long()].double()[..., None, None])
    assert ops.page_values(k, v, pages[:0])[0].shape == (0, heads, PAGE, dim)


def within(got, want, size, p_rounding):
    """``p_rounding``: half a step of the type that probabilities are rounded to; the sum they are divided by may hold them rounded or not. 2^-13
    for scores in 32 bits (up to 2^7 in units of ln 2, off by 2^-20 of that) and the exponential."""
    got = got.double().cpu()
    assert torch.isfinite(got).all()
    bound = (2 * p_rounding + 2.0 ** -13) * size + 2.0 ** -8 * want.abs() + 2.0 ** -120
    worst = ((got - want).abs() / bound).max()
    assert worst <= 1, worst


LENS = [(1,), (0, 5), (15, 16, 17), (250, 3, 1000), (2049,)]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("n_q, n_kv, dim", [(1, 1, 64), (8, 8, 128), (32, 8, 128), (32, 8, 64), (8, 1, 128), (24, 2, 64), (20, 1, 128)])
@pytest.mark.parametrize("q_per_seq, window, chunk, sinks, splits", [(1, 0, 0, False, 1), (1, 0, 0, True, 2), (3, 100, 0, True, 3), (5, 0, 64, False, 8), (2, 1, 0, False, 11),
                                                                     (9, 0, 0, False, 40)])
@pytest.mark.parametrize("lens", range(len(LENS)))
def test_decode_attention(device, n_q, n_kv, dim, q_per_seq, window, chunk, sinks, splits, lens):
    seq_lens = LENS[lens]
    num, table = layout(seq_lens, device, wider=3)
    k, v = (filled(num, n_kv, dim, device, seed=i) for i in range(2))
    g = torch.Generator().manual_seed(n_q)
    q = torch.randn((len(seq_lens) * q_per_seq, n_q, dim), generator=g).bfloat16().to(device)
    s = torch.randn(n_q, generator=g).to(device) if sinks else None
    scale = 1.5 * dim ** -0.5
    got = ops.attention_decode(q, k, v, table, ints(seq_lens, device), q_per_seq, scale, splits=splits, window=window, sinks=s, chunk=chunk)
    within(got, *attended(q, k.values(), v.values(), table, seq_lens, [q_per_seq] * len(seq_lens), scale, window, chunk, s), 2.0 ** -11)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("n_q, n_kv, dim", [(4, 1, 64), (32, 8, 128), (6, 2, 128), (3, 3, 64)])
@pytest.mark.parametrize("old, new, window, chunk, sinks", [((0,), (1,), 0, 0, False), ((0, 5, 130), (300, 1, 45), 0, 0, True), ((700, 0), (20, 129), 100, 0, False), ((40, 130), (70, 9), 0, 64, False),
                                                            ((1000, 3, 0), (2, 0, 0), 0, 0, False)])
def test_prefill_attention(device, n_q, n_kv, dim, old, new, window, chunk, sinks):
    seq_lens = [a + n for a, n in zip(old, new)]
    num, table = layout(seq_lens, device, wider=2)
    k, v = (filled(num, n_kv, dim, device, seed=i) for i in range(2))
    g = torch.Generator().manual_seed(n_q)
    q = torch.randn((sum(new), n_q, dim), generator=g).bfloat16().to(device)
    s = torch.randn(n_q, generator=g).to(device) if sinks else None
    cu = ints([sum(new[:i]) for i in range(len(new) + 1)], device)
    for known in (0, max(seq_lens)):
        got = ops.attention_prefill(q, k, v, table, ints(seq_lens, device), cu, max(new), dim ** -0.5, window=window, sinks=s, chunk=chunk, max_kv_len=known)
        within(got, *attended(q, k.values(), v.values(), table, seq_lens, new, dim ** -0.5, window, chunk, s), 2.0 ** -8)


@pytest.mark.gpu
@pytest.mark.parametrize("n_q, n_kv, dim", [(8, 2, 64), (32, 8, 128), (7, 1, 128)])
@pytest.mark.parametrize("old, rows, window, chunk, sinks", [((4000,), 17, 0, 0, False), ((0, 500, 37), 9, 0, 0, True), ((300, 290), 33, 70, 0, False), ((90, 300), 12, 0, 64, True),
                                                             ((9000,), 21, 0, 0, False), ((100,), 130, 0, 0, False)])
def test_portions_of_equally_many_rows(n_q, n_kv, dim, old, rows, window, chunk, sinks):
    """Few rows behind what is cached, as many for every sequence, with and without the longest length known."""
    assert kv8.decode_pays(1, 45, 32, 8, 128, 512) and not kv8.decode_pays(1, 64, 32, 8, 128, 4160) and not kv8.decode_pays(1, 4096, 32, 8, 64, 4096)
    test_prefill_attention("cuda", n_q, n_kv, dim, old, (rows,) * len(old), window, chunk, sinks)


@pytest.mark.gpu
@pytest.mark.parametrize("n_q, n_kv, dim", [(8, 2, 64), (32, 8, 128), (7, 1, 128)])
@pytest.mark.parametrize("old, rows, window, chunk, sinks", [((4000,), 17, 0, 0, False), ((0, 500, 37), 9, 0, 0, True), ((300, 290), 33, 70, 0, False), ((90, 300), 12, 0, 64, True),
                                                             ((9000,), 21, 0, 0, False), ((100,), 130, 0, 0, False)])
def test_portions_that_the_caller_knows_to_be_equal(n_q, n_kv, dim, old, rows, window, chunk, sinks):
    seq_lens = [a + rows for a in old]
    num, table = layout(seq_lens, "cuda", wider=1)
    k, v = (filled(num, n_kv, dim, "cuda", seed=i) for i in range(2))
    q = torch.randn((rows * len(old), n_q, dim), generator=torch.Generator().manual_seed(rows)).bfloat16().cuda()
    s = torch.randn(n_q, device="cuda") if sinks else None
    cu = ints([rows * i for i in range(len(old) + 1)], "cuda")
    got = ops.attention_prefill(q, k, v, table, ints(seq_lens, "cuda"), cu, rows, dim ** -0.5, window=window, sinks=s, chunk=chunk, max_kv_len=max(seq_lens), equal=True)
    within(got, *attended(q, k.values(), v.values(), table, seq_lens, [rows] * len(old), dim ** -0.5, window, chunk, s), 2.0 ** -8)
    with pytest.raises(ValueError):
        ops.attention_prefill(q[1:], k, v, table, ints(seq_lens, "cuda"), cu, rows, dim ** -0.5, max_kv_len=max(seq_lens), equal=True)


def test_pages_that_are_seen():
    """Counted as defined: a page is seen when a key of it lies in some query's reach."""
    g = torch.Generator().manual_seed(0)
    for _ in range(300):
        old, new, wide = (int(torch.randint(0, n, (), generator=g)) for n in (200, 50, 20))
        window, chunk = ((0, 0), (1 + old % 70, 0), (0, 1 + new))[int(torch.randint(0, 3, (), generator=g))]
        seen = set()
        for pos in range(old, old + new):
            low = max(0, pos - window + 1) if window else pos - pos % chunk if chunk else 0
            seen |= {j // PAGE for j in range(low, pos + 1)}
        # (pages between those of the first and of the last query count, and so does the chunk of the first query)
        span = range(min(seen), max(seen) + 1) if seen else ()
        assert kv8.seen_pages([(old, new)], window, chunk, wide) == len([p for p in span if p < wide])
    assert kv8.seen_pages([(10, 3), (0, 0), (100, 0), (31, 2)], 0, 0, 99) == 1 + 3


@pytest.mark.gpu
@pytest.mark.parametrize("n_q, n_kv, dim", [(8, 2, 64), (32, 8, 128)])
@pytest.mark.parametrize("window, chunk, sinks", [(0, 0, False), (100, 0, True), (0, 64, False)])
@pytest.mark.parametrize("old, new", [((8000,) + (30,) * 40, (3,) + tuple(range(40))), ((500, 0, 900, 17), (40, 0, 200, 1)), ((0, 5), (1, 0)), ((3000,), (70,)), ((40,) * 300 + (600,), (2,) * 300 + (9,))])
def test_memory_of_a_prefill_is_what_its_sequences_see(n_q, n_kv, dim, window, chunk, sinks, old, new):
    """Beside the output and two tables; and the values are those of rows that are as wide as the longest."""
    seq_lens = [a + n for a, n in zip(old, new)]
    num, table = layout(seq_lens, "cuda", wider=2)
    k, v = (filled(num, n_kv, dim, "cuda", seed=i) for i in range(2))
    q = torch.randn((sum(new) + 5, n_q, dim), generator=torch.Generator().manual_seed(n_q)).bfloat16().cuda()   # rows behind the last: left as they were
    s = torch.randn(n_q, device="cuda") if sinks else None
    cu, lens = ints([sum(new[:i]) for i in range(len(new) + 1)], "cuda"), ints(seq_lens, "cuda")
    how = dict(window=window, sinks=s, chunk=chunk)
    want = ops.attention_prefill(q, k, v, table, lens, cu, max(new), dim ** -0.5, out=torch.full_like(q, 3.0), max_kv_len=max(seq_lens), **how)
    out = torch.full_like(q, 3.0)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    ops.attention_prefill(q, k, v, table, lens, cu, max(new), dim ** -0.5, out=out, max_kv_len=max(seq_lens), portions=list(zip(old, new)), **how)
    peak = torch.cuda.max_memory_allocated() - before
    seen = kv8.seen_pages(zip(old, new), window, chunk, table.shape[1])
    # the allocator rounds up to 2 MB at most where a block is taken apart
    assert peak <= 2 * 2 * max(1, seen) * n_kv * PAGE * dim + 4 * len(old) * (table.shape[1] + 8) + (2 << 20)
    assert torch.equal(out, want) and (out[sum(new):] == 3).all()
    ops.native.check_status(torch.device("cuda"))


@pytest.mark.gpu
def test_portions_that_are_not_those_of_the_device():
    """Sequences that are longer than the caller says: nothing is written behind what was allocated, and the status word says so. Wrong numbers of portions are refused."""
    lens, new = (400, 300), (20, 30)
    num, table = layout(lens, "cuda")
    k, v = (filled(num, 2, 64, "cuda", seed=i) for i in range(2))
    q = torch.randn((50, 8, 64), device="cuda").bfloat16()
    cu = ints([0, 20, 50], "cuda")
    with pytest.raises(ValueError, match="portions"):
        ops.attention_prefill(q, k, v, table, ints(lens, "cuda"), cu, 30, 0.1, portions=[(380, 20)])
    ops.attention_prefill(q, k, v, table, ints(lens, "cuda"), cu, 30, 0.1, max_kv_len=400, portions=[(10, 20), (270, 30)])
    with pytest.raises(RuntimeError, match="bad argument"):
        ops.native.check_status(torch.device("cuda"))


@pytest.mark.gpu
def test_padded_rows_of_a_prefill_are_left_as_they_were():
    """As many rows as sequences times the longest portion, some of them behind the last sequence."""
    n_q, n_kv, dim, lens, new = 8, 2, 128, (300, 40), (32, 20)
    num, table = layout(lens, "cuda")
    k, v = (filled(num, n_kv, dim, "cuda", seed=i) for i in range(2))
    q = torch.randn((64, n_q, dim), generator=torch.Generator().manual_seed(0)).bfloat16().cuda()
    out = torch.full_like(q, 7.0)
    ops.attention_prefill(q, k, v, table, ints(lens, "cuda"), ints([0, 32, 52], "cuda"), 32, dim ** -0.5, out=out, max_kv_len=300)
    within(out[:52], *attended(q[:52], k.values(), v.values(), table, lens, new, dim ** -0.5), 2.0 ** -8)
    assert (out[52:] == 7).all()


def expanded(pages, dim):
    """Pages whose scales differ by far more than f16 holds."""
    g = torch.Generator().manual_seed(5)
    pages.scales.copy_(torch.exp2(torch.randint(-60, 41, pages.scales.shape, generator=g).float()))
    return pages


@pytest.mark.gpu
@pytest.mark.parametrize("seed", [0, 795])
@pytest.mark.parametrize("splits", [1, 4, 12])
def test_decode_attention_of_far_apart_scales(splits, seed):
    """Values from 2^-60 to 2^47 beside one another. f16 rounds what a token weighs, its probability times its scale, to 11 bits down to 2^-14 of the row's
    largest, and to a multiple of 2^-24 of it below: there a token is off by half of that, 2^-25 times its code. A channel in which the largest tokens have codes of zero
    consists of such (seed 795 has one)."""
    dim, seq_lens, scale = 128, (400, 1700), 0.3
    num, table = layout(seq_lens, "cuda")
    k, v = filled(num, 2, dim, "cuda"), expanded(filled(num, 2, dim, "cuda", seed=1), dim)
    q = torch.randn((2, 8, dim), generator=torch.Generator().manual_seed(seed)).bfloat16().cuda()

    def fits(got, queries, scale):
        want, size = attended(queries, k.values(), v.values(), table, seq_lens, (1, 1), scale)
        least = torch.zeros_like(size)
        for b, n in enumerate(seq_lens):
            at = table[b, :-(-n // PAGE)].long().cpu()
            for h in range(8):
                keys, codes = (t.double().cpu()[at, h // 4].reshape(-1, dim)[:n] for t in (k.values(), v.codes))
                weight = torch.softmax(keys @ queries[b, h].double().cpu() * scale, 0) * v.scales.double().cpu()[at, h // 4].repeat_interleave(PAGE)[:n]
                least[b, h] = 2.0 ** -25 * weight.max() * codes.abs().sum(0)
        # (as a part of what `within` allows for the size)
        within(got, want, size + least / (2 * 2.0 ** -11 + 2.0 ** -13), 2.0 ** -11)

    fits(ops.attention_decode(q, k, v, table, ints(seq_lens, "cuda"), 1, scale, splits=splits), q, scale)
    # and queries as small and as large as bf16 holds, with a scale of scores to match
    for size in (2.0 ** -120, 2.0 ** 100):
        far = (q.float() * size).bfloat16()
        fits(ops.attention_decode(far, k, v, table, ints(seq_lens, "cuda"), 1, scale / size, splits=splits), far, scale / size)


@pytest.mark.gpu
def test_what_is_no_number_reaches_only_those_who_see_it():
    dim, seq_lens = 64, (40, 40)
    num, table = layout(seq_lens, "cuda")
    k, v = (filled(num, 1, dim, "cuda", seed=i) for i in range(2))
    q = torch.randn((4, 4, dim), device="cuda").bfloat16()
    v.scales[table[0, 2].item()] = math.nan           # the last eight tokens of the first sequence, seen by its second query alone in windows of 7
    k.scales[table[1, 0].item()] = math.nan           # the first page of the second sequence
    got = ops.attention_decode(q, k, v, table, ints(seq_lens, "cuda"), 2, 0.1, window=7)
    assert got[:2].isnan().all() and not got[2:].isnan().any()
    got = ops.attention_decode(q, k, v, table, ints([32, 40], "cuda"), 2, 0.1)
    assert not got[:2].isnan().any() and got[2:].isnan().all()
    # a query that is no number
    q[0, 1, 3], q[1, 2, 5] = math.nan, math.inf
    got = ops.attention_decode(q, k, v, table, ints([32, 40], "cuda"), 2, 0.1)
    assert got[0, 1].isnan().all() and not got[0, [0, 2, 3]].isnan().any() and got[1, 2].isnan().all()


@pytest.mark.gpu
@pytest.mark.parametrize("dim, n_q, n_kv", [(64, 4, 1), (128, 32, 2)])
@pytest.mark.parametrize("splits", [1, 3, 0])
@pytest.mark.parametrize("apart", [0.0, 200.0])
def test_values_that_are_no_numbers_give_none(dim, n_q, n_kv, splits, apart):
    """A block of values that a write has marked: every code is the same, so that no sum of products of both signs stands in for what is no number. Also where the
    block's tokens weigh nothing (scores that are ``apart`` below the others' in units of log2: a product of zero and no number is none)."""
    seq_lens = (400, 90)
    num, table = layout(seq_lens, "cuda")
    k, v = (filled(num, n_kv, dim, "cuda", seed=i) for i in range(2))
    q = torch.ones((2, n_q, dim), dtype=torch.bfloat16, device="cuda")
    k.codes.fill_(1)
    k.scales.fill_(1.0)
    marked = table[0, 7].item()
    rows = torch.full((PAGE, n_kv, dim), 1 - apart / dim, dtype=torch.bfloat16, device="cuda")
    bad = torch.ones_like(rows)
    bad[3, :, 5] = math.nan
    ops.store_kv(rows, bad, torch.arange(marked * PAGE, (marked + 1) * PAGE, device="cuda"), k, v)
    assert v.scales[marked].isnan().all()
    got = ops.attention_decode(q, k, v, table, ints(seq_lens, "cuda"), 1, math.log(2.0), splits=splits)
    assert got[0].isnan().all() and torch.isfinite(got[1]).all()
    cu = ints([0, 1, 2], "cuda")
    assert ops.attention_prefill(q, k, v, table, ints(seq_lens, "cuda"), cu, 1, math.log(2.0))[0].isnan().all()
    # and where nobody sees it, nobody has it
    got = ops.attention_decode(q, k, v, table, ints(seq_lens, "cuda"), 1, math.log(2.0), splits=splits, window=200)
    assert torch.isfinite(got).all()


@pytest.mark.gpu
def test_block_tables_that_are_part_of_a_wider_one():
    """Rows of another pitch than their width; lengths that say more than the table has are cut there, and nothing behind the table is read."""
    seq_lens = (70, 33)
    num, table = layout(seq_lens, "cuda")
    k, v = (filled(num, 2, 64, "cuda", seed=i) for i in range(2))
    q = torch.randn((2, 8, 64), generator=torch.Generator().manual_seed(1)).bfloat16().cuda()
    lens, cu = ints(seq_lens, "cuda"), ints([0, 1, 2], "cuda")
    wide = torch.full((2, 40), 1 << 20, dtype=torch.int32, device="cuda")
    part = wide[:, 30:30 + table.shape[1]]
    part.copy_(table)
    for splits in (1, 3, 0):
        assert torch.equal(ops.attention_decode(q, k, v, part, lens, 1, 0.1, splits=splits), ops.attention_decode(q, k, v, table, lens, 1, 0.1, splits=splits))
    assert torch.equal(ops.attention_prefill(q, k, v, part, lens, cu, 1, 0.1), ops.attention_prefill(q, k, v, table, lens, cu, 1, 0.1))
    short = wide[:, 30:32]
    for splits in (1, 3, 0):
        got = ops.attention_decode(q, k, v, short, lens, 1, 0.1, splits=splits)
        within(got, *attended(q, k.values(), v.values(), table, (32, 32), (1, 1), 0.1), 2.0 ** -11)
    ops.native.check_status(torch.device("cuda"))


@pytest.mark.gpu
def test_pages_behind_four_gigabytes():
    """Codes at offsets that no 32-bit number holds."""
    heads, dim, num = 8, 128, 270_000
    k, v = (Pages8(torch.empty((num, heads, PAGE, dim), dtype=torch.int8, device="cuda"), torch.empty((num, heads), device="cuda")) for _ in "kv")
    g = torch.Generator().manual_seed(3)
    rows = torch.randn((2, 37, heads, dim), generator=g).bfloat16().cuda()
    table = ints([[num - 1, 5, num - 70]], "cuda")
    at = torch.arange(37)
    slots = (table[0].cpu()[at // PAGE].long() * PAGE + at % PAGE).cuda()
    ops.store_kv(rows[0], rows[1], slots, k, v)
    q = torch.randn((1, 32, dim), generator=g).bfloat16().cuda()
    small = [Pages8(t.codes[table[0].long()], t.scales[table[0].long()]) for t in (k, v)]
    near = torch.arange(3, dtype=torch.int32, device="cuda")[None]
    lens = ints([37], "cuda")
    assert torch.equal(ops.attention_decode(q, k, v, table, lens, 1, 0.1), ops.attention_decode(q, *small, near, lens, 1, 0.1))
    cu = ints([0, 1], "cuda")
    assert torch.equal(ops.attention_prefill(q, k, v, table, lens, cu, 1, 0.1), ops.attention_prefill(q, *small, near, lens, cu, 1, 0.1))
    off = (small[0].values().transpose(1, 2).reshape(-1, heads, dim)[:37] - rows[0].float()).abs()
    assert (off <= small[0].scales[at.cuda() // PAGE][..., None] / 2).all()
    ops.copy_pages((k.codes[None], v.codes[None]), [num - 1], [num - 2])
    assert torch.equal(k.codes[num - 1], k.codes[num - 2]) and torch.equal(v.codes[num - 1], v.codes[num - 2])


@pytest.mark.gpu
def test_steps_captured_and_replayed_beside_others():
    """Two captured steps (each with partial sums of its own) and an eager one, on three streams, repeatedly: what each gives alone."""
    n_q, n_kv, dim = 8, 2, 128
    steps = []
    for i, splits in enumerate((12, 12, 3)):
        seq_lens = (900 + 10 * i, 350)
        num, table = layout(seq_lens, "cuda", seed=i)
        k, v = (filled(num, n_kv, dim, "cuda", seed=2 * i + j) for j in range(2))
        old = [n - 1 for n in seq_lens]
        args = dict(qkv=torch.randn((2, (n_q + 2 * n_kv) * dim), device="cuda").bfloat16(), positions=ints(old, "cuda"),
                    slots=torch.stack([table[b, n // PAGE].long() * PAGE + n % PAGE for b, n in enumerate(old)]), lens=ints(seq_lens, "cuda"))
        freq = torch.tensor([1e4 ** (-2 * j / dim) for j in range(dim // 2)], device="cuda")
        steps.append(lambda a=args, k=k, v=v, t=table, s=splits, f=freq: ops.attention_decode_rope(
            a["qkv"], k, v, t, a["lens"], 1, dim ** -0.5, a["positions"], a["slots"], f, n_q, n_kv, dim, splits=s))
    want = [f().clone() for f in steps]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for f in steps[:2]:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(f())
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in range(3)]
    for _ in range(20):
        for s, graph in zip(streams, graphs):
            with torch.cuda.stream(s):
                graph.replay()
        with torch.cuda.stream(streams[2]):
            last = steps[2]()
    torch.cuda.synchronize()
    ops.native.check_status(torch.device("cuda"))
    assert all(torch.equal(a, b) for a, b in zip(outs + [last], want))


# ------------------------------------------------------------------------------------------ one step
@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("n_q, n_kv, dim", [(4, 4, 64), (32, 8, 128), (32, 4, 128), (18, 2, 64)])
@pytest.mark.parametrize("old, new, norm", [((0,), 1, False), ((15, 700, 16), 1, True), ((30, 0, 333), 5, False), ((1040, 14), 8, True)])
@pytest.mark.parametrize("splits", [1, 4, 10])
def test_decode_step_from_the_projection(device, n_q, n_kv, dim, old, new, norm, splits):
    """Rotation, write and attention in one call: pages as rope_kv leaves them, attention over these pages."""
    seq_lens = [a + new for a in old]
    num, table = layout(seq_lens, device, wider=1)
    g = torch.Generator().manual_seed(n_q + sum(old))
    rows = len(old) * new
    qkv = (torch.randn((rows, (n_q + 2 * n_kv) * dim), generator=g) * 2).bfloat16().to(device)
    weights = [(1 + 0.1 * torch.randn(dim, generator=g)).to(device) if norm else None for _ in "qk"]
    freq = torch.tensor([1e4 ** (-2 * j / dim) for j in range(dim // 2)], device=device)
    at = torch.cat([torch.arange(a, a + new) for a in old])
    seq = torch.repeat_interleave(torch.arange(len(old)), new)
    slots = table.cpu()[seq, at // PAGE].long() * PAGE + at % PAGE
    pages = [filled(num, n_kv, dim, device, seed=i) for i in range(2)]
    again = [Pages8(p.codes.clone(), p.scales.clone()) for p in pages]
    common = dict(q_norm_w=weights[0], k_norm_w=weights[1], norm_eps=1e-6)
    got = ops.attention_decode_rope(qkv, *pages, table, ints(seq_lens, device), new, dim ** -0.5, at.to(torch.int32).to(device), slots.to(device), freq, n_q, n_kv,
                                    dim, splits=splits, **common)
    q = ops.rope_kv(qkv, at.to(torch.int32).to(device), slots.to(device), freq, *again, n_q, n_kv, dim, **common)
    for a, b in zip(pages, again):
        assert torch.equal(a.codes, b.codes) and torch.equal(a.scales, b.scales)
    want, size = attended(q, pages[0].values(), pages[1].values(), table, seq_lens, [new] * len(old), dim ** -0.5)
    # the step may keep queries in more bits than rope_kv returns: half a bf16 step in every component moves a score by 2^-8 of the sum of |q k|
    moved, start = 0.0, 0
    for b, n in enumerate(seq_lens):
        pg = table[b, :-(-n // PAGE)].long()
        for h in range(n_kv):
            kk = pages[0].values()[pg, h].reshape(-1, dim)[:n].double().cpu()
            qq = q[start:start + new, h * (n_q // n_kv):(h + 1) * (n_q // n_kv)].double().cpu().reshape(-1, dim)
            moved = max(moved, float((qq.abs() @ kk.abs().t()).max()) * dim ** -0.5 * 2.0 ** -8)
        start += new
    got = got.double().cpu()
    bound = (2 * 2.0 ** -11 + 2.0 ** -13 + 2 * math.expm1(moved)) * size + 2.0 ** -8 * want.abs() + 2.0 ** -120
    assert ((got - want).abs() <= bound).all()


@pytest.mark.gpu
@pytest.mark.parametrize("n_q, n_kv, dim", [(8, 2, 64), (8, 2, 128)])
@pytest.mark.parametrize("old, new", [((4203,), 3), ((2046, 250), 4), ((127, 4095), 1)])
@pytest.mark.parametrize("splits", [1, 2])
def test_steps_far_behind_what_a_warp_reads_first(n_q, n_kv, dim, old, new, splits):
    """New rows in pages that a CTA comes to late, and in the first ones of its second look at the table."""
    test_decode_step_from_the_projection("cuda", n_q, n_kv, dim, old, new, False, splits)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("n_q, n_kv, dim", [(4, 4, 64), (16, 4, 128)])
@pytest.mark.parametrize("settled", [False, True])
def test_rows_of_a_step_that_are_not_stored(device, n_q, n_kv, dim, settled):
    """Sequences of which the first, the last or no new rows go to their pages: attention reads what is there."""
    new, old = 4, (30, 13, 44, 100)
    seq_lens = [a + new for a in old]
    num, table = layout(seq_lens, device)
    g = torch.Generator().manual_seed(dim)
    qkv = torch.randn((len(old) * new, (n_q + 2 * n_kv) * dim), generator=g).bfloat16().to(device)
    freq = torch.tensor([1e4 ** (-2 * j / dim) for j in range(dim // 2)], device=device)
    at = torch.cat([torch.arange(a, a + new) for a in old])
    seq = torch.repeat_interleave(torch.arange(len(old)), new)
    slots = table.cpu()[seq, at // PAGE].long() * PAGE + at % PAGE
    slots[[0, 1, 7, 8, 9, 10, 11]] = -1
    slots, at = slots.to(device), at.to(torch.int32).to(device)
    pages = [filled(num, n_kv, dim, device, seed=i) for i in range(2)]
    again = [Pages8(p.codes.clone(), p.scales.clone()) for p in pages]
    got = ops.attention_decode_rope(qkv, *pages, table, ints(seq_lens, device), new, dim ** -0.5, at, slots, freq, n_q, n_kv, dim, splits=2, settled=settled)
    q = ops.rope_kv(qkv, at, slots, freq, *again, n_q, n_kv, dim)
    for a, b in zip(pages, again):
        assert torch.equal(a.codes, b.codes) and torch.equal(a.scales, b.scales)
    want, size = attended(q, pages[0].values(), pages[1].values(), table, seq_lens, [new] * len(old), dim ** -0.5)
    keys = pages[0].values().double().abs().amax((0, 2)).cpu()                 # [n_kv, dim]: no key is larger
    most = (q.double().cpu().abs().view(-1, n_kv, n_q // n_kv, dim) * keys[None, :, None]).sum(-1).max()
    moved = float(most) * dim ** -0.5 * 2.0 ** -8                              # half a bf16 step in every component of a query
    bound = (2 * 2.0 ** -11 + 2.0 ** -13 + 2 * math.expm1(moved)) * size + 2.0 ** -8 * want.abs() + 2.0 ** -120
    assert ((got.double().cpu() - want).abs() <= bound).all()


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [33, 300, 700, 2000])
@pytest.mark.parametrize("n_q, n_kv, dim, rot", [(8, 8, 128, 128), (14, 2, 64, 64), (3, 3, 128, 32), (32, 2, 64, 8)])
def test_runs_of_all_kinds_whatever_tile_they_begin_in(rows, n_q, n_kv, dim, rot):
    """Runs of any length and offset with rows between them that are not stored. The angles are zero, so that codes and scales are those of the rows themselves."""
    g = torch.Generator().manual_seed(rows + n_q)
    draw = lambda low, high: int(torch.randint(low, high + 1, (), generator=g))     # noqa: E731
    slots, page = [], 0
    while len(slots) < rows:
        if draw(0, 9) == 0:
            slots += [-1] * draw(1, 5)
        first = draw(0, 15) if draw(0, 2) == 0 else 0
        slots += [page * PAGE + first + i for i in range(16 - first if draw(0, 1) else draw(1, 16 - first))]
        page += 1
    slots = torch.tensor(slots[:rows])
    x = (torch.randn((rows, (n_q + 2 * n_kv) * dim), generator=g) * torch.exp(torch.randn((rows, 1), generator=g))).bfloat16()
    pages = [filled(page, n_kv, dim, "cpu", seed=i) for i in range(2)]
    have = [Pages8(p.codes.cuda(), p.scales.cuda()) for p in pages]
    k, v = x.view(rows, -1, dim)[:, n_q:].split(n_kv, 1)
    for part, p in zip((k, v), pages):
        kv8.store_rows_ref(part, slots, p)
    q = ops.rope_kv(x.cuda(), torch.arange(rows, dtype=torch.int32, device="cuda"), slots.cuda(), torch.zeros(rot // 2, device="cuda"), *have, n_q, n_kv, dim, rot=rot)
    assert torch.equal(q.cpu().view(rows, -1), x[:, :n_q * dim])
    for a, b in zip(have, pages):
        assert torch.equal(a.scales.cpu(), b.scales) and torch.equal(a.codes.cpu(), b.codes)


def test_argument_blocks_hold_what_the_header_declares():
    """Pointers, then ints, then floats, as many of each as the formats have."""
    header = (Path(ops.__file__).resolve().parent.parent / "csrc/common/kv8_args.h").read_text()
    for name, block in (("Kv8StoreArgs", kv8._STORE), ("Kv8ValuesArgs", kv8._VALUES), ("Kv8AttentionArgs", kv8._ATTENTION)):
        body = re.sub(r"//.*", "", re.search(rf"struct {name} {{(.*?)}};", header, re.S).group(1))
        kinds = ""
        for line in filter(None, (part.strip() for part in body.split(";"))):
            pointer = "*" in line or line.startswith("cudaStream_t")
            kinds += ("Q" if pointer else "f" if line.startswith("float ") else "i") * len(line.split(","))
        assert "".join(letter * int(n) for n, letter in re.findall(r"(\d+)([Qif])", block.format)) == kinds, name


@pytest.mark.gpu
@pytest.mark.parametrize("name, block", [("eredu_kv8_store", kv8._STORE), ("eredu_kv8_values", kv8._VALUES), ("eredu_attn_kv8_decode", kv8._ATTENTION),
                                         ("eredu_attn_kv8_step", kv8._ATTENTION)])
def test_argument_blocks_are_as_long_as_the_library_has_them(name, block):
    call, nothing = getattr(ops.native.lib(), name), bytes(block.size)        # no rows, no sequences: nothing is launched
    assert call(nothing, block.size) == 0
    assert call(nothing + b"    ", block.size + 4) != 0 and call(nothing, 8) != 0


# ------------------------------------------------------------------------------------------ moving
@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("kind, heads, dim", [(torch.bfloat16, 8, 128), (torch.float32, 1, 4), (torch.int8, 3, 64), (torch.bfloat16, 1, 1)])
def test_pages_are_copied_in_all_layers(device, kind, heads, dim):
    g = torch.Generator().manual_seed(0)
    pools = [torch.randint(-100, 100, (layers, 12, heads, PAGE, dim), generator=g).to(kind).to(device) for layers in (3, 3, 1)]
    pools.append(torch.randn((3, 12, heads), generator=g).to(device))
    want = [p.clone() for p in pools]
    src, dst = [3, 11, 4], [1, 2, 7]
    for w in want:
        w[:, dst] = w[:, src]
    lists = [ints(x, device) for x in (src, dst)] if device == "cuda" else [src, dst]
    ops.copy_pages(pools, *lists)
    assert all(torch.equal(a, b) for a, b in zip(pools, want))
    ops.copy_pages(pools, src, dst)
    assert all(torch.equal(a, b) for a, b in zip(pools, want))
    ops.copy_pages(pools, [], [])


@pytest.mark.gpu
def test_more_tensors_than_one_launch_holds():
    pools = [torch.randn((2, 5, 3, PAGE, 8), device="cuda") for _ in range(11)]
    want = [p.clone() for p in pools]
    for w in want:
        w[:, 4] = w[:, 1]
    ops.copy_pages(pools, [1], [4])
    assert all(torch.equal(a, b) for a, b in zip(pools, want))


# ------------------------------------------------------------------------------------------ refusals
def test_copies_that_are_refused():
    pools = [torch.zeros((2, 6, 1, PAGE, 4))]
    for src, dst, kind in [([1], [6], IndexError), ([-1], [2], IndexError), ([1, 2], [3, 3], ValueError), ([1, 2], [2, 3], ValueError), ([1, 2], [3], ValueError)]:
        with pytest.raises(kind):
            ops.copy_pages(pools, src, dst)
    with pytest.raises(ValueError, match="same pages"):
        ops.copy_pages([pools[0], torch.zeros((2, 7, 1, PAGE, 4))], [1], [2])
    with pytest.raises(ValueError, match="contiguous"):
        ops.copy_pages([torch.zeros((2, 6, 4, PAGE)).transpose(2, 3)], [1], [2])
    with pytest.raises(ValueError, match="words"):
        ops.copy_pages([torch.zeros((2, 6, 3), dtype=torch.int8)], [1], [2])


@pytest.mark.parametrize("device", DEVICES)
def test_pages_that_are_refused(device):
    k, v = (Pages8.empty(4, 2, 64, device) for _ in "kv")
    rows, slots = torch.zeros((3, 2, 64), dtype=torch.bfloat16, device=device), torch.arange(16, 19, device=device)
    ops.store_kv(rows, rows, slots, k, v)
    with pytest.raises(TypeError):
        ops.store_kv(rows, rows, slots, k, v.codes)
    with pytest.raises(ValueError, match="do not go together"):
        ops.store_kv(rows, rows, slots[:2], k, v)
    with pytest.raises(ValueError, match="no pages of"):
        ops.store_kv(rows[:, :1], rows[:, :1], slots, k, v)
    with pytest.raises(ValueError, match="no pages of"):
        ops.store_kv(rows, rows, slots, k, Pages8(v.codes, v.scales.double()))
    with pytest.raises(ValueError, match="contiguous"):
        ops.store_kv(rows, rows, slots, k, Pages8(torch.zeros((4, 2, 64, PAGE), dtype=torch.int8, device=device).transpose(2, 3), v.scales))
    with pytest.raises(ValueError, match="same pages"):
        ops.store_kv(rows, rows, slots, k, Pages8.empty(5, 2, 64, device))
    if device == "cpu":
        with pytest.raises(IndexError):
            ops.store_kv(rows, rows, slots + 48, k, v)


@pytest.mark.gpu
def test_slots_and_pages_out_of_range_are_reported():
    """The kernels check them: nothing is written or read there, and the status word says so."""
    dev = torch.device("cuda")
    k, v = (Pages8.empty(4, 2, 64, dev) for _ in "kv")
    rows = torch.ones((3, 2, 64), dtype=torch.bfloat16, device=dev)
    ops.store_kv(rows, rows, torch.tensor([16, 64, 1 << 40], device=dev), k, v)
    with pytest.raises(RuntimeError, match="bad argument"):
        ops.native.check_status(dev)
    assert (k.codes[1, :, 0] == 64).all() and not k.codes[2:].any()
    ops.copy_pages((k.codes[None], v.codes[None]), ints([1, 1], dev), ints([2, 4], dev))
    with pytest.raises(RuntimeError, match="bad argument"):
        ops.native.check_status(dev)
    assert torch.equal(k.codes[2], k.codes[1])
    q = torch.zeros((1, 2, 64), dtype=torch.bfloat16, device=dev)
    ops.attention_decode(q, k, v, ints([[1, 9]], dev), ints([20], dev), 1, 1.0)
    with pytest.raises(RuntimeError, match="bad argument"):
        ops.native.check_status(dev)
    ops.page_values(k, v, ints([-1], dev))
    with pytest.raises(RuntimeError, match="bad argument"):
        ops.native.check_status(dev)


@pytest.mark.gpu
def test_calls_that_are_refused_on_a_gpu():
    dev = torch.device("cuda")
    k, v = (Pages8.empty(4, 2, 64, dev) for _ in "kv")
    q = torch.zeros((2, 4, 64), dtype=torch.bfloat16, device=dev)
    table, lens = ints([[1], [2]], dev), ints([3, 4], dev)
    ops.attention_decode(q, k, v, table, lens, 1, 1.0)
    bad = [dict(q=q.float()), dict(q=q[:1]), dict(q=q.transpose(0, 1)), dict(q=q[:, :3].contiguous()), dict(lens=lens.long()), dict(table=table.long()), dict(table=table[:1]), dict(table=table.cpu()),
           dict(sinks=torch.zeros(3, device=dev)), dict(out=torch.zeros((2, 4, 32), dtype=torch.bfloat16, device=dev))]
    for change in bad:
        a = dict(q=q, table=table, lens=lens, sinks=None, out=None) | change
        with pytest.raises(ValueError):
            ops.attention_decode(a["q"], k, v, a["table"], a["lens"], 1, 1.0, sinks=a["sinks"], out=a["out"])
    for pair in ((k, v.codes), (k.codes, v)):
        with pytest.raises(TypeError):
            ops.attention_decode(q, *pair, table, lens, 1, 1.0)
        with pytest.raises(TypeError):
            ops.attention_prefill(q, *pair, table, lens, ints([0, 1, 2], dev), 1, 1.0)
    with pytest.raises(NotImplementedError):
        wide = [Pages8.empty(4, 2, 256, dev) for _ in "kv"]
        ops.attention_decode(torch.zeros((2, 4, 256), dtype=torch.bfloat16, device=dev), *wide, table, lens, 1, 1.0)
    with pytest.raises(ValueError):
        ops.attention_prefill(q, k, v, table, lens, ints([0, 2], dev), 2, 1.0)
    qkv, pos, slots = torch.zeros((2, 8 * 64), dtype=torch.bfloat16, device=dev), ints([0, 0], dev), torch.tensor([16, 32], device=dev)
    freq = torch.ones(32, device=dev)
    ops.rope_kv(qkv, pos, slots, freq, k, v, 4, 2, 64)
    for change in [dict(qkv=qkv.float()), dict(qkv=qkv[:, :400]), dict(pos=pos.long()), dict(slots=slots.int()), dict(freq=freq[:16]), dict(pos=pos[:1])]:
        a = dict(qkv=qkv, pos=pos, slots=slots, freq=freq) | change
        with pytest.raises(ValueError):
            ops.rope_kv(a["qkv"], a["pos"], a["slots"], a["freq"], k, v, 4, 2, 64)
    with pytest.raises(NotImplementedError):
        ops.attention_decode_rope(qkv, k, v, table, lens, 1, 1.0, pos, slots, freq, 4, 2, 64, value_norm=True, norm_whole=True)
