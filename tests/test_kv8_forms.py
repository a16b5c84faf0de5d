"""Steps over 8-bit pages in all their forms, rows that are taken back and written again, and what a user of speculation over such pages gets."""
import math

import pytest
import torch

from eredu_b200 import ops
from eredu_b200.ops import kv8
from eredu_b200.ops.kv8 import PAGE, Pages8
from eredu_b200.runtime.engine import Engine
from eredu_b200.runtime.speculative import SpeculativeDecoder
from test_kv8 import attended, filled, ints, layout, stored
from test_kv8_engine import GREEDY, build, pages_of, prompt

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


# ------------------------------------------------------------------------------------------ the step's forms
@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("n_q, n_kv, dim", [(4, 4, 64), (32, 8, 128), (24, 2, 64), (32, 4, 128)])
@pytest.mark.parametrize("how", [dict(rot=32), dict(interleaved=True), dict(rot=16, interleaved=True), dict(rot=8, norm=True, norm_w_off=1.0),
                                 dict(norm=True, interleaved=True, attn_factor=1.3)])
@pytest.mark.parametrize("old, new, window, chunk, sinks", [((70, 0, 333), 2, 40, 0, True), ((30, 126, 64), 4, 0, 32, False), ((15, 250), 1, 7, 0, False), ((1000,), 5, 300, 0, True)])
@pytest.mark.parametrize("splits", [1, 3, 0])
def test_steps_of_all_forms(device, n_q, n_kv, dim, how, old, new, window, chunk, sinks, splits):
    """Rotations of a part, of neighbours, with norms and factors, under windows, chunks and sinks: pages as rope_kv leaves them, attention over these pages.
    Rows begin inside a window's first page, a chunk and a page."""
    how = dict(how)
    norm = how.pop("norm", False)
    rot = how.get("rot", dim)
    seq_lens = [a + new for a in old]
    num, table = layout(seq_lens, device, wider=1)
    g = torch.Generator().manual_seed(n_q + rot + sum(old))
    rows = len(old) * new
    qkv = (torch.randn((rows, (n_q + 2 * n_kv) * dim), generator=g) * 1.5).bfloat16().to(device)
    weights = [((0.0 if "norm_w_off" in how else 1.0) + 0.1 * torch.randn(dim, generator=g)).to(device) if norm else None for _ in "qk"]
    freq = torch.tensor([1e4 ** (-2 * j / rot) for j in range(rot // 2)], device=device)
    s = torch.randn(n_q, generator=g).to(device) if sinks else None
    at = torch.cat([torch.arange(a, a + new) for a in old])
    seq = torch.repeat_interleave(torch.arange(len(old)), new)
    slots = (table.cpu()[seq, at // PAGE].long() * PAGE + at % PAGE).to(device)
    at = at.to(torch.int32).to(device)
    pages = [filled(num, n_kv, dim, device, seed=i) for i in range(2)]
    again = [Pages8(p.codes.clone(), p.scales.clone()) for p in pages]
    common = dict(q_norm_w=weights[0], k_norm_w=weights[1], norm_eps=1e-6, **how)
    scale = 0.5 * dim ** -0.5
    got = ops.attention_decode_rope(qkv, *pages, table, ints(seq_lens, device), new, scale, at, slots, freq, n_q, n_kv, dim, splits=splits, window=window, chunk=chunk,
                                    sinks=s, **common)
    q = ops.rope_kv(qkv, at, slots, freq, *again, n_q, n_kv, dim, **common)
    for a, b in zip(pages, again):
        assert torch.equal(a.codes, b.codes) and torch.equal(a.scales, b.scales)
    want, size = attended(q, pages[0].values(), pages[1].values(), table, seq_lens, [new] * len(old), scale, window, chunk, s)
    # the step may keep queries in more bits than rope_kv returns: half a bf16 step in every component moves a score by 2^-8 of the sum of |q k|
    keys = pages[0].values().double().abs().amax((0, 2)).cpu()                 # [n_kv, dim]: no key is larger
    moved = float((q.double().cpu().abs().view(-1, n_kv, n_q // n_kv, dim) * keys[None, :, None]).sum(-1).max()) * scale * 2.0 ** -8
    bound = (2 * 2.0 ** -11 + 2.0 ** -13 + 2 * math.expm1(moved)) * size + 2.0 ** -8 * want.abs() + 2.0 ** -120
    assert ((got.double().cpu() - want).abs() <= bound).all()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("n_q, n_kv, dim, section", [(8, 2, 64, (16, 8, 8)), (32, 8, 128, (24, 20, 20))])
def test_positions_of_three_axes(device, n_q, n_kv, dim, section):
    """By tensor operations: on a GPU a key is rounded to bf16 and then to its code, on a CPU to its code alone."""
    rows, half = 37, dim // 2
    g = torch.Generator().manual_seed(dim)
    qkv = torch.randn((rows, (n_q + 2 * n_kv) * dim), generator=g).bfloat16().to(device)
    positions = torch.stack([torch.randint(0, 60, (rows,), generator=g) for _ in range(3)]).to(torch.int32).to(device)
    freq = torch.tensor([1e4 ** (-2 * j / dim) for j in range(half)])
    slots = torch.arange(20, 20 + rows, device=device)
    pages = [Pages8.empty(5, n_kv, dim, device) for _ in "kv"]
    pages[0].scales[1], pages[1].scales[1] = 2.0 ** -9, 2.0 ** -9
    got = ops.rope_kv(qkv, positions, slots, freq.to(device), *pages, n_q, n_kv, dim, mrope_section=section)
    axis = torch.zeros(half, dtype=torch.long)
    for a in (1, 2):
        axis[a:3 * section[a]:3] = a
    angle = positions.double().cpu()[axis].t() * freq.double()
    cos, sin = angle.cos()[:, None], angle.sin()[:, None]
    x = qkv.double().cpu().view(rows, -1, dim)[:, :n_q + n_kv]
    a, b = x.chunk(2, -1)
    want = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    # angles are 32-bit products below 2^6: off by 2^-18, and so are sines and cosines
    fine = 2.0 ** -17 * x.abs().amax(-1, keepdim=True)
    assert ((got.double().cpu() - want[:, :n_q]).abs() <= 2.0 ** -8 * want[:, :n_q].abs() + fine[:, :n_q]).all()
    k, v = (p.values()[slots // PAGE, :, slots % PAGE].double().cpu() for p in pages)
    scale = pages[0].scales[slots // PAGE].double().cpu()[..., None]
    assert ((k - want[:, n_q:]).abs() <= scale / 2 + 2.0 ** -8 * want[:, n_q:].abs() + fine[:, n_q:]).all()
    # no larger scale than the rounded rows need: 127 of them are above half of their block's largest magnitude
    page = (slots // PAGE).cpu()
    for p in page.unique().tolist():
        top = want[:, n_q:][page == p].abs().amax((0, 2)) * (1 + 2.0 ** -8) + 2.0 ** -16
        assert (pages[0].scales[p].double().cpu() <= (2 * top / 127).clamp_min(2.0 ** -9)).all()
    codes, scales = stored(qkv.view(rows, -1, dim)[:, n_q + n_kv:], slots, Pages8.empty(5, n_kv, dim, "cpu"))
    assert torch.equal(v[12:], (codes * scales[..., None, None])[slots.cpu() // PAGE, :, slots.cpu() % PAGE][12:])


# ------------------------------------------------------------------------------------------ rows that are taken back
@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("n_q, n_kv, dim", [(8, 2, 64), (16, 4, 128), (32, 2, 128)])
@pytest.mark.parametrize("splits", [1, 2])
def test_rows_that_are_refused_and_written_again(device, n_q, n_kv, dim, splits):
    """A verification writes rows a hundred times as large as the others, one of them stays and the next verification writes over the rest: codes and scales are those of the
    definition over both writes (a block keeps the scale that the refused rows have raised, one that is opened again does not), and attention is that of these pages."""
    new, old = 4, (10, 30, 47, 5, 15)
    lens = [a + 1 + new for a in old]
    num, table = layout(lens, device)
    g = torch.Generator().manual_seed(dim)
    pages = [filled(num, n_kv, dim, device, seed=i) for i in range(2)]
    for p in pages:
        p.scales.fill_(2.0 ** -6)
    freq = torch.zeros(dim // 2, device=device)                     # rows are stored as they are
    held = [Pages8(p.codes.cpu().clone(), p.scales.cpu().clone()) for p in pages]
    for first, size in ((0, 100.0), (1, 1.0)):
        begin = [a + first for a in old]
        at = torch.cat([torch.arange(a, a + new) for a in begin])
        seq = torch.repeat_interleave(torch.arange(len(old)), new)
        slots = table.cpu()[seq, at // PAGE].long() * PAGE + at % PAGE
        qkv = torch.randn((len(old) * new, n_q + 2 * n_kv, dim), generator=g)
        qkv[:, n_q:] *= size
        qkv[::new, n_q:] /= size                                    # the row that stays is an ordinary one
        qkv = qkv.bfloat16()
        for p, x in zip(held, (qkv[:, n_q:n_q + n_kv], qkv[:, n_q + n_kv:])):
            codes, scales = stored(x, slots, p)
            p.codes.copy_(codes)
            p.scales.copy_(scales)
        seq_lens = [a + new for a in begin]
        got = ops.attention_decode_rope(qkv.view(len(qkv), -1).to(device), *pages, table, ints(seq_lens, device), new, 0.02, at.to(torch.int32).to(device), slots.to(device),
                                        freq, n_q, n_kv, dim, splits=splits)
        for p, h in zip(pages, held):
            assert torch.equal(p.codes.cpu(), h.codes) and torch.equal(p.scales.cpu(), h.scales)
        want, magnitude = attended(qkv[:, :n_q], held[0].values(), held[1].values(), table, seq_lens, [new] * len(old), 0.02)
        # What a token weighs, its probability times its block's scale, is held in f16 relative to a maximum that the row's largest weight reaches or passes: 11 bits down to
        # 2^-14 of it, whole multiples of 2^-24 of it below. There a token is off by half of that, 2^-25 of the largest weight at most, times its code. In a channel in which
        # the largest tokens have codes of zero (ordinary rows beside refused ones a hundred times as large) nothing else is left.
        least = torch.zeros_like(want)
        for b, n in enumerate(seq_lens):
            pg = table[b, :-(-n // PAGE)].long().cpu()
            for h in range(n_q):
                keys, codes = (t.double()[pg, h // (n_q // n_kv)].reshape(-1, dim)[:n] for t in (held[0].values(), held[1].codes))
                steps = held[1].scales.double()[pg, h // (n_q // n_kv)].repeat_interleave(PAGE)[:n]
                for i in range(new):
                    to = n - new + i + 1
                    weight = torch.softmax(keys[:to] @ qkv[b * new + i, h].double() * 0.02, 0) * steps[:to]
                    least[b * new + i, h] = 2.0 ** -25 * weight.max() * codes[:to].abs().sum(0)
        bound = (2 * 2.0 ** -11 + 2.0 ** -13) * magnitude + 2.0 ** -8 * want.abs() + least + 2.0 ** -120
        assert ((got.double().cpu() - want).abs() <= bound).all()
    raised, opened = table[0, 0].item(), table[4, 1].item()          # rows 10 to 13 and 11 to 14; 15 to 18, then 16 to 19
    assert (held[0].scales[raised] >= 1).all() and (held[0].scales[opened] <= 2.0 ** -4).all()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("lengths", [(21,), (5, 40)])
def test_tokens_that_speculation_keeps_are_the_target_s_own(device, lengths):
    """Fed to the target one after the other, each is its choice or next to it. A cached value is off by a per cent (half a step of 1/90 of a block's largest, three times a typical value; two
    where refused rows have raised the scale), so are logits of two layers by up to five, in units of their spread, and the distance of two logits in two passes by ten:
    half a spread is five times that, where a token chosen from wrong pages lies three spreads below the largest. Drafts of the same weights are near ties apart, drafts of others
    are kept by chance."""
    model, other = build(device), build(device, seed=9)
    prompts = [prompt(n, seed=n) for n in lengths]
    for draft, rate in ((model, (0.5, 1.0)), (other, (0.0, 0.2))):
        dec = SpeculativeDecoder(*(Engine(m, max_batch=2, max_seq_len=128, kv_bits=8) for m in (model, draft)), k=3)
        out = dec.generate(prompts, GREEDY, max_new_tokens=40)
        assert rate[0] <= dec.stats.accepted / dec.stats.proposed <= rate[1]
        solo = Engine(model, max_batch=2, max_seq_len=128, kv_bits=8)
        for p, tokens in zip(prompts, out):
            assert len(tokens) == 40
            s = solo.new_sequence(p, GREEDY, max_new_tokens=41)
            logits = solo.feed_logits(s, p).float()
            for t in tokens:
                assert logits.max() - logits[t] <= 0.5 * logits.std()
                logits = solo.feed_logits(s, [t]).float()
            solo.release(s)


@pytest.mark.parametrize("device", DEVICES)
def test_portions_of_whole_pages_leave_the_same_scales(device):
    """The first layer's rows come from the tokens alone; products of another number of rows may round a value to its other neighbour in bf16. A scale then differs where a
    block's largest value lies next to a border, by a factor of two, and values by a step of it."""
    model = build(device)
    held = []
    for limits in ((70,), (32, 16, 22)):
        eng = Engine(model, max_batch=1, max_seq_len=128, kv_bits=8)
        seq = eng.new_sequence(prompt(70), GREEDY, max_new_tokens=8)
        for n in limits:
            eng.prefill([seq], limits=[n])
        held.append([t[:4].double().cpu() for t in pages_of(eng, seq)])
    for i in (0, 2):
        codes, scales = zip(*(h[i:i + 2] for h in held))
        assert (scales[0] > 2.0 ** -30).all() and (torch.log2(scales[0] / scales[1]).abs() <= 1).all() and (scales[0] == scales[1]).double().mean() >= 0.9
        a, b = (c * s[..., None, None] for c, s in zip(codes, scales))
        assert ((a - b).abs() <= torch.maximum(*scales)[..., None, None] + 2.0 ** -7 * a.abs()).all()
        if device == "cpu":
            assert torch.equal(a, b)


# ------------------------------------------------------------------------------------------ refusals
def beside(t, elements):
    """The same contents, contiguous, ``elements`` behind where an allocation begins."""
    room = torch.empty(t.numel() + 64, dtype=t.dtype, device=t.device)
    at = room[elements:elements + t.numel()].view(t.shape)
    at.copy_(t)
    assert at.is_contiguous()
    return at


@pytest.mark.parametrize("kind", [torch.bfloat16, torch.float32])
def test_rows_to_be_stored_are_brought_to_where_they_can_be_read(kind):
    x = torch.randn((5, 3, 64)).to(kind)
    for t in (x, beside(x, 1), beside(x, 2), x[1:], torch.randn((5, 4, 64)).to(kind)[:, 1:], x.expand(5, 3, 64), x[:1].expand(4, 3, 64), torch.randn((5, 194)).to(kind)[:, :192].view(5, 3, 64),
              x.transpose(1, 2).contiguous().transpose(1, 2)):
        got = kv8._aligned_rows(t, 64)
        assert got.dtype == torch.bfloat16 and got.data_ptr() % 8 == 0 and got.stride()[1:] == (64, 1) and got.stride(0) % 4 == 0 and torch.equal(got, t.bfloat16())


@pytest.mark.gpu
def test_addresses_that_the_kernels_cannot_take_are_refused():
    """Contiguous tensors that begin inside an allocation: an access that is wider than their alignment would end the process's use of the GPU. And rows on the host."""
    dev = torch.device("cuda")
    n_q, n_kv, dim = 4, 2, 64
    k, v = (filled(4, n_kv, dim, dev, seed=i) for i in range(2))
    rows, slots = torch.zeros((3, n_kv, dim), dtype=torch.bfloat16, device=dev), torch.arange(16, 19, device=dev)
    q, table, lens, cu = torch.zeros((2, n_q, dim), dtype=torch.bfloat16, device=dev), ints([[1], [2]], dev), ints([3, 4], dev), ints([0, 1, 2], dev)
    qkv, pos, to, freq = torch.zeros((2, 8 * dim), dtype=torch.bfloat16, device=dev), ints([2, 3], dev), torch.tensor([18, 35], device=dev), torch.ones(32, device=dev)
    calls = dict(
        store=lambda k, v, q, out: ops.store_kv(rows, rows, slots, k, v),
        rope=lambda k, v, q, out: ops.rope_kv(qkv, pos, to, freq, k, v, n_q, n_kv, dim, q_out=out),
        values=lambda k, v, q, out: ops.page_values(k, v, ints([1, 2], dev)),
        decode=lambda k, v, q, out: ops.attention_decode(q, k, v, table, lens, 1, 1.0, out=out),
        prefill=lambda k, v, q, out: ops.attention_prefill(q, k, v, table, lens, cu, 1, 1.0, out=out),
        equal=lambda k, v, q, out: ops.attention_prefill(q, k, v, table, lens, cu, 1, 1.0, out=out, max_kv_len=4, equal=True),
        step=lambda k, v, q, out: ops.attention_decode_rope(qkv, k, v, table, lens, 1, 1.0, pos, to, freq, n_q, n_kv, dim))
    for name, call in calls.items():
        call(k, v, q, torch.empty_like(q))
        for by in (1, 4, 8):
            for pair in ((Pages8(beside(k.codes, by), k.scales), v), (k, Pages8(beside(v.codes, by), v.scales))):
                with pytest.raises(ValueError, match="16 bytes"):
                    call(*pair, q, torch.empty_like(q))
        call(Pages8(beside(k.codes, 16), beside(k.scales, 1)), Pages8(beside(v.codes, 32), beside(v.scales, 3)), beside(q, 8), beside(q, 16))
        for by in (1, 2, 4):
            if name in ("decode", "prefill", "equal"):
                with pytest.raises(ValueError, match="16 bytes"):
                    call(k, v, beside(q, by), torch.empty_like(q))
            if name in ("rope", "decode", "prefill", "equal"):
                with pytest.raises(ValueError, match="16 bytes"):
                    call(k, v, q, beside(q, by))
    for a, b in ((rows.cpu(), rows), (rows, rows.cpu())):
        with pytest.raises(ValueError, match="pages on cuda"):
            ops.store_kv(a, b, slots, k, v)
    # rows to be stored, and the projection's, may begin anywhere that is said
    ops.store_kv(beside(rows, 1), beside(rows, 3), slots, k, v)
    with pytest.raises(ValueError, match="8-byte aligned"):
        ops.rope_kv(beside(qkv, 2), pos, to, freq, k, v, n_q, n_kv, dim)
    torch.cuda.synchronize()
    ops.native.check_status(dev)
