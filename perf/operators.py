"""Keys and values held in 8 bits: the operators that write, read and move the pages of such a cache, as cases that can be timed and compared.

A page holds 16 tokens. The rows of one key / value head in a page are a block [16, head size]: int8 codes from -127 to 127 and one scale, a
power of two, so that ``code * scale`` is the value. ``code = round(x / scale)`` (ties to even) with the smallest scale that keeps all codes
in range, 2^-100 at least. Rows are written in the order of their tokens:

* a row at offset 0 opens its block: the scale is what the rows of this call need;
* rows behind others keep the block's scale or, where one of them needs a larger one, raise it; the codes in front are then rounded again.

The paths are those of a decoder's attention layer:

* ``store``: a portion of a prompt - queries and keys rotated by their positions, keys and values written to their pages;
* ``step``: a decode or verify step from the projection's output to attention's: rotation, the write, attention over all tokens;
* ``decode``: attention of a few queries per sequence over its pages;
* ``prefill``: attention of prompts, or of portions of them behind what is cached;
* ``copy``: pages copied from one place of the pools to another in all layers (a sequence that is forked, a pool that is compacted).

Heads and head sizes are those of :mod:`eredu_b200.models.config`: Llama-3-8B (32 over 8 of 128), Llama-3-70B (64 over 8 of 128),
Qwen3-30B-A3B (32 over 4 of 128, normalised) and the 16-layer draft model (32 over 8 of 64).
"""
from __future__ import annotations

import math
import random

import torch

own = False

PAGE = 16
THETA = 500000.0
EPS = 1e-5
FLOOR = 2.0 ** -100         # smallest scale of a block
HEADS = {"8b": (32, 8, 128), "70b": (64, 8, 128), "moe": (32, 4, 128), "draft": (32, 8, 64)}


# ------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # a long prompt, whole pages of one sequence; the next messages of five chats, which begin and end inside a page
        dict(name="store prompt", op="store", heads="8b", batch=1, context=0, new=4096, window=0, sinks=False),
        dict(name="store turns draft", op="store", heads="draft", batch=5, context=1003, new=77, window=0, sinks=False),
        # the smallest steps there are: the drafter between two verifications
        dict(name="step draft", op="step", heads="draft", batch=1, context=512, new=1, window=0, sinks=False),
        # a full decode batch; one user far into a long document; the verification of four drafted tokens with normalised heads
        dict(name="step 8b batch", op="step", heads="8b", batch=32, context=2048, new=1, window=0, sinks=False),
        dict(name="step 70b long", op="step", heads="70b", batch=1, context=65536, new=1, window=0, sinks=False),
        dict(name="step moe verify", op="step", heads="moe", batch=4, context=3001, new=5, window=0, sinks=False),
        # as many long sequences as such a cache is chosen for; three verifications behind a sliding window with sinks
        dict(name="decode 8b wide", op="decode", heads="8b", batch=64, context=8192, new=1, window=0, sinks=False),
        dict(name="decode window", op="decode", heads="draft", batch=3, context=1777, new=3, window=500, sinks=True),
        # the second half of a long prompt; the next message of a chat; prompts of all lengths that arrive together
        dict(name="prefill 8b portion", op="prefill", heads="8b", batch=1, context=4096, new=4096, window=0, sinks=False),
        dict(name="prefill moe turn", op="prefill", heads="moe", batch=1, context=4096, new=45, window=0, sinks=False),
        # the last pages of sixteen forked sequences; a third of a pool moved to its front
        dict(name="copy fork", op="copy", heads="8b", layers=32, pages=300, moved=16, type="bf16"),
        dict(name="copy compact", op="copy", heads="draft", layers=16, pages=6001, moved=2000, type="bf16"),
    ]


def draw(rng):
    def spread(low, high):
        return max(low, min(high, int(low * (max(high, low) / low) ** rng.random() + rng.random())))

    op, heads = rng.choice(["store", "step", "step", "decode", "prefill", "copy"]), rng.choice(list(HEADS))
    sinks = rng.random() < 0.25
    if op == "copy":
        moved = spread(1, 2000)
        layers = spread(1, max(1, min(32, 32000 // moved)))
        return dict(op=op, heads=heads, layers=layers, pages=2 * moved + spread(1, 500), moved=moved, type=rng.choice(["bf16", "fp32"]) if layers < 16 else "bf16")
    if op in ("step", "decode"):
        batch = spread(1, 64)
        context = spread(1, min(65536, 262144 // batch))
        return dict(op=op, heads=heads, batch=batch, context=context, new=rng.choice([1, 1, 2, 3, 5, 8]), window=rng.choice([0, 0, spread(16, 4096)]), sinks=sinks)
    batch = spread(1, 8)
    most = 4096 * 32 // HEADS[heads][0] // batch
    new = spread(1, most)
    context = rng.choice([0, spread(1, most)])
    return dict(op=op, heads=heads, batch=batch, context=context, new=new, window=rng.choice([0, 0, spread(16, 4096)]) if op == "prefill" else 0, sinks=sinks and op == "prefill")


def lengths(case):
    """(cached tokens, new tokens) of every sequence: the first has as many as the case says, the others between half of that and all;
    those of a step bring equally many."""
    rng = random.Random(f"{case['batch']} {case['context']} {case['new']}")
    part = lambda n, first: n if first or n < 2 else rng.randint(n // 2, n)     # noqa: E731
    same = case["op"] in ("step", "decode")
    return [(part(case["context"], i == 0), case["new"] if same else part(case["new"], i == 0)) for i in range(case["batch"])]


# ------------------------------------------------------------------------------------------ inputs
def needed(amax):
    """The smallest power of two that brings ``amax`` down to 127."""
    m, e = torch.frexp(amax.double().clamp_min(FLOOR) / 127)
    return torch.ldexp(torch.ones_like(m), torch.where(m == 0.5, e - 1, e)).clamp_min(FLOOR).float()


def filled(pages, heads, dim, valid, spread, g):
    """Codes and scales of pages whose first ``valid`` rows hold tokens; what is behind them is left from earlier use. Some channels of a
    head are larger than others, and so are some tokens, by ``spread`` (in powers of e) - keys more than values."""
    x = torch.randn((pages, heads, PAGE, dim), generator=g, device="cuda", dtype=torch.bfloat16).float()
    x *= torch.exp(0.5 * spread * torch.randn((heads, 1, dim), generator=g, device="cuda"))
    x *= torch.exp(0.3 * spread * torch.randn((pages, 1, PAGE, 1), generator=g, device="cuda"))
    there = torch.arange(PAGE, device="cuda")[None, None, :, None] < valid[:, None, None, None]
    amax = (x.abs() * there).amax((2, 3))
    scales = torch.where(valid[:, None] > 0, needed(amax), torch.full_like(amax, 2.0 ** -7))
    return (x / scales[:, :, None, None]).round_().clamp_(-127, 127).to(torch.int8), scales


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    n_q, n_kv, dim = HEADS[case["heads"]]
    state = dict(case=case, n_q=n_q, n_kv=n_kv, dim=dim, scale=dim ** -0.5)
    if case["op"] == "copy":
        kind = torch.bfloat16 if case["type"] == "bf16" else torch.float32
        shape = (case["layers"], case["pages"], n_kv, PAGE, dim)
        state["k"], state["v"] = (torch.randn(shape, generator=g, device="cuda", dtype=kind) for _ in "kv")
        # pages from anywhere behind the front to the free places in front (page 0 belongs to nobody)
        order = 1 + torch.randperm(case["pages"] - 1, generator=g, device="cuda")
        state["src"], state["dst"] = (order[i * case["moved"]:(i + 1) * case["moved"]].to(torch.int32) for i in range(2))
        return state
    spans = lengths(case)
    old, new = ([s[i] for s in spans] for i in range(2))
    total = [a + n for a, n in spans]
    count = [-(-t // PAGE) for t in total]
    wide, rows = max(count), sum(new)
    place = 1 + torch.randperm(sum(count) + 7, generator=g, device="cuda")[:sum(count)]
    table = torch.zeros((len(spans), wide), dtype=torch.int32, device="cuda")
    table[torch.arange(wide, device="cuda") < torch.tensor(count, device="cuda")[:, None]] = place.to(torch.int32)
    # tokens in place when the call is made: the cached ones where it writes the new ones itself, else all
    held = old if case["op"] in ("store", "step") else total
    valid = torch.zeros(sum(count) + 8, dtype=torch.long, device="cuda")
    valid[place] = torch.cat([(torch.tensor(h) - PAGE * torch.arange(c)).clamp(0, PAGE) for h, c in zip(held, count)]).cuda()
    for name, wild in (("k", 1.0), ("v", 0.5)):
        state[name + "_codes"], state[name + "_scales"] = filled(len(valid), n_kv, dim, valid, wild, g)
    at = torch.cat([torch.arange(a, a + n) for a, n in spans]).cuda()
    seq = torch.repeat_interleave(torch.arange(len(spans)), torch.tensor(new)).cuda()
    page = table[seq, at // PAGE].long()
    state.update(
        table=table, seq_lens=torch.tensor(total, dtype=torch.int32, device="cuda"), longest=max(total), most=max(new), positions=at.to(torch.int32),
        slots=page * PAGE + at % PAGE, touched=torch.unique(page).to(torch.int32),
        cu_q=torch.tensor([sum(new[:i]) for i in range(len(new) + 1)], dtype=torch.int32, device="cuda"),
        sinks=torch.randn(n_q, generator=g, device="cuda") if case["sinks"] else None)
    if case["op"] in ("store", "step"):
        # keys twice as large as in the cache here and there: some blocks need a larger scale
        state["qkv"] = torch.randn((rows, (n_q + 2 * n_kv) * dim), generator=g, device="cuda", dtype=torch.bfloat16) * 1.5
        state["inv_freq"] = torch.tensor([THETA ** (-2 * i / dim) for i in range(dim // 2)], dtype=torch.float32, device="cuda")
        for name in ("q_norm", "k_norm"):
            state[name] = 1.4 + 0.1 * torch.randn(dim, generator=g, device="cuda") if case["heads"] == "moe" else None
    else:
        state["q"] = torch.randn((rows, n_q, dim), generator=g, device="cuda", dtype=torch.bfloat16) * 1.4
    return state


# ------------------------------------------------------------------------------------------ passes
def run(state):
    """``store``: queries, keys and values of the pages written. ``step``: attention's output, keys and values of the pages written.
    ``decode``, ``prefill``: attention's output. ``copy``: the pools."""
    return through_the_framework(state) if own else plain(state)


def through_the_framework(s):
    from eredu_b200 import ops

    case, op = s["case"], s["case"]["op"]
    if op == "copy":
        ops.copy_pages((s["k"], s["v"]), s["src"], s["dst"])
        return s["k"], s["v"]
    k, v = ops.Pages8(s["k_codes"], s["k_scales"]), ops.Pages8(s["v_codes"], s["v_scales"])
    shared = dict(window=case["window"], sinks=s["sinks"])
    if op == "store":
        q = ops.rope_kv(s["qkv"], s["positions"], s["slots"], s["inv_freq"], k, v, s["n_q"], s["n_kv"], s["dim"],
                        q_norm_w=s["q_norm"], k_norm_w=s["k_norm"], norm_eps=EPS)
        return (q, *ops.page_values(k, v, s["touched"]))
    if op == "prefill":
        return ops.attention_prefill(s["q"], k, v, s["table"], s["seq_lens"], s["cu_q"], s["most"], s["scale"], max_kv_len=s["longest"], **shared)
    splits = ops.decode_splits(case["batch"], s["n_kv"], s["longest"], rows=s["most"] * s["n_q"] // s["n_kv"], head_dim=s["dim"], bits=8)
    if op == "decode":
        return ops.attention_decode(s["q"], k, v, s["table"], s["seq_lens"], case["new"], s["scale"], splits=splits, **shared)
    out = ops.attention_decode_rope(s["qkv"], k, v, s["table"], s["seq_lens"], case["new"], s["scale"], s["positions"], s["slots"], s["inv_freq"],
                                    s["n_q"], s["n_kv"], s["dim"], q_norm_w=s["q_norm"], k_norm_w=s["k_norm"], norm_eps=EPS, splits=splits, **shared)
    return (out, *ops.page_values(k, v, s["touched"]))


def plain(s):
    op = s["case"]["op"]
    if op == "copy":
        src, dst = s["src"].long(), s["dst"].long()
        s["k"][:, dst] = s["k"][:, src]
        s["v"][:, dst] = s["v"][:, src]
        return s["k"], s["v"]
    if op in ("decode", "prefill"):
        return attended(s, s["q"].float()).bfloat16()
    n_q, n_kv, dim = s["n_q"], s["n_kv"], s["dim"]
    q, k, v = s["qkv"].float().view(-1, n_q + 2 * n_kv, dim).split((n_q, n_kv, n_kv), 1)
    angle = (s["positions"].double()[:, None] * s["inv_freq"].double())[:, None]
    cos, sin = angle.cos().float(), angle.sin().float()

    def turned(x, weight):
        if weight is not None:
            x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * weight
        a, b = x.chunk(2, -1)
        return torch.cat((a * cos - b * sin, b * cos + a * sin), -1)

    q = turned(q, s["q_norm"])
    written(s, s["k_codes"], s["k_scales"], turned(k, s["k_norm"]))
    written(s, s["v_codes"], s["v_scales"], v)
    touched = s["touched"].long()
    values = [(s[x + "_codes"][touched].float() * s[x + "_scales"][touched][:, :, None, None]).bfloat16() for x in "kv"]
    return ((q if op == "store" else attended(s, q)).bfloat16(), *values)


def written(s, codes, scales, x):
    """Rows ``x`` [tokens, heads, dim] into their blocks."""
    page, offset = s["slots"] // PAGE, s["slots"] % PAGE
    touched = s["touched"].long()
    which = torch.searchsorted(touched, page)
    first = torch.full_like(touched, PAGE).scatter_reduce(0, which, offset, "amin")
    amax = torch.zeros((len(touched), x.shape[1]), device=x.device).index_reduce_(0, which, x.abs().amax(-1), "amax")
    before = scales[touched]
    scale = torch.where(first[:, None] > 0, torch.maximum(before, needed(amax)), needed(amax))
    held = codes[touched]
    again = (held.float() * (before / scale)[:, :, None, None]).round().to(torch.int8)
    in_front = (torch.arange(PAGE, device=x.device) < first[:, None])[:, None, :, None]
    codes[touched] = torch.where(in_front, again, held)
    scales[touched] = scale
    codes[page, :, offset] = (x / scale[which][:, :, None]).round().to(torch.int8)


def attended(s, q):
    """Attention of ``q`` [rows, heads, dim] in 32 bits; the rows of a sequence are its last tokens. Sequences are padded to the longest."""
    case, table, n_kv = s["case"], s["table"].long(), s["n_kv"]
    batch, wide = table.shape
    k, v = ((s[x + "_codes"][table].float() * s[x + "_scales"][table][..., None, None]).transpose(2, 3).reshape(batch, wide * PAGE, n_kv, -1) for x in "kv")
    begin, lens = s["cu_q"].long(), s["seq_lens"].long()
    count = begin[1:] - begin[:-1]
    row = torch.arange(s["most"], device=q.device)
    there = row < count[:, None]
    at = (begin[:-1, None] + row).clamp_max(len(q) - 1)
    padded = q[at].view(batch, s["most"], n_kv, -1, s["dim"])
    score = torch.einsum("bqhgd,bkhd->bhgqk", padded, k) * s["scale"]
    where = (lens - count)[:, None] + row
    key = torch.arange(wide * PAGE, device=q.device)
    seen = (key <= where[..., None]) & (key < lens[:, None, None])
    if case["window"]:
        seen &= key > where[..., None] - case["window"]
    score = score.masked_fill_(~seen[:, None, None], float("-inf"))
    top = score.amax(-1, keepdim=True)
    if s["sinks"] is not None:
        sink = s["sinks"].view(1, n_kv, -1, 1, 1)
        top = torch.maximum(top, sink)
    p = torch.exp_(score.sub_(top))
    total = p.sum(-1, keepdim=True)
    if s["sinks"] is not None:
        total = total + torch.exp(sink - top)
    out = torch.einsum("bhgqk,bkhd->bqhgd", p, v) / total.permute(0, 3, 1, 2, 4)
    return out.flatten(2, 3)[there]


# ------------------------------------------------------------------------------------------ what a pass cannot do without
def work(case):
    n_q, n_kv, dim = HEADS[case["heads"]]
    if case["op"] == "copy":
        # every page moved is read and written, in keys and in values
        return {"bytes": 2 * 2 * case["layers"] * case["moved"] * n_kv * PAGE * dim * (2 if case["type"] == "bf16" else 4), "flops": 0}
    spans, op, window = lengths(case), case["op"], case["window"]
    rows = sum(n for _, n in spans)
    block = 2 * n_kv * (PAGE * dim + 4)                                          # keys and values of a page, in 8 bits
    touched = sum(-(-(a + n) // PAGE) - a // PAGE for a, n in spans)
    pairs = sum(min(a + i + 1, window or a + n) for a, n in spans for i in range(n))
    reached = sum(min(a + n, window + n - 1 if window else a + n) for a, n in spans)
    attention = 2 * n_q * dim * rows + reached * block / PAGE                    # the output, and the tokens that some query sees
    read_back = touched * (block + 2 * 2 * n_kv * PAGE * dim)                    # the pages written, as values
    entry = 2 * (n_q + 2 * n_kv) * dim * rows                                    # the projection's output
    if op == "store":
        return {"bytes": entry + 2 * n_q * dim * rows + rows * block / PAGE + read_back, "flops": 0}
    if op == "step":
        return {"bytes": entry + attention + rows * block / PAGE + read_back, "flops": 4 * n_q * dim * pairs}
    return {"bytes": 2 * n_q * dim * rows + attention, "flops": 4 * n_q * dim * pairs}


# ------------------------------------------------------------------------------------------ the same in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "copy":
        out = []
        for pool in (s["k"], s["v"]):
            moved = pool.clone()
            for a, b in zip(s["src"].tolist(), s["dst"].tolist()):
                moved[:, b] = pool[:, a]
            out.append(moved)
        return tuple(out)
    n_q, n_kv, dim, table = s["n_q"], s["n_kv"], s["dim"], s["table"].tolist()
    key, value = ((s[x + "_codes"], s[x + "_scales"].double()) for x in "kv")
    spans = lengths(case)
    starts = [sum(n for _, n in spans[:i]) for i in range(len(spans))]
    if case["op"] in ("store", "step"):
        x = s["qkv"].double().view(-1, n_q + 2 * n_kv, dim)
        q, new_k, new_v = x[:, :n_q], x[:, n_q:n_q + n_kv], x[:, n_q + n_kv:]
        if s["q_norm"] is not None:
            q = q / (q.pow(2).mean(-1, True) + EPS).sqrt() * s["q_norm"].double()
            new_k = new_k / (new_k.pow(2).mean(-1, True) + EPS).sqrt() * s["k_norm"].double()
        turn = torch.polar(torch.ones_like(s["positions"], dtype=torch.float64)[:, None], s["positions"].double()[:, None] * s["inv_freq"].double())[:, None]

        def turned(t):
            z = torch.complex(t[..., :dim // 2].contiguous(), t[..., dim // 2:].contiguous()) * turn
            return torch.cat((z.real, z.imag), -1)

        q, new_k = turned(q), turned(new_k)
        for (codes, scales), fresh in ((key, new_k), (value, new_v)):
            for (a, n), start, pages in zip(spans, starts, table):
                for i in range(a // PAGE, -(-(a + n) // PAGE)):
                    lo, hi = max(a, i * PAGE), min(a + n, (i + 1) * PAGE)
                    rows, front, p = fresh[start + lo - a:start + hi - a].transpose(0, 1), lo % PAGE, pages[i]
                    scale = torch.exp2(torch.ceil(torch.log2(rows.abs().amax((1, 2)) / 127))).clamp_min(FLOOR)
                    if front:
                        scale = torch.maximum(scale, scales[p])
                        codes[p, :, :front] = torch.round(codes[p, :, :front].double() * (scales[p] / scale)[:, None, None]).to(torch.int8)
                    scales[p] = scale
                    codes[p, :, front:front + hi - lo] = torch.round(rows / scale[:, None, None]).to(torch.int8)
        at = s["touched"].long()
        values = [codes[at].double() * scales[at][:, :, None, None] for codes, scales in (key, value)]
        if case["op"] == "store":
            return (q, *values)
    else:
        q = s["q"].double()
    out = torch.zeros((len(q), n_q, dim), dtype=torch.float64, device="cuda")
    group = n_q // n_kv
    for (a, n), start, pages in zip(spans, starts, table):
        at = torch.tensor(pages[:-(-(a + n) // PAGE)], device="cuda")
        where = torch.arange(a, a + n, device="cuda")[:, None]
        there = torch.arange(a + n, device="cuda")
        hidden = there > where
        if case["window"]:
            hidden |= there <= where - case["window"]
        for h in range(n_kv):
            k, v = ((codes[at, h].double() * scales[at, h][:, None, None]).view(-1, dim)[:a + n] for codes, scales in (key, value))
            for head in range(h * group, (h + 1) * group):
                score = (q[start:start + n, head] @ k.t() * s["scale"]).masked_fill(hidden, -math.inf)
                if s["sinks"] is not None:
                    score = torch.cat((score, s["sinks"][head].double().expand(n, 1)), 1)
                out[start:start + n, head] = torch.softmax(score, 1)[:, :a + n] @ v
    return out if case["op"] in ("decode", "prefill") else (out, *values)
