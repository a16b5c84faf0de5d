"""A cache that gives up its least attended tokens: attention that adds up the weight every cached token gets, and the eviction that goes by it,
as cases that can be timed and compared.

Pages hold 16 tokens of bf16 keys and values. Beside them lies one fp32 number for every token and key / value head: the sum of the softmax weights
that the token was given, over the query rows that counted and over the query heads that share the head. The paths are:

* ``step``: a decode step, or a few tokens at once - attention over all cached tokens, weights added up. The tokens that the call brings begin with what
  the call itself gives them;
* ``prompt``: attention of prompts, or of portions of them behind what is cached, with the same sums over all rows, or over the last ``observed`` rows
  of every sequence;
* ``evict``: sequences longer than ``keep`` tokens are brought down to it, for every layer and head by itself: the first few tokens and the recent ones
  stay, and of those between them the ones with the largest sums (the earlier one of equal sums); what stays moves to the front in its order.

Heads and head sizes are those of :mod:`eredu_b200.models.config`: Llama-3-8B (32 over 8 of 128), Llama-3-70B (64 over 8 of 128),
Qwen3-30B-A3B (32 over 4 of 128) and the 16-layer draft model (32 over 8 of 64).
"""
from __future__ import annotations

import math
import random

import torch

own = False

PAGE = 16
HEADS = {"8b": (32, 8, 128), "70b": (64, 8, 128), "moe": (32, 4, 128), "draft": (32, 8, 64)}


# ------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # the smallest steps there are: the drafter over a cache of bounded size
        dict(name="step draft", op="step", heads="draft", batch=1, context=512, new=1, window=0, sinks=False),
        # a full decode batch whose caches are near their bound; one user far into a document before its first eviction
        dict(name="step 8b batch", op="step", heads="8b", batch=32, context=2175, new=1, window=0, sinks=False),
        dict(name="step 70b long", op="step", heads="70b", batch=1, context=32768, new=1, window=0, sinks=False),
        # a few known tokens at once in four chats, with a window and sinks
        dict(name="step moe turn", op="step", heads="moe", batch=4, context=3001, new=5, window=2000, sinks=True),
        # as many sequences as bounded caches allow
        dict(name="step 8b wide", op="step", heads="8b", batch=64, context=4096, new=1, window=0, sinks=False),
        # a prompt of which every row counts; the next messages of five chats; a long prompt judged by its last 64 rows; the second portion of one
        dict(name="prompt 8b", op="prompt", heads="8b", batch=1, context=0, new=4096, window=0, sinks=False, observed=0),
        dict(name="prompt draft turns", op="prompt", heads="draft", batch=5, context=1003, new=333, window=0, sinks=False, observed=0),
        dict(name="prompt moe observed", op="prompt", heads="moe", batch=1, context=0, new=8192, window=0, sinks=False, observed=64),
        dict(name="prompt 70b portion", op="prompt", heads="70b", batch=1, context=2000, new=1025, window=0, sinks=True, observed=32),
        # a batch of conversations that have passed their bound, or have not; a long prompt cut down once; one sequence of a stage of four layers
        dict(name="evict 8b batch", op="evict", heads="8b", layers=32, batch=8, context=1152, keep=1024, recent=128, first=4),
        dict(name="evict draft prompt", op="evict", heads="draft", layers=16, batch=1, context=32768, keep=2048, recent=256, first=4),
        dict(name="evict moe stage", op="evict", heads="moe", layers=4, batch=1, context=600, keep=513, recent=33, first=0),
    ]


def draw(rng):
    def spread(low, high):
        return max(low, min(high, int(low * (max(high, low) / low) ** rng.random() + rng.random())))

    op, heads = rng.choice(["step", "step", "prompt", "evict"]), rng.choice(list(HEADS))
    if op == "evict":
        context = spread(2, 32768)
        batch = spread(1, max(1, min(16, 40000 // context)))
        layers = spread(1, max(1, min(32, 300000 // (context * batch))))
        keep = spread(1, context - 1)
        recent = rng.choice([0, rng.randint(0, keep // 2)])
        return dict(op=op, heads=heads, layers=layers, batch=batch, context=context, keep=keep, recent=recent, first=rng.choice([0, 0, min(4, keep - recent)]))
    shared = dict(heads=heads, sinks=rng.random() < 0.25, window=rng.choice([0, 0, spread(16, 4096)]))
    if op == "step":
        batch = spread(1, 64)
        return dict(op=op, batch=batch, context=spread(1, min(65536, 262144 // batch)), new=rng.choice([1, 1, 1, 2, 3, 5, 8]), **shared)
    batch = spread(1, 8)
    most = 4096 * 32 // HEADS[heads][0] // batch
    return dict(op=op, batch=batch, context=rng.choice([0, spread(1, most)]), new=spread(1, most), observed=rng.choice([0, 0, spread(1, 256)]), **shared)


def lengths(case):
    """(cached tokens, new tokens) of every sequence: the first has as many as the case says, the others between half of that and all (those that
    may be cut down: between seven eighths and all); those of a step bring equally many."""
    rng = random.Random(f"{case['batch']} {case['context']} {case.get('new')}")
    part = lambda n, first, least=1: n if first or n < 2 else rng.randint(n * least // (least + 1), n)     # noqa: E731
    spans = []
    for i in range(case["batch"]):
        old = part(case["context"], i == 0, 7 if case["op"] == "evict" else 1)
        spans.append((old, 0 if case["op"] == "evict" else case["new"] if case["op"] == "step" else part(case["new"], i == 0)))
    return spans


# ------------------------------------------------------------------------------------------ inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    n_q, n_kv, dim = HEADS[case["heads"]]
    spans = lengths(case)
    total = [a + n for a, n in spans]
    count = [-(-t // PAGE) for t in total]
    wide, pages = max(count), sum(count) + 8
    place = 1 + torch.randperm(sum(count) + 7, generator=g, device="cuda")[:sum(count)]
    table = torch.zeros((len(spans), wide), dtype=torch.int32, device="cuda")
    table[torch.arange(wide, device="cuda") < torch.tensor(count, device="cuda")[:, None]] = place.to(torch.int32)
    layers = (case["layers"],) if case["op"] == "evict" else ()
    state = dict(case=case, n_q=n_q, n_kv=n_kv, dim=dim, scale=dim ** -0.5, table=table, longest=max(total),
                 seq_lens=torch.tensor(total, dtype=torch.int32, device="cuda"))
    # some channels of a head are larger than others, keys more than values
    for name, wild in (("k", 0.5), ("v", 0.25)):
        x = torch.randn((*layers, pages, n_kv, PAGE, dim), generator=g, device="cuda", dtype=torch.bfloat16)
        state[name] = x.mul_(torch.exp(wild * torch.randn((n_kv, 1, dim), generator=g, device="cuda")).bfloat16())
    # sums of earlier calls: few tokens have most of the weight, some have none at all; what lies behind a sequence's end is left from earlier use
    w = torch.exp(2 * torch.randn((*layers, pages, n_kv, PAGE), generator=g, device="cuda"))
    state["weights"] = w * (torch.rand(w.shape, generator=g, device="cuda") > 0.1)
    if case["op"] != "evict":
        new = [n for _, n in spans]
        state["q"] = torch.randn((sum(new), n_q, dim), generator=g, device="cuda", dtype=torch.bfloat16) * 1.4
        state["cu_q"] = torch.tensor([sum(new[:i]) for i in range(len(new) + 1)], dtype=torch.int32, device="cuda")
        state["most"] = max(new)
        state["sinks"] = torch.randn(n_q, generator=g, device="cuda") if case["sinks"] else None
    return state


# ------------------------------------------------------------------------------------------ passes
def run(state):
    """``step``, ``prompt``: attention's output and the sums. ``evict``: keys, values, sums and the tokens that every sequence has left."""
    return through_the_framework(state) if own else plain(state)


def through_the_framework(s):
    from eredu_b200 import ops

    case = s["case"]
    if case["op"] == "evict":
        left = ops.evict_tokens(s["k"], s["v"], s["weights"], s["table"], s["seq_lens"], case["keep"], recent=case["recent"], first=case["first"],
                                max_kv_len=s["longest"])
        return s["k"], s["v"], s["weights"], left
    shared = dict(window=case["window"], sinks=s["sinks"], weights=s["weights"], max_kv_len=s["longest"])
    if case["op"] == "step":
        out = ops.attention_decode(s["q"], s["k"], s["v"], s["table"], s["seq_lens"], case["new"], s["scale"], **shared)
    else:
        out = ops.attention_prefill(s["q"], s["k"], s["v"], s["table"], s["seq_lens"], s["cu_q"], s["most"], s["scale"], observed=case["observed"], **shared)
    return out, s["weights"]


def plain(s):
    if s["case"]["op"] == "evict":
        return evicted(s)
    case, n_kv, group = s["case"], s["n_kv"], s["n_q"] // s["n_kv"]
    out, start = [], 0
    if case["op"] == "step":
        return stepped(s)
    for i, (old, new) in enumerate(lengths(case)):
        n = old + new
        pages = s["table"][i, :-(-n // PAGE)].long()
        k, v = (s[x][pages].float().transpose(0, 1).reshape(n_kv, -1, s["dim"])[:, :n] for x in "kv")
        q = s["q"][start:start + new].float().view(new, n_kv, group, -1).permute(1, 2, 0, 3)             # [heads, group, rows, dim]
        start += new
        score = torch.matmul(q, k[:, None].transpose(-1, -2)).mul_(s["scale"])
        at, key = torch.arange(old, n, device=q.device)[:, None], torch.arange(n, device=q.device)
        hidden = key > at
        if case["window"]:
            hidden |= key <= at - case["window"]
        p = normalised(score.masked_fill_(hidden, float("-inf")), s["sinks"], n_kv)
        out.append(torch.matmul(p, v[:, None]).permute(2, 0, 1, 3).reshape(new, s["n_q"], -1))
        counted = min(new, case["observed"] or new)
        given = p[:, :, new - counted:].sum((1, 2))                                                      # [heads, tokens]
        page, offset = pages[key // PAGE], key % PAGE
        before = s["weights"][page, :, offset] * (key < old)[:, None]
        s["weights"][page, :, offset] = before + given.t()
    return torch.cat(out).bfloat16(), s["weights"]


def normalised(score, sinks, n_kv):
    """Softmax over the last dimension of ``score`` [..., heads, group, rows, tokens], in place; sinks enter the sum."""
    top = score.amax(-1, keepdim=True)
    if sinks is not None:
        sink = sinks.view(n_kv, -1, 1, 1)
        top = torch.maximum(top, sink)
    p = score.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    if sinks is not None:
        total = total + torch.exp(sink - top)
    return p.div_(total)


def stepped(s):
    """All sequences of a step at once, padded to the longest."""
    case, n_kv, new = s["case"], s["n_kv"], s["case"]["new"]
    table, lens = s["table"].long(), s["seq_lens"].long()
    batch, wide = table.shape
    key = torch.arange(wide * PAGE, device=table.device)
    k, v = (s[x][table].float().transpose(2, 3).reshape(batch, wide * PAGE, n_kv, -1).transpose(1, 2) for x in "kv")
    q = s["q"].float().view(batch, new, n_kv, -1, s["dim"]).permute(0, 2, 3, 1, 4)                       # [batch, heads, group, rows, dim]
    score = torch.matmul(q, k[:, :, None].transpose(-1, -2)).mul_(s["scale"])
    at = (lens - new)[:, None] + torch.arange(new, device=q.device)
    seen = key <= at[..., None]
    if case["window"]:
        seen &= key > at[..., None] - case["window"]
    p = normalised(score.masked_fill_(~seen[:, None, None], float("-inf")), s["sinks"], n_kv)
    out = torch.matmul(p, v[:, :, None]).permute(0, 3, 1, 2, 4).flatten(2, 3).flatten(0, 1).bfloat16()
    given = p.sum((2, 3)).transpose(1, 2)                                                                # [batch, tokens, heads]
    page, offset = table[:, key // PAGE], (key % PAGE).expand(batch, -1)
    before = s["weights"][page, :, offset]
    there = key < lens[:, None]
    after = torch.where((key < (lens - new)[:, None])[..., None], before, torch.zeros_like(before)) + given
    s["weights"][page[there], :, offset[there]] = after[there]
    return out, s["weights"]


def evicted(s):
    case, n_kv = s["case"], s["n_kv"]
    keep, recent, first = case["keep"], case["recent"], case["first"]
    heads = torch.arange(n_kv, device="cuda")[:, None]
    for layer in range(case["layers"]):
        k, v, w = s["k"][layer], s["v"][layer], s["weights"][layer]
        for i, (n, _) in enumerate(lengths(case)):
            if n <= keep:
                continue
            pages, t = s["table"][i].long(), torch.arange(n, device="cuda")
            rank = w[pages[t // PAGE], :, t % PAGE].t().clone()                                          # [heads, tokens]
            rank[:, :first] = float("inf")
            rank[:, n - recent:] = float("inf")
            stays = torch.sort(rank, dim=1, descending=True, stable=True)[1][:, :keep].sort(1)[0]
            source = pages[stays // PAGE], heads, stays % PAGE
            target = pages[t[:keep] // PAGE], heads, t[:keep] % PAGE
            for x in (k, v, w):
                x[target] = x[source]
    return s["k"], s["v"], s["weights"], s["seq_lens"].clamp_max(keep)


# ------------------------------------------------------------------------------------------ what a pass cannot do without
def work(case):
    n_q, n_kv, dim = HEADS[case["heads"]]
    spans, row = lengths(case), 2 * 2 * n_kv * dim                                                       # bytes of a token's keys and values
    if case["op"] == "evict":
        # the sums of all tokens; what stays, read and written (the first tokens are where they belong)
        shrunk, moved = [n for n, _ in spans if n > case["keep"]], case["keep"] - case["first"]
        return {"bytes": case["layers"] * sum(4 * n_kv * (n + moved) + 2 * moved * row for n in shrunk), "flops": 0}
    window = case["window"]
    rows = sum(n for _, n in spans)
    reached = sum(min(a + n, window + n - 1 if window else a + n) for a, n in spans)
    pairs = sum(min(a + i + 1, window or a + n) for a, n in spans for i in range(n))
    # queries and output, the tokens that some row sees, their sums (those of new tokens are written only)
    return {"bytes": 2 * 2 * n_q * dim * rows + reached * (row + 8 * n_kv) - 4 * n_kv * min(rows, reached), "flops": 4 * n_q * dim * pairs}


# ------------------------------------------------------------------------------------------ the same in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    n_q, n_kv, dim, table = s["n_q"], s["n_kv"], s["dim"], s["table"].tolist()
    spans = lengths(case)
    if case["op"] == "evict":
        keep, recent, first = case["keep"], case["recent"], case["first"]
        for i, (n, _) in enumerate(spans):
            if n <= keep:
                continue
            at = torch.tensor(table[i][:-(-n // PAGE)], device="cuda")
            between, quota = n - first - recent, keep - first - recent
            for layer in range(case["layers"]):
                sums = s["weights"][layer, at].transpose(0, 1).reshape(n_kv, -1)[:, :n]
                some = sums[:, first:n - recent].double()
                stays = torch.ones_like(sums, dtype=torch.bool)
                if quota == 0:
                    stays[:, first:n - recent] = False
                else:
                    border = some.kthvalue(between - quota + 1, dim=1, keepdim=True)[0]
                    above, equal = some > border, some == border
                    stays[:, first:n - recent] = above | (equal & (equal.cumsum(1) <= quota - above.sum(1, keepdim=True)))
                for x in (s["k"], s["v"], s["weights"]):
                    flat = x[layer, at].transpose(0, 1).flatten(1, 2)                                    # [heads, tokens of the pages, ...]
                    for h in range(n_kv):
                        flat[h, :keep] = flat[h, :n][stays[h]]
                    x[layer, at] = flat.unflatten(1, (len(at), PAGE)).transpose(0, 1)
        return s["k"], s["v"], s["weights"], torch.tensor([min(n, keep) for n, _ in spans], dtype=torch.int32, device="cuda")
    out = torch.zeros((len(s["q"]), n_q, dim), dtype=torch.float64, device="cuda")
    sums = s["weights"].double()
    group, start = n_q // n_kv, 0
    for i, (a, n) in enumerate(spans):
        at = torch.tensor(table[i][:-(-(a + n) // PAGE)], device="cuda")
        where, there = torch.arange(a, a + n, device="cuda")[:, None], torch.arange(a + n, device="cuda")
        hidden = there > where
        if case["window"]:
            hidden |= there <= where - case["window"]
        counted = min(n, case.get("observed") or n)
        for h in range(n_kv):
            k, v = (s[x][at, h].double().reshape(-1, dim)[:a + n] for x in "kv")
            given = torch.zeros(len(at) * PAGE, dtype=torch.float64, device="cuda")
            for head in range(h * group, (h + 1) * group):
                score = (s["q"][start:start + n, head].double() @ k.t() * s["scale"]).masked_fill_(hidden, -math.inf)
                if s["sinks"] is not None:
                    score = torch.cat((score, s["sinks"][head].double().expand(n, 1)), 1)
                p = torch.softmax(score, 1)[:, :a + n]
                out[start:start + n, head] = p @ v
                given[:a + n] += p[n - counted:].sum(0)
            held = sums[at, h].reshape(-1)
            held[:a] += given[:a]
            held[a:a + n] = given[a:a + n]
            sums[at, h] = held.view(-1, PAGE)
        start += n
    return out, sums
