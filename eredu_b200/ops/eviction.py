"""Caches that give up tokens: the weight that attention gives every cached token, added up, and eviction by it.

Beside the pages of a layer lies a tensor of sums, fp32 [pages, heads, 16]: for every token and key / value head the softmax weights that query rows have
given the token, summed over the rows that counted and over the query heads that share the head. :func:`.core.attention_decode` and
:func:`.core.attention_prefill` keep it where they are given it (``weights``): tokens that stood in the cache before the call are added to, the
tokens of the call's own rows - the last ones of every sequence - begin with what the call gives them, so that a page needs no clearing.
What a page holds behind its sequence's last token means nothing.

:func:`evict_tokens` brings sequences down to a number of tokens by these sums, for every layer and head by itself. The heads of a sequence then hold
different tokens at the same place, in their order. A key keeps the rotation of the position that it had; new tokens come behind what is left, with positions that
go on counting. Masks go by places in the cache: a row sees all that stands in front of it, and a window counts tokens that are left.

The kernels take bf16 pages with heads of 64 or 128 (:func:`evict_tokens`: keys and values of any type whose rows are multiples of 16 bytes). What lies behind a sequence's
last token may be anything; a value that is no number may reach rows that do not see its token where these see its neighbours (later tokens of the same call, the edge of
a window). A page is one sequence's: sequences that share pages would add to the same sums at once.
"""
from __future__ import annotations

import struct

import torch

from . import native
from .kv8 import Pages8, _need, address
from .native import check, lib, status_word, stream_ptr

PAGE = 16
HEAD_DIMS = (64, 128)        # head sizes of the kernels
DECODE_ROWS = 64             # query rows that share a head in the decode kernel; more go to the prefill kernels
CLUSTER = 16                 # splits of a sequence and head that meet in a cluster, where the device has room for one of so many
MAX_SPLITS = 64
HELD_SCORES = 16 << 10       # bytes of scores that a CTA of the decode kernel may hold in shared memory
HELD_TOKENS = 48 * 1024      # longest sequence whose weights the eviction kernel holds in shared memory
LIST_BYTES = 64 << 20        # scratch that a call takes for the lists of what stays where they are longer: layers go in portions of it

_devices: dict = {}


def _device(device) -> tuple:
    """(SMs, largest cluster of the decode kernel) of a device, asked once."""
    known = _devices.get(device)
    if known is None:
        with torch.cuda.device(device):
            known = torch.cuda.get_device_properties(device).multi_processor_count, CLUSTER if lib().eredu_weighed_clusters() else 8
        _devices[device] = known
    return known


P, I = native.P, native.I
# the arguments of a call in one block, laid out as csrc/common/weights_args.h has them
_EVICT, _DECODE, _PROMPT = struct.Struct("9Q12i"), struct.Struct("13Q11if"), struct.Struct("12Q13if")
native.register("eredu_evict_tokens", I, [P, I])
native.register("eredu_weighed_decode", I, [P, I])
native.register("eredu_weighed_clusters", I, [])
native.register("eredu_weighed_prefill", I, [P, I])


_current = getattr(torch._C, "_cuda_getDevice", lambda: -1)       # the current device, without the checks around it


def _elsewhere(t) -> bool:
    """Whether a tensor lies on another GPU than the current one, whose stream a launch would take."""
    at = t.get_device()
    return at >= 0 and at != _current()


# ------------------------------------------------------------------------------------------ attention
def _kernels_take(q, k_cache, v_cache, block_table, seq_lens, sinks, weights, out, rows, chunk) -> bool:
    """Whether the call is one for the kernels; CPU tensors and other head sizes take tensor operations, and what neither can take is refused.
    (One condition for the common case: these checks are a good part of what a short call costs.)"""
    at, shape, row = q.get_device(), k_cache.shape, q.shape
    if at >= 0 and sinks is None and out is None and not chunk and type(k_cache) is not Pages8 and type(v_cache) is not Pages8 and len(row) == 3 and len(shape) == 4:
        m, n_q, dim = row
        if (dim in HEAD_DIMS and shape[3] == dim and v_cache.shape == shape and shape[2] == PAGE and weights.shape == shape[:3] and n_q % shape[1] == 0
                and (rows is None or m == rows) and at == k_cache.get_device() == v_cache.get_device() == weights.get_device() == seq_lens.get_device() == block_table.get_device()
                and q.dtype is torch.bfloat16 and k_cache.dtype is torch.bfloat16 and v_cache.dtype is torch.bfloat16 and weights.dtype is torch.float32
                and seq_lens.dtype is torch.int32 and block_table.dtype is torch.int32 and seq_lens.dim() == 1 and block_table.dim() == 2
                and block_table.shape[0] == seq_lens.shape[0] and block_table.stride(1) == 1 and q.is_contiguous() and k_cache.is_contiguous()
                and v_cache.is_contiguous() and weights.is_contiguous() and seq_lens.is_contiguous()
                and (q.data_ptr() | k_cache.data_ptr() | v_cache.data_ptr()) % 16 == 0):
            return True
    return _check_attention(q, k_cache, v_cache, block_table, seq_lens, sinks, weights, out, rows, chunk)


def _check_attention(q, k_cache, v_cache, block_table, seq_lens, sinks, weights, out, rows, chunk) -> bool:
    if isinstance(k_cache, Pages8) or isinstance(v_cache, Pages8):
        raise NotImplementedError("weights are added up over pages of the model's type, not over 8-bit ones")
    if chunk:
        raise NotImplementedError("weights are not added up over chunks of positions")
    if q.dim() != 3 or k_cache.dim() != 4 or v_cache.dim() != 4 or k_cache.shape[2] != PAGE or k_cache.shape[3] != q.shape[2] or v_cache.shape[:3] != k_cache.shape[:3]:
        raise ValueError(f"queries {tuple(q.shape)}, keys {tuple(k_cache.shape)} and values {tuple(v_cache.shape)} do not go together")
    n_q, n_kv, dev = q.shape[1], k_cache.shape[1], k_cache.device
    if n_q % n_kv:
        raise ValueError(f"{n_q} query heads do not share {n_kv} key / value heads evenly")
    if rows is not None and q.shape[0] != rows:
        raise ValueError(f"{q.shape[0]} query rows, not {rows}")
    if weights.shape != k_cache.shape[:3]:
        raise ValueError(f"weights {tuple(weights.shape)} for pages {tuple(k_cache.shape[:3])}")
    _need("weights", weights, torch.float32, dev)
    _need("seq_lens", seq_lens, torch.int32, dev)
    _need("sinks", sinks, torch.float32, dev)
    if sinks is not None and sinks.numel() != n_q:
        raise ValueError(f"{sinks.numel()} sinks for {n_q} query heads")
    _check_table(block_table, seq_lens, dev)
    if q.device != dev or v_cache.device != dev:
        raise ValueError(f"queries on {q.device} and values on {v_cache.device} for keys on {dev}")
    if out is not None and (out.shape != (*q.shape[:2], v_cache.shape[3]) or out.dtype != q.dtype or out.device != dev):
        raise ValueError(f"out {tuple(out.shape)} {out.dtype} for queries {tuple(q.shape)} {q.dtype}")
    if not q.is_cuda or q.shape[2] not in HEAD_DIMS or v_cache.shape[3] != q.shape[2]:
        return False
    for name, t in (("q", q), ("keys", k_cache), ("values", v_cache), ("out", out)):
        _need(name, t, torch.bfloat16, dev, 16)
    return True


def _check_table(block_table, seq_lens, dev) -> None:
    if block_table.dtype != torch.int32 or block_table.dim() != 2 or seq_lens.dim() != 1 or block_table.stride(1) != 1 \
            or block_table.shape[0] != seq_lens.shape[0] or block_table.device != dev:
        raise ValueError("block_table: int32 rows, one per sequence")


def _narrow(window, tokens) -> int:
    """A window that no sequence of ``tokens`` fills hides nothing (0): what the kernels add to one stays within 32 bits."""
    return window if window < tokens else 0


def _named(block_table, seq_lens, pages) -> list:
    """The lengths, behind a look at them and at the pages that they reach: tensor operations follow whatever they are given."""
    wide = block_table.shape[1]
    held = torch.arange(wide, device=block_table.device) * PAGE < seq_lens[:, None]
    wrong = (seq_lens > wide * PAGE).any() | (held & ((block_table < 0) | (block_table >= pages))).any()
    if bool(wrong):
        raise ValueError(f"lengths beyond {wide * PAGE} tokens of a table's row, or pages in it that are none of {pages}")
    return seq_lens.tolist()


def weighed_attention_ref(q, k_cache, v_cache, block_table, seq_lens, q_lens, scale, window=0, sinks=None, weights=None, observed=0, out=None):
    """Attention of the last ``q_lens[b]`` tokens of every sequence, by tensor operations, with ``weights`` kept as above. ``observed`` > 0: the last so many
    rows of a sequence count. A row that sees nothing gives zeros."""
    from .core import _gather_kv

    n_q, n_kv = q.shape[1], k_cache.shape[1]
    out = q.new_empty((*q.shape[:2], v_cache.shape[3])) if out is None else out
    start = 0
    for b, (n, m) in enumerate(zip(_named(block_table, seq_lens, k_cache.shape[0]), q_lens)):
        if m == 0:
            continue
        k, v = (_gather_kv(c, block_table[b], n).float() for c in (k_cache, v_cache))
        rows = q[start:start + m].float().view(m, n_kv, n_q // n_kv, -1).permute(1, 2, 0, 3)
        s = torch.matmul(rows, k[:, None].transpose(-1, -2)) * scale                                    # [heads, group, rows, tokens]
        at, key = torch.arange(n - m, n, device=q.device)[:, None], torch.arange(n, device=q.device)
        seen = key <= at
        if window > 0:
            seen &= key > at - window
        s = s.masked_fill(~seen, float("-inf"))
        if sinks is not None:
            s = torch.cat((s, sinks.float().view(n_kv, -1, 1, 1).expand(*s.shape[:3], 1)), -1)
        p = torch.softmax(s, -1)[..., :n].masked_fill(~seen.any(-1)[:, None], 0.0)
        out[start:start + m] = torch.matmul(p, v[:, None]).permute(2, 0, 1, 3).flatten(1, 2).to(q.dtype)
        given = p[:, :, max(0, m - observed) if observed > 0 else 0:].sum((1, 2)).t()                    # [tokens, heads]
        page, offset = block_table[b, key // PAGE].long(), key % PAGE
        held = weights[page, :, offset]
        weights[page, :, offset] = torch.where((key < n - m)[:, None], held, torch.zeros_like(held)) + given
        start += m
    return out


def weighed_splits(batch, n_kv, max_kv_len, sm_count=148, cluster=CLUSTER, rows=1):
    """CTAs that share a sequence and head of the decode kernel, each with eight pages at least. Three CTAs fit an SM, clusters not quite: as many splits as find room on
    nine tenths of that, up to eight (us with 4 / 6 / 8: 8 x 8 heads of 1024 to 2048 tokens 17.2 / 15.4 / 20.8; 4 x 8 of 2048 to 4096 18.6 / 17.0 / 17.4). Where sequences and
    heads fill most of the room by themselves, three even out what they differ by while all run at once, as does one where they do not and contexts are short; two or eight where they are long
    (1 / 2 / 3 / 4 / 8: 32 x 8 heads of 1088 to 2175 tokens 49 / 48 / 44 / 46 / 59; 64 x 8 of 500 to 1000 43 / 47 / 51 / 55 / 85, of 2048 to 4096 142 / 138 / 139 / 139 / 152;
    16 x 8 of 8192 to 16384 184 / 182 / 153 / 150 / 144; with 20 ``rows`` a head 32 x 8 of 1000 to 2000 86 / 84 / 75 / 80 / 105). Few sequences and heads have sixteen
    (``cluster``: what the device has room for; 16 heads of 32768 with 8 / 16: 57 / 53), and very few with long contexts more, whose parts a second kernel joins (8 heads with
    8 / 16 / 24 / 40: 16384 tokens 28 / 21 / 19 / 19, 32768 50 / 37 / 33 / 33, 131072 167 / 108 / 92 / 94)."""
    heads, pages = max(1, batch * n_kv), max(1, -(-max_kv_len // PAGE))
    most = max(1, pages // 8)
    if heads * cluster <= 2 * sm_count:
        if heads * cluster <= sm_count and pages >= 1024:
            return min(max(cluster + 1, 27 * sm_count // (20 * heads)), MAX_SPLITS)
        return min(cluster, most)
    fit = 27 * sm_count // (10 * heads)
    if fit > 3:
        return min(8 if fit > 6 else fit, most)
    if pages >= 192:
        return 8 if pages >= 768 else 2
    return 3 if pages >= 96 and (heads <= 3 * sm_count or rows > 16) else 1


def weighed_decode(q, k_cache, v_cache, block_table, seq_lens, q_per_seq, scale, window, sinks, weights, out, chunk, max_kv_len):
    """The form of :func:`.core.attention_decode` that keeps ``weights``. ``max_kv_len``: the largest of ``seq_lens`` at least, where the host knows it (0: what
    a row of the table holds); the call takes memory for the scores of so many tokens of every sequence. A sequence of length 0 - one that does not step - gives rows of
    zeros and leaves all sums as they are."""
    if _elsewhere(q):
        with torch.cuda.device(q.device):
            return weighed_decode(q, k_cache, v_cache, block_table, seq_lens, q_per_seq, scale, window, sinks, weights, out, chunk, max_kv_len)
    B = seq_lens.shape[0]
    if not _kernels_take(q, k_cache, v_cache, block_table, seq_lens, sinks, weights, out, B * q_per_seq, chunk):
        return weighed_attention_ref(q, k_cache, v_cache, block_table, seq_lens, [q_per_seq] * B, scale, window, sinks, weights, 0, out)
    total, n_q, dim = q.shape
    pages, n_kv = k_cache.shape[:2]
    dev, most = q.device, block_table.shape[1] * PAGE
    rows = q_per_seq * (n_q // n_kv)
    longest = max_kv_len if 0 < max_kv_len < most else most
    window = _narrow(window, most)
    if rows > DECODE_ROWS:
        cu_q = torch.arange(0, (B + 1) * q_per_seq, q_per_seq, dtype=torch.int32, device=dev)
        return weighed_prefill(q, k_cache, v_cache, block_table, seq_lens, cu_q, q_per_seq, scale, window, sinks, weights, out, 0, longest, 0)
    if out is None:
        out = torch.empty_like(q)
    if total == 0 or most == 0:
        return out.zero_() if most == 0 else out
    sms, cluster = _device(dev)
    splits = weighed_splits(B, n_kv, min(longest, window + q_per_seq + PAGE) if window > 0 else longest, sms, cluster, rows)
    room, pad = -(-longest // PAGE) * PAGE, (rows + 3) // 4 * 4
    # few scores stay in shared memory, where a third CTA of an SM would have nothing to do in any case: no scratch to allocate (1.7 us of the host's)
    at = part_o = part_ml = 0
    joined = splits > cluster                # a second kernel joins what so many splits leave in memory
    if joined or B * n_kv * splits > 2 * sms or -(-room // (PAGE * splits)) * PAGE * pad * 4 > HELD_SCORES:
        scored, parts = B * n_kv * room * pad, B * n_kv * splits * rows if joined else 0
        scratch = torch.empty(scored + parts * (dim + 2), dtype=torch.float32, device=dev)
        at = scratch.data_ptr()
        if parts:
            part_o, part_ml = at + 4 * scored, at + 4 * (scored + parts * dim)
    code = lib().eredu_weighed_decode(_DECODE.pack(
        q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), out.data_ptr(), block_table.data_ptr(), seq_lens.data_ptr(), 0 if sinks is None else sinks.data_ptr(),
        weights.data_ptr(), at, part_o, part_ml, status_word(dev).data_ptr(), stream_ptr(dev), B, q_per_seq, block_table.stride(0), most, room, pages, n_q, n_kv, dim, splits,
        window, scale), _DECODE.size)
    check(code, "eredu_weighed_decode")
    return out


def prompt_ranks(batch, n_q, n_kv, max_q_len, max_kv_len, observed, sm_count=148):
    """CTAs that share the rows of a block of 256 keys in the kernel of prompts' weights, one to an SM: 1, 2, 4 or 8. Early blocks are seen by more rows than late ones, and
    a CTA costs what 14 of its tiles of 128 rows take beside them; the choice is the one with the least of the longest CTA or the mean over SMs, and that cost for every
    round (us of the whole call with 1 / 2 / 4 / 8, 32 heads over 8: 4096 tokens 346 / 244 / 267 / 311, 2048 149 / 102 / 88 / 109, 512 45 / 35 / 29 / 32, eight of 512
    80 / 80 / 92 / 127; 8192 tokens over 4 heads, the last 64 rows 490 / 497 / 509 / 566)."""
    group, blocks = n_q // n_kv, -(-max_kv_len // 256)
    shared = min(group & -group, 32)                                          # query heads of a tile
    rows = min(observed, max_q_len) if observed > 0 else max_q_len
    longest = -(-rows * shared // 128) * (group // shared)
    ctas = blocks * n_kv * batch
    mean = ctas * longest * (1 - 0.5 * min(1.0, rows / max_kv_len)) / sm_count
    return min((1, 2, 4, 8), key=lambda r: (max(longest / r, mean) + 14 * -(-ctas * r // sm_count) + r / 2, r))


def weighed_prefill(q, k_cache, v_cache, block_table, seq_lens, cu_q, max_q_len, scale, window, sinks, weights, out, chunk, max_kv_len, observed):
    """The form of :func:`.core.attention_prefill` that keeps ``weights``; ``observed`` > 0: the last so many rows of every sequence count, 0: all of them."""
    if _elsewhere(q):
        with torch.cuda.device(q.device):
            return weighed_prefill(q, k_cache, v_cache, block_table, seq_lens, cu_q, max_q_len, scale, window, sinks, weights, out, chunk, max_kv_len, observed)
    kernels = _kernels_take(q, k_cache, v_cache, block_table, seq_lens, sinks, weights, out, None, chunk)
    B, dev = seq_lens.shape[0], k_cache.device
    _need("cu_q", cu_q, torch.int32, dev)
    if cu_q.shape != (B + 1,):
        raise ValueError(f"{cu_q.numel()} query offsets for {B} sequences")
    if observed < 0:
        raise ValueError(f"the last {observed} rows")
    if not kernels:
        return weighed_attention_ref(q, k_cache, v_cache, block_table, seq_lens, (cu_q[1:] - cu_q[:-1]).tolist(), scale, window, sinks, weights, observed, out)
    if not scale > 0:
        if scale != scale:
            raise ValueError(f"a scale of {scale}")
        # the kernels take scales above zero: the sign goes to the queries, or they are nothing (bf16 holds both without rounding)
        q, scale = (-q, -scale) if scale < 0 else (q * 0, 1.0)
    total, n_q, dim = q.shape
    pages, n_kv = k_cache.shape[:2]
    block_table = block_table.contiguous()
    wide = block_table.shape[1]
    if out is None:
        out = torch.empty_like(q)
    if total == 0 or B == 0 or wide == 0:
        return out.zero_() if wide == 0 else out
    window = _narrow(window, wide * PAGE)
    longest, sms = min(max_kv_len, wide * PAGE) if max_kv_len > 0 else wide * PAGE, _device(dev)[0]
    lse = torch.empty(total * n_q, dtype=torch.float32, device=dev)
    code = lib().eredu_weighed_prefill(_PROMPT.pack(
        q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), out.data_ptr(), lse.data_ptr(), block_table.data_ptr(), seq_lens.data_ptr(), cu_q.data_ptr(),
        address(sinks), weights.data_ptr(), status_word(dev).data_ptr(), stream_ptr(dev), B, total, max_q_len, longest, wide, pages, n_q, n_kv, dim,
        window, observed, prompt_ranks(B, n_q, n_kv, max_q_len, longest, observed, sms), sms, scale), _PROMPT.size)
    check(code, "eredu_weighed_prefill")
    return out


# ------------------------------------------------------------------------------------------ eviction
def evict_tokens_ref(k, v, weights, block_table, seq_lens, keep, recent=0, first=0):
    for b, n in enumerate(_named(block_table, seq_lens, k.shape[1])):
        if n <= keep:
            continue
        t = torch.arange(n, device=k.device)
        page, offset = block_table[b, t // PAGE].long(), t % PAGE
        for layer in range(k.shape[0]):
            rank = weights[layer][page, :, offset].double().t()                                          # [heads, tokens]
            rank = torch.where(torch.isnan(rank), torch.full_like(rank, float("-inf")), rank.clamp_min(torch.finfo(torch.float32).min * 2))
            between = torch.zeros_like(rank, dtype=torch.bool)
            between[:, first:n - recent] = True
            order = torch.sort(torch.where(between, rank, torch.full_like(rank, float("inf"))), dim=1, descending=True, stable=True)[1]
            # (an infinite sum is not ahead of the tokens that stay in any case)
            order = order.gather(1, torch.sort(between.gather(1, order), dim=1, stable=True)[1])
            stays = order[:, :keep].sort(1)[0]
            heads = torch.arange(k.shape[2], device=k.device)[:, None]
            for x in (k[layer], v[layer], weights[layer]):
                x[page[:keep], :, offset[:keep]] = x[page[stays], heads, offset[stays]].transpose(0, 1)
    return seq_lens.clamp_max(keep)


def _check_eviction(k, v, weights, block_table, seq_lens) -> None:
    if isinstance(k, Pages8) or isinstance(v, Pages8) or k.dtype == torch.int8:
        raise NotImplementedError("tokens of 8-bit pages share the scale of their block: they are not evicted one by one")
    if k.dim() != 5 or v.dim() != 5 or k.shape[3] != PAGE or v.shape[:4] != k.shape[:4] or weights.shape != k.shape[:4]:
        raise ValueError(f"keys {tuple(k.shape)}, values {tuple(v.shape)} and weights {tuple(weights.shape)} do not go together")
    dev = k.device
    _need("keys", k, k.dtype, dev)
    _need("values", v, k.dtype, dev)
    _need("weights", weights, torch.float32, dev)
    _need("seq_lens", seq_lens, torch.int32, dev)
    _check_table(block_table, seq_lens, dev)


def _apart(*pools) -> bool:
    """Whether the layers of some pool, each contiguous, do not lie one behind the other (a part of a larger pool's pages)."""
    return (all(torch.is_tensor(t) and t.dim() > 1 and t.shape[0] == pools[0].shape[0] > 1 and t[0].is_contiguous() for t in pools)
            and not all(t.is_contiguous() for t in pools))


def evict_tokens(k, v, weights, block_table, seq_lens, keep, recent=0, first=0, max_kv_len=0):
    """Brings every sequence of more than ``keep`` tokens down to ``keep``, in place, and returns the tokens that each has left (int32 [B]). ``k``, ``v``: pages
    of all layers [layers, pages, heads, 16, width], ``weights`` [layers, pages, heads, 16] fp32 (see above). For every layer and head by itself
    the ``first`` tokens of a sequence and its ``recent`` last ones stay, and of those between them the ones with the largest weights; of equal weights the
    earlier token, and what is no number goes first. What stays moves to the front in its order - keys, values and weights, bit by bit -, and the rows
    behind it are left as they were. A page belongs to one sequence of the call only (shared pages are copied first, :func:`.kv8.copy_pages`).
    ``max_kv_len``: the largest of ``seq_lens`` at least, where the host knows it. Layers that do not lie one behind the other are brought down one by one."""
    if keep < 1 or recent < 0 or first < 0 or recent + first > keep:
        raise ValueError(f"of {keep} tokens the first {first} and the last {recent} cannot stay")
    shape, at = k.shape, -1 if type(k) is Pages8 else k.get_device()
    # (one condition for the common case, as above)
    if not (at >= 0 and type(v) is not Pages8 and len(shape) == 5 and shape[3] == PAGE and v.shape == shape and weights.shape == shape[:4] and k.dtype is v.dtype
            and k.dtype is not torch.int8 and weights.dtype is torch.float32 and seq_lens.dtype is torch.int32 and block_table.dtype is torch.int32
            and seq_lens.dim() == 1 and block_table.dim() == 2 and block_table.shape[0] == seq_lens.shape[0] and block_table.stride(1) == 1
            and at == v.get_device() == weights.get_device() == seq_lens.get_device() == block_table.get_device() and k.is_contiguous() and v.is_contiguous()
            and weights.is_contiguous() and seq_lens.is_contiguous()):
        if _apart(k, v, weights):
            for i in range(shape[0]):
                left = evict_tokens(k[i:i + 1], v[i:i + 1], weights[i:i + 1], block_table, seq_lens, keep, recent, first, max_kv_len)
            return left
        _check_eviction(k, v, weights, block_table, seq_lens)
    dev = k.device
    layers, pages, n_kv = shape[:3]
    B, wide = block_table.shape
    if at < 0:
        return evict_tokens_ref(k, v, weights, block_table, seq_lens, keep, recent, first)
    size = k.element_size()
    k_row, v_row = shape[4] * size, v.shape[4] * size
    ka, va, wa = k.data_ptr(), v.data_ptr(), weights.data_ptr()
    if (k_row | v_row) % 16:
        raise NotImplementedError(f"rows of {k_row} and {v_row} bytes: the kernel moves whole pieces of 16 bytes")
    if (ka | va | wa) % 16:
        raise ValueError("keys, values and weights have to begin at multiples of 16 bytes")
    if at != _current():
        with torch.cuda.device(dev):
            return evict_tokens(k, v, weights, block_table, seq_lens, keep, recent, first, max_kv_len)
    left = torch.empty_like(seq_lens)
    longest = min(max_kv_len, wide * PAGE) if max_kv_len > 0 else wide * PAGE
    if B == 0 or layers == 0 or longest <= keep:
        return left.copy_(seq_lens)
    step, lists, done = layers, None, 0
    if longest > HELD_TOKENS:
        step = max(1, min(layers, LIST_BYTES // (4 * B * n_kv * keep)))
        lists = torch.empty(step * B * n_kv * keep, dtype=torch.int32, device=dev)
    page = pages * n_kv * PAGE                                                                           # tokens and heads of a layer
    status, stream = status_word(dev).data_ptr(), stream_ptr(dev)
    while done < layers:
        some = min(step, layers - done)
        code = lib().eredu_evict_tokens(_EVICT.pack(
            ka + done * page * k_row, va + done * page * v_row, wa + done * page * 4, block_table.data_ptr(), seq_lens.data_ptr(), left.data_ptr(), address(lists),
            status, stream, some, B, n_kv, pages, block_table.stride(0), longest, keep, recent, first, k_row, v_row, _device(dev)[0]), _EVICT.size)
        check(code, "eredu_evict_tokens")
        done += some
    return left
