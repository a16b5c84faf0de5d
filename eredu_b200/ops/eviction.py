"""Caches that give up tokens: the weight that attention gives every cached token, added up, and eviction by it.

Beside the pages of a layer lies a tensor of sums, fp32 [pages, heads, 16]: for every token and key / value head the softmax weights that query rows have
given the token, summed over the rows that counted and over the query heads that share the head. :func:`.core.attention_decode` and
:func:`.core.attention_prefill` keep it where they are given it (``weights``): tokens that stood in the cache before the call are added to, the
tokens of the call's own rows - the last ones of every sequence - begin with what the call gives them, so that a page needs no clearing.
What a page holds behind its sequence's last token means nothing.

:func:`evict_tokens` brings sequences down to a number of tokens by these sums, for every layer and head by itself. The heads of a sequence then hold
different tokens at the same place, in their order. A key keeps the rotation of the position that it had; new tokens come behind what is left, with positions that
go on counting. Masks go by places in the cache: a row sees all that stands in front of it, and a window counts tokens that are left.

The kernels take bf16 pages with heads of 64 or 128 (:func:`evict_tokens`: keys and values of any type whose rows are multiples of 16 bytes). Values of tokens that
a row does not see have to be finite where they belong to the same call.
"""
from __future__ import annotations

import struct

import torch

from . import native
from .kv8 import Pages8, _need, address
from .native import check, lib, status_word, stream_ptr

PAGE = 16
HEAD_DIMS = (64, 128)        # head sizes of the kernels
DECODE_ROWS = 16             # query rows that share a head in the decode kernel; more go to the prefill kernels
CLUSTER = 8                  # splits of a sequence and head that meet in a cluster
MAX_SPLITS = 64
LIST_BYTES = 64 << 20        # scratch that a call of evict_tokens takes for the lists of what stays: layers go in portions of it

_sms: dict = {}


def _sm_count(device) -> int:
    n = _sms.get(device)
    if n is None:
        n = _sms[device] = torch.cuda.get_device_properties(device).multi_processor_count
    return n


P, I, F = native.P, native.I, native.F
# the arguments of a call in one block, laid out as csrc/common/weights_args.h has them
_EVICT, _DECODE, _PROMPT = struct.Struct("9Q12i"), struct.Struct("13Q11if"), struct.Struct("9Q13if")
native.register("eredu_evict_tokens", I, [P, I])
native.register("eredu_weighed_decode", I, [P, I])
native.register("eredu_prompt_weights", I, [P, I])
native.register("eredu_attn_prefill_tc_lse", I, [P] * 9 + [I] * 11 + [F, P, P])


# ------------------------------------------------------------------------------------------ attention
def _check_attention(q, k_cache, v_cache, block_table, seq_lens, sinks, weights, out, rows, chunk, splits=1):
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
    if block_table.dtype != torch.int32 or block_table.dim() != 2 or block_table.stride(1) != 1 or block_table.shape[0] != seq_lens.shape[0] \
            or block_table.device != dev:
        raise ValueError("block_table: int32 rows, one per sequence")
    if q.device != dev or v_cache.device != dev:
        raise ValueError(f"queries on {q.device} and values on {v_cache.device} for keys on {dev}")
    if out is not None and (out.shape != (*q.shape[:2], v_cache.shape[3]) or out.dtype != q.dtype or out.device != dev):
        raise ValueError(f"out {tuple(out.shape)} {out.dtype} for queries {tuple(q.shape)} {q.dtype}")


def _kernels_take(q, k_cache, v_cache, out) -> bool:
    """Whether the call is one for the kernels; other head sizes take tensor operations, and what the kernels cannot read is refused."""
    if not q.is_cuda or q.shape[2] not in HEAD_DIMS or v_cache.shape[3] != q.shape[2]:
        return False
    for name, t in (("q", q), ("keys", k_cache), ("values", v_cache), ("out", out)):
        _need(name, t, torch.bfloat16, k_cache.device, 16)
    return True


def weighed_attention_ref(q, k_cache, v_cache, block_table, seq_lens, q_lens, scale, window=0, sinks=None, weights=None, observed=0, out=None):
    """Attention of the last ``q_lens[b]`` tokens of every sequence, by tensor operations, with ``weights`` kept as above. ``observed`` > 0: the last so many
    rows of a sequence count. A row that sees nothing gives zeros."""
    from .core import _gather_kv

    n_q, n_kv = q.shape[1], k_cache.shape[1]
    out = q.new_empty((*q.shape[:2], v_cache.shape[3])) if out is None else out
    start = 0
    for b, (n, m) in enumerate(zip(seq_lens.tolist(), q_lens)):
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


def weighed_splits(batch, n_kv, max_kv_len, sm_count=148):
    """CTAs that share a sequence and head of the decode kernel: as many as there is room for (two to an SM), with two pages for each of the four warps
    at least. Up to eight meet in a cluster; more leave their parts to a second kernel, which pays where eight have long shares."""
    heads, pages = max(1, batch * n_kv), max(1, -(-max_kv_len // PAGE))
    want = max(1, 2 * sm_count // heads)
    if want > CLUSTER and pages > 64 * CLUSTER:
        return min(want, pages // 32, MAX_SPLITS)
    return max(1, min(want, pages // 8, CLUSTER))


def weighed_decode(q, k_cache, v_cache, block_table, seq_lens, q_per_seq, scale, window, sinks, weights, out, chunk, max_kv_len):
    """The form of :func:`.core.attention_decode` that keeps ``weights``. ``max_kv_len``: the largest of ``seq_lens`` at least, where the host knows it (0: what
    a row of the table holds); the call takes memory for the scores of so many tokens of every sequence."""
    B = seq_lens.shape[0]
    _check_attention(q, k_cache, v_cache, block_table, seq_lens, sinks, weights, out, B * q_per_seq, chunk)
    if not _kernels_take(q, k_cache, v_cache, out):
        return weighed_attention_ref(q, k_cache, v_cache, block_table, seq_lens, [q_per_seq] * B, scale, window, sinks, weights, 0, out)
    n_q, dim = q.shape[1:]
    pages, n_kv = k_cache.shape[:2]
    dev, wide = k_cache.device, block_table.shape[1]
    rows = q_per_seq * (n_q // n_kv)
    longest = min(max_kv_len, wide * PAGE) if max_kv_len > 0 else wide * PAGE
    if rows > DECODE_ROWS:
        cu_q = torch.arange(0, (B + 1) * q_per_seq, q_per_seq, dtype=torch.int32, device=dev)
        return weighed_prefill(q, k_cache, v_cache, block_table, seq_lens, cu_q, q_per_seq, scale, window, sinks, weights, out, 0, longest, 0)
    if out is None:
        out = torch.empty_like(q)
    if q.shape[0] == 0 or wide == 0:
        return out.zero_() if wide == 0 else out
    splits = weighed_splits(B, n_kv, min(longest, window + q_per_seq + PAGE) if window > 0 else longest, _sm_count(dev))
    room, pad = -(-longest // PAGE) * PAGE, 2 if rows <= 2 else 4 if rows <= 4 else 8 if rows <= 8 else 16
    scored = B * n_kv * room * pad
    parts = B * n_kv * splits * rows if splits > CLUSTER else 0
    scratch = torch.empty(scored + parts * (dim + 2), dtype=torch.float32, device=dev)
    at = scratch.data_ptr()
    code = lib().eredu_weighed_decode(_DECODE.pack(
        q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), out.data_ptr(), block_table.data_ptr(), seq_lens.data_ptr(), address(sinks), weights.data_ptr(),
        at, at + 4 * scored if parts else 0, at + 4 * (scored + parts * dim) if parts else 0, status_word(dev).data_ptr(), stream_ptr(dev),
        B, q_per_seq, block_table.stride(0), wide * PAGE, room, pages, n_q, n_kv, dim, splits, int(window), scale), _DECODE.size)
    check(code, "eredu_weighed_decode")
    return out


def weighed_prefill(q, k_cache, v_cache, block_table, seq_lens, cu_q, max_q_len, scale, window, sinks, weights, out, chunk, max_kv_len, observed):
    """The form of :func:`.core.attention_prefill` that keeps ``weights``; ``observed`` > 0: the last so many rows of every sequence count, 0: all of them."""
    _check_attention(q, k_cache, v_cache, block_table, seq_lens, sinks, weights, out, None, chunk)
    _need("cu_q", cu_q, torch.int32, k_cache.device)
    B, total, dev = seq_lens.shape[0], q.shape[0], k_cache.device
    if cu_q.shape != (B + 1,):
        raise ValueError(f"{cu_q.numel()} query offsets for {B} sequences")
    if observed < 0:
        raise ValueError(f"the last {observed} rows")
    if not _kernels_take(q, k_cache, v_cache, out):
        return weighed_attention_ref(q, k_cache, v_cache, block_table, seq_lens, (cu_q[1:] - cu_q[:-1]).tolist(), scale, window, sinks, weights, observed, out)
    n_q, dim = q.shape[1:]
    pages, n_kv = k_cache.shape[:2]
    block_table = block_table.contiguous()
    wide = block_table.shape[1]
    if out is None:
        out = torch.empty_like(q)
    if total == 0 or B == 0 or wide == 0:
        return out
    sms, status, stream = _sm_count(dev), status_word(dev).data_ptr(), stream_ptr(dev)
    lse = torch.empty((total, n_q), dtype=torch.float32, device=dev)
    code = lib().eredu_attn_prefill_tc_lse(
        q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), out.data_ptr(), lse.data_ptr(), block_table.data_ptr(), seq_lens.data_ptr(), cu_q.data_ptr(),
        address(sinks) or None, B, total, max_q_len, wide, pages, n_q, n_kv, dim, int(window), int(max_kv_len), sms, scale, status, stream)
    check(code, "eredu_attn_prefill_tc_lse")
    longest = min(max_kv_len, wide * PAGE) if max_kv_len > 0 else wide * PAGE
    code = lib().eredu_prompt_weights(_PROMPT.pack(
        q.data_ptr(), k_cache.data_ptr(), lse.data_ptr(), block_table.data_ptr(), seq_lens.data_ptr(), cu_q.data_ptr(), weights.data_ptr(), status, stream,
        B, total, max_q_len, longest, wide, wide, pages, n_q, n_kv, dim, int(window), int(observed), sms, scale), _PROMPT.size)
    check(code, "eredu_prompt_weights")
    return out


# ------------------------------------------------------------------------------------------ eviction
def evict_tokens_ref(k, v, weights, block_table, seq_lens, keep, recent=0, first=0):
    for b, n in enumerate(seq_lens.tolist()):
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


def evict_tokens(k, v, weights, block_table, seq_lens, keep, recent=0, first=0, max_kv_len=0):
    """Brings every sequence of more than ``keep`` tokens down to ``keep``, in place, and returns the tokens that each has left (int32 [B]). ``k``, ``v``: pages
    of all layers [layers, pages, heads, 16, width], ``weights`` [layers, pages, heads, 16] fp32 (see above). For every layer and head by itself
    the ``first`` tokens of a sequence and its ``recent`` last ones stay, and of those between them the ones with the largest weights; of equal weights the
    earlier token, and what is no number goes first. What stays moves to the front in its order - keys, values and weights, bit by bit -, and the rows
    behind it are left as they were. A page belongs to one sequence of the call only (shared pages are copied first, :func:`.kv8.copy_pages`).
    ``max_kv_len``: the largest of ``seq_lens`` at least, where the host knows it."""
    if isinstance(k, Pages8) or isinstance(v, Pages8) or k.dtype == torch.int8:
        raise NotImplementedError("tokens of 8-bit pages share the scale of their block: they are not evicted one by one")
    if k.dim() != 5 or v.dim() != 5 or k.shape[3] != PAGE or v.shape[:4] != k.shape[:4] or weights.shape != k.shape[:4]:
        raise ValueError(f"keys {tuple(k.shape)}, values {tuple(v.shape)} and weights {tuple(weights.shape)} do not go together")
    dev = k.device
    _need("keys", k, k.dtype, dev)
    _need("values", v, k.dtype, dev)
    _need("weights", weights, torch.float32, dev)
    _need("seq_lens", seq_lens, torch.int32, dev)
    if block_table.dtype != torch.int32 or block_table.dim() != 2 or block_table.stride(1) != 1 or block_table.shape[0] != seq_lens.shape[0] \
            or block_table.device != dev:
        raise ValueError("block_table: int32 rows, one per sequence")
    if keep < 1 or recent < 0 or first < 0 or recent + first > keep:
        raise ValueError(f"of {keep} tokens the first {first} and the last {recent} cannot stay")
    layers, pages, n_kv = k.shape[:3]
    B, wide = block_table.shape
    if not k.is_cuda:
        return evict_tokens_ref(k, v, weights, block_table, seq_lens, keep, recent, first)
    k_row, v_row = k.shape[4] * k.element_size(), v.shape[4] * v.element_size()
    if (k_row | v_row) % 16 or (k.data_ptr() | v.data_ptr()) % 16:
        raise NotImplementedError(f"rows of {k_row} and {v_row} bytes: the kernel moves whole pieces of 16 bytes")
    left = torch.empty_like(seq_lens)
    longest = min(max_kv_len, wide * PAGE) if max_kv_len > 0 else wide * PAGE
    if B == 0 or layers == 0 or longest <= keep:
        return torch.clamp(seq_lens, max=keep, out=left)
    step = max(1, min(layers, LIST_BYTES // (4 * B * n_kv * keep)))
    lists = torch.empty(step * B * n_kv * keep, dtype=torch.int32, device=dev)
    for at in range(0, layers, step):
        some = min(step, layers - at)
        code = lib().eredu_evict_tokens(_EVICT.pack(
            k[at].data_ptr(), v[at].data_ptr(), weights[at].data_ptr(), block_table.data_ptr(), seq_lens.data_ptr(), left.data_ptr(), lists.data_ptr(),
            status_word(dev).data_ptr(), stream_ptr(dev), some, B, n_kv, pages, block_table.stride(0), longest, keep, recent, first, k_row, v_row, 0), _EVICT.size)
        check(code, "eredu_evict_tokens")
    return left
