"""Keys and values held in 8 bits.

The cache of a layer is a pair of :class:`Pages8` in place of two bf16 tensors; :func:`rope_kv`, :func:`attention_prefill`,
:func:`attention_decode`, :func:`attention_decode_rope` and :func:`attention_ref` of :mod:`.core` take either.

A block is the 16 rows of one key / value head in a page: int8 codes in [-127, 127] and one fp32 scale, a power of two, value = code * scale.
``code = round(x / scale)`` (ties to even) with the smallest scale that keeps all codes in range, 2^-100 at least: a value is off by at most
half a scale, between 1/254 and 1/127 of the block's largest magnitude. (With positions of three axes a key is rotated by tensor operations, and on a GPU rounded to bf16
in front of its code.)
Rows are written in the order of their tokens. A row at offset 0 opens its block and sets the scale; rows behind others keep the scale or,
where one of them needs a larger one, raise it, and the codes in front are rounded again (at least twofold each time, so that all roundings of a value
together stay below one scale). What lies behind the last row written is left from earlier use and means nothing. A row with an infinity or a NaN
makes the scale, and with it the whole block, no number until the block is opened again. Rows that are taken back and written again (a verification) leave the scale they
have raised.
"""
from __future__ import annotations

import struct
from typing import NamedTuple

import torch

from . import native
from .native import check, lib, ptr, status_word, stream_ptr

PAGE = 16
FLOOR = 2.0 ** -100          # smallest scale
KV8_HEAD_DIMS = (64, 128)    # head sizes of the kernels
CLUSTER = 8                  # splits of a sequence and head that meet in a cluster
EVEN_CTAS = 3                # CTAs to an SM that take even shares of all pages

_sms: dict = {}


def _sm_count(device) -> int:
    n = _sms.get(device)
    if n is None:
        n = _sms[device] = torch.cuda.get_device_properties(device).multi_processor_count
    return n


P, I, F = native.P, native.I, native.F
# the arguments of a call in one block, laid out as csrc/common/kv8_args.h has them
_STORE, _VALUES, _ATTENTION = struct.Struct("15Q11i3f"), struct.Struct("12Q10i"), struct.Struct("20Q16i4f")
native.register("eredu_kv8_store", I, [P, I])
native.register("eredu_kv8_values", I, [P, I])
native.register("eredu_attn_kv8_decode", I, [P, I])
native.register("eredu_attn_kv8_step", I, [P, I])
native.register("eredu_copy_pages", I, [P, I, P, P, I, I, P, P])


class Pages8(NamedTuple):
    """``codes`` [pages, heads, 16, head size] int8 and ``scales`` [pages, heads] fp32 of the keys or of the values of a layer."""
    codes: torch.Tensor
    scales: torch.Tensor

    @property
    def shape(self):
        return self.codes.shape

    @property
    def is_cuda(self) -> bool:
        return self.codes.is_cuda

    @property
    def device(self):
        return self.codes.device

    def values(self, pages=None) -> torch.Tensor:
        """fp32 values of ``pages`` (all by default), by tensor operations; :func:`page_values` is the kernel."""
        codes, scales = (self.codes, self.scales) if pages is None else (self.codes[pages], self.scales[pages])
        return codes.float() * scales[..., None, None]

    @classmethod
    def empty(cls, pages: int, heads: int, head_dim: int, device) -> "Pages8":
        """Zeroed blocks."""
        return cls(torch.zeros((pages, heads, PAGE, head_dim), dtype=torch.int8, device=device),
                   torch.full((pages, heads), FLOOR, dtype=torch.float32, device=device))


def _check_pair(k, v) -> None:
    if type(k) is not Pages8 or type(v) is not Pages8:
        raise TypeError("keys and values: a pair of Pages8 is expected, both or neither")


def check_pages8(k: Pages8, v: Pages8, n_kv: int, head_dim: int) -> None:
    _check_pair(k, v)
    (kc, ks), (vc, vs) = k, v
    shape = kc.shape
    # (one condition for the common case: these checks are a good part of what a short call costs)
    if (kc.dtype is torch.int8 and vc.dtype is torch.int8 and ks.dtype is torch.float32 and vs.dtype is torch.float32 and vc.shape == shape and len(shape) == 4
            and shape[1] == n_kv and shape[2] == PAGE and shape[3] == head_dim and ks.shape == shape[:2] and vs.shape == shape[:2]
            and kc.is_contiguous() and vc.is_contiguous() and ks.is_contiguous() and vs.is_contiguous()
            and kc.get_device() == vc.get_device() == ks.get_device() == vs.get_device()
            and (not kc.is_cuda or (head_dim in KV8_HEAD_DIMS and (kc.data_ptr() | vc.data_ptr()) % 16 == 0))):
        return
    for name, t in (("keys", k), ("values", v)):
        if t.codes.dtype != torch.int8 or t.scales.dtype != torch.float32 or tuple(t.codes.shape[1:]) != (n_kv, PAGE, head_dim) \
                or t.scales.shape != t.codes.shape[:2]:
            raise ValueError(f"{name}: codes {tuple(t.codes.shape)} {t.codes.dtype} with scales {tuple(t.scales.shape)} {t.scales.dtype} are no pages of "
                             f"{n_kv} heads of {head_dim}")
        if not t.codes.is_contiguous() or not t.scales.is_contiguous() or t.scales.device != t.codes.device:
            raise ValueError(f"{name}: codes and scales have to be contiguous and on one device")
    if kc.shape[0] != vc.shape[0] or kc.device != vc.device:
        raise ValueError("keys and values have to have the same pages")
    if (kc.data_ptr() | vc.data_ptr()) % 16:
        raise ValueError("codes have to begin at a multiple of 16 bytes")
    raise NotImplementedError(f"the kernels of 8-bit pages are built for head sizes {KV8_HEAD_DIMS}, not {head_dim}")


def address(t) -> int:
    """Where a tensor lies, 0 for none."""
    return 0 if t is None else t.data_ptr()


def _need(name, t, dtype, device, align=1) -> None:
    """``align``: bytes of the widest access that a kernel makes."""
    if t is not None and (t.dtype is not dtype or not t.is_contiguous() or t.device != device):
        raise ValueError(f"{name}: a contiguous {dtype} tensor on {device} is expected, not {t.dtype} on {t.device}")
    if align > 1 and t is not None and t.data_ptr() % align:
        raise ValueError(f"{name} has to begin at a multiple of {align} bytes")


# ------------------------------------------------------------------------------------------ writing
def needed_scale(amax: torch.Tensor) -> torch.Tensor:
    """The smallest power of two that brings ``amax`` down to 127 (at least :data:`FLOOR`); no number for what is none."""
    m, e = torch.frexp(amax.double().clamp_min(FLOOR) / 127)
    s = torch.ldexp(torch.ones_like(m), torch.where(m == 0.5, e - 1, e)).clamp_min(FLOOR)
    return torch.where(torch.isfinite(amax), s, torch.full_like(s, float("nan"))).float()


def store_rows_ref(x, slots, pages: Pages8) -> None:
    """Rows ``x`` [M, heads, head size] into their blocks, run by run (rows that follow one another in a page)."""
    at, i = slots.tolist(), 0
    while i < len(at):
        n = 1
        if at[i] >= 0:
            page, first = divmod(at[i], PAGE)
            if page >= pages.shape[0]:
                raise IndexError(f"slot {at[i]} lies behind the last of {pages.shape[0]} pages")
            while i + n < len(at) and first + n < PAGE and at[i + n] == at[i] + n:
                n += 1
            rows = x[i:i + n].float().transpose(0, 1)                          # [heads, n, head size]
            before = pages.scales[page]
            scale = needed_scale(rows.abs().amax((1, 2)))
            if first:
                scale = torch.maximum(scale, before)                           # (keeps what is no number)
                front = pages.codes[page, :, :first].float() * (before / scale)[:, None, None]
                pages.codes[page, :, :first] = torch.nan_to_num(front.round()).to(torch.int8)
            pages.scales[page] = scale
            pages.codes[page, :, first:first + n] = torch.nan_to_num((rows / scale[:, None, None]).round()).to(torch.int8)
        i += n


def _store(q, k, v, slots, k_cache, v_cache, q_out, positions, inv_freq, n_q, n_kv, head_dim, rot, interleaved, attn_factor, q_norm_w, k_norm_w,
           norm_eps, norm_w_off, ld):
    dev = k_cache.device
    code = lib().eredu_kv8_store(_STORE.pack(
        q, k, v, address(q_out), k_cache.codes.data_ptr(), v_cache.codes.data_ptr(), k_cache.scales.data_ptr(), v_cache.scales.data_ptr(), address(positions), slots.data_ptr(),
        address(inv_freq), address(q_norm_w), address(k_norm_w), status_word(dev).data_ptr(), stream_ptr(dev), slots.shape[0], *ld, n_q, n_kv, head_dim, rot,
        1 if interleaved else 0, k_cache.codes.shape[0], 0, attn_factor, norm_eps, norm_w_off), _STORE.size)
    check(code, "eredu_kv8_store")


def _aligned_rows(t, head_dim):
    """Rows as the kernel reads them: bf16, four values at a time."""
    if t.dtype == torch.bfloat16 and t.stride()[1:] == (head_dim, 1) and t.stride(0) % 4 == 0 and t.data_ptr() % 8 == 0:
        return t
    t = t.to(torch.bfloat16).contiguous()
    return t if t.data_ptr() % 8 == 0 else t.clone()      # (what is bf16 and contiguous already has not moved)


def store_kv(k, v, slots, k_cache: Pages8, v_cache: Pages8) -> None:
    """Keys and values [M, heads, head size] (as they are: rotated where the model rotates them; on a GPU in bf16, others are rounded to it first) into the blocks of ``slots`` [M] int64 (page * 16 +
    offset; negative: not stored). The rows of a page follow one another in the order of their offsets, and a page occurs once in a call."""
    if k.shape != v.shape or k.dim() != 3 or slots.shape != k.shape[:1]:
        raise ValueError(f"keys {tuple(k.shape)}, values {tuple(v.shape)} and slots {tuple(slots.shape)} do not go together")
    n_kv, head_dim = k.shape[1:]
    check_pages8(k_cache, v_cache, n_kv, head_dim)
    if not k_cache.is_cuda:
        store_rows_ref(k, slots, k_cache)
        store_rows_ref(v, slots, v_cache)
        return
    _need("slots", slots, torch.int64, k_cache.device)
    if k.device != k_cache.device or v.device != k_cache.device:
        raise ValueError(f"keys on {k.device} and values on {v.device} for pages on {k_cache.device}")
    k, v = _aligned_rows(k, head_dim), _aligned_rows(v, head_dim)
    _store(0, k.data_ptr(), v.data_ptr(), slots, k_cache, v_cache, None, None, None, 0, n_kv, head_dim, 0, False, 1.0, None, None, 0.0, 0.0,
           (0, k.stride(0), v.stride(0)))


def _check_qkv(qkv, M, positions, slots, inv_freq, k_cache, v_cache, n_q, n_kv, head_dim, rot, q_norm_w, k_norm_w):
    check_pages8(k_cache, v_cache, n_kv, head_dim)
    dev = k_cache.codes.device
    if qkv.dtype != torch.bfloat16 or qkv.device != dev or qkv.dim() != 2 or qkv.shape[0] != M or qkv.stride(1) != 1 or qkv.stride(0) % 4 \
            or qkv.data_ptr() % 8 or qkv.shape[1] < (n_q + 2 * n_kv) * head_dim or n_q % n_kv:
        raise ValueError(f"qkv: {M} bf16 rows of {n_q} + 2 * {n_kv} heads of {head_dim}, 8-byte aligned, on {dev} are expected")
    if rot % 8 or rot > head_dim or inv_freq.numel() != rot // 2:
        raise ValueError(f"{rot} rotated dims with {inv_freq.numel()} frequencies: a multiple of 8 up to the head size, and half as many frequencies")
    if positions.shape != (M,) or slots.shape != (M,):
        raise ValueError("one position and one slot per row are expected")
    _need("positions", positions, torch.int32, dev)
    _need("slots", slots, torch.int64, dev)
    _need("inv_freq", inv_freq, torch.float32, dev)
    for w in (q_norm_w, k_norm_w):
        if w is not None:
            _need("norm weights", w, torch.float32, dev)
            if w.numel() != head_dim:
                raise ValueError(f"a norm has {w.numel()} weights for heads of {head_dim}")


def rope_kv8(qkv, positions, slots, inv_freq, k_cache: Pages8, v_cache: Pages8, n_q, n_kv, head_dim, rot, interleaved, attn_factor, q_norm_w, k_norm_w,
             norm_eps, norm_w_off, q_out):
    """The form of :func:`.core.rope_kv` for 8-bit pages on a GPU. Norm and rotation run in 32 bits throughout; a key is rounded once, to its code.
    Angles (position times frequency) are good below 2^22."""
    dev, M = k_cache.codes.device, qkv.shape[0]
    _check_qkv(qkv, M, positions, slots, inv_freq, k_cache, v_cache, n_q, n_kv, head_dim, rot, q_norm_w, k_norm_w)
    if q_out is None:
        q_out = qkv.new_empty((M, n_q, head_dim))
    else:
        _need("q_out", q_out, qkv.dtype, dev, 16)
        if q_out.numel() != M * n_q * head_dim:
            raise ValueError(f"q_out has {q_out.numel()} elements for {M} rows of {n_q} heads of {head_dim}")
    ld, at = qkv.stride(0), qkv.data_ptr()
    _store(at, at + 2 * n_q * head_dim, at + 2 * (n_q + n_kv) * head_dim, slots, k_cache, v_cache, q_out, positions, inv_freq, n_q, n_kv, head_dim, rot,
           interleaved, attn_factor, q_norm_w, k_norm_w, norm_eps, norm_w_off, (ld, ld, ld))
    return q_out


# ------------------------------------------------------------------------------------------ reading
def page_values(k_cache: Pages8, v_cache: Pages8, pages):
    """Keys and values of ``pages`` [n] int32 as bf16 [n, heads, 16, head size] each (exact: a code has seven bits)."""
    _check_pair(k_cache, v_cache)
    (kc, ks), (vc, vs) = k_cache, v_cache
    num, n_kv, _, dim = kc.shape
    check_pages8(k_cache, v_cache, n_kv, dim)
    if not kc.is_cuda:
        return tuple(t.values(pages.long()).to(torch.bfloat16) for t in (k_cache, v_cache))
    dev, n = kc.device, pages.shape[0]
    _need("pages", pages, torch.int32, dev)
    out = kc.new_empty((2, n, n_kv, PAGE, dim), dtype=torch.bfloat16)
    if n:
        at = out.data_ptr()
        code = lib().eredu_kv8_values(_VALUES.pack(
            kc.data_ptr(), vc.data_ptr(), ks.data_ptr(), vs.data_ptr(), at, at + 2 * n * n_kv * PAGE * dim, pages.data_ptr(), 0, 0, 0, status_word(dev).data_ptr(),
            stream_ptr(dev), 1, n, n, n, n_kv, dim, num, 0, 0, 0), _VALUES.size)
        check(code, "eredu_kv8_values")
    return out.unbind(0)


def _check_batch(n_q, n_kv, block_table, seq_lens, sinks, dev):
    if n_q % n_kv:
        raise ValueError(f"{n_q} query heads do not share {n_kv} key / value heads evenly")
    _need("seq_lens", seq_lens, torch.int32, dev)
    _need("sinks", sinks, torch.float32, dev)
    if block_table.dtype != torch.int32 or block_table.dim() != 2 or block_table.stride(1) != 1 or block_table.shape[0] != seq_lens.shape[0] \
            or block_table.device != dev:
        raise ValueError("block_table: int32 rows, one per sequence")
    if sinks is not None and sinks.numel() != n_q:
        raise ValueError(f"{sinks.numel()} sinks for {n_q} query heads")


def check_attention8(q, k_cache, v_cache, block_table, seq_lens, sinks, out, cu_q=None):
    _check_pair(k_cache, v_cache)
    n_q, dim = q.shape[1:]
    n_kv, dev = k_cache.codes.shape[1], k_cache.codes.device
    check_pages8(k_cache, v_cache, n_kv, dim)
    _check_batch(n_q, n_kv, block_table, seq_lens, sinks, dev)
    _need("q", q, torch.bfloat16, dev, 16)
    _need("out", out, torch.bfloat16, dev, 16)
    _need("cu_q", cu_q, torch.int32, dev)
    if cu_q is not None and cu_q.shape[0] != seq_lens.shape[0] + 1:
        raise ValueError(f"{cu_q.shape[0]} query offsets for {seq_lens.shape[0]} sequences")
    if out is not None and out.shape != q.shape:
        raise ValueError(f"out {tuple(out.shape)} for queries {tuple(q.shape)}")


def _shares(splits, rows, dim, dev):
    """(splits, CTAs, scratch, addresses in it) of a decode call."""
    if 1 <= splits <= CLUSTER:
        return splits, 0, None, 0, 0, 0
    ctas = EVEN_CTAS * _sm_count(dev)
    n = 2 * ctas * (8 if rows <= 8 else 16)
    part = torch.empty(n * (dim + 4) + 4 * ctas, dtype=torch.float32, device=dev)
    at = part.data_ptr()
    return 0, ctas, part, at, at + n * dim * 4, at + n * (dim + 4) * 4


def attention_decode8(q, k_cache: Pages8, v_cache: Pages8, block_table, seq_lens, q_per_seq, scale, splits, window, sinks, out, chunk):
    """The form of :func:`.core.attention_decode` for 8-bit pages on a GPU. ``splits`` from 1 to 8: CTAs for a sequence and head, which meet in a cluster;
    any other number: even shares of all pages whatever the sequences' lengths are, partial sums in memory that the call allocates, and a second kernel
    that adds them up."""
    check_attention8(q, k_cache, v_cache, block_table, seq_lens, sinks, out)
    if q.shape[0] != seq_lens.shape[0] * q_per_seq:
        raise ValueError(f"{q.shape[0]} query rows for {seq_lens.shape[0]} sequences of {q_per_seq}")
    return _decode8(q, k_cache, v_cache, block_table, seq_lens, q_per_seq, scale, splits, window, sinks, out, chunk)


def _decode8(q, k_cache, v_cache, block_table, seq_lens, q_per_seq, scale, splits, window, sinks, out, chunk):
    dev, B = q.device, seq_lens.shape[0]
    n_q, dim = q.shape[1:]
    n_kv = k_cache.codes.shape[1]
    if out is None:
        out = torch.empty_like(q)
    splits, ctas, part, part_o, part_ml, joins = _shares(splits, q_per_seq * (n_q // n_kv), dim, dev)
    code = lib().eredu_attn_kv8_decode(_ATTENTION.pack(
        q.data_ptr(), 0, k_cache.codes.data_ptr(), v_cache.codes.data_ptr(), k_cache.scales.data_ptr(), v_cache.scales.data_ptr(), out.data_ptr(), block_table.data_ptr(),
        seq_lens.data_ptr(), address(sinks), part_o, part_ml, joins, 0, 0, 0, 0, 0, status_word(dev).data_ptr(), stream_ptr(dev), 0, B, q_per_seq, block_table.shape[1],
        block_table.stride(0), k_cache.codes.shape[0], n_q, n_kv, dim, 0, 0, splits, ctas, int(window), int(chunk), 0, scale, 0.0, 0.0, 0.0), _ATTENTION.size)
    check(code, "eredu_attn_kv8_decode")
    return out


def attention_step8(qkv, k_cache: Pages8, v_cache: Pages8, block_table, seq_lens, q_per_seq, scale, positions, slots, inv_freq, n_q, n_kv, dim, rot, interleaved,
                    attn_factor, q_norm_w, k_norm_w, norm_eps, norm_w_off, splits, window, sinks, chunk, settled):
    """The form of :func:`.core.attention_decode_rope` for 8-bit pages on a GPU: queries keep 16 bits from the rotation to the scores."""
    dev, B = k_cache.codes.device, seq_lens.shape[0]
    M = B * q_per_seq
    _check_qkv(qkv, M, positions, slots, inv_freq, k_cache, v_cache, n_q, n_kv, dim, rot, q_norm_w, k_norm_w)
    _check_batch(n_q, n_kv, block_table, seq_lens, sinks, dev)
    out = qkv.new_empty((M, n_q, dim))
    rows = q_per_seq * (n_q // n_kv)
    splits, ctas, part, part_o, part_ml, joins = _shares(splits, rows, dim, dev)
    q32 = torch.empty(M * n_q * dim, dtype=torch.float32, device=dev) if rows > 16 or q_per_seq > 8 else None
    code = lib().eredu_attn_kv8_step(_ATTENTION.pack(
        qkv.data_ptr(), address(q32), k_cache.codes.data_ptr(), v_cache.codes.data_ptr(), k_cache.scales.data_ptr(), v_cache.scales.data_ptr(), out.data_ptr(),
        block_table.data_ptr(), seq_lens.data_ptr(), address(sinks), part_o, part_ml, joins, positions.data_ptr(), slots.data_ptr(), inv_freq.data_ptr(), address(q_norm_w),
        address(k_norm_w), status_word(dev).data_ptr(), stream_ptr(dev), qkv.stride(0), B, q_per_seq, block_table.shape[1], block_table.stride(0), k_cache.codes.shape[0],
        n_q, n_kv, dim, rot, 1 if interleaved else 0, splits, ctas, int(window), int(chunk), 1 if settled else 0, scale, attn_factor, norm_eps, norm_w_off),
        _ATTENTION.size)
    check(code, "eredu_attn_kv8_step")
    return out


def decode_splits8(batch, n_kv, max_kv_len, sm_count=148, rows=0):
    """Split factor of the decode kernel for 8-bit pages: 1 to 8 CTAs for a sequence and head, or 0 for even shares.

    Three CTAs fit an SM, clusters not quite: as many splits as find room on nine tenths of that (two where that is all), with a pair of pages for each of a CTA's
    four warps. Even shares cost a second kernel and the way to a CTA's place, 2 to 4 us, and pay where clusters leave SMs empty and a CTA has many pairs: more
    than 48 of eight splits, which most often are all that a cluster may have and not all there is room for, and more than 84 of fewer (us, 32 heads of 128 over 8,
    even / best cluster: one sequence of 8192 tokens 13.3 / 11.9, of 12000 14.5 / 13.9, of 16384 15.2 / 17.6, of 65536 32 / 54; four of 8192 16.4 / 15.3, of 16384
    22.5 / 26.0; eight of 8192 24.2 / 23.1, of 12000 35.6 / 34.2, of 16384 43.2 / 43.6, of 32768 79 / 81; 20 of 8192 51 / 52).
    More sequences and heads than that go one CTA each, or, where they are long enough for the tail of the longest to count, two or three
    (us with 1 / 2 / 3 / even: 32 of 1024 16 / 17 / 17 / 19, of 4096 48 / 46 / 42 / 44; 64 of 2048 43 / 43 / 46 / 46, of 4096 77 / 72 / 75 / 74), or even shares where
    they are longer still. Three splits are up to a twentieth faster there when all are about as long, and far slower when one is longer than the others
    (3 / even: 64 of 8192 136 / 142, 32 of 16384 132 / 135, one of 16384 with 31 of 1024 48 / 23; 64 of 8192 with four new tokens 158 / 155)."""
    tiles = -(-max(rows, 1) // (8 if rows <= 8 else 16))
    heads = max(1, batch * n_kv * tiles)
    pairs = max(1, -(-max_kv_len // (2 * PAGE)))
    room = EVEN_CTAS * sm_count
    if heads > room // 2 + 2:
        if pairs < 96:
            return 1
        if pairs < 192:
            return 3 if 3 * heads <= 2 * room else 2
        return 0
    splits = max(1, min(max(2, room * 9 // 10 // heads), pairs // 4, CLUSTER))
    if splits == 7:             # six or eight fill a GPC better
        splits = 6
    return 0 if pairs > (48 if splits == CLUSTER else 84) * splits else splits


def decode_pays(batch, new, n_q, n_kv, dim, seen, sm_count=148):
    """Whether the decode kernel takes ``new`` query rows of each of ``batch`` sequences behind ``seen`` tokens in less time than the prefill kernel (estimates of either in us).
    The former reads the pages once for every 16 rows that share a head, 0.6 ns a page, and a tile of them costs 9 ns beside that (head size 128, about half of 64).
    The latter has a CTA for every head and 256 rows, however few they are. Those of one round take 2.1 us for 1000 keys; of more rounds each takes 4 us, and they read
    keys and values, in bf16 and once for each query head, at 6.5 TB/s. Before, the pages are brought to bf16, three bytes a value.
    Measured, decode / prefill, 32 heads of 128 over 8: 45 rows behind 512 10.4 / 15.5, behind 4096 24.2 / 24.9, behind 32768 123 / 104; 16 rows behind 32768 52 / 92; 64
    behind 4096 29 / 26; 32 sequences with 9 rows behind 200 17 / 61; 64 with 9 behind 500 46 / 187; 100 with 20 rows 53 / 129, 8 with 100 25 / 17; one with 128
    7.4 / 8.8, with 256 14.7 / 12.0. Heads of 64: 45 rows behind 4096 17.3 / 19.6, 64 rows 20.7 / 19.8, 300 rows 13.8 / 9.6."""
    part = dim / 128
    tiles = batch * n_kv * -(-new * (n_q // n_kv) // 16)
    decode = 7 + tiles * (0.002 + 0.007 * part + 0.6e-3 * part * seen / PAGE)
    ctas, keys = batch * n_q * -(-new // 256), -(-seen // 128) * 128
    attention = 2.1e-3 * part * keys
    if ctas > sm_count:
        attention = max(attention, ctas * keys * 4 * dim / 6.5e6) + 4 * (ctas / sm_count - 1)
    prefill = 12 + attention + batch * n_kv * seen * 6 * dim / 6.5e6
    return decode < prefill


def seen_pages(portions, window, chunk, wide):
    """Pages that some query of a sequence sees, of the first ``wide`` of its table, added up over sequences of (cached tokens, new tokens)."""
    count = 0
    for old, new in portions:
        if new > 0:
            low = max(0, old - window + 1) if window > 0 else old - old % chunk if chunk > 0 else 0
            count += max(0, min(wide, -(-(old + new) // PAGE)) - low // PAGE)
    return count


def attention_prefill8(q, k_cache: Pages8, v_cache: Pages8, block_table, seq_lens, cu_q, max_q_len, scale, window, sinks, out, chunk, max_kv_len, equal=False,
                       portions=None):
    """The form of :func:`.core.attention_prefill` for 8-bit pages on a GPU. The pages that some query sees are brought to bf16, in pages and a block table of
    their own, and the prefill kernel reads these: once for all query tiles and heads that share them, where a kernel that reads codes would convert
    each tile again for every one of them. Entries of that table that nobody sees point behind the last page, where the kernel's tensor maps read
    zeros; its rows are whole key tiles of eight pages. Memory: as many pages as sequences see in all where the caller states ``portions``, else as many times the
    longest row of the table as there are sequences. Where the caller says that sequences bring equally many rows (what ``cu_q`` holds is not known
    here, and rows behind its last entry are left as they are), few of them go to the decode kernel."""
    check_attention8(q, k_cache, v_cache, block_table, seq_lens, sinks, out, cu_q)
    (kc, ks), (vc, vs) = k_cache, v_cache
    dev, B, (total, n_q, dim) = q.device, seq_lens.shape[0], q.shape
    num, n_kv = kc.shape[:2]
    if out is None:
        out = torch.empty_like(q)
    if total == 0 or B == 0:
        return out
    if portions:
        if len(portions) != B:
            raise ValueError(f"{len(portions)} portions for {B} sequences")
        max_kv_len = max_kv_len or max(old + new for old, new in portions)
        equal = equal or (total == B * max_q_len and all(new == max_q_len for _, new in portions))
    if equal and max_kv_len > 0:
        seen = min(max_kv_len, window + max_q_len if window > 0 else chunk + max_q_len if chunk > 0 else max_kv_len)
        if decode_pays(B, max_q_len, n_q, n_kv, dim, seen, _sm_count(dev)):
            splits = decode_splits8(B, n_kv, seen, _sm_count(dev), max_q_len * (n_q // n_kv))
            return _decode8(q, k_cache, v_cache, block_table, seq_lens, max_q_len, scale, splits, window, sinks, out, chunk)
    wide = block_table.shape[1]
    if max_kv_len > 0:
        wide = min(wide, -(-max_kv_len // PAGE))
    wide = -(-wide // 8) * 8
    room, entries = B * wide, 0
    if portions:
        seen = max(1, seen_pages(portions, window, chunk, block_table.shape[1]))
        if seen < room:
            room = entries = seen
    half = room * n_kv * PAGE * dim * 2                                      # bytes of the keys
    held = torch.empty(2 * half + 4 * B * wide, dtype=torch.uint8, device=dev)
    at = held.data_ptr()
    table, status, stream = at + 2 * half, status_word(dev).data_ptr(), stream_ptr(dev)
    lens, cu = seq_lens.data_ptr(), cu_q.data_ptr()
    code = lib().eredu_kv8_values(_VALUES.pack(
        kc.data_ptr(), vc.data_ptr(), ks.data_ptr(), vs.data_ptr(), at, at + half, block_table.data_ptr(), lens, cu, table, status, stream, B, block_table.stride(0),
        block_table.shape[1], wide, n_kv, dim, num, int(window), int(chunk), entries), _VALUES.size)
    check(code, "eredu_kv8_values")
    code = lib().eredu_attn_prefill_tc(q.data_ptr(), at, at + half, out.data_ptr(), table, lens, cu, ptr(sinks), B, total, max_q_len, wide, room, n_q, n_kv, dim, dim,
                                       int(window), int(chunk), int(max_kv_len), _sm_count(dev), scale, status, stream)
    check(code, "eredu_attn_prefill_tc")
    return out


# ------------------------------------------------------------------------------------------ moving
def _page_list(pages, device):
    t = pages if torch.is_tensor(pages) else torch.as_tensor(list(pages), dtype=torch.int32)
    if t.is_cuda:
        return t
    return t.to(torch.int32).pin_memory().to(device, non_blocking=True) if device.type == "cuda" else t.to(torch.int32)


def copy_pages(pools, src, dst) -> None:
    """Page ``src[i]`` to page ``dst[i]`` in every layer of every tensor of ``pools``, in one launch (for eight tensors). ``pools``: tensors
    [layers, pages, ...] with pages that are contiguous. ``src``, ``dst``: page numbers on the host, which are checked (in range, no destination twice, none
    that is a source as well), or int32 tensors on the pools' device, for which that is the caller's part (pages out of range are not copied, and reported)."""
    if not pools:
        return
    dev, num = pools[0].device, pools[0].shape[1]
    words = []                  # address, bytes between layers, bytes of a page, layers
    for t in pools:
        shape, size = t.shape, t.element_size()
        if t.device != dev or len(shape) < 2 or shape[1] != num:
            raise ValueError("the pools have to have the same pages, on one device")
        if not shape[0]:
            continue
        if not t.is_contiguous() and not t[0].is_contiguous():
            raise ValueError("the pages of a layer have to be contiguous")
        page = t.stride(1) * size if num > 1 else t[0].numel() * size
        at = t.data_ptr()
        if page % 4 or at % 4:
            raise ValueError("pages have to be whole words")
        words.append((at, t.stride(0) * size, page, shape[0]))
    on_host = [x for x in (src, dst) if not (torch.is_tensor(x) and x.is_cuda)]
    if len(on_host) == 2:
        a, b = ([int(i) for i in (x.tolist() if torch.is_tensor(x) else x)] for x in (src, dst))
        if len(a) != len(b):
            raise ValueError(f"{len(a)} sources for {len(b)} destinations")
        if any(not 0 <= i < num for i in a + b):
            raise IndexError(f"a page is not one of {num}")
        if len(set(b)) != len(b) or set(a) & set(b):
            raise ValueError("a page is the destination of two copies, or a destination and a source")
        if not a:
            return
        src, dst = a, b
    elif on_host:
        raise ValueError("sources and destinations are either both on the host or both on the device")
    elif src.shape != dst.shape or src.dim() != 1 or any(t.dtype != torch.int32 or not t.is_contiguous() or t.device != dev for t in (src, dst)):
        raise ValueError(f"src, dst: int32 vectors of one length on {dev}")
    if dev.type != "cuda":
        for t in pools:
            t[:, list(dst)] = t[:, list(src)]
        return
    if on_host:
        both = _page_list(src + dst, dev)
        src, dst = both[:len(src)], both[len(src):]
    n = src.shape[0]
    if n == 0:
        return
    for i in range(0, len(words), 8):
        part = words[i:i + 8]
        code = lib().eredu_copy_pages(struct.pack(f"{4 * len(part)}q", *(w for t in part for w in t)), len(part), src.data_ptr(), dst.data_ptr(), n, num,
                                      status_word(dev).data_ptr(), stream_ptr(dev))
        check(code, "eredu_copy_pages")
