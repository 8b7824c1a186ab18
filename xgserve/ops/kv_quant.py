"""The 8-bit paged KV cache, the attentions over it, and decode attention of sequences that share a prefix.

`QuantKVCache` holds keys and values of one layer in pages as 8-bit codes with one fp32 scale per token, kv head and side. A row
x of D bf16 numbers whose largest magnitude is a is held as

    int8   code = round(127 x / a), ties to even              value = code a / 127
    fp8    code = round(448 x / a) to E4M3, ties to even      value = code a / 448

(off by at most a / 254 for int8; for fp8 by 2^-4 of the number, or by 2^-10 a / 448 where that is more: codes below 2^-6 have
steps of 2^-9). A row of zeros reads back as zeros; a row that holds an infinity or NaN reads back as NaN throughout, and so does
what attends to it.

Attention sums in 32 bits; weights (times the values' scales) are rounded to bf16 before their product, which takes an output's
error from 1.6e-3 of it in root mean square (its own rounding) to 2.0 to 2.4e-3. Values may be of any size that bf16 holds, as long
as a sequence whose first keys' values are below 2^-64 has none above 2^50 later.

All GPU calls go to the current stream of the current device, allocate nothing but their outputs and (without a workspace)
the parts of a split, and can be captured; a workspace belongs to one call at a time, so captured graphs that may run at the
same time, or eager calls beside them, each need their own. Page numbers of a table are kept within the cache.
"""
from __future__ import annotations

import math
from dataclasses import dataclass
from typing import List, Optional, Sequence, Tuple, Union

import torch

from ._native import kernels, loaded, ptr, stream_ptr, use_native
from .attention import DecodeWorkspace, _attend
from .rope import _rotate

KV_BF16, KV_FP8, KV_INT8 = 0, 1, 2
KV_FORMATS = {"fp8": KV_FP8, "int8": KV_INT8}
LARGEST = {"fp8": 448.0, "int8": 127.0}
TILE = 16           # tokens whose codes lie together in the order of the matrix instructions (csrc/kernels/kv_quant.h)
MAX_SPLITS = 64
# us of decode, one part / the parts that this makes: 1 sequence of 640 keys 5.9 / 7.7, 1280 8.2 / 7.9, 5120 36 / 10.3; 16 of 640
# 8.9 / 11.7, 5120 44 / 35; 48 of 1280 24.6 / 32.6 (8 kv heads of 128, fp8). Below SPLIT_FROM keys a second launch costs more
SPLIT_WGS = 512     # workgroups that fill the chip: two a CU
SPLIT_KEYS = 128    # a workgroup's four waves have a 32-key tile each
WHOLE_UNITS = 16    # units of SPLIT_KEYS that stay whole where the sequences alone fill most of the chip
SPLIT_FROM = 1024
# the common parts of shared prefixes: at most one workgroup a CU leaves room for the sequences' own keys beside them (64 sequences
# behind 4096 keys, bf16: 256 workgroups 34.5 us, 384 39.0, 512 42.7, 768 46.7; 64 heads on 8 of 20 behind 3000: 18.3, 19.4, 24.4, 26.5),
# or two a CU where one would have PREFIX_LONG 32-key tiles and more (fp8, 256 / 384 / 512: 27 behind 40 k with up to 100 keys of their own
# 48 / 47 / 40, up to 900 51 / 49 / 46; 5 groups of 27 behind 5 - 30 k 111 / 85 / 85; 27 behind 60 k 72 / 64 / 55. Shorter ones, 64 behind
# 16 k with up to 900, have 43 / 46 / 51)
PREFIX_WGS = 256
PREFIX_LONG = 144


def _need(ok: bool, what: str) -> None:
    if not ok:
        raise ValueError(what)


def _int32(t: torch.Tensor, name: str, dims: int, device) -> None:
    if t.dtype != torch.int32:
        raise TypeError(f"{name} must be int32, got {t.dtype}")
    _need(t.dim() == dims and (t.numel() == 0 or t.shape[-1] == 1 or t.stride(-1) == 1),
          f"{name} must have {dims} dimension(s), contiguous in the last")
    _need(t.device == device, f"{name} is on {t.device}, the cache on {device}")


# ---------------------------------------------------------------------------------------------------------------- the cache
@dataclass
class QuantKVCache:
    """One layer's keys and values in pages. `k`, `v`: codes [num_blocks, Hkv, block_size, D] uint8, where the 16 D codes of 16 tokens
    lie in tile order (`kv_quant_read` gives rows); `scales` [num_blocks, Hkv, 2, block_size] fp32: the keys', then the values'. A
    page is the same bytes wherever it lies, so whole pages may be copied, saved and moved."""
    k: torch.Tensor
    v: torch.Tensor
    scales: torch.Tensor
    fmt: str

    @classmethod
    def alloc(cls, num_blocks: int, num_kv_heads: int, block_size: int, head_dim: int, fmt: str = "fp8",
              device="cuda") -> "QuantKVCache":
        """An empty cache: every row reads back as zeros."""
        shape = (num_blocks, num_kv_heads, block_size, head_dim)
        return cls(torch.zeros(shape, dtype=torch.uint8, device=device), torch.zeros(shape, dtype=torch.uint8, device=device),
                   torch.zeros(num_blocks, num_kv_heads, 2, block_size, dtype=torch.float32, device=device), fmt)

    def __post_init__(self):
        _need(self.fmt in KV_FORMATS, f"format must be one of {sorted(KV_FORMATS)}, got {self.fmt!r}")
        _need(self.k.dim() == 4 and self.k.shape == self.v.shape, "k and v must be [num_blocks, Hkv, block_size, D] alike")
        nb, hkv, bs, d = self.k.shape
        _need(nb >= 1 and hkv >= 1, "a cache has at least one page and one head")
        _need(d in (64, 128), f"heads of 64 or 128 numbers, got {d}")
        _need(bs >= TILE and bs % TILE == 0, f"pages of a multiple of {TILE} tokens, got {bs}")
        _need(nb * bs < 1 << 31, "slots are 32-bit numbers")
        if self.k.dtype != torch.uint8 or self.v.dtype != torch.uint8 or self.scales.dtype != torch.float32:
            raise TypeError("codes are uint8 and scales float32")
        _need(tuple(self.scales.shape) == (nb, hkv, 2, bs), "scales must be [num_blocks, Hkv, 2, block_size]")
        _need(all(t.is_contiguous() for t in (self.k, self.v, self.scales)), "a cache is contiguous")
        _need(self.k.device == self.v.device == self.scales.device, "a cache is on one device")
        _need(all(t.data_ptr() % 16 == 0 for t in (self.k, self.v, self.scales)), "a cache's parts begin at multiples of 16 bytes")
        self.num_blocks, self.num_kv_heads, self.block_size, self.head_dim = self.dims = nb, hkv, bs, d
        self.device, self.code = self.k.device, KV_FORMATS[self.fmt]
        self.index = self.k.get_device()   # -1: host

    def nbytes(self) -> int:
        return self.k.numel() + self.v.numel() + 4 * self.scales.numel()


def _native(cache_tensor: torch.Tensor) -> bool:
    index = cache_tensor.get_device()
    if index < 0:
        return False
    if index != torch._C._cuda_getDevice():
        raise ValueError(f"the cache is on {cache_tensor.device}, which is not the current device")
    return loaded() or use_native(cache_tensor)


# Arguments are looked over twice: one condition asks whether all is as it nearly always is, each shape and stride asked for once (a call
# of single tokens is mostly host time), and where it is not, `_check_*` and `_int32` allow it or say what is wrong.
_BF16, _I32 = torch.bfloat16, torch.int32


def _plain_lists(index: int, n: int, *lists: torch.Tensor) -> bool:
    for t in lists:
        if t.dtype is not _I32 or t.shape != (n,) or not t.is_contiguous() or t.get_device() != index:
            return False
    return True


# ------------------------------------------------------------------------------------------------------ plain (CPU) forms
_ORDERS = {}


def _order(D: int, device) -> Tuple[torch.Tensor, torch.Tensor]:
    """Bytes of codes (t, d) of a tile, keys' and values', [16, D]."""
    key = (D, str(device))
    if key not in _ORDERS:
        t, d = torch.arange(TILE)[:, None], torch.arange(D)[None]
        k = ((d // 16) * 16 + t) * 16 + d % 16
        v = ((d // 64) * 64 + 16 * (t // 4) + d % 16) * 16 + (d // 16) % 4 * 4 + t % 4
        _ORDERS[key] = (k.to(device), v.to(device))
    return _ORDERS[key]


def quantize_rows_ref(x: torch.Tensor, fmt: str) -> Tuple[torch.Tensor, torch.Tensor]:
    """Codes (uint8 bytes) and fp32 scales of rows [..., D]."""
    a = x.abs().amax(-1, keepdim=True).double()
    bad = ~torch.isfinite(x).all(-1, keepdim=True)
    y = torch.where(bad | (a == 0), 0.0, x.double() * LARGEST[fmt] / torch.where(bad | (a == 0), 1.0, a))
    codes = y.float().to(torch.float8_e4m3fn) if fmt == "fp8" else y.round().to(torch.int8)
    scale = torch.where(bad, math.nan, a).float() / torch.tensor(LARGEST[fmt], device=x.device)
    return codes.view(torch.uint8), scale[..., 0]


def _tile_index(cache: QuantKVCache, slots: torch.Tensor):
    """Pages, offsets in a page, and bytes of the page's rows of a head, keys' and values' [n, D], of slots."""
    slots = slots.long()
    pages, offs = slots // cache.block_size, slots % cache.block_size
    ko, vo = _order(cache.head_dim, cache.device)
    base = ((offs // TILE) * TILE * cache.head_dim)[:, None]
    return pages, offs, base + ko[offs % TILE], base + vo[offs % TILE]


def kv_quant_append_ref(k, v, cache: QuantKVCache, slot_mapping) -> None:
    real = (slot_mapping >= 0) & (slot_mapping.long() < cache.num_blocks * cache.block_size)
    if not bool(real.any()):
        return
    pages, offs, ko, vo = _tile_index(cache, slot_mapping[real])
    flat = (cache.num_blocks, cache.num_kv_heads, cache.block_size * cache.head_dim)
    heads = torch.arange(cache.num_kv_heads, device=cache.device)
    for side, (x, codes, order) in enumerate(((k, cache.k, ko), (v, cache.v, vo))):
        c, s = quantize_rows_ref(x[real], cache.fmt)
        codes.view(flat)[pages[:, None, None], heads[None, :, None], order[:, None, :]] = c
        cache.scales[pages, :, side, offs] = s


def _rows_ref(cache: QuantKVCache, slots: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """fp32 rows [n, Hkv, D] of slots."""
    pages, offs, ko, vo = _tile_index(cache, slots)
    flat = (cache.num_blocks, cache.num_kv_heads, cache.block_size * cache.head_dim)
    heads = torch.arange(cache.num_kv_heads, device=cache.device)
    out = []
    for side, (codes, order) in enumerate(((cache.k, ko), (cache.v, vo))):
        c = codes.view(flat)[pages[:, None, None], heads[None, :, None], order[:, None, :]]
        c = c.view(torch.float8_e4m3fn if cache.fmt == "fp8" else torch.int8).float()
        out.append(c * cache.scales[pages, :, side, offs][..., None])
    return out[0], out[1]


def _slots_ref(table_row: torch.Tensor, bs: int, lo: int, hi: int, num_blocks: int) -> torch.Tensor:
    at = torch.arange(lo, hi, device=table_row.device)
    return table_row.long()[at // bs].clamp(0, num_blocks - 1) * bs + at % bs


def _any_rows_ref(kv, table_row, lo: int, hi: int) -> Tuple[torch.Tensor, torch.Tensor]:
    if isinstance(kv, QuantKVCache):
        return _rows_ref(kv, _slots_ref(table_row, kv.block_size, lo, hi, kv.num_blocks))
    bs, nb = kv[0].shape[2], kv[0].shape[0]
    slots = _slots_ref(table_row, bs, lo, hi, nb)
    return tuple(x[slots // bs, :, slots % bs].float() for x in kv)


def _attend_causal(q, k, v, first: int, scale: float) -> torch.Tensor:
    """q [n, Hq, D] at positions first .. over fp32 rows; a value that is NaN reaches the queries that see it and no others."""
    n, Hq, _ = q.shape
    pos = torch.arange(first, first + n, device=q.device)
    bad = v.isnan().any(-1)                                           # [L, Hkv]
    out = _attend(q, k, v.masked_fill(bad[..., None], 0.0), pos, scale)
    reached = (bad.cumsum(0) > 0)[pos.clamp(max=k.shape[0] - 1)] if k.shape[0] else bad.new_zeros(n, bad.shape[1])
    return out.masked_fill(reached.repeat_interleave(Hq // bad.shape[1], 1)[..., None], math.nan)


# --------------------------------------------------------------------------------------------------------- write and read
def _check_rows(x: torch.Tensor, name: str, cache: QuantKVCache, T: int) -> None:
    if x.dtype != torch.bfloat16:
        raise TypeError(f"{name} must be bfloat16, got {x.dtype}")
    H, D = cache.num_kv_heads, cache.head_dim
    _need(x.dim() == 3 and tuple(x.shape) == (T, H, D), f"{name} must be [{T}, {H}, {D}], got {tuple(x.shape)}")
    _need(x.device == cache.device, f"{name} is on {x.device}, the cache on {cache.device}")
    if T:
        _need(x.stride(2) == 1 and (H == 1 or x.stride(1) == D), f"{name}'s heads must be contiguous within a token")
        _need(x.stride(0) % (D // 16) == 0 and x.data_ptr() % (D // 8) == 0, f"{name}'s tokens must begin at multiples of {D // 8} bytes")


def kv_quant_append(k: torch.Tensor, v: torch.Tensor, cache: QuantKVCache, slot_mapping: torch.Tensor) -> None:
    """Writes rows k, v [T, Hkv, D] bf16 (tokens may be strided: views into the projection's rows) to the cache's slots
    slot_mapping [T] int32; tokens with a slot below 0 or behind the cache are left out. A slot may occur once in a call."""
    (nb, Hkv, bs, D), index, shape, sk, sv = cache.dims, cache.index, k.shape, k.stride(), v.stride()
    T, kp, vp = shape[0], k.data_ptr(), v.data_ptr()
    if not (shape == (T, Hkv, D) and v.shape == shape and sk[2] == 1 == sv[2] and sk[1] == D == sv[1] and sk[0] % (D // 16) == 0
            and sv[0] % (D // 16) == 0 and kp % (D // 8) == 0 and vp % (D // 8) == 0 and k.dtype is _BF16 and v.dtype is _BF16
            and k.get_device() == index and v.get_device() == index and _plain_lists(index, T, slot_mapping)):
        _check_rows(k, "k", cache, T)
        _check_rows(v, "v", cache, T)
        _int32(slot_mapping, "slot_mapping", 1, cache.device)
        _need(slot_mapping.shape[0] == T, f"slot_mapping must have {T} entries")
    if T == 0:
        return
    if not _native(cache.k):
        return kv_quant_append_ref(k, v, cache, slot_mapping)
    kernels().kv_append(cache.code, 0, kp, sk[0], vp, sv[0], slot_mapping.data_ptr(), 0, 0, cache.k.data_ptr(), cache.v.data_ptr(),
                        cache.scales.data_ptr(), nb, T, 0, Hkv, D, bs, stream_ptr())


def _check_cos_sin(cos_sin: torch.Tensor, cache: QuantKVCache) -> None:
    if cos_sin.dtype is not torch.float32:
        raise TypeError("cos_sin must be float32")
    if not (cos_sin.dim() == 2 and cos_sin.shape[1] == cache.head_dim and cos_sin.is_contiguous() and cos_sin.get_device() == cache.index):
        raise ValueError(f"cos_sin must be a contiguous [max_pos, {cache.head_dim}] table beside the cache")


def rope_kv_quant(qkv: torch.Tensor, positions: torch.Tensor, cos_sin: torch.Tensor, cache: QuantKVCache,
                  slot_mapping: torch.Tensor, num_heads: int, apply_rope: bool = True) -> None:
    """`rope_cache` for an 8-bit cache: rows qkv [T, (Hq + 2 Hkv) D] bf16, q rotated in place, k rotated (to bf16, as the bf16
    cache holds it) and v written to the cache in 8 bits. positions [T] int32 within cos_sin [max_pos, D] fp32."""
    H, D, T = cache.num_kv_heads, cache.head_dim, qkv.shape[0]
    _need(qkv.dim() == 2 and qkv.shape[1] >= (num_heads + 2 * H) * D and (T == 0 or qkv.stride(1) == 1),
          "qkv must be [T, (Hq + 2 Hkv) D], contiguous in the last dimension")
    _need(T < 2 or qkv.stride(0) >= qkv.shape[1], "qkv's tokens must not overlap")
    k = qkv[:, num_heads * D:(num_heads + H) * D].unflatten(1, (H, D))
    v = qkv[:, (num_heads + H) * D:(num_heads + 2 * H) * D].unflatten(1, (H, D))
    if not apply_rope:
        return kv_quant_append(k, v, cache, slot_mapping)
    _check_rows(k, "qkv", cache, T)
    _int32(slot_mapping, "slot_mapping", 1, cache.device)
    _int32(positions, "positions", 1, cache.device)
    _need(slot_mapping.shape[0] == T and positions.shape[0] == T, f"slot_mapping and positions must have {T} entries")
    _check_cos_sin(cos_sin, cache)
    if T == 0:
        return
    if not _native(cache.k):
        cs = cos_sin[positions.long()]
        cos, sin = cs[:, None, :D // 2], cs[:, None, D // 2:]
        q = qkv[:, :num_heads * D].unflatten(1, (num_heads, D))
        q.copy_(_rotate(q.float(), cos, sin).to(qkv.dtype))
        return kv_quant_append_ref(_rotate(k.float(), cos, sin).to(torch.bfloat16), v, cache, slot_mapping)
    nb, _, bs, _ = cache.dims
    kernels().kv_append(cache.code, qkv.data_ptr(), k.data_ptr(), k.stride(0), v.data_ptr(), v.stride(0), slot_mapping.data_ptr(),
                        positions.data_ptr(), cos_sin.data_ptr(), cache.k.data_ptr(), cache.v.data_ptr(), cache.scales.data_ptr(), nb, T,
                        num_heads, H, D, bs, stream_ptr())


def rope_kv_quant_partials(pend, positions: torch.Tensor, cos_sin: torch.Tensor, cache: QuantKVCache, slot_mapping: torch.Tensor,
                           num_heads: int, apply_rope: bool = True) -> torch.Tensor:
    """`rope_cache_partials` for an 8-bit cache: QKV as split-K partial sums (PendingSum [S, T, (Hq + 2 Hkv) D]); k and v to the
    cache, q -> [T, Hq D] bf16."""
    H, D = cache.num_kv_heads, cache.head_dim
    S, T, W = pend.part.shape
    index = cache.index
    if not (W == (num_heads + 2 * H) * D and pend.part.dtype is torch.float32 and pend.part.is_contiguous()
            and pend.part.get_device() == index and pend.part.data_ptr() % 16 == 0):
        raise ValueError(f"partial sums must be contiguous float32 [S, T, {(num_heads + 2 * H) * D}] beside the cache")
    if not (_plain_lists(index, T, slot_mapping, positions)):
        _int32(slot_mapping, "slot_mapping", 1, cache.device)
        _int32(positions, "positions", 1, cache.device)
        _need(slot_mapping.shape[0] == T and positions.shape[0] == T, f"slot_mapping and positions must have {T} entries")
    _check_cos_sin(cos_sin, cache)
    q = torch.empty(T, num_heads * D, dtype=torch.bfloat16, device=cache.device)
    if T == 0:
        return q
    if not _native(cache.k):
        qkv = pend.part.sum(0)
        k, v = (qkv[:, (num_heads + i * H) * D:(num_heads + (i + 1) * H) * D].unflatten(1, (H, D)) for i in (0, 1))
        x = qkv[:, :num_heads * D].unflatten(1, (num_heads, D))
        if apply_rope:
            cs = cos_sin[positions.long()]
            x, k = (_rotate(y, cs[:, None, :D // 2], cs[:, None, D // 2:]) for y in (x, k))
        kv_quant_append_ref(k.to(torch.bfloat16), v.to(torch.bfloat16), cache, slot_mapping)
        return q.copy_(x.flatten(1))
    nb, _, bs, _ = cache.dims
    kernels().kv_append_partials(cache.code, pend.part.data_ptr(), S, q.data_ptr(), num_heads * D, slot_mapping.data_ptr(),
                                 positions.data_ptr(), cos_sin.data_ptr() if apply_rope else 0, cache.k.data_ptr(),
                                 cache.v.data_ptr(), cache.scales.data_ptr(), nb, T, num_heads, H, D, bs, stream_ptr())
    return q


def kv_quant_read(cache: QuantKVCache, block_tables: torch.Tensor, starts: torch.Tensor, cu_tokens: torch.Tensor, num_tokens: int,
                  out: Optional[Tuple[torch.Tensor, torch.Tensor]] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Cached rows as bf16: tokens starts[s] .. starts[s] + cu_tokens[s + 1] - cu_tokens[s] of each sequence, packed
    -> k, v [num_tokens, Hkv, D]. block_tables [S, W], starts [S], cu_tokens [S + 1] (from 0, not falling) int32; num_tokens =
    cu_tokens[S]. Tokens behind a sequence's table have no row: theirs stay as they were in `out`."""
    nb, Hkv, bs, D = cache.dims
    index, counts, table, steps = cache.index, starts.shape, block_tables.shape, block_tables.stride()
    S = counts[0]
    if not (len(counts) == 1 and len(table) == 2 and table[0] == S and table[1] > 0 and steps[1] == 1 and cu_tokens.shape == (S + 1,)
            and starts.is_contiguous() and cu_tokens.is_contiguous() and block_tables.dtype is _I32 and starts.dtype is _I32
            and cu_tokens.dtype is _I32 and block_tables.get_device() == index and starts.get_device() == index
            and cu_tokens.get_device() == index and num_tokens >= 0):
        _int32(block_tables, "block_tables", 2, cache.device)
        _int32(starts, "starts", 1, cache.device)
        _int32(cu_tokens, "cu_tokens", 1, cache.device)
        _need(block_tables.shape[0] == S and cu_tokens.shape[0] == S + 1, "starts must have an entry a sequence, cu_tokens one more")
        _need(num_tokens >= 0, "num_tokens must not be negative")
    W, shape = table[1], (num_tokens, Hkv, D)
    if out is None:
        k = torch.empty_strided(shape, (Hkv * D, D, 1), dtype=_BF16, device=cache.device)   # (half of empty's host time)
        v = torch.empty_like(k)
    else:
        k, v = out
        for t in (k, v):
            _need(t.dtype == torch.bfloat16 and tuple(t.shape) == shape and t.is_contiguous() and t.device == cache.device
                  and t.data_ptr() % 16 == 0, f"out must be two contiguous, aligned bfloat16 {list(shape)} beside the cache")
    if num_tokens == 0 or S == 0 or W == 0:
        return k, v
    if not _native(cache.k):
        for s in range(S):
            lo, a, b = int(starts[s]), int(cu_tokens[s]), min(int(cu_tokens[s + 1]), num_tokens)
            n = min(b - a, W * cache.block_size - lo)
            if n > 0 and lo >= 0:
                k[a:a + n], v[a:a + n] = _rows_ref(cache, _slots_ref(block_tables[s], cache.block_size, lo, lo + n, cache.num_blocks))
        return k, v
    kernels().kv_read(cache.code, cache.k.data_ptr(), cache.v.data_ptr(), cache.scales.data_ptr(), block_tables.data_ptr(),
                      steps[0], W, starts.data_ptr(), cu_tokens.data_ptr(), S, num_tokens, nb, Hkv, D, bs,
                      k.data_ptr(), v.data_ptr(), stream_ptr())
    return k, v


# -------------------------------------------------------------------------------------------------------------- attention
def _check_q(q: torch.Tensor, Hkv: int, D: int, device) -> None:
    if q.dtype != torch.bfloat16:
        raise TypeError(f"q must be bfloat16, got {q.dtype}")
    _need(q.dim() == 3 and q.shape[2] == D and q.shape[1] >= 1 and q.shape[1] % Hkv == 0,
          f"q must be [tokens, a multiple of {Hkv} heads, {D}], got {tuple(q.shape)}")
    _need(q.device == device, f"q is on {q.device}, the cache on {device}")
    if q.shape[0]:
        _need(q.stride(2) == 1 and (q.shape[1] == 1 or q.stride(1) == D), "q's heads must be contiguous within a token")
        _need(q.stride(0) % 8 == 0 and q.data_ptr() % 16 == 0, "q's tokens must begin at multiples of 16 bytes")


def _check_out(out: Optional[torch.Tensor], q: torch.Tensor) -> Tuple[torch.Tensor, int]:
    """The output, and the stride of its tokens."""
    if out is None:
        return torch.empty_like(q, memory_format=torch.contiguous_format), q.shape[1] * q.shape[2]
    if out.dtype != q.dtype:
        raise TypeError(f"out must be {q.dtype}, got {out.dtype}")
    _need(out.shape == q.shape and out.device == q.device, f"out must be {list(q.shape)} beside q")
    _need(q.shape[0] < 2 or out.stride(0) >= q.shape[1] * q.shape[2], "out's tokens must not overlap")
    if q.shape[0]:
        _need(out.stride(2) == 1 and (q.shape[1] == 1 or out.stride(1) == q.shape[2]) and out.stride(0) % 4 == 0
              and out.data_ptr() % 8 == 0, "out's heads must be contiguous within a token, and tokens begin at multiples of 8 bytes")
    return out, out.stride()[0]


def _check_tables(block_tables, seq_lens, device, S: int) -> None:
    _int32(block_tables, "block_tables", 2, device)
    _int32(seq_lens, "seq_lens", 1, device)
    _need(block_tables.shape[0] == S and seq_lens.shape[0] == S, f"block_tables and seq_lens must have {S} rows")
    _need(block_tables.shape[1] >= 1 or S == 0, "block_tables must have a column")


def _check_queries(q, Hkv: int, D: int, index: int, device, block_tables, seq_lens, S: int) -> Tuple[int, int, int, int, int]:
    """q, and tables and lengths of S sequences -> tokens, query heads, columns, strides of q's tokens and of the table's rows."""
    shape, sq, table, st = q.shape, q.stride(), block_tables.shape, block_tables.stride()
    if not (len(shape) == 3 and shape[2] == D == sq[1] and sq[2] == 1 and sq[0] % 8 == 0 and shape[1] % Hkv == 0 < shape[1]
            and len(table) == 2 and table[0] == S and table[1] > 0 and st[1] == 1 and seq_lens.shape == (S,)
            and seq_lens.is_contiguous() and q.dtype is _BF16 and block_tables.dtype is _I32 and seq_lens.dtype is _I32
            and q.get_device() == index and block_tables.get_device() == index and seq_lens.get_device() == index
            and q.data_ptr() % 16 == 0):
        _check_q(q, Hkv, D, device)
        _check_tables(block_tables, seq_lens, device, S)
    return shape[0], shape[1], table[1], sq[0], st[0]


def _splits(num_splits: Optional[int], wgs: int, max_keys: int) -> int:
    """Parts of the key range: enough workgroups to fill the chip, each with a tile for each of its waves."""
    if num_splits is None:
        return 1 if max_keys < SPLIT_FROM else max(1, min(-(-SPLIT_WGS // max(1, wgs)), -(-max_keys // SPLIT_KEYS), MAX_SPLITS))
    if not 1 <= num_splits <= MAX_SPLITS:
        raise ValueError(f"num_splits must be 1 to {MAX_SPLITS}, got {num_splits}")
    return int(num_splits)


def _shares(num_splits: Optional[int], B: int, wgs: int, max_keys: int) -> Tuple[int, int]:
    """Shares of a batch's keys, which the kernel gives out by the sequences' lengths: B for one part each. wgs: workgroups a share.
    And the units that a share has at least. Where the sequences alone fill most of the chip, only those longer than the mean and
    than WHOLE_UNITS are cut, and none where none can be long: us whole and with that, 64 of 500 - 8000 keys on 8 kv heads 111 / 120,
    1 of 60 k beside 63 of 500 428 / 41. The kernel cuts a sequence into 128 parts at most."""
    if num_splits is None:
        full = 8 * B * wgs >= 3 * SPLIT_WGS
        if max_keys < SPLIT_FROM * (4 if full else 1):
            return B, 1
        more = min(-(-SPLIT_WGS // wgs), B * -(-max_keys // SPLIT_KEYS))
        return (B + min(more, B), WHOLE_UNITS) if full else (B + more, 1)
    return B * _splits(num_splits, 1, 0), 1


def _parts(workspace: Optional[DecodeWorkspace], parts: int, D: int, device):
    """The parts' buffer and the addresses of outputs [parts, D] and log-sums [parts] in it."""
    if workspace is None:
        buf = torch.empty_strided((parts * (D + 1),), (1,), dtype=torch.float32, device=device)
        at = buf.data_ptr()
        return buf, at, at + 4 * parts * D
    if workspace.part_lse.device != device or workspace.part_lse.numel() < parts or workspace.part_out.numel() < parts * D:
        raise ValueError(f"the workspace is too small for {parts} parts of {D}, or on another device")
    return workspace, workspace.part_out.data_ptr(), workspace.part_lse.data_ptr()


def quant_decode_attention(q: torch.Tensor, cache: QuantKVCache, block_tables: torch.Tensor, seq_lens: torch.Tensor, scale: float,
                           num_splits: Optional[int] = None, workspace: Optional[DecodeWorkspace] = None,
                           out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """`decode_attention` over an 8-bit cache: q [B, Hq, D] bf16 (tokens may be strided), one new token of each sequence, whose own
    key is in the cache already -> [B, Hq, D]. block_tables [B, W], seq_lens [B] int32; a length of 0 gives zeros, one behind the
    table means the whole table. num_splits: parts that a sequence's keys are cut into on average, more the longer it is; a workspace
    needs B num_splits of them (None: by the batch and the table's width, at most B + 512)."""
    (nb, Hkv, bs, D), dev = cache.dims, cache.device
    B, Hq, W, q_stride, t_stride = _check_queries(q, Hkv, D, cache.index, dev, block_tables, seq_lens, q.shape[0])
    out, out_stride = _check_out(out, q)
    blocks = -(-Hq // Hkv // 16)
    shares, least = _shares(num_splits, B, Hkv * blocks, W * bs)
    if B == 0:
        return out
    if shares * blocks > 65535:
        raise ValueError("at most 65535 parts (for each 16 query heads of a kv head)")
    if not _native(cache.k):
        for b in range(B):
            L = min(int(seq_lens[b]), W * bs)
            out[b] = 0
            if L > 0:
                k, v = _any_rows_ref(cache, block_tables[b], 0, L)
                out[b] = _attend(q[b:b + 1], k, v, torch.tensor([L - 1], device=q.device), scale)[0].to(q.dtype)
        return out
    keep, po, pl = _parts(workspace, shares * Hq, D, dev) if shares > B else (None, 0, 0)
    kernels().quant_decode_attention(cache.code, q.data_ptr(), q_stride, cache.k.data_ptr(), cache.v.data_ptr(),
                                     cache.scales.data_ptr(), block_tables.data_ptr(), t_stride, W,
                                     seq_lens.data_ptr(), po, pl, out.data_ptr(), out_stride, B, Hq, Hkv, D, bs, nb, scale,
                                     shares, least, stream_ptr())
    return out


def _row_tiles(rows: int, lists: int) -> int:
    """16-row tiles of a workgroup over `lists` lists of up to `rows` rows: one or two for all four waves, each with keys of its own, or
    eight, two a wave, over the same keys. More rows read and widen the keys less often; fewer make more workgroups. us with 1, 2
    and 8 (8 kv heads, G = 4): a prompt of 128 tokens 5.4 / 7.2 / 11.5, 512 14.1 / 11.5 / 20.4, 2048 76.3 / 56.6 / 60.3, four of
    2000 behind 1500 tokens 515 / 380 / 342 (int8 714 / 474 / 358)."""
    if lists * -(-rows // 128) >= 2 * SPLIT_WGS:
        return 8
    return 2 if lists * -(-rows // 32) >= SPLIT_WGS else 1


def quant_prefill_attention(q: torch.Tensor, cache: QuantKVCache, block_tables: torch.Tensor, query_start_loc: torch.Tensor,
                            seq_lens: torch.Tensor, max_q_len: int, scale: float, num_splits: Optional[int] = None,
                            workspace: Optional[DecodeWorkspace] = None, out: Optional[torch.Tensor] = None,
                            row_tiles: Optional[int] = None) -> torch.Tensor:
    """`prefill_attention` over an 8-bit cache: q [T, Hq, D] bf16 packed; sequence s has the tokens query_start_loc[s] ..
    query_start_loc[s + 1], the last of its seq_lens[s], and each sees the keys up to its own, all of them in the cache already.
    max_q_len: at least the tokens of the longest portion. Rows of no sequence stay as they were in `out`. row_tiles (tests / A/B
    sweeps; None = `_row_tiles`): 1, 2 or 8."""
    (nb, Hkv, bs, D), dev, index = cache.dims, cache.device, cache.index
    S = seq_lens.shape[0]
    T, Hq, W, q_stride, t_stride = _check_queries(q, Hkv, D, index, dev, block_tables, seq_lens, S)
    if not _plain_lists(index, S + 1, query_start_loc):
        _int32(query_start_loc, "query_start_loc", 1, dev)
        _need(query_start_loc.shape[0] == S + 1, "query_start_loc must have one entry more than seq_lens")
    _need(0 <= max_q_len, "max_q_len must not be negative")
    out, out_stride = _check_out(out, q)
    if T == 0 or S == 0 or max_q_len == 0:
        return out
    G = Hq // Hkv
    max_q_len = min(max_q_len, T)
    rt = _row_tiles(max_q_len * G, S * Hkv) if row_tiles is None else row_tiles
    if rt not in (1, 2, 8):
        raise ValueError(f"row_tiles must be 1, 2 or 8, got {rt}")
    blocks = -(-max_q_len * G // (16 * rt))
    splits = _splits(num_splits, S * Hkv * blocks, W * bs)
    if S * splits > 65535 or blocks > 65535:
        raise ValueError("at most 65535 sequences (times splits), and blocks of rows")
    if not _native(cache.k):
        for s in range(S):
            a, b = int(query_start_loc[s]), int(query_start_loc[s + 1])
            n, L = min(b - a, max_q_len), int(seq_lens[s])
            if n > 0:
                k, v = _any_rows_ref(cache, block_tables[s], 0, max(0, min(L, W * bs)))
                out[a:a + n] = _attend_causal(q[a:a + n], k, v, max(L - (b - a), 0), scale).to(q.dtype)
        return out
    keep, po, pl = _parts(workspace, T * Hq * splits, D, dev) if splits > 1 else (None, 0, 0)
    kernels().quant_prefill_attention(cache.code, q.data_ptr(), q_stride, cache.k.data_ptr(), cache.v.data_ptr(),
                                      cache.scales.data_ptr(), block_tables.data_ptr(), t_stride, W,
                                      query_start_loc.data_ptr(), seq_lens.data_ptr(), po, pl, out.data_ptr(), out_stride, T, S,
                                      max_q_len, Hq, Hkv, D, bs, nb, scale, rt, splits, stream_ptr())
    return out


# ----------------------------------------------------------------------------------------------------------- shared prefixes
@dataclass
class PrefixWork:
    """What the workgroups of the groups' common keys do."""
    row_tiles: int               # 16-row tiles of a workgroup
    slots: int                   # most parts that a prefix is cut into
    items: torch.Tensor          # [n, 8] int32: first sequence, sequences, block of rows, first key, end key, slot
    counts: torch.Tensor         # [num_seqs] int32: parts of each sequence's prefix
    n: int                       # items


@dataclass
class SharedPrefixPlan:
    """Which sequences of a decode batch share which prefix, and the launch's work (`shared_prefix_plan`)."""
    num_seqs: int
    num_heads: int
    num_kv_heads: int
    work: PrefixWork
    wide: Optional[PrefixWork]   # of bf16 pages, where blocks of 128 rows pay
    slots: int                   # most parts of either
    prefix: torch.Tensor         # [num_seqs] int32: keys that the common part covers
    group_sizes: Tuple[int, ...]
    prefix_lens: Tuple[int, ...]
    shortest: int                # prefix
    longest: int


# bf16 pages, whose K and V each wave turns through LDS: blocks of 128 rows share that, from rows that nearly fill one and a share of
# the work on which their longer start is lost. us with blocks of 32 / 128 rows: 5 groups of 108 rows behind 5 - 30 k keys 132 / 113, 108
# rows behind 40 k 61 / 52, 512 behind 8000 47 / 44, 256 behind 4096 (32 tiles a workgroup) 35 / 38; fp8 81 / 104 and 52 / 55 (first and third).
WIDE_ROWS = 96
WIDE_TILES = 48


def _prefix_work(sizes, lens, G: int, Hkv: int, rt: int, each: int, put) -> PrefixWork:
    """each: 32-key tiles of a workgroup, at most (where MAX_SPLITS parts do: 1 sequence of 8 / 1 heads behind 100 k keys has 64
    workgroups, 17.4 us in fp8 for a floor of 5.5)."""
    items: List[List[int]] = []
    counts, at = [], 0
    for n, p in zip(sizes, lens):
        blocks, tiles = -(-n * G // (16 * rt)), -(-p // 32)
        parts = min(MAX_SPLITS, -(-tiles // each))
        share = -(-tiles // parts) * 32 if parts else 0
        parts = -(-p // share) if parts else 0
        # (the blocks of one range of keys side by side: they read the same bytes)
        items += [[at, n, i, j * share, min(p, (j + 1) * share), j, 0, 0] for j in range(parts) for i in range(blocks)]
        counts += [parts] * n
        at += n
    _need(len(items) <= 65535, "too many groups")
    return PrefixWork(rt, max(counts, default=0), put(items, (8,)), put(counts, ()), len(items))


def shared_prefix_plan(group_sizes: Sequence[int], prefix_lens: Sequence[int], num_heads: int, num_kv_heads: int,
                       device="cuda") -> SharedPrefixPlan:
    """Plan of a decode batch whose sequences come in groups: group_sizes[g] sequences in a row of the batch share their first
    prefix_lens[g] tokens (0: nothing shared). A program makes it when the batch changes, not for every step; it holds for any
    lengths of the sequences and for all layers."""
    sizes, lens = [int(n) for n in group_sizes], [int(n) for n in prefix_lens]
    _need(len(sizes) == len(lens), "a prefix length for each group")
    _need(all(n >= 1 for n in sizes) and all(0 <= n < 1 << 30 for n in lens), "groups of at least one sequence, lengths of at least 0")
    _need(num_kv_heads >= 1 and num_heads >= 1 and num_heads % num_kv_heads == 0, "num_heads must be a multiple of num_kv_heads")
    G = num_heads // num_kv_heads

    def put(rows, width):
        return torch.tensor(rows, dtype=torch.int32).reshape(-1, *width).to(device)

    def tiles(rt, wgs):   # of a workgroup, where so many have them all (or nearly: no more than twice the mean)
        work = [(num_kv_heads * -(-n * G // (16 * rt)), -(-p // 32)) for n, p in zip(sizes, lens)]
        lo = max(4, -(-sum(b * t for b, t in work) // wgs))
        hi = 2 * lo
        while lo < hi:
            mid = (lo + hi) // 2
            lo, hi = (lo, mid) if sum(b * -(-t // mid) for b, t in work) <= wgs else (mid + 1, hi)
        return lo

    most = max([n * G for n, p in zip(sizes, lens) if p > 0], default=0)
    rt = 1 if most <= 16 else 2
    each = tiles(rt, PREFIX_WGS)
    wide = None
    if most >= WIDE_ROWS and each >= WIDE_TILES:
        wide = _prefix_work(sizes, lens, G, num_kv_heads, 8, tiles(8, PREFIX_WGS), put)
    if each >= PREFIX_LONG:
        each = tiles(rt, PREFIX_WGS * 2)
    work = _prefix_work(sizes, lens, G, num_kv_heads, rt, each, put)
    prefix = [p for n, p in zip(sizes, lens) for _ in range(n)]
    return SharedPrefixPlan(len(prefix), num_heads, num_kv_heads, work, wide, max(work.slots, wide.slots if wide else 0),
                            put(prefix, ()), tuple(sizes), tuple(lens), min(lens, default=0), max(lens, default=0))


def shared_prefix_attention(q: torch.Tensor, kv: Union[QuantKVCache, Tuple[torch.Tensor, torch.Tensor]], block_tables: torch.Tensor,
                            seq_lens: torch.Tensor, plan: SharedPrefixPlan, scale: float, num_splits: Optional[int] = None,
                            workspace: Optional[DecodeWorkspace] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Decode attention q [B, Hq, D] bf16 of sequences in groups with a common prefix, whose keys are read once for the group: of a
    group, the first prefix_lens[g] keys of every sequence are those of its first sequence's table, the rest its own table's; a
    sequence shorter than the prefix sees as much of it as it is long. kv: a `QuantKVCache`, or the bf16 pages (k, v) [NB, Hkv, bs,
    D]. num_splits: parts of the keys behind the prefix, as in `quant_decode_attention`. A workspace needs these and B plan.slots."""
    quant = isinstance(kv, QuantKVCache)
    if quant:
        kc, vc, (nb, Hkv, bs, D), fmt = kv.k, kv.v, kv.dims, kv.code
    else:
        kc, vc = kv
        if kc.dtype is not torch.bfloat16 or vc.dtype is not torch.bfloat16:
            raise TypeError("kv must be a QuantKVCache or bfloat16 pages")
        if not (kc.dim() == 4 and kc.shape == vc.shape and kc.is_contiguous() and vc.is_contiguous()
                and kc.get_device() == vc.get_device() and kc.data_ptr() % 16 == 0 and vc.data_ptr() % 16 == 0):
            raise ValueError("pages must be contiguous [NB, Hkv, bs, D] alike")
        (nb, Hkv, bs, D), fmt = kc.shape, KV_BF16
        if D not in (64, 128) or bs < TILE or bs % TILE or nb < 1 or Hkv < 1:
            raise ValueError(f"heads of 64 or 128 numbers in pages of a multiple of {TILE} tokens")
    dev, index = kc.device, kc.get_device()
    B, Hq, W, q_stride, t_stride = _check_queries(q, Hkv, D, index, dev, block_tables, seq_lens, q.shape[0])
    if plan.num_seqs != B or plan.num_heads != Hq or plan.num_kv_heads != Hkv:
        raise ValueError(f"the plan is for {plan.num_seqs} sequences of {plan.num_heads} / {plan.num_kv_heads} heads, not {B} of {Hq} / {Hkv}")
    if plan.prefix.get_device() != index or plan.longest > W * bs:
        raise ValueError(f"the plan is on {plan.prefix.device}, the cache on {dev}" if plan.prefix.device != dev
                         else "a prefix is longer than the tables")
    out, out_stride = _check_out(out, q)
    blocks = -(-Hq // Hkv // 16)
    shares, least = _shares(num_splits, B, Hkv * blocks, W * bs - plan.shortest)
    work = plan.work if quant or plan.wide is None else plan.wide
    if work.n + shares * blocks > 65535:
        raise ValueError("at most 65535 parts (for each 16 query heads of a kv head)")
    if B == 0:
        return out
    if not _native(kc):
        at = 0
        for n, p in zip(plan.group_sizes, plan.prefix_lens):
            for b in range(at, at + n):
                L = max(0, min(int(seq_lens[b]), W * bs))
                out[b] = 0
                if L > 0:
                    front, back = _any_rows_ref(kv, block_tables[at], 0, min(p, L)), _any_rows_ref(kv, block_tables[b], min(p, L), L)
                    k, v = (torch.cat(x) for x in zip(front, back))
                    out[b] = _attend(q[b:b + 1], k, v, torch.tensor([L - 1], device=q.device), scale)[0].to(q.dtype)
            at += n
        return out
    keep, po, pl = _parts(workspace, (B * work.slots + shares) * Hq, D, dev) if work.slots or shares > B else (None, 0, 0)
    kernels().shared_prefix_attention(fmt, q.data_ptr(), q_stride, kc.data_ptr(), vc.data_ptr(), ptr(kv.scales if quant else None),
                                      block_tables.data_ptr(), t_stride, W, seq_lens.data_ptr(), po, pl,
                                      out.data_ptr(), out_stride, B, Hq, Hkv, D, bs, nb, scale, work.items.data_ptr(),
                                      work.n, plan.prefix.data_ptr(), work.counts.data_ptr(), work.slots,
                                      work.row_tiles, shares, least, stream_ptr())
    return out
