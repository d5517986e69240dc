"""The 4-bit KV cache on the host: the format of the engine's ``kv4`` mode, and its cache pages' bookkeeping.

A separate, NON-PARITY mode (the reference keeps K and V in f16): K and V are quantised when they are written to the cache
and attention reads the codes. One scale and zero point serve 64 neighbouring elements of a token's row of one KV head:

    lo = min(0, min x), hi = max(0, max x)
    scale = (hi - lo) / 15, rounded UP to seven significant bits (below 2^-14: to a multiple of 2^-20)
    zero = rint(-lo / scale), code = clamp(rint(x / scale) + zero, 0, 15), value = scale * (code - zero)

Seven bits times the four of ``code - zero`` fit the eleven of an f16, so an f16 holds every value exactly (next to the largest
f16 number a step that would pass it is not taken). A group of zeros has scale 0; one that holds an infinity or a NaN stands for NaN throughout.

A cache is u8 ``[pages, kv_heads, page, row_bytes(head_dim)]``. The bytes of one (page, head) are first the page's rows of codes,
``head_dim / 2`` bytes each, then its rows of 16-bit headers: the f16 scale with the zero point in its low four bits. Eight
elements e0..e7 take one little-endian 32-bit word, nibbles e0 e2 e4 e6 e1 e3 e5 e7 from the low end.
"""
from __future__ import annotations

from typing import Iterable, List, Tuple

import numpy as np

GROUP = 64
_ORDER = [0, 4, 1, 5, 2, 6, 3, 7]  # element i of a word is nibble _ORDER[i]


def groups(head_dim: int) -> int:
    return -(-head_dim // GROUP)


def row_bytes(head_dim: int) -> int:
    """Bytes of one token's row of one KV head (codes and headers)."""
    return head_dim // 2 + 2 * groups(head_dim)


def quantize(x: np.ndarray) -> Tuple[np.ndarray, np.ndarray]:
    """Rows f16 ``[..., D]`` -> codes u8 ``[..., D]`` and headers u16 ``[..., groups(D)]``, as the device makes them."""
    x = np.asarray(x, np.float16).astype(np.float32)
    d = x.shape[-1]
    codes = np.zeros(x.shape, np.uint8)
    heads = np.zeros(x.shape[:-1] + (groups(d),), np.uint16)
    for i in range(groups(d)):
        g = x[..., i * GROUP:(i + 1) * GROUP]
        bad = ~np.isfinite(g).all(-1)
        g = np.where(bad[..., None], np.float32(0), g)
        lo, hi = np.minimum(g.min(-1), np.float32(0)), np.maximum(g.max(-1), np.float32(0))
        r = (hi.astype(np.float64) - lo.astype(np.float64)) / 15  # (two f16 numbers may need 41 bits side by side)
        step = np.exp2(np.maximum(np.frexp(r)[1], -13) - 7.0)
        scale = (np.ceil(r / step) * step).astype(np.float32)
        div = np.where(scale > 0, scale, np.float32(1))
        zero = np.minimum(np.rint(-lo / div), np.float32(15))
        most = np.floor(np.float32(65504) / div)[..., None]
        q = np.clip(np.clip(np.rint(g / div[..., None]), -most, most) + zero[..., None], 0, 15)
        codes[..., i * GROUP:(i + 1) * GROUP] = np.where((bad | (scale == 0))[..., None], 0, q)
        heads[..., i] = np.where(bad, 0x7E00, scale.astype(np.float16).view(np.uint16) | zero.astype(np.uint16))
    return codes, heads


def values(codes: np.ndarray, heads: np.ndarray) -> np.ndarray:
    """What codes ``[..., D]`` and headers ``[..., groups(D)]`` stand for: f16 ``[..., D]``."""
    d = codes.shape[-1]
    scale = (heads & np.uint16(0xFFF0)).view(np.float16).astype(np.float32)
    zero = (heads & np.uint16(15)).astype(np.float32)
    wide = lambda a: np.repeat(a, GROUP, axis=-1)[..., :d]
    return ((codes.astype(np.float32) - wide(zero)) * wide(scale)).astype(np.float16)


def pack(codes: np.ndarray) -> np.ndarray:
    """Codes u8 ``[..., D]`` -> bytes u8 ``[..., D / 2]``."""
    c = codes.reshape(codes.shape[:-1] + (-1, 8)).astype(np.uint32)
    w = sum(c[..., i] << np.uint32(4 * n) for i, n in enumerate(_ORDER)).astype("<u4")
    return np.ascontiguousarray(w).view(np.uint8).reshape(codes.shape[:-1] + (codes.shape[-1] // 2,))


def unpack(rows: np.ndarray) -> np.ndarray:
    """Bytes u8 ``[..., D / 2]`` -> codes u8 ``[..., D]``."""
    w = np.ascontiguousarray(rows).view("<u4")
    c = np.stack([(w >> np.uint32(4 * n)) & np.uint32(15) for n in _ORDER], -1)
    return c.reshape(rows.shape[:-1] + (rows.shape[-1] * 2,)).astype(np.uint8)


def parts(cache: np.ndarray, head_dim: int) -> Tuple[np.ndarray, np.ndarray]:
    """Views of a C-contiguous cache u8 ``[pages, kv_heads, page, row_bytes]``: the code rows u8 ``[pages, kv_heads, page,
    D / 2]`` and the header rows u16 ``[pages, kv_heads, page, groups(D)]``."""
    n, g, p, _ = cache.shape
    flat, cut = cache.reshape(n, g, -1), p * head_dim // 2
    heads = flat.view(np.uint16)[..., cut // 2:].reshape(n, g, p, groups(head_dim))
    return flat[..., :cut].reshape(n, g, p, head_dim // 2), heads


def write(cache: np.ndarray, slots: Iterable[int], rows: np.ndarray) -> None:
    """Quantises rows f16 ``[T, kv_heads, D]`` into ``cache`` at ``slots`` (page * P + offset); a slot outside it is dropped."""
    n, _, p, _ = cache.shape
    code, head = parts(cache, rows.shape[-1])
    assert np.shares_memory(code, cache) and np.shares_memory(head, cache)
    for t, s in enumerate(slots):
        if 0 <= s < n * p:
            c, h = quantize(rows[t])
            code[s // p, :, s % p], head[s // p, :, s % p] = pack(c), h


def read(cache: np.ndarray, head_dim: int) -> np.ndarray:
    """All of a cache as f16 ``[pages, page, kv_heads, D]``: the shape of the f16 cache."""
    code, head = parts(np.ascontiguousarray(cache), head_dim)
    return np.ascontiguousarray(values(unpack(code), head).transpose(0, 2, 1, 3))


def copy_waves(pairs: Iterable[Tuple[int, int]], pages: int) -> List[List[Tuple[int, int]]]:
    """Orders page copies (source, destination) so that every one reads its source as it was before the first: a list of
    waves, each a set of copies that may run at once. A page that is written twice, a page outside the cache, or copies
    that wait for one another in a circle (two pages exchanged) are refused with ValueError."""
    left = [(int(s), int(d)) for s, d in pairs]
    for s, d in left:
        if not (0 <= s < pages and 0 <= d < pages):
            raise ValueError(f"page copy {s} -> {d}: the cache has {pages} pages")
    if len({d for _, d in left}) != len(left):
        raise ValueError("page copies: a page is written twice")
    left = [(s, d) for s, d in left if s != d]
    waves = []
    while left:
        # A page may be overwritten once no copy that is still to run reads it, this wave's included.
        read_by = {s for s, _ in left}
        now = [(s, d) for s, d in left if d not in read_by]
        if not now:
            raise ValueError("page copies: pages exchanged in a circle (copy one of them to a free page first)")
        waves.append(now)
        gone = {d for _, d in now}
        left = [(s, d) for s, d in left if d not in gone]
    return waves
