"""Host side of the paged 4-bit KV cache (include/b200q.h, "several sequences"): Q4_0 quantization of K and V rows and the
bytes of the cache's pages, for callers that fill a cache from host memory; on the device kv4_store does the same."""
from __future__ import annotations

import numpy as np

from . import kv4_page_bytes


def quantize(x: np.ndarray):
    """Q4_0 of FP32 rows [..., dim]: (codes uint8, FP16 scales [..., dim / 32]), in the format's own FP32 steps; a block
    that holds a NaN or an infinity gets a NaN scale."""
    b = np.asarray(x, np.float32).reshape(*x.shape[:-1], -1, 32)
    bad = ~np.isfinite(b).all(-1, keepdims=True)
    b = np.where(bad | (b == 0), np.float32(0), b)
    d = (np.take_along_axis(b, np.abs(b).argmax(-1)[..., None], -1) / np.float32(-8)).astype(np.float32)
    with np.errstate(divide="ignore", over="ignore", invalid="ignore"):
        inv = np.where(d != 0, np.float32(1) / d, np.float32(0)).astype(np.float32)
        codes = np.clip(b * inv + np.float32(8.5), 0, 15).astype(np.uint8)
        d16 = np.where(bad, np.float16(np.nan), d.astype(np.float16))
    return codes.reshape(x.shape), d16[..., 0]


def pack_pages(k: np.ndarray, v: np.ndarray, page: int, n_pages: int) -> np.ndarray:
    """The bytes of n_pages pages [n_pages, page bytes] that hold the tokens of k and v [tokens, n_kv, dim] in order from
    page 0 on; places behind the last token are zero."""
    tokens, n_kv, dim = k.shape
    if kv4_page_bytes(page, n_kv, dim) == 0 or tokens > page * n_pages:
        raise ValueError("a shape the cache does not take, or more tokens than the pages hold")
    nb = dim // 32
    out = []
    for x in (k, v):
        codes, d = quantize(x)
        full = np.full((page * n_pages, n_kv, dim), 8, np.uint8)
        full[:tokens] = codes
        scale = np.zeros((page * n_pages, n_kv, nb), np.float16)
        scale[:tokens] = d
        # page, head, tile, token, ...
        full = full.reshape(n_pages, page // 16, 16, n_kv, nb, 2, 4, 4).transpose(0, 3, 1, 2, 4, 5, 6, 7)
        words = full[..., 0, :, :] | full[..., 1, :, :] << 4  # page, head, tile, token, block, word, byte
        out.append((words, scale.reshape(n_pages, page // 16, 16, n_kv, nb).transpose(0, 3, 1, 2, 4)))
    lead = (n_pages, n_kv, page // 16)
    parts = []
    for which, (words, _) in enumerate(out):
        for p in range(0, nb, 4):
            w = words[..., p:p + 4, :, :].swapaxes(-3, -2)  # token, word, block, byte
            if which:  # token / 8, token % 2, word, token / 2 % 4, block, byte
                w = w.reshape(*lead, 2, 4, 2, 4, -1, 4).transpose(0, 1, 2, 3, 5, 6, 4, 7, 8)
            parts.append(np.ascontiguousarray(w).reshape(*lead, -1))
    parts += [np.ascontiguousarray(s).view(np.uint8).reshape(*lead, -1) for _, s in out]
    return np.concatenate(parts, -1).reshape(n_pages, -1)
