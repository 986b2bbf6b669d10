"""Plain restatements, in numpy and 64 bits, of the operators that serve several sequences: the paged 4-bit cache's layout
and quantizer, attention over it, block maps, beam selection and the reorderings. Written from the formulas of
include/b200q.h, element by element where that is simplest."""
import numpy as np

NO_SLOT = 0xFFFFFFFF


def tile_bytes(dim):
    return 18 * dim


def code_place(which, dim):
    """(byte, shift) of every code in a tile: arrays [16, dim]; which 0: K, 1: V."""
    t, e = np.meshgrid(np.arange(16), np.arange(dim), indexing="ij")
    b, j = e // 32, e % 32
    plane = b // 4
    nb = np.minimum(4, dim // 32 - 4 * plane)
    word, byte = j % 16 // 4, j % 4
    if which == 0:
        at = (t * 4 + word) * nb + b % 4
    else:
        at = (((t // 8 * 2 + t % 2) * 4 + word) * 4 + t // 2 % 4) * nb + b % 4
    return which * 8 * dim + plane * 1024 + at * 4 + byte, j // 16 * 4


def scale_place(which, dim):
    t, b = np.meshgrid(np.arange(16), np.arange(dim // 32), indexing="ij")
    return 16 * dim + which * dim + (t * (dim // 32) + b) * 2


def quantize(x):
    """GGUF Q4_0 of FP32 rows [..., dim]: (codes, FP16 scales), each step rounded to FP32; non-finite blocks: NaN scale."""
    b = np.asarray(x, np.float32).reshape(-1, 32)
    bad = ~np.isfinite(b).all(1)
    b = np.where(bad[:, None] | (b == 0), np.float32(0), b)  # (the search for the largest starts from +0)
    d = (b[np.arange(len(b)), np.abs(b).argmax(1)] / np.float32(-8)).astype(np.float32)
    with np.errstate(divide="ignore", over="ignore", invalid="ignore"):
        inv = np.where(d != 0, np.float32(1) / d, np.float32(0)).astype(np.float32)
        codes = np.clip((b * inv[:, None] + np.float32(8.5)), 0, 15).astype(np.uint8)
        d16 = d.astype(np.float16)
    d16[bad] = np.nan
    return codes.reshape(np.shape(x)), d16.reshape(*np.shape(x)[:-1], -1)


class Pool:
    """A layer's pages as numpy bytes [n_pages, n_kv, tiles, tile bytes]."""

    def __init__(self, n_pages, page, n_kv, dim, fill=0):
        self.n_pages, self.page, self.n_kv, self.dim = n_pages, page, n_kv, dim
        self.bytes = np.full((n_pages, n_kv, page // 16, tile_bytes(dim)), fill, np.uint8)

    def store(self, slots, k, v):
        for i, s in enumerate(np.asarray(slots).astype(np.int64) & NO_SLOT):
            if s == NO_SLOT or s // self.page >= self.n_pages:
                continue
            p, t, r = s // self.page, s % self.page // 16, s % 16
            for which, x in ((0, k), (1, v)):
                codes, d = quantize(x[i].reshape(self.n_kv, self.dim))
                at, shift = code_place(which, self.dim)
                at, shift = at[r], shift[r]
                tile = self.bytes[p, :, t]
                for e in range(self.dim):
                    keep = tile[:, at[e]] & (0xF0 if shift[e] == 0 else 0x0F)
                    tile[:, at[e]] = keep | (codes[:, e] << shift[e])
                sp = scale_place(which, self.dim)[r]
                raw = d.view(np.uint8).reshape(self.n_kv, -1, 2)
                tile[:, sp], tile[:, sp + 1] = raw[:, :, 0], raw[:, :, 1]

    def values(self, which, page, token):
        """[n, n_kv, dim] float64 of tokens (page, place) of the pool."""
        page, token = np.asarray(page), np.asarray(token)
        tile = self.bytes[page, :, token // 16]  # n, n_kv, bytes
        at, shift = code_place(which, self.dim)
        sp = scale_place(which, self.dim)
        r = token % 16
        idx = np.arange(len(page))[:, None, None], np.arange(self.n_kv)[None, :, None]
        codes = (tile[(*idx, at[r][:, None, :])] >> shift[r][:, None, :]) & 15
        lo, hi = tile[(*idx, sp[r][:, None, :])], tile[(*idx, sp[r][:, None, :] + 1)]
        d = (lo.astype(np.uint16) | hi.astype(np.uint16) << 8).view(np.float16).astype(np.float64)
        return (codes.astype(np.float64) - 8) * np.repeat(d, 32, axis=-1)


def attention(pool, q, table, q_start, kv_len, scale, window=0):
    """(y, per-element magnitude sum p |v|, per-row (row, head) largest scale sum |q k|): float64, rows of all requests."""
    rows, n_head, dim = q.shape
    group = n_head // pool.n_kv
    y, mag, big = np.zeros(q.shape), np.zeros(q.shape), np.zeros((rows, n_head))
    for r in range(len(kv_len)):
        a, b, n = int(q_start[r]), int(q_start[r + 1]), int(kv_len[r])
        key = np.arange(n)
        pages = table[r][key // pool.page] if n else np.zeros(0, int)
        k, v = (pool.values(i, pages, key % pool.page) if n else np.zeros((0, pool.n_kv, dim)) for i in (0, 1))
        for i in range(a, b):
            pos = n - (b - a) + (i - a)
            lo = max(0, pos - window + 1) if window else 0
            if pos < 0:
                continue
            for h in range(n_head):
                kk, vv = k[lo:pos + 1, h // group], v[lo:pos + 1, h // group]
                qk = kk * q[i, h].astype(np.float64) * scale
                s = qk.sum(-1)
                p = np.exp(s - s.max())
                p /= p.sum()
                y[i, h], mag[i, h] = p @ vv, p @ np.abs(vv)
                big[i, h] = np.abs(qk).sum(-1).max()
    return y, mag, big


def block_map(past, fresh, table, page, free, cursor, n_rows):
    """(table, kv_len, q_start, slots, positions, cursor, short)."""
    table = np.array(table, np.int64)
    cap = table.shape[1] * page
    kv_len, q_start, slots, positions, short, at = [], [0], [], [], False, cursor
    for r, (p, f) in enumerate(zip(past, fresh)):
        kv = p + f
        if kv > cap:
            kv, short = cap, True
        for b in range(-(-p // page), -(-kv // page)):
            if at < len(free):
                table[r, b] = free[at]
            else:
                table[r, b], short = NO_SLOT, True
            at += 1
        kv_len.append(kv)
        q_start.append(q_start[-1] + f)
        for pos in range(p, p + f):
            s = NO_SLOT
            if pos < cap and table[r, pos // page] != NO_SLOT:
                s = table[r, pos // page] * page + pos % page
            slots.append(s)
            positions.append(pos if pos < cap else 0)
    pad = n_rows - len(slots)
    slots, positions = (slots + [NO_SLOT] * pad)[:n_rows], (positions + [0] * pad)[:n_rows]
    return table, kv_len, q_start, slots, positions, max(cursor, min(at, len(free))), short


def select(logits, scores, n_req, beams, n_out):
    """Per request a list of (score, parent, token), best first."""
    out = []
    vocab = logits.shape[1]
    for r in range(n_req):
        all_ = []
        for b in range(beams):
            x = logits[r * beams + b].astype(np.float64)
            sc = float(scores[r * beams + b])
            ok = x > -np.inf  # NaN: false
            if not np.isfinite(sc) or not ok.any() or np.isposinf(x[ok]).any():
                continue
            m = x[ok].max()
            lse = m + np.log(np.exp(x[ok] - m).sum())
            for t in np.nonzero(ok)[0]:
                all_.append((-(sc + (x[t] - lse)), b * vocab + int(t)))
        all_.sort()
        out.append([(-s, i // vocab, i % vocab) for s, i in all_[:n_out]])
    return out
